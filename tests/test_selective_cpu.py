"""The selective state space block's entry points without a GPU: refusals that
return before any HIP call, size queries, and the model's shapes."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from pathtile_amd import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libpathtile_hip.so not built (python -m pathtile_amd.build)")
    return _lib.load()


def _scan(B=2, L=5, H=8, N=16, G=1, dtype=0, ptr=4096, b_row=16, b_group=16):
    from pathtile_amd import _lib

    return _lib.ScanInputs(ptr, ptr, ptr, ptr, ptr, None, None, None, None,
                           L * H, H, L * H, H, L * b_row, b_row, b_group, L * b_row, b_row, b_group,
                           dtype, B, L, H, N, G, 1)


def test_scan_refusals(lib):
    from pathtile_amd import _lib

    def fwd(**kw):
        return lib.pt_selective_scan_fwd(ctypes.byref(_scan(**kw)), 4096, None, None, None, 0, None)

    for kw in ({"L": 0}, {"L": (1 << 30) + 1}, {"H": 0}, {"N": 0}, {"N": 65}, {"G": 0}, {"G": 3}, {"B": -1},
               {"b_group": -1}, {"b_group": 2**31}):
        assert fwd(**kw) == _lib.PT_ERR_SHAPE, kw
    assert fwd(dtype=2) == _lib.PT_ERR_CONFIG
    assert fwd(ptr=None) == _lib.PT_ERR_NULL
    assert fwd() == _lib.PT_ERR_WORKSPACE
    assert fwd(B=0) == _lib.PT_OK
    s = _scan()
    assert lib.pt_selective_scan_fwd(None, 4096, None, None, None, 0, None) == _lib.PT_ERR_NULL
    assert lib.pt_selective_scan_fwd(ctypes.byref(s), None, None, None, None, 0, None) == _lib.PT_ERR_NULL
    bwd = [4096] * 12
    assert lib.pt_selective_scan_bwd(ctypes.byref(s), *bwd[:11], None, 0, None) == _lib.PT_ERR_WORKSPACE
    bwd[5] = None  # the gradient of A
    assert lib.pt_selective_scan_bwd(ctypes.byref(s), *bwd, 1 << 30, None) == _lib.PT_ERR_NULL
    assert lib.pt_selective_scan_step(ctypes.byref(s), None, None, 2, 4096, None) == _lib.PT_ERR_NULL
    assert lib.pt_selective_scan_step(ctypes.byref(s), 4096, None, -1, 4096, None) == _lib.PT_ERR_SHAPE


def test_scan_sizes(lib):
    from pathtile_amd import _lib

    def sizes(**kw):
        out = [ctypes.c_size_t(0) for _ in range(3)]
        _lib.check(lib.pt_selective_scan_sizes(ctypes.byref(_scan(**kw)), *map(ctypes.byref, out)), "")
        return [v.value for v in out]

    B, L, H = 2, 33, 8
    ws, saved, bwd = sizes(B=B, L=L, H=H)
    bc = B * 48 * 2 * 16 * 4  # B and C of whole tiles, as the kernels read them
    assert ws == bc and saved == B * 3 * 16 * H * 4 + bc  # a state before each of three tiles
    assert bwd >= B * L * 2 * 16 * 4
    assert sizes(B=B, L=L, H=H, N=13) == [ws, saved, bwd]
    assert sizes(B=B, L=L, H=H, N=17)[1] > saved
    assert sizes(B=0)[1:] == [0, 0]
    # 64-bit sizes
    big = sizes(B=64, L=1 << 20, H=4096, N=64)
    assert big[1] > 64 * (1 << 16) * 64 * 4096 * 4


def test_conv_refusals(lib):
    from pathtile_amd import _lib

    def fwd(dtype=0, B=2, L=5, H=8, K=4, x=4096):
        return lib.pt_causal_conv_fwd(dtype, x, L * H, H, 4096, None, None, None, 4096, None,
                                      B, L, H, K, 1, None)

    for kw in ({"B": -1}, {"L": 0}, {"L": (1 << 30) + 1}, {"H": 0}, {"K": 0}, {"K": 9}):
        assert fwd(**kw) == _lib.PT_ERR_SHAPE, kw
    assert fwd(dtype=7) == _lib.PT_ERR_CONFIG
    assert fwd(x=None) == _lib.PT_ERR_NULL
    assert fwd(B=0, x=None) == _lib.PT_OK
    n = ctypes.c_size_t(0)
    assert lib.pt_causal_conv_bwd_workspace_bytes(0, 2, 5, 8, 4, ctypes.byref(n)) == _lib.PT_OK
    assert n.value >= 2 * 8 * 5 * 4
    args = [0, 4096, 40, 8] + [4096] * 10
    assert lib.pt_causal_conv_bwd(*args, 4096, n.value - 1, 2, 5, 8, 4, 1, None) == _lib.PT_ERR_WORKSPACE
    assert lib.pt_causal_conv_bwd(*args, None, n.value, 2, 5, 8, 4, 1, None) == _lib.PT_ERR_WORKSPACE
    assert lib.pt_causal_conv_step(0, 4096, 8, 4096, None, None, None, 4096, 2, 8, 4, 2, 1,
                                   None) == _lib.PT_ERR_NULL
    assert lib.pt_causal_conv_step(0, 4096, 8, 4096, None, 4096, None, 4096, 2, 8, 4, -1, 1,
                                   None) == _lib.PT_ERR_SHAPE


def test_norm_refusals(lib):
    from pathtile_amd import _lib

    def gated(dtype=0, rows=2, H=8, groups=1, x=4096):
        return lib.pt_gated_norm_fwd(dtype, x, H, 4096, H, 4096, 4096, None, rows, H, groups, 1e-5, None)

    for kw in ({"rows": -1}, {"H": 0}, {"groups": 0}, {"groups": 3}, {"H": 16385}):
        assert gated(**kw) == _lib.PT_ERR_SHAPE, kw
    assert gated(dtype=5) == _lib.PT_ERR_CONFIG
    assert gated(x=None) == _lib.PT_ERR_NULL
    assert gated(rows=0) == _lib.PT_OK

    def residual(dtype=0, res=0, rows=2, H=8, x=4096):
        return lib.pt_residual_norm_fwd(dtype, res, x, H, None, 0, None, None, 4096, 4096, 4096, None,
                                        None, rows, H, 1e-5, None)

    assert residual(H=16385) == residual(rows=-1) == _lib.PT_ERR_SHAPE
    assert residual(res=1) == residual(dtype=2) == _lib.PT_ERR_CONFIG  # a sum below x's type
    assert residual(x=None) == _lib.PT_ERR_NULL
    n = ctypes.c_size_t(0)
    assert lib.pt_residual_norm_bwd_workspace_bytes(0, 5, 8, 4, ctypes.byref(n)) == _lib.PT_ERR_CONFIG
    assert lib.pt_residual_norm_bwd_workspace_bytes(0, 5, 8, 3, ctypes.byref(n)) == _lib.PT_OK
    assert lib.pt_gated_norm_bwd(0, 4096, 8, 4096, 8, *[4096] * 6, None, 0, 2, 8, 1,
                                 None) == _lib.PT_ERR_WORKSPACE


def test_tensors_of_the_host_are_refused():
    from pathtile_amd import selective as sel

    x, w, v = torch.zeros(1, 4, 8), torch.zeros(8, 4), torch.zeros(8)
    A, bc = torch.zeros(8, 16), torch.zeros(1, 4, 16)
    for call in (lambda: sel.causal_conv(x, w), lambda: sel.causal_conv_step(x[:, 0], w, x),
                 lambda: sel.selective_scan(x, x, A, bc, bc),
                 lambda: sel.selective_scan_step(x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], x),
                 lambda: sel.gated_norm(x, x, v), lambda: sel.residual_norm(x, None, v)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


def test_model_parameters_and_cache():
    from pathtile_amd.selective_model import SelectiveModel

    model = SelectiveModel(vocab=11, hidden=32, blocks=2, state=8, taps=3, groups=2)
    block = model.blocks[0]
    assert block.in_proj.weight.shape == (128, 32) and block.in_proj.weight.dtype == torch.bfloat16
    assert block.x_proj.weight.shape == (2 + 2 * 2 * 8, 64)
    assert block.conv_weight.dtype == block.log_A.dtype == torch.float32
    step = torch.nn.functional.softplus(block.dt_bias)
    assert (step > 9e-4).all() and (step < 0.11).all()
    cache = model.new_cache(pool=3)
    assert [t.shape for t in cache.conv] == [(3, 2, 64)] * 2
    assert [t.shape for t in cache.scan] == [(3, 64, 8)] * 2
    cache.scan[0] += 1
    cache.clear(torch.tensor([2]))
    assert cache.scan[0][0].all() and not cache.scan[0][2].any()


def test_workspaces_are_aligned(lib):
    """Workspaces that are read and written by vectors are refused at odd addresses."""
    from pathtile_amd import _lib

    conv = [0, 4096, 40, 8] + [4096] * 10
    assert lib.pt_causal_conv_bwd(*conv, 4100, 1 << 20, 2, 5, 8, 4, 1, None) == _lib.PT_ERR_ALIGN
    s = ctypes.byref(_scan())
    assert lib.pt_selective_scan_fwd(s, 4096, None, None, 4112, 1 << 20, None) == _lib.PT_ERR_ALIGN
    assert lib.pt_selective_scan_fwd(s, 4096, None, 4112, 4096, 1 << 20, None) == _lib.PT_ERR_ALIGN
    assert lib.pt_selective_scan_bwd(s, *[4096] * 11, 4112, 1 << 20, None) == _lib.PT_ERR_ALIGN
