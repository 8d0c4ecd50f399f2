"""The operators of the selective state space block on the GPU (marked
``gpu``) against plain loops in 64 bits, at the sizes, layouts and masks where
tiles, runs and rows end: outputs, final states and every gradient; the token
steps against the prompts; gradients also against differences.

Bars, of the 2-norm of the 64-bit result. FP32 (unit roundoff u = 6e-8): a
convolution or norm rounds some ten times and sums by trees or short chains:
1e-6. A scan's state rounds twice a token and forgets as it goes; over the up
to 300 tokens here sqrt(600) u = 1.5e-6, and its gradients do so twice more:
1e-5. Parameter gradients add up to 1e4 products in chains of at most a few
hundred: 1e-5. BF16 outputs are rounded once, by at most 2^-8 of each value (a
significand of 8 bits), and FP32's error besides: 4e-3."""

from __future__ import annotations

import itertools

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

BF16_TOL = 4e-3
EPS = 1e-5


@pytest.fixture(scope="module")
def sel():
    from pathtile_amd import selective

    return selective


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    return float((got - want).norm() / want.norm().clamp_min(1e-30))


def _check(got, want, tol, what):
    bar = BF16_TOL if got.dtype == torch.bfloat16 else tol
    err = _rel(got, want)
    assert err <= bar, f"{what}: {err:.2e} > {bar:.0e}"


def _gen(*key):
    return torch.Generator().manual_seed(sum((i + 1) * 7919 * int(k) for i, k in enumerate(key)))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def _wide(t):
    """The same values as a slice of a wider tensor."""
    room = torch.full((*t.shape[:-1], t.shape[-1] + 5), float("nan"), dtype=t.dtype, device=t.device)
    room[..., 3:-2] = t
    return room[..., 3:-2]


def _grads(outs, inputs, gouts):
    return torch.autograd.grad(outs, inputs, gouts)


# --- plain forms in 64 bits ------------------------------------------------------
def _conv64(x, w, bias, state, lengths, silu):
    B, L, H = x.shape
    K = w.shape[1]
    state = x.new_zeros(B, K - 1, H) if state is None else state
    seen = torch.cat((state, x), 1)
    p = 0 if bias is None else bias
    p = p + sum(w[:, j] * seen[:, j:j + L] for j in range(K))
    y = F.silu(p) if silu else p
    n = [L] * B if lengths is None else [min(max(int(k), 0), L) for k in lengths]
    keep = torch.stack([(torch.arange(L, device=x.device) < k).double() for k in n])[..., None]
    return y * keep, torch.stack([seen[b, k:k + K - 1] for b, k in enumerate(n)])


def _scan64(x, dt, A, b, c, D, dt_bias, state, lengths, softplus):
    B, L, H = x.shape
    G, N = b.shape[-2:]
    s = x.new_zeros(B, H, N) if state is None else state
    v = dt if dt_bias is None else dt + dt_bias
    d = F.softplus(v, threshold=50) if softplus else v
    n = torch.tensor([L] * B if lengths is None else [min(max(int(k), 0), L) for k in lengths],
                     device=x.device)
    ys = []
    for t in range(L):
        bt, ct = (m[:, t].repeat_interleave(H // G, 1) for m in (b, c))  # [B, H, N]
        new = torch.exp(d[:, t, :, None] * A) * s + (d[:, t] * x[:, t])[..., None] * bt
        inside = (n > t)[:, None, None]
        s = torch.where(inside, new, s)
        y = (ct * s).sum(-1) + (0 if D is None else D * x[:, t])
        ys.append(torch.where(inside[..., 0], y, torch.zeros_like(y)))
    return torch.stack(ys, 1), s


def _rms64(u, groups=1):
    v = u.unflatten(-1, (groups, -1))
    return (v / (v.square().mean(-1, keepdim=True) + EPS).sqrt()).flatten(-2)


def _double(ts):
    return [None if t is None else t.detach().double().requires_grad_(True) for t in ts]


def _leaves(ts):
    return [None if t is None else t.detach().requires_grad_(True) for t in ts]


def _some(ts):
    return [t for t in ts if t is not None]


# --- causal convolution ------------------------------------------------------------
CONV = [
    # B, L, H, K, bias, state, lengths, silu
    (1, 1, 1, 4, True, False, None, True),
    (2, 3, 8, 4, True, True, None, True),
    (3, 17, 7, 3, False, True, (17, 0, 5), True),
    (2, 64, 64, 1, True, False, (64, 63), True),
    (2, 65, 24, 2, True, True, (1, 65), False),
    (4, 130, 100, 4, True, True, (0, 2, 129, 130), True),
    (1, 300, 130, 8, True, True, (299,), True),
    (2, 33, 513, 5, False, False, None, True),
    (5, 16, 256, 7, True, True, (3, 2, 1, 0, 16), True),
    (2, 40, 16, 6, True, True, (-3, 99), True),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", CONV)
def test_causal_conv(sel, case, dtype):
    B, L, H, K, has_bias, has_state, lens, silu = case
    g = _gen(B, L, H, K)
    x = _wide(_randn(g, B, L, H, dtype=dtype))
    w, bias = _randn(g, H, K), _randn(g, H) if has_bias else None
    state = _randn(g, B, K - 1, H, dtype=dtype) if has_state else None
    gy, gs = _randn(g, B, L, H, dtype=dtype), _randn(g, B, K - 1, H, dtype=dtype)
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    act = "silu" if silu else None

    want_in = _double((x, w, bias, state))
    wy, ws = _conv64(*want_in, lens, silu)
    y, s = sel.causal_conv(x, w, bias, activation=act, state=state, lengths=lengths,
                           return_state=True)
    _check(y, wy, 1e-6, "y")
    assert torch.equal(s.double(), ws.detach())  # tokens, not computed values
    got_in = _leaves((x, w, bias, state))
    y2, s2 = sel.causal_conv(*got_in[:3], activation=act, state=got_in[3], lengths=lengths,
                             return_state=True)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    got = _grads((y2, s2) if K > 1 else y2, _some(got_in), (gy, gs) if K > 1 else gy)
    want = _grads((wy, ws) if K > 1 else wy, _some(want_in),
                  (gy.double(), gs.double()) if K > 1 else gy.double())
    for a, b, name in zip(got, want, ("x", "w", "bias", "state")):
        _check(a, b, 1e-5 if a.dtype == torch.float32 and name in ("w", "bias") else 2e-6, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,K", [(64, 4), (100, 3), (7, 2), (24, 8), (16, 1)])
def test_causal_conv_step_goes_on_from_a_prompt(sel, H, K, dtype):
    g = _gen(H, K)
    B, L, pool = 3, 9, 6
    x, w, bias = _randn(g, B, L, H, dtype=dtype), _randn(g, H, K), _randn(g, H)
    whole = sel.causal_conv(x, w, bias)
    _, s = sel.causal_conv(x[:, :4], w, bias, return_state=True)
    slots = torch.tensor([4, 0, 3], dtype=torch.int32, device="cuda")
    state = torch.full((pool, K - 1, H), 7.0, dtype=dtype, device="cuda")
    state[slots.long()] = s
    for t in range(4, L):
        y = sel.causal_conv_step(x[:, t], w, state, bias, slots=slots)
        assert torch.equal(y, whole[:, t])
    rest = [i for i in range(pool) if i not in (4, 0, 3)]
    assert (state[rest] == 7.0).all()


# --- scan ----------------------------------------------------------------------------
SCAN = [
    # B, L, H, N, G, D, dt_bias, state, lengths, softplus
    (1, 1, 1, 1, 1, False, False, False, None, True),
    (2, 15, 64, 16, 1, True, True, True, None, True),
    (2, 16, 64, 16, 1, True, True, True, (16, 0), True),
    (3, 17, 65, 16, 1, True, True, True, (17, 1, 16), True),
    (1, 300, 100, 16, 2, True, True, True, None, True),
    (2, 33, 130, 13, 1, False, True, True, (32, 33), True),
    (4, 50, 96, 8, 3, True, False, False, (0, 49, 50, 7), False),
    (2, 48, 128, 64, 1, True, True, True, None, True),
    (1, 100, 70, 32, 5, True, True, True, (65,), True),
    (2, 21, 66, 33, 1, True, True, False, (21, 20), True),
    (1, 64, 7, 64, 7, True, True, True, (40,), True),
    (2, 40, 64, 17, 1, True, True, True, (-5, 400), True),
    (1, 290, 64, 4, 1, True, True, True, (273,), True),
]


def _scan_case(case, dtype, wide=True):
    B, L, H, N, G, has_d, has_bias, has_state, lens, softplus = case
    g = _gen(B, L, H, N, G)
    strided = _wide if wide else (lambda t: t)
    x = strided(_randn(g, B, L, H, dtype=dtype))
    dt = strided(_randn(g, B, L, H, dtype=dtype))
    if not softplus:  # steps themselves, not negative
        dt = strided((dt.float().abs() * 0.1).to(dtype))
    A = -torch.exp(_randn(g, H, N, scale=0.5)) * torch.arange(1, N + 1, device="cuda") * 0.2
    bc = _randn(g, B, L, 2, G, N, dtype=dtype)
    b, c = (strided(bc[:, :, i].flatten(2)).unflatten(-1, (G, N)) for i in (0, 1))
    D = _randn(g, H) if has_d else None
    dt_bias = _randn(g, H, scale=0.5) - 3.0 if has_bias else None
    state = _randn(g, B, H, N) if has_state else None
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    return (x, dt, A, b, c, D, dt_bias, state), lens, lengths, softplus, g


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", SCAN)
def test_selective_scan(sel, case, dtype, wide):
    ins, lens, lengths, softplus, g = _scan_case(case, dtype, wide)
    x = ins[0]
    gy, gs = _randn(g, *x.shape, dtype=dtype), _randn(g, x.shape[0], *ins[2].shape)
    want_in = _double(ins)
    wy, ws = _scan64(*want_in, lens, softplus)

    def run(x, dt, A, b, c, D, dt_bias, state):
        return sel.selective_scan(x, dt, A, b, c, D, dt_bias=dt_bias, softplus=softplus,
                                  state=state, lengths=lengths, return_state=True)

    y, s = run(*ins)
    _check(y, wy, 1e-5, "y")
    _check(s, ws, 1e-5, "state")
    got_in = _leaves(ins)
    y2, s2 = run(*got_in)
    got = _grads((y2, s2), _some(got_in), (gy, gs))
    want = _grads((wy, ws), _some(want_in), (gy.double(), gs.double()))
    names = [n for n, t in zip(("x", "dt", "A", "B", "C", "D", "dt_bias", "state"), ins)
             if t is not None]
    for a, b, name in zip(got, want, names):
        _check(a, b, 1e-5, name)
    again = run(*_leaves(ins))
    assert torch.equal(again[0], y2) and torch.equal(again[1], s2)


@pytest.mark.parametrize("B,L,H,N", [(1, 1000, 64, 16), (1, 4097, 130, 16), (2, 2500, 64, 33)])
def test_selective_scan_long(sel, B, L, H, N):
    """Sequences that a launch may split; the chain is longer than the short
    ones' by sqrt(4097 / 300) = 3.7: 4e-5."""
    ins, lens, lengths, softplus, g = _scan_case((B, L, H, N, 1, True, True, True,
                                                  (L - 5, L)[-B:], True), torch.float32)
    ins = list(ins)
    ins[6] = ins[6] - 2.0  # smaller steps: long memory
    gy, gs = _randn(g, B, L, H), _randn(g, B, H, N)
    want_in = _double(ins)
    wy, ws = _scan64(*want_in, lens, softplus)
    got_in = _leaves(ins)
    y, s = sel.selective_scan(*got_in[:6], dt_bias=got_in[6], state=got_in[7], lengths=lengths,
                              return_state=True)
    _check(y, wy, 4e-5, "y")
    _check(s, ws, 4e-5, "state")
    for a, b, name in zip(_grads((y, s), got_in, (gy, gs)),
                          _grads((wy, ws), want_in, (gy.double(), gs.double())),
                          ("x", "dt", "A", "B", "C", "D", "dt_bias", "state")):
        _check(a, b, 4e-5, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_places_are_not_read(sel, dtype):
    """Infinities and NaN past a sequence's end reach nothing."""
    ins, lens, lengths, _, g = _scan_case((3, 40, 72, 16, 1, True, True, True, (23, 0, 40), True),
                                          dtype, False)
    gy = _randn(g, *ins[0].shape, dtype=dtype)
    w, bias = _randn(g, 72, 4), _randn(g, 72)

    def run(poison):
        bad = [t.clone() for t in (*ins[:2], *ins[3:5], gy)]
        for t, v in zip(bad, itertools.cycle((float("nan"), float("inf"), -float("inf")))):
            for b, n in enumerate(lens):
                t[b, n:] = v if poison else 0.0
        x, dt, b, c, gyb = bad
        given = _leaves((x, dt, ins[2], b, c, ins[5], ins[6], ins[7]))
        y, s = sel.selective_scan(*given[:6], dt_bias=given[6], state=given[7], lengths=lengths,
                                  return_state=True)
        out = [y, s, *_grads((y, s), given, (gyb, torch.ones_like(s)))]
        conv = _leaves((x, w, bias))
        y, s = sel.causal_conv(*conv, lengths=lengths, return_state=True)
        return out + [y, s, *_grads((y, s), conv, (gyb, torch.ones_like(s)))]

    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b)
        assert torch.isfinite(a).all()


def test_nan_tokens_stay_in_their_channel(sel):
    ins, *_ = _scan_case((1, 20, 64, 16, 1, True, True, False, None, True), torch.float32, False)
    x, dt = ins[0].clone(), ins[1].clone()
    x[0, 5, 3] = float("nan")
    dt[0, 7, 9] = float("nan")
    y = sel.selective_scan(x, dt, *ins[2:6], dt_bias=ins[6])
    bad = torch.isnan(y[0])
    want = torch.zeros_like(bad)
    want[5:, 3] = True
    want[7:, 9] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,N,G", [(64, 16, 1), (100, 13, 2), (7, 64, 7), (256, 8, 1), (66, 3, 3),
                                   (128, 32, 2)])
def test_selective_scan_step_goes_on_from_a_prompt(sel, H, N, G, dtype):
    ins, _, _, _, g = _scan_case((3, 9, H, N, G, True, True, False, None, True), dtype)
    x, dt, A, b, c, D, dt_bias, _ = ins
    want, ws = _scan64(*_double(ins), None, True)
    _, s = sel.selective_scan(x[:, :4], dt[:, :4], A, b[:, :4], c[:, :4], D, dt_bias=dt_bias,
                              return_state=True)
    slots = torch.tensor([4, 0, 3], dtype=torch.int32, device="cuda")
    state = torch.full((6, H, N), 7.0, device="cuda")
    state[slots.long()] = s
    for t in range(4, 9):
        y = sel.selective_scan_step(x[:, t], dt[:, t], A, b[:, t], c[:, t], state, D,
                                    dt_bias=dt_bias, slots=slots)
        _check(y, want[:, t], 1e-5, f"token {t}")
    _check(state[slots.long()], ws, 1e-5, "state")
    assert (state[[1, 2, 5]] == 7.0).all()


def test_steps_of_rows_without_a_sequence(sel):
    g = _gen(5)
    B, H, N, K, pool = 4, 40, 16, 4, 3
    x, dt, b, c = (_randn(g, B, n) for n in (H, H, N, N))
    A, w = -_randn(g, H, N).abs(), _randn(g, H, K)
    slots = torch.tensor([-1, 2, 3, 2**31 - 1], dtype=torch.int32, device="cuda")
    scan, conv = _randn(g, pool, H, N), _randn(g, pool, K - 1, H)
    before = scan.clone(), conv.clone()
    y = sel.selective_scan_step(x, dt, A, b, c, scan, slots=slots)
    z = sel.causal_conv_step(x, w, conv, slots=slots)
    for out, now, was in ((y, scan, before[0]), (z, conv, before[1])):
        assert (out[[0, 2, 3]] == 0).all() and (out[1] != 0).any()
        assert torch.equal(now[:2], was[:2]) and not torch.equal(now[2], was[2])


def test_chunks_of_a_prompt(sel):
    ins, *_ = _scan_case((2, 100, 64, 16, 1, True, True, False, None, True), torch.float32, False)
    x, dt, A, b, c, D, dt_bias, _ = ins
    whole, last = sel.selective_scan(x, dt, A, b, c, D, dt_bias=dt_bias, return_state=True)
    s, parts = None, []
    for lo, hi in ((0, 1), (1, 32), (32, 99), (99, 100)):
        y, s = sel.selective_scan(x[:, lo:hi], dt[:, lo:hi], A, b[:, lo:hi], c[:, lo:hi], D,
                                  dt_bias=dt_bias, state=s, return_state=True)
        parts.append(y)
    _check(torch.cat(parts, 1), whole, 1e-6, "y")
    _check(s, last, 1e-6, "state")


def _differences(f, ins, grads, gouts, h):
    """Directional derivatives by central differences against the gradients."""
    g = _gen(17)
    for i, (t, grad) in enumerate(zip(ins, grads)):
        v = _randn(g, *t.shape)
        v = v / v.norm() * (grad.double().norm() / grad.double().norm())
        v = 0.5 * v + 0.5 * (grad / grad.norm()).float()  # along the gradient too

        def loss(sign):
            moved = [a + sign * h * v if j == i else a for j, a in enumerate(ins)]
            return sum((o.double() * q.double()).sum() for o, q in zip(f(*moved), gouts))

        want = float((loss(1) - loss(-1)) / (2 * h))
        got = float((grad.double() * v.double()).sum())
        # second order in h, and the outputs' rounding over 2 h
        assert abs(got - want) <= 5e-3 * abs(want) + 1e-3, (i, got, want)


def test_gradients_against_differences(sel):
    ins, *_ = _scan_case((1, 24, 20, 16, 2, True, True, True, None, True), torch.float32, False)
    g = _gen(3)
    gouts = _randn(g, 1, 24, 20), _randn(g, 1, 20, 16)

    def scan(x, dt, A, b, c, D, dt_bias, state):
        return sel.selective_scan(x, dt, A, b, c, D, dt_bias=dt_bias, state=state,
                                  return_state=True)

    given = _leaves(ins)
    _differences(scan, ins, _grads(scan(*given), given, gouts), gouts, 1e-2)

    ins = _randn(g, 2, 12, 16), _randn(g, 16, 4), _randn(g, 16), _randn(g, 2, 3, 16)
    gouts = _randn(g, 2, 12, 16), _randn(g, 2, 3, 16)

    def conv(x, w, bias, state):
        return sel.causal_conv(x, w, bias, state=state, return_state=True)

    given = _leaves(ins)
    _differences(conv, ins, _grads(conv(*given), given, gouts), gouts, 1e-2)

    ins = _randn(g, 6, 24), _randn(g, 6, 24), _randn(g, 24)
    gouts = (_randn(g, 6, 24),)

    def gated(x, gate, w):
        return (sel.gated_norm(x, gate, w, groups=2),)

    given = _leaves(ins)
    _differences(gated, ins, _grads(gated(*given), given, gouts), gouts, 1e-2)

    ins = tuple(_randn(g, 6, 24) for _ in range(2)) + tuple(_randn(g, 24) for _ in range(3))
    gouts = _randn(g, 6, 24), _randn(g, 6, 24)

    def residual(x, r, w, post, scale):
        return sel.residual_norm(x, r, w, post_weight=post, scale=scale)

    given = _leaves(ins)
    _differences(residual, ins, _grads(residual(*given), given, gouts), gouts, 1e-2)


# --- norms ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,H,groups", [
    (1, 1, 1), (3, 7, 1), (5, 8, 1), (70, 64, 2), (9, 100, 4), (33, 512, 1), (4, 513, 1),
    (65, 1000, 5), (2, 1024, 1), (3, 1025, 1), (6, 4096, 1), (2, 4100, 1), (3, 16384, 1),
    (2, 32768, 2), (2100, 40, 5),
])
def test_gated_norm(sel, rows, H, groups, dtype):
    g = _gen(rows, H, groups)
    x, z = _wide(_randn(g, rows, H, dtype=dtype)), _randn(g, rows, 2 * H, dtype=dtype)[:, H:]
    w, gy = 1 + _randn(g, H, scale=0.2), _randn(g, rows, H, dtype=dtype)
    want_in = _double((x, z, w))
    want = _rms64(want_in[0] * F.silu(want_in[1]), groups) * want_in[2]
    got_in = _leaves((x, z, w))
    y = sel.gated_norm(*got_in, groups=groups)
    assert torch.equal(y, sel.gated_norm(x, z, w, groups=groups))
    _check(y, want, 1e-6, "y")
    for a, b, name in zip(_grads(y, got_in, gy), _grads(want, want_in, gy.double()), "xzw"):
        # one channel: u / |u| has no slope but for eps, what is left is rounding
        if H // groups > 1:
            _check(a, b, 1e-5 if name == "w" else 2e-6, name)


@pytest.mark.parametrize("dtype,wide", [(torch.float32, True), (torch.bfloat16, True),
                                        (torch.bfloat16, False)])
@pytest.mark.parametrize("post,scaled,given", list(itertools.product((False, True), repeat=3)))
@pytest.mark.parametrize("rows,H", [(3, 7), (70, 64), (5, 513), (65, 1000), (2, 2048), (3, 4100),
                                    (2, 16384)])
def test_residual_norm(sel, rows, H, post, scaled, given, dtype, wide):
    g = _gen(rows, H, post, scaled, given)
    rt = torch.float32 if wide or dtype == torch.float32 else dtype
    x = _wide(_randn(g, rows, H, dtype=dtype))
    r = _wide(_randn(g, rows, H, dtype=rt, scale=2.0)) if given else None
    w = 1 + _randn(g, H, scale=0.2)
    p = 1 + _randn(g, H, scale=0.2) if post else None
    s = 0.5 + _randn(g, H, scale=0.2) if scaled else None
    out_t = rt if given else dtype
    gy, gr = _randn(g, rows, H, dtype=dtype), _randn(g, rows, H, dtype=out_t)
    want_in = _double((x, r, w, p, s))
    f = _rms64(want_in[0]) * want_in[3] if post else want_in[0]
    f = f * want_in[4] if scaled else f
    wr = f + want_in[1] if given else f
    wy = _rms64(wr) * want_in[2]
    got_in = _leaves((x, r, w, p, s))
    y, out = sel.residual_norm(*got_in[:3], post_weight=got_in[3], scale=got_in[4])
    assert y.dtype == dtype and out.dtype == out_t
    _check(y, wy, 1e-6, "y")
    _check(out, wr, 1e-6, "sum")
    names = [n for n, t in zip(("x", "residual", "weight", "post_weight", "scale"), got_in)
             if t is not None]
    for a, b, name in zip(_grads((y, out), _some(got_in), (gy, gr)),
                          _grads((wy, wr), _some(want_in), (gy.double(), gr.double())), names):
        _check(a, b, 1e-5, name)


def test_norms_of_one_output(sel):
    """Only one of the two outputs has a gradient."""
    g = _gen(2)
    x, r, w = _randn(g, 5, 32), _randn(g, 5, 32), _randn(g, 32)
    for i in (0, 1):
        got_in, want_in = _leaves((x, r, w)), _double((x, r, w))
        wr = want_in[0] + want_in[1]
        want = (_rms64(wr) * want_in[2], wr)[i].square().sum()
        got = sel.residual_norm(*got_in)[i].square().sum()
        n = 3 - i
        for a, b in zip(torch.autograd.grad(got, got_in[:n]), torch.autograd.grad(want, want_in[:n])):
            _check(a, b, 1e-5, f"output {i}")


def test_norms_of_rows_of_zeros_and_large_values(sel):
    x = torch.zeros(4, 96, device="cuda")
    x[1], x[2, 5] = 1e18, 3e-20
    w = torch.ones(96, device="cuda")
    y, s = sel.residual_norm(x, None, w)
    want = _rms64(x.double())
    assert torch.equal(s, x) and torch.isfinite(y).all()
    assert float((y.double() - want).abs().max()) <= 1e-6
    assert (sel.gated_norm(x, torch.zeros_like(x), w) == 0).all()


# --- in a program ----------------------------------------------------------------------
def test_other_streams(sel):
    ins, *_ = _scan_case((2, 64, 128, 13, 1, True, True, True, None, True), torch.float32)
    x, dt, A, b, c, D, dt_bias, state = ins
    want = sel.selective_scan(x, dt, A, b, c, D, dt_bias=dt_bias, state=state)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        late = x * 1.0  # produced on the stream that the call uses
        got = sel.selective_scan(late, dt, A, b, c, D, dt_bias=dt_bias, state=state)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


def test_steps_in_a_graph(sel):
    g = _gen(23)
    B, H, N, K = 4, 64, 16, 4
    x, dt, b, c, z = (_randn(g, B, n, dtype=torch.bfloat16) for n in (H, H, N, N, H))
    A, w, nw = -_randn(g, H, N).abs(), _randn(g, H, K), torch.ones(H, device="cuda")
    conv, scan = torch.zeros(B, K - 1, H, dtype=torch.bfloat16, device="cuda"), torch.zeros(
        B, H, N, device="cuda")

    def token():
        u = sel.causal_conv_step(x, w, conv)
        return sel.gated_norm(sel.selective_scan_step(u, dt, A, b, c, scan), z, nw)

    token()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        token()
    torch.cuda.current_stream().wait_stream(stream)
    with torch.cuda.graph(graph):
        out = token()
    conv.zero_(), scan.zero_()
    want = [token().clone() for _ in range(3)]
    conv.zero_(), scan.zero_()
    for i in range(3):
        x.add_(0)  # eager work between replays
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


def test_offsets_past_32_bits(sel):
    """A tensor of more than 2^31 values: its last tokens against a call on
    them alone."""
    H, K = 2048, 4
    L = 2**31 // H + 100
    x = torch.randn(1, 4096, H, device="cuda", dtype=torch.bfloat16).repeat(1, L // 4096 + 1, 1)[:, :L]
    w = torch.randn(H, K, device="cuda")
    y, s = sel.causal_conv(x, w, return_state=True)
    want = sel.causal_conv(x[:, -200:], w)
    assert torch.equal(y[:, -190:], want[:, -190:]) and torch.equal(s, x[:, -3:])
    del y, want
    rows = x.view(-1, H)
    nw = torch.ones(H, device="cuda")
    assert torch.equal(sel.gated_norm(rows, rows, nw)[-50:], sel.gated_norm(rows[-50:], rows[-50:], nw))
    del x, rows
    N, pool = 64, 2**31 // (H * 64) + 3
    scan = torch.zeros(pool, H, N, device="cuda")
    slots = torch.tensor([pool - 1], dtype=torch.int32, device="cuda")
    u, bc = torch.randn(1, H, device="cuda"), torch.randn(1, N, device="cuda")
    A = -torch.rand(H, N, device="cuda")
    small = torch.zeros(1, H, N, device="cuda")
    for _ in range(2):
        assert torch.equal(sel.selective_scan_step(u, u, A, bc, bc, scan, slots=slots),
                           sel.selective_scan_step(u, u, A, bc, bc, small))
    assert torch.equal(scan[-1], small[0]) and not scan[0].any()


def test_no_tokens_and_no_rows(sel):
    w, A = torch.randn(8, 4, device="cuda"), -torch.rand(8, 16, device="cuda")
    for B, L in ((2, 0), (0, 5)):
        x, bc = torch.zeros(B, L, 8, device="cuda"), torch.zeros(B, L, 16, device="cuda")
        state = torch.randn(B, 8, 16, device="cuda")
        y, s = sel.selective_scan(x, x, A, bc, bc, state=state, return_state=True)
        assert y.shape == x.shape and torch.equal(s, state)
        last = torch.randn(B, 3, 8, device="cuda")
        y, s = sel.causal_conv(x, w, state=last, return_state=True)
        assert y.shape == x.shape and torch.equal(s, last)
    e = torch.zeros(0, 8, device="cuda")
    assert sel.causal_conv_step(e, w, torch.zeros(0, 3, 8, device="cuda")).shape == (0, 8)
    assert sel.gated_norm(e, e, w[:, 0]).shape == (0, 8)
    given = _leaves((e, e, torch.ones(8, device="cuda")))
    grads = torch.autograd.grad(sel.gated_norm(*given).sum(), given)
    assert (grads[2] == 0).all()


def test_refusals(sel):
    x, w = torch.zeros(2, 5, 8, device="cuda"), torch.zeros(8, 4, device="cuda")
    A, bc = torch.zeros(8, 16, device="cuda"), torch.zeros(2, 5, 16, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    vec = torch.zeros(8, device="cuda")
    bad = [
        lambda: sel.causal_conv(x.cpu(), w),
        lambda: sel.causal_conv(x.half(), w),
        lambda: sel.causal_conv(x[0], w),
        lambda: sel.causal_conv(x, w[:7]),
        lambda: sel.causal_conv(x, w.bfloat16()),
        lambda: sel.causal_conv(x, torch.zeros(8, 9, device="cuda")),
        lambda: sel.causal_conv(x, w, activation="gelu"),
        lambda: sel.causal_conv(x, w, state=torch.zeros(2, 4, 8, device="cuda")),
        lambda: sel.causal_conv(x, w, state=torch.zeros(2, 3, 8, device="cuda").bfloat16()),
        lambda: sel.causal_conv(x, w, lengths=n.float()),
        lambda: sel.causal_conv(x, w, lengths=n[:1]),
        lambda: sel.causal_conv(x, w, lengths=n.cpu()),
        lambda: sel.causal_conv_step(x[:, 0], w, torch.zeros(1, 3, 8, device="cuda")),
        lambda: sel.causal_conv_step(x[:, 0], w, torch.zeros(2, 8, 3, device="cuda").mT),
        lambda: sel.causal_conv_step(x[:, 0], w, torch.zeros(2, 3, 8, device="cuda"), slots=n.long()),
        lambda: sel.selective_scan(x, x[:, :4], A, bc, bc),
        lambda: sel.selective_scan(x, x, A[:, :0], bc[..., :0], bc[..., :0]),
        lambda: sel.selective_scan(x, x, torch.zeros(8, 65, device="cuda"), bc, bc),
        lambda: sel.selective_scan(x, x, A, bc[..., :8], bc),
        lambda: sel.selective_scan(x, x, A, bc, bc.bfloat16()),
        lambda: sel.selective_scan(x, x, A, bc.view(2, 5, 1, 16).expand(2, 5, 3, 16),
                                   bc.view(2, 5, 1, 16).expand(2, 5, 3, 16)),
        lambda: sel.selective_scan(x, x, A, bc, bc, vec[:4]),
        lambda: sel.selective_scan(x, x, A, bc, bc, state=torch.zeros(2, 16, 8, device="cuda")),
        lambda: sel.selective_scan_step(x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0],
                                        torch.zeros(2, 8, 16, device="cuda").bfloat16()),
        lambda: sel.gated_norm(x, x[..., :4], vec),
        lambda: sel.gated_norm(x, x, vec, groups=3),
        lambda: sel.gated_norm(x, x.bfloat16(), vec),
        lambda: sel.residual_norm(x, x.bfloat16(), vec),
        lambda: sel.residual_norm(x, x[:, :1], vec),
        lambda: sel.residual_norm(x, None, vec, scale=vec[:1]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_no_second_order(sel):
    x = torch.randn(1, 4, 8, device="cuda", requires_grad=True)
    y = sel.causal_conv(x, torch.randn(8, 4, device="cuda"))
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 0.1)])
def test_model_prompts_steps_and_training(dtype, tol):
    """Chunks of prompts and single tokens give the logits of whole sequences
    (in BF16 to a few roundings of the linear layers, whose shapes differ),
    and a training step lowers the loss."""
    from pathtile_amd.selective_model import SelectiveModel

    torch.manual_seed(0)
    model = SelectiveModel(vocab=50, hidden=64, blocks=2, groups=2, dtype=dtype).cuda()
    tokens = torch.randint(0, 50, (3, 40), device="cuda")
    with torch.no_grad():
        whole = model(tokens).double()

    def close(got, want):
        assert float((got.double() - want).norm() / want.norm()) <= tol

    cache, slots = model.new_cache(pool=5), torch.tensor([3, 0, 4], dtype=torch.int32, device="cuda")
    n = torch.tensor([20, 7, 13], dtype=torch.int32, device="cuda")
    at = torch.arange(3, device="cuda")
    close(model.prompt(tokens[:, :20], cache, slots, n), whole[at, n.long() - 1])
    more = torch.stack([tokens[i, k:k + 5] for i, k in enumerate(n.tolist())])
    close(model.prompt(more, cache, slots), whole[at, n.long() + 4])
    for t in range(5, 9):
        step = torch.stack([tokens[i, k + t] for i, k in enumerate(n.tolist())])
        close(model.step(step, cache, slots), whole[at, n.long() + t])
    cache.clear(slots)
    close(model.prompt(tokens, cache, slots), whole[:, -1])

    opt = torch.optim.SGD(model.parameters(), lr=0.05)

    def loss():
        logits = model(tokens[:, :-1]).float().flatten(0, 1)
        return F.cross_entropy(logits, tokens[:, 1:].flatten())

    first = loss()
    first.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    opt.step()
    assert loss().item() < first.item()
