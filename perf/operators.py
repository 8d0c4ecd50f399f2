"""The operators of a selective state space block that are measured: the short
causal convolution, the selective scan, the gated norm and the residual norm,
for training, for prompts and for single tokens.

Each is there twice: in its plain form (elementary torch operations in 32
bits) and as a user calls the framework's own (``own`` true). Notation: B
sequences of L tokens, H channels, N states per channel, G groups of channels
that share their B and C, K taps.

``conv``       ``causal_conv`` (``mode`` "prompt": outputs and final state;
               "train": outputs and gradients) and ``causal_conv_step``.
``scan``       ``selective_scan`` and ``selective_scan_step``, the same modes.
``gated``      ``gated_norm``: ``rmsnorm(x * silu(gate)) * weight``.
``residual``   ``residual_norm``: post-norm, scale, residual and pre-norm.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5


def listed():
    return [
        # One new token of one sequence: launch cost only.
        dict(name="conv_step_one", op="conv", mode="step", B=1, H=256, K=4, pool=4, dtype="bf16"),
        # A chunk of ragged prompts that goes on from earlier tokens; one of
        # them is empty. Odd channels and lengths, x a slice of a projection.
        dict(name="conv_prompt_ragged", op="conv", mode="prompt", B=5, L=1021, H=1000, K=3,
             ragged=True, dtype="fp32"),
        # A layer of a training step, x one half of the input projection.
        dict(name="conv_train", op="conv", mode="train", B=8, L=2048, H=4096, K=4, ragged=False,
             dtype="bf16"),
        # One token for each of a full serving batch, states in a pool.
        dict(name="scan_step_batch", op="scan", mode="step", B=256, H=4096, N=16, G=1, pool=320,
             dtype="bf16"),
        # One long prompt: few channels to work on, many tokens.
        dict(name="scan_prompt_long", op="scan", mode="prompt", B=1, L=16384, H=2048, N=16, G=1,
             ragged=False, dtype="bf16"),
        # Ragged prompts that go on from earlier states; odd everything, two
        # groups of channels.
        dict(name="scan_prompt_ragged", op="scan", mode="prompt", B=5, L=777, H=1000, N=13, G=2,
             ragged=True, dtype="fp32"),
        # A layer of a training step.
        dict(name="scan_train", op="scan", mode="train", B=8, L=2048, H=2048, N=16, G=1,
             ragged=False, dtype="bf16"),
        # The S4ConvD model's rows, channels and states: many short sequences.
        dict(name="scan_train_rows", op="scan", mode="train", B=2048, L=48, H=128, N=64, G=1,
             ragged=False, dtype="fp32"),
        # The norm after the scan for one token of a serving batch.
        dict(name="gated_norm_step", op="gated", mode="prompt", rows=64, H=4096, groups=1,
             dtype="bf16"),
        # The same in a training step.
        dict(name="gated_norm_train", op="gated", mode="train", rows=16384, H=4096, groups=1,
             dtype="bf16"),
        # The end of a block for a few tokens, odd channels.
        dict(name="residual_norm_few", op="residual", mode="prompt", rows=77, H=1000, post=False,
             dtype="fp32", wide=True),
        # The same in a training step: both norms, the residual in 32 bits.
        dict(name="residual_norm_train", op="residual", mode="train", rows=16384, H=2048,
             post=True, dtype="bf16", wide=True),
    ]


# The largest listed cases: scanned values B L H N, elements of the others.
MOST_SCAN = 2048 * 48 * 128 * 64
MOST_ELEMENTS = 8 * 2048 * 4096
MOST_STATE = 256 * 4096 * 16


def draw(rng):
    def spread(lo, hi):
        n = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
        return max(lo, min(hi, int(n)))

    op = rng.choice(("conv", "conv", "scan", "scan", "scan", "gated", "residual"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if op in ("gated", "residual"):
        mode, H = rng.choice(("prompt", "train")), spread(64, 4096)
        rows = spread(1, min(16384, MOST_ELEMENTS // H))
        if op == "gated":
            groups = rng.choice((1, 1, 2, 4))
            return dict(op=op, mode=mode, rows=rows, H=H // groups * groups, groups=groups,
                        dtype=dtype)
        return dict(op=op, mode=mode, rows=rows, H=H, post=rng.random() < 0.5, dtype=dtype,
                    wide=rng.random() < 0.5)
    mode, H = rng.choice(("step", "prompt", "train")), spread(64, 4096)
    if op == "conv":
        K = rng.choice((2, 3, 4, 4, 4, 5, 8))
        if mode == "step":
            B = spread(1, 256)
            return dict(op=op, mode=mode, B=B, H=H, K=K, pool=B + B // 4 + 1, dtype=dtype)
        L = spread(1, 16384)
        B = spread(1, max(1, min(64, MOST_ELEMENTS // (L * H))))
        return dict(op=op, mode=mode, B=B, L=min(L, MOST_ELEMENTS // (B * H)), H=H, K=K,
                    ragged=rng.random() < 0.5, dtype=dtype)
    G = rng.choice((1, 1, 1, 2))
    H, N = H // G * G, rng.choice((8, 16, 16, 16, 13, 32, 64))
    if mode == "step":
        B = spread(1, max(1, min(256, MOST_STATE // (H * N))))
        return dict(op=op, mode=mode, B=B, H=H, N=N, G=G, pool=B + B // 4 + 1, dtype=dtype)
    L = spread(1, 16384)
    L = min(L, MOST_SCAN // (2 * H * N))
    B = spread(1, max(1, min(64, MOST_SCAN // (2 * L * H * N))))
    return dict(op=op, mode=mode, B=B, L=L, H=H, N=N, G=G, ragged=rng.random() < 0.5, dtype=dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    H, s = case["H"], {"case": case}
    if case["op"] == "gated":
        # x and gate as the scan and one half of the input projection give them
        s.update(x=normal(case["rows"], H, dtype=t),
                 gates=normal(case["rows"], 2 * H, dtype=t),
                 weight=1.0 + normal(H, scale=0.1), gy=normal(case["rows"], H, dtype=t))
        return s
    if case["op"] == "residual":
        r = torch.float32 if case["wide"] else t
        s.update(x=normal(case["rows"], H, dtype=t), residual=normal(case["rows"], H, dtype=r, scale=2.0),
                 weight=1.0 + normal(H, scale=0.1), scale=0.5 + normal(H, scale=0.1),
                 post_weight=1.0 + normal(H, scale=0.1) if case["post"] else None,
                 gy=normal(case["rows"], H, dtype=t), gr=normal(case["rows"], H, dtype=r))
        return s
    B, L = case["B"], case.get("L", 1)
    lengths = state = None
    if case["mode"] == "step":
        s["slots"] = torch.randperm(case["pool"], generator=g, device="cuda")[:B].to(torch.int32)
    elif case["ragged"]:  # from a state, lengths over the whole range, the first row empty
        lengths = (uniform(B) * (L + 1)).to(torch.int32).clamp_(max=L)
        lengths[0] = 0
        state = True
    s["lengths"] = lengths
    if case["op"] == "conv":
        K = case["K"]
        # x is one half of an input projection's output
        s.update(xz=normal(B, L, 2 * H, dtype=t), weight=normal(H, K, scale=K ** -0.5),
                 bias=normal(H, scale=0.1))
        rows = case["pool"] if case["mode"] == "step" else B if state else 0
        s["state"] = normal(rows, K - 1, H, dtype=t) if rows else None
    else:
        N, G = case["N"], case["G"]
        # B and C are parts of one projection; dt's bias puts softplus between 1e-3 and 1e-1
        step = torch.exp(uniform(H) * math.log(100.0) + math.log(1e-3))
        s.update(x=normal(B, L, H, dtype=t), dt=normal(B, L, H, dtype=t, scale=0.5),
                 bc=normal(B, L, 2 * G * N, dtype=t),
                 A=-torch.arange(1, N + 1, device="cuda") * torch.exp(normal(H, N, scale=0.1)),
                 D=1.0 + normal(H, scale=0.1), dt_bias=step + torch.log(-torch.expm1(-step)))
        rows = case["pool"] if case["mode"] == "step" else B if state else 0
        s["state"] = normal(rows, H, N) if rows else None
    if case["mode"] == "train":
        s["gy"] = normal(B, L, H, dtype=t)
    return s


def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](state, case)


# --- the framework's operators -------------------------------------------------
def _own_conv(s, case):
    from pathtile_amd import selective

    x = s["xz"][..., :case["H"]]
    if case["mode"] == "step":
        y = selective.causal_conv_step(x[:, 0], s["weight"], s["state"], s["bias"],
                                       slots=s["slots"])
        return y, s["state"]
    if case["mode"] == "prompt":
        return selective.causal_conv(x, s["weight"], s["bias"], state=s["state"],
                                     lengths=s["lengths"], return_state=True)
    given = [x, s["weight"], s["bias"]] + ([s["state"]] if s["state"] is not None else [])
    given = [v.detach().requires_grad_(True) for v in given]
    y = selective.causal_conv(*given[:3], state=given[3] if len(given) > 3 else None,
                              lengths=s["lengths"])
    return y, torch.autograd.grad(y, given, s["gy"])


def _own_scan(s, case):
    from pathtile_amd import selective

    G, N = case["G"], case["N"]
    Bm, Cm = (v.unflatten(-1, (G, N)) for v in s["bc"].split(G * N, -1))
    if case["mode"] == "step":
        y = selective.selective_scan_step(s["x"][:, 0], s["dt"][:, 0], s["A"], Bm[:, 0], Cm[:, 0],
                                          s["state"], s["D"], dt_bias=s["dt_bias"],
                                          slots=s["slots"])
        return y, s["state"]
    if case["mode"] == "prompt":
        return selective.selective_scan(s["x"], s["dt"], s["A"], Bm, Cm, s["D"],
                                        dt_bias=s["dt_bias"], state=s["state"],
                                        lengths=s["lengths"], return_state=True)
    given = [s["x"], s["dt"], s["A"], Bm, Cm, s["D"], s["dt_bias"]]
    given += [s["state"]] if s["state"] is not None else []
    given = [v.detach().requires_grad_(True) for v in given]
    y = selective.selective_scan(*given[:6], dt_bias=given[6],
                                 state=given[7] if len(given) > 7 else None, lengths=s["lengths"])
    return y, torch.autograd.grad(y, given, s["gy"])


def _own_gated(s, case):
    from pathtile_amd import selective

    gate = s["gates"][:, case["H"]:]
    if case["mode"] == "prompt":
        return selective.gated_norm(s["x"], gate, s["weight"], groups=case["groups"], eps=EPS)
    given = [v.detach().requires_grad_(True) for v in (s["x"], gate, s["weight"])]
    y = selective.gated_norm(*given, groups=case["groups"], eps=EPS)
    return y, torch.autograd.grad(y, given, s["gy"])


def _own_residual(s, case):
    from pathtile_amd import selective

    if case["mode"] == "prompt":
        return selective.residual_norm(s["x"], s["residual"], s["weight"], scale=s["scale"],
                                       post_weight=s["post_weight"], eps=EPS)
    given = [s["x"], s["residual"], s["weight"], s["scale"]]
    given += [s["post_weight"]] if case["post"] else []
    given = [v.detach().requires_grad_(True) for v in given]
    y, r = selective.residual_norm(*given[:3], scale=given[3],
                                   post_weight=given[4] if case["post"] else None, eps=EPS)
    return y, r, torch.autograd.grad((y, r), given, (s["gy"], s["gr"]))


_own = dict(conv=_own_conv, scan=_own_scan, gated=_own_gated, residual=_own_residual)


# --- the plain forms -------------------------------------------------------------
def _silu_grad(p):
    sig = torch.sigmoid(p)
    return sig * (1.0 + p * (1.0 - sig))


def _inside(lengths, L):
    """[B, L, 1]: 1 at a sequence's tokens, 0 past them."""
    return (torch.arange(L, device=lengths.device) < lengths[:, None]).float()[..., None]


def _plain_conv(s, case):
    t, w, H, K = s["xz"].dtype, s["weight"], case["H"], case["K"]
    x = s["xz"][..., :H].float()
    if case["mode"] == "step":
        at = s["slots"].long()
        window = torch.cat((s["state"][at].float(), x), 1)  # [B, K, H]
        p = (window * w.t()).sum(1) + s["bias"]
        s["state"][at] = window[:, 1:].to(t)
        return (p * torch.sigmoid(p)).to(t), s["state"]
    B, L = case["B"], case["L"]
    before = x.new_zeros(B, K - 1, H) if s["state"] is None else s["state"].float()
    padded = torch.cat((before, x), 1)
    windows = padded.unfold(1, K, 1)  # [B, L, H, K]
    p = (windows * w).sum(-1) + s["bias"]
    inside = 1.0 if s["lengths"] is None else _inside(s["lengths"], L)
    y = (p * torch.sigmoid(p) * inside).to(t)
    if case["mode"] == "prompt":
        n = torch.full((B,), L, device=x.device) if s["lengths"] is None else s["lengths"].long()
        last = n[:, None] + torch.arange(K - 1, device=x.device)
        return y, padded.gather(1, last[..., None].expand(-1, -1, H)).to(t)
    gp = s["gy"].float() * _silu_grad(p) * inside
    gw = (gp[..., None] * windows).sum((0, 1))
    ahead = torch.cat((x.new_zeros(B, K - 1, H), gp, x.new_zeros(B, K - 1, H)), 1)
    gpad = (ahead.unfold(1, K, 1) * w.flip(1)).sum(-1)  # [B, K - 1 + L, H]
    grads = [gpad[:, K - 1:].to(t), gw, gp.sum((0, 1))]
    return y, grads + ([gpad[:, :K - 1].to(t)] if s["state"] is not None else [])


def _recurrence(a, u):
    """s[l] = a[l] s[l - 1] + u[l] along the first axis, by doubling."""
    d = 1
    while d < a.shape[0]:
        u = torch.cat((u[:d], torch.addcmul(u[d:], a[d:], u[:-d])))
        a = torch.cat((a[:d], a[d:] * a[:-d]))
        d *= 2
    return u


def _channels(v, H):
    """[L, B, G, N] as [L, B, H, N]: a group's values for each of its channels."""
    return v.float().repeat_interleave(H // v.shape[-2], -2)


def _groups(v, G):
    """The sums of [L, B, H, N] over the channels of each group."""
    return v.unflatten(-2, (G, -1)).sum(-2)


def _plain_scan(s, case):
    t, A, D, H, G, N = s["x"].dtype, s["A"], s["D"], case["H"], case["G"], case["N"]
    x = s["x"].float().transpose(0, 1)  # the tokens first
    v = s["dt"].float().transpose(0, 1) + s["dt_bias"]
    delta = torch.where(v > 20.0, v, torch.log1p(torch.exp(v)))
    b, c = (_channels(m.transpose(0, 1).unflatten(-1, (G, N)), H)
            for m in s["bc"].split(G * N, -1))
    decay = torch.exp(delta[..., None] * A)  # [L, B, H, N]
    if case["mode"] == "step":
        at = s["slots"].long()
        h = decay[0] * s["state"][at] + (delta[0] * x[0])[..., None] * b[0]
        s["state"][at] = h
        return ((c[0] * h).sum(-1) + D * x[0]).to(t), s["state"]
    inside = within = 1.0
    if s["lengths"] is not None:  # past its length a sequence keeps its state
        inside = _inside(s["lengths"], case["L"]).transpose(0, 1)
        within = inside[..., None]
        decay = torch.where(within > 0, decay, 1.0)
    u = (delta * x * inside)[..., None] * b
    if s["state"] is not None:
        u[0] += decay[0] * s["state"]
    h = _recurrence(decay, u)
    y = (((c * h).sum(-1) + D * x) * inside).transpose(0, 1).to(t)
    if case["mode"] == "prompt":
        return y, h[-1].clone()
    gy = s["gy"].float().transpose(0, 1) * inside
    # gh[l] = c[l] gy[l] + decay[l + 1] gh[l + 1]
    after = torch.cat((decay[1:], torch.ones_like(decay[:1])))
    gh = _recurrence(after.flip(0), (c * gy[..., None]).flip(0)).flip(0)
    before = torch.zeros_like(h[:1]) if s["state"] is None else s["state"][None]
    gdecay = gh * torch.cat((before, h[:-1])) * decay * within
    gu = (gh * b).sum(-1) * inside
    gdelta = gu * x + (gdecay * A).sum(-1)
    gdt = gdelta * torch.sigmoid(v)
    gb = _groups(gh * (delta * x * inside)[..., None], G)
    gc = _groups(h * gy[..., None], G)
    grads = [(gu * delta + D * gy).transpose(0, 1).to(t), gdt.transpose(0, 1).to(t),
             (gdecay * delta[..., None]).sum((0, 1)), gb.transpose(0, 1).to(t),
             gc.transpose(0, 1).to(t), (gy * x).sum((0, 1)), gdt.sum((0, 1))]
    return y, grads + ([gh[0] * decay[0]] if s["state"] is not None else [])


def _plain_gated(s, case):
    t, w, H, groups = s["x"].dtype, s["weight"], case["H"], case["groups"]
    x, z = s["x"].float(), s["gates"][:, H:].float()
    sig = torch.sigmoid(z)
    u = (x * z * sig).unflatten(-1, (groups, -1))
    r = torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS)
    n = (u * r).flatten(1)
    y = (n * w).to(t)
    if case["mode"] == "prompt":
        return y
    gy = s["gy"].float()
    gn = (gy * w).unflatten(-1, (groups, -1))
    gu = (r * (gn - u * r * (gn * u * r).mean(-1, keepdim=True))).flatten(1)
    return y, [(gu * z * sig).to(t), (gu * x * _silu_grad(z)).to(t), (gy * n).sum(0)]


def _plain_residual(s, case):
    t, w, scale, post = s["x"].dtype, s["weight"], s["scale"], s["post_weight"]
    x, base = s["x"].float(), s["residual"].float()
    f = n = x
    if case["post"]:
        rx = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * rx
        f = n * post
    r = base + scale * f
    rr = torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)
    m = r * rr
    y, out = (m * w).to(t), r.to(s["residual"].dtype)
    if case["mode"] == "prompt":
        return y, out
    gy, gm = s["gy"].float(), s["gy"].float() * w
    gr = s["gr"].float() + rr * (gm - m * (gm * m).mean(-1, keepdim=True))
    gf = gr * scale
    gx = gf
    if case["post"]:
        gn = gf * post
        gx = rx * (gn - n * (gn * n).mean(-1, keepdim=True))
    grads = [gx.to(t), gr.to(out.dtype), (gy * m).sum(0), (gr * f).sum(0)]
    return y, out, grads + ([(gf * n).sum(0)] if case["post"] else [])


_plain = dict(conv=_plain_conv, scan=_plain_scan, gated=_plain_gated, residual=_plain_residual)


# --- what a pass cannot do without ------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    op, mode, H = case["op"], case["mode"], case["H"]
    train = mode == "train"
    if op == "gated":
        e = case["rows"] * H
        return {"bytes": e * size * (6 if train else 3) + 4 * H * (2 if train else 1),
                "flops": e * (38 if train else 12)}
    if op == "residual":
        e, wide = case["rows"] * H, 4 if case["wide"] else size
        n = 3 if case["post"] else 2
        # x, y (and gy, gx); residual, its sum (and their gradients)
        return {"bytes": e * (2 * size + 2 * wide) * (2 if train else 1)
                + 4 * H * n * (2 if train else 1), "flops": e * (30 if train else 10)}
    B, L = case["B"], case.get("L", 1)
    e = B * L * H
    if op == "conv":
        K = case["K"]
        par = 4 * H * (K + 1)
        if mode == "step":
            return {"bytes": e * size * (2 + 2 * (K - 1)) + par, "flops": e * (2 * K + 5)}
        ends = B * (K - 1) * H * size
        state = ends * ((1 if case["ragged"] else 0) + (0 if train else 1))
        if train:  # x, gy; y, gx
            return {"bytes": e * size * 4 + 2 * par + 2 * state, "flops": e * (6 * K + 15)}
        return {"bytes": e * size * 2 + par + state, "flops": e * (2 * K + 5)}
    N, G = case["N"], case["G"]
    bc, par = 2 * B * L * G * N * size, 4 * H * (N + 2)
    if mode == "step":
        return {"bytes": e * size * 3 + bc + par + 8 * B * H * N, "flops": e * (7 * N + 12)}
    state = 4 * B * H * N * ((1 if case["ragged"] else 0) + (0 if train else 1))
    if train:  # x, dt, gy; y, gx, gdt
        return {"bytes": e * size * 6 + 2 * bc + 2 * par + 2 * state, "flops": e * (20 * N + 30)}
    return {"bytes": e * size * 3 + bc + par + state, "flops": e * (7 * N + 12)}


# --- the definition in 64 bits -----------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    given = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v
             for k, v in s.items()}
    with torch.set_grad_enabled(case["mode"] == "train"):
        got = dict(conv=_exact_conv, scan=_exact_scan, gated=_exact_gated,
                   residual=_exact_residual)[case["op"]](given, case)
    return got


def _leaf(v, train):
    return v.clone().requires_grad_(True) if train else v


def _exact_conv(s, case):
    train, K, w, bias = case["mode"] == "train", case["K"], s["weight"], s["bias"]
    x, w, bias = (_leaf(v, train) for v in (s["xz"][..., :case["H"]], w, bias))
    B, L, H = x.shape
    state = s["state"]
    if case["mode"] == "step":
        rows = s["slots"].tolist()
        pool, ys = state.clone(), []
        for i, at in enumerate(rows):
            seen = torch.cat((state[at], x[i]))  # K tokens
            p = bias + sum(w[:, j] * seen[j] for j in range(K))
            ys.append(torch.nn.functional.silu(p))
            pool[at] = seen[1:]
        return torch.stack(ys), pool
    if state is None:
        state = torch.zeros(B, K - 1, H, dtype=x.dtype, device=x.device)
    state = _leaf(state, train)
    seen = torch.cat((state, x), 1)
    p = bias + sum(w[:, j] * seen[:, j:j + L] for j in range(K))
    n = [L] * B if s["lengths"] is None else s["lengths"].tolist()
    keep = torch.zeros(B, L, 1, dtype=x.dtype, device=x.device)
    for i, k in enumerate(n):
        keep[i, :k] = 1.0
    y = torch.nn.functional.silu(p) * keep
    if train:
        of = [x, w, bias] + ([state] if s["state"] is not None else [])
        return y.detach(), list(torch.autograd.grad(y, of, s["gy"]))
    return y, torch.stack([seen[i, k:k + K - 1] for i, k in enumerate(n)])


def _exact_scan(s, case):
    train, G, N, H = case["mode"] == "train", case["G"], case["N"], case["H"]
    names = ("x", "dt", "A", "D", "dt_bias")
    x, dt, A, D, dt_bias = (_leaf(s[k], train) for k in names)
    b, c = (_leaf(v.unflatten(-1, (G, N)), train) for v in s["bc"].split(G * N, -1))
    B, L = x.shape[:2]
    delta = torch.nn.functional.softplus(dt + dt_bias)
    first = s["state"]
    if case["mode"] == "step":
        first = first[s["slots"].long()]
    elif first is None:
        first = torch.zeros(B, H, N, dtype=x.dtype, device=x.device)
    first = _leaf(first, train)
    h = first.unflatten(1, (G, H // G))  # [B, G, channels of a group, N]
    A_g = A.unflatten(0, (G, H // G))
    ys = []
    keep = None if s["lengths"] is None else s["lengths"][:, None, None, None]
    steps = zip(*(v.unbind(1) for v in (x, delta, b, c)))
    for l, (x_l, d_l, b_l, c_l) in enumerate(steps):
        x_l, d_l = (v.unflatten(1, (G, H // G)).unsqueeze(-1) for v in (x_l, d_l))
        new = torch.exp(d_l * A_g) * h + d_l * x_l * b_l.unsqueeze(2)
        h = new if keep is None else torch.where(keep > l, new, h)
        ys.append(torch.matmul(h, c_l.unsqueeze(-1)).flatten(1))
    y = torch.stack(ys, 1) + D * x
    if keep is not None:
        y = torch.where(torch.arange(L, device=x.device)[:, None] < s["lengths"][:, None, None],
                        y, 0.0)
    if train:
        of = [x, dt, A, b, c, D, dt_bias] + ([first] if s["state"] is not None else [])
        return y.detach(), list(torch.autograd.grad(y, of, s["gy"]))
    if case["mode"] == "step":
        pool = s["state"].clone()
        pool[s["slots"].long()] = h.flatten(1, 2)
        return y[:, 0], pool
    return y, h.flatten(1, 2)


def _norm64(v, n=1):
    u = v.unflatten(-1, (n, -1))
    return (u / (u.square().mean(-1, keepdim=True) + EPS).sqrt()).flatten(-2)


def _exact_gated(s, case):
    train, H = case["mode"] == "train", case["H"]
    x, z, w = (_leaf(v, train) for v in (s["x"], s["gates"][:, H:], s["weight"]))
    y = _norm64(x * torch.nn.functional.silu(z), case["groups"]) * w
    return (y.detach(), list(torch.autograd.grad(y, (x, z, w), s["gy"]))) if train else y


def _exact_residual(s, case):
    train = case["mode"] == "train"
    names = ("x", "residual", "weight", "scale") + (("post_weight",) if case["post"] else ())
    given = {k: _leaf(s[k], train) for k in names}
    f = _norm64(given["x"]) * given["post_weight"] if case["post"] else given["x"]
    r = given["residual"] + given["scale"] * f
    y = _norm64(r) * given["weight"]
    if not train:
        return y, r
    grads = torch.autograd.grad((y, r), list(given.values()), (s["gy"], s["gr"]))
    return y.detach(), r.detach(), list(grads)
