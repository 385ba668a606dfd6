"""Workloads of `neumesh_amd.ops`: dense layers with a fused epilogue and the gated linear recurrence, each forward and as a
training step, at sizes from one sample to whole batches of rays.

`own = False` computes a workload with elementary torch operations in 32 bits, `own = True` through `neumesh_amd.ops`.
"""
import math

import numpy as np
import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_ACTS = ("none", "relu", "softplus", "sigmoid", "silu", "gelu_tanh")
_DENSE_FLOPS_MAX = 6 * 131072 * 256 * 256      # of a drawn layer: the largest listed one
_DENSE_ELEMS_MAX = 131072 * 256
_SCAN_ELEMS_MAX = 4 * 16384 * 512


def _dense(name, M, K, N, dtype, act, residual, train):
    return dict(name=name, op="dense", M=M, K=K, N=N, dtype=dtype, act=act, bias=True, residual=residual, train=train)


def _scan(name, B, T, D, dtype, gate, shared, blend, reverse, packed, states, h0, train):
    return dict(name=name, op="scan", B=B, T=T, D=D, dtype=dtype, gate=gate, shared=shared, blend=blend, reverse=reverse,
                packed=packed, states=states, h0=h0, train=train)


def listed():
    return [
        # one sample through a hidden layer: a probe or a picked point, latency only
        _dense("dense_one_row", 1, 256, 256, "fp16", "softplus", False, False),
        # the colour network's first layer over a batch of rays (512 rays x 128 samples; 207 embedded inputs: odd rows)
        _dense("dense_color_in_bf16", 65536, 207, 256, "bf16", "relu", False, False),
        # a wider residual block, bound by the matrix pipe
        _dense("dense_wide_bf16", 16384, 1024, 1024, "bf16", "gelu_tanh", True, False),
        # a geometry layer of a training step in the framework's own arithmetic
        _dense("dense_geo_train_fp32", 65536, 256, 256, "fp32", "softplus", False, True),
        # the same batch twice as large in 16 bits, with a residual
        _dense("dense_train_bf16", 131072, 256, 256, "bf16", "softplus", True, True),
        # embedded geometry inputs (177 wide) of a ragged batch into an odd head
        _dense("dense_ragged_train_fp16", 10007, 177, 131, "fp16", "silu", False, True),
        # one step of a batch of carried states
        _scan("scan_step", 512, 1, 256, "fp32", "fp32", False, False, False, False, True, True, False),
        # colours of 32768 rays composited far to near (127 mid-points, one opacity for three channels)
        _scan("scan_rays_rgb", 32768, 127, 3, "fp32", "fp32", True, True, True, False, False, True, False),
        # 32 feature channels of a training batch of rays, 16-bit features under 32-bit opacities
        _scan("scan_rays_train", 2048, 127, 32, "bf16", "fp32", True, True, True, False, False, False, True),
        # rays that kept different numbers of samples, packed one after the other (empty ones among them)
        _scan("scan_packed_train", 8192, 96, 32, "fp32", "fp32", False, False, False, True, True, True, True),
        # long sequences, a gate per channel
        _scan("scan_long_bf16", 4, 16384, 512, "bf16", "bf16", False, False, False, False, True, False, False),
        # one very long sequence in training
        _scan("scan_long_train", 1, 32768, 256, "bf16", "bf16", False, False, False, False, True, True, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        dtype, train = rng.choice(("fp32", "bf16", "fp16")), rng.random() < 0.5
        K, N, M = _log_int(rng, 1, 1024), _log_int(rng, 1, 1024), _log_int(rng, 1, 131072)
        if rng.random() < 0.3:
            K, N = max(8, K // 16 * 16), max(8, N // 16 * 16)
        scale = _SIZE[dtype] // 2
        M = max(1, min(M, _DENSE_FLOPS_MAX // ((6 if train else 2) * K * N * scale), _DENSE_ELEMS_MAX // (max(K, N) * scale)))
        # ReLU's derivative jumps at 0, where the last bit of a 32-bit sum decides: training passes take the smooth ones
        act = rng.choice([n for n in _ACTS if not (train and n == "relu")])
        return dict(op="dense", M=M, K=K, N=N, dtype=dtype, act=act, bias=rng.random() < 0.8,
                    residual=rng.random() < 0.4, train=train)
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    D, T = _log_int(rng, 1, 1024), _log_int(rng, 1, 32768)
    cap = _SCAN_ELEMS_MAX // (4 * _SIZE[dtype] // 2)
    T = max(1, min(T, cap // D))
    B = max(1, min(_log_int(rng, 1, 32768), cap // (D * T)))
    return dict(op="scan", B=B, T=T, D=D, dtype=dtype, gate=rng.choice((dtype, "fp32")), shared=rng.random() < 0.4,
                blend=rng.random() < 0.5, reverse=rng.random() < 0.5, packed=rng.random() < 0.3, states=rng.random() < 0.7,
                h0=rng.random() < 0.5, train=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    s = dict(case=case)
    if case["op"] == "dense":
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = normal(M, K)
        s["weight"] = normal(N, K, scale=K ** -0.5)
        s["bias"] = normal(N, scale=0.1) if case["bias"] else None
        s["residual"] = normal(M, N) if case["residual"] else None
        s["g"] = normal(M, N) if case["train"] else None
        s["beta"] = 100.0
        return s
    B, T, D = case["B"], case["T"], case["D"]
    gdt, Dg = _DT[case["gate"]], 1 if case["shared"] else D
    if case["packed"]:
        # B sequences of T steps on average, cut at random places; a few rows of padding behind the last one
        cuts = np.sort(np.random.default_rng(seed).integers(0, B * T + 1, B - 1))
        cu = np.concatenate([[0], cuts, [B * T]]).astype(np.int32)
        s["cu"], s["max_len"] = torch.from_numpy(cu).cuda(), int(np.diff(cu).max())
        lead = (B * T + 5,)
    else:
        s["cu"], s["max_len"] = None, T
        lead = (B, T)
    s["x"] = normal(*lead, D)
    if case["blend"]:       # opacities: mostly empty space, some of it solid
        s["gate"] = torch.sigmoid(normal(*lead, Dg, scale=2.0, dtype=torch.float32) - 3.0).to(gdt)
    else:                   # retention, from forgetting at once to nearly for ever
        s["gate"] = torch.sigmoid(normal(*lead, Dg, scale=2.0, dtype=torch.float32) + 2.0).to(gdt)
    s["h0"] = normal(B, D, dtype=torch.float32) if case["h0"] else None
    s["g"] = normal(*lead, D) if case["train"] and case["states"] else None
    s["g_last"] = normal(B, D, dtype=torch.float32) if case["train"] else None
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["op"] == "dense":
        return _dense_own(case, state) if own else _dense_plain(case, state)
    return _scan_own(case, state) if own else _scan_plain(case, state)


def _leaf(t):
    return None if t is None else t.detach().requires_grad_(True)


def _grads(outputs, cotangents, named):
    pairs = [(o, c) for o, c in zip(outputs, cotangents) if c is not None]
    names = [n for n, t in named.items() if t is not None]
    got = torch.autograd.grad([o for o, _ in pairs], [named[n] for n in names], [c for _, c in pairs])
    return {"d_" + n: g for n, g in zip(names, got)}


def _dense_own(case, s):
    from neumesh_amd import ops
    if not case["train"]:
        with torch.no_grad():
            return ops.dense(s["x"], s["weight"], s["bias"], s["residual"], activation=case["act"], beta=s["beta"])
    t = {n: _leaf(s[n]) for n in ("x", "weight", "bias", "residual")}
    y = ops.dense(t["x"], t["weight"], t["bias"], t["residual"], activation=case["act"], beta=s["beta"])
    return {"y": y.detach(), **_grads([y], [s["g"]], t)}


def _scan_own(case, s):
    from neumesh_amd import ops
    kw = dict(cu_seqlens=s["cu"], reverse=case["reverse"], blend=case["blend"], need_states=case["states"])
    if not case["train"]:
        with torch.no_grad():
            h, last = ops.gated_scan(s["gate"], s["x"], s["h0"], **kw)
        return {"states": h, "last": last} if case["states"] else {"last": last}
    t = {n: _leaf(s[n]) for n in ("gate", "x", "h0")}
    h, last = ops.gated_scan(t["gate"], t["x"], t["h0"], **kw)
    grads = _grads([h, last], [s["g"], s["g_last"]], t)
    return {**({"states": h.detach()} if case["states"] else {}), "last": last.detach(), **grads}


# ------------------------------------------------------------------------------------------------ plain forms
def _act(name, z, beta):
    """act(z) and act'(z)."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "softplus":
        e = torch.exp(-(beta * z).abs())
        return z.clamp(min=0) + torch.log1p(e) / beta, torch.sigmoid(beta * z)
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    sg = torch.sigmoid(z)
    return (sg, sg * (1 - sg)) if name == "sigmoid" else (z * sg, sg * (1 + z * (1 - sg)))


def _dense_plain(case, s):
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    h, d = _act(case["act"], z, s["beta"])
    y = (h if s["residual"] is None else h + s["residual"].float()).to(s["x"].dtype)
    if not case["train"]:
        return y
    dz = s["g"].float() * d
    out = {"y": y, "d_x": (dz @ w).to(y.dtype), "d_weight": (dz.t() @ x).to(y.dtype)}
    if s["bias"] is not None:
        out["d_bias"] = dz.sum(0).to(y.dtype)
    if s["residual"] is not None:
        out["d_residual"] = s["g"]
    return out


def _doubling(r, u, first, max_len):
    """h_i = r_i h_{i-1} + u_i over the rows of u [L,D], r [L,D] or [L,1]; rows marked in `first` [L,1] start anew."""
    r, h, k = torch.where(first, torch.zeros_like(r), r), u, 1
    while k < max_len:
        h = torch.cat([h[:k], h[k:] + r[k:] * h[:-k]])
        r = torch.cat([r[:k], r[k:] * r[:-k]])
        k *= 2
    return h


def _scan_plain(case, s):
    B, T, D, blend = case["B"], case["T"], case["D"], case["blend"]
    x, a = s["x"].float().reshape(-1, D), s["gate"].float()
    a = a.reshape(-1, a.shape[-1])
    L, dev = x.shape[0], x.device
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(B + 1, device=dev) * T
    seq = torch.bucketize(torch.arange(L, device=dev), cu[1:], right=True)     # sequence of every row, B: padding
    live = (seq < B)[:, None]
    filled = cu[1:] > cu[:-1]
    lo, hi = cu[:-1][filled], cu[1:][filled] - 1
    first_rows, last_rows = (hi, lo) if case["reverse"] else (lo, hi)
    turn = (lambda t: t.flip(0)) if case["reverse"] else (lambda t: t)
    mark = torch.zeros((L, 1), dtype=torch.bool, device=dev)
    first, final = mark.clone(), mark.clone()
    first[first_rows], final[last_rows] = True, True
    h0 = s["h0"] if s["h0"] is not None else torch.zeros((B, D), device=dev)
    r = 1 - a if blend else a
    start = torch.zeros((L, D), device=dev)
    start[first_rows] = h0[filled]
    u = (a * x if blend else x) + torch.where(first, r * start, torch.zeros_like(start))
    u = torch.where(live, u, torch.zeros_like(u))
    h = turn(_doubling(turn(r), turn(u), turn(first | ~live), s["max_len"]))
    last = h0.clone()
    last[filled] = h[last_rows]
    states = h.to(s["x"].dtype).reshape(s["x"].shape)
    if not case["train"]:
        return {"states": states, "last": last} if case["states"] else {"last": last}
    g = s["g"].float().reshape(-1, D).clone() if s["g"] is not None else torch.zeros((L, D), device=dev)
    g = torch.where(live, g, torch.zeros_like(g))
    g[last_rows] += s["g_last"][filled]
    step = -1 if case["reverse"] else 1
    lam = _doubling(turn(torch.roll(r, -step, 0)).flip(0), turn(g).flip(0), turn(final | ~live).flip(0), s["max_len"])
    lam = turn(lam.flip(0))
    before = torch.where(first, start, torch.roll(h, step, 0))
    da = torch.where(live, lam * (x - before if blend else before), torch.zeros_like(lam))
    if case["shared"]:
        da = da.sum(1, keepdim=True)
    dx = a * lam if blend else lam
    out = {"states": states} if case["states"] else {}
    out.update(last=last, d_gate=da.to(s["gate"].dtype).reshape(s["gate"].shape),
               d_x=torch.where(live, dx, torch.zeros_like(dx)).to(s["x"].dtype).reshape(s["x"].shape))
    if s["h0"] is not None:
        dh0 = s["g_last"].clone()
        dh0[filled] = (r * lam)[first_rows]
        out["d_h0"] = dh0
    return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "dense":
        M, K, N = case["M"], case["K"], case["N"]
        elems = M * K + N * K + M * N + N * case["bias"] + M * N * case["residual"]
        if case["train"]:       # in: g; out: gradients of x, the weight, the bias and the residual
            elems += M * N + M * K + N * K + N * case["bias"] + M * N * case["residual"]
        return {"bytes": e * elems, "flops": (6 if case["train"] else 2) * M * N * K}
    B, T, D = case["B"], case["T"], case["D"]
    L, Dg = B * T, 1 if case["shared"] else D
    gate = _SIZE[case["gate"]] * L * Dg
    total = e * L * D * (1 + case["states"]) + gate + 4 * B * D * (1 + case["h0"])
    if case["train"]:
        total += e * L * D * (1 + case["states"]) + gate + 4 * B * D * (1 + case["h0"])
    return {"bytes": total, "flops": (8 if case["train"] else 2) * L * D}


# ------------------------------------------------------------------------------------------------ 64-bit definitions
def exact(case, seed):
    s = prepare(case, seed)
    return _dense_exact(case, s) if case["op"] == "dense" else _scan_exact(case, s)


def _dense_exact(case, s):
    x, w = s["x"].double(), s["weight"].double()
    z = torch.mm(x, w.t().contiguous())
    if s["bias"] is not None:
        z += s["bias"].double()
    b, act = s["beta"], case["act"]
    if act == "none":
        y, d = z, torch.ones_like(z)
    elif act == "relu":
        y, d = torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).double()
    elif act == "softplus":
        y, d = torch.logaddexp(b * z, torch.zeros_like(z)) / b, 1 / (1 + torch.exp(-b * z))
    elif act == "sigmoid":
        y = 1 / (1 + torch.exp(-z))
        d = y / (1 + torch.exp(z))
    elif act == "silu":
        q = 1 / (1 + torch.exp(-z))
        y, d = z * q, q + z * q / (1 + torch.exp(z))
    else:       # z sigma(2 v), v = sqrt(2 / pi) (z + 0.044715 z^3)
        v2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        q = 1 / (1 + torch.exp(-v2))
        y, d = z * q, q + z * q / (1 + torch.exp(v2)) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
    if s["residual"] is not None:
        y = y + s["residual"].double()
    if not case["train"]:
        return y
    dz = s["g"].double() * d
    out = {"y": y, "d_x": torch.mm(dz, w), "d_weight": torch.mm(dz.t().contiguous(), x)}
    if s["bias"] is not None:
        out["d_bias"] = dz.sum(0)
    if s["residual"] is not None:
        out["d_residual"] = s["g"].double()
    return out


def _scan_exact(case, s):
    """Step by step over sequences padded to the longest one."""
    B, T, D, blend, rev = case["B"], case["T"], case["D"], case["blend"], case["reverse"]
    dev, tmax = s["x"].device, s["max_len"]
    if case["packed"]:
        lens = (s["cu"][1:] - s["cu"][:-1]).long()
        base = s["cu"][:-1].long()
    else:
        lens = torch.full((B,), T, device=dev)
        base = torch.arange(B, device=dev) * T
    if B * tmax * D > 3 * 10 ** 8 or tmax > 200000:
        return None
    i = torch.arange(tmax, device=dev)
    valid = i[None] < lens[:, None]                                             # [B,tmax] in the order of the recurrence
    row = base[:, None] + (lens[:, None] - 1 - i[None] if rev else i[None])
    row = torch.where(valid, row, 0).t().contiguous()                           # [tmax,B]
    valid = valid.t().contiguous()[..., None]
    x2, a2 = s["x"].reshape(-1, D), s["gate"].reshape(-1, s["gate"].shape[-1])
    h = s["h0"].double() if s["h0"] is not None else torch.zeros((B, D), dtype=torch.float64, device=dev)
    prev = torch.empty((tmax, B, D), dtype=torch.float64, device=dev)
    for k in range(tmax):
        prev[k] = h
        a, x = a2[row[k]].double(), x2[row[k]].double()
        n = h + a * (x - h) if blend else a * h + x
        h = torch.where(valid[k], n, h)
    out = {}
    sel = valid[..., 0]

    def scatter(t, like):
        flat = torch.zeros((like.numel() // like.shape[-1], t.shape[-1]), dtype=torch.float64, device=dev)
        flat[row[sel]] = t[sel]
        return flat.reshape(like.shape)

    if case["states"]:
        nxt = torch.cat([prev[1:], h[None]])
        out["states"] = scatter(nxt, s["x"])
        del nxt
    out["last"] = h
    if not case["train"]:
        return out
    g2 = s["g"].reshape(-1, D) if s["g"] is not None else None
    lam = s["g_last"].double()
    dx = torch.empty_like(prev)
    da = torch.empty((tmax, B, s["gate"].shape[-1]), dtype=torch.float64, device=dev)
    for k in range(tmax - 1, -1, -1):
        a, x = a2[row[k]].double(), x2[row[k]].double()
        here = lam + (g2[row[k]].double() if g2 is not None else 0.0)
        step = here * (x - prev[k]) if blend else here * prev[k]
        da[k] = step.sum(-1, keepdim=True) if case["shared"] else step
        dx[k] = a * here if blend else here
        lam = torch.where(valid[k], (1 - a) * here if blend else a * here, lam)
    out["d_gate"], out["d_x"] = scatter(da, s["gate"]), scatter(dx, s["x"])
    if s["h0"] is not None:
        out["d_h0"] = lam
    return out
