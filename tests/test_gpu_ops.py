"""neumesh_amd.ops against plain 64-bit forms: dense layers (forward, gradients) and the gated linear recurrence, at the sizes, strides, masks and
orders where they can go wrong.  Tolerances are elementwise bounds from the arithmetic (unit roundoff u = 2^-24 of the fp32 sums, eps / 2 of
the output type), computed beside each reference."""
import math

import numpy as np
import pytest
import torch

from neumesh_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -23            # one fp32 operation inside a matrix instruction may truncate: a whole unit in the last place
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half of the smallest subnormal: what rounding may lose near zero."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def close(got, want, bound, what):
    got, want, bound = got.detach().double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / bound).nan_to_num(1e9).max()):.3g} x the bound"


# ------------------------------------------------------------------------------------------------ dense
def act64(name, z, beta):
    """act, act', a bound of |act''|."""
    s = torch.sigmoid(z)
    if name == "none":
        return z, torch.ones_like(z), 0.0
    if name == "relu":
        return z.clamp(min=0), (z > 0).double(), 0.0
    if name == "softplus":
        return torch.logaddexp(beta * z, torch.zeros_like(z)) / beta, torch.sigmoid(beta * z), beta / 4
    if name == "sigmoid":
        return s, s * (1 - s), 0.1
    if name == "silu":
        return z * s, s * (1 + z * (1 - s)), 0.5
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z), 1.2


def dense_reference(x, w, b, r, act, beta, g=None):
    """64-bit outputs and their bounds: y, and with a cotangent dx, dw, db."""
    t = x.dtype
    x, w = x.detach().double().cpu(), w.detach().double().cpu()
    K, N, M = x.shape[1], w.shape[0], x.shape[0]
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, mag = z + b.detach().double().cpu(), mag + b.detach().double().cpu().abs()
    # K products and sums; fp32 operands in three pieces drop less than 2^-21 of every product
    ez = ((K + 2) * U + (2.0 ** -21 if t == torch.float32 else 0.0)) * mag
    h, d, curve = act64(act, z, beta)
    y = h if r is None else h + r.detach().double().cpu()
    # act is 1.13-Lipschitz at most and evaluated to 3e-6 relative (its argument beta z to one ulp: beta |z| ulps of h at most, h >= its slope there)
    ey = 1.13 * ez + 3e-6 * h.abs() + 2 * U * (h.abs() + y.abs()) + (1e-6 / beta if act == "softplus" else 0.0)
    by = ey + half_step(t) * (y.abs() + ey) + tiny(t)
    if g is None:
        return y, by
    g = g.double().cpu()
    dz = g * d
    # act' is kept with 24 significant bits beside fp32 rows, 12 beside fp16 and 11 beside bf16 rows: half a step is
    keep = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -12, torch.bfloat16: 2.0 ** -11}[t]
    edz = g.abs() * (curve * ez + (keep + 4e-6) * d.abs() + 2.0 ** -24) + 2.0 ** -15 * dz.abs() * (t != torch.float32) + 2 * U * dz.abs() + tiny(t)
    extra = 2.0 ** -21 if t == torch.float32 else 0.0

    def out(v, e, typ):
        return v, e + half_step(typ) * (v.abs() + e) + tiny(typ)
    grads = {"x": out(dz @ w, edz @ w.abs() + ((N + 2) * U + extra) * (dz.abs() @ w.abs()), t),
             "weight": out(dz.t() @ x, edz.t() @ x.abs() + ((M + 2) * U + extra) * (dz.abs().t() @ x.abs()), t)}
    if b is not None:
        grads["bias"] = out(dz.sum(0), edz.sum(0) + (M + 2) * U * dz.abs().sum(0), b.dtype)
    return y, by, grads


def dense_inputs(M, K, N, t, seed, residual=True, exact=False):
    gen = torch.Generator().manual_seed(seed)

    def make(*s, scale=1.0):
        v = torch.randn(*s, generator=gen) * scale
        return (torch.round(v * 4) / 4 if exact else v).to(t).cuda()
    return make(M, K), make(N, K, scale=1.0 if exact else max(K, 1) ** -0.5), make(N, scale=0.3), make(M, N) if residual else None, make(M, N)


SIZES = [(1, 1, 1), (1, 256, 256), (2, 300, 20), (3, 7, 5), (8, 64, 33), (9, 16, 16), (12, 3, 300), (31, 177, 131), (128, 8, 9), (129, 207, 256), (257, 256, 257),
         (300, 1, 300), (70, 300, 1), (640, 72, 40), (1000, 520, 130),
         (8200, 264, 1030), (4200, 521, 2050), (50000, 3, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_dense_forward_and_gradients(size, dtype):
    M, K, N = size
    t = TYPES[dtype]
    names = [n for n in ops.ACTIVATIONS if n != "relu"]
    for i, act in enumerate(names if M * K * N < 3e6 else [names[(M + K) % len(names)]]):
        x, w, b, r, g = dense_inputs(M, K, N, t, 7 * M + K + N + i, residual=i % 2 == 0)
        leaves = [v.requires_grad_(True) for v in (x, w, b)] + ([r.requires_grad_(True)] if r is not None else [])
        beta = 100.0 if i % 2 else 3.0
        y = ops.dense(x, w, b, r, activation=act, beta=beta)
        got = torch.autograd.grad(y, leaves, g)
        yw, by, grads = dense_reference(x, w, b, r, act, beta, g)
        close(y, yw, by, f"{act} y")
        for name, v in zip(("x", "weight", "bias"), got):
            close(v, *grads[name], f"{act} d_{name}")
        if r is not None:
            assert torch.equal(got[3], g)
        with torch.no_grad():
            assert torch.equal(ops.dense(x, w, b, r, activation=act, beta=beta), y)     # (no second variant behind no_grad)


@pytest.mark.parametrize("dtype", TYPES)
def test_dense_relu_and_its_border(dtype):
    """Inputs on a grid: z is exact in every order of summation, zeros among it, so ReLU's derivative is decided without rounding."""
    for M, K, N in ((5, 24, 40), (200, 40, 72)):
        x, w, b, r, g = dense_inputs(M, K, N, TYPES[dtype], M, exact=True)
        for v in (x, w, b, r):
            v.requires_grad_(True)
        assert ((x.double() @ w.double().t() + b.double()) == 0).any()
        y = ops.dense(x, w, b, r, activation="relu")
        got = torch.autograd.grad(y, (x, w, b), g)
        yw, by, grads = dense_reference(x, w, b, r, "relu", 1.0, g)
        close(y, yw, by, "y")
        for name, v in zip(("x", "weight", "bias"), got):
            close(v, *grads[name], name)


@pytest.mark.parametrize("dtype", TYPES)
def test_dense_strides_and_shapes(dtype):
    t = TYPES[dtype]
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(60, 401, generator=gen).to(t).cuda()
    base = torch.randn(70, 300, generator=gen).to(t).cuda()
    w = base[:, 3:180]                                        # rows of 177 inside rows of 300
    x = wide[:, 5:182]
    out = ops.dense(x, w, None, wide[:, 200:270], activation="silu")
    want = ops.dense(x.contiguous(), w.contiguous(), None, wide[:, 200:270].contiguous(), activation="silu")
    assert torch.equal(out, want)
    assert torch.equal(ops.dense(x.reshape(3, 4, 5, 177), w, activation="silu").reshape(60, 70), ops.dense(x, w, activation="silu"))
    xt = torch.randn(177, 60, generator=gen).to(t).cuda().t()                              # columns first
    assert torch.equal(ops.dense(xt, w), ops.dense(xt.contiguous(), w))
    wt = torch.randn(177, 70, generator=gen).to(t).cuda().t()
    assert torch.equal(ops.dense(x, wt), ops.dense(x, wt.contiguous()))
    one = x[:1].expand(20, 177)
    assert torch.equal(ops.dense(one, w), ops.dense(one.contiguous(), w))
    assert torch.equal(ops.dense(x[7], w), ops.dense(x[7:8], w)[0])                        # a vector
    # cotangents as autograd makes them: expanded, and transposed
    for make in (lambda y: y.sum(), lambda y: (y.t().float() * torch.arange(60, device="cuda")).sum()):
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = ops.dense(xs, ws, activation="sigmoid")
        a = torch.autograd.grad(make(y), (xs, ws), retain_graph=True)
        gy = torch.autograd.grad(make(y), y, retain_graph=True)[0].contiguous()
        bb = torch.autograd.grad(y, (xs, ws), gy)
        assert all(torch.equal(p, q) for p, q in zip(a, bb))


@pytest.mark.parametrize("dtype", TYPES)
def test_dense_rows_do_not_touch_each_other(dtype):
    """Infinities and NaN stay in their rows; padded columns and the last pieces of odd rows bring nothing in."""
    t = TYPES[dtype]
    for M, K, N in ((5, 41, 19), (150, 41, 19), (150, 207, 130)):
        x, w, b, _, g = dense_inputs(M, K, N, t, 3, residual=False)
        clean = ops.dense(x, w, b, activation="silu")
        bad = x.clone()
        bad[2, K - 1], bad[4, 0] = float("inf"), float("nan")
        y = ops.dense(bad, w, b, activation="silu")
        rows = [i for i in range(M) if i not in (2, 4)]
        assert torch.equal(y[rows], clean[rows])
        assert y[4].isnan().all() and not y[2].isfinite().logical_and(y[2] != 0).any()
        wb = w.clone()
        wb[3, K - 2] = float("nan")
        z = ops.dense(x, wb, b)
        cols = [i for i in range(N) if i != 3]
        assert torch.equal(z[:, cols], ops.dense(x, w, b)[:, cols]) and z[:, 3].isnan().all()
        # gradients: a bad row of the cotangent reaches its row of dx alone
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        gb = g.clone()
        gb[2, N - 1] = float("inf")
        dx0 = torch.autograd.grad(ops.dense(xs, ws, activation="silu"), xs, g)[0]
        dx1, dw1 = torch.autograd.grad(ops.dense(xs, ws, activation="silu"), (xs, ws), gb)
        assert torch.equal(dx0[[i for i in range(M) if i != 2]], dx1[[i for i in range(M) if i != 2]])
        assert not dx1[2].isfinite().any() and not dw1[N - 1].isfinite().any() and dw1[:N - 1].isfinite().all()


def test_dense_infinities_follow_ieee_in_16_bits():
    for t in (torch.float16, torch.bfloat16):
        x = torch.ones(40, 37, dtype=t, device="cuda")
        x[1, 36], x[2, 0], x[3, 5] = float("inf"), float("-inf"), float("inf")
        w = torch.full((24, 37), 0.5, dtype=t, device="cuda")
        y = ops.dense(x, w)
        want = x.double() @ w.double().t()
        assert torch.equal(y.double(), want)


@pytest.mark.parametrize("act", ["softplus", "sigmoid", "silu", "gelu_tanh", "relu"])
def test_dense_activations_at_extremes(act):
    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 5.0, -5.0, 30.0, -30.0, 90.0, -90.0, 1e4, -1e4, 3e4, -3e4, 1e30, -1e30], device="cuda")
    for n in (1, 40):                                         # both row forms
        x = z.reshape(-1, 1).expand(-1, 1)[:, None].expand(-1, n, 1).reshape(-1, 1) if n > 1 else z.reshape(-1, 1)
        x = x.contiguous().requires_grad_(True)
        w = torch.ones(3, 1, device="cuda")
        y = torch.cat([ops.dense(x[i:i + 8], w, activation=act, beta=2.0) for i in range(0, x.shape[0], 8)]) if n == 1 else ops.dense(x, w, activation=act, beta=2.0)
        dx = torch.autograd.grad(y[:, 0].sum(), x)[0]
        h, d, _ = act64(act, x.detach().double(), 2.0)
        assert y.isfinite().all() and dx.isfinite().all()
        assert ((y[:, :1].double() - h).abs() <= 2e-6 * h.abs() + 1e-7).all()
        assert ((dx.double() - d).abs() <= 2e-6 * d.abs() + 1e-6).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", ["softplus", "sigmoid", "silu", "gelu_tanh", "relu"])
def test_dense_16_bit_activations_at_extremes(act, dtype):
    t = TYPES[dtype]
    top = 60000.0 if dtype == "fp16" else 2e38
    z = torch.tensor([0.0, -0.0, 1e-3, -1e-3, 0.5, -0.5, 5.0, -5.0, 12.0, -12.0, 30.0, -30.0, 90.0, -90.0, 1e4, -1e4, top, -top], device="cuda").to(t)
    special = torch.tensor([float("inf"), float("nan")], device="cuda").to(t)
    for n in (1, 40):                                         # both row forms
        x = torch.cat([z, special]).repeat_interleave(n)[:, None].contiguous().requires_grad_(True)
        w = torch.ones(3, 1, device="cuda", dtype=t)
        y = torch.cat([ops.dense(v, w, activation=act, beta=2.0) for v in x.split(8)]) if n == 1 else ops.dense(x, w, activation=act, beta=2.0)
        dx = torch.autograd.grad(y[:, 0].sum(), x)[0]
        m = z.numel() * n
        h, d, _ = act64(act, x.detach().double()[:m], 2.0)
        # relative: the result's rounding and 3e-6 of the evaluation (the argument's rounding, |u| < 20 where q is not 0 or 1 in 16 bits); softplus: 1e-7 absolute
        # near 1 + e = 1, over beta; derivatives are kept with 11 bits at least and rounded once more as dx
        assert ((y[:m, :1].double() - h).abs() <= (half_step(t) + 5e-6) * h.abs() + tiny(t) + 1e-7).all()
        assert ((dx[:m].double() - d).abs() <= (half_step(t) + 2.0 ** -11 + 5e-6) * d.abs() + tiny(t) + 2.0 ** -24).all()
        assert (y[m:m + n, 0] == (1.0 if act == "sigmoid" else float("inf"))).all() and y[m + n:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_dense_zero_sizes(dtype):
    t = TYPES[dtype]
    for M, K, N in ((0, 5, 7), (4, 0, 7), (20, 0, 7), (4, 5, 0), (0, 0, 0)):
        x = torch.randn(M, K, device="cuda").to(t).requires_grad_(True)
        w = torch.randn(N, K, device="cuda").to(t).requires_grad_(True)
        b = torch.randn(N, device="cuda").to(t).requires_grad_(True)
        y = ops.dense(x, w, b, activation="sigmoid")
        assert y.shape == (M, N)
        if K == 0:
            close(y, torch.sigmoid(b.double()).expand(M, N), torch.full((M, N), 2 * half_step(t)), "act(b)")
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert dx.shape == x.shape and dw.shape == w.shape and (dx == 0).all() and (M > 0 or ((dw == 0).all() and (db == 0).all()))


def test_dense_some_gradients_only():
    x, w, b, r, g = dense_inputs(200, 50, 30, torch.bfloat16, 11)
    full = [v.clone().requires_grad_(True) for v in (x, w, b, r)]
    want = torch.autograd.grad(ops.dense(*full, activation="silu"), full, g)
    for mask in range(1, 16):
        v = [p.clone().requires_grad_(bool(mask >> i & 1)) for i, p in enumerate((x, w, b, r))]
        wanted = [p for p in v if p.requires_grad]
        got = torch.autograd.grad(ops.dense(*v, activation="silu"), wanted, g)
        for q, p in zip(got, [want[i] for i in range(4) if mask >> i & 1]):
            assert torch.equal(q, p)
    b32 = b.float().requires_grad_(True)                      # an fp32 bias beside 16-bit rows keeps its type
    db = torch.autograd.grad(ops.dense(x, w, b32, activation="silu"), b32, g)[0]
    assert db.dtype == torch.float32 and torch.equal(db.to(torch.bfloat16), want[2])


def test_dense_gradient_against_differences():
    x, w, b, r, g = (v.float() for v in dense_inputs(20, 17, 9, torch.float32, 5))
    for act in ops.ACTIVATIONS:
        if act == "relu":
            continue
        v = [p.clone().requires_grad_(True) for p in (x, w, b, r)]
        grads = torch.autograd.grad(ops.dense(*v, activation=act, beta=2.0), v, g)
        for i, (p, gr) in enumerate(zip(v, grads)):
            d = torch.randn(p.shape, generator=torch.Generator().manual_seed(i)).cuda()
            e = 2.0 ** -9
            args = [q.detach().double().cpu() for q in v]

            def f(s):
                a = list(args)
                a[i] = a[i] + s * d.double().cpu()
                h = act64(act, a[0] @ a[1].t() + a[2], 2.0)[0] + a[3]
                return float((h * g.double().cpu()).sum())
            diff = (f(e) - f(-e)) / (2 * e)                   # truncation e^2 / 6 |f'''| < 1e-6 x a few hundred terms
            assert abs(diff - float((gr.double().cpu() * d.double().cpu()).sum())) < 2e-3 * (1 + abs(diff)), (act, i)


# ------------------------------------------------------------------------------------------------ gated scan
def scan_reference(gate, x, h0, cu, reverse, blend, g=None, g_last=None):
    """Step by step in 64 bits on the CPU -> {name: (value, bound)}.  `cu`: list of row borders; x [L,D], gate [L,1 or D]."""
    a, v = gate.detach().double().cpu().numpy(), x.detach().double().cpu().numpy()
    L, D = v.shape
    S = len(cu) - 1
    h0n = np.zeros((S, D)) if h0 is None else h0.detach().double().cpu().numpy()
    st, eb, before, ebefore = np.zeros((L, D)), np.zeros((L, D)), np.zeros((L, D)), np.zeros((L, D))
    last, elast = h0n.copy(), np.zeros((S, D))
    r, u = (1 - a, a * v) if blend else (np.broadcast_to(a, v.shape), v)
    r = np.broadcast_to(r, v.shape)
    mr = (np.abs(1.0) + np.abs(a)) * np.ones_like(v) if blend else np.abs(r)
    longest = 1
    for s in range(S):
        rows = range(cu[s], cu[s + 1])[::-1] if reverse else range(cu[s], cu[s + 1])
        h, m, n = h0n[s], np.abs(h0n[s]), 0
        longest = max(longest, cu[s + 1] - cu[s])
        for i in rows:
            n += 1
            before[i], ebefore[i] = h, m * n
            h = r[i] * h + u[i]
            m = np.abs(r[i]) * m + np.abs(u[i]) + (np.abs(h) if blend else 0)
            st[i], eb[i] = h, m * (n + 4)
        last[s], elast[s] = h, m * (n + 4)
    # every step is two rounded operations (blend: four); maps of n steps are products of n rounded factors
    c = 4 * U if blend else 2 * U
    tx = x.dtype
    out = {"states": (st, c * eb + half_step(tx) * (np.abs(st) + c * eb) + tiny(tx)), "last": (last, c * elast + 1e-37)}
    if g is None and g_last is None:
        return out
    gn = np.zeros((L, D)) if g is None else g.double().cpu().numpy()
    gl = np.zeros((S, D)) if g_last is None else g_last.double().cpu().numpy()
    dx, da, edx, eda, dh0, edh0 = (np.zeros((L, D)) for _ in range(6))
    dh0, edh0 = gl.copy(), np.zeros((S, D))
    for s in range(S):
        rows = list(range(cu[s], cu[s + 1])[::-1] if reverse else range(cu[s], cu[s + 1]))
        f, m, n = gl[s], np.abs(gl[s]), 0
        for i in rows[::-1]:
            n += 1
            lam = gn[i] + f
            mag = np.abs(gn[i]) + m
            e = c * (n + 4) * mag
            dx[i], edx[i] = (a[i] * lam, np.abs(a[i]) * e + U * mag) if blend else (lam, e)
            w = v[i] - before[i] if blend else before[i]
            da[i] = lam * w
            eda[i] = e * np.abs(w) + mag * (c * (ebefore[i] + 4 * np.abs(before[i])) + U * (np.abs(v[i]) + np.abs(before[i]))) + U * np.abs(da[i])
            f, m = r[i] * lam, np.abs(r[i]) * mag
        dh0[s], edh0[s] = f, c * (len(rows) + 4) * m
    if gate.shape[1] != D:
        tot = np.abs(da).sum(1, keepdims=True)
        da, eda = da.sum(1, keepdims=True), eda.sum(1, keepdims=True) + (D + 2) * U * tot
    tg = gate.dtype
    out["gate"] = (da, eda + half_step(tg) * (np.abs(da) + eda) + tiny(tg) + 1e-37)
    out["x"] = (dx, edx + half_step(tx) * (np.abs(dx) + edx) + tiny(tx) + 1e-37)
    out["h0"] = (dh0, edh0 + 1e-37)
    return out


def scan_case(lead, D, shared, blend, tx, tg, S, h0, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*lead, D, generator=gen).to(tx).cuda()
    a = torch.sigmoid(torch.randn(*lead, 1 if shared else D, generator=gen) * 2 + (-2.0 if blend else 2.0))
    if not blend:
        a = a * torch.where(torch.rand(a.shape, generator=gen) < 0.2, -1.0, 1.0)      # negative gates too
    a = torch.where(torch.rand(a.shape, generator=gen) < 0.05, torch.full_like(a, float(torch.rand(1, generator=gen) < 0.5)), a).to(tg).cuda()
    return a, x, torch.randn(S, D, generator=gen).cuda() if h0 else None, torch.randn(*lead, D, generator=gen).to(tx).cuda(), torch.randn(S, D, generator=gen).cuda()


def check_scan(a, x, h0, cu, D, shared, blend, reverse, packed, states=True, use_g=True, use_last=True, g=None, gl=None):
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda") if packed else None
    leaves = [v.clone().requires_grad_(True) for v in (a, x)] + ([h0.clone().requires_grad_(True)] if h0 is not None else [])
    kw = dict(cu_seqlens=cu_t, reverse=reverse, blend=blend, need_states=states)
    st, last = ops.gated_scan(leaves[0], leaves[1], leaves[2] if h0 is not None else None, **kw)
    assert (st is None) == (not states)
    flat = lambda v: v.reshape(-1, v.shape[-1])
    use_g = use_g and states
    ref = scan_reference(flat(a), flat(x), h0, cu, reverse, blend, flat(g) if use_g else None, gl if use_last or not use_g else None)
    as_t = lambda n: tuple(torch.from_numpy(np.ascontiguousarray(q)) for q in ref[n])
    if states:
        close(flat(st), *as_t("states"), "states")
    close(last, *as_t("last"), "last")
    outs, cots = ([st] if use_g else []) + ([last] if use_last or not use_g else []), ([g] if use_g else []) + ([gl] if use_last or not use_g else [])
    grads = torch.autograd.grad(outs, leaves, cots)
    for n, v in zip(("gate", "x", "h0"), grads):
        close(flat(v), *as_t(n), "d_" + n)
    with torch.no_grad():
        s2, l2 = ops.gated_scan(a, x, h0, **kw)
        assert torch.equal(l2, last) and (s2 is None or torch.equal(s2, st))


SCANS = [(1, 1, 1), (3, 1, 5), (512, 1, 9), (2, 7, 3), (5, 127, 3), (40, 16, 2), (4, 64, 32), (2, 1000, 8), (1, 5000, 4), (3, 129, 257), (2, 40, 6), (1, 2300, 1), (6, 300, 33),
         (1, 700, 1030), (40, 100, 33), (180, 35, 1030)]


@pytest.mark.parametrize("dtype", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")], ids="/".join)
@pytest.mark.parametrize("size", SCANS, ids=lambda s: "x".join(map(str, s)))
def test_scan_of_equal_lengths(size, dtype):
    B, T, D = size
    cu = [T * b for b in range(B + 1)]
    for k in range(8 if B * T * D < 20000 else 4):
        shared, blend, reverse, h0 = k & 1 == 1, k & 2 == 2, (k >> 2 ^ k) & 1 == 1, k % 3 != 0
        a, x, h, g, gl = scan_case((B, T), D, shared, blend, TYPES[dtype[0]], TYPES[dtype[1]], B, h0, 13 * k + D)
        check_scan(a, x, h, cu, D, shared and D > 1, blend, reverse, False, states=k != 3, use_g=k != 2, use_last=k != 1, g=g, gl=gl)


@pytest.mark.parametrize("dtype", [("fp32", "fp32"), ("bf16", "fp32"), ("fp16", "fp16")], ids="/".join)
@pytest.mark.parametrize("D", [1, 3, 4, 37, 300])
def test_scan_of_packed_sequences(D, dtype):
    """Empty sequences at both ends and between, one-step ones, long ones, rows of no sequence before the first and behind the last."""
    for k, cu in enumerate(([0, 0, 1, 1, 1, 5, 900, 901, 1600, 1600], [3, 3, 40, 41, 200, 200, 203], [0, 6000], [2, 2], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10])):
        L, S = cu[-1] + (7 if k < 4 else 0), len(cu) - 1
        for blend, reverse in ((False, False), (True, True)):
            a, x, h, g, gl = scan_case((L,), D, k % 2 == 1, blend, TYPES[dtype[0]], TYPES[dtype[1]], S, k != 2, 5 * k + D)
            check_scan(a, x, h, cu, D, k % 2 == 1 and D > 1, blend, reverse, True, g=g, gl=gl)


def test_scan_long_sequence_over_many_ranges():
    """Ranges beyond one round of the carry launch, slow decay: what crosses them decides the result."""
    T, D = 30000, 130
    gen = torch.Generator().manual_seed(2)
    a = (1 - 1e-3 * torch.rand(1, T, D, generator=gen)).cuda()
    x, g, gl = torch.randn(1, T, D, generator=gen).cuda(), torch.randn(1, T, D, generator=gen).cuda(), torch.randn(1, D, generator=gen).cuda()
    check_scan(a, x, None, [0, T], D, False, False, False, False, g=g, gl=gl)


def test_scan_continues_from_its_last_state():
    a, x, h, _, _ = scan_case((3, 400), 20, False, False, torch.float32, torch.float32, 3, True, 4)
    whole, end = ops.gated_scan(a, x, h)
    state, parts = h, []
    for lo, hi in ((0, 1), (1, 2), (2, 130), (130, 400)):     # single steps and stretches
        st, state = ops.gated_scan(a[:, lo:hi], x[:, lo:hi], state)
        parts.append(st)
    ref = scan_reference(a.reshape(-1, 20), x.reshape(-1, 20), h, [0, 400, 800, 1200], False, False)
    close(torch.cat(parts, 1).reshape(-1, 20), torch.from_numpy(ref["states"][0]), torch.from_numpy(ref["states"][1]), "parts")
    close(state, torch.from_numpy(ref["last"][0]), torch.from_numpy(ref["last"][1]), "state")


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("D", [3, 40])
def test_scan_sequences_do_not_touch_each_other(D, packed):
    """Infinities and NaN in one sequence, and in rows of none, leave every other one as it is, forward and backward."""
    T, S = 150, 40
    lead = (S * T,) if packed else (S, T)
    for blend in (False, True):
        a, x, h, g, gl = scan_case(lead, D, False, blend, torch.float32, torch.float32, S, True, 9)
        cu = torch.arange(S + 1, dtype=torch.int32, device="cuda") * T if packed else None
        if packed:                                            # a pad behind, full of NaN
            a, x, g = (torch.cat([v, torch.full((33, v.shape[1]), float("nan"), device="cuda")]) for v in (a, x, g))

        def run(a, x, h, g, gl):
            v = [p.clone().requires_grad_(True) for p in (a, x, h)]
            st, last = ops.gated_scan(*v, cu_seqlens=cu, blend=blend)
            return [st.detach()[:S * T] if packed else st.detach(), last.detach()] + [q[:S * T] if packed and q.shape[0] > S else q for q in torch.autograd.grad((st, last), v, (g, gl))], st
        clean, st = run(a, x, h, g, gl)
        assert all(v.isfinite().all() for v in clean)
        if packed:
            assert (st[S * T:] == 0).all()
        xb, gb, hb = x.clone(), g.clone(), h.clone()
        row = (7 * T + 149,) if packed else (7, 149)
        xb[row], gb[(11 * T,) if packed else (11, 0)], hb[20] = float("inf"), float("nan"), float("nan")
        dirty, _ = run(a, xb, hb, gb, gl)
        keep = [i for i in range(S) if i not in (7, 11, 20)]
        for p, q in zip(clean, dirty):
            n = p.shape[0] // S if packed and p.shape[0] != S else 1
            pick = (lambda v: v.reshape(S, n, D)[keep]) if packed and p.shape[0] != S else (lambda v: v[keep])
            assert torch.equal(pick(p), pick(q))


def test_scan_gate_extremes():
    """Gates of exactly 0 and 1, and opacities of 1 in front of infinities further back (blend: 0 times infinity is the formula's NaN, as in 64 bits)."""
    T, D = 300, 8
    x = torch.randn(2, T, D, device="cuda")
    for v, want in ((0.0, x), (1.0, x.double().cumsum(1))):
        st, _ = ops.gated_scan(torch.full((2, T, 1), v, device="cuda"), x)
        assert ((st.double() - want).abs() <= 2 * T * U * x.double().abs().cumsum(1) + 1e-30).all()
    st, last = ops.gated_scan(torch.ones(2, T, 1, device="cuda"), x, blend=True)
    assert torch.equal(st, x) and torch.equal(last, x[:, -1])


def test_scan_zero_sizes():
    for B, T, D in ((0, 5, 3), (2, 0, 3), (2, 5, 0)):
        a, x, h = torch.rand(B, T, D, device="cuda"), torch.randn(B, T, D, device="cuda"), torch.randn(B, D, device="cuda").requires_grad_(True)
        x.requires_grad_(True)
        st, last = ops.gated_scan(a, x, h)
        assert st.shape == x.shape and last.shape == (B, D)
        if T == 0:
            assert torch.equal(last, h)
            assert torch.equal(torch.autograd.grad(last, h, torch.ones_like(last))[0], torch.ones_like(last))
    cu = torch.zeros(4, dtype=torch.int64, device="cuda")
    st, last = ops.gated_scan(torch.rand(0, 2, device="cuda"), torch.rand(0, 2, device="cuda"), cu_seqlens=cu)
    assert st.shape == (0, 2) and torch.equal(last, torch.zeros(3, 2, device="cuda"))
    st, last = ops.gated_scan(torch.rand(6, 2, device="cuda"), torch.rand(6, 2, device="cuda"), cu_seqlens=cu[:1])      # rows of no sequence
    assert (st == 0).all() and last.shape == (0, 2)


def test_scan_ill_formed_borders_stay_inside():
    """What the kernels index is bounded whatever cu_seqlens holds (its values are not read on the host)."""
    for cu in ([0, 50, 20, 200], [-5, 10, 2 ** 31 - 1], [90, 3], [10, 10, 10, 5000]):
        v = [torch.rand(100, 6, device="cuda").requires_grad_(True) for _ in range(2)] + [torch.rand(len(cu) - 1, 6, device="cuda").requires_grad_(True)]
        st, last = ops.gated_scan(*v, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"))
        torch.autograd.grad((st, last), v, (torch.ones_like(st), torch.ones_like(last)))
    torch.cuda.synchronize()


def test_scan_strided_inputs():
    big = torch.rand(4, 90, 50, device="cuda")
    a, x = big[:, :, 3:23], torch.randn(90, 4, 20, device="cuda").transpose(0, 1)
    for p, q in zip(ops.gated_scan(a, x), ops.gated_scan(a.contiguous(), x.contiguous())):
        assert torch.equal(p, q)
    off = torch.rand(4 * 90 * 20 + 1, device="cuda")[1:].reshape(4, 90, 20)              # 4-byte aligned only
    assert torch.equal(ops.gated_scan(off, x)[0], ops.gated_scan(off.clone(), x)[0])


def test_composite_features_is_the_renderers_compositing():
    """rgb, and any other channels, with the weights of volume_render (alpha_to_w) and a background."""
    from neumesh_amd.renderer import alpha_to_w
    gen = torch.Generator().manual_seed(0)
    alpha = torch.sigmoid(torch.randn(300, 127, generator=gen) * 3 - 3).cuda()
    feats, bg = torch.randn(300, 127, 19, generator=gen).cuda(), torch.randn(300, 19, generator=gen).cuda()
    w = alpha_to_w(alpha.double().cpu())
    want = (w.unsqueeze(-1) * feats.double().cpu()).sum(1) + (1 - w.sum(1, keepdim=True)) * bg.double().cpu()
    got = ops.composite_features(alpha, feats, bg)
    assert (got.double().cpu() - want).abs().max() < 2e-5      # 127 steps x 4 roundings x |features| <= 5 and the renderer's 1e-10 in the transmittance
    lens = torch.randint(0, 128, (300,), generator=gen)
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).cuda()
    keep = torch.arange(127)[None] < lens[:, None]
    packed = ops.composite_features(alpha[keep.cuda()], feats[keep.cuda()], bg, cu_seqlens=cu)
    masked = ops.composite_features(torch.where(keep.cuda(), alpha, 0.0), feats, bg)
    assert (packed - masked).abs().max() < 2e-5


# ------------------------------------------------------------------------------------------------ together, streams, graphs
def make_head(t, seed=0):
    gen = torch.Generator().manual_seed(seed)
    shapes = [(64, 45), (64,), (64, 64), (64,), (64, 64), (64,), (1, 64), (1,), (12, 64), (12,)]
    return [(torch.randn(*s, generator=gen) * (s[-1] ** -0.5 if len(s) == 2 else 0.1)).to(t).cuda().requires_grad_(True) for s in shapes]


def head_step(p, pts, cu, bg, dense, composite):
    """A feature field along packed rays: layers with a residual block, opacities and features, composited."""
    h = dense(pts, p[0], p[1], None, "softplus")
    h = dense(dense(h, p[2], p[3], None, "silu"), p[4], p[5], h, "none")
    alpha = dense(h, p[6], p[7], None, "sigmoid")[:, 0]
    return composite(alpha, dense(h, p[8], p[9], None, "none"), bg, cu)


def own_step(p, pts, cu, bg):
    return head_step(p, pts, cu, bg, lambda x, w, b, r, act: ops.dense(x, w, b, r, activation=act, beta=5.0),
                     lambda al, f, bg, cu: ops.composite_features(al, f, bg, cu_seqlens=cu))


def plain_step(p, pts, cu, bg):
    def dense(x, w, b, r, act):
        h = act64(act, x @ w.t() + b, 5.0)[0]
        return h if r is None else h + r

    def composite(al, f, bg, cu):
        rows = []
        for s in range(len(cu) - 1):
            lo, hi = int(cu[s]), int(cu[s + 1])
            tr = torch.cat([torch.ones(1, dtype=al.dtype), torch.cumprod(1 - al[lo:hi], 0)])
            rows.append((tr[:-1, None] * al[lo:hi, None] * f[lo:hi]).sum(0) + tr[-1] * bg[s])
        return torch.stack(rows)
    return head_step(p, pts, cu, bg, dense, composite)


def head_data(t, seed):
    gen = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, 60, (50,), generator=gen)
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])
    return torch.randn(int(cu[-1]), 45, generator=gen).to(t).cuda(), cu.cuda(), torch.randn(50, 12, generator=gen).cuda(), torch.randn(50, 12, generator=gen).cuda()


@pytest.mark.parametrize("dtype", TYPES)
def test_feature_field_along_rays_end_to_end(dtype):
    t = TYPES[dtype]
    p, (pts, cu, bg, g) = make_head(t), head_data(t, 3)
    out = own_step(p, pts, cu, bg)
    grads = torch.autograd.grad(out, p, g)
    p64 = [v.detach().double().cpu().requires_grad_(True) for v in p]
    want = plain_step(p64, pts.double().cpu(), cu.cpu(), bg.double().cpu())
    wgrads = torch.autograd.grad(want, p64, g.double().cpu())
    # five layers deep, each output rounded to the type and amplified at most a few times on the way: 32 half steps of the largest value
    tol = 32 * max(half_step(t), 2.0 ** -20)
    assert (out.double().cpu() - want).abs().max() <= tol * want.abs().max()
    for a, b in zip(grads, wgrads):
        assert (a.double().cpu() - b).norm() <= tol * b.norm() + 1e-30


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_dense_tiles_of_strided_rows(dtype):
    """Enough rows and columns for 256 x 256 tiles: odd strides and offsets give the bits of contiguous tensors."""
    t = TYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(13000, 231, generator=gen, device="cuda").to(t)[:, 5:208]
    w = torch.randn(1030, 301, generator=gen, device="cuda").to(t)[:, 3:206]
    r = torch.randn(13000, 1101, generator=gen, device="cuda").to(t)[:, 7:1037]
    b = torch.randn(1030, generator=gen, device="cuda")
    y = ops.dense(x, w, b, r, activation="silu")
    assert torch.equal(y, ops.dense(x.contiguous(), w.contiguous(), b, r.contiguous(), activation="silu"))
    want, bound = dense_reference(x[-300:], w, b, r[-300:], "silu", 1.0)
    close(y[-300:], want, bound, "last rows")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_dense_tiles_keep_non_finite_values_apart(dtype):
    """... of rows in rows, of weights in columns; last pieces of odd contraction lengths included."""
    t = TYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, w = torch.randn(13000, 203, generator=gen, device="cuda").to(t), torch.randn(1030, 203, generator=gen, device="cuda").to(t)
    clean = ops.dense(x, w)
    assert clean.isfinite().all()
    bad, wbad = x.clone(), w.clone()
    bad[5], bad[300, 202], bad[12999, 196], bad[700, 0] = float("nan"), float("inf"), float("-inf"), float("inf")
    rows = torch.tensor([5, 300, 700, 12999], device="cuda")
    y = ops.dense(bad, w)
    keep = torch.ones(13000, dtype=torch.bool, device="cuda").index_fill(0, rows, False)
    assert torch.equal(y[keep], clean[keep]) and not y[rows].isfinite().any()
    wbad[7, 200], wbad[1029, 0] = float("inf"), float("nan")
    y = ops.dense(x, wbad)
    cols = torch.ones(1030, dtype=torch.bool, device="cuda").index_fill(0, torch.tensor([7, 1029], device="cuda"), False)
    assert torch.equal(y[:, cols], clean[:, cols]) and y[:, 1029].isnan().all()


def test_captured_large_layers_and_scans_replay():
    """The kernels of large sizes (tiles, split gradients, ranges with carried states) captured together, replayed on new data."""
    t = torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(13000, 200, generator=gen, device="cuda").to(t)
    p = [torch.randn(1030, 200, generator=gen, device="cuda").to(t).mul_(0.07).requires_grad_(True), torch.randn(1030, generator=gen, device="cuda").requires_grad_(True)]
    cu = torch.tensor([0, 0, 900, 901, 7000, 12990], device="cuda")
    gate = torch.rand(13000, 1, generator=gen, device="cuda")
    g, gs = torch.randn(5, 1030, generator=gen, device="cuda"), torch.randn(13000, 1030, generator=gen, device="cuda").to(t)

    def step(p):
        states, last = ops.gated_scan(gate, ops.dense(x, p[0], p[1], activation="silu"), cu_seqlens=cu, blend=True)
        return [states, last] + list(torch.autograd.grad((states, last), p, (gs, g)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(p)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(p)
    for i in range(3):
        x.copy_(torch.randn(x.shape, generator=gen, device="cuda").to(t))
        graph.replay()
        want = step([v.detach().clone().requires_grad_(True) for v in p])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_offsets_beyond_32_bits():
    """More than 2^31 elements and 2^32 bytes: the far end against the same rows on their own."""
    L, D = 8_500_000, 256
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.empty(L, D, device="cuda", dtype=torch.bfloat16).uniform_(-1, 1, generator=gen)

    def near(a, b):                                           # two roundings of one value to 8 bits, sums in another order
        return bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-4).all())
    w = torch.randn(D, D, generator=gen, device="cuda").to(torch.bfloat16) / 16
    y = ops.dense(x, w, activation="relu")
    assert near(y[-70000:], ops.dense(x[-70000:], w, activation="relu"))
    del y
    gate = torch.empty(1, L, 1, device="cuda").uniform_(0.2, 0.9, generator=gen)      # 3000 steps: nothing is left of what was before
    v = x[None].requires_grad_(True)
    states, last = ops.gated_scan(gate, v)
    tail, end = ops.gated_scan(gate[:, -5000:], x[None, -5000:])
    assert near(states[0, -2000:], tail[0, -2000:]) and near(last, end)
    dx = torch.autograd.grad(states, v, torch.ones_like(states))[0]
    u = x[None, -5000:].clone().requires_grad_(True)
    du = torch.autograd.grad(ops.gated_scan(gate[:, -5000:], u)[0], u, torch.ones_like(u))[0]
    assert near(dx[0, -5000:], du[0])
    cu = torch.tensor([0, 10, L - 3000, L], device="cuda")
    st, last = ops.gated_scan(gate[0], x, cu_seqlens=cu)
    one, end = ops.gated_scan(gate[:, -3000:], x[None, -3000:])
    assert near(st[-3000:], one[0]) and near(last[2:], end)


def test_same_bits_again_and_on_other_streams():
    p, (pts, cu, bg, g) = make_head(torch.bfloat16), head_data(torch.bfloat16, 5)
    ref = own_step(p, pts, cu, bg)
    ref = [ref] + list(torch.autograd.grad(ref, p, g))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:                                     # calls of the streams in turn, nothing waited for in between
            with torch.cuda.stream(s):
                out = own_step(p, pts, cu, bg)
                got.append([out] + list(torch.autograd.grad(out, p, g)))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, ref))


def test_captured_graphs_replay_and_do_not_share_scratch():
    """Two captured training steps (forward and backward) on other data, replayed in turn with eager work between; leaves of their own."""
    graphs = []
    for seed in (6, 7):
        p, (pts, cu, bg, g) = make_head(torch.float16, seed), head_data(torch.float16, seed)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(2):
                out = own_step(p, pts, cu, bg)
                torch.autograd.grad(out, p, g)
        torch.cuda.current_stream().wait_stream(stream)
        del out
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = own_step(p, pts, cu, bg)
            grads = torch.autograd.grad(out, p, g)
        graphs.append((gr, p, pts, cu, bg, g, [out] + list(grads)))
    for i in range(4):
        for gr, p, pts, cu, bg, g, held in graphs:
            with torch.no_grad():
                pts.copy_(torch.randn(pts.shape, generator=torch.Generator().manual_seed(100 + i)).to(pts.dtype))
            gr.replay()
            q = [v.detach().clone().requires_grad_(True) for v in p]
            out = own_step(q, pts, cu, bg)
            want = [out] + list(torch.autograd.grad(out, q, g))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_second_derivatives_are_refused():
    """... instead of leaving a penalty on a gradient without its gradient."""
    x, w = torch.randn(20, 8, device="cuda", requires_grad=True), torch.randn(4, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="dense: its gradient cannot be differentiated again"):
        torch.autograd.grad(ops.dense(x, w, activation="silu").sum(), x, create_graph=True)
    v = torch.randn(2, 8, 4, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="gated_scan: its gradient cannot be differentiated again"):
        torch.autograd.grad(ops.gated_scan(torch.rand(2, 8, 4, device="cuda"), v)[1].sum(), v, create_graph=True)


def test_in_place_change_between_forward_and_backward_is_an_error():
    x, w = torch.randn(20, 8, device="cuda", requires_grad=True), torch.randn(4, 8, device="cuda", requires_grad=True)
    y = ops.dense(x, w, activation="silu")
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
