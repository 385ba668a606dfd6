"""neumesh_amd.ops at the ends of its ranges: sizes beyond one launch, sums over nothing, cotangents and derivatives from the smallest to the largest numbers.
Tolerances are elementwise bounds from the arithmetic, as in test_gpu_ops.py."""
import pytest
import torch
import torch.utils.checkpoint

from neumesh_amd import ops

pytestmark = pytest.mark.gpu


def test_states_beyond_32_bits_of_empty_sequences():
    """Packed sequences, nearly all of them empty, with more than 2^32 states: those pass through, the few rows are scanned, and back."""
    S, D, L = (1 << 22) + 3, 1024, 40
    cu = torch.full((S + 1,), 10, dtype=torch.int32, device="cuda")      # rows 0 .. 9 in sequence 0, 10 .. 34 in the last one, 5 rows in none
    cu[0], cu[S] = 0, 35
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, gate = torch.randn(L, D, generator=gen, device="cuda").requires_grad_(True), torch.rand(L, 1, generator=gen, device="cuda").requires_grad_(True)
    h0 = torch.empty(S, D, device="cuda").uniform_(-1, 1, generator=gen).requires_grad_(True)
    states, last = ops.gated_scan(gate, x, h0, cu_seqlens=cu)
    assert torch.equal(last[1:-1], h0.detach()[1:-1]) and (states[35:] == 0).all()
    ends = torch.tensor([0, 10, 35], device="cuda")
    leaves = [v.detach().clone().requires_grad_(True) for v in (gate, x)] + [h0.detach()[[0, -1]].clone().requires_grad_(True)]
    few, end = ops.gated_scan(leaves[0], leaves[1], leaves[2], cu_seqlens=ends)
    assert torch.equal(states, few) and torch.equal(last[[0, -1]], end)
    g = h0.detach()                                           # (cotangent of the last states: the same values again)
    grads = torch.autograd.grad(last, (gate, x, h0), g)
    want = torch.autograd.grad(end, leaves, g[[0, -1]].contiguous())
    assert torch.equal(grads[0], want[0]) and torch.equal(grads[1], want[1]) and torch.equal(grads[2][[0, -1]], want[2])
    assert torch.equal(grads[2][1:-1], g[1:-1])
    # no rows at all
    _, last = ops.gated_scan(gate.detach()[:0], x.detach()[:0], g, cu_seqlens=torch.zeros_like(cu))
    assert torch.equal(last, g)


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
def test_gradient_of_a_shared_gate_over_no_channels(types):
    """An empty sum: 0, whatever the memory of the result held before."""
    for packed in (False, True):
        lead = (300,) if packed else (3, 100)
        gate = torch.rand(*lead, 1, device="cuda").to(types[1]).requires_grad_(True)
        x = torch.rand(*lead, 0, device="cuda").to(types[0]).requires_grad_(True)
        cu = torch.tensor([0, 100, 290], device="cuda") if packed else None
        states, last = ops.gated_scan(gate, x, cu_seqlens=cu)
        torch.full((300,), float("nan"), device="cuda", dtype=types[1])      # (freed at once: what the allocator hands out next)
        dgate, dx = torch.autograd.grad((states, last), (gate, x), (torch.ones_like(states), torch.ones_like(last)))
        assert dgate.shape == gate.shape and (dgate == 0).all() and dx.shape == x.shape
    alpha = torch.rand(5, 60, device="cuda").requires_grad_(True)
    out = ops.composite_features(alpha, torch.rand(5, 60, 0, device="cuda"))
    torch.full((300,), float("nan"), device="cuda")
    assert (torch.autograd.grad(out, alpha, torch.ones_like(out))[0] == 0).all()


# ------------------------------------------------------------------------------------------------ gradients of dense over the ranges of their types
def derivative(act, z, beta):
    """act'(z) in 64 bits, the size of its terms (what its evaluation's relative errors act on), |act''| at most over a small neighbourhood of z, and |u| of the exponential exp(-|u|)."""
    if act == "softplus":
        d = torch.sigmoid(beta * z)
        return d, d, beta * d, beta * z.abs()
    c1, c3 = (2 * (2 / torch.pi) ** 0.5, 0.044715) if act == "gelu_tanh" else (1.0, 0.0)
    u, du = c1 * (z + c3 * z ** 3), c1 * (1 + 3 * c3 * z * z)
    q, q1 = torch.sigmoid(u), torch.sigmoid(-u)
    if act == "sigmoid":
        return q * q1, q * q1, q * q1, u.abs()
    size = q + z.abs() * q * q1 * du
    # (q + z q q1 u')' = 2 q q1 u' + z q q1 (u'^2 (1 - 2 q) + u'')
    return q + z * q * q1 * du, size, q * q1 * (2 * du + z.abs() * (du * du + 6 * c1 * c3 * z.abs())), u.abs()


def gradient_bounds(x, w, b, act, beta, g, keep):
    """64-bit dx, dW, db and elementwise bounds.  Nothing absolute stands in them but the last rounding of each result: act' is kept to `keep` of itself, dz = g act' enters
    the products with 16 bits at least (fp32: in three exact pieces), sums are fp32."""
    t = x.dtype
    u32 = 2.0 ** -23                                          # one operation of a matrix instruction may truncate
    half, tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    x, w, b, g = (v.detach().double().cpu() for v in (x, w, b, g))
    K, N, M = x.shape[1], w.shape[0], x.shape[0]
    extra = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -16, torch.bfloat16: 0.0}[t]        # piece products that are dropped, of each product at most
    z = x @ w.t() + b
    ez = ((K + 2) * u32 + (extra if t == torch.float32 else 0.0)) * (x.abs() @ w.abs().t() + b.abs())
    d, size, curve, u = derivative(act, z, beta)
    # the exponential's argument: five roundings and three rounded constants at most; exponential and reciprocal are off by 1e-6 in all
    ed = curve * 1.01 * ez + (2e-6 + 8 * 2.0 ** -24 * u) * size + keep * d.abs()
    dz = g * d
    edz = g.abs() * ed + (0.0 if t == torch.float32 else 2.0 ** -16) * dz.abs() + u32 * dz.abs()

    def out(v, e):
        return v, e + half * (v.abs() + e) + tiny
    return (out(dz @ w, edz @ w.abs() + ((N + 2) * u32 + extra) * (dz.abs() @ w.abs())),
            out(dz.t() @ x, edz.t() @ x.abs() + ((M + 2) * u32 + extra) * (dz.abs().t() @ x.abs())),
            out(dz.sum(0), edz.sum(0) + (M + 2) * u32 * dz.abs().sum(0)))


def check_gradients(x, w, b, act, beta, g, keep, what):
    v = [p.detach().clone().requires_grad_(True) for p in (x, w, b)]
    got = torch.autograd.grad(ops.dense(*v, activation=act, beta=beta), v, g)
    for name, p, (want, bound) in zip(("d_x", "d_weight", "d_bias"), got, gradient_bounds(x, w, b, act, beta, g, keep)):
        off = (p.double().cpu() - want).abs()
        assert (off <= bound).all(), f"{what} {name}: {int((~(off <= bound)).sum())} of {off.numel()} off, worst {float((off / bound).nan_to_num(1e9).max()):.3g} x the bound"
        tiny = torch.finfo(p.dtype).smallest_normal * torch.finfo(p.dtype).eps
        assert (want.abs() > 4 * bound).float().mean() > 0.5 or want.abs().max() < 64 * tiny, f"{what} {name}: the bound says nothing"


# few rows; resident weights; streamed weights and a gradient without a split; many rows and a split gradient
GRAD_SIZES = [(5, 24, 40), (300, 130, 70), (1500, 520, 700), (70000, 40, 24)]
SCALES = {"fp16": (2.0 ** -24, 2.0 ** -21, 2.0 ** -17, 2.0 ** -12, 1.0), "bf16": (1e-30, 1e-12, 1e25), "fp32": (1e-25, 1e-6, 1e25)}
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", GRAD_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_dense_gradients_of_small_and_large_cotangents(size, dtype):
    """Cotangents over the range of their type: those of a mean over many outputs (fp16: down to its smallest number) as exact as those of size one."""
    (M, K, N), t = size, TYPES[dtype]
    gen = torch.Generator().manual_seed(M + K)
    for i, scale in enumerate(SCALES[dtype]):
        # all of one sign, so that the sums keep what their terms have; z within a few units of 0
        x, w = 0.5 + torch.rand(M, K, generator=gen), (0.5 + torch.rand(N, K, generator=gen)) / K
        b, g = torch.randn(N, generator=gen) * 0.3 - 0.5, (1 + torch.rand(M, N, generator=gen)) * scale
        x, w, b, g = (v.to(t).cuda() for v in (x, w, b, g))
        check_gradients(x, w, b, ("sigmoid", "silu", "softplus", "gelu_tanh", "sigmoid")[i], 1.0, g, 2.0 ** -11, f"{scale:g}")


@pytest.mark.parametrize("size", GRAD_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_dense_fp16_cotangents_near_the_maximum(size):
    """g act' beyond fp16's range (act' up to 1.13) inside, finite results outside."""
    M, K, N = size
    gen = torch.Generator().manual_seed(M)
    for act, z in (("gelu_tanh", 1.4), ("silu", 2.4)):
        x, w = 2.0 ** -14 * (1 + torch.rand(M, K, generator=gen)), 2.0 ** -12 * (1 + torch.rand(N, K, generator=gen))
        b, g = z + 0.1 * torch.rand(N, generator=gen), 61000 + 4000 * torch.rand(M, N, generator=gen)
        if M > 10000:                                         # (dW within fp16: most rows without a cotangent)
            g[torch.rand(M, 1, generator=gen).expand(M, N) < 0.95] = 0
        x, w, g = (v.half().cuda() for v in (x, w, g))
        b = b.cuda()
        v = [p.clone().requires_grad_(True) for p in (x, w, b)]
        dx, dw, db = torch.autograd.grad(ops.dense(*v, activation=act), v, g)
        dz = g.double() * derivative(act, x.double() @ w.double().t() + b.double(), 1.0)[0]
        assert dz.max() > 65504 and dx.isfinite().all() and dw.isfinite().all() and db.isfinite().all()
        for name, p, (want, bound) in zip(("d_x", "d_weight"), (dx, dw), gradient_bounds(x, w, b, act, 1.0, g, 2.0 ** -11)):
            off = (p.double().cpu() - want).abs()
            assert (off <= bound).all(), f"{act} {name}: worst {float((off / bound).max()):.3g} x the bound"


def test_dense_fp16_infinities_in_the_cotangent_stay_in_their_rows():
    x, w = torch.randn(200, 41, device="cuda").half(), torch.randn(19, 41, device="cuda").half()
    g = torch.randn(200, 19, device="cuda").half()
    bad = g.clone()
    bad[3, 4], bad[100, 18] = float("inf"), float("nan")
    grads = []
    for c in (g, bad):
        v = [p.clone().requires_grad_(True) for p in (x, w)]
        grads.append(torch.autograd.grad(ops.dense(*v, activation="silu"), v, c))
    rows = [i for i in range(200) if i not in (3, 100)]
    cols = [i for i in range(19) if i not in (4, 18)]
    assert torch.equal(grads[0][0][rows], grads[1][0][rows]) and not grads[1][0][[3, 100]].isfinite().any()
    assert torch.equal(grads[0][1][cols], grads[1][1][cols]) and not grads[1][1][[4, 18]].isfinite().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", GRAD_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_dense_gradients_in_the_tails_of_activations(size, dtype):
    """Units far below 0 on every row: their small derivatives are kept as exactly as large ones (half a step of 16 significant bits, 24 beside fp32), not to an absolute step."""
    (M, K, N), t = size, TYPES[dtype]
    gen = torch.Generator().manual_seed(M + N)
    cases = [("sigmoid", -15.0, 1.0), ("sigmoid", -18.0, 1.0), ("silu", -17.0, 1.0), ("gelu_tanh", -4.6, 1.0), ("softplus", -0.45, 50.0 if dtype == "fp16" else 100.0)]
    if dtype != "fp16":
        cases += [("sigmoid", -60.0, 1.0), ("softplus", -0.7, 100.0), ("gelu_tanh", -8.0, 1.0)]
    for act, shift, beta in cases:
        x, w = 0.5 + torch.rand(M, K, generator=gen), (0.5 + torch.rand(N, K, generator=gen)) / (8 * K)
        b, g = shift - 0.1 * torch.rand(N, generator=gen), (1 + torch.rand(M, N, generator=gen)) * 2.0 ** (12 if dtype == "fp16" else 0)
        x, w, b, g = (v.to(t).cuda() for v in (x, w, b, g))
        assert (x.double() @ w.double().t() + b.double()).max() < 0.6 * shift
        check_gradients(x, w, b.float(), act, beta, g, 2.0 ** -24 if dtype == "fp32" else 2.0 ** -16, f"{act} at {shift}")


# ------------------------------------------------------------------------------------------------ what a forward pass keeps for the backward pass
def both_ways(make, wrap):
    """Gradients of make() -> (outputs, leaves, cotangents), plainly and with the forward pass inside wrap()."""
    out, leaves, cots = make()
    want = torch.autograd.grad(out, leaves, cots)
    with wrap():
        out, leaves, cots = make()
    got = torch.autograd.grad(out, leaves, cots)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def dense_slices():
    """Rows that are slices of wider tensors, on both sides."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(300, 401, generator=gen, device="cuda").half()[:, 5:182].detach().requires_grad_(True)
    w = torch.randn(70, 300, generator=gen, device="cuda").half()[:, 3:180].detach().requires_grad_(True)
    return ops.dense(x, w, activation="silu"), (x, w), torch.randn(300, 70, generator=gen, device="cuda").half()


def packed_scan():
    gen = torch.Generator(device="cuda").manual_seed(3)
    gate = torch.rand(40, 800, generator=gen, device="cuda").t().detach().requires_grad_(True)     # columns first
    x, h0 = torch.randn(800, 50, generator=gen, device="cuda")[:, 4:44].detach().requires_grad_(True), torch.randn(3, 40, generator=gen, device="cuda").requires_grad_(True)
    states, last = ops.gated_scan(gate, x, h0, cu_seqlens=torch.tensor([0, 1, 500, 790], device="cuda"))
    return (states, last), (gate, x, h0), (torch.randn(800, 40, generator=gen, device="cuda"), torch.randn(3, 40, generator=gen, device="cuda"))


@pytest.mark.parametrize("make", [dense_slices, packed_scan])
def test_saved_tensors_may_come_back_with_other_strides(make):
    """Hooks that keep saved tensors on the host give them back contiguous; others give them back spread out."""
    both_ways(make, torch.autograd.graph.save_on_cpu)

    def spread(t):
        wide = torch.empty((*t.shape[:-1], 2 * t.shape[-1] + 3), dtype=t.dtype, device=t.device)
        return wide[..., 1:1 + 2 * t.shape[-1]:2].copy_(t) if t.dim() > 1 else t
    both_ways(make, lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread))


@pytest.mark.parametrize("make", [dense_slices, packed_scan])
def test_kept_tensors_are_saved_variables(make):
    """What the forward pass keeps beside its inputs (act'(z), states) is released by the backward pass while the outputs live, passes through hooks on saved
    tensors, and is made again under checkpointing."""
    _, leaves, cots = make()
    sizes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (sizes.append(t.numel() * t.element_size()), t)[1], lambda t: t):
        make()
    if make is dense_slices:
        assert sizes[-1] == 300 * 70 * 3                      # act'(z)
    else:
        assert sizes[-1] > 800 * 4                            # the sequences of the rows, and states
    leaves = [v.detach().requires_grad_(True) for v in leaves]

    def run(*v):
        return ops.dense(*v, activation="silu") if make is dense_slices else ops.gated_scan(*v, cu_seqlens=torch.tensor([0, 1, 500, 790], device="cuda"))
    want = torch.autograd.grad(run(*leaves), leaves, cots)
    got = torch.autograd.grad(torch.utils.checkpoint.checkpoint(run, *leaves, use_reentrant=False), leaves, cots)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_memory_falls_after_backward_while_outputs_live():
    x, w = torch.randn(20000, 64, device="cuda", requires_grad=True), torch.randn(256, 64, device="cuda", requires_grad=True)
    gate, v = torch.rand(1, 40000, 64, device="cuda", requires_grad=True), torch.randn(1, 40000, 64, device="cuda", requires_grad=True)
    for run, leaves, kept in ((lambda: ops.dense(x, w, activation="silu"), (x, w), 20000 * 256 * 4), (lambda: ops.gated_scan(gate, v)[0], (gate, v), 40000 // 64 * 64 * 4)):
        y = run()
        before = torch.cuda.memory_allocated()
        grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
        del grads
        assert torch.cuda.memory_allocated() <= before - kept and y.grad_fn is not None
        with pytest.raises(RuntimeError, match="backward through the graph a second time"):
            torch.autograd.grad(y, leaves, torch.ones_like(y))


@pytest.mark.parametrize("rows", [4, 40, 20000])              # few rows, streamed or resident weights, a split gradient
def test_fp32_products_are_fp32_products(rows):
    """Layers of one and a few inputs, where nothing hides what a product loses: operands whose bits below the first eight are all ones, and the largest numbers there
    are.  Piece products of 2^-23 of a product are left out at most, and its largest one is added with an error of one unit in the last place."""
    def near(got, a, b):
        a, b, got = a.detach().double().cpu(), b.detach().double().cpu(), got.detach().double().cpu()
        terms = ((a != 0).double() @ (b != 0).double()).clamp(min=1)
        return ((got - a @ b).abs() <= (2.0 ** -23 + (2 * terms - 1) * 2.0 ** -23 + 2.0 ** -26) * (a.abs() @ b.abs())).all()
    for K in (1, 3):
        gen = torch.Generator().manual_seed(K)
        ones = torch.tensor([1.0 + 2.0 ** -7 - 2.0 ** -23, 1.0 + 2.0 ** -8 - 2.0 ** -23, 2.0 - 2.0 ** -23, 1.0 + 2.0 ** -6 - 2.0 ** -14])

        def some(*shape):
            return ones[torch.randint(0, 4, shape, generator=gen)]
        x, w = some(rows, K) * 2.0 ** torch.randint(-40, 40, (rows, 1), generator=gen), some(24, K) * 2.0 ** torch.randint(-20, 20, (24, 1), generator=gen)
        g = (some(rows, 24) * torch.nn.functional.one_hot(torch.arange(rows) % 24, 24)).cuda()      # one term in every sum of dx
        x, w = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
        y = ops.dense(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), g)
        assert near(y, x, w.t()) and near(dx, g, w) and near(dw, g.t(), x), K
    top = torch.full((rows, 8), 3.4e38).cuda()                # (sums in any order stay finite)
    w = torch.tensor([[0.1, -0.1] * 4, [2.0 ** -4] * 8, [2.0 ** -126] * 8]).cuda()
    y = ops.dense(top, w)
    assert y.isfinite().all() and near(y, top, w.t())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_kept_derivatives_of_rows_of_any_width(dtype):
    """The gradient of an fp32 bias is a sum of kept derivatives that nothing rounds again: 16 significant bits of each, whatever the width of the rows."""
    t = TYPES[dtype]
    gen = torch.Generator().manual_seed(5)
    for N in (1, 2, 3, 5, 7, 8, 9, 13, 31, 33, 57, 129, 250, 517):
        for M in (1, 7, 9, 50, 700):                          # few rows, narrow and wide blocks of columns
            x, w, b = (torch.randn(*s, generator=gen) for s in ((M, 3), (N, 3), (N,)))
            x, w, b = x.to(t).cuda(), w.to(t).cuda(), (b - 3).cuda().requires_grad_(True)
            for act in ("sigmoid", "gelu_tanh"):
                db = torch.autograd.grad(ops.dense(x, w, b, activation=act), b, torch.ones(M, N, dtype=t, device="cuda"))[0]
                z = x.double() @ w.double().t() + b.double()
                d, size, curve, u = derivative(act, z, 1.0)
                bound = ((2.0 ** -16 + M * 2.0 ** -23) * d.abs() + (2e-6 + 8 * 2.0 ** -24 * u) * size + curve * 1.01 * 5 * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.abs())).sum(0)
                assert ((db - d.sum(0)).abs() <= bound).all(), (N, M, act)


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_inputs_keep_to_their_rows_in_gradients(dtype):
    t = TYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(7)
    for M, K, N in ((6, 20, 37), (150, 41, 19), (400, 700, 600)):
        x, w, g = (torch.randn(*s, generator=gen, device="cuda").to(t) for s in ((M, K), (N, K), (M, N)))
        bad = x.clone()
        bad[3, K - 1] = float("nan")
        grads = []
        for v in (x, bad):
            leaves = [p.clone().requires_grad_(True) for p in (v, w)]
            grads.append(torch.autograd.grad(ops.dense(*leaves, activation="silu"), leaves, g))
        rows = [i for i in range(M) if i != 3]
        assert torch.equal(grads[0][0][rows], grads[1][0][rows]) and grads[1][0][3].isnan().all() and grads[1][1].isnan().all()


def test_training_layer_beyond_32_bits():
    """More than 2^32 bytes of kept derivatives: gradients of the far end against the same rows on their own."""
    M, D = 8_500_000, 256
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.empty(M, D, device="cuda", dtype=torch.bfloat16).uniform_(-1, 1, generator=gen).requires_grad_(True)
    w, b = (torch.randn(D, D, generator=gen, device="cuda") / 16).bfloat16(), torch.zeros(D, device="cuda", requires_grad=True)
    g = torch.zeros(M, D, device="cuda", dtype=torch.bfloat16)
    g[-70000:].uniform_(-1, 1, generator=gen)
    dx, db = torch.autograd.grad(ops.dense(x, w, b, activation="silu"), (x, b), g)
    assert (dx[:-70000] == 0).all()
    u, c = x.detach()[-70000:].clone().requires_grad_(True), torch.zeros(D, device="cuda", requires_grad=True)
    du, dc = torch.autograd.grad(ops.dense(u, w, c, activation="silu"), (u, c), g[-70000:])
    # sums of 70000 terms of size one in two orders; rounding of one value to 8 bits twice
    assert ((dx[-70000:].float() - du.float()).abs() <= 2.0 ** -7 * du.float().abs() + 1e-5).all() and (db - dc).abs().max() <= 70000 * 2.0 ** -22


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_widest_layers_and_scans(dtype):
    """2^20 inputs, outputs and channels: the last ones of each as exact as the first."""
    t, W = TYPES[dtype], 1 << 20
    gen = torch.Generator(device="cuda").manual_seed(9)

    def rand(*s):
        return torch.rand(s, generator=gen, device="cuda").to(t)
    half = torch.finfo(t).eps / 2
    for M, K, N in ((3, W, 2), (20, W, 3), (3, 2, W), (20, 5, W)):
        x, w, g = rand(M, K).requires_grad_(True), rand(N, K).requires_grad_(True), rand(M, N)
        y = ops.dense(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), g)
        x64, w64, g64 = x.detach().double(), w.detach().double(), g.double()
        for got, want, terms in ((y, x64 @ w64.t(), K), (dx, g64 @ w64, N), (dw, g64.t() @ x64, M)):
            # terms of one sign: every matrix instruction (16 terms at least) may truncate a unit in the last place of the sum so far, and so may each of its pieces
            assert ((got.double() - want).abs() <= (half + (terms / 16 * 6 + 8) * 2.0 ** -23) * want.abs()).all(), (M, K, N)
    for T, packed in ((1, False), (5, False), (9, True)):
        gate, x = (rand(2, T, 1) if not packed else rand(T, 1)).requires_grad_(True), (rand(2, T, W) if not packed else rand(T, W)).requires_grad_(True)
        cu = torch.tensor([0, 4, 8], device="cuda") if packed else None
        states, last = ops.gated_scan(gate, x, cu_seqlens=cu)
        dgate, dx = torch.autograd.grad(last, (gate, x), torch.ones_like(last))
        rows = [range(0, 4), range(4, 8)] if packed else [range(T)] * 2
        for s in range(2):
            a, v = (gate if packed else gate[s]).detach().double(), (x if packed else x[s]).detach().double()
            h = [torch.zeros(W, dtype=torch.float64, device="cuda")]
            for i in rows[s]:
                h.append(a[i] * h[-1] + v[i])
            f = torch.ones(W, dtype=torch.float64, device="cuda")
            assert ((last[s].double() - h[-1]).abs() <= 16 * 2.0 ** -23 * h[-1]).all()
            for k, i in reversed(list(enumerate(rows[s]))):
                got_x, got_a = (dx if packed else dx[s])[i].double(), (dgate if packed else dgate[s])[i].double()
                assert ((got_x - f).abs() <= (half + 16 * 2.0 ** -23) * f).all()
                want = (f * h[k]).sum()
                assert abs(got_a - want) <= (half + 2.6e-4) * want     # (2^20 terms in 4096 blocks of 256, then the blocks in order: 4096 + 20 roundings of 2^-24)
                f = f * a[i]
        if packed:
            assert (states[8:] == 0).all() and (dx[8:] == 0).all() and (dgate[8:] == 0).all()


def test_backward_twice_through_one_graph():
    for make in (dense_slices, packed_scan):
        out, leaves, cots = make()
        first = torch.autograd.grad(out, leaves, cots, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(out, leaves, cots)))
