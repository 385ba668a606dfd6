"""neumesh_amd.ops at the ends of its ranges: sizes beyond one launch, sums over nothing, cotangents and derivatives from the smallest to the largest numbers.
Tolerances are elementwise bounds from the arithmetic, as in test_gpu_ops.py."""
import pytest
import torch

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
