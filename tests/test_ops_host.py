"""CPU: what neumesh_amd.ops refuses before any launch, and what the C entries refuse."""
import ctypes as C
import os
import sys

import numpy as np
import pytest
import torch

from neumesh_amd import _lib, ops


def test_dense_refuses_bad_arguments():
    x, w = torch.randn(4, 6), torch.randn(5, 6)
    for bad in (dict(activation="tanh"), dict(activation="softplus", beta=0.0), dict(activation="softplus", beta=float("nan"))):
        with pytest.raises(ValueError):
            ops.dense(x, w, **bad)
    for args in ((x, torch.randn(5, 7)), (x, torch.randn(6)), (x, w, torch.randn(4)), (x, w, None, torch.randn(4, 4)), (x, w, None, torch.randn(5)),
                 (x.double(), w.double()), (x.half(), w), (x, w, torch.randn(5).half()), (x.half(), w.half(), torch.randn(5).bfloat16()),
                 (x.half(), w.half(), None, torch.randn(4, 5)), (x.int(), w.int()), (x, [1.0]), (1.0, w), (torch.tensor(1.0), w)):
        with pytest.raises(ValueError):
            ops.dense(*args)


def test_scan_refuses_bad_arguments():
    a, x, cu = torch.rand(2, 5, 3), torch.randn(2, 5, 3), torch.tensor([0, 5], dtype=torch.int32)
    for args, kw in (((a[0], x), {}), ((a[:, :4], x), {}), ((a[..., :2], x), {}), ((a, x, torch.randn(2, 4)), {}), ((a, x, torch.randn(3, 3)), {}), ((a[0], x[0]), {}),
                     ((a, x), dict(cu_seqlens=cu)), ((a[0], x[0]), dict(cu_seqlens=cu.float())), ((a[0], x[0]), dict(cu_seqlens=cu[None])),
                     ((a[0], x[0]), dict(cu_seqlens=cu[:0])), ((a[0], x[0], torch.randn(2, 3)), dict(cu_seqlens=cu)), ((a.double(), x.double()), {}),
                     ((a.half(), x), {}), ((a.half(), x.bfloat16()), {}), ((None, x), {})):
        with pytest.raises(ValueError):
            ops.gated_scan(*args, **kw)
    with pytest.raises(ValueError):
        ops.composite_features(a, x)


def test_no_cpu_fallback():
    with pytest.raises(_lib.NeuMeshHipError, match="HIP device"):
        ops.dense(torch.randn(4, 6), torch.randn(5, 6))
    with pytest.raises(_lib.NeuMeshHipError, match="HIP device"):
        ops.gated_scan(torch.rand(2, 5, 3), torch.randn(2, 5, 3))


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_c_entries_refuse(dtype):
    """Invalid calls return an error before anything is launched (the pointers here are never followed)."""
    lib = _lib.load(require_device=False)
    p = C.c_void_p(4096)

    def fwd(x=p, ldx=8, w=p, ldw=8, bdt=dtype, r=None, ldr=0, M=20, K=8, N=4, dt=dtype, act=0, beta=1.0, y=p, ldy=4, ws=p, n=1 << 30):
        return lib.nm_dense_forward(x, ldx, w, ldw, None, bdt, r, ldr, M, K, N, dt, act, beta, y, ldy, None, ws, n, None)
    for bad in (dict(dt=3), dict(bdt=7), dict(act=6), dict(act=-1), dict(act=2, beta=0.0), dict(x=None), dict(w=None), dict(y=None), dict(ldx=7), dict(ldw=7), dict(ldy=3), dict(ldx=(1 << 24) + 1),
                dict(r=p, ldr=3), dict(M=-1), dict(K=-1), dict(N=-1), dict(K=(1 << 20) + 1, ldx=1 << 21, ldw=1 << 21), dict(K=4096, ldx=4096, ldw=4096, N=700, ldy=700, n=16),
                dict(K=4096, ldx=4096, ldw=4096, N=700, ldy=700, n=-1), dict(K=4096, ldx=4096, ldw=4096, N=700, ldy=700, ws=None)):
        assert fwd(**bad) == 1 and lib.nm_last_error(), bad
    assert fwd(M=0, x=None, y=None) == 0 and fwd(N=0, y=None) == 0

    def bwd(g=p, ldg=4, x=p, ldx=8, w=p, ldw=8, M=20, K=8, N=4, dt=dtype, dx=p, lddx=8, dw=p, db=p, bdt=dtype, ws=p, n=1 << 30):
        return lib.nm_dense_backward(g, ldg, None, x, ldx, w, ldw, M, K, N, dt, dx, lddx, dw, db, bdt, ws, n, None)
    for bad in (dict(g=None), dict(x=None), dict(w=None), dict(ldg=3), dict(ldx=7), dict(ldw=7), dict(lddx=7), dict(dt=5), dict(bdt=5), dict(M=3000, n=16), dict(M=3000, n=-1), dict(M=3000, ws=None), dict(M=-2)):
        assert bwd(**bad) == 1 and lib.nm_last_error(), bad
    assert bwd(dx=None, dw=None, db=None, g=None) == 0

    def scan(gate=p, gdt=dtype, x=p, dt=dtype, cu=None, L=12, S=3, D=4, last=p, ws=p, n=1 << 30):
        return lib.nm_scan_forward(gate, gdt, 0, x, dt, None, cu, L, S, D, 0, 0, None, last, None, ws, n, None)
    for bad in (dict(gate=None), dict(x=None), dict(last=None), dict(gdt=9), dict(dt=9), dict(L=13), dict(L=-1), dict(S=-1), dict(D=-1), dict(S=0), dict(L=1 << 31, S=1, D=1),
                dict(cu=p, n=4), dict(cu=p, ws=None)):
        assert scan(**bad) == 1 and lib.nm_last_error(), bad
    assert scan(D=0) == 0 and scan(L=0, S=0) == 0

    def back(gate=p, x=p, keep=p, dt=dtype, cu=None, L=12000, S=3, D=4, dgate=p, dx=p, dh0=p, ws=p, n=1 << 30):
        return lib.nm_scan_backward(gate, dt, 0, x, dt, None, cu, L, S, D, 0, 0, keep, None, None, dgate, dx, dh0, ws, n, None)
    for bad in (dict(gate=None), dict(x=None), dict(keep=None), dict(dt=9), dict(L=12001), dict(cu=p, n=4), dict(cu=p, ws=None)):
        assert back(**bad) == 1 and lib.nm_last_error(), bad
    assert back(dgate=None, dx=None, dh0=None) == 0
    for sizes in ((0, 0, 0), (0, 3, 3), (3, 0, 3), (3, 3, 0)):                # sizes of zero are answered
        assert lib.nm_dense_workspace_bytes(*sizes, dtype, 0) >= 0 and lib.nm_dense_workspace_bytes(*sizes, dtype, 1) >= 0
        assert lib.nm_scan_workspace_bytes(0, sizes[0], sizes[1], dtype, 0, 1) >= 0 and lib.nm_scan_keep_elems(0, sizes[0], sizes[1], dtype, 0, 0) >= 0
    assert lib.nm_dense_workspace_bytes(-1, 1, 1, dtype, 0) == -1 and lib.nm_scan_workspace_bytes(5, 2, 1, dtype, 0, 0) == -1 and lib.nm_scan_keep_elems(5, 2, 1, dtype, 0, 0) == -1


def test_workspaces_cover_every_subset_of_gradients():
    """The bias gradient alone runs on a plan of its own: the workspace of a backward pass has room for it beside dx."""
    lib = _lib.load(require_device=False)
    for M in (1, 9, 300, 70000):
        for N in (1, 100, 256, 1500):
            for K in (1, 130, 1024):
                assert lib.nm_dense_workspace_bytes(M, K, N, 2, 1) >= lib.nm_dense_workspace_bytes(M, 1, N, 2, 1)


def test_packed_rows_and_ranges():
    """The row -> sequence search and the starts / ends of partial reductions (nm_scan_index.h): right for ascending borders, inside the buffers
    whatever the borders hold."""
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    from hostcheck import loader
    lib = loader.load()
    rng = np.random.default_rng(0)
    L = 60
    for k in range(300):
        S = int(rng.integers(0, 9))
        good = k % 2 == 0
        cu = np.sort(rng.integers(0, L + 1, S + 1)) if good else rng.choice([-2 ** 31, -5, 0, 3, 30, L, L + 9, 2 ** 31 - 1], S + 1)
        cu = np.ascontiguousarray(cu, np.int32)
        rows = np.zeros(L, np.int32)
        lib.hc_scan_sequences(cu.ctypes.data, S, L, rows.ctypes.data)
        assert ((rows >= -1) & (rows < S)).all()
        if good:
            want = np.full(L, -1)
            for s in range(S):
                want[cu[s]:cu[s + 1]] = s
            assert (rows == want).all()
        for _ in range(20):
            c0 = int(rng.integers(0, L))
            c1 = int(rng.integers(c0 + 1, L + 1))
            for reverse in (0, 1):
                row = (lambda i: L - 1 - i) if reverse else (lambda i: i)
                lo = lib.hc_scan_reduce(cu.ctypes.data, int(rows[row(c1 - 1)]), reverse, L, c0, c1, 0)
                hi = lib.hc_scan_reduce(cu.ctypes.data, int(rows[row(c0)]), reverse, L, c0, c1, 1)
                assert c0 <= lo < c1 and c0 <= hi < c1
                if good:
                    seq = [int(rows[row(i)]) for i in range(c0, c1)]
                    first = c1 - 1
                    while first > c0 and seq[-1] >= 0 and seq[first - 1 - c0] == seq[-1]:
                        first -= 1
                    last = c0
                    while last < c1 - 1 and seq[0] >= 0 and seq[last + 1 - c0] == seq[0]:
                        last += 1
                    assert (lo, hi) == (first, last)


def test_launches_beyond_32_bits_of_threads_are_refused():
    """A launch's threads are counted in 32 bits: more is an error of the call's own, before anything is launched (the pointers are never followed)."""
    lib = _lib.load(require_device=False)
    p = C.c_void_p(4096)
    L, S, D = 1 << 30, 1 << 25, 2048                          # ranges of 32 steps x 8 blocks of channels: 2^28 workgroups
    assert lib.nm_scan_forward(p, 0, 0, p, 0, None, None, L, S, D, 0, 0, p, p, None, p, 1 << 62, None) == 1
    assert b"exceed one launch" in lib.nm_last_error()
    assert lib.nm_scan_backward(p, 0, 0, p, 0, None, None, L, S, D, 0, 0, p, p, p, p, p, p, p, 1 << 62, None) == 1
    assert b"exceed one launch" in lib.nm_last_error()
    assert lib.nm_dense_forward(p, 1024, p, 1024, None, 2, None, 0, 1 << 31, 1024, 1024, 2, 0, 1.0, p, 1024, None, p, 1 << 62, None) == 1     # 256 x 256 tiles
    assert b"exceed one launch" in lib.nm_last_error()


def test_tangents_are_refused():
    """Forward-mode derivatives: an error, with and without inputs that require grad, in every differentiable argument; never a result without its tangent."""
    from torch.autograd import forward_ad as fa
    x, w, b, r = torch.randn(4, 6), torch.randn(5, 6), torch.randn(5), torch.randn(4, 5)
    gate, v, h = torch.rand(2, 5, 3), torch.randn(2, 5, 3), torch.randn(2, 3)
    alpha, feats, bg = torch.rand(2, 5), torch.randn(2, 5, 3), torch.randn(2, 3)
    for fn, args in ((ops.dense, (x, w, b, r)), (ops.gated_scan, (gate, v, h)), (ops.composite_features, (alpha, feats, bg))):
        for i in range(len(args)):
            for leaf in (False, True):
                with fa.dual_level():
                    a = list(args)
                    a[i - 1] = a[i - 1].clone().requires_grad_(leaf)
                    a[i] = fa.make_dual(a[i], torch.ones_like(a[i]))
                    with pytest.raises(RuntimeError, match="forward-mode derivatives are not supported"):
                        fn(*a)
                    with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode derivatives are not supported"):
                        fn(*a)
        with fa.dual_level(), pytest.raises(_lib.NeuMeshHipError, match="HIP device"):      # no input with a tangent: the call goes on
            fn(*args)
    with pytest.raises(RuntimeError, match="forward-mode derivatives are not supported"):
        torch.func.jvp(lambda t: ops.dense(t, w), (x,), (x,))


def test_softplus_refuses_what_fp32_does_not_hold():
    """beta goes to the kernels in fp32, with its reciprocal: 1e39 would arrive as an infinity, 1e-46 as 0."""
    x, w = torch.randn(4, 6), torch.randn(5, 6)
    for beta in (1e39, 1e-46, 1e-40, 2.0 ** 127, -1.0, float("inf")):
        with pytest.raises(ValueError, match="beta"):
            ops.dense(x, w, activation="softplus", beta=beta)
        with pytest.raises(_lib.NeuMeshHipError, match="HIP device"):
            ops.dense(x, w, activation="silu", beta=beta)     # (ignored by the others)
    lib, p = _lib.load(require_device=False), C.c_void_p(4096)
    for beta in (float("inf"), 1e-40, 1.5e38):
        assert lib.nm_dense_forward(p, 8, p, 8, None, 0, None, 0, 20, 8, 4, 0, 2, beta, p, 4, None, p, 1 << 30, None) == 1 and b"beta" in lib.nm_last_error()
