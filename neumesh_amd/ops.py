"""Free-standing differentiable operators for models built around the field: dense layers of any width (feature, semantic or
appearance heads, other hidden widths) and the gated linear recurrence along rays or other sequences.

    dense(x, weight, bias, residual, activation=...)        act(x W^T + b) + r in one kernel, with its gradient
    gated_scan(gate, x, h0, cu_seqlens=..., blend=...)      h_i = gate_i h_{i-1} + x_i along sequences, with its gradient
    composite_features(alpha, features, background)         alpha compositing of any number of channels along rays

They stand beside the field's own layers (`NeuMesh`, fp32 tensors and fixed networks) and its own compositing (`volume_render`: rgb, depth,
normals): tensors are fp32, fp16 or bf16 on a HIP device, sums and states are fp32, results are rounded once.  Calls run on the
current stream of the tensors' device, do not synchronise, can be captured into a graph and give the same bits from run to run.  Their
gradients are not differentiable a second time, and tangents of forward-mode differentiation are refused.  A backward pass is captured
with leaves of its own (`detach().requires_grad_()`): where an eager graph of the same leaves still lives, autograd makes the captured
stream wait for that graph's, which ends the capture.
"""
from __future__ import annotations

import contextlib
import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
ACTIVATIONS = {"none": 0, "relu": 1, "softplus": 2, "sigmoid": 3, "silu": 4, "gelu_tanh": 5}   # NM_ACT_* (include/neumesh_hip.h)


_MAX_STRIDE = 1 << 24     # elements from row to row (nm_dense_*)


def _ptr(t):
    return None if t is None else t.data_ptr()


_SAME = contextlib.nullcontext()


def _on(dev):
    """The tensors' device as the current one (kernels are launched on it)."""
    return _SAME if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream(dev):
    """Handle of the device's current stream (torch.cuda.current_stream builds an object first: 3 us of a 17 us call)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _check(who, tensors, types):
    """Same HIP device for all; element types out of `types`."""
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{who}: {name} must be a tensor")
        if t.dtype not in types.get(name, _DTYPES):
            raise ValueError(f"{who}: {name} is {t.dtype}, expected one of {sorted(map(str, types.get(name, _DTYPES)))}")
        dev = dev or t.device
        if t.device != dev:
            raise ValueError(f"{who}: {name} is on {t.device}, the first tensor on {dev}")
    return dev


def _on_device(who, dev):
    if dev.type != "cuda":
        raise _lib.NeuMeshHipError(f"{who}: tensors must be on a HIP device (no CPU fallback)")


def _once(who):
    """Grad mode is on inside a backward pass only under create_graph=True: the gradients made here carry no graph, and a second derivative
    through them would silently be taken as zero."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{who}: its gradient cannot be differentiated again (backward with create_graph=True)")


def _no_tangents(who, *tensors):
    """Forward-mode differentiation is not offered: a tangent would be dropped silently, since a dual tensor need not require grad.  (The level is -1
    outside of every dual_level, the one thing that a call pays for.)"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{who}: forward-mode derivatives are not supported (an input carries a tangent)")


# ------------------------------------------------------------------------------------------------ dense layers
def _rows(t, n: int):
    """[..., n] as rows with a unit last stride -> (tensor [M, n], row stride in elements)."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), n)
    if t.is_contiguous():
        return t, n
    m, k = t.stride()
    if (n > 1 and k != 1) or (t.shape[0] > 1 and not n <= m <= _MAX_STRIDE):
        return t.contiguous(), n
    return t, (m if t.shape[0] > 1 else n)


def _dense_forward(x, weight, bias, residual, act: int, beta: float, want_deriv: bool):
    """-> (y, sizes and element type; rows of x, rows of the weight, act'(z))"""
    lib = _lib.load()
    N, K = weight.shape
    x2, ldx = _rows(x, K)
    w2, ldw = _rows(weight, K)
    M, dt, dev = x2.shape[0], _DTYPES[x.dtype], x.device
    y = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=dev)
    r2, ldr = (None, 0) if residual is None else _rows(residual, N)
    b = None if bias is None else bias.contiguous()
    deriv = torch.empty((M * N * (4 if dt == _lib.DTYPE_F32 else 3),), dtype=torch.uint8, device=dev) if want_deriv and act else None
    nbytes = lib.nm_dense_workspace_bytes(M, K, N, dt, 0)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes > 0 else None
    with _on(dev):
        _lib.check(lib.nm_dense_forward(x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(b), dt if b is None else _DTYPES[b.dtype], _ptr(r2), ldr, M, K, N, dt, act, beta,
                                        y.data_ptr(), N, _ptr(deriv), _ptr(ws), nbytes, _stream(dev)), "nm_dense_forward")
    return y, (M, K, N, dt), x2, w2, deriv


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, beta):
        need = ctx.needs_input_grad
        y, ctx.sizes, x2, w2, deriv = _dense_forward(x, weight, bias, residual, act, beta, need[0] or need[1] or need[2])
        ctx.save_for_backward(x2 if need[1] else None, w2 if need[0] else None, deriv)      # (released with the graph, and seen by hooks on saved tensors)
        ctx.x_shape, ctx.weight_dtype, ctx.bias_dtype = x.shape, weight.dtype, None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, g):
        # (runs on the engine's own thread, where every Python line costs twice: sizes come from the forward pass.  Strides do not: hooks on saved tensors, which
        # move them to the host and back, keep values and sizes only.)
        _once("dense")
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            lib, dev, empty = _lib.load(), g.device, torch.empty
            x2, w2, deriv = ctx.saved_tensors
            M, K, N, dt = ctx.sizes
            g2, ldg = (g, N) if g.is_contiguous() else _rows(g, N)
            x2, ldx = (None, K) if x2 is None else _rows(x2, K)
            w2, ldw = (None, K) if w2 is None else _rows(w2, K)
            if need_x:
                dx = empty(ctx.x_shape, dtype=ctx.weight_dtype, device=dev)
            if need_w:
                dw = empty((N, K), dtype=ctx.weight_dtype, device=dev)
            if need_b:
                db = empty((N,), dtype=ctx.bias_dtype, device=dev)
            nbytes = lib.nm_dense_workspace_bytes(M, K, N, dt, 1)
            ws = empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes > 0 else None
            with _on(dev):
                _lib.check(lib.nm_dense_backward(g2.data_ptr(), ldg, _ptr(deriv), _ptr(x2), ldx, _ptr(w2), ldw, M, K, N, dt, _ptr(dx), K, _ptr(dw), _ptr(db),
                                                 dt if db is None else _DTYPES[db.dtype], _ptr(ws), nbytes, _stream(dev)), "nm_dense_backward")
        return dx, dw, db, (g if need_r else None), None, None


def dense(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, *, activation: str = "none",
          beta: float = 100.0) -> torch.Tensor:
    """act(x weight^T + bias) + residual.

    x [..., K], weight [N, K] (as nn.Linear stores it), bias [N], residual [..., N] -> [..., N], all of one element type (fp32, fp16, bf16; the
    bias may be fp32 beside 16-bit rows); K, N <= 2^20.  activation: one of ACTIVATIONS; softplus is log(1 + exp(beta z)) / beta, beta in
    [2^-126, 2^126] (100 as in the geometry network), GELU its tanh form.  Differentiable in all four tensors: act'(z) is kept for the backward
    pass (3 bytes per output beside 16-bit rows, 4 beside fp32).  Rows may be strided (a column slice of a wider tensor); other layouts are copied.
    One row to many: up to 8 rows go through a form that reads the weights once and in place.
    fp32 products are as accurate as an fp32 matrix product; a non-finite operand makes the outputs it enters NaN there, and so in gradients
    beside an activation."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"dense: activation={activation!r}, expected one of {sorted(ACTIVATIONS)}")
    if not isinstance(x, torch.Tensor) or not isinstance(weight, torch.Tensor) or weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"dense: x [..., K] and weight [N, K] expected, got {tuple(getattr(x, 'shape', ()))} and {tuple(getattr(weight, 'shape', ()))}")
    same = {x.dtype} if x.dtype in _DTYPES else set(_DTYPES)
    dev = _check("dense", dict(x=x, weight=weight, bias=bias, residual=residual), dict(weight=same, residual=same, bias=same | {torch.float32}))
    N = weight.shape[0]
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"dense: bias has shape {tuple(bias.shape)}, expected ({N},)")
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], N):
        raise ValueError(f"dense: residual has shape {tuple(residual.shape)}, expected {(*x.shape[:-1], N)}")
    beta = float(beta)
    if activation == "softplus" and not 2.0 ** -126 <= beta <= 2.0 ** 126:      # (beta and 1 / beta are normal fp32 numbers)
        raise ValueError(f"dense: beta={beta} must be in [2^-126, 2^126]")
    _no_tangents("dense", x, weight, bias, residual)
    _on_device("dense", dev)
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or (residual is not None and residual.requires_grad)):
        return _Dense.apply(x, weight, bias, residual, act, beta)
    return _dense_forward(x, weight, bias, residual, act, beta, False)[0]


# ------------------------------------------------------------------------------------------------ gated linear recurrence
def _scan_sizes(x, cu):
    """(steps, sequences, channels) of x [B,T,D] or packed x [L,D]."""
    D = x.shape[-1]
    return (x.shape[0], cu.shape[0] - 1, D) if cu is not None else (x.shape[0] * x.shape[1], x.shape[0], D)


def _scan_forward(gate, x, h0, cu, reverse, blend, need_states, want_keep):
    lib = _lib.load()
    dev, dt = x.device, _DTYPES[x.dtype]
    L, S, D = _scan_sizes(x, cu)
    packed, shared = int(cu is not None), int(gate.shape[-1] != D)
    states = torch.empty_like(x) if need_states else None
    last = torch.empty((S, D), dtype=torch.float32, device=dev)
    keep = torch.empty((lib.nm_scan_keep_elems(L, S, D, dt, shared, packed),), dtype=torch.float32, device=dev) if want_keep else None
    nbytes = lib.nm_scan_workspace_bytes(L, S, D, dt, shared, packed)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes > 0 else None
    with _on(dev):
        _lib.check(lib.nm_scan_forward(gate.data_ptr(), _DTYPES[gate.dtype], shared, x.data_ptr(), dt, _ptr(h0), _ptr(cu), L, S, D, int(reverse),
                                       int(blend), _ptr(states), last.data_ptr(), _ptr(keep), _ptr(ws), nbytes, _stream(dev)), "nm_scan_forward")
    return states, last, keep


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, h0, cu, reverse, blend, need_states):
        ctx.set_materialize_grads(False)
        states, last, keep = _scan_forward(gate, x, h0, cu, reverse, blend, need_states, ctx.needs_input_grad[0] or cu is not None)
        ctx.save_for_backward(gate, x, h0, cu, keep)
        ctx.reverse, ctx.blend = reverse, blend
        return states, last

    @staticmethod
    def backward(ctx, g_states, g_last):
        _once("gated_scan")
        lib = _lib.load()
        gate, x, h0, cu, keep = (None if t is None else t.contiguous() for t in ctx.saved_tensors)      # (hooks on saved tensors keep values and sizes only)
        dev, dt = x.device, _DTYPES[x.dtype]
        L, S, D = _scan_sizes(x, cu)
        packed, shared = int(cu is not None), int(gate.shape[-1] != D)
        need_gate, need_x, need_h0 = ctx.needs_input_grad[:3]
        g_states = None if g_states is None else g_states.contiguous()
        g_last = None if g_last is None else g_last.contiguous()
        dgate = torch.empty_like(gate) if need_gate else None
        dx = torch.empty_like(x) if need_x else None
        dh0 = torch.empty_like(h0) if need_h0 else None
        nbytes = lib.nm_scan_workspace_bytes(L, S, D, dt, shared, packed)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes > 0 else None
        with _on(dev):
            _lib.check(lib.nm_scan_backward(gate.data_ptr(), _DTYPES[gate.dtype], shared, x.data_ptr(), dt, _ptr(h0), _ptr(cu), L, S, D,
                                            int(ctx.reverse), int(ctx.blend), _ptr(keep), _ptr(g_states), _ptr(g_last), _ptr(dgate), _ptr(dx), _ptr(dh0),
                                            _ptr(ws), nbytes, _stream(dev)), "nm_scan_backward")
        return dgate, dx, dh0, None, None, None, None


def gated_scan(gate: torch.Tensor, x: torch.Tensor, h0: Optional[torch.Tensor] = None, *, cu_seqlens: Optional[torch.Tensor] = None, reverse: bool = False,
               blend: bool = False, need_states: bool = True) -> Tuple[Optional[torch.Tensor], torch.Tensor]:
    """The linear recurrence h_i = gate_i h_{i-1} + x_i along sequences, every channel for itself -> (states, last).

    blend=True: h_i = (1 - gate_i) h_{i-1} + gate_i x_i.  reverse=True: from the last row of every sequence to its first.
    x [B,T,D]: B sequences of T rows; or x [L,D] with cu_seqlens [S+1] (int32 / int64, on the device, ascending): sequence s is rows
    cu_seqlens[s] .. cu_seqlens[s+1] - 1, rows outside belong to none (states and gradients 0).
    gate: as x, or [..., 1]: one for all channels of a row; of x's element type or fp32.  |gate| <= 1 (blend: 0 <= gate <= 1).
    h0 [B,D] / [S,D]: the state before each sequence (None = 0).  states as x (None with need_states=False: nothing is written), last [B,D] / [S,D]
    fp32: the state behind each sequence, h0 of the next call where a sequence goes on.  Differentiable in gate, x and h0.  Less than 2^31 rows and
    sequences, at most 2^20 channels."""
    if not isinstance(x, torch.Tensor) or not isinstance(gate, torch.Tensor):
        raise ValueError("gated_scan: gate and x must be tensors")
    packed = cu_seqlens is not None
    if x.dim() != (2 if packed else 3):
        raise ValueError(f"gated_scan: x [L,D] with cu_seqlens or [B,T,D] without expected, got {tuple(x.shape)}")
    D = x.shape[-1]
    if gate.shape[:-1] != x.shape[:-1] or gate.dim() != x.dim() or gate.shape[-1] not in (1, D):
        raise ValueError(f"gated_scan: gate has shape {tuple(gate.shape)}, expected {tuple(x.shape)} or {(*x.shape[:-1], 1)}")
    own = {x.dtype, torch.float32} if x.dtype in _DTYPES else set(_DTYPES)
    dev = _check("gated_scan", dict(x=x, gate=gate, h0=h0, cu_seqlens=cu_seqlens), dict(gate=own, cu_seqlens={torch.int32, torch.int64}))
    if packed and (cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1):
        raise ValueError("gated_scan: cu_seqlens must be a vector of at least one element")
    S = cu_seqlens.shape[0] - 1 if packed else x.shape[0]
    if h0 is not None and tuple(h0.shape) != (S, D):
        raise ValueError(f"gated_scan: h0 has shape {tuple(h0.shape)}, expected {(S, D)}")
    _no_tangents("gated_scan", gate, x, h0)
    _on_device("gated_scan", dev)
    h0 = None if h0 is None else h0.float().contiguous()
    cu = cu_seqlens.to(torch.int32).contiguous() if packed else None
    gate, x = gate.contiguous(), x.contiguous()
    if torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(gate, x, h0, cu, bool(reverse), bool(blend), bool(need_states))
    return _scan_forward(gate, x, h0, cu, bool(reverse), bool(blend), bool(need_states), False)[:2]


def composite_features(alpha: torch.Tensor, features: torch.Tensor, background: Optional[torch.Tensor] = None, *, cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Alpha compositing of any number of channels along rays: sum_i T_i alpha_i features_i + T_N background, T_i = prod_{j<i} (1 - alpha_j).

    alpha [R,N] and features [R,N,C] ordered near to far, as volume_render's detailed `alpha` and its samples are, or packed alpha [L] and
    features [L,C] with cu_seqlens [R+1] for rays with different numbers of samples.  alpha in [0,1], of the features' type or fp32; background [R,C].
    -> [R,C] fp32, differentiable in all three.  (volume_render's own `alpha` carries no gradient unless it composites with NEUMESH_COMPOSITE=torch: to
    train the geometry through these features, take alpha from the sdf with torch, as renderer.sdf_to_alpha does.)"""
    if not isinstance(alpha, torch.Tensor) or not isinstance(features, torch.Tensor) or alpha.shape != features.shape[:-1]:
        raise ValueError(f"composite_features: alpha {tuple(getattr(alpha, 'shape', ()))} must have the shape of features {tuple(getattr(features, 'shape', ()))} without channels")
    return gated_scan(alpha.unsqueeze(-1), features, background, cu_seqlens=cu_seqlens, reverse=True, blend=True, need_states=False)[1]
