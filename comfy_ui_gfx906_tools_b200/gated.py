"""The gated feed-forward product of a transformer block, with gradients:
act(x Wg^T + bg) * (x Wu^T + bu) in float16 or bfloat16.

The reference's models leave it to their host framework (two linears, an
activation, a product). Here both projections, the activation and the product
are one kernel (csrc/gated.cu behind the C ABI ``gated_linear``), and the
backward is one elementwise kernel and two products
(``gated_linear_backward``). ``GatedMLP`` is the block around it.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib, ops

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [rows, cols] with contiguous, 16-byte aligned rows: t itself where it lies so (a slice of a wider matrix,
    say), else a copy."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _ptr(t: torch.Tensor | None):
    return t.data_ptr() if t is not None else None


def _forward(x, w_gate, w_up, b_gate, b_up, act, keep):
    """(h, the float32 projections that a backward wants: [2, M, F], or None)"""
    (M, K), N, dev = x.shape, w_gate.shape[0], x.device
    lib = _lib.load()
    h = x.new_empty((M, N))
    save = x.new_empty((2, M, N), dtype=torch.float32) if keep else None
    with ops._on(dev):
        stream, need = ops._stream(dev), lib.gated_linear_workspace_bytes(M, K, N)
        ws = ops._workspace(dev, stream, need) if need else None
        rc = lib.gated_linear(x.data_ptr(), x.stride(0), w_gate.data_ptr(), w_gate.stride(0), w_up.data_ptr(),
                              w_up.stride(0), _ptr(b_gate), _ptr(b_up), ops._DTYPE_CODE[x.dtype], act, h.data_ptr(),
                              _ptr(save), M, K, N, _ptr(ws), ws.numel() if need else 0, stream)
    if rc:
        ops._check_gemm("gated_linear", dev, rc)
    return h, save


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        h, save = _forward(x, w_gate, w_up, b_gate, b_up, act, True)
        ctx.act = act
        ctx.save_for_backward(x, w_gate, w_up, save)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, save = ctx.saved_tensors
        (M, K), N = x.shape, w_gate.shape[0]
        dh, dev, lib = _rows(dh), x.device, _lib.load()
        shapes = ((M, K), (N, K), (N, K), (N,), (N,))
        grads = [x.new_empty(s) if need else None for s, need in zip(shapes, ctx.needs_input_grad)]
        with ops._on(dev):
            ws = x.new_empty(lib.gated_linear_backward_workspace_bytes(M, K, N), dtype=torch.uint8)
            rc = lib.gated_linear_backward(
                dh.data_ptr(), dh.stride(0), x.data_ptr(), x.stride(0), w_gate.data_ptr(), w_gate.stride(0),
                w_up.data_ptr(), w_up.stride(0), save.data_ptr(), ops._DTYPE_CODE[x.dtype], ctx.act,
                *[g.data_ptr() if g is not None else None for g in grads], M, K, N, ws.data_ptr(), ws.numel(),
                ops._stream(dev))
        if rc:
            ops._check_gemm("gated_linear_backward", dev, rc)
        return (*grads, None)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                 b_up: torch.Tensor | None = None, activation: str = "silu") -> torch.Tensor:
    """act(x Wg^T + bg) * (x Wu^T + bu): x [..., K], w_gate / w_up [F, K],
    biases [F] or None, all of one dtype, float16 or bfloat16; returns [..., F].

    K and F are multiples of 8; rows may lie in a wider matrix (the two halves
    of a fused [2F, K] weight are read in place). activation: "silu", "gelu"
    or "gelu_tanh". Products accumulate in float32 and the result is rounded
    once. Differentiable in every tensor; a call that needs a gradient keeps
    both projections in float32 (8 bytes for each element of the result).
    Forward-mode derivatives are refused."""
    ops._require_cuda(x, "x")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"x must be float16 or bfloat16, got {x.dtype}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation in {list(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.shape[1] != x.shape[-1] or w_up.shape != w_gate.shape:
        raise RuntimeError(f"expected x [..., K], w_gate and w_up [F, K]; got x {tuple(x.shape)} w_gate "
                           f"{tuple(w_gate.shape)} w_up {tuple(w_up.shape)}")
    N, K = w_gate.shape
    if K % 8 or N % 8 or K == 0 or N == 0:
        raise RuntimeError(f"expected K % 8 == 0 and F % 8 == 0, got K={K} F={N}")
    dt, index = x.dtype, x.get_device()
    for t, name, shape in ((w_gate, "w_gate", None), (w_up, "w_up", None), (b_gate, "b_gate", (N,)),
                           (b_up, "b_up", (N,))):
        if t is None:
            continue
        if t.dtype is not dt or t.get_device() != index:
            raise RuntimeError(f"{name} must be {dt} on {x.device}, got {t.dtype} on {t.device}")
        if shape and t.shape != shape:
            raise RuntimeError(f"{name} must have {N} elements, got {tuple(t.shape)}")
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, K)
    if x2.shape[0] > 2 ** 30:
        raise RuntimeError(f"at most 2^30 tokens, got {x2.shape[0]}")
    args = (_rows(x2), _rows(w_gate), _rows(w_up), b_gate.contiguous() if b_gate is not None else None,
            b_up.contiguous() if b_up is not None else None)
    if (torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in args])) or ops._has_tangent(*args):
        h = _GatedLinear.apply(*args, ACTIVATIONS[activation])
    else:
        h = _forward(*args, ACTIVATIONS[activation], False)[0]
    return h if flat else h.reshape(*x.shape[:-1], N)


class GatedMLP(torch.nn.Module):
    """down(act(gate(x)) * up(x)): ``gated_linear`` and a plain down projection, with ``gate``, ``up`` and ``down``
    linears as the usual checkpoints name them."""

    def __init__(self, hidden: int, features: int, activation: str = "silu", bias: bool = False, device=None,
                 dtype=torch.bfloat16):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation in {list(ACTIVATIONS)}, got {activation!r}")
        self.activation = activation
        self.gate = torch.nn.Linear(hidden, features, bias=bias, device=device, dtype=dtype)
        self.up = torch.nn.Linear(hidden, features, bias=bias, device=device, dtype=dtype)
        self.down = torch.nn.Linear(features, hidden, bias=bias, device=device, dtype=dtype)

    def forward(self, x):
        h = gated_linear(x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias, self.activation)
        return F.linear(h, self.down.weight, self.down.bias)
