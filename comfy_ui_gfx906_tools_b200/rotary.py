"""q/k RMS normalisation with multi-axis rotary positions, with gradients.

``flux_dit`` normalises q and k per head and turns them by axial rotary
positions in torch, some ten kernels each way (the reference leaves both to
its host framework's model). Here the two are one kernel (csrc/rotary.cu
behind the C ABI ``qk_norm_rope`` / ``qk_norm_rope_backward``): it reads q and
k where the packed qkv projection left them, computes in float32, rounds once,
and writes the [B, H, L, D] layout that attention takes.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

_POSITIONS = {torch.float32: 0, torch.int32: 1, torch.int64: 2}


def _strides(t: torch.Tensor | None):
    return (ctypes.c_int64 * 3)(*t.stride()[:3]) if t is not None else None


def _ptr(t: torch.Tensor | None):
    return t.data_ptr() if t is not None else None


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with a contiguous last dimension, which is all that the kernel asks of its layout."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _like_tokens(x: torch.Tensor) -> torch.Tensor:
    """An empty [B, H, L, D] dense in x's own order of heads and tokens, so the gradient of heads cut out of a
    [B, L, H * D] projection lies as that projection does."""
    if x.stride(1) < x.stride(2):
        B, H, L, D = x.shape
        return torch.empty(B, L, H, D, dtype=x.dtype, device=x.device).transpose(1, 2)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, q_scale, k_scale, axes, theta, eps, interleaved):
        B, H, L, D = q.shape
        q_out = torch.empty(B, H, L, D, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=q.dtype, device=q.device) if k is not None else None
        scale = q_scale if q_scale is not None else k_scale
        code = ops._dtype_code(q.dtype)
        ctx.tail = (B, H, k.shape[1] if k is not None else 0, L, D, axes, len(axes), float(theta), int(interleaved),
                    float(eps))
        ctx.pos_args = (_POSITIONS[positions.dtype], (ctypes.c_int64 * 3)(*positions.stride()))
        ctx.codes = (code, ops._dtype_code(scale.dtype) if scale is not None else code)
        with torch.cuda.device(q.device):
            _lib.call("qk_norm_rope", q.data_ptr(), _strides(q), _ptr(k), _strides(k), code, positions.data_ptr(),
                      *ctx.pos_args, _ptr(q_scale), _ptr(k_scale), ctx.codes[1], q_out.data_ptr(), _strides(q_out),
                      _ptr(k_out), _strides(k_out), *ctx.tail, ops._stream(q.device))
        ctx.save_for_backward(q, k, positions, q_scale, k_scale)
        return q_out, k_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, positions, q_scale, k_scale = ctx.saved_tensors
        B, H, Hk, L, D = ctx.tail[:5]
        dq_out = _rows(dq_out)
        dk_out = _rows(dk_out) if k is not None else None
        dq, dk = _like_tokens(q), _like_tokens(k) if k is not None else None
        dqs = torch.empty_like(q_scale) if q_scale is not None and ctx.needs_input_grad[3] else None
        dks = torch.empty_like(k_scale) if k_scale is not None and ctx.needs_input_grad[4] else None
        with torch.cuda.device(q.device):
            ws = None
            if dqs is not None or dks is not None:
                ws = torch.empty(_lib.load().qk_norm_rope_workspace_bytes(D), dtype=torch.uint8, device=q.device)
            _lib.call("qk_norm_rope_backward", dq_out.data_ptr(), _strides(dq_out), _ptr(dk_out), _strides(dk_out),
                      q.data_ptr(), _strides(q), _ptr(k), _strides(k), ctx.codes[0], positions.data_ptr(),
                      *ctx.pos_args, _ptr(q_scale), _ptr(k_scale), ctx.codes[1], dq.data_ptr(), _strides(dq),
                      _ptr(dk), _strides(dk), _ptr(dqs), _ptr(dks), *ctx.tail, _ptr(ws),
                      ws.numel() if ws is not None else 0, ops._stream(q.device))
        return dq, dk, None, dqs, dks, None, None, None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, axes_dims, theta: float = 10000.0,
                 q_scale: torch.Tensor | None = None, k_scale: torch.Tensor | None = None, eps: float = 1e-6,
                 interleaved: bool = True):
    """(q, k) RMS-normalised per head row where they have a scale, then turned
    by rotary positions of several axes; contiguous [B, H, L, D] each.

    q [B, H, L, D], k [B, KVH, L, D] or None: float32 / float16 / bfloat16 of
    one dtype, any strides of batch, head and token (views of a packed qkv
    projection are read in place), D a multiple of 8 up to 256. positions
    [L, axes] or [B, L, axes], float32 / int32 / int64. axes_dims: the even
    number of elements each axis turns, in order; they may add up to less than
    D, the rest passes through. ``interleaved``: neighbouring elements form a
    pair (``flux_dit.apply_rope``'s layout), else element i and
    i + sum(axes_dims) / 2. Pair j of an axis of d elements turns by
    position * theta^(-2j/d). q_scale / k_scale [D]: the norm's scale (None:
    that tensor is not normalised). Differentiable in q, k and the scales."""
    for t, name in ((q, "q"), (k, "k")):
        if t is None:
            continue
        ops._require_cuda(t, name)
        ops._dtype_code(t.dtype)
        if t.dim() != 4:
            raise RuntimeError(f"{name} must be [B, H, L, D], got {tuple(t.shape)}")
    B, _, L, D = q.shape
    if k is not None and (k.shape[0] != B or k.shape[2] != L or k.shape[3] != D or k.dtype != q.dtype
                          or k.device != q.device):
        raise RuntimeError(f"k must be {q.dtype} [{B}, KVH, {L}, {D}] on {q.device}, got {k.dtype} {tuple(k.shape)} on "
                           f"{k.device}")
    axes = tuple(int(d) for d in axes_dims)
    if positions.dtype not in _POSITIONS:
        raise RuntimeError(f"positions must be float32, int32 or int64, got {positions.dtype}")
    if positions.device != q.device:
        raise RuntimeError(f"positions must be on {q.device}, got {positions.device}")
    if positions.dim() == 2:
        positions = positions[None]
    if positions.dim() != 3 or positions.shape[0] not in (1, B) or tuple(positions.shape[1:]) != (L, len(axes)):
        raise RuntimeError(f"positions must be [{L}, {len(axes)}] or [{B}, {L}, {len(axes)}], got "
                           f"{tuple(positions.shape)}")
    positions = positions.expand(B, L, len(axes))
    scales = [s for s in (q_scale, k_scale) if s is not None]
    for s in scales:
        if s.numel() != D or s.dtype != scales[0].dtype or s.device != q.device:
            raise RuntimeError(f"scales must be [{D}] of one dtype on {q.device}, got {s.dtype} {tuple(s.shape)} on "
                               f"{s.device}")
        ops._dtype_code(s.dtype)
    if k is None and k_scale is not None:
        raise RuntimeError("k_scale without k")
    q, k = _rows(q), _rows(k) if k is not None else None
    q_scale, k_scale = (s.contiguous() if s is not None else None for s in (q_scale, k_scale))
    return _QkNormRope.apply(q, k, positions, q_scale, k_scale, (ctypes.c_int * len(axes))(*axes), theta, eps,
                             interleaved)
