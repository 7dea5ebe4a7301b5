"""q/k RMS normalisation with multi-axis rotary positions, with gradients.

``flux_dit`` normalises q and k per head and turns them by axial rotary
positions in torch, some ten kernels each way (the reference leaves both to
its host framework's model). Here the two are one kernel (csrc/rotary.cu
behind the C ABI ``qk_norm_rope`` / ``qk_norm_rope_backward``): it reads q and
k where the packed qkv projection left them, computes in float32, rounds once,
and writes the [B, H, L, D] layout that attention takes.
"""
from __future__ import annotations

import array
import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

_POSITIONS = {torch.float32: 0, torch.int32: 1, torch.int64: 2}


@functools.lru_cache(maxsize=64)
def _axes(dims: tuple):
    return (ctypes.c_int * len(dims))(*[int(d) for d in dims])


def _strides(*lists):
    """One int64 array of three strides for each list, and the address of each."""
    flat = array.array("q")
    for x in lists:
        flat.extend(x[:3])
    at = flat.buffer_info()[0]
    return flat, range(at, at + 24 * len(lists), 24)


_NONE = (0, 0, 0)


def _of(t: torch.Tensor | None):
    return t.stride() if t is not None else _NONE


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
        return x.new_empty((B, L, H, D)).transpose(1, 2)
    return x.new_empty(x.shape)


def _forward(q, k, positions, pos_strides, q_scale, k_scale, call):
    B, H, L, D = q.shape
    dev = q.device
    code, scale_code, pos_code, kv, tail = call
    q_out = q.new_empty((B, H, L, D))
    q_strides, k_strides = (H * L * D, L * D, D), (kv * L * D, L * D, D)
    k_at = k_out_at = k_out = None
    if k is not None:
        k_out = q.new_empty((B, kv, L, D))
        k_at, k_out_at = k.data_ptr(), k_out.data_ptr()
    keep, (qs, ks, ps, qos, kos) = _strides(q.stride(), _of(k), pos_strides, q_strides, k_strides)
    with ops._on(dev):
        rc = _lib.load().qk_norm_rope(q.data_ptr(), qs, k_at, ks, code, positions.data_ptr(), pos_code, ps,
                                      _ptr(q_scale), _ptr(k_scale), scale_code, q_out.data_ptr(), qos, k_out_at, kos,
                                      B, H, kv, L, D, *tail, ops._stream(dev))
    if rc:
        raise _lib.GfxError("qk_norm_rope", rc, _lib.last_error())
    return q_out, k_out


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, q_scale, k_scale, pos_strides, call):
        ctx.pos_strides, ctx.call = pos_strides, call
        ctx.save_for_backward(q, k, positions, q_scale, k_scale)
        return _forward(q, k, positions, pos_strides, q_scale, k_scale, call)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, positions, q_scale, k_scale = ctx.saved_tensors
        B, H, L, D = q.shape
        dev, code, scale_code, pos_code, kv, tail = q.device, *ctx.call
        dq_out = _rows(dq_out)
        dk_out = _rows(dk_out) if k is not None else None
        dq, dk = _like_tokens(q), _like_tokens(k) if k is not None else None
        dqs = torch.empty_like(q_scale) if q_scale is not None and ctx.needs_input_grad[3] else None
        dks = torch.empty_like(k_scale) if k_scale is not None and ctx.needs_input_grad[4] else None
        keep, (dqo, dko, qs, ks, ps, dqi, dki) = _strides(dq_out.stride(), _of(dk_out), q.stride(), _of(k),
                                                          ctx.pos_strides, dq.stride(), _of(dk))
        with ops._on(dev):
            ws = None
            if dqs is not None or dks is not None:
                ws = q.new_empty(_lib.load().qk_norm_rope_workspace_bytes(D), dtype=torch.uint8)
            rc = _lib.load().qk_norm_rope_backward(
                dq_out.data_ptr(), dqo, _ptr(dk_out), dko, q.data_ptr(), qs, _ptr(k), ks, code, positions.data_ptr(),
                pos_code, ps, _ptr(q_scale), _ptr(k_scale), scale_code, dq.data_ptr(), dqi, _ptr(dk),
                dki, _ptr(dqs), _ptr(dks), B, H, kv, L, D, *tail, _ptr(ws), ws.numel() if ws is not None else 0,
                ops._stream(dev))
        if rc:
            raise _lib.GfxError("qk_norm_rope_backward", rc, _lib.last_error())
        return dq, dk, None, dqs, dks, None, None


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
    that tensor is not normalised). Differentiable in q, k and the scales
    (backward only; forward-mode derivatives are refused)."""
    index, dt, shape = q.get_device(), q.dtype, q.shape
    if index < 0:
        ops._require_cuda(q, "q")
    code = ops._dtype_code(dt)
    if len(shape) != 4:
        raise RuntimeError(f"q must be [B, H, L, D], got {tuple(shape)}")
    B, _, L, D = shape
    kv = 0
    if k is not None:
        other = k.shape
        if (len(other) != 4 or other[0] != B or other[2] != L or other[3] != D or k.dtype is not dt
                or k.get_device() != index):
            raise RuntimeError(f"k must be {dt} [{B}, KVH, {L}, {D}] on {q.device}, got {k.dtype} {tuple(other)} on "
                               f"{k.device}")
        kv = other[1]
    elif k_scale is not None:
        raise RuntimeError("k_scale without k")
    axes = _axes(tuple(axes_dims))
    n, pos_code = len(axes), _POSITIONS.get(positions.dtype)
    if pos_code is None:
        raise RuntimeError(f"positions must be float32, int32 or int64, got {positions.dtype}")
    if positions.get_device() != index:
        raise RuntimeError(f"positions must be on {q.device}, got {positions.device}")
    given, ps = positions.shape, positions.stride()
    if given == (L, n):
        ps = (0, *ps)
    elif given == (1, L, n):
        ps = (0, ps[1], ps[2])
    elif given != (B, L, n):
        raise RuntimeError(f"positions must be [{L}, {n}] or [{B}, {L}, {n}], got {tuple(given)}")
    scale_code = code
    first = q_scale if q_scale is not None else k_scale
    if first is not None:
        scale_type = first.dtype
        for s in (q_scale, k_scale):
            if s is not None and (s.numel() != D or s.dtype is not scale_type or s.get_device() != index):
                raise RuntimeError(f"scales must be [{D}] of one dtype on {q.device}, got {s.dtype} {tuple(s.shape)} on "
                                   f"{s.device}")
        scale_code = ops._dtype_code(scale_type)
        q_scale, k_scale = (s.contiguous() if s is not None else None for s in (q_scale, k_scale))
    q, k = _rows(q), _rows(k) if k is not None else None
    call = (code, scale_code, pos_code, kv, (axes, n, float(theta), int(interleaved), float(eps)))
    if ((torch.is_grad_enabled() and (q.requires_grad or any([t is not None and t.requires_grad
                                                             for t in (k, q_scale, k_scale)])))
            or ops._has_tangent(q, k, positions, q_scale, k_scale)):
        return _QkNormRope.apply(q, k, positions, q_scale, k_scale, ps, call)
    return _forward(q, k, positions, ps, q_scale, k_scale, call)
