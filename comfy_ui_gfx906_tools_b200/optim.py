"""AdamW over many tensors in one launch, with moments in 32 or in 8 bits.

The reference's training code (nodes/ComfyUI-Gfx906Int4/train_linear.py) leaves
the optimizer to torch; these are the step a fine-tuning run takes here
(csrc/adamw.cu behind the C ABI ``adamw_step``):

  * ``AdamW``: a ``torch.optim.Optimizer`` over the functions below;
  * ``adamw_step`` / ``adamw_step_8bit``: the step on plain tensor lists;
  * ``moment_values``: what 8-bit moments stand for.

8-bit moments: one float32 scale s for each 256 consecutive elements of a
tensor. A first moment's code c in [-127, 127] stands for c |c| s. A second
moment's code c in [0, 255] stands for (c^2 s)^2: its root is held, so that the
ratio of the largest to the smallest held value is 255^4 within a block, and a
positive second moment keeps at least the code 1.
"""
from __future__ import annotations

import array
import operator

import torch

from . import _lib, ops

BLOCK = 256  # elements that share one scale of an 8-bit moment


def moment_scales(numel: int) -> int:
    """Scales that an 8-bit moment of ``numel`` elements has."""
    return -(-numel // BLOCK)


# Whole lists at a time, without a loop of Python's own: a step over many small tensors is bound by this side.
_DTYPES, _SHAPES, _DEVICES = operator.attrgetter("dtype"), operator.attrgetter("shape"), torch.Tensor.get_device
_NUMELS, _CONTIGUOUS, _ADDRESSES = torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.data_ptr


def _lists(params, others):
    """Checks the lists of one step: others is [(name, tensors, dtype or None for the first one's, scales)], the
    gradients first, which have the parameters' shapes, where the rest have their numbers of elements; returns
    (device, elements of each parameter), or None where there is nothing to do."""
    n = len(params)
    for name, tensors, _, _ in others:
        if len(tensors) != n:
            raise RuntimeError(f"{name} has {len(tensors)} tensors, params {n}")
    if n == 0:
        return None
    ops._require_cuda(params[0], "params[0]")
    dev, index, numel = params[0].device, params[0].get_device(), list(map(_NUMELS, params))
    ops._dtype_code(params[0].dtype)
    here, yes, shapes = [index] * n, [True] * n, list(map(_SHAPES, params))
    for name, tensors, dtype, scales in (("params", params, None, False), *others):
        dtype = dtype or tensors[0].dtype
        size, want = (_SHAPES, shapes) if name in ("params", "grads") else (
            _NUMELS, list(map(moment_scales, numel)) if scales else numel)
        if (list(map(_DTYPES, tensors)) != [dtype] * n or list(map(_DEVICES, tensors)) != here
                or (tensors is not params and list(map(size, tensors)) != want)
                or list(map(_CONTIGUOUS, tensors)) != yes):
            i = next(i for i, t in enumerate(tensors) if t.dtype != dtype or t.get_device() != index
                     or size(t) != want[i] or not t.is_contiguous())
            t, asked = tensors[i], f"shape {tuple(want[i])}" if want is shapes else f"{want[i]} elements"
            raise RuntimeError(f"{name}[{i}] must be contiguous, {dtype} on {dev} with {asked}; got {t.dtype} on "
                               f"{t.device}, {tuple(t.shape)}, strides {t.stride()}")
    return dev, numel


def _call(dev, numel, lists, bits, step, lr, betas, eps, weight_decay, grad_scale):
    """lists: params, grads, m, v and, with 8 bits, the moments' scales."""
    scale = None
    if grad_scale is not None:
        if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != dev:
            raise RuntimeError(f"grad_scale must be one float32 value on {dev}, got {grad_scale.dtype} "
                               f"{tuple(grad_scale.shape)} on {grad_scale.device}")
        scale = grad_scale.data_ptr()
    params, grads = lists[:2]
    n = len(params)
    # one host array: a row of pointers for each list, then the element counts
    table = array.array("Q")
    for tensors in lists:
        table.extend(map(_ADDRESSES, tensors))
    table.extend(numel)
    at = table.buffer_info()[0]
    where = [at + 8 * n * i for i in range(len(lists) + 1)]
    with ops._on(dev):
        _lib.call("adamw_step", *where[:4], *(where[4:6] if bits == 8 else (None, None)), where[-1], n,
                  ops._dtype_code(params[0].dtype), ops._dtype_code(grads[0].dtype), bits, int(step), float(lr),
                  float(betas[0]), float(betas[1]), float(eps), float(weight_decay), scale, ops._stream(dev))
    torch.autograd.graph.increment_version(params)  # autograd sees the kernel's write as any in-place change


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step: int, lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.01, grad_scale: torch.Tensor | None = None) -> None:
    """One AdamW step in place on lists of tensors.

    params: contiguous CUDA tensors of one dtype (float32 / float16 /
    bfloat16); grads: the same shapes, one dtype; exp_avgs, exp_avg_sqs:
    float32. ``step`` counts from 1. ``grad_scale`` (one float32 value on the
    device) multiplies every gradient, for clipping or unscaling without a
    pass of its own. No tensor may overlap another. Captured in a CUDA graph,
    the launch keeps the ``step`` and ``lr`` of the capture in every replay."""
    found = _lists(params, [("grads", grads, None, False), ("exp_avgs", exp_avgs, torch.float32, False),
                            ("exp_avg_sqs", exp_avg_sqs, torch.float32, False)])
    if found:
        _call(*found, (params, grads, exp_avgs, exp_avg_sqs), 32, step, lr, betas, eps, weight_decay, grad_scale)


def adamw_step_8bit(params, grads, m_codes, m_scales, v_codes, v_scales, *, step: int, lr: float, betas=(0.9, 0.999),
                    eps: float = 1e-8, weight_decay: float = 0.01, grad_scale: torch.Tensor | None = None) -> None:
    """``adamw_step`` with moments in 8 bits: m_codes int8 and v_codes uint8
    with a tensor's elements, m_scales and v_scales float32 with one value per
    256 elements (``moment_scales``). Zeros are a fresh state. The parameters
    move by the moments as computed, before they are rounded to codes."""
    found = _lists(params, [("grads", grads, None, False), ("m_codes", m_codes, torch.int8, False),
                            ("v_codes", v_codes, torch.uint8, False), ("m_scales", m_scales, torch.float32, True),
                            ("v_scales", v_scales, torch.float32, True)])
    if found:
        _call(*found, (params, grads, m_codes, v_codes, m_scales, v_scales), 8, step, lr, betas, eps, weight_decay,
              grad_scale)


def moment_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float32 values that 8-bit moments stand for, in codes' shape: int8
    codes are a first moment's, uint8 codes a second's."""
    ops._require_cuda(codes, "codes")
    if codes.dtype not in (torch.int8, torch.uint8):
        raise RuntimeError(f"codes must be int8 (first moment) or uint8 (second moment), got {codes.dtype}")
    if scales.dtype != torch.float32 or scales.numel() != moment_scales(codes.numel()) or scales.device != codes.device:
        raise RuntimeError(f"scales must be {moment_scales(codes.numel())} float32 values on {codes.device}, got "
                           f"{scales.dtype} {tuple(scales.shape)} on {scales.device}")
    c, s = codes.contiguous(), scales.contiguous()
    out = torch.empty(codes.shape, dtype=torch.float32, device=codes.device)
    with ops._on(codes.device):
        _lib.call("adamw_moment_values", c.data_ptr(), s.data_ptr(), out.data_ptr(), c.numel(),
                  int(codes.dtype == torch.uint8), ops._stream(codes.device))
    return out


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay on CUDA parameters; ``state_bits`` 32
    or 8 chooses how both moments are held. Each group's parameters move in as
    few launches as their number asks for (one per 56 tensors), separately for
    each pair of parameter and gradient dtype. ``step(grad_scale=...)`` as
    ``adamw_step``'s. ``step`` refuses to be captured in a CUDA graph: the
    step's number and bias corrections are arguments of the launch, and every
    replay would repeat the captured ones."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def add_param_group(self, param_group):
        """torch's, with the settings checked: the constructor's and the group's own."""
        own = {**self.defaults, **param_group}
        if own["state_bits"] not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {own['state_bits']}")
        if not (own["lr"] >= 0 and own["eps"] >= 0 and own["weight_decay"] >= 0
                and all(0 <= b < 1 for b in own["betas"])):
            raise ValueError(f"expected lr, eps, weight_decay >= 0 and betas in [0, 1); got lr={own['lr']} "
                             f"eps={own['eps']} weight_decay={own['weight_decay']} betas={own['betas']}")
        super().add_param_group(param_group)

    def _fresh(self, p: torch.Tensor, bits: int) -> dict:
        if bits == 32:
            return {"step": 0, "exp_avg": torch.zeros(p.shape, dtype=torch.float32, device=p.device),
                    "exp_avg_sq": torch.zeros(p.shape, dtype=torch.float32, device=p.device)}
        n = moment_scales(p.numel())
        return {"step": 0, "m_codes": torch.zeros(p.shape, dtype=torch.int8, device=p.device),
                "m_scales": torch.zeros(n, dtype=torch.float32, device=p.device),
                "v_codes": torch.zeros(p.shape, dtype=torch.uint8, device=p.device),
                "v_scales": torch.zeros(n, dtype=torch.float32, device=p.device)}

    def load_state_dict(self, state_dict):
        """torch's loader casts a parameter's state to the parameter's dtype;
        the moments keep their own."""
        super().load_state_dict(state_dict)
        index = {i: p for g, h in zip(state_dict["param_groups"], self.param_groups)
                 for i, p in zip(g["params"], h["params"])}
        for i, saved in state_dict["state"].items():
            p = index[i]
            self.state[p] = {k: (v.detach().clone().to(p.device) if torch.is_tensor(v) else v)
                             for k, v in saved.items()}

    @torch.no_grad()
    def step(self, closure=None, grad_scale: torch.Tensor | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for index in set().union(*(map(_DEVICES, group["params"]) for group in self.param_groups)):
            if index >= 0:
                with ops._on(torch.device("cuda", index)):
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW.step cannot be captured in a CUDA graph: every replay would take the "
                                           "captured step's number and learning rate")
        for group in self.param_groups:
            lists: dict = {}
            bits = group["state_bits"]
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    continue
                if grad.is_sparse:
                    raise RuntimeError("AdamW takes dense gradients")
                st = self.state[p]
                if not st:
                    st.update(self._fresh(p, bits))
                key = (p.device, p.dtype, grad.dtype, st["step"] + 1)
                lists.setdefault(key, []).append((p, grad.contiguous(), st))
            for (*_, step), items in lists.items():
                ps, gs, sts = zip(*items)
                more = dict(step=step, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                            weight_decay=group["weight_decay"], grad_scale=grad_scale)
                if bits == 32:
                    adamw_step(ps, gs, [s["exp_avg"] for s in sts], [s["exp_avg_sq"] for s in sts], **more)
                else:
                    adamw_step_8bit(ps, gs, *([s[k] for s in sts]
                                              for k in ("m_codes", "m_scales", "v_codes", "v_scales")), **more)
                for st in sts:  # a call that was refused is not a step
                    st["step"] = step
        return loss
