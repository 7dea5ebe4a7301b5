"""Edges of q/k normalisation with rotary positions (rotary.qk_norm_rope): eps = 0 with heads that leave lanes and steps
without a row.

Tolerances, with u = 2^-24: a scale's gradient sums n products of a turned gradient (40 u of its pair's length) with a
normalised value (20 u of itself), so it is off by at most (n + 64) u of their sizes; dx has 64 u of its terms' sizes;
half a step of the output's type comes on top."""
import pytest
import torch

from comfy_ui_gfx906_tools_b200 import rotary

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def _turned(x, angle):
    """Neighbouring pairs turned, and each element's pair length."""
    y, size = x.clone(), x.abs()
    a, b = x[..., 0::2], x[..., 1::2]
    y[..., 0::2], y[..., 1::2] = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    size[..., 0::2] = size[..., 1::2] = torch.hypot(a, b)
    return y, size


def _close(got, want, far):
    got = got.detach().double().cpu()
    assert bool(torch.isfinite(got).all())
    d = (got - want).abs()
    assert bool((d <= far).all()), f"off by up to {float((d / far).max()):.3g} of what is allowed"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,KV,L,D", [(1, 3, 1, 5, 64), (2, 4, 2, 33, 64), (1, 9, 5, 700, 64), (1, 5, 1, 17, 128),
                                        (2, 1, 3, 6, 256), (1, 12, 4, 9, 72), (1, 1, 1, 3000, 8)])
def test_gradients_without_eps(cuda, B, H, KV, L, D, dtype):
    """eps = 0 is a plain RMS norm for rows that are not zero, whatever the number of heads: every gradient is finite
    and the formula's."""
    g = torch.Generator().manual_seed(41)
    q, k = (torch.randn(B, n, L, D, generator=g).to(dtype).to(cuda).requires_grad_(True) for n in (H, KV))
    ws = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype).to(cuda).requires_grad_(True) for _ in range(2)]
    dq, dk = (torch.randn(B, n, L, D, generator=g).to(dtype).to(cuda) for n in (H, KV))
    pos = torch.randint(0, 300, (L, 1), generator=g)
    out = rotary.qk_norm_rope(q, k, pos.to(cuda), (D,), 10000.0, *ws, eps=0.0)
    grads = torch.autograd.grad(out, [q, k, *ws], [dq, dk])
    angle = pos.double() * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    for x, w, dy, dx, dw in ((q, ws[0], dq, grads[0], grads[2]), (k, ws[1], dk, grads[1], grads[3])):
        x, w64 = x.detach().double().cpu(), w.detach().double().cpu()
        r = x.pow(2).mean(-1, keepdim=True).rsqrt()
        xh = x * r
        dz, size = _turned(dy.double().cpu(), -angle)
        want = (dz * xh).sum((0, 1, 2))
        far = (dz[..., 0].numel() + 64) * U * (size * xh.abs()).sum((0, 1, 2))
        _close(dw, want, far + HALF_STEP[dtype] * (want.abs() + far) + TINY[dtype])
        t = dz * w64
        want = r * (t - xh * (t * xh).mean(-1, keepdim=True))
        s = size * w64.abs()
        far = 64 * U * r * (s + xh.abs() * (s * xh.abs()).mean(-1, keepdim=True))
        _close(dx, want, far + HALF_STEP[dtype] * (want.abs() + far) + TINY[dtype])
