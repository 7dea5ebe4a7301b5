"""Edges of q/k normalisation with rotary positions (rotary.qk_norm_rope): eps = 0 with heads that leave lanes and steps
without a row, and infinities and NaN among the elements that pass through.

Tolerances, with u = 2^-24: a scale's gradient sums n products of a turned gradient (40 u of its pair's length) with a
normalised value (20 u of itself), so it is off by at most (n + 64) u of their sizes; dx has 64 u of its terms' sizes;
half a step of the output's type comes on top. Where a value has to be untouched by a neighbour, bits are compared."""
import math

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


PARTLY = [(96, (32, 32), True), (96, (32, 32), False), (200, (30, 70), True), (16, (6,), True), (16, (8,), False),
          (256, (2,), True), (72, (24, 24), False)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,axes,interleaved", PARTLY, ids=str)
def test_elements_that_pass_through_are_left_alone(cuda, D, axes, interleaved, dtype):
    """Without a norm, an infinity or NaN past the rotated elements comes out as it went in and reaches no other
    element, in either direction."""
    B, H, L, r = 2, 5, 11, sum(axes)
    g = torch.Generator().manual_seed(43)
    x = torch.randn(B, H, L, D, generator=g).to(dtype).to(cuda)
    dy = torch.randn(B, H, L, D, generator=g).to(dtype).to(cuda)
    pos = torch.randint(1, 300, (L, len(axes)), generator=g).to(cuda)
    mark = torch.zeros(B, H, L, D, dtype=torch.bool)
    for i, v in enumerate((math.inf, -math.inf, math.nan)):
        mark.view(-1, D)[i::3, r + i % (D - r)] = True
        mark.view(-1, D)[i::7, D - 1] = True
    mark = mark.to(cuda)
    bad = torch.tensor([math.inf, -math.inf, math.nan]).to(dtype).to(cuda)[torch.arange(B * H * L, device=cuda) % 3]
    bad = bad.view(B, H, L, 1).expand(B, H, L, D)

    def both(x, dy):
        x = x.detach().clone().requires_grad_(True)
        y, _ = rotary.qk_norm_rope(x, None, pos, axes, interleaved=interleaved)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    y0, d0 = both(x, dy)
    y1, d1 = both(torch.where(mark, bad, x), torch.where(mark, bad, dy))
    for base, got in ((y0, y1), (d0, d1)):
        assert torch.equal(base[~mark], got[~mark])
        assert torch.equal(got[mark].nan_to_num(7.0, 8.0, 9.0), bad[mark].nan_to_num(7.0, 8.0, 9.0))


@pytest.mark.parametrize("D,axes,interleaved", PARTLY, ids=str)
def test_norm_with_an_infinite_element_that_passes_through(cuda, D, axes, interleaved):
    """The norm takes such a row's finite elements to 0 (they are divided by an infinite root) and leaves inf / inf, a
    NaN, in its own place alone. An infinite gradient of one such element makes that element's scale gradient
    infinite and no other's."""
    r = sum(axes)
    g = torch.Generator().manual_seed(44)
    x = torch.randn(1, 2, 3, D, generator=g).to(cuda)
    x[0, 1, 1, r] = math.inf
    pos = torch.randint(1, 300, (3, len(axes)), generator=g).to(cuda)
    w = torch.ones(D, device=cuda)
    y, _ = rotary.qk_norm_rope(x, None, pos, axes, q_scale=w, interleaved=interleaved)
    row = y[0, 1, 1]
    assert bool(torch.isnan(row[r])) and bool((row[torch.arange(D, device=cuda) != r] == 0).all())
    assert bool(torch.isfinite(y[0, 0]).all())

    x = torch.randn(1, 2, 3, D, generator=g).to(cuda)
    w.requires_grad_(True)
    y, _ = rotary.qk_norm_rope(x, None, pos, axes, q_scale=w, interleaved=interleaved)
    dy = torch.randn(1, 2, 3, D, generator=g).to(cuda)
    base = torch.autograd.grad(y, w, dy, retain_graph=True)[0]
    dy[0, 1, 2, r] = math.inf
    dw = torch.autograd.grad(y, w, dy)[0]
    others = torch.arange(D, device=cuda) != r
    assert torch.equal(dw[others], base[others]) and bool(torch.isinf(dw[r]))


def test_forward_mode_is_refused(cuda):
    """No tangent is lost in silence: there is no forward-mode derivative, and a call with one says so."""
    x, pos = torch.randn(1, 2, 3, 64, device=cuda), torch.zeros(3, 1, device=cuda)
    w = torch.ones(64, device=cuda)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward"):
            rotary.qk_norm_rope(dual, None, pos, (64,))
        with pytest.raises(RuntimeError, match="forward"):
            rotary.qk_norm_rope(x, None, pos, (64,), q_scale=torch.autograd.forward_ad.make_dual(w, w))
        rotary.qk_norm_rope(x, None, pos, (64,))  # a call without a tangent goes through
