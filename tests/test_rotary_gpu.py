"""q/k normalisation with multi-axis rotary positions (rotary.qk_norm_rope; C ABI qk_norm_rope and
qk_norm_rope_backward) against the formula in 64 bits, and its gradient against the formula's and against differences.

Tolerances, with u = 2^-24. A normalised value is off by at most 20 u of itself (a sum of D <= 256 squares in at most
13 steps, the reciprocal root, three products); turning it adds 4 u for the sines (their angle's fraction of a turn is
rounded once) and 3 u for the arithmetic, of the pair's length: 40 u in all. The gradient has the same steps once more:
64 u of its terms' sizes. A scale's gradient adds n terms, at most (n + 64) u of their sizes. Half a step of the
output's type comes on top."""
import math

import pytest
import torch

from comfy_ui_gfx906_tools_b200 import flux_dit, rotary

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
EPS = 1e-6


def _angles(positions, axes, theta):
    out = []
    for a, d in enumerate(axes):
        f = theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        out.append(positions[..., a].double()[..., None] * f)
    return torch.cat(out, -1)[:, None]


def _turn(x, angle, interleaved):
    """(turned x, each element's pair length)"""
    r = 2 * angle.shape[-1]
    y, size = x.clone(), x.abs()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    size[..., first] = size[..., second] = torch.hypot(a, b)
    return y, size


def _reference(x, scale, angle, interleaved, dy=None):
    """y and how far it may be off; with dy, also dx, its bound, the scale's gradient and its bound."""
    x64 = x.detach().double().cpu()
    w = scale.detach().double().cpu() if scale is not None else None
    r = (x64.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    xh = x64 * r
    y, size = _turn(x64 if w is None else xh * w, angle, interleaved)
    far = 40 * U * size
    far = far + HALF_STEP[x.dtype] * (y.abs() + far) + TINY[x.dtype]
    if dy is None:
        return y, far
    dz, size = _turn(dy.double().cpu(), -angle, interleaved)
    if w is None:
        f = 40 * U * size
        return y, far, dz, f + HALF_STEP[x.dtype] * (dz.abs() + f) + TINY[x.dtype], None, None
    dw, dw_size = (dz * xh).sum((0, 1, 2)), (size * xh.abs()).sum((0, 1, 2))
    t = dz * w
    dx = r * (t - xh * (t * xh).mean(-1, keepdim=True))
    f = 64 * U * r * ((size * w.abs()) + xh.abs() * (size * w.abs() * xh.abs()).mean(-1, keepdim=True))
    n = dz[..., 0].numel()
    fw = (n + 64) * U * dw_size
    return (y, far, dx, f + HALF_STEP[x.dtype] * (dx.abs() + f) + TINY[x.dtype], dw,
            fw + HALF_STEP[scale.dtype] * (dw.abs() + fw) + TINY[scale.dtype])


def _close(got, want, far):
    d = (got.detach().double().cpu() - want).abs()
    assert bool((d <= far).all()), f"off by up to {float((d / far).max()):.3g} of what is allowed"


def _inputs(cuda, B, H, KV, L, D, dtype, layout, seed):
    """q, k of the layout, as leaves."""
    g = torch.Generator().manual_seed(seed)
    if layout == "packed":  # cut out of a projection [B, L, (H + 2 KV) D]
        y = torch.randn(B, L, (H + 2 * KV) * D, generator=g).to(dtype).to(cuda)
        q = y[..., :H * D].view(B, L, H, D).transpose(1, 2)
        k = y[..., H * D:(H + KV) * D].view(B, L, KV, D).transpose(1, 2)
    elif layout == "odd":   # rows that no 16-byte access may touch
        y = torch.randn(B, H + KV, L, D + 3, generator=g).to(dtype).to(cuda)[..., 1:D + 1]
        q, k = y[:, :H], y[:, H:]
    else:
        q, k = (torch.randn(B, n, L, D, generator=g).to(dtype).to(cuda) for n in (H, KV))
    return q.detach().requires_grad_(True), k.detach().requires_grad_(True)


def _positions(B, L, n, kind, seed):
    g = torch.Generator().manual_seed(seed + 1)
    if kind == "float":
        return torch.rand(B, L, n, generator=g) * 200 - 100
    if kind == "large":
        return torch.randint(0, 1 << 20, (B, L, n), generator=g)
    return torch.randint(-5, 300, (L, n), generator=g).to(torch.int32)


CASES = [
    # B, H, KV, L, D, axes, interleaved, (q scale, k scale), positions, layout
    (1, 24, 24, 33, 128, (16, 56, 56), True, (True, True), "int", "packed"),
    (2, 8, 2, 131, 64, (16, 24, 24), False, (True, True), "large", "packed"),
    (3, 5, 3, 17, 96, (32, 32), True, (False, False), "float", "plain"),
    (1, 3, 1, 40, 72, (24, 24, 24), False, (True, False), "int", "odd"),
    (2, 4, 4, 1, 256, (64, 64, 64, 64), True, (False, True), "large", "plain"),
    (1, 1, 1, 1, 8, (2,), True, (True, True), "int", "plain"),
    (1, 7, 2, 300, 80, (16, 32, 32), False, (True, True), "float", "odd"),
    (2, 2, 1, 9, 200, (30, 70), True, (True, True), "int", "plain"),
    (1, 3, 1, 6001, 64, (16, 24, 24), False, (True, True), "int", "packed"),  # more tokens than a backward's blocks hold
    (2, 5, 2, 1003, 128, (16, 56, 56), True, (True, True), "large", "odd"),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])))
def test_forward_and_gradient(cuda, case, dtype):
    B, H, KV, L, D, axes, interleaved, (qs, ks), kind, layout = case
    q, k = _inputs(cuda, B, H, KV, L, D, dtype, layout, 17)
    pos = _positions(B, L, len(axes), kind, 17)
    g = torch.Generator().manual_seed(4)
    scales = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype).to(cuda).requires_grad_(True) if on else None
              for on in (qs, ks)]
    dq, dk = (torch.randn(B, n, L, D, generator=g).to(dtype).to(cuda) for n in (H, KV))
    yq, yk = rotary.qk_norm_rope(q, k, pos.to(cuda), axes, 10000.0, *scales, eps=EPS, interleaved=interleaved)
    assert yq.is_contiguous() and yk.is_contiguous()
    leaves = [t for t in (q, k, *scales) if t is not None]
    grads = dict(zip(map(id, leaves), torch.autograd.grad([yq, yk], leaves, [dq, dk])))
    angle = _angles(pos if pos.dim() == 3 else pos.expand(B, L, len(axes)), axes, 10000.0)
    for x, w, y, dy in ((q, scales[0], yq, dq), (k, scales[1], yk, dk)):
        want, far, dx, far_dx, dw, far_dw = _reference(x, w, angle, interleaved, dy)
        _close(y, want, far)
        _close(grads[id(x)], dx, far_dx)
        if w is not None:
            _close(grads[id(w)], dw, far_dw)


@pytest.mark.parametrize("dtype,scale_dtype", [(torch.float32, torch.bfloat16), (torch.float16, torch.float32),
                                               (torch.bfloat16, torch.float16)])
def test_scales_of_another_type_and_heads_in_one(cuda, dtype, scale_dtype):
    """A scale of its own type; k as one head expanded over four: its gradient is their sum, made by autograd from the
    kernel's gradient of each."""
    q, _ = _inputs(cuda, 2, 3, 1, 21, 64, dtype, "plain", 30)
    g = torch.Generator().manual_seed(31)
    one = torch.randn(2, 1, 21, 64, generator=g).to(dtype).to(cuda).requires_grad_(True)
    w = (1 + 0.2 * torch.randn(64, generator=g)).to(scale_dtype).to(cuda).requires_grad_(True)
    pos = _positions(2, 21, 3, "int", 30)
    dq, dk = (torch.randn(2, n, 21, 64, generator=g).to(dtype).to(cuda) for n in (3, 4))
    yq, yk = rotary.qk_norm_rope(q, one.expand(2, 4, 21, 64), pos.to(cuda), (16, 24, 24), 10000.0, w, w)
    gq, gk, gw = torch.autograd.grad([yq, yk], [q, one, w], [dq, dk])
    angle = _angles(pos.expand(2, 21, 3), (16, 24, 24), 10000.0)
    want, far, dx, far_dx, dw, far_dw = _reference(q, w, angle, True, dq)
    _close(yq, want, far)
    _close(gq, dx, far_dx)
    want, far, dx, far_dx, dw2, far_dw2 = _reference(one.expand(2, 4, 21, 64), w, angle, True, dk)
    _close(yk, want, far)
    # autograd adds four gradients of the type, rounding each of three sums
    total = dx.sum(1, keepdim=True)
    _close(gk, total, far_dx.sum(1, keepdim=True) + 4 * HALF_STEP[dtype] * dx.abs().sum(1, keepdim=True))
    # the two scales' gradients, of the scale's type each, added in it
    _close(gw, dw + dw2, far_dw + far_dw2 + HALF_STEP[scale_dtype] * (dw + dw2).abs() * 1.01)


def test_gradient_against_differences(cuda):
    """Directional derivatives of sum(y dy): central differences with step h are off by h^2 / 6 of the third derivative
    (a row's norm is of order 1, so of the order of the value itself) and by the outputs' rounding over h."""
    q, k = _inputs(cuda, 2, 3, 2, 5, 64, torch.float32, "plain", 5)
    pos = _positions(2, 5, 3, "float", 5).to(cuda)
    g = torch.Generator().manual_seed(6)
    qs, ks = ((1 + 0.2 * torch.randn(64, generator=g)).to(cuda).requires_grad_(True) for _ in range(2))
    dq, dk = (torch.randn(2, n, 5, 64, generator=g).to(cuda) for n in (3, 2))

    def value(*leaves):
        a, b = rotary.qk_norm_rope(leaves[0], leaves[1], pos, (16, 24, 24), 100.0, *leaves[2:], eps=EPS,
                                   interleaved=False)
        return (a.double() * dq).sum() + (b.double() * dk).sum()

    leaves = (q, k, qs, ks)
    grads = torch.autograd.grad(value(*leaves), leaves)
    h = 1e-2
    for i, x in enumerate(leaves):
        v = torch.randn(x.shape, generator=g).to(cuda)
        with torch.no_grad():
            up = value(*leaves[:i], x + h * v, *leaves[i + 1:])
            down = value(*leaves[:i], x - h * v, *leaves[i + 1:])
        slope, want = float((up - down) / (2 * h)), float((grads[i].double() * v).sum())
        size = float((grads[i].double() * v).abs().sum())
        assert abs(slope - want) <= 1e-3 * size, (i, slope, want)


def test_equals_the_models_own_layers(cuda):
    """flux_dit's RMSNorm and apply_rope, which round to bfloat16 between their steps: within four of its half steps."""
    B, H, L, D, axes = 1, 4, 50, 128, (16, 56, 56)
    q, k = _inputs(cuda, B, H, H, L, D, torch.bfloat16, "packed", 8)
    norm = flux_dit.RMSNorm(D, device=cuda, dtype=torch.bfloat16)
    ids = torch.randint(0, 64, (B, L, 3), generator=torch.Generator().manual_seed(1)).float().to(cuda)
    pe = flux_dit.rope_tables(ids, axes, 10000.0)
    with torch.no_grad():
        got, _ = rotary.qk_norm_rope(q, k, ids, axes, 10000.0, norm.scale, norm.scale)
        want = flux_dit.apply_rope(norm(q), pe)
    size = _turn(want.double().cpu(), torch.zeros(B, 1, L, D // 2, dtype=torch.float64), True)[1]
    assert bool(((got - want).double().cpu().abs() <= 4 * 2.0 ** -8 * size + 1e-6).all())


def test_rows_do_not_touch_each_other(cuda):
    """A NaN row, an infinite one and one of zeros: every other row's output and gradient is what it is without them."""
    q, k = _inputs(cuda, 1, 4, 4, 6, 64, torch.float32, "plain", 9)
    pos = _positions(1, 6, 1, "int", 9).to(cuda)
    w = torch.ones(64, device=cuda)

    def both(x):
        x = x.detach().clone().requires_grad_(True)
        y, _ = rotary.qk_norm_rope(x, None, pos, (64,), q_scale=w)
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0]

    y0, d0 = both(q)
    x = q.detach().clone()
    x[0, 0, 0, 3], x[0, 1, 1, 5], x[0, 2, 2] = float("nan"), float("inf"), 0.0
    y1, d1 = both(x)
    same = torch.ones(1, 4, 6, dtype=torch.bool, device=cuda)
    same[0, 0, 0] = same[0, 1, 1] = same[0, 2, 2] = False
    assert torch.equal(y0[same], y1[same]) and torch.equal(d0[same], d1[same])
    assert bool(torch.isnan(y1[0, 0, 0]).all())
    assert bool((y1[0, 2, 2] == 0).all()) and bool(torch.isfinite(d1[0, 2, 2]).all())


def test_repeats_bit_for_bit_and_on_another_stream(cuda):
    q, k = _inputs(cuda, 2, 6, 2, 700, 128, torch.bfloat16, "packed", 10)
    pos = _positions(2, 700, 3, "large", 10).to(cuda)
    w = torch.ones(128, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    dq, dk = torch.randn(2, 6, 700, 128, device=cuda).bfloat16(), torch.randn(2, 2, 700, 128, device=cuda).bfloat16()

    def once():
        y = rotary.qk_norm_rope(q, k, pos, (16, 56, 56), q_scale=w, k_scale=w)
        return [*y, *torch.autograd.grad(y, [q, k, w], [dq, dk])]

    first = once()
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        second = once()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("B,H,L", [(0, 2, 3), (1, 2, 0)])
def test_nothing_to_do(cuda, B, H, L):
    x = torch.zeros(B, H, L, 64, device=cuda, requires_grad=True)
    w = torch.ones(64, device=cuda, requires_grad=True)
    y, none = rotary.qk_norm_rope(x, None, torch.zeros(L, 1, device=cuda), (64,), q_scale=w)
    assert none is None and y.shape == x.shape
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert dx.shape == x.shape and bool((dw == 0).all())


def test_refusals(cuda):
    def call(q=(1, 2, 3, 64), k=(1, 1, 3, 64), pos=(3, 1), axes=(64,), dt=torch.float32, kdt=None, pdt=torch.float32,
             dev=cuda, **more):
        return rotary.qk_norm_rope(torch.zeros(q, dtype=dt, device=dev),
                                   torch.zeros(k, dtype=kdt or dt, device=cuda) if k else None,
                                   torch.zeros(pos, dtype=pdt, device=cuda), axes, **more)

    call()
    for match, more in (("q must be on a CUDA device", dict(dev="cpu")),
                        ("unsupported dtype", dict(dt=torch.float64)),
                        (r"must be \[B, H, L, D\]", dict(q=(2, 3, 64))),
                        ("k must be", dict(k=(1, 1, 4, 64))),
                        ("k must be", dict(kdt=torch.float16)),
                        ("positions must be float32", dict(pdt=torch.float64)),
                        (r"positions must be \[3, 1\]", dict(pos=(4, 1))),
                        (r"positions must be \[3, 2\]", dict(axes=(32, 32))),
                        ("multiple of 8", dict(q=(1, 2, 3, 20), k=None, axes=(4,))),
                        ("multiple of 8", dict(q=(1, 2, 3, 264), k=None, axes=(4,))),
                        ("even", dict(axes=(5,))),
                        ("add up to 66", dict(axes=(66,))),
                        ("split halves", dict(axes=(12,), interleaved=False)),
                        ("theta", dict(theta=0.0)),
                        ("eps", dict(eps=-1.0)),
                        ("scales must be", dict(q_scale=torch.ones(32, device=cuda))),
                        ("scales must be", dict(q_scale=torch.ones(64, device=cuda),
                                                k_scale=torch.ones(64, device=cuda, dtype=torch.float16))),
                        ("k_scale without k", dict(k=None, k_scale=torch.ones(64, device=cuda)))):
        with pytest.raises(RuntimeError, match=match):
            call(**more)


def test_angles_of_large_positions(cuda):
    """A position of 2^24 - 1 on the fastest pair: the fraction of a turn is kept (float32 could not hold the angle)."""
    x = torch.zeros(1, 1, 1, 8, device=cuda)
    x[..., 0] = 1
    p = (1 << 24) - 1
    y, _ = rotary.qk_norm_rope(x, None, torch.tensor([[p]], device=cuda), (2,))
    assert abs(float(y[0, 0, 0, 0]) - math.cos(p)) <= 8 * U and abs(float(y[0, 0, 0, 1]) - math.sin(p)) <= 8 * U
