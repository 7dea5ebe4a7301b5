"""The gated feed-forward product (gated.gated_linear; C ABI gated_linear, gated_linear_backward) against the formula in
64 bits, its gradients against the formula's and against differences.

Tolerances, with u = 2^-24 and e half a step of the 16-bit type (2^-11 or 2^-8). A projection's products are exact in
float32 and its K + 1 sums are off by at most 2 u each of the terms' sizes (an accumulator may truncate):
d = 2 u (K + 2) (sum |x w| + |b|). The activation moves that by at most 1.2 (its largest slope, and its slope's) and is
itself within 16 u of its value; the product has both factors' errors, and the result half a step of its own.
A gradient is made of dg and du with these errors and one rounding to the type (float16's smallest steps included), all
of which may add up; its own sums and rounding come on top. With random signs the roundings do not add up: the whole
error's 2-norm stays below 2 e of the result's."""
import math

import pytest
import torch

from comfy_ui_gfx906_tools_b200 import gated

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ACTS = list(gated.ACTIVATIONS)


def _act(g, name):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * k * (g + 0.044715 * g ** 3))
    return g * s, s + g * s * (1 - s) * 2 * k * (1 + 3 * 0.044715 * g * g)


def _reference(x, wg, wu, bg, bu, act, dh=None):
    """h and how far it may be off; with dh, the gradients of x, wg, wu, bg, bu."""
    X, G, W = (t.detach().double() for t in (x, wg, wu))
    b = [t.detach().double() if t is not None else torch.zeros(wg.shape[0], dtype=torch.float64, device=x.device)
         for t in (bg, bu)]
    g, u = X @ G.T + b[0], X @ W.T + b[1]
    k = 2 * U * (x.shape[1] + 2)
    far_g, far_u = (k * (X.abs() @ w.abs().T + c.abs()) for w, c in ((G, b[0]), (W, b[1])))
    a, da = _act(g, act)
    far_a = 1.2 * far_g + 16 * U * a.abs()
    h = a * u
    far = far_a * (u.abs() + far_u) + a.abs() * far_u
    e = HALF_STEP[x.dtype]
    far = far + e * (h.abs() + far) + 2.0 ** -24
    if dh is None:
        return h, far
    d, tiny = dh.double(), 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    dg, du = d * u * da, d * a
    off_g = d.abs() * 1.2 * (far_u + (u.abs() + far_u) * far_g) + (32 * U + e) * dg.abs() + tiny
    off_u = d.abs() * far_a + e * du.abs() + tiny

    def bounded(want, terms):
        """(want, its bound) from (|factor|, |other|, the factor's own error) of each product"""
        n = 2 * U * (len(terms) * terms[0][0].shape[1] + 2)
        far = sum(off @ other + n * (size @ other) for size, other, off in terms)
        return want, far + e * (want.abs() + far) + tiny

    one = torch.ones(x.shape[0], 1, dtype=torch.float64, device=x.device)
    weights = [bounded((t.T @ X), [(t.abs().T, X.abs(), o.T)]) for t, o in ((dg, off_g), (du, off_u))]
    biases = [bounded(t.sum(0)[:, None], [(t.abs().T, one, o.T)]) for t, o in ((dg, off_g), (du, off_u))]
    dx = bounded(dg @ G + du @ W, [(dg.abs(), G.abs(), off_g), (du.abs(), W.abs(), off_u)])
    return h, far, [dx, *weights, *((v[:, 0], o[:, 0]) for v, o in biases)]


def _inputs(cuda, M, K, F, dtype, bias, seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, wg, wu = make(M, K), make(F, K) / math.sqrt(K), make(F, K) / math.sqrt(K)
    b = [make(F) * 0.3, make(F) * 0.3] if bias else [None, None]
    leaves = [t.to(dtype).to(cuda).requires_grad_(True) if t is not None else None for t in (x, wg, wu, *b)]
    return leaves, (make(M, F) * 0.5).to(dtype).to(cuda)


def _close(got, want, far):
    d = (got.detach().double() - want).abs()
    assert bool((d <= far).all()), f"off by up to {float((d / far).max()):.3g} of what is allowed"


def _near(got, want, far, name):
    """Within the bound everywhere, within 2 e in the 2-norm; infinite where the exact value passes the type's range."""
    fine = torch.isfinite(want.to(got.dtype))
    assert torch.equal(torch.isfinite(got), fine), name
    _close(got[fine], want[fine], far[fine])
    norm = float(want[fine].norm())
    assert float((got[fine].detach().double() - want[fine]).norm()) <= 2 * HALF_STEP[got.dtype] * norm, name


SHAPES = [(1, 8, 8), (2, 2056, 72), (3, 64, 128), (17, 72, 1000), (33, 136, 264), (64, 512, 256), (129, 1032, 520),
          (300, 256, 1016), (513, 520, 136), (1000, 64, 384)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_without_gradient(cuda, shape, dtype):
    M, K, F = shape
    for act, bias in (("silu", False), ("gelu", True), ("gelu_tanh", True)):
        leaves, _ = _inputs(cuda, M, K, F, dtype, bias, 3)
        with torch.no_grad():
            h = gated.gated_linear(*leaves, activation=act)
        _close(h, *_reference(*leaves, act))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,bias", [("silu", True), ("gelu", False), ("gelu_tanh", True)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients(cuda, shape, act, bias, dtype):
    M, K, F = shape
    leaves, dh = _inputs(cuda, M, K, F, dtype, bias, 4)
    h = gated.gated_linear(*leaves, activation=act)
    want, far, grads = _reference(*leaves, act, dh)
    _close(h, want, far)
    named = [(n, t, g) for n, t, g in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), leaves, grads) if t is not None]
    got = torch.autograd.grad(h, [t for _, t, _ in named], dh)
    for (name, _, w), t in zip(named, got):
        _near(t, *w, name)


@pytest.mark.parametrize("shape", [(3, 64, 20000), (2600, 136, 6008), (1300, 1032, 4808), (5000, 72, 520)], ids=str)
def test_many_tiles(cuda, shape):
    """Several waves of tiles: the few-token kernel with more tiles than SMs, the products with one and two row blocks a
    tile, a contraction shorter than the pipeline, a last wave that is cut."""
    M, K, F = shape
    leaves, dh = _inputs(cuda, M, K, F, torch.bfloat16, True, 21)
    h = gated.gated_linear(*leaves)
    want, far, grads = _reference(*leaves, "silu", dh)
    _close(h, want, far)
    with torch.no_grad():
        assert torch.equal(gated.gated_linear(*leaves), h)
    for name, t, w in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), torch.autograd.grad(h, leaves, dh), grads):
        _near(t, *w, name)


def test_gradient_against_differences(cuda):
    """Along the gradient's own signs with an exact step, in float16: the slope is the sum of the gradient's sizes.
    A step of 2^-9 bends the value by parts in a thousand; h's rounding (2^-12 of each of 64 x 256 elements, random
    signs) over the step is parts in a thousand of the slope too."""
    M, K, F, h = 64, 128, 256, 2.0 ** -9
    leaves, dh = _inputs(cuda, M, K, F, torch.float16, True, 6)
    leaves = [(t.detach() * 256).round().div(256).requires_grad_(True) for t in leaves]  # t +- h is exact
    for act in ACTS:
        out = gated.gated_linear(*leaves, activation=act)
        grads = torch.autograd.grad(out, leaves, dh)
        for i, g in enumerate(grads):
            v = g.sign()
            with torch.no_grad():
                up, down = (gated.gated_linear(*leaves[:i], leaves[i] + s * h * v, *leaves[i + 1:], activation=act)
                            for s in (1, -1))
            slope = float(((up.double() - down.double()) * dh.double()).sum() / (2 * h))
            want = float(g.double().abs().sum())
            assert abs(slope - want) <= 2e-2 * want, (act, i, slope, want)


def test_operands_in_wider_matrices(cuda):
    """A fused [2F, K] weight's halves, tokens out of a wider row, a broadcast output gradient, and rows that no 16-byte
    access may touch give what their dense copies give."""
    g = torch.Generator().manual_seed(8)
    w = (torch.randn(2 * 264, 200, generator=g) / 14).to(torch.bfloat16).to(cuda)
    wide = torch.randn(70, 3, 208, generator=g).to(torch.bfloat16).to(cuda)
    for K, x in ((200, wide[:, 1, :200]), (192, wide[:, 1, 3:195])):
        wk = w[:, :K]
        views = [t.detach().requires_grad_(True) for t in (x, wk[:264], wk[264:])]
        dense = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in views]
        dh = torch.ones(264, device=cuda, dtype=torch.bfloat16).expand(70, 264)
        a, b = gated.gated_linear(*views), gated.gated_linear(*dense)
        assert torch.equal(a, b)
        for p, q in zip(torch.autograd.grad(a, views, dh), torch.autograd.grad(b, dense, dh.contiguous())):
            assert torch.equal(p, q)


def test_leading_dimensions_and_gradients_on_demand(cuda):
    """[B, L, K] tokens; gradients of x alone (frozen weights) or of one weight alone are those of the whole set."""
    leaves, dh = _inputs(cuda, 2 * 45, 72, 136, torch.bfloat16, True, 9)
    x = leaves[0].detach().view(2, 45, 72).requires_grad_(True)
    full = torch.autograd.grad(gated.gated_linear(x, *leaves[1:]), [x, *leaves[1:]], dh.view(2, 45, 136))
    assert full[0].shape == (2, 45, 72)
    for i in range(5):
        one = [t.detach().requires_grad_(j == i) for j, t in enumerate([x, *leaves[1:]])]
        h = gated.gated_linear(*one)
        assert h.shape == (2, 45, 136)
        assert torch.equal(torch.autograd.grad(h, one[i], dh.view(2, 45, 136))[0], full[i])


@pytest.mark.parametrize("M", [4, 70, 300])
@pytest.mark.parametrize("act", ACTS)
def test_far_gates(cuda, act, M):
    """Gates from -100 to 100: far negative ones keep their relative precision down to the type's smallest steps, far
    positive ones are the up projection; gradients follow, and are infinite only where the exact ones pass float16."""
    K, F = 64, 128
    x = torch.zeros(M, K, device=cuda, dtype=torch.float16)
    x[:, 0] = torch.linspace(-100, 100, M, device=cuda)
    x[:, 1] = 1
    wg, wu = torch.zeros(F, K, device=cuda, dtype=torch.float16), torch.zeros(F, K, device=cuda, dtype=torch.float16)
    wg[:, 0], wu[:, 1] = torch.linspace(0, 1, F, device=cuda), 2
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    h = gated.gated_linear(*leaves, activation=act)
    _close(h, *_reference(*leaves, None, None, act))
    with torch.no_grad():
        _close(gated.gated_linear(*leaves, activation=act), *_reference(*leaves, None, None, act))
    dh = torch.ones_like(h)
    _, _, want = _reference(*leaves, None, None, act, dh)
    for t, w in zip(torch.autograd.grad(h, leaves, dh), want):
        _near(t, *w, act)


@pytest.mark.parametrize("M", [5, 40, 400])
def test_rows_do_not_touch_each_other(cuda, M):
    """A NaN token and an infinite weight row: the other tokens' and features' results are what they are without."""
    leaves, dh = _inputs(cuda, M, 72, 264, torch.bfloat16, False, 12)
    with torch.no_grad():
        base = gated.gated_linear(*leaves)
        x, wg, wu = (t.detach().clone() if t is not None else None for t in leaves[:3])
        x[M // 2, 3] = float("nan")
        wu[100, 5] = float("inf")
        h = gated.gated_linear(x, wg, wu)
    keep = torch.ones(M, 264, dtype=torch.bool, device=cuda)
    keep[M // 2], keep[:, 100] = False, False
    assert torch.equal(h[keep], base[keep])
    assert bool(torch.isnan(h[M // 2]).all()) and not bool(torch.isfinite(h[:, 100]).any())


def test_repeats_bit_for_bit_and_on_another_stream(cuda):
    leaves, dh = _inputs(cuda, 700, 264, 520, torch.bfloat16, True, 13)

    def once():
        h = gated.gated_linear(*leaves)
        return [h, *torch.autograd.grad(h, leaves, dh)]

    first = once()
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        second = once()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_nothing_to_do(cuda):
    leaves, _ = _inputs(cuda, 3, 64, 72, torch.bfloat16, True, 14)
    x = torch.zeros(0, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    h = gated.gated_linear(x, *leaves[1:])
    assert h.shape == (0, 72)
    grads = torch.autograd.grad(h, [x, *leaves[1:]], torch.zeros_like(h))
    assert grads[0].shape == (0, 64) and all(bool((g == 0).all()) for g in grads[1:])


def test_module_is_its_parts(cuda):
    torch.manual_seed(3)
    mlp = gated.GatedMLP(64, 176, "gelu_tanh", bias=True, device=cuda)
    x = torch.randn(5, 7, 64, device=cuda).bfloat16()
    h = gated.gated_linear(x, mlp.gate.weight, mlp.up.weight, mlp.gate.bias, mlp.up.bias, "gelu_tanh")
    assert torch.equal(mlp(x), torch.nn.functional.linear(h, mlp.down.weight, mlp.down.bias))
    mlp(x).float().sum().backward()
    assert all(p.grad is not None for p in mlp.parameters())


def test_refusals(cuda):
    def call(x=(3, 64), wg=(72, 64), wu=(72, 64), bg=None, dt=torch.bfloat16, wdt=None, dev=cuda, act="silu"):
        z = lambda s, d: torch.zeros(s, dtype=d, device=cuda)  # noqa: E731
        return gated.gated_linear(torch.zeros(x, dtype=dt, device=dev), z(wg, wdt or dt), z(wu, wdt or dt),
                                  z(bg, dt) if bg else None, activation=act)

    call()
    for match, more in (("x must be on a CUDA device", dict(dev="cpu")), ("float16 or bfloat16", dict(dt=torch.float32)),
                        ("expected x", dict(wg=(72, 72))), ("expected x", dict(wu=(80, 64))),
                        ("K % 8", dict(x=(3, 60), wg=(72, 60), wu=(72, 60))),
                        ("F % 8", dict(wg=(70, 64), wu=(70, 64))), ("w_gate must be", dict(wdt=torch.float16)),
                        ("b_gate must have 72", dict(bg=(64,)))):
        with pytest.raises(RuntimeError, match=match):
            call(**more)
    with pytest.raises(ValueError, match="activation in"):
        call(act="relu")
    with pytest.raises(ValueError, match="activation in"):
        gated.GatedMLP(64, 64, "relu")
