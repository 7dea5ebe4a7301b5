"""AdamW (optim.adamw_step, adamw_step_8bit, AdamW; C ABI adamw_step) on the GPU against the formula in 64 bits, and
the 8-bit coding against its own definition.

Tolerances. A float32 operation is off by at most u = 2^-24 of its result. The new first moment is a sum of two
products with a rounded coefficient each: at most 5 u of T = |b1 m| + |(1 - b1) g|; the second moment, with one product
more, 6 u of itself (its terms are positive). The update is a moment over a root: 5 u (moment), 3 u + u (half the
second moment's, and the root), and six more operations, at most 16 u of step T / denom; the parameter's own part has
three roundings. float16 / bfloat16 parameters add half a step of their type to that."""
import math

import numpy as np
import pytest
import torch

from comfy_ui_gfx906_tools_b200 import optim

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
SIZES = [(1,), (3, 85), (256,), (257,), (0,), (1000,), (8, 4097), (2, 3, 5, 7)]
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def _tensors(cuda, sizes, dtype, gdtype, seed, shift=0):
    """params, grads, m, v; every array starts `shift` elements past an allocation's start."""
    g = torch.Generator().manual_seed(seed)

    def make(size, scale, dt, square=False):
        x = torch.randn(math.prod(size) + shift, generator=g) * scale
        x = (x.square() if square else x).to(dt).to(cuda)
        return x[shift:].view(size)

    return ([make(s, 0.02, dtype) for s in sizes], [make(s, 1e-3, gdtype) for s in sizes],
            [make(s, 3e-4, torch.float32) for s in sizes], [make(s, 1e-3, torch.float32, True) for s in sizes])


def _formula(p, g, m, v, step, lr, betas, eps, weight_decay, scale=1.0):
    """p, m, v after the step in 64 bits, and how far 32 bits may be off each."""
    p64, g64, m, v = p.double(), g.double() * scale, m.double(), v.double()
    b1, b2 = betas
    t = (b1 * m).abs() + ((1 - b1) * g64).abs()
    m, v = b1 * m + (1 - b1) * g64, b2 * v + (1 - b2) * g64 * g64
    denom = (v / (1 - b2 ** step)).sqrt() + eps
    size = lr / (1 - b1 ** step)
    new = p64 * (1 - lr * weight_decay) - size * m / denom
    far = U * (4 * p64.abs() + 16 * size * t / denom + 2 * new.abs())
    return new, m, v, far + HALF_STEP[p.dtype] * (new.abs() + far) + TINY[p.dtype], 5 * U * t + 1e-45, 6 * U * v + 1e-45


def _close(got, want, far):
    d = (got.double() - want).abs()
    assert bool((d <= far).all()), f"off by up to {float((d / far).max()):.3g} of what is allowed"


@pytest.mark.parametrize("step", [1, 1000])
@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float32), (torch.float32, torch.bfloat16)])
def test_step_against_the_formula(cuda, dtype, gdtype, shift, step):
    p, g, m, v = _tensors(cuda, SIZES, dtype, gdtype, 5 + step, shift)
    want = [_formula(*x, step=step, **HYPER) for x in zip(p, g, m, v)]
    optim.adamw_step(p, g, m, v, step=step, **HYPER)
    for (wp, wm, wv, fp, fm, fv), a, b, c in zip(want, p, m, v):
        _close(a, wp, fp)
        _close(b, wm, fm)
        _close(c, wv, fv)


def test_many_tensors_take_several_launches(cuda):
    """More tensors than one launch's table holds (56), empty ones among them, each with its own size."""
    sizes = [(i % 7 * 37,) for i in range(150)]
    p, g, m, v = _tensors(cuda, sizes, torch.float32, torch.float32, 1)
    want = [_formula(*x, step=3, **HYPER) for x in zip(p, g, m, v)]
    optim.adamw_step(p, g, m, v, step=3, **HYPER)
    for (wp, wm, wv, fp, fm, fv), a, b, c in zip(want, p, m, v):
        _close(a, wp, fp)
        _close(b, wm, fm)
        _close(c, wv, fv)


def test_large_tensor(cuda):
    """Enough elements that a warp takes several blocks, in both forms."""
    size = (4_000_003,)
    p, g, m, v = _tensors(cuda, [size], torch.bfloat16, torch.bfloat16, 6)
    want = _formula(p[0], g[0], m[0], v[0], step=9, **HYPER)
    optim.adamw_step(p, g, m, v, step=9, **HYPER)
    for got, w, far in zip((p[0], m[0], v[0]), want[:3], want[3:]):
        _close(got, w, far)
    p, g, mc, ms, vc, vs, n = _eight(cuda, size, torch.bfloat16, torch.bfloat16, 7)
    m0, r0 = _value(mc.cpu(), ms.cpu()), _value(vc.cpu(), vs.cpu())
    want = _formula(p.cpu(), g.cpu(), m0, r0 * r0, step=9, **HYPER)
    gf, (b1, b2) = g.cpu().float(), HYPER["betas"]
    f = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    m1 = m0 * f(b1) + gf * f(1 - b1)
    v1 = r0 * r0 * f(b2) + gf * gf * f(1 - b2)
    optim.adamw_step_8bit([p], [g], [mc], [ms], [vc], [vs], step=9, **HYPER)
    _close(p.cpu(), want[0], want[3])
    for code, scale, x, top in ((mc, ms, m1, 127), (vc, vs, _sqrt(v1), 255)):
        wc, ws = _encode(x, top)
        assert torch.equal(code.cpu().float(), wc) and torch.equal(scale.cpu(), ws)


def test_neighbours_of_a_tensor_are_not_written(cuda):
    """Views of one buffer with a gap between them: the gaps keep their values."""
    buf = [torch.full((1000,), 7.0, device=cuda) for _ in range(4)]
    views = [[b[1:300], b[301:555], b[560:561]] for b in buf]
    optim.adamw_step(*views, step=1, **HYPER)
    gap = torch.ones(1000, dtype=torch.bool, device=cuda)
    for a, b in ((1, 300), (301, 555), (560, 561)):
        gap[a:b] = False
    for b in (buf[0], buf[2], buf[3]):
        assert bool((b[gap] == 7.0).all()) and bool((b[~gap] != 7.0).all())


def test_grad_scale_and_other_stream(cuda):
    p, g, m, v = _tensors(cuda, [(1000,)], torch.float32, torch.bfloat16, 9)
    scale = torch.tensor([0.25], device=cuda)
    want = _formula(p[0], g[0], m[0], v[0], step=2, scale=0.25, **HYPER)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        optim.adamw_step(p, g, m, v, step=2, grad_scale=scale, **HYPER)
    side.synchronize()
    _close(p[0], want[0], want[3])
    _close(m[0], want[1], want[4])


# ---------------------------------------------------------------------------------------------------------------
# 8-bit moments
# ---------------------------------------------------------------------------------------------------------------
def _sqrt(x):
    """Correctly rounded, which torch's own on the CPU is not always."""
    return torch.from_numpy(np.sqrt(x.numpy()))


def _encode(x, top):
    """The coding by its definition, one block of 256 at a time, in float32 on the CPU."""
    n = x.numel()
    b = torch.nn.functional.pad(x.reshape(-1), (0, -n % 256)).view(-1, 256)
    scale = b.abs().amax(1, keepdim=True) * torch.tensor(1.0 / (top * top))
    fine = scale >= 2.0 ** -126
    inv = torch.where(fine, 1.0 / torch.where(fine, scale, 1.0), 0.0)
    scale = torch.where(fine, scale, 0.0)
    code = _sqrt(b.abs() * inv).round().clamp(max=top)
    if top == 255:
        code = torch.where((b > 0) & fine, code.clamp(min=1), code)
    return (code * b.sign()).reshape(-1)[:n], scale.reshape(-1)


def _value(code, scale):
    c = code.float().reshape(-1)
    return c * c.abs() * scale.repeat_interleave(256)[:c.numel()]


def _eight(cuda, size, dtype, gdtype, seed, shift=0):
    (p,), (g,), (m,), (v,) = _tensors(cuda, [size], dtype, gdtype, seed, shift)
    n = p.numel()
    mc, ms = _encode(m.cpu(), 127)
    vc, vs = _encode(_sqrt(v.cpu()), 255)

    def at(x, dt):
        return torch.cat([torch.zeros(shift), x]).to(dt).to(cuda)[shift:].view(size)

    return p, g, at(mc, torch.int8), ms.to(cuda), at(vc, torch.uint8), vs.to(cuda), n


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("size", [(1,), (255,), (256,), (513,), (64, 1031)])
@pytest.mark.parametrize("dtype,gdtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16)])
def test_8bit_step_is_its_definition(cuda, dtype, gdtype, size, shift):
    """Codes and scales equal the definition computed in float32 on the CPU, bit for bit (every operation of the coding
    is correctly rounded); the parameters follow the formula in 64 bits."""
    p, g, mc, ms, vc, vs, n = _eight(cuda, size, dtype, gdtype, 11, shift)
    m0, r0 = _value(mc.cpu(), ms.cpu()), _value(vc.cpu(), vs.cpu())
    v0 = r0 * r0
    want = _formula(p.cpu().reshape(-1), g.cpu().reshape(-1), m0, v0, step=7, **HYPER)
    gf, (b1, b2) = g.cpu().float().reshape(-1), HYPER["betas"]
    f = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    m1 = m0 * f(b1) + gf * f(1 - b1)
    v1 = v0 * f(b2) + gf * gf * f(1 - b2)
    optim.adamw_step_8bit([p], [g], [mc], [ms], [vc], [vs], step=7, **HYPER)
    _close(p.cpu().reshape(-1), want[0], want[3])
    for code, scale, x, top in ((mc, ms, m1, 127), (vc, vs, _sqrt(v1), 255)):
        wc, ws = _encode(x, top)
        assert torch.equal(code.cpu().float().reshape(-1), wc)
        assert torch.equal(scale.cpu(), ws)
    assert torch.equal(optim.moment_values(mc, ms).cpu().reshape(-1), _value(mc.cpu(), ms.cpu()))
    r = _value(vc.cpu(), vs.cpu())
    assert torch.equal(optim.moment_values(vc, vs).cpu().reshape(-1), r * r)


def test_8bit_moments_are_within_half_a_code(cuda):
    """Against 64 bits: the root of |m| / scale is within half a code, plus what the float32 moment's own error (5 u of
    its terms) can move a root, which is at most the root of that error."""
    p, g, mc, ms, vc, vs, n = _eight(cuda, (4096,), torch.float32, torch.float32, 3)
    m0 = _value(mc.cpu(), ms.cpu())
    v0 = _value(vc.cpu(), vs.cpu()) ** 2
    _, m, v, _, fm, fv = _formula(p.cpu(), g.cpu(), m0, v0, step=7, **HYPER)
    optim.adamw_step_8bit([p], [g], [mc], [ms], [vc], [vs], step=7, **HYPER)
    sm, sv = (s.cpu().double().repeat_interleave(256) for s in (ms, vs))
    code = mc.cpu().double()
    assert bool(((m.abs() / sm).sqrt() - code.abs()).abs().le(0.5 + 1e-3 + (fm / sm).sqrt()).all())
    assert bool(((code == 0) | (code.sign() == m.sign())).all())
    root = (v.sqrt() / sv).sqrt()
    assert bool((root.clamp(min=1) - vc.cpu().double()).abs().le(0.5 + 1e-3).all())


def test_8bit_edges(cuda):
    """A fresh state; a block of zero gradients; gradients whose block is too small for a normal scale; a positive second
    moment far below its block's largest keeps the code 1; an infinite and a NaN gradient."""
    n = 256 * 5 + 10
    p = torch.ones(n, device=cuda)
    g = torch.zeros(n, device=cuda)
    g[256:512] = 1e-3
    g[300] = 1e4           # the others of the block lie 1e7 below
    g[512:768] = 1e-38
    g[800] = float("inf")
    g[1030] = float("nan")
    mc, vc = torch.zeros(n, dtype=torch.int8, device=cuda), torch.zeros(n, dtype=torch.uint8, device=cuda)
    ms, vs = torch.zeros(6, device=cuda), torch.zeros(6, device=cuda)
    optim.adamw_step_8bit([p], [g], [mc], [ms], [vc], [vs], step=1, lr=0.1, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0)
    assert bool((p[:256] == 1).all()) and int(mc[:256].abs().max()) == 0 and float(ms[0]) == 0 and float(vs[0]) == 0
    assert int(vc[256:512].min()) >= 1 and int(vc[300]) == 255 and int(mc[300]) == 127
    # the first step moves a parameter by lr whatever its gradient's size: an element of the outlier's block too
    assert bool(((p[256:512] - 0.9).abs() < 1e-3).all())
    assert bool((mc[512:768] == 0).all()) and bool(torch.isfinite(p[512:768]).all())
    bad = ~torch.isfinite(p)
    assert bool(bad[1030]) and int(bad.sum()) <= 2  # only where the gradient was not finite
    assert math.isnan(float(ms[3])) and math.isnan(float(vs[3])) and math.isnan(float(ms[4]))
    assert math.isfinite(float(ms[1])) and math.isfinite(float(ms[2])) and float(ms[5]) == 0
    optim.adamw_step_8bit([p], [g.zero_()], [mc], [ms], [vc], [vs], step=2, lr=0.1, betas=(0.9, 0.99))
    assert bool(torch.isnan(p[768:1280]).all()) and bool(torch.isfinite(p[:768]).all())  # loud, and only there


def test_optimizer_follows_the_functions_and_keeps_its_state(cuda):
    for bits in (32, 8):
        g = torch.Generator().manual_seed(2)
        w0 = [torch.randn(37, 19, generator=g), torch.randn(300, generator=g)]
        mine = [torch.nn.Parameter(x.to(cuda)) for x in w0] + [torch.nn.Parameter(torch.ones(4, device=cuda))]
        opt = optim.AdamW(mine, lr=1e-2, weight_decay=0.1, state_bits=bits)
        grads = [[torch.randn(x.shape, generator=g) for x in w0] for _ in range(4)]
        ref = [torch.nn.Parameter(x.clone()) for x in w0]
        ropt = torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.1)
        for i in range(4):
            if i == 2:  # through a state dict, into another optimizer over the same parameters
                saved = opt.state_dict()
                opt = optim.AdamW(mine, lr=1e-2, weight_decay=0.1, state_bits=bits)
                opt.load_state_dict(saved)
            for q, r, x in zip(mine, ref, grads[i]):
                q.grad, r.grad = x.to(cuda), x.clone()
            version = mine[0]._version
            opt.step()
            ropt.step()
            assert mine[0]._version > version
        assert bool((mine[2] == 1).all()) and mine[2] not in opt.state  # no gradient: not touched
        for q, r in zip(mine, ref):
            d = (q.detach().cpu() - r.detach()).abs().max()
            # four steps of at most 1.1 lr each; 8-bit moments are within half a code, under 1/8 of the value
            # wherever the code is 4 or more, and the updates of this test's normal gradients lie above that
            assert float(d) <= (1e-6 if bits == 32 else 0.25 * 4 * 1.1e-2)


def test_refusals(cuda):
    t = lambda *s, dt=torch.float32, dev=cuda: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
    more = dict(step=1, lr=1e-3)
    optim.adamw_step([], [], [], [], **more)  # nothing to do
    with pytest.raises(RuntimeError, match="exp_avgs has 0"):
        optim.adamw_step([t(4)], [t(4)], [], [t(4)], **more)
    with pytest.raises(RuntimeError, match="must be on a CUDA device"):
        optim.adamw_step(*([t(4, dev="cpu")] for _ in range(4)), **more)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        optim.adamw_step([t(4, dt=torch.float64)], [t(4)], [t(4)], [t(4)], **more)
    with pytest.raises(RuntimeError, match="contiguous"):
        optim.adamw_step([t(4, 4).t()[:, :2]], [t(8)], [t(8)], [t(8)], **more)
    with pytest.raises(RuntimeError, match=r"grads\[1\]"):
        optim.adamw_step([t(4), t(4)], [t(4), t(5)], [t(4), t(4)], [t(4), t(4)], **more)
    with pytest.raises(RuntimeError, match=r"exp_avgs\[0\].*float32"):
        optim.adamw_step([t(4)], [t(4)], [t(4, dt=torch.bfloat16)], [t(4)], **more)
    with pytest.raises(RuntimeError, match="step counts from 1"):
        optim.adamw_step([t(4)], [t(4)], [t(4)], [t(4)], step=0, lr=1e-3)
    with pytest.raises(RuntimeError, match="betas"):
        optim.adamw_step([t(4)], [t(4)], [t(4)], [t(4)], step=1, lr=1e-3, betas=(1.0, 0.9))
    with pytest.raises(RuntimeError, match="lr, eps"):
        optim.adamw_step([t(4)], [t(4)], [t(4)], [t(4)], step=1, lr=float("nan"))
    with pytest.raises(RuntimeError, match="grad_scale"):
        optim.adamw_step([t(4)], [t(4)], [t(4)], [t(4)], grad_scale=t(2), **more)
    with pytest.raises(RuntimeError, match=r"m_scales\[0\].*with 2 elements"):
        optim.adamw_step_8bit([t(257)], [t(257)], [t(257, dt=torch.int8)], [t(1)], [t(257, dt=torch.uint8)], [t(2)],
                              **more)
    with pytest.raises(RuntimeError, match="int8"):
        optim.moment_values(t(4), t(1))
    with pytest.raises(RuntimeError, match="2 float32 values"):
        optim.moment_values(t(257, dt=torch.int8), t(1))
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([torch.nn.Parameter(t(4))], state_bits=16)
