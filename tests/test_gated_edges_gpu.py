"""Edges of the gated feed-forward product (gated.gated_linear): far negative gates against their own size,
joins of a cut contraction with many tokens, forward-mode derivatives, a workspace that grows after a CUDA graph was
captured, one that is made inside a capture, and one launch of several seconds."""
import math

import pytest
import torch

from comfy_ui_gfx906_tools_b200 import gated, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half the smallest step
ACTS = list(gated.ACTIVATIONS)
K2 = 2 * math.sqrt(2 / math.pi)


def _act(g, name):
    """a, a' as its two terms, and the size of the exponential's argument, in 64 bits without cancellation."""
    if name == "silu":
        s, t, e = torch.sigmoid(g), torch.sigmoid(-g), g.abs()
        return g * s, (s, g * s * t), e
    if name == "gelu":
        c, e = 0.5 * torch.erfc(-g / math.sqrt(2)), g * g / 2
        return g * c, (c, g * torch.exp(-e) / math.sqrt(2 * math.pi)), e
    y = K2 * (g + 0.044715 * g ** 3)
    s, t = torch.sigmoid(y), torch.sigmoid(-y)
    return g * s, (s, g * s * t * K2 * (1 + 3 * 0.044715 * g * g)), y.abs()


def _relative(e):
    """How far an activation may be off, of its value, where its exponential's argument has the size e.

    CUDA's fast exponential is documented to 2 + 1.173 e steps (2 u each), its fast division to 2; the argument has up
    to four roundings (u of e each, which the exponential turns into a relative error), the rest some ten (u each).
    Phi's polynomial is within 2e-6."""
    return (2 * (2 + 1.173 * e) + 4 + 4 * e + 10) * U + 2e-6


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 40, 160])
def test_far_gates_keep_their_precision(cuda, act, M, dtype):
    """Every gate is one exact product and every up projection is 2 or 1, so a result is off by its activation and its
    own rounding alone, of its own size, however small that is; the same for dg and du, which one token's weight
    gradients show as they are (a sum of one product with 1). a' is a sum of two terms: the error is of their sizes."""
    K, F = 72, 8192
    gates = torch.cat([-torch.linspace(0, 6, F // 2), -torch.linspace(6, 100, F // 2)]).to(dtype)
    x, wg, wu = torch.zeros(M, K, dtype=dtype), torch.zeros(F, K, dtype=dtype), torch.zeros(F, K, dtype=dtype)
    x[:, 0] = 1 - 0.25 * (torch.arange(M) % 2)
    x[:, 1] = 1
    wg[:, 0] = gates
    wu[:, 1] = 1 + torch.arange(F) % 2
    x, wg, wu = (t.to(cuda) for t in (x, wg, wu))
    g = x[:, :1].double() * wg[:, 0].double()
    u = wu[:, 1].double().expand(M, F)
    a, terms, e = _act(g, act)
    off = _relative(e)
    e16, tiny = HALF_STEP[dtype], TINY[dtype]

    def close(got, want, size):
        far = off[:got.shape[0]] * size
        far = far + e16 * (want.abs() + far) + tiny
        d = (got.double() - want).abs()
        i = int((d / far).argmax())
        assert bool((d <= far).all()), (f"{float((d / far).max()):.3g} of what is allowed at gate "
                                        f"{float(g.expand_as(d).reshape(-1)[i]):.6g}: {float(got.reshape(-1)[i]):.6g}, "
                                        f"want {float(want.reshape(-1)[i]):.6g}")

    with torch.no_grad():
        close(gated.gated_linear(x, wg, wu, activation=act), a * u, (a * u).abs())
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    h = gated.gated_linear(*leaves, activation=act)
    close(h.detach(), a * u, (a * u).abs())
    if M == 1:
        dwg, dwu = torch.autograd.grad(h, leaves[1:], torch.ones_like(h))
        close(dwg[:, 0][None], u * sum(terms), u * sum(t.abs() for t in terms))
        close(dwu[:, 1][None], a, a.abs())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,F", [(65, 1032, 264), (100, 2056, 520), (128, 4104, 136), (128, 1544, 1000), (77, 776, 72)])
def test_few_tokens_with_a_cut_contraction(cuda, M, K, F, dtype):
    """65 to 128 tokens and a contraction that is cut among the CTAs of a cluster. A projection of K + 1 terms is off by
    at most 2 u each of the terms' sizes; the activation (slope 1.2 at most) and the product carry that on, and the
    result has half a step of its own."""
    g = torch.Generator().manual_seed(51)
    x = torch.randn(M, K, generator=g).to(dtype).to(cuda)
    wg, wu = ((torch.randn(F, K, generator=g) / math.sqrt(K)).to(dtype).to(cuda) for _ in range(2))
    bg, bu = ((torch.randn(F, generator=g) * 0.3).to(dtype).to(cuda) for _ in range(2))
    X, G, W, cg, cu = (t.double() for t in (x, wg, wu, bg, bu))
    gate, up = X @ G.T + cg, X @ W.T + cu
    n = 2 * U * (K + 2)
    far_g, far_u = n * (X.abs() @ G.abs().T + cg.abs()), n * (X.abs() @ W.abs().T + cu.abs())
    for act in ACTS:
        a, _, e = _act(gate, act)
        far_a = 1.2 * far_g + _relative(e) * a.abs()
        far = far_a * (up.abs() + far_u) + a.abs() * far_u
        far = far + HALF_STEP[dtype] * ((a * up).abs() + far) + TINY[dtype]
        with torch.no_grad():
            h = gated.gated_linear(x, wg, wu, bg, bu, activation=act)
            assert torch.equal(h, gated.gated_linear(x, wg, wu, bg, bu, activation=act))
        d = (h.double() - a * up).abs()
        assert bool((d <= far).all()), f"{act}: off by up to {float((d / far).max()):.3g} of what is allowed"
    # the same sums are kept for a backward
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, bg, bu)]
    assert torch.equal(gated.gated_linear(*leaves, activation=ACTS[-1]), h)


def test_forward_mode_is_refused(cuda):
    """No tangent is lost in silence: there is no forward-mode derivative, and a call with one says so."""
    x, w = torch.randn(3, 64, device=cuda).bfloat16(), torch.randn(72, 64, device=cuda).bfloat16()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward"):
            gated.gated_linear(dual, w, w)
        with pytest.raises(RuntimeError, match="forward"):
            gated.gated_linear(x, w, torch.autograd.forward_ad.make_dual(w, w))
        gated.gated_linear(x, w, w)  # a call without a tangent goes through


def _cut(cuda, M, K, F, seed):
    """Operands of a product whose few tiles are cut along K, which takes a workspace."""
    from comfy_ui_gfx906_tools_b200 import _lib
    assert _lib.load().gated_linear_workspace_bytes(M, K, F) > 1 << 18
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).bfloat16().to(cuda)
    return x, *((torch.randn(F, K, generator=g) / math.sqrt(K)).bfloat16().to(cuda) for _ in range(2))


def _captured(stream, args):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        h = gated.gated_linear(*args)
    return graph, h


def test_a_graph_outlives_a_grown_workspace(cuda):
    """A larger call on the stream of a capture replaces the workspace; the graph still joins its tiles in its own, and
    writes into nobody else's memory."""
    small, large = _cut(cuda, 200, 2048, 136, 61), _cut(cuda, 700, 6400, 72, 62)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    ops._workspaces.pop((0, side.cuda_stream), None)
    with torch.cuda.stream(side):
        want = gated.gated_linear(*small)
        held = ops._workspaces[(0, side.cuda_stream)].data_ptr()
    side.synchronize()
    graph, h = _captured(side, small)
    with torch.cuda.stream(side):
        gated.gated_linear(*large)
        assert ops._workspaces[(0, side.cuda_stream)].data_ptr() != held
        # whatever is allocated from now on is not the graph's
        mine = [torch.full((1 << 20,), 0x5A, dtype=torch.uint8, device=cuda) for _ in range(64)]
    side.synchronize()
    for _ in range(3):
        h.zero_()
        graph.replay()
        torch.cuda.synchronize(cuda)
        assert torch.equal(h, want)
    assert all(bool((t == 0x5A).all()) for t in mine)


def test_a_workspace_made_in_a_capture_is_the_graphs_own(cuda):
    """No call before the capture: eager calls on the same stream, before any replay, have a zeroed workspace too."""
    args = _cut(cuda, 200, 2048, 136, 63)
    want = gated.gated_linear(*args)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    ops._workspaces.pop((0, side.cuda_stream), None)
    graph, h = _captured(side, args)
    with torch.cuda.stream(side):
        eager = gated.gated_linear(*args)
    side.synchronize()
    assert torch.equal(eager, want)
    for _ in range(2):
        h.zero_()
        graph.replay()
        torch.cuda.synchronize(cuda)
        assert torch.equal(h, want)


def test_a_launch_of_several_seconds(cuda):
    """5.6e15 operations in one launch, longer than the limit of a wait for one stage, with a call right behind it: both
    are right and no wait gave up. Operands are +-1 and +-2^-9, whose sums are exact in float32, so a sampled result is
    off by its activation (1e-5 of it) and its own rounding alone."""
    M, K, F = 65536, 163840, 131072
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(cuda)[0] < 100 * 2 ** 30:
        pytest.skip("needs 100 GB of free memory")
    g = torch.Generator(device=cuda).manual_seed(71)
    x = torch.empty(M, K, device=cuda, dtype=torch.bfloat16).bernoulli_(0.5, generator=g).mul_(2).sub_(1)
    w = torch.empty(F, K, device=cuda, dtype=torch.bfloat16).bernoulli_(0.5, generator=g).sub_(0.5).mul_(2.0 ** -8)
    with torch.no_grad():
        h = gated.gated_linear(x, w, w)
        few = gated.gated_linear(x[:40], w[:520], w[:520])
    rows, cols = (torch.randperm(n, generator=g, device=cuda)[:128] for n in (M, F))
    gate = x[rows].double() @ w[cols].double().T
    want = gate * torch.sigmoid(gate) * gate
    got = h[rows][:, cols].double()
    assert bool(((got - want).abs() <= (2.0 ** -8 + 1e-5) * want.abs()).all())
    assert torch.equal(few, h[:40, :520])
    assert ops.device_status(cuda) == 0
    del x, w, h
    torch.cuda.empty_cache()
