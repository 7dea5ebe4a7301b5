"""The training operators together (train_dit): a block's output and gradients against the same block written from
plain torch operations in 64 bits, and training runs whose loss falls, with moments in 32 and in 8 bits."""
import math

import pytest
import torch

from comfy_ui_gfx906_tools_b200 import flux_dit, train_dit

pytestmark = pytest.mark.gpu


def _plain_block(block, p, x, vec, ids):
    """GatedBlock.forward from the formulas, with the parameters p in 64 bits."""
    cfg, (B, L, h) = block.cfg, x.shape
    n, kv, d = cfg.heads, cfg.kv_heads, cfg.head_dim

    def norm(y):
        return (y - y.mean(-1, keepdim=True)) / torch.sqrt(y.var(-1, unbiased=False, keepdim=True) + 1e-6)

    m = (vec * torch.sigmoid(vec)) @ p["mod.lin.weight"].T + p["mod.lin.bias"]
    m = m[:, None].chunk(6, dim=-1)
    y = (((1 + m[1]) * norm(x) + m[0]) @ p["qkv.weight"].T).view(B, L, n + 2 * kv, d).transpose(1, 2)
    q, k, v = y.split((n, kv, kv), dim=1)
    ang = torch.cat([ids[..., a].double()[:, None] * cfg.theta ** (-torch.arange(0, w, 2, device=x.device).double() / w)
                     for a, w in enumerate(cfg.axes_dims)], -1)

    def turned(t, w):
        t = t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * w
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).flatten(-2)

    q, k = turned(q, p["q_scale"]), turned(k, p["k_scale"])
    k, v = (t.repeat_interleave(n // kv, dim=1) for t in (k, v))
    o = torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(d), dim=-1) @ v
    x = x + m[2] * (o.transpose(1, 2).reshape(B, L, n * d) @ p["proj.weight"].T)
    y = (1 + m[4]) * norm(x) + m[3]
    g, u = y @ p["mlp.gate.weight"].T, y @ p["mlp.up.weight"].T
    return x + m[5] * ((g * torch.sigmoid(g) * u) @ p["mlp.down.weight"].T)


def test_block_against_the_formulas(cuda):
    """Every step of the block rounds to bfloat16 (half a step: 2^-8 of the value, a third of it in the mean): some
    fifteen of them in a row forward and as many back leave the 2-norm's error below 15 * 2^-8 / 3 = 2e-2 of the
    result's forward; gradients go through both, 4e-2."""
    cfg = train_dit.GatedDiTConfig()
    make = flux_dit.float_linear_factory(cuda, torch.bfloat16, 3)
    block = train_dit.GatedBlock(cfg, make, cuda)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 48, cfg.hidden, generator=g).bfloat16().to(cuda).requires_grad_(True)
    vec = torch.randn(2, cfg.hidden, generator=g).bfloat16().to(cuda)
    dy = torch.randn(2, 48, cfg.hidden, generator=g).bfloat16().to(cuda)
    ids = train_dit.grid_ids(6, 8, cuda)
    y = block(x, vec, ids)
    y.backward(dy)
    p = {n: t.detach().double().requires_grad_(True) for n, t in block.named_parameters()}
    x64 = x.detach().double().requires_grad_(True)
    want = _plain_block(block, p, x64, vec.double(), ids)
    want.backward(dy.double())

    def off(a, b):
        return float((a.double() - b).norm() / b.norm())

    assert off(y.detach(), want.detach()) <= 2e-2
    assert off(x.grad, x64.grad) <= 4e-2
    for n, t in block.named_parameters():
        assert off(t.grad, p[n].grad) <= 4e-2, n


@pytest.mark.parametrize("bits", [32, 8])
def test_training_lowers_the_loss(cuda, bits):
    losses = train_dit.train(train_dit.GatedDiTConfig(), 60, state_bits=bits)
    assert all(math.isfinite(v) for v in losses)
    assert sum(losses[-10:]) / 10 < 0.6 * sum(losses[:3]) / 3


def test_runs_repeat(cuda):
    a = train_dit.train(train_dit.GatedDiTConfig(depth=1), 5, state_bits=8)
    b = train_dit.train(train_dit.GatedDiTConfig(depth=1), 5, state_bits=8)
    assert len(a) == 5 and a[0] == b[0]  # the first forward is the same bit for bit
    assert all(abs(x - y) <= 1e-2 * abs(x) for x, y in zip(a, b))


def test_operators_in_a_cuda_graph(cuda):
    """Forward calls and an AdamW step captured once and replayed on new contents of the same tensors."""
    from comfy_ui_gfx906_tools_b200 import gated, optim, rotary
    g = torch.Generator().manual_seed(5)
    make = lambda *s: torch.randn(*s, generator=g).bfloat16().to(cuda)  # noqa: E731
    few, many, w = make(40, 264), make(700, 264), make(2 * 1032, 264) / 16
    q, ids = make(1, 4, 33, 64), train_dit.grid_ids(3, 11, cuda)
    p, grad = torch.ones(5000, device=cuda), torch.randn(5000, generator=g).to(cuda)
    m, v = torch.zeros(5000, device=cuda), torch.zeros(5000, device=cuda)

    def once():
        outs = [gated.gated_linear(x, w[:1032], w[1032:]) for x in (few, many)]
        outs.append(rotary.qk_norm_rope(q, None, ids, (16, 24, 24), q_scale=q[0, 0, 0])[0])
        optim.adamw_step([p], [grad], [m], [v], step=3, lr=1e-2)
        return outs

    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        once()  # workspaces are made outside the capture
    torch.cuda.current_stream(cuda).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = once()
    for t in (few, many, q):
        t.copy_(make(*t.shape))
    for t in (p, m, v):
        t.fill_(0.5)
    graph.replay()
    got = [t.clone() for t in outs + [p, m, v]]
    for t in (p, m, v):
        t.fill_(0.5)
    want = once() + [p, m, v]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
