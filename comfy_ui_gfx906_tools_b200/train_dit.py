"""A small diffusion transformer trained with this package's training operators:
q/k norm and multi-axis rotary positions (``rotary``), the gated feed-forward
product (``gated``) and AdamW with moments in 32 or 8 bits (``optim``).

    python -m comfy_ui_gfx906_tools_b200.train_dit --steps 100 --state-bits 8

The model is a single-stream transformer in ``flux_dit``'s manner (adaLN
modulation from the timestep, axial positions) whose feed-forward is gated; its
matrix products besides the gated one are torch's, its attention is
``flux_dit.attention``. It learns the velocity of straight paths from noise to
synthetic patches, which are smooth waves over the grid, so that the loss falls
within a few dozen steps.
"""
from __future__ import annotations

import argparse
import dataclasses
import time

import torch
import torch.nn.functional as F

from . import flux_dit, gated, optim, rotary


@dataclasses.dataclass
class GatedDiTConfig:
    hidden: int = 256
    heads: int = 4
    kv_heads: int = 2
    features: int = 704
    depth: int = 2
    in_channels: int = 64
    axes_dims: tuple = (16, 24, 24)  # index, row, column
    theta: float = 10000.0

    @property
    def head_dim(self) -> int:
        return self.hidden // self.heads


class GatedBlock(torch.nn.Module):
    """Attention and a gated feed-forward, each behind an adaLN modulation."""

    def __init__(self, cfg: GatedDiTConfig, make, device=None, dtype=torch.bfloat16):
        super().__init__()
        self.cfg = cfg
        h, d = cfg.hidden, cfg.head_dim
        self.mod = flux_dit.Modulation(make, h, 6)
        self.qkv = make(h, (cfg.heads + 2 * cfg.kv_heads) * d, bias=False)
        self.q_scale = torch.nn.Parameter(torch.ones(d, device=device, dtype=dtype))
        self.k_scale = torch.nn.Parameter(torch.ones(d, device=device, dtype=dtype))
        self.proj = make(h, h, bias=False)
        self.mlp = gated.GatedMLP(h, cfg.features, "silu", device=device, dtype=dtype)
        self.mlp.gate, self.mlp.up, self.mlp.down = (  # from the model's own seed
            make(i, o, bias=False) for i, o in ((h, cfg.features), (h, cfg.features), (cfg.features, h)))

    def forward(self, x, vec, ids):
        cfg, (B, L, _) = self.cfg, x.shape
        n, kv, d = cfg.heads, cfg.kv_heads, cfg.head_dim
        m = self.mod(vec)
        y = self.qkv((1 + m[1]) * flux_dit.layer_norm(x) + m[0]).view(B, L, n + 2 * kv, d).transpose(1, 2)
        q, k, v = y.split((n, kv, kv), dim=1)
        q, k = rotary.qk_norm_rope(q, k, ids, cfg.axes_dims, cfg.theta, self.q_scale, self.k_scale)
        k, v = (t.repeat_interleave(n // kv, dim=1) for t in (k, v))
        o = flux_dit.attention(q, k, v).transpose(1, 2).reshape(B, L, n * d)
        x = x + m[2] * self.proj(o)
        return x + m[5] * self.mlp((1 + m[4]) * flux_dit.layer_norm(x) + m[3])


class GatedDiT(torch.nn.Module):
    def __init__(self, cfg: GatedDiTConfig, device=None, dtype=torch.bfloat16, seed: int = 0):
        super().__init__()
        make = flux_dit.float_linear_factory(device, dtype, seed)
        self.cfg = cfg
        self.img_in = make(cfg.in_channels, cfg.hidden)
        self.time_in = flux_dit.MLPEmbedder(make, 256, cfg.hidden)
        self.blocks = torch.nn.ModuleList([GatedBlock(cfg, make, device, dtype) for _ in range(cfg.depth)])
        self.final_mod = flux_dit.Modulation(make, cfg.hidden, 2)
        self.final_out = make(cfg.hidden, cfg.in_channels)

    def forward(self, img, ids, t):
        """img [B, L, in_channels], ids [L, 3] or [B, L, 3], t [B] -> [B, L, in_channels]."""
        x = self.img_in(img)
        vec = self.time_in(flux_dit.timestep_embedding(t).to(img.dtype))
        for block in self.blocks:
            x = block(x, vec, ids)
        shift, scale = self.final_mod(vec)
        return self.final_out((1 + scale) * flux_dit.layer_norm(x) + shift)


def grid_ids(rows: int, cols: int, device) -> torch.Tensor:
    """(0, row, column) of each patch: [rows * cols, 3]."""
    i = torch.arange(rows * cols, device=device)
    return torch.stack([torch.zeros_like(i), i // cols, i % cols], dim=-1)


def synthetic_batch(cfg: GatedDiTConfig, batch: int, ids: torch.Tensor, generator: torch.Generator):
    """(patches [B, L, in_channels], noise, t [B]): each channel a wave over the grid with its image's own phase."""
    dev = ids.device
    wave = torch.linspace(0.2, 1.0, cfg.in_channels, device=dev)
    phase = torch.rand(batch, 1, 1, generator=generator, device=dev) * 6.28
    x = torch.sin(ids[:, 1:2].float() * wave + ids[:, 2:3].float() * wave.flip(0) + phase)
    noise = torch.randn(x.shape, generator=generator, device=dev)
    return x, noise, torch.rand(batch, generator=generator, device=dev)


def train_step(model, opt, x, noise, t, ids, clip: float = 1.0):
    """One step; returns the loss (on the device). Gradients are clipped to a norm of ``clip`` by the scale that the
    optimizer multiplies them with, without a pass over them."""
    dtype = model.img_in.weight.dtype
    path = (t[:, None, None] * noise + (1 - t[:, None, None]) * x).to(dtype)
    loss = F.mse_loss(model(path, ids, t).float(), noise - x)
    loss.backward()
    grads = [p.grad for p in model.parameters()]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g, dtype=torch.float32) for g in grads]))
    opt.step(grad_scale=(clip / norm.clamp(min=clip)).view(1))
    opt.zero_grad()
    return loss.detach()


def train(cfg: GatedDiTConfig, steps: int, batch: int = 4, grid: int = 16, lr: float = 2e-3, state_bits: int = 32,
          device="cuda", seed: int = 0, log=None) -> list:
    """Trains a fresh model on synthetic batches; returns the loss of every step."""
    device = torch.device(device)
    model = GatedDiT(cfg, device, seed=seed)
    opt = optim.AdamW(model.parameters(), lr=lr, betas=(0.9, 0.95), weight_decay=0.01, state_bits=state_bits)
    gen = torch.Generator(device=device).manual_seed(seed)
    ids = grid_ids(grid, grid, device)
    losses, began = [], time.perf_counter()
    for i in range(steps):
        losses.append(train_step(model, opt, *synthetic_batch(cfg, batch, ids, gen), ids))
        if log and (i + 1) % log == 0:
            print(f"step {i + 1}: loss {losses[-1].item():.4f}  "
                  f"{(time.perf_counter() - began) / (i + 1) * 1e3:.1f} ms a step", flush=True)
    return torch.stack(losses).tolist() if losses else []


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--grid", type=int, default=16, help="patches along each side")
    ap.add_argument("--hidden", type=int, default=256)
    ap.add_argument("--depth", type=int, default=2)
    ap.add_argument("--lr", type=float, default=2e-3)
    ap.add_argument("--state-bits", type=int, choices=(32, 8), default=32)
    a = ap.parse_args()
    if a.hidden % 64:
        ap.error("--hidden must be a multiple of 64 (heads of 64)")
    heads = a.hidden // 64
    cfg = GatedDiTConfig(hidden=a.hidden, heads=heads, kv_heads=2 if heads % 2 == 0 else 1,
                         features=(a.hidden * 11 // 4 + 7) // 8 * 8, depth=a.depth)
    losses = train(cfg, a.steps, a.batch, a.grid, a.lr, a.state_bits, log=10)
    if losses:
        print(f"loss {losses[0]:.4f} -> {sum(losses[-10:]) / len(losses[-10:]):.4f}")


if __name__ == "__main__":
    main()
