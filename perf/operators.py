"""The training operators of a DiT block, as they are measured: the gated feed-forward product with its backward
pass, q/k normalisation with multi-axis rotary positions with its backward pass, and the AdamW step over many
tensors with moments in 32 or 8 bits.

``run`` computes a case with elementary torch operations in 32 bits where ``own`` is false, and through this
package's operators where it is true. ``exact`` restates each operator in 64 bits from its definition.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_BLOCK = 256           # elements that share one scale of an 8-bit moment
_BETAS, _EPS, _WEIGHT_DECAY = (0.9, 0.95), 1e-8, 0.1
_ROPE_EPS = 1e-6


def listed():
    return [
        # one vector through a block's feed-forward at the diffusion transformer's own width: serving, latency-bound
        {"name": "gated token", "op": "gated", "tokens": 1, "hidden": 3072, "features": 12288, "dtype": "bf16",
         "act": "silu", "bias": False, "train": False},
        # a text prompt's 77 tokens through a small text block, half precision with biases, widths off any tile
        {"name": "gated prompt", "op": "gated", "tokens": 77, "hidden": 2056, "features": 5640, "dtype": "fp16",
         "act": "gelu_tanh", "bias": True, "train": False},
        # fine-tuning a small block on a ragged batch of tokens: forward and every gradient
        {"name": "gated train ragged", "op": "gated", "tokens": 1531, "hidden": 1160, "features": 3000,
         "dtype": "fp16", "act": "gelu", "bias": True, "train": True},
        # a training step's feed-forward at the diffusion transformer's width: 1024 x 1024 image, 512 text tokens
        {"name": "gated train image", "op": "gated", "tokens": 4608, "hidden": 3072, "features": 12288,
         "dtype": "bf16", "act": "silu", "bias": False, "train": True},
        # one new token's q and k: the smallest call
        {"name": "rope token", "op": "rope", "batch": 1, "tokens": 1, "heads": 24, "kv_heads": 24, "axes": "16,56,56",
         "dim": 128, "interleaved": True, "norm": True, "dtype": "bf16", "train": False},
        # sampling at 1024 x 1024 with 512 text tokens, q and k cut out of the packed qkv projection
        {"name": "rope image", "op": "rope", "batch": 1, "tokens": 4608, "heads": 24, "kv_heads": 24,
         "axes": "16,56,56", "dim": 128, "interleaved": True, "norm": True, "dtype": "bf16", "train": False},
        # training on video latents, grouped heads, half-split pairs, time / height / width: forward and gradients
        {"name": "rope train video", "op": "rope", "batch": 2, "tokens": 9991, "heads": 32, "kv_heads": 8,
         "axes": "16,24,24", "dim": 64, "interleaved": False, "norm": True, "dtype": "bf16", "train": True},
        # a float32 run on two axes that rotate part of the head, an odd count of tokens, no normalisation
        {"name": "rope train float", "op": "rope", "batch": 3, "tokens": 331, "heads": 12, "kv_heads": 4,
         "axes": "32,32", "dim": 96, "interleaved": True, "norm": False, "dtype": "fp32", "train": True},
        # low-rank adapters of two layers: twenty small tensors, latency-bound
        {"name": "adamw adapters", "op": "adamw", "kind": "adapter", "hidden": 3072, "features": 12288, "layers": 2,
         "rank": 4, "dtype": "fp32", "grad": "bf16", "bits": 32},
        # one full block of the diffusion transformer, bfloat16 weights, moments in 32 bits
        {"name": "adamw block", "op": "adamw", "kind": "block", "hidden": 3072, "features": 12288, "layers": 1,
         "rank": 0, "dtype": "bf16", "grad": "bf16", "bits": 32},
        # the same weights with moments in 8 bits
        {"name": "adamw block 8-bit", "op": "adamw", "kind": "block", "hidden": 3072, "features": 12288, "layers": 1,
         "rank": 0, "dtype": "bf16", "grad": "bf16", "bits": 8},
        # a small float32 model whose tensors have odd sizes, moments in 8 bits
        {"name": "adamw odd 8-bit", "op": "adamw", "kind": "block", "hidden": 515, "features": 1373, "layers": 3,
         "rank": 0, "dtype": "fp32", "grad": "fp32", "bits": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gated", "rope", "adamw"])
    if op == "gated":
        train = rng.random() < 0.5
        # widths are multiples of 8, as the operator asks; tokens are any number
        hidden, features = 8 * _log(rng, 32, 384), 8 * _log(rng, 32, 1536)
        return {"op": op, "tokens": _log(rng, 64 if train else 1, 4608), "hidden": hidden, "features": features,
                "dtype": rng.choice(["bf16", "fp16"]), "act": rng.choice(["silu", "gelu", "gelu_tanh"]),
                "bias": rng.random() < 0.5, "train": train}
    if op == "rope":
        train = rng.random() < 0.5
        dim = rng.choice([64, 80, 96, 128])
        axes = {64: "16,24,24", 80: "16,32,32", 96: "32,32", 128: "16,56,56"}[dim]
        kv = rng.choice([1, 2, 4, 8])
        return {"op": op, "batch": rng.choice([1, 1, 2, 3]), "tokens": _log(rng, 1, 5000),
                "heads": kv * rng.choice([1, 3, 4]), "kv_heads": kv, "axes": axes, "dim": dim,
                "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.7,
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "train": train}
    kind = rng.choice(["adapter", "block"])
    hidden = _log(rng, 64, 1536)
    return {"op": op, "kind": kind, "hidden": hidden, "features": hidden * 3 + rng.randrange(0, 99),
            "layers": rng.choice([1, 2, 3]), "rank": rng.choice([4, 8, 13]) if kind == "adapter" else 0,
            "dtype": rng.choice(["bf16", "fp32"]), "grad": rng.choice(["bf16", "fp32"]), "bits": rng.choice([8, 32])}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"gated": _prepare_gated, "rope": _prepare_rope, "adamw": _prepare_adamw}[case["op"]](case, g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_gated(case, g):
    m, k, f, dt = case["tokens"], case["hidden"], case["features"], _DTYPES[case["dtype"]]
    s = {"case": case, "x": _randn(g, m, k).to(dt), "w_gate": (_randn(g, f, k) / math.sqrt(k)).to(dt),
         "w_up": (_randn(g, f, k) / math.sqrt(k)).to(dt), "b_gate": None, "b_up": None}
    if case["bias"]:
        s["b_gate"], s["b_up"] = (_randn(g, f) * 0.1).to(dt), (_randn(g, f) * 0.1).to(dt)
    if case["train"]:
        s["dh"] = (_randn(g, m, f) * 0.5).to(dt)
        for n in ("x", "w_gate", "w_up", "b_gate", "b_up"):
            if s[n] is not None:
                s[n].requires_grad_(True)
    return s


def _prepare_rope(case, g):
    b, n, h, kv, d = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    dt = _DTYPES[case["dtype"]]
    axes = [int(a) for a in case["axes"].split(",")]
    qkv = _randn(g, b, n, (h + 2 * kv) * d).to(dt)  # a block's packed projection; q and k are read in place
    q = qkv[..., :h * d].view(b, n, h, d).transpose(1, 2)
    k = qkv[..., h * d:(h + kv) * d].view(b, n, kv, d).transpose(1, 2)
    # the ids of a grid of patches: (row, column), with the frame before them where there are three axes
    w = max(1, int(math.sqrt(n / 2)))
    i = torch.arange(n, device="cuda") + torch.randint(0, 64, (b, 1), generator=g, device="cuda")
    per = [i % w, i // w] if len(axes) == 2 else [i // (w * w), (i // w) % w, i % w]
    s = {"case": case, "axes": axes, "q": q, "k": k, "positions": torch.stack(per, dim=-1), "q_scale": None,
         "k_scale": None}
    if case["norm"]:
        s["q_scale"], s["k_scale"] = (1 + 0.1 * _randn(g, d)).to(dt), (1 + 0.1 * _randn(g, d)).to(dt)
    if case["train"]:
        s["dq"], s["dk"] = _randn(g, b, h, n, d).to(dt), _randn(g, b, kv, n, d).to(dt)
        for name in ("q", "k", "q_scale", "k_scale"):
            if s[name] is not None:
                s[name] = s[name].detach().requires_grad_(True)
    return s


def _shapes(case):
    h, f, r = case["hidden"], case["features"], case["rank"]
    weights = [(3 * h, h), (h, h), (f, h), (f, h), (h, f)]  # qkv, out, gate, up, down
    if case["kind"] == "adapter":
        return [s for o, i in weights for s in ((r, i), (o, r))] * case["layers"]
    return (weights + [(h,), (f,), (128,), (128,)]) * case["layers"]


def _spans(case):
    """(offset, shape) of each tensor in one flat buffer, each at a whole number of blocks, and the buffer's length."""
    at, spans = 0, []
    for s in _shapes(case):
        spans.append((at, s))
        at += -(-math.prod(s) // _BLOCK) * _BLOCK
    return spans, at


def _views(flat, spans):
    return [flat[o:o + math.prod(s)].view(s) for o, s in spans]


def _prepare_adamw(case, g):
    spans, n = _spans(case)
    inside = torch.zeros(n, device="cuda")  # 1 where an element belongs to a tensor, 0 in the gaps behind them
    for v in _views(inside, spans):
        v.fill_(1)
    p = (_randn(g, n) * 0.02 * inside).to(_DTYPES[case["dtype"]])
    grad = (_randn(g, n) * 1e-3 * inside).to(_DTYPES[case["grad"]])
    m = _randn(g, n) * 3e-4 * inside
    v = (_randn(g, n) * 1e-3 * inside).square() + 1e-8 * inside
    s = {"case": case, "step": 100, "lr": 1e-3, "p_flat": p, "g_flat": grad, "p": _views(p, spans),
         "g": _views(grad, spans)}
    if case["bits"] == 32:
        s.update(m_flat=m, v_flat=v, m=_views(m, spans), v=_views(v, spans))
        return s
    mc, ms = _encode(m, 127)
    vc, vs = _encode(v.sqrt(), 255)
    s.update(m_flat=mc.to(torch.int8), v_flat=vc.to(torch.uint8), ms_flat=ms, vs_flat=vs)
    s["m"], s["v"] = ([t[o:o + math.prod(z)] for o, z in spans] for t in (s["m_flat"], s["v_flat"]))
    blocks = [(o // _BLOCK, -(-math.prod(z) // _BLOCK)) for o, z in spans]
    s["ms"], s["vs"] = ([t[o:o + c] for o, c in blocks] for t in (ms, vs))
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    return {"gated": _run_gated, "rope": _run_rope, "adamw": _run_adamw}[state["case"]["op"]](state)


def _run_gated(s):
    c, w = s["case"], ("x", "w_gate", "w_up", "b_gate", "b_up")
    if own:
        from comfy_ui_gfx906_tools_b200 import gated
        h = gated.gated_linear(*(s[n] for n in w), activation=c["act"])
    else:
        h = _plain_gated(*(None if s[n] is None else s[n].float() for n in w), c["act"]).to(s["x"].dtype)
    if not c["train"]:
        return h
    return [h.detach(), *torch.autograd.grad(h, [s[n] for n in w if s[n] is not None], s["dh"])]


def _plain_gated(x, wg, wu, bg, bu, act):
    gate, up = x @ wg.t(), x @ wu.t()
    if bg is not None:
        gate, up = gate + bg, up + bu
    if act == "silu":
        a = gate / (1 + torch.exp(-gate))
    elif act == "gelu":
        a = 0.5 * gate * (1 + torch.erf(gate * math.sqrt(0.5)))
    else:
        a = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
    return a * up


def _run_rope(s):
    c = s["case"]
    if own:
        from comfy_ui_gfx906_tools_b200 import rotary
        q, k = rotary.qk_norm_rope(s["q"], s["k"], s["positions"], s["axes"], theta=10000.0, q_scale=s["q_scale"],
                                   k_scale=s["k_scale"], eps=_ROPE_EPS, interleaved=c["interleaved"])
    else:
        cos, sin = _plain_tables(s["positions"], s["axes"])
        q = _plain_rope(s["q"], s["q_scale"], cos, sin, c["interleaved"])
        k = _plain_rope(s["k"], s["k_scale"], cos, sin, c["interleaved"])
    if not c["train"]:
        return q, k
    leaves = [s[n] for n in ("q", "k", "q_scale", "k_scale") if s[n] is not None]
    return [q.detach(), k.detach(), *torch.autograd.grad([q, k], leaves, [s["dq"], s["dk"]])]


def _plain_tables(positions, axes):
    """cos and sin [B, 1, L, pairs]; the angle is formed in 64 bits, as the package's own rope tables form it, because
    an angle of some thousand radians in 32 bits is off by more than a 32-bit result may be."""
    parts = []
    for a, d in enumerate(axes):
        freq = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        parts.append(positions[..., a].double()[..., None] * freq)
    angle = torch.remainder(torch.cat(parts, dim=-1), 2 * math.pi).float()[:, None]
    return torch.cos(angle), torch.sin(angle)


def _plain_rope(x, scale, cos, sin, interleaved):
    y, r = x.float(), 2 * cos.shape[-1]
    if scale is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + _ROPE_EPS) * scale.float()
    if interleaved:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, y[..., r:]], dim=-1).to(x.dtype)


def _run_adamw(s):
    c = s["case"]
    if own:
        from comfy_ui_gfx906_tools_b200 import optim
        more = dict(step=s["step"], lr=s["lr"], betas=_BETAS, eps=_EPS, weight_decay=_WEIGHT_DECAY)
        if c["bits"] == 32:
            optim.adamw_step(s["p"], s["g"], s["m"], s["v"], **more)
            return s["p_flat"], s["m_flat"], s["v_flat"]
        optim.adamw_step_8bit(s["p"], s["g"], s["m"], s["ms"], s["v"], s["vs"], **more)
        return (s["p_flat"], optim.moment_values(s["m_flat"], s["ms_flat"]),
                optim.moment_values(s["v_flat"], s["vs_flat"]))
    m, v = s["m_flat"], s["v_flat"]
    if c["bits"] == 8:
        m, v = _decode(m, s["ms_flat"]), _decode(v, s["vs_flat"])
        v = v * v
    grad = s["g_flat"].float()
    m = m * _BETAS[0] + grad * (1 - _BETAS[0])
    v = v * _BETAS[1] + grad * grad * (1 - _BETAS[1])
    root = torch.sqrt(v)
    denom = root * (1 / math.sqrt(1 - _BETAS[1] ** s["step"])) + _EPS
    p = s["p_flat"].float() * (1 - s["lr"] * _WEIGHT_DECAY) - m / denom * (s["lr"] / (1 - _BETAS[0] ** s["step"]))
    s["p_flat"].copy_(p)
    if c["bits"] == 32:
        s["m_flat"].copy_(m)
        s["v_flat"].copy_(v)
        return s["p_flat"], s["m_flat"], s["v_flat"]
    for name, x, top in (("m", m, 127), ("v", root, 255)):
        codes, scale = _encode(x, top)
        s[name + "_flat"].copy_(codes)
        s[name + "s_flat"].copy_(scale)
    root = _decode(s["v_flat"], s["vs_flat"])
    return s["p_flat"], _decode(s["m_flat"], s["ms_flat"]), root * root


def _encode(x, top):
    """Codes in [-top, top] (a first moment) or [0, top] (the root of a second one) and one scale a block: the code is
    the root of |x| / scale to the nearest whole number, the scale the block's largest |x| over top squared. A positive
    root of a second moment keeps at least the code 1, so that no update divides by a lost one."""
    x = x.view(-1, _BLOCK)
    scale = x.abs().amax(dim=1, keepdim=True) * torch.tensor(1.0 / (top * top), device="cuda")
    fine = scale >= 2.0 ** -126
    inv = torch.where(fine, torch.ones_like(scale) / torch.where(fine, scale, torch.ones_like(scale)), 0)
    scale = torch.where(fine, scale, 0)
    code = torch.sqrt(x.abs() * inv).round().clamp(max=top)
    if top == 255:
        code = torch.where((x > 0) & fine, code.clamp(min=1), code)
    return (code * torch.sign(x)).flatten(), scale.flatten()


def _decode(codes, scale):
    c = codes.view(-1, _BLOCK).float()
    return (c * c.abs() * scale[:, None]).flatten()


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "gated":
        m, k, f, e = case["tokens"], case["hidden"], case["features"], _BYTES[case["dtype"]]
        b = 2 * f if case["bias"] else 0
        once = m * k + 2 * f * k + b
        if not case["train"]:
            return {"bytes": e * (once + m * f), "flops": 4 * m * k * f}
        # forward, both weights' gradients, x's: six products of 2 m k f; every input read and output written once
        return {"bytes": e * (2 * once + 2 * m * f), "flops": 12 * m * k * f}
    if case["op"] == "rope":
        d, e = case["dim"], _BYTES[case["dtype"]]
        rows = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"])
        axes, norm = len(case["axes"].split(",")), 2 * d * e if case["norm"] else 0
        ids = case["batch"] * case["tokens"] * axes * 8
        # forward: q and k in and out; backward: the outputs' gradients in, the inputs' out
        times = 4 if case["train"] else 2
        return {"bytes": times * rows * d * e + ids + (2 if case["train"] else 1) * norm, "flops": times * 5 * rows * d}
    n = sum(math.prod(s) for s in _shapes(case))
    per = 2 * _BYTES[case["dtype"]] + _BYTES[case["grad"]]
    if case["bits"] == 32:
        return {"bytes": n * (per + 16), "flops": 16 * n}
    # 8-bit moments: codes and scales read and written, and the values that they stand for written as outputs
    return {"bytes": n * (per + 4 + 16 / _BLOCK + 8), "flops": 32 * n}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"gated": _exact_gated, "rope": _exact_rope, "adamw": _exact_adamw}[case["op"]](s)


def _exact_gated(s):
    """h = a(g) u with g = x Wg' + bg, u = x Wu' + bu; dg = dh u a'(g), du = dh a(g); dx = dg Wg + du Wu,
    dWg = dg' x, dWu = du' x, db = the columns' sums."""
    c = s["case"]
    x, wg, wu = (s[n].double() for n in ("x", "w_gate", "w_up"))
    g, u = torch.mm(x, wg.T), torch.mm(x, wu.T)
    if c["bias"]:
        g += s["b_gate"].double()
        u += s["b_up"].double()
    if c["act"] == "silu":
        z = torch.sigmoid(g)
        a, da = g * z, z * (1 + g * (1 - z))
    elif c["act"] == "gelu":
        z = 0.5 * torch.erfc(-g / math.sqrt(2))
        a, da = g * z, z + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    else:
        q = math.sqrt(2 / math.pi)
        t = torch.tanh(q * g * (1 + 0.044715 * g * g))
        a, da = g * (1 + t) / 2, (1 + t) / 2 + g / 2 * (1 - t * t) * q * (1 + 3 * 0.044715 * g * g)
    h = a * u
    if not c["train"]:
        return h
    dh = s["dh"].double()
    dg, du = dh * u * da, dh * a
    out = [h, torch.mm(dg, wg) + torch.mm(du, wu), torch.mm(dg.T, x), torch.mm(du.T, x)]
    return out + [dg.sum(0), du.sum(0)] if c["bias"] else out


def _exact_rope(s):
    """Pairs as complex numbers: the forward turns them by the angle, the backward turns back."""
    c = s["case"]
    angle = torch.cat([s["positions"][..., a].double().unsqueeze(-1)
                       * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"),
                                   -2.0 * torch.arange(d // 2, device="cuda").double() / d)
                       for a, d in enumerate(s["axes"])], -1).unsqueeze(1)
    turn = torch.polar(torch.ones_like(angle), angle)
    r = 2 * angle.shape[-1]

    def rotated(x, by):
        y = x.clone()
        if c["interleaved"]:
            z = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * by
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        else:
            z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * by
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        return y

    out, grads, scales = [], [], []
    for n in ("q", "k"):
        x, w = s[n].double(), s[n + "_scale"]
        if w is not None:
            inv = (x.pow(2).mean(-1, keepdim=True) + _ROPE_EPS).pow(-0.5)
            unit = x * inv
        out.append(rotated(x if w is None else unit * w.double(), turn))
        if c["train"]:
            d = rotated(s["d" + n].double(), turn.conj())
            if w is not None:
                scales.append((d * unit).sum((0, 1, 2)))
                d = d * w.double()
                d = inv * (d - unit * (d * unit).mean(-1, keepdim=True))
            grads.append(d)
    return out + grads + scales if c["train"] else tuple(out)


def _exact_adamw(s):
    b1, b2, lr, t = *_BETAS, s["lr"], s["step"]
    p, g = s["p_flat"].double(), s["g_flat"].double()
    if s["case"]["bits"] == 32:
        m, v = s["m_flat"].double(), s["v_flat"].double()
    else:
        def value(c, q):
            c = c.double().reshape(-1, _BLOCK)
            return (c.sign() * c.pow(2) * q.double().reshape(-1, 1)).reshape(-1)
        m, v = value(s["m_flat"], s["ms_flat"]), value(s["v_flat"], s["vs_flat"]).pow(2)
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g.pow(2)
    p = p - lr * (_WEIGHT_DECAY * p + (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + _EPS))
    if s["case"]["bits"] == 32:
        return p, m, v

    def held(x, top):
        x = x.reshape(-1, _BLOCK)
        q = x.abs().amax(1, keepdim=True) / top ** 2
        c = (x.abs() / q.clamp(min=1e-300)).sqrt().round()
        if top == 255:
            c = torch.where(x > 0, c.clamp(min=1), c)
        return (x.sign() * c.pow(2) * q).reshape(-1)

    return p, held(m, 127), held(v.sqrt(), 255).pow(2)
