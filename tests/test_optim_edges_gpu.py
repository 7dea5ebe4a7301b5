"""Edges of the AdamW operators (optim): a step inside a CUDA graph capture, refused steps, gradients of another shape,
groups with their own settings."""
import pytest
import torch

from comfy_ui_gfx906_tools_b200 import optim

pytestmark = pytest.mark.gpu


def _param(cuda, *shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    p = torch.nn.Parameter(torch.randn(*shape, generator=g).to(dtype).to(cuda))
    p.grad = torch.randn(*shape, generator=g).to(dtype).to(cuda)
    return p


@pytest.mark.parametrize("bits", [32, 8])
def test_step_refuses_a_graph_capture(cuda, bits):
    """The step's number and its bias corrections are arguments of the launch: a replay would repeat the captured ones.
    The refusal leaves parameters and state as they were."""
    p = _param(cuda, 300)
    opt = optim.AdamW([p], lr=1e-2, state_bits=bits)
    opt.step()
    before, other = p.detach().clone(), torch.zeros(4, device=cuda)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        other.add_(1)
        with pytest.raises(RuntimeError, match="CUDA graph"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize(cuda)
    assert torch.equal(p.detach(), before) and opt.state[p]["step"] == 1 and bool((other == 1).all())
    opt.step()
    assert opt.state[p]["step"] == 2 and not torch.equal(p.detach(), before)


@pytest.mark.parametrize("bits", [32, 8])
def test_refused_step_is_not_counted(cuda, bits):
    """A call that is refused moves no step counter: the next one is the first step, bit for bit."""
    a, b = _param(cuda, 37, 5), _param(cuda, 37, 5)
    mine, fresh = (optim.AdamW([p], lr=1e-2, state_bits=bits) for p in (a, b))
    for _ in range(3):
        with pytest.raises(RuntimeError, match="grad_scale"):
            mine.step(grad_scale=torch.ones(2, device=cuda))
    mine.step()
    fresh.step()
    assert torch.equal(a, b) and mine.state[a]["step"] == fresh.state[b]["step"] == 1


def test_only_what_moved_is_counted(cuda):
    """Two launches of one step, the second one refused: the first one's parameters moved and are counted."""
    good, bad = _param(cuda, 50), _param(cuda, 6, 8, dtype=torch.bfloat16)
    bad.data = bad.data.t()
    bad.grad = torch.ones(8, 6, device=cuda, dtype=torch.bfloat16)
    before = good.detach().clone()
    opt = optim.AdamW([good, bad], lr=1e-2)
    with pytest.raises(RuntimeError, match="contiguous"):
        opt.step()
    assert opt.state[good]["step"] == 1 and not torch.equal(good.detach(), before)
    assert opt.state[bad]["step"] == 0


def test_gradient_of_another_shape_is_refused(cuda):
    """As many elements in another order are another tensor's gradient."""
    p, g = torch.ones(3, 2, device=cuda), torch.ones(2, 3, device=cuda)
    m, v = torch.zeros(3, 2, device=cuda), torch.zeros(3, 2, device=cuda)
    with pytest.raises(RuntimeError, match=r"grads\[0\].*\(3, 2\).*\(2, 3\)"):
        optim.adamw_step([p], [g], [m], [v], step=1, lr=1e-2)
    with pytest.raises(RuntimeError, match=r"grads\[1\]"):
        optim.adamw_step([p, p.clone()], [g.t().contiguous(), g.view(6)], [m, m.clone()], [v, v.clone()], step=1,
                         lr=1e-2)
    assert bool((p == 1).all()) and bool((m == 0).all())
    z = lambda dt: torch.zeros(6, dtype=dt, device=cuda)  # noqa: E731
    with pytest.raises(RuntimeError, match=r"grads\[0\]"):
        optim.adamw_step_8bit([p], [g], [z(torch.int8)], [z(torch.float32)[:1]], [z(torch.uint8)],
                              [z(torch.float32)[:1]], step=1, lr=1e-2)


def test_group_settings_are_checked(cuda):
    """A group's own settings meet the checks of the constructor's."""
    for more in (dict(state_bits=16), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(betas=(0.9, 1.0)),
                 dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            optim.AdamW([{"params": [_param(cuda, 4)], **more}])
        opt = optim.AdamW([_param(cuda, 4)])
        with pytest.raises(ValueError):
            opt.add_param_group({"params": [_param(cuda, 4)], **more})
        assert len(opt.param_groups) == 1
    a, b = _param(cuda, 300, seed=1), _param(cuda, 300, seed=1)
    opt = optim.AdamW([{"params": [a], "state_bits": 8}, {"params": [b]}], lr=1e-2)
    opt.step()
    assert "m_codes" in opt.state[a] and "exp_avg" in opt.state[b]
