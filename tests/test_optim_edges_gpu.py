"""Edges of the AdamW operators (optim): a step inside a CUDA graph capture."""
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
