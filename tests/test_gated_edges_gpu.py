"""Edges of the gated feed-forward product (gated.gated_linear): forward-mode derivatives."""
import pytest
import torch

from comfy_ui_gfx906_tools_b200 import gated

pytestmark = pytest.mark.gpu


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
