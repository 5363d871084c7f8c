"""No-GPU check: a tensor with a forward-mode tangent is refused before anything else looks at it."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from paraattention_b200 import _lib as L
from paraattention_b200 import build_ext


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_tangents_are_refused(which, grad):
    build_ext.build()
    ext = L.load_torch_ext()
    xs = [torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16, requires_grad=grad) for _ in range(3)]
    w = torch.ones(64, dtype=torch.bfloat16, requires_grad=grad)
    with fwAD.dual_level():
        xs[which] = fwAD.make_dual(xs[which], torch.ones_like(xs[which]))
        with pytest.raises(NotImplementedError, match="forward"):
            ext.cross_attention(*xs, None, 0.125, False, 0, 0)
        norm = [xs[0], xs[1], fwAD.make_dual(w, torch.ones_like(w)) if which == 2 else w, w]
        with pytest.raises(NotImplementedError, match="forward"):
            ext.qk_norm_rotary(*norm, None, None, 0, True, 1e-6)
