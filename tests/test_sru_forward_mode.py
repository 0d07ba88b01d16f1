"""Forward-mode derivatives of the SRU scan (ops.sru_compute): there are none, and a dual tensor is refused rather than taken
for a constant.  The refusal comes before any look at the device.
"""
import pytest
import torch
from torch.autograd import forward_ad

import dms_amd
from dms_amd import ops


@pytest.mark.parametrize("at", range(4))
@pytest.mark.parametrize("grad", [True, False])
def test_dual_tensors_are_refused(at, grad):
    args = [torch.randn(5, 2, 4, 3), torch.randn(5, 2, 4), torch.zeros(8), torch.zeros(2, 4)]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        args[at] = forward_ad.make_dual(args[at], torch.ones_like(args[at]))
        with pytest.raises(RuntimeError, match="dms_amd.sru_compute: no forward-mode derivatives"):
            ops.sru_compute(*args)


@pytest.mark.parametrize("grad", [True, False])
def test_layer_refuses_dual_tensors(grad):
    layer = dms_amd.SRU(4, 4, 2)
    x = torch.randn(5, 2, 4)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="no forward-mode derivatives"):
            layer(forward_ad.make_dual(x, x))
