"""Forward-mode derivatives (torch.autograd.forward_ad) of the linear-attention operators: there are none, and a dual tensor is
refused rather than taken for a constant.  The refusal comes before any launch, so all of it runs without a GPU.
"""
import pytest
import torch
from torch.autograd import forward_ad

import dms_amd
from dms_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def calls(device):
    x, g = torch.randn(3, 1, 2, 8, device=device), torch.zeros(3, 1, 2, device=device)
    s, w = torch.zeros(1, 2, 8, 8, device=device), torch.ones(8, device=device)
    token = torch.randn(1, 2, 8, device=device)
    return {"linear_attention": (ops.linear_attention, [x, x + 1, x - 1, g, s]),
            "linear_attention_step": (ops.linear_attention_step, [token, token + 1, token - 1, g[0], s]),
            "head_norm_rotary": (lambda q, k, wq, wk: ops.head_norm_rotary(q, k, wq, wk, None, ()), [x, x + 1, w, w + 1])}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["linear_attention", "linear_attention_step", "head_norm_rotary"])
def test_dual_tensors_are_refused(name, grad, device):
    call, args = calls(device)[name]
    for i in range(len(args)):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            dual = list(args)
            dual[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match="dms_amd.%s: no forward-mode derivatives" % name):
                call(*dual)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [True, False])
def test_layer_refuses_dual_tensors(grad, device):
    layer = dms_amd.LinearAttention(8, 16, 2, sections=(2,)).to(device)
    x, pos, state = torch.randn(3, 1, 8, device=device), torch.zeros(3, 1, 1, dtype=torch.int64, device=device), torch.zeros(1, 2, 8, 8, device=device)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = forward_ad.make_dual(x, x)
        for run in (lambda: layer(dual, None, pos), lambda: layer.step(dual[0], state, pos[0]),
                    lambda: torch.func.functional_call(layer, {"weight": forward_ad.make_dual(layer.weight.detach(), layer.weight.detach())},
                                                       (x, None, pos))):
            with pytest.raises(RuntimeError, match="no forward-mode derivatives"):
                run()


@pytest.mark.gpu
def test_tensors_without_a_tangent_pass_inside_a_level():
    for name, (call, args) in calls("cuda").items():
        with torch.no_grad():
            want = call(*[a.clone() for a in args])
            with forward_ad.dual_level():
                got = call(*[a.clone() for a in args])
        for a, b in zip((want,) if torch.is_tensor(want) else want, (got,) if torch.is_tensor(got) else got):
            assert torch.equal(a, b), name
