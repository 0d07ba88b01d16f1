"""Gradients of norm + rotation (ops.head_norm_rotary) over more tokens than one turn of the backward's grid takes (1024
workgroups of 256 lanes): groups of lanes walk several tokens each, the last turn is not full, and the weights' gradients are summed
over all of it.

Bounds as derived for single turns: 2^-18 of the magnitudes for the rows' gradients; a weight's gradient is a chain of a
group's rows (at most 3 here) and of at most 256 groups of a workgroup before the sum goes on in 64 bits: 2^-18 + 260 * 2^-24 <
2^-15.
"""
import pytest
import torch

from dms_amd import ops
from test_head_norm_rotary import DEV, angles, bounded, make, plain


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,T,B,Hq,Hk,D,sections,weights", [
    ("fp32", 9001, 1, 1, 1, 256, (64, 64), "fp32"),            # 4 tokens a workgroup
    ("bf16", 3307, 5, 1, 2, 256, (100,), "same"),              # 8
    ("fp32", 300007, 1, 1, 1, 7, (1, 2), "fp32"),              # 128
    ("fp16", 2 * 4097, 3, 2, 1, 100, (10, 20, 20), "fp32"),    # 8
    ("bf16", 4099, 9, 1, 1, 64, (8, 12, 12), "fp32"),          # 32: one turn and the beginning of a second
])
def test_more_tokens_than_one_turn(dtype, T, B, Hq, Hk, D, sections, weights):
    q, k, wq, wk, pos, dq, dk = make(dtype, T, B, Hq, Hk, D, len(sections), weights, seed=T)
    dev = [x.to(DEV).requires_grad_() for x in (q, k, wq, wk)]
    y = ops.head_norm_rotary(*dev, pos.to(DEV), sections, base=500.0, eps=1e-5)
    grads = torch.autograd.grad(y, dev, [dq.to(DEV), dk.to(DEV)])
    angle = angles(pos, sections, (D + 1) // 2, 500.0)
    for m, (x, w, d) in enumerate(((q, wq, dq), (k, wk, dk))):
        want = plain(x.double(), w.double(), angle, 1e-5, d.double())
        bounded(y[m], want[0], want[1], 2.0 ** -20)
        bounded(grads[m], want[2], want[3], 2.0 ** -18)
        bounded(grads[2 + m], want[4], want[5], 2.0 ** -15)
        # the bound by magnitudes is wide for a long sum; by the norm, rows of either sign leave sqrt(rows) roundings of terms
        # and the result grows with the same root
        off = grads[2 + m].cpu().double() - want[4]
        assert float(off.norm()) <= (torch.finfo(grads[2 + m].dtype).eps / 2 + 2.0 ** -18) * float(want[4].norm())
