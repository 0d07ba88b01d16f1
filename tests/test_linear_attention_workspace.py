"""Workspace of linear attention's backward pass: what is asked for is what is used, and nothing for gradients that nobody wants."""
import pytest
import torch

from dms_amd import _lib, ops

DEV = "cuda"


def floats(kind, dtype, *sizes):
    return _lib.query("dmn_linear_attention_workspace_floats", dtype, kind, *sizes)


def test_frozen_decays_ask_for_no_meeting_states():
    sizes = (2000, 64, 16, 16, 16, 16, 64, 64)                 # T, B, H, Hq, Hk, Hv, dk, dv
    states, dots = 2 * 64 * 16 * 7 * 64 * 64, 2 * 2000 * 64 * 16
    assert floats(1, 1, *sizes) >= states + dots
    assert floats(2, 1, *sizes) == 0                           # enough heads for one segment: nothing else to keep
    shared = (2000, 64, 16, 8, 16, 16, 64, 64)
    assert floats(2, 1, *shared) == 2000 * 64 * 16 * 64        # the queries' gradient before its heads are summed
    few = (2000, 1, 2, 2, 2, 2, 64, 64)
    assert 0 < floats(2, 0, *few) < floats(1, 0, *few)
    assert floats(2, 3, *few) == -1 and floats(2, 0, 2000, 1, 2, 3, 2, 2, 64, 64) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("T,B,H,Hq,Hk,Hv,dk,dv", [(300, 1, 2, 2, 2, 2, 64, 64), (300, 2, 4, 2, 1, 4, 33, 100), (700, 9, 30, 30, 15, 30, 16, 16),
                                                  (5, 2, 2, 1, 2, 1, 20, 128)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("decays", [False, True])
def test_nothing_is_written_behind_the_workspace(dtype, decays, T, B, H, Hq, Hk, Hv, dk, dv):
    sizes = (T, B, H, Hq, Hk, Hv, dk, dv)
    gen = torch.Generator().manual_seed(T)
    t = [torch.float32, torch.bfloat16, torch.float16][dtype]
    q, k, v, do = (torch.randn(T, B, h, d, generator=gen).to(t).to(DEV) for h, d in ((Hq, dk), (Hk, dk), (Hv, dv), (H, dv)))
    g = torch.nn.functional.logsigmoid(torch.randn(T, B, H, generator=gen)).to(DEV)
    s0, ds = (torch.randn(B, H, dk, dv, generator=gen).to(DEV) for _ in range(2))
    grads = [torch.empty_like(x) for x in (q, k, v, g, s0)]
    n, guard = max(floats(1 if decays else 2, dtype, *sizes), 4), 4096
    ws = torch.full((n + guard,), 7.0, device=DEV)
    p = [x.data_ptr() for x in grads]
    _lib.call("dmn_linear_attention_bwd", dtype, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), s0.data_ptr(), None, 0, do.data_ptr(),
              ds.data_ptr(), p[0], p[1], p[2], p[3] if decays else None, 0, p[4],
              ops._strides(q.stride()[:3], k.stride()[:3], v.stride()[:3], g.stride(), do.stride()[:3]), ws.data_ptr(), *sizes, dk ** -0.5,
              torch.cuda.current_stream().cuda_stream)
    assert (ws[n:] == 7.0).all()
    leaves = [x.requires_grad_(decays or i != 3) for i, x in enumerate((q, k, v, g, s0))]
    out = ops.linear_attention(*leaves)
    want = torch.autograd.grad(out, [x for x in leaves if x.requires_grad], [do, ds])
    assert all(torch.equal(a, b) for a, b in zip([x for i, x in enumerate(grads) if decays or i != 3], want))
