"""The layer dms_amd.LinearAttention: norm, rotation, recurrence, its step and the projections round them together, against
the same layer in 64 bits.

Bound.  Products of n <= 64 terms in fp32 are right to 64 * 2^-24 of the sum of their absolute values, the recurrence to 2^-16
of it and the rotation to 2^-20 (tests of the operators).  The layer chains a projection, a rotation, the recurrence and a
projection; where terms of size 1 add up to a sum about 8 times smaller than their absolute values, each stage gives at most
8 * 2^-16 of the norm and passes on what came in: 4 * 8 * 2^-16 = 2^-11.  A backward pass chains the same stages once more: 2^-10.
"""
import pytest
import torch
import torch.nn.functional as F

import dms_amd
from dms_amd import ops

DEV = "cuda"


def plain(p, layer, x, state, pos, lengths):
    """The layer in float64 on the CPU from its parameters p."""
    T, B = x.shape[:2]
    W, Hq, H = layer.width, layer.qk_heads, layer.heads
    q, k, v = (x @ p["weight"]).split([Hq * W, Hq * W, H * W], -1)
    q, k, v = q.view(T, B, Hq, W), k.view(T, B, Hq, W), v.view(T, B, H, W)
    g = F.logsigmoid(x @ p["gate"] + p["gate_bias"]) * layer.DECAY_SCALE

    def turned(y, w):
        y = y * (y.square().mean(-1, keepdim=True) + layer.eps).rsqrt() * w
        if not layer.sections:
            return y
        angle = torch.cat([pos[..., a:a + 1].double() * torch.tensor([layer.base ** (-j / n) for j in range(n)], dtype=torch.float64)
                           for a, n in enumerate(layer.sections)], -1)
        angle = F.pad(angle, (0, (W + 1) // 2 - angle.shape[-1])).view(T, -1, 1, (W + 1) // 2)
        z = F.pad(y, (0, W % 2)).unflatten(-1, (-1, 2))
        return torch.stack([z[..., 0] * angle.cos() - z[..., 1] * angle.sin(), z[..., 0] * angle.sin() + z[..., 1] * angle.cos()],
                           -1).flatten(-2)[..., :W]

    q, k = (turned(y, p[n]).repeat_interleave(H // Hq, 2) for y, n in ((q, "q_norm"), (k, "k_norm")))
    S = torch.zeros(B, H, W, W, dtype=torch.float64) if state is None else state
    out = []
    for t in range(T):
        live = (torch.ones(B, dtype=torch.bool) if lengths is None else t < lengths).view(B, 1, 1, 1)
        S = torch.where(live, S * g[t].exp()[..., None, None] + k[t][..., :, None] * v[t][..., None, :], S)
        out.append(torch.where(live[..., 0], (q[t][..., :, None] * S).sum(-2) * W ** -0.5, 0.0))
    return torch.stack(out).view(T, B, H * W) @ p["out"], S


def near(got, want, bound):
    got = got.detach().cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all()
    assert float((got - want).norm()) <= bound * float(want.norm()), float((got - want).norm() / want.norm())


def make(dtype=torch.float32, sections=(4, 5, 5), heads=4, qk=2, width=29):
    torch.manual_seed(0)
    layer = dms_amd.LinearAttention(40, heads * width, heads, qk, sections).to(dtype).to(DEV)
    with torch.no_grad():
        layer.gate_bias.uniform_(-1, 3)
        layer.q_norm.uniform_(0.5, 1.5)
        layer.k_norm.uniform_(0.5, 1.5)
    return layer


@pytest.mark.gpu
def test_layer_with_its_gradients():
    layer = make()
    H, W, L, B = 3, 4, 6, 2
    T = H * W * L
    gen = torch.Generator().manual_seed(1)
    x, s0 = torch.randn(T, B, 40, generator=gen), torch.randn(B, 4, 29, 29, generator=gen)
    dh, ds = torch.randn(T, B, layer.n_out, generator=gen), torch.randn(s0.shape, generator=gen)
    pos = ops.map_positions(H, W, L, DEV)
    lengths = torch.tensor([T, 41])
    xd, sd = x.to(DEV).requires_grad_(), s0.to(DEV).requires_grad_()
    h, s = layer(xd, sd, pos, lengths.to(DEV))
    named = dict(layer.named_parameters())
    grads = torch.autograd.grad([h, s], [xd, sd] + list(named.values()), [dh.to(DEV), ds.to(DEV)])
    p = {n: w.detach().cpu().double().requires_grad_() for n, w in named.items()}
    xr, sr = x.double().requires_grad_(), s0.double().requires_grad_()
    want = plain(p, layer, xr, sr, pos.cpu().unsqueeze(1), lengths)
    wg = torch.autograd.grad(want, [xr, sr] + [p[n] for n in named], [dh.double(), ds.double()])
    near(h, want[0].detach(), 2.0 ** -11)
    near(s, want[1].detach(), 2.0 ** -11)
    assert not h[41:, 1].any()
    for name, a, b in zip(["x", "state"] + list(named), grads, wg):
        near(a, b, 2.0 ** -10)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_captured_steps(dtype):
    """A prompt of two lengths, then single tokens through one captured graph, against the layer over the whole sequences."""
    layer = make(dtype, width=32, sections=(6, 6)).eval()
    gen = torch.Generator().manual_seed(2)
    T, new, B = 50, 5, 2
    lengths = torch.tensor([50, 33], dtype=torch.int32, device=DEV)
    x = torch.randn(T + new, B, 40, generator=gen).to(dtype).to(DEV)
    at = torch.arange(T + new, device=DEV)
    pos = torch.stack([at, at // 7], -1).unsqueeze(1).repeat(1, B, 1)
    for b in range(B):                                     # the new tokens follow on each sample's own last one
        n = int(lengths[b])
        pos[T:, b] = torch.stack([torch.arange(n, n + new, device=DEV), torch.arange(n, n + new, device=DEV) // 7], -1)
    with torch.no_grad():
        _, state = layer(x[:T], None, pos[:T], lengths)
        token, where = x[T].clone(), pos[T].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        scratch = state.clone()
        with torch.cuda.stream(side):
            layer.step(token, scratch, where)
        torch.cuda.current_stream().wait_stream(side)
        graph, live = torch.cuda.CUDAGraph(), state.clone()
        with torch.cuda.graph(graph):
            h = layer.step(token, live, where)
        live.copy_(state)
        got = []
        for t in range(T, T + new):
            token.copy_(x[t])
            where.copy_(pos[t])
            eager = layer.step(x[t], state, pos[t])
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(h, eager) and torch.equal(live, state)
            got.append(eager)
    p = {n: w.detach().cpu().double() for n, w in layer.named_parameters()}
    # bf16: each stage rounds its result to half a step, 2^-9 rms and less; five stages in a row and their products: 2^-5
    bound = 2.0 ** -11 if dtype == torch.float32 else 2.0 ** -5
    for b in range(B):
        n = int(lengths[b])
        rows = list(range(n)) + list(range(T, T + new))
        want, s = plain(p, layer, x.cpu().double()[rows][:, b:b + 1], None, pos.cpu()[rows][:, b:b + 1], None)
        near(torch.stack(got)[:, b], want[n:, 0], bound)
        near(state[b], s[0], bound)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_nothing_to_read_leaves_the_state(grad):
    layer = make(torch.float32, width=16, sections=(3,))
    state = torch.randn(2, layer.heads, 16, 16, device=DEV)
    with torch.set_grad_enabled(grad):
        for T, B in ((0, 2), (3, 0)):
            h, after = layer(torch.zeros(T, B, 40, device=DEV), state[:B], torch.zeros(T, B, 1, dtype=torch.int32, device=DEV))
            assert h.shape == (T, B, layer.n_out) and torch.equal(after, state[:B])
            if grad:
                (h.sum() + after.sum()).backward()
    if grad:
        assert all(p.grad is None or not p.grad.any() for p in layer.parameters())


def test_layer_refusals():
    with pytest.raises(ValueError, match="multiple"):
        dms_amd.LinearAttention(8, 30, 4)
    with pytest.raises(ValueError, match="multiple"):
        dms_amd.LinearAttention(8, 32, 4, 3)
    with pytest.raises(ValueError, match="at most 128"):
        dms_amd.LinearAttention(8, 400, 2)
    layer = dms_amd.LinearAttention(8, 32, 4, 2, (2,))
    assert {n: tuple(p.shape) for n, p in layer.named_parameters()} == {
        "weight": (8, 64), "gate": (8, 4), "gate_bias": (4,), "q_norm": (8,), "k_norm": (8,), "out": (32, 32)}
    with pytest.raises(ValueError, match="expects"):
        layer(torch.zeros(3, 1, 9))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layer(torch.zeros(3, 1, 8), positions=torch.zeros(3, 1, dtype=torch.long))
