"""What linear attention keeps of its numbers (ops.linear_attention): cases where the result is an exact small number that a
kernel with fewer bits cannot give, and bounds on the norm of the error.
"""
import pytest
import torch

from dms_amd import ops

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------ 24 bits of scores and states
# 2^20 + 2^10 + 1 takes 21 bits and has gaps too wide for two parts of 8 bits: less 2^20 + 2^10 it is 1, and 0 if its last bit was lost.
BIG = torch.tensor([1024.0, 32.0, 1.0])
LESS = torch.tensor([-1024.0, -32.0, 0.0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("width", [16, 48, 64, 128])
@pytest.mark.parametrize("T,first,second,reader", [(3, 0, 1, 2), (64, 3, 20, 63), (60, 10, 12, 50), (200, 130, 140, 159)])
def test_scores_keep_24_bits(dtype, width, T, first, second, reader):
    """Two tokens of one chunk whose scores with a third are 2^20 + 2^10 + 1 and -(2^20 + 2^10): o and the gradients that read
    them are exactly 1, each asked for alone and with the decays' gradient."""
    def at(*rows):
        x = torch.zeros(T, 1, 1, width)
        for t, r in rows:
            x[t, 0, 0, :len(r)] = r
        return x.to(DTYPES[dtype]).to(DEV)

    ones = torch.ones(width)
    g = torch.zeros(T, 1, 1, device=DEV)
    with torch.no_grad():
        o, _ = ops.linear_attention(at((reader, BIG)), at((first, BIG), (second, LESS)), at((first, ones), (second, ones)), g, scale=1.0)
    assert (o[reader] == 1).all()

    back = (T - 1 - reader, T - 1 - second, T - 1 - first) if T != 200 else (reader - 29, reader - 19, reader)   # reader before the two
    one, x, y = back
    zero = at()
    for leaf, q, k, v, do, token in (
            ("q", zero, at((first, ones), (second, ones)), at((first, BIG), (second, LESS)), at((reader, BIG)), reader),
            ("k", at((x, ones), (y, ones)), zero, at((one, BIG)), at((x, BIG), (y, LESS)), one),
            ("v", at((x, BIG), (y, LESS)), at((one, BIG)), zero, at((x, ones), (y, ones)), one)):
        for decays in (False, True):
            args = {"q": q.clone(), "k": k.clone(), "v": v.clone(), "g": g.clone()}
            args[leaf].requires_grad_()
            args["g"].requires_grad_(decays)
            o, _ = ops.linear_attention(**args, scale=1.0)
            got = torch.autograd.grad(o, [args[leaf]] + ([args["g"]] if decays else []), do)[0]
            assert (got[token] == 1).all(), (leaf, decays)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("width", [16, 64, 128])
def test_states_keep_24_bits(dtype, width):
    """States of 2^20 + 2^10 + 1 and -(2^20 + 2^10), read by a query, a key and a value of ones."""
    state = torch.zeros(1, 1, width, width, device=DEV)
    state[0, 0, 0], state[0, 0, 1] = 2.0 ** 20 + 1025, -(2.0 ** 20 + 1024)
    x = torch.zeros(3, 1, 1, width, device=DEV, dtype=DTYPES[dtype])
    two = x.clone()
    two[1, 0, 0, :2] = 1
    g = torch.zeros(3, 1, 1, device=DEV)
    with torch.no_grad():
        o, _ = ops.linear_attention(two, x, x, g, state, scale=1.0)
    assert (o[1] == 1).all()
    for decays in (False, True):
        for leaf in "qkv":
            args = {n: x.clone() for n in "qkv"}
            args["g"] = g.clone().requires_grad_(decays)
            args["state0"] = state.transpose(2, 3).contiguous() if leaf == "q" else torch.zeros_like(state)
            if leaf != "q":
                args["v" if leaf == "k" else "k"].copy_(two)
            args[leaf].requires_grad_()
            o, s = ops.linear_attention(**args, scale=1.0)
            ds = torch.zeros_like(s) if leaf == "q" else (state.transpose(2, 3).contiguous() if leaf == "k" else state)
            got = torch.autograd.grad([o, s], [args[leaf]] + ([args["g"]] if decays else []), [two if leaf == "q" else x, ds])[0]
            assert (got[1] == 1).all(), (leaf, decays)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("dk,dv,H", [(64, 64, 3), (32, 100, 2), (125, 125, 2), (20, 32, 260)])
def test_frozen_decays_leave_the_other_gradients_as_they_are(dtype, dk, dv, H):
    gen = torch.Generator().manual_seed(dk)
    T, B = 150, 1
    make = lambda *shape: torch.randn(shape, generator=gen).to(DTYPES[dtype]).to(DEV)  # noqa: E731
    q, k, v, do = make(T, B, H, dk), make(T, B, H, dk), make(T, B, H, dv), make(T, B, H, dv)
    g = torch.nn.functional.logsigmoid(torch.randn(T, B, H, generator=gen)).to(DEV)
    state, ds = (torch.randn(B, H, dk, dv, generator=gen).to(DEV) for _ in range(2))
    got = []
    for decays in (False, True):
        leaves = [x.clone().requires_grad_() for x in (q, k, v, state)]
        gate = g.clone().requires_grad_(decays)
        out = ops.linear_attention(*leaves[:3], gate, leaves[3])
        got.append(torch.autograd.grad(out, leaves + ([gate] if decays else []), [do, ds])[:4])
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------ the decays' gradient
def recurrence(q, k, v, g, state, scale):
    """One head, float64: q, k (T, B, dk), v (T, B, dv), g (T, B), state (B, dk, dv); returns o, state."""
    out = []
    for t in range(q.shape[0]):
        state = state * g[t].exp()[:, None, None] + k[t][:, :, None] * v[t][:, None, :]
        out.append(scale * (q[t][:, :, None] * state).sum(1))
    return torch.stack(out), state


def recurrence_grads(args, scale, do, ds):
    leaves = [x.clone().requires_grad_() for x in args]
    o, s = recurrence(*leaves, scale)
    return [o.detach(), s.detach()] + list(torch.autograd.grad((o * do).sum() + (s * ds).sum(), leaves))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("dk,dv", [(24, 16), (64, 64), (64, 100), (100, 128), (128, 128)])
def test_decays_gradient_does_not_carry_errors_past_a_256th_token(dtype, dk, dv):
    """Tokens 0 to 249 are 2^6 times the others in q, k, v and their output's gradient, their dots 2^24 times; a reset behind
    them.  From token 256 on the gradient starts anew from the states that meet there, so that it is right to 2^-15 of the
    magnitudes of its own 256 tokens (derived for the gradient far from either end: twice the dots' errors, and the two ends')."""
    T, B = 600, 1
    gen = torch.Generator().manual_seed(dk + dv)
    make = lambda *shape: torch.randn(shape, generator=gen)  # noqa: E731
    q, k, v, do, ds, state = make(T, B, dk), make(T, B, dk), make(T, B, dv), make(T, B, dv), make(B, dk, dv), make(B, dk, dv)
    for x in (q, k, v, do):
        x[:250] *= 64
    q, k, v, do = (x.to(DTYPES[dtype]) for x in (q, k, v, do))
    g = 0.1 * torch.nn.functional.logsigmoid(make(T, B))
    g[250] = -1e4                                              # a reset that autograd in 64 bits has a gradient of: 0
    dev = [x.unsqueeze(2).to(DEV) for x in (q, k, v, g)] + [state.unsqueeze(1).to(DEV)]
    dev[3].requires_grad_()
    out = ops.linear_attention(*dev)
    got, = torch.autograd.grad(out, [dev[3]], [do.unsqueeze(2).to(DEV), ds.unsqueeze(1).to(DEV)])
    args = [x.double() for x in (q, k, v, g, state)]
    scale = dk ** -0.5
    want = recurrence_grads(args, scale, do.double(), ds.double())[5]
    size = [x if i == 3 else x.abs() for i, x in enumerate(args)]
    mag = recurrence_grads(size, scale, do.double().abs(), ds.double().abs())
    flow = (size[0] * mag[2] + size[1] * mag[3]).sum(-1)
    for t in (256, 512):
        end = min(t + 256, T)
        far = mag[5][end] if end < T else (mag[1] * ds.double().abs()).sum((-1, -2))
        bound = mag[5][t] + far + 2 * flow[t:end].sum(0)
        over = (got[t:end, :, 0].cpu().double() - want[t:end]).abs() - (2.0 ** -15 * bound + 2.0 ** -24 * want[t:end].abs())
        assert float(over.max()) <= 0.0, (t, float(over.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("T", [901, 1301])
def test_gradient_of_one_decay_for_each_head_sums_in_64_bits(dtype, T):
    """Whole numbers in one column, no decay: every token's gradient is a whole number below 2^24, each sample's sum is beyond
    it, and the samples cancel down to a number that 32 bits hold again: the result is exact only if no sum was rounded."""
    B, H, width = 2, 3, 16
    def ones(sign=None):                                       # noqa: E306
        x = torch.zeros(T, B, H, width)
        x[..., 0] = 1
        if sign is not None:
            x[:, 1, :, 0] = sign
        return x
    k, do = ones(), ones(-1.0)
    k[0, 1, :, 0] = 2
    S, R = k[..., 0].double().cumsum(0), do[..., 0].double().flip(0).cumsum(0).flip(0)
    tokens = torch.cat([torch.zeros(1, B, H, dtype=torch.float64), S[:-1] * R[1:]])
    parts = tokens.sum(0)
    want = parts.sum(0)
    assert float(tokens.abs().max()) < 2 ** 24 and float(parts.abs().min()) > 2 ** 24 and float(want.abs().max()) < 2 ** 24
    assert (parts.float().double().sum(0) != want).all()       # with sums in 32 bits the test would not hold
    q, k, v, do = (x.to(DTYPES[dtype]).to(DEV) for x in (ones(), k, ones(), do))
    g = torch.zeros(H, device=DEV, requires_grad=True)
    o, _ = ops.linear_attention(q, k, v, g, scale=1.0)
    got, = torch.autograd.grad(o, g, do)
    assert torch.equal(got.cpu().double(), want)


# ------------------------------------------------------------------------------------ decays that last
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,chunk", [("bf16", 64), ("fp32", 32), ("fp16", 32)])
@pytest.mark.parametrize("H,chunks", [(256, 1024), (1, 4096)])
def test_one_decay_for_every_token_does_not_add_up_its_rounding(dtype, chunk, H, chunks):
    """A state that only decays, by the same factor for every chunk, forwards and (its gradient) backwards, in one piece and cut
    into segments.  The factor is one that 32 bits miss by a quarter of a step, 2^-26, or more: kept there, it is off by
    chunks * 2^-26 after them.  What remains is a rounding of the state for each chunk, at most 2^-24 and of either sign over its
    elements: sqrt(chunks) * 2^-24 of the norm."""
    T, width = chunks * chunk, 16
    for i in range(1000):                                      # until the chunk's factor lies that far from a float
        g = torch.full((H,), -8.0 / T * (1 + i / 1000))
        factor = (chunk * g[0].double()).exp()
        if 2.0 ** -26 <= abs(float(factor.float().double() / factor - 1)):
            break
    else:
        raise AssertionError("no such decay")
    gen = torch.Generator().manual_seed(1)
    state, ds = (torch.randn(1, H, width, width, generator=gen).to(DEV) for _ in range(2))
    x = torch.zeros(1, 1, 1, width, dtype=DTYPES[dtype], device=DEV).expand(T, 1, H, width)
    state.requires_grad_()
    _, s = ops.linear_attention(x, x, x, g.to(DEV), state)
    grad, = torch.autograd.grad(s, state, ds)
    whole = (T * g[0].double()).exp()
    for got, start in ((s, state), (grad, ds)):
        want = start.detach().double().cpu() * whole
        off = (got.detach().cpu().double() - want).norm() / want.norm()
        assert float(off) <= chunks ** 0.5 * 2.0 ** -24, float(off)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("width,T", [(16, 8192), (64, 4096), (128, 4096)])
def test_a_state_is_rounded_once_for_32_tokens(dtype, width, T):
    """No decay, terms of either sign: the state grows with the root of the tokens, |S_n|^2 = |S_N|^2 n / N after n of N times 32
    tokens.  A rounding to nearest is off by 2^-24 / sqrt(3) of the number in the mean square; one for each 32 tokens adds up to
    sqrt(N / 2) of that, and what the tokens add, |S_N|^2 over all, is a chain of at most 8 roundings itself:
    2^-24 / sqrt(3) sqrt(N / 2 + 8) of the norm over at least 2^16 elements.  (A rounding for each product would be 2 to 6 for 32.)"""
    H = 256
    gen = torch.Generator(device=DEV).manual_seed(width)
    a, b = (torch.randn(T, 1, H, width, generator=gen, device=DEV).to(DTYPES[dtype]) for _ in range(2))
    zero = torch.zeros(1, 1, 1, width, dtype=DTYPES[dtype], device=DEV).expand(T, 1, H, width)
    want = torch.bmm(a[:, 0].permute(1, 2, 0).double().contiguous(), b[:, 0].transpose(0, 1).double().contiguous())
    g = torch.zeros(H, device=DEV)
    with torch.no_grad():
        _, s = ops.linear_attention(zero, a, b, g, scale=1.0)
    state = torch.zeros(1, H, width, width, device=DEV, requires_grad=True)
    o, _ = ops.linear_attention(a, zero, zero, g, state, scale=1.0)
    ds, = torch.autograd.grad(o, state, b)
    for x in (s, ds):
        off = float((x[0].double() - want).norm() / want.norm())
        assert off <= 2.0 ** -24 * ((T / 64 + 8) / 3) ** 0.5, off


# ------------------------------------------------------------------------------------ by the norm
def norm_case(seed, T, dk, dv):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, generator=gen)  # noqa: E731
    B = 2
    args = [rnd(T, B, dk), rnd(T, B, dk), rnd(T, B, dv), 0.2 * torch.nn.functional.logsigmoid(1 + rnd(T, B)), rnd(B, dk, dv)]
    return args, rnd(T, B, dv), rnd(B, dk, dv), dk ** -0.5


# Of the norm.  Three planes leave 2^-26 of an operand in the mean, a sum passes about 32 roundings of 2^-24 / sqrt(3) with what it
# has gathered, sqrt(32) of them in the mean square: 2^-22.3, and three such stages (scores, state, output) below 2^-21.  The
# decays' gradient gathers the dots of up to 256 tokens, whose errors grow with the root of the distance to a meeting state as
# the gradient itself does with the root of what a state remembers, here about 20 tokens: sqrt(128 / 20) of that.
NORM, NORM_DECAYS = 2.0 ** -21, 2.0 ** -19.6
NAMES = ("o", "state", "q", "k", "v", "g", "state0")
NORM_CASES = [(20, 64, 64), (300, 64, 64), (700, 100, 36), (290, 128, 128), (1100, 32, 24)]


def norm_of_error(got, want):
    return float((got.detach().cpu().double().reshape(want.shape) - want).norm() / want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("T,dk,dv", NORM_CASES)
def test_fp32_results_by_their_norm(T, dk, dv):
    args, do, ds, scale = norm_case(T, T, dk, dv)
    dev = [x.unsqueeze(2 if i < 4 else 1).to(DEV).requires_grad_() for i, x in enumerate(args)]
    out = ops.linear_attention(*dev)
    got = list(out) + list(torch.autograd.grad(out, dev, [do.unsqueeze(2).to(DEV), ds.unsqueeze(1).to(DEV)]))
    want = recurrence_grads([x.double() for x in args], scale, do.double(), ds.double())
    for name, x, y in zip(NAMES, got, want):
        assert norm_of_error(x, y) <= (NORM_DECAYS if name == "g" else NORM), (name, norm_of_error(x, y))


@pytest.mark.parametrize("at,T", [(0, 300), (1, 300), (2, 300), (4, 20)])        # the first state fades
def test_a_lost_plane_would_be_seen(at, T):
    """The same bounds reject 64-bit results of inputs of which one kept two planes, 16 bits, only."""
    args, do, ds, scale = norm_case(T, T, 64, 64)
    args = [x.double() for x in args]
    want = recurrence_grads(args, scale, do.double(), ds.double())
    high = args[at].bfloat16().double()
    spoilt = list(args)
    spoilt[at] = high + (args[at] - high).bfloat16().double()
    got = recurrence_grads(spoilt, scale, do.double(), ds.double())
    assert any(norm_of_error(x, y) > (NORM_DECAYS if name == "g" else NORM) for name, x, y in zip(NAMES, got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("T", [65, 200, 256])
def test_decays_gradient_is_tied_behind_the_last_token(dtype, T):
    """Tokens of the first half 2^6 times the others in q, k, v and their output's gradient, their dots 2^24 times; a reset behind
    them.  What the sum has missed up to there, E, stays with it; known behind the last token as well, E is spread over the T tokens:
    E (1 - t / T) is left at t, E / T at the last, twice that for its rounding, where a sum that only starts right leaves E."""
    B, dk, dv, half = 16, 32, 32, T // 2
    gen = torch.Generator().manual_seed(T)
    make = lambda *shape: torch.randn(shape, generator=gen)  # noqa: E731
    q, k, v, do, ds, state = make(T, B, dk), make(T, B, dk), make(T, B, dv), make(T, B, dv), make(B, dk, dv), make(B, dk, dv)
    for x in (q, k, v, do):
        x[:half] *= 64
    q, k, v, do = (x.to(DTYPES[dtype]) for x in (q, k, v, do))
    g = 0.1 * torch.nn.functional.logsigmoid(make(T, B))
    g[half] = -1e4
    dev = [x.unsqueeze(2).to(DEV) for x in (q, k, v, g)] + [state.unsqueeze(1).to(DEV)]
    dev[3].requires_grad_()
    got, = torch.autograd.grad(ops.linear_attention(*dev), [dev[3]], [do.unsqueeze(2).to(DEV), ds.unsqueeze(1).to(DEV)])
    args = [x.double() for x in (q, k, v, g, state)]
    want = recurrence_grads(args, dk ** -0.5, do.double(), ds.double())[5]
    off = (got[:, :, 0].cpu().double() - want).abs()
    first, last = off[half + 1], off[-1]
    missed = first / (1 - (half + 1) / T)
    # the small tokens' own errors: 2^-15 of their magnitudes, as for every such sum
    size = [x if i == 3 else x.abs() for i, x in enumerate(args)]
    mag = recurrence_grads(size, dk ** -0.5, do.double().abs(), ds.double().abs())
    flow = (size[0] * mag[2] + size[1] * mag[3]).sum(-1)[half + 1:].sum(0)
    own = 2.0 ** -15 * ((mag[1] * ds.double().abs()).sum((-1, -2)) + 2 * flow)
    assert (last <= 2 * missed / T + own).all(), (last / missed).max()
    assert float(missed.median()) > 8 * float(own.median())    # else nothing was told apart
