"""Linear attention (ops.linear_attention) over more than a million tokens and over far rows: padded columns stay zero and
offsets hold wherever a token lies.
"""
import pytest
import torch

from dms_amd import ops

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NAMES = ("q", "k", "v", "g")


def recurrence(q, k, v, g, scale):
    """One sample, one head, float64: o (T, dv)."""
    S, out = torch.zeros(q.shape[1], v.shape[1], dtype=torch.float64), []
    for t in range(q.shape[0]):
        S = S * g[t].exp() + k[t][:, None] * v[t]
        out.append(scale * (q[t] @ S))
    return torch.stack(out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dk,dv", [("bf16", 40, 40), ("bf16", 36, 100), ("fp32", 36, 20), ("fp32", 100, 100), ("fp16", 48, 72)])
def test_columns_behind_a_row_stay_out_of_sequences_of_more_than_2_20_tokens(dtype, dk, dv):
    """Rows lie in a wider tensor of NaN.  The chunks before the last 2^20 tokens know only their neighbours, as the decays of
    exp(-1/2) leave e^-100 of a token after 200 others: the ends of the long sequence are the ends of short ones.

    Bound, of the norm over 100 tokens: the output's half step (2^-8, 2^-11, 2^-24) and 2^-16 for the kernel's own sums, which
    are right to 2^-20 of sums of absolute values that are at most 2^3 of the results' norm here."""
    T, n, far = (1 << 20) + 700, 100, 300
    gen = torch.Generator(device=DEV).manual_seed(dk)

    def rows(d):
        room = torch.full((T, 1, 1, d + 8), float("nan"), dtype=DTYPES[dtype], device=DEV)
        room[..., :d] = torch.randn(T, 1, 1, d, generator=gen, device=DEV).to(DTYPES[dtype])
        return room[..., :d]

    dev = {"q": rows(dk), "k": rows(dk), "v": rows(dv), "g": torch.full((T, 1, 1), -0.5, device=DEV)}
    do = rows(dv)
    leaves = [dev[x].requires_grad_() for x in NAMES]
    o, s = ops.linear_attention(**dev)
    got = [o] + list(torch.autograd.grad(o, leaves, do))
    for name, x in zip(("o",) + NAMES, got):
        assert torch.isfinite(x).all(), name
    assert torch.isfinite(s).all()
    scale, bound = dk ** -0.5, torch.finfo(DTYPES[dtype]).eps / 2 + 2.0 ** -16
    for lo, hi, first in ((0, far, 0), (T - far, T, far - n)):                # the first n tokens, the last n
        short = [dev[x][lo:hi, 0, 0].detach().cpu().double().requires_grad_() for x in NAMES]
        want = recurrence(*short, scale)
        grads = torch.autograd.grad(want, short, do[lo:hi, 0, 0].cpu().double())
        for name, x, y in zip(("o",) + NAMES, got, (want.detach(),) + grads):
            x, y = x[lo:hi, 0, 0].detach().cpu().double()[first:first + n], y[first:first + n]
            assert float((x - y).norm()) <= bound * float(y.norm()), (name, lo, float((x - y).norm() / y.norm()))


@pytest.mark.gpu
def test_gradient_of_the_output_in_rows_too_far_apart():
    """What flows back is whatever the next operator made, here a slice of a far wider tensor: the result is that of its copy."""
    T, H, d = 3, 2, 16
    gen = torch.Generator().manual_seed(4)
    leaves = [torch.randn(T, 1, H, d, generator=gen).bfloat16().to(DEV).requires_grad_() for _ in range(3)]
    g = torch.full((T, 1, H), -0.1, device=DEV, requires_grad=True)
    o, _ = ops.linear_attention(*leaves, g)
    do = torch.randn(T, 1, H, d, generator=gen).bfloat16().to(DEV)
    room = torch.full((T, (1 << 24) + (1 << 20) + 8), float("nan"), dtype=torch.bfloat16, device=DEV)
    room[:, :H * d] = do.view(T, H * d)
    want = torch.autograd.grad(o, leaves + [g], do, retain_graph=True)
    got = torch.autograd.grad(o, leaves + [g], torch.as_strided(room, do.shape, (room.shape[1], H * d, d, 1)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_gradients_at_offsets_beyond_32_bits():
    """Rows 2^24 + 8 elements apart in the forward and backward pass: the last ones start behind 2^32 elements."""
    T, H, d, gap = 260, 2, 64, (1 << 24) + 8
    gen = torch.Generator().manual_seed(2)
    small = [torch.randn(T, 1, H, d, generator=gen).bfloat16().to(DEV) for _ in range(4)]
    g = torch.nn.functional.logsigmoid(torch.randn(T, 1, H, generator=gen)).to(DEV)
    room = torch.empty((T - 1) * gap + 4 * H * d, dtype=torch.bfloat16, device=DEV)
    far = [torch.as_strided(room, (T, 1, H, d), (gap, H * d, d, 1), i * H * d) for i in range(4)]
    for x, y in zip(far, small):
        x.copy_(y)

    def run(q, k, v, do):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, g)]
        out = ops.linear_attention(*leaves)
        return list(out) + list(torch.autograd.grad(out[0], leaves, do))

    for a, b in zip(run(*far), run(*small)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_decays_gradient_at_meeting_states_beyond_32_bits():
    """2^27 + 1024 tokens of one wide head: the states that meet at every 256th token take more than 2^31 groups of four.  All
    tokens are alike, so that far from either end S = k^T v / (1 - a), dS = scale q^T do / (1 - a) and the gradient is
    a <S, dS>, for every token the same.  Bound: sums of 24-bit products over the at most 60 tokens that exp(-t/2) leaves, the two
    states' and 256 dots' of the size of (1 - a)^2 / a = 0.26 of the gradient: 2^-15 of it."""
    T, d = (1 << 27) + 1024, 65
    if torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved() < 120 << 30:
        pytest.skip("needs 120 GiB of free GPU memory")
    torch.cuda.empty_cache()
    gen = torch.Generator().manual_seed(3)
    one = [torch.rand(1, 1, 1, d, generator=gen).bfloat16().to(DEV) for _ in range(4)]
    q, k, v, do = (x.expand(T, 1, 1, d) for x in one)
    g = torch.full((T, 1, 1), -0.5, device=DEV, requires_grad=True)
    o, _ = ops.linear_attention(q, k, v, g)
    got, = torch.autograd.grad(o, g, do)
    a, (q, k, v, do) = torch.tensor(-0.5, dtype=torch.float64).exp(), (x.double().cpu().flatten() for x in one)
    want = float(a * d ** -0.5 * (q @ k) * (v @ do) / (1 - a) ** 2)
    off = (got[512:T - 512] - want).abs_().max()
    assert float(off) <= 2.0 ** -15 * want, float(off) / want
    del o, got
    torch.cuda.empty_cache()
