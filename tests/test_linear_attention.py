"""Linear attention with a decay for each head (ops.linear_attention, ops.linear_attention_step) against the recurrence
in 64 bits, and its refusals.

Bounds.  Every output is a sum of products; `plain` run on the absolute values of the inputs gives the sum of their
absolute values, `mag`.  A computed operand is kept in planes that leave at most 2^-18 of it (two bf16 planes, beside bf16
and fp16 inputs) or 2^-27 (three, beside fp32), products of planes that are left out are of that size again, and a
term meets at most 3 such operands (the decayed value in the state, the state, the product inside a chunk).  A decay's
exponent is right to half a step of itself, |x| 2^-25 for 2^x: terms with |x| > 32 are below 2^-32 of the others, so 2^-20.
Every fp32 accumulation adds half a step, 2^-24: a term passes 1 + 2 * 3 of them (scaling; matrix instructions) in every
chunk that the state lives through and at most 32 in its own output's chunk, so with the at most 10 chunks here
(T <= 320, 32 tokens and more in a chunk) fewer than 128: 2^-17.  Together
    |error| <= DELTA * mag + eps/2 * |value|,   DELTA = 2^-15 for 16-bit types (6 * 2^-18 + 2^-20 + 2^-17), 2^-16 for fp32,
with eps/2 the rounding of the output's type.
"""
import math

import pytest
import torch

from dms_amd import _lib, ops

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DELTA = {"fp32": 2.0 ** -16, "bf16": 2.0 ** -15, "fp16": 2.0 ** -15}


# ------------------------------------------------------------------------------------ the recurrence in 64 bits
def plain(q, k, v, g, state0, lengths, scale):
    """Token by token; every argument float64 on the CPU, heads as given.  Returns o, state."""
    T, B, H = q.shape[0], q.shape[1], g.shape[-1]
    q, k, v = (x.repeat_interleave(H // x.shape[2], 2) for x in (q, k, v))
    g = g.expand(T, B, H)
    S = torch.zeros(B, H, q.shape[3], v.shape[3], dtype=torch.float64) if state0 is None else state0
    out = []
    for t in range(T):
        live = torch.ones(B, dtype=torch.bool) if lengths is None else t < lengths
        w = live.view(B, 1, 1, 1)
        new = S * g[t].exp()[..., None, None] + k[t][..., :, None] * v[t][..., None, :]
        S = torch.where(w, new, S)
        out.append(torch.where(w[..., 0], scale * (q[t][..., :, None] * S).sum(-2), 0.0))
    o = torch.stack(out) if T else torch.zeros(0, B, H, v.shape[3], dtype=torch.float64)
    return o, S


def plain_grads(q, k, v, g, state0, lengths, scale, do, ds):
    leaves = [x.clone().requires_grad_() for x in (q, k, v, g)] + ([state0.clone().requires_grad_()] if state0 is not None else [])
    o, s = plain(*leaves[:4], leaves[4] if state0 is not None else None, lengths, scale)
    loss = (s * ds).sum() + (o * do).sum()
    return [o.detach(), s.detach()] + [x if x is not None else torch.zeros_like(l) for x, l in
                                       zip(torch.autograd.grad(loss, leaves, allow_unused=True), leaves)]


def rnd(gen, *shape):
    return torch.randn(shape, generator=gen)


def make(dtype, T, B, H, dk, dv, Hq=None, Hk=None, Hv=None, fixed=False, ragged=False, state=False, resets=(), seed=0):
    gen = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    q, k, v = (rnd(gen, T, B, h or H, d).to(dt) for h, d in ((Hq, dk), (Hk, dk), (Hv, dv)))
    g = torch.nn.functional.logsigmoid(1 + 2 * rnd(gen, *((H,) if fixed else (T, B, H))))
    for t in resets:
        g[t] = -math.inf
    s0 = rnd(gen, B, H, dk, dv) if state else None
    lengths = torch.randint(0, T + 1, (B,), generator=gen, dtype=torch.int32) if ragged else None
    do, ds = rnd(gen, T, B, H, dv).to(dt), rnd(gen, B, H, dk, dv)
    return dict(q=q, k=k, v=v, g=g, state0=s0, lengths=lengths), do, ds, float(dk) ** -0.5


def f64(x):
    return None if x is None else x.detach().cpu().double()


def bounded(got, want, mag, dtype, delta):
    got, want = f64(got), want
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny                       # a subnormal's half step, and what the exponential flushes
    over = (got - want).abs() - (delta * mag + half * want.abs() + tiny)
    assert float(over.max() if over.numel() else 0.0) <= 0.0, "off by %g beyond its bound" % float(over.max())


def check_forward(a, scale, dtype, **call):
    dev = {n: (x.to(DEV) if x is not None else None) for n, x in a.items()}
    dev.update(call)
    with torch.no_grad():
        o, s = ops.linear_attention(**dev)
    args = [f64(a[n]) for n in ("q", "k", "v", "g", "state0")] + [a["lengths"]]
    want = plain(*args, scale)
    mag = plain(*[x.abs() if x is not None and i != 3 else x for i, x in enumerate(args[:5])], args[5], scale)
    assert o.dtype == DTYPES[dtype] and s.dtype == torch.float32
    bounded(o, want[0], mag[0], o.dtype, DELTA[dtype])
    bounded(s, want[1], mag[1], s.dtype, DELTA[dtype])
    return o, s


CASES = [
    # dtype, T, B, H, dk, dv, more
    ("fp32", 1, 1, 1, 1, 1, {}),
    ("fp32", 1, 3, 2, 125, 125, dict(state=True)),
    ("bf16", 2, 2, 3, 3, 5, dict(fixed=True)),
    ("fp32", 20, 1, 8, 125, 125, {}),
    ("bf16", 31, 2, 2, 16, 32, dict(state=True)),
    ("fp32", 32, 2, 2, 32, 32, dict(ragged=True)),
    ("fp32", 33, 2, 2, 33, 16, dict(ragged=True, state=True)),
    ("bf16", 64, 2, 2, 64, 64, dict(ragged=True)),
    ("bf16", 65, 1, 4, 64, 64, dict(state=True, Hq=2, Hk=2)),
    ("fp16", 63, 2, 4, 100, 100, dict(Hk=1, Hv=1, ragged=True)),
    ("fp16", 129, 1, 2, 128, 64, dict(state=True)),
    ("fp32", 130, 2, 4, 64, 128, dict(Hq=2, Hk=2, resets=(0, 40, 64, 129), state=True)),
    ("bf16", 300, 2, 2, 128, 128, dict(ragged=True, state=True, resets=(63, 64, 128))),
    ("bf16", 257, 3, 1, 70, 40, dict(Hq=1, ragged=True, fixed=True)),
    ("fp32", 320, 1, 2, 100, 100, dict(state=True)),
    ("fp16", 200, 2, 2, 32, 17, dict(ragged=True, state=True, resets=(7,))),
    ("fp32", 70, 2, 4, 64, 64, dict(Hq=2, Hk=1, Hv=2)),
    ("bf16", 140, 1, 4, 64, 100, dict(Hq=1, Hv=2, state=True)),
]


def _id(c):
    return "%s-T%d-B%d-H%d-%dx%d-%s" % (c[:6] + ("_".join(sorted(c[6])) or "plain",))


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_forward(case):
    dtype, T, B, H, dk, dv, more = case
    a, _, _, scale = make(dtype, T, B, H, dk, dv, seed=T, **more)
    check_forward(a, scale, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_backward(case):
    dtype, T, B, H, dk, dv, more = case
    a, do, ds, scale = make(dtype, T, B, H, dk, dv, seed=T + 1, **more)
    names = ["q", "k", "v", "g"] + (["state0"] if a["state0"] is not None else [])
    dev = {n: (x.to(DEV) if x is not None else None) for n, x in a.items()}
    for n in names:
        dev[n].requires_grad_()
    o, s = ops.linear_attention(**dev)
    got = [o, s] + list(torch.autograd.grad([o, s], [dev[n] for n in names], [do.to(DEV), ds.to(DEV)]))
    args = [f64(a[n]) for n in ("q", "k", "v", "g", "state0")] + [a["lengths"], scale]
    want = plain_grads(*args, f64(do), f64(ds))
    absolute = [x.abs() if x is not None and i != 3 else x for i, x in enumerate(args[:5])] + args[5:]
    mag = plain_grads(*absolute, f64(do).abs(), f64(ds).abs())
    # the decay's gradient is a running sum over the tokens before it of what enters through the queries and leaves through
    # the keys, from what came in with the first state: each summand is bounded by its own magnitude
    rep = lambda x: x.sum(-1).reshape(T, B, -1)  # noqa: E731
    full = [f64(a[n]).abs().repeat_interleave(H // a[n].shape[2], 2) for n in ("q", "k", "v")]
    wide = plain_grads(*full, f64(a["g"]).expand(T, B, H), absolute[4], a["lengths"], scale, f64(do).abs(), f64(ds).abs())
    flow = rep(full[0] * wide[2]) + rep(full[1] * wide[3])
    mag_g = flow.cumsum(0) + ((wide[6] * absolute[4]).sum((-1, -2))[None] if a["state0"] is not None else 0.0)
    mag[5] = mag_g.sum((0, 1)) if a["g"].dim() == 1 else mag_g
    for n, x, y, m in zip(["o", "state"] + names, got, want, mag):
        bounded(x, y, m, x.dtype, DELTA[dtype] * (2 if n == "g" else 1))       # g: two operands carry the error


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,T,dk,dv,end", [("fp32", 1100, 16, 16, True), ("bf16", 1100, 16, 24, True), ("fp16", 513, 24, 16, False),
                                               ("bf16", 257, 64, 64, False), ("fp32", 512, 33, 16, True), ("bf16", 1100, 100, 128, True),
                                               ("fp32", 1025, 128, 100, False)])
def test_gradient_of_the_decays_far_from_either_end(dtype, T, dk, dv, end):
    """Lengths on both sides of every 256th token, where (at every second one for wide states) the gradient is known from the
    states that meet there.  In between it is a sum of at most 256 (512) dots that starts at one of them and is corrected at the next, so that its error stays below that of the two
    and twice that of the dots: 24 bits of each operand beside every type (2 * 2^-26), 2^-20 for the exponents, and 7 roundings of
    2^-24 in at most 35 chunks with 64 for the dot and its chunk, 2^-15.7: 2^-15."""
    lengths = [n for n in (0, 1, 255, 256, 257, 511, 512, 513, 1024, 1025, 1100) if n <= T]
    a, do, ds, scale = make(dtype, T, len(lengths), 1, dk, dv, state=True, resets=(128, 256), seed=T + 5)
    a["g"] = a["g"] * 0.1                                  # states that live for a while
    a["lengths"] = torch.tensor(lengths)
    ds = ds if end else torch.zeros_like(ds)
    dev = {n: x.to(DEV) for n, x in a.items()}
    dev["g"].requires_grad_()
    o, s = ops.linear_attention(**dev)
    got, = torch.autograd.grad([o, s] if end else [o], [dev["g"]], [do.to(DEV), ds.to(DEV)][:2 if end else 1])
    args = [f64(a[n]) for n in ("q", "k", "v", "g", "state0")]
    want = plain_grads(*args, a["lengths"], scale, f64(do), f64(ds))[5]
    size = [x.abs() if i != 3 else x for i, x in enumerate(args)]
    mag = plain_grads(*size, a["lengths"], scale, f64(do).abs(), f64(ds).abs())
    ends = (mag[1] * f64(ds).abs()).sum((-1, -2))          # what meets behind the last token
    flow = (size[0] * mag[2] + size[1] * mag[3]).sum(-1)
    bound = torch.zeros_like(want)
    step = 256 if max(dk, dv) <= 64 else 512
    for t in range(0, T, step):
        far = torch.where((torch.tensor(lengths) > t + step)[:, None], mag[5][min(t + step, T - 1)], ends)
        bound[t:t + step] = mag[5][t] + far + 2 * flow[t:t + step].sum(0)
    bounded(got, want, bound, torch.float32, 2.0 ** -15)


def test_plain_gradients_are_differences():
    """The 64-bit gradients that the kernels are held to, against central differences."""
    a, do, ds, scale = make("fp32", 5, 2, 2, 3, 2, Hk=1, state=True, ragged=True, seed=4)
    args = [f64(a[n]) for n in ("q", "k", "v", "g", "state0")]
    grads = plain_grads(*args, a["lengths"], scale, f64(do), f64(ds))[2:]
    value = lambda xs: sum((x * w).sum() for x, w in zip(plain(*xs, a["lengths"], scale), (f64(do), f64(ds))))  # noqa: E731
    for i, (x, gr) in enumerate(zip(args, grads)):
        way = torch.randn(x.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        h = 1e-5
        up, down = list(args), list(args)
        up[i], down[i] = x + h * way, x - h * way
        assert abs(float((value(up) - value(down)) / (2 * h) - (gr * way).sum())) <= 1e-7 * float((gr * way).abs().sum() + 1)


@pytest.mark.gpu
def test_backward_is_a_difference_of_the_kernel_itself():
    a, do, ds, scale = make("fp32", 70, 1, 2, 16, 16, state=True, seed=9)
    dev = {n: x.to(DEV) for n, x in a.items() if x is not None}
    leaves = [dev[n].requires_grad_() for n in ("q", "k", "v", "g", "state0")]
    do, ds = do.to(DEV), ds.to(DEV)
    grads = torch.autograd.grad(ops.linear_attention(**dev), leaves, [do, ds])
    with torch.no_grad():
        for i, (x, gr) in enumerate(zip(leaves, grads)):
            way = torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(DEV)
            h = 2.0 ** -6
            ends = []
            for sign in (1, -1):
                xs = [y + sign * h * way if j == i else y for j, y in enumerate(leaves)]
                o, s = ops.linear_attention(*xs)
                ends.append(((o * do).double().sum() + (s * ds).double().sum()).item())
            want = (gr * way).double().sum().item()
            # the difference of two sums of 70 * 32 + 512 terms of size 4, each right to 2^-17, over 2 h = 2^-5, and h^2 times a
            # third derivative that only g has: below |way|^3 / 6 of sums that fade within a few tokens
            assert abs((ends[0] - ends[1]) / (2 * h) - want) <= 0.02 * float((gr * way).abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dk,dv", [("bf16", 64, 64), ("fp32", 64, 100), ("fp16", 32, 20)])
def test_one_gradient_at_a_time(dtype, dk, dv):
    """Each leaf alone, and each output alone: other launches than all together, each within the bound of its own."""
    a, do, ds, scale = make(dtype, 300, 2, 4, dk, dv, Hq=2, Hv=1, state=True, ragged=True, seed=21)
    names = ("q", "k", "v", "g", "state0")
    do, ds = do.to(DEV), ds.to(DEV)

    def run(wanted, outs=(0, 1)):
        dev = {n: x.to(DEV) for n, x in a.items()}
        leaves = [dev[n].requires_grad_() for n in wanted]
        out = ops.linear_attention(**dev)
        return torch.autograd.grad([out[i] for i in outs], leaves, [(do, ds)[i] for i in outs], allow_unused=True)

    full = run(names)
    want = plain_grads(*[f64(a[n]) for n in names], a["lengths"], scale, f64(do), f64(ds))[2:]
    size = [f64(a[n]).abs() if n != "g" else f64(a[n]) for n in names]
    mag = plain_grads(*size, a["lengths"], scale, f64(do).abs(), f64(ds).abs())[2:]
    for n, x, y, m, all_of_them in zip(names, [run((n,))[0] for n in names], want, mag, full):
        if n == "g":                                       # its own bound is that of test_backward; here only the same sums differ
            assert (f64(x) - f64(all_of_them)).abs().max() <= DELTA[dtype] * m.max()
        else:
            bounded(x, y, m, x.dtype, DELTA[dtype])
    parts = [run(names, (i,)) for i in (0, 1)]
    assert parts[1][0] is None or not parts[1][0].any()    # the state does not depend on q
    for n, x, y, z, m in zip(names[1:], parts[0][1:], parts[1][1:], full[1:], mag[1:]):
        half = 2 * torch.finfo(z.dtype).eps * (f64(x).abs() + f64(y).abs())
        slack = 4 * DELTA[dtype] * (m if n != "g" else m.max())
        assert ((f64(x) + f64(y) - f64(z)).abs() <= half + slack).all(), n


@pytest.mark.gpu
def test_rows_behind_the_lengths_are_neither_read_nor_counted():
    a, do, ds, scale = make("bf16", 150, 4, 2, 64, 64, state=True, seed=3)
    a["lengths"] = torch.tensor([0, 1, 64, 150], dtype=torch.int64)
    want, wstate = check_forward(a, scale, "bf16")
    for b, n in enumerate(a["lengths"].tolist()):
        for x in ("q", "k", "v"):
            a[x][n:, b] = float("nan")
        a["g"][n:, b] = float("nan")
        do[n:, b] = float("inf")
    dev = {n: x.to(DEV) for n, x in a.items()}
    names = ("q", "k", "v", "g", "state0")
    leaves = [dev[n].requires_grad_() for n in names]
    o, s = ops.linear_attention(**dev)
    assert torch.equal(o, want) and torch.equal(s, wstate)
    grads = torch.autograd.grad([o, s], leaves, [do.to(DEV), ds.to(DEV)])
    for n, gr in zip(names, grads):
        assert torch.isfinite(gr).all(), n
        if n != "state0":
            for b, m in enumerate(a["lengths"].tolist()):
                assert not gr[m:, b].any(), n
    assert not o[1:, 1].any() and not o[:, 0].any()
    assert torch.equal(s[0], dev["state0"][0]) and torch.equal(grads[4][0].cpu(), ds[0])
    # lengths out of range count as the nearest that is in it
    dev["lengths"] = torch.tensor([-5, 1, 64, 4000], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        o2, s2 = ops.linear_attention(**dev)
    assert torch.equal(o2, want) and torch.equal(s2, wstate)


@pytest.mark.gpu
def test_a_reset_cuts_the_sequence_and_lowest_values_are_resets_too():
    a, do, ds, scale = make("fp32", 100, 2, 2, 40, 40, resets=(37,), state=True, seed=5)
    o, s = check_forward(a, scale, "fp32")
    low = {n: x.to(DEV) for n, x in a.items() if x is not None}
    low["g"] = low["g"].clone()
    low["g"][37] = torch.finfo(torch.float32).min
    with torch.no_grad():
        o2, s2 = ops.linear_attention(**low)
        assert torch.equal(o, o2) and torch.equal(s, s2)
        # the tokens from the reset on do not know what was before it
        again, state = ops.linear_attention(**{n: x[37:] for n, x in low.items() if n in ("q", "k", "v", "g")})
    mag = plain(*[f64(a[n][37:]).abs() if n != "g" else f64(a[n][37:]) for n in ("q", "k", "v", "g")], None, None, scale)
    bounded(again, f64(o2[37:]), 2 * mag[0], torch.float32, DELTA["fp32"])
    bounded(state, f64(s2), 2 * mag[1], torch.float32, DELTA["fp32"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("fp32", 100), ("fp16", 36), ("bf16", 33)])
def test_strides_give_the_same_bits(dtype, d):
    T, B, H = 70, 3, 4
    gen = torch.Generator().manual_seed(1)
    fused = torch.randn(T, B, 3 * H * d, generator=gen).to(DTYPES[dtype]).to(DEV)
    q, k, v = (x.view(T, B, H, d) for x in fused.split(H * d, -1))
    g = torch.nn.functional.logsigmoid(torch.randn(B, H, T, generator=gen)).to(DEV).permute(2, 0, 1)
    with torch.no_grad():
        want = ops.linear_attention(*(x.contiguous() for x in (q, k, v, g)))
        flipped = [x.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3) for x in (q, k, v)]
        shifted = []
        for x in (q, k, v):                                   # rows that start one element off
            room = torch.full((x.numel() + 1,), float("nan"), dtype=x.dtype, device=DEV)
            shifted.append(room[1:].view(x.shape).copy_(x))
        for other in ((q, k, v, g), (*flipped, g), (*shifted, g)):
            got = ops.linear_attention(*other)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        same = ops.linear_attention(q, k[:, :, :1].expand(T, B, H, d), v, g)
        shared = ops.linear_attention(q, k[:, :, :1], v, g)
        assert torch.equal(same[0], shared[0]) and torch.equal(same[1], shared[1])


@pytest.mark.gpu
def test_gradient_of_a_strided_and_of_an_expanded_output():
    a, do, ds, scale = make("fp32", 40, 2, 2, 24, 24, seed=6)
    dev = {n: x.to(DEV) for n, x in a.items() if x is not None}
    leaves = [dev[n].requires_grad_() for n in ("q", "k", "v", "g")]
    o, s = ops.linear_attention(**dev)
    want = torch.autograd.grad(o, leaves, torch.ones_like(o), retain_graph=True)
    got = torch.autograd.grad(o.sum(), leaves, retain_graph=True)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    w = do.to(DEV)
    want = torch.autograd.grad(o, leaves, w, retain_graph=True)
    got = torch.autograd.grad(o, leaves, w.permute(3, 1, 2, 0).contiguous().permute(3, 1, 2, 0), retain_graph=True)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    # the state alone, and one leaf alone
    want = torch.autograd.grad([o, s], leaves, [torch.zeros_like(o), ds.to(DEV)], retain_graph=True)
    got = torch.autograd.grad(s, leaves, ds.to(DEV), retain_graph=True)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    full = torch.autograd.grad([o, s], leaves, [w, ds.to(DEV)])
    for i, n in enumerate(("q", "k", "v", "g")):
        alone = {m: x.detach().requires_grad_(m == n) for m, x in dev.items()}
        out = ops.linear_attention(**alone)
        assert torch.equal(torch.autograd.grad(out, [alone[n]], [w, ds.to(DEV)])[0], full[i]), n


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows 2^24 + 8 elements apart: the last ones start behind 4 GiB (and behind 2^32 elements)."""
    T, H, d, gap = 260, 2, 64, (1 << 24) + 8
    gen = torch.Generator().manual_seed(2)
    small = [torch.randn(T, 1, H, d, generator=gen).bfloat16().to(DEV) for _ in range(3)]
    g = torch.nn.functional.logsigmoid(torch.randn(T, 1, H, generator=gen)).to(DEV)
    room = torch.empty((T - 1) * gap + 3 * H * d, dtype=torch.bfloat16, device=DEV)
    far = [torch.as_strided(room, (T, 1, H, d), (gap, H * d, d, 1), i * H * d) for i in range(3)]
    for x, y in zip(far, small):
        x.copy_(y)
    with torch.no_grad():
        want, got = ops.linear_attention(*small, g), ops.linear_attention(*far, g)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.gpu
def test_empty_sizes():
    for T, B in ((0, 2), (3, 0)):
        q, k, v = (torch.zeros(T, B, 2, 8, device=DEV, requires_grad=True) for _ in range(3))
        g = torch.zeros(2, device=DEV, requires_grad=True)
        s0 = torch.randn(B, 2, 8, 8, device=DEV, requires_grad=True)
        o, s = ops.linear_attention(q, k, v, g, s0)
        assert o.shape == (T, B, 2, 8) and torch.equal(s, s0)
        grads = torch.autograd.grad([o, s], [q, k, v, g, s0], [torch.ones_like(o), torch.ones_like(s)])
        assert not grads[3].any() and torch.equal(grads[4], torch.ones_like(s0))
    o = ops.linear_attention_step(*(torch.zeros(0, 2, 8, device=DEV) for _ in range(3)), torch.zeros(0, 2, device=DEV),
                                  torch.zeros(0, 2, 8, 8, device=DEV))
    assert o.shape == (0, 2, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,B,H,dk,dv,share", [("fp32", 1, 8, 125, 125, 1), ("bf16", 5, 4, 64, 64, 2), ("fp16", 40, 16, 128, 128, 1),
                                                   ("bf16", 3, 2, 1, 1, 1), ("fp32", 2, 3, 100, 36, 3), ("bf16", 300, 4, 16, 70, 1)])
def test_step(dtype, B, H, dk, dv, share):
    T = 6
    a, _, _, scale = make(dtype, T, B, H, dk, dv, Hq=H // share, Hv=H // share, state=True, resets=(3,), seed=dk)
    dev = {n: (x.to(DEV) if x is not None else None) for n, x in a.items()}
    room = torch.full((B, 2, H, dk, dv), 7.0, device=DEV)
    state = room[:, 1]                                       # every second state of a pool
    state.copy_(dev["state0"])
    outs = [ops.linear_attention_step(dev["q"][t], dev["k"][t], dev["v"][t], dev["g"][t], state) for t in range(T)]
    args = [f64(a[n]) for n in ("q", "k", "v", "g", "state0")]
    want = plain(*args, None, scale)
    mag = plain(*[x.abs() if i != 3 else x for i, x in enumerate(args)], None, scale)
    bounded(torch.stack(outs), want[0], mag[0], DTYPES[dtype], 2.0 ** -16)     # fp32 throughout: T decays and dk additions
    bounded(state, want[1], mag[1], torch.float32, 2.0 ** -16)
    assert (room[:, 0] == 7.0).all()
    fixed = ops.linear_attention_step(dev["q"][0], dev["k"][0], dev["v"][0], dev["g"][0, 0], state.clone())
    spread = ops.linear_attention_step(dev["q"][0], dev["k"][0], dev["v"][0], dev["g"][0, :1].expand(B, H), state.clone())
    assert torch.equal(fixed, spread)


@pytest.mark.gpu
def test_prompt_then_tokens_is_the_whole_sequence():
    a, _, _, scale = make("bf16", 90, 2, 4, 64, 64, Hk=2, seed=8)
    dev = {n: x.to(DEV) for n, x in a.items() if x is not None}
    with torch.no_grad():
        o, state = ops.linear_attention(**{n: x[:80] for n, x in dev.items()})
        late = [ops.linear_attention_step(*(dev[n][t] for n in ("q", "k", "v", "g")), state) for t in range(80, 90)]
    args = [f64(a[n]) for n in ("q", "k", "v", "g")]
    want, mag = plain(*args, None, None, scale), plain(*[x.abs() if i != 3 else x for i, x in enumerate(args)], None, None, scale)
    bounded(torch.cat([o, torch.stack(late)]), want[0], mag[0], torch.bfloat16, DELTA["bf16"])
    bounded(state, want[1], mag[1], torch.float32, DELTA["bf16"])


@pytest.mark.gpu
def test_other_streams_and_repeats_give_the_same_bits():
    a, do, ds, scale = make("bf16", 700, 1, 2, 64, 64, state=True, seed=10)
    dev = {n: x.to(DEV) for n, x in a.items() if x is not None}
    leaves = [dev[n].requires_grad_() for n in ("q", "k", "v", "g", "state0")]
    do, ds = do.to(DEV), ds.to(DEV)
    run = lambda: [*(out := ops.linear_attention(**dev)), *torch.autograd.grad(out, leaves, [do, ds])]  # noqa: E731
    want = run()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:                                           # two at once, each with its own workspace
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in side:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(x, y) for x, y in zip(r, want))


@pytest.mark.gpu
def test_capture_and_replay():
    """Forward with its gradients, and single tokens, captured and replayed three times between eager work."""
    a, do, ds, scale = make("bf16", 300, 1, 4, 64, 64, Hk=2, state=True, ragged=True, seed=11)
    dev = {n: x.to(DEV) for n, x in a.items()}
    names = ("q", "k", "v", "g", "state0")
    do, ds = do.to(DEV), ds.to(DEV)
    stat = {n: x.clone() for n, x in dev.items()}

    def run(d):
        d = {n: (x.detach().requires_grad_() if n in names else x) for n, x in d.items()}
        out = ops.linear_attention(**d)
        return [x.detach() for x in out] + list(torch.autograd.grad(out, [d[n] for n in names], [do, ds]))

    def token(d, state):
        with torch.no_grad():
            return ops.linear_attention_step(d["q"][0], d["k"][0], d["v"][0], d["g"][0], state)

    pool = stat["state0"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(stat)
        token(stat, pool)
    torch.cuda.current_stream().wait_stream(side)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        outs = run(stat)
    with torch.cuda.graph(second):
        o1 = token(stat, pool)
    for i in range(3):
        gen = torch.Generator().manual_seed(100 + i)
        for n in ("q", "k", "v"):
            stat[n].copy_(torch.randn(stat[n].shape, generator=gen).to(stat[n].dtype))
        pool.copy_(stat["state0"])
        want = run({n: x.clone() for n, x in stat.items()})
        eager = stat["state0"].clone()
        wtok = token(stat, eager)
        torch.cuda.synchronize()
        first.replay()
        second.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want)), i
        assert torch.equal(o1, wtok) and torch.equal(pool, eager)


@pytest.mark.gpu
def test_step_marks_its_state_as_changed():
    a, do, ds, _ = make("fp32", 4, 1, 1, 8, 8, state=True, seed=12)
    dev = {n: x.to(DEV) for n, x in a.items() if x is not None}
    q = dev["q"].requires_grad_()
    o, s = ops.linear_attention(q, dev["k"], dev["v"], dev["g"], dev["state0"])
    with torch.no_grad():
        ops.linear_attention_step(q[0], dev["k"][0], dev["v"][0], dev["g"][0], dev["state0"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o.sum(), q)


# ------------------------------------------------------------------------------------ refusals
def test_entry_points_refuse_bad_arguments_without_a_gpu():
    lib = _lib.load()
    ok = [0, 4, 1, 2, 2, 2, 2, 8, 8]                          # dtype, T, B, H, Hq, Hk, Hv, dk, dv
    size = lambda *a: int(lib.dmn_linear_attention_workspace_floats(a[0], 0, *a[1:]))  # noqa: E731
    assert size(*ok) == 0
    assert int(lib.dmn_linear_attention_workspace_floats(ok[0], 1, *ok[1:])) > 0
    for at, value, word in ((0, 3, b"dtype"), (1, -1, b"bad sizes"), (2, -1, b"bad sizes"), (3, 0, b"bad sizes"), (4, 3, b"multiple"),
                            (7, 0, b"widths"), (7, 129, b"widths"), (8, 200, b"widths"), (2, 1 << 17, b"2^17"), (1, (1 << 29) + 1, b"2^29")):
        bad = list(ok)
        bad[at] = value
        assert size(*bad) == -1 and word in lib.dmn_last_error(), (at, value)
    assert size(0, 1 << 20, 1 << 12, 1, 1, 1, 1, 8, 8) == -1 and b"2^32" in lib.dmn_last_error()
    strides = ops._strides([16, 16, 8] * 5)
    for args, word in (((1, 1, 1, 1, None, None, 0, None, None, strides, None), "null pointer"),
                       ((1, 1, 1, 1, None, None, 0, 1, None, None, None), "null pointer"),
                       ((None, 1, 1, 1, None, None, 0, 1, None, strides, None), "null pointer")):
        with pytest.raises(RuntimeError, match=word):
            _lib.call("dmn_linear_attention_fwd", 0, *args, *ok[1:], 1.0, None)
    long = [0, 4096, 1, 2, 2, 2, 2, 8, 8]
    assert size(*long) > 0
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.call("dmn_linear_attention_fwd", 0, 16, 16, 16, 16, None, None, 0, 16, None, strides, None, *long[1:], 1.0, None)
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.call("dmn_linear_attention_bwd", 0, 16, 16, 16, 16, None, None, 0, 16, None, 16, 16, 16, None, 0, None, strides, 8, *ok[1:], 1.0, None)
    for at, value in ((0, (1 << 24) + (1 << 20) + 1), (3, -8), (6, 1 << 40)):
        far = [16, 16, 8] * 5
        far[at] = value
        with pytest.raises(RuntimeError, match="stride"):
            _lib.call("dmn_linear_attention_fwd", 0, 16, 16, 16, 16, None, None, 0, 16, None, ops._strides(far), None, *ok[1:], 1.0, None)
    with pytest.raises(RuntimeError, match="null pointer"):
        _lib.call("dmn_linear_attention_step", 0, 16, 16, 16, 16, None, 16, strides, 1, 2, 2, 2, 2, 8, 8, 1.0, None)


def test_cpu_tensors_are_refused():
    x, g = torch.zeros(3, 1, 2, 8), torch.zeros(3, 1, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_attention(x, x, x, g)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_attention_step(x[0], x[0], x[0], g[0], torch.zeros(1, 2, 8, 8))


@pytest.mark.gpu
def test_refusals():
    x, g = torch.zeros(3, 1, 2, 8, device=DEV), torch.zeros(3, 1, 2, device=DEV)
    s = torch.zeros(1, 2, 8, 8, device=DEV)
    call = ops.linear_attention
    for bad, word in (
            (lambda: call(x.double(), x, x, g), "float32, bfloat16 or float16"),
            (lambda: call(x, x.bfloat16(), x, g), "expected torch.float32 for k"),
            (lambda: call(x, x, x, g.bfloat16()), "g must be float32"),
            (lambda: call(x, x, x, g[:2]), "g must be float32"),
            (lambda: call(x, x, x, g[:, :, :1].expand(3, 1, 3)), "multiple"),
            (lambda: call(x, x[:2], x, g), "expected shape"),
            (lambda: call(x, x[..., :4], x, g), "expected shape"),
            (lambda: call(x[..., ::2], x[..., :4], x, g), "unit stride"),
            (lambda: call(x, x, x[0], g), "axes"),
            (lambda: call(x[0], x[0], x[0], g), "q must be"),
            (lambda: call(torch.zeros(3, 1, 2, 129, device=DEV), torch.zeros(3, 1, 2, 129, device=DEV), x, g), "widths"),
            (lambda: call(x, x, x, g, s[:, :1]), "expected shape"),
            (lambda: call(x, x, x, g, s.transpose(2, 3)), "contiguous"),
            (lambda: call(x, x, x, g, s.bfloat16()), "expected float32"),
            (lambda: call(x, x, x, g, lengths=torch.zeros(2, dtype=torch.int32, device=DEV)), "lengths"),
            (lambda: call(x, x, x, g, lengths=torch.zeros(1, device=DEV)), "lengths"),
            (lambda: call(x, x, x, g, lengths=[3]), "lengths"),
            (lambda: call(x, x, x, g, lengths=torch.zeros(1, dtype=torch.int32)), "lengths"),
            (lambda: call(x, x.cpu(), x, g), "no CPU fallback"),
            (lambda: ops.linear_attention_step(x[0], x[0], x[0], g[0], s.transpose(2, 3)), "contiguous"),
            (lambda: ops.linear_attention_step(x[0], x[0], x[0], g[0], s.bfloat16()), "float32"),
            (lambda: ops.linear_attention_step(x[0], x[0], x[0], g[0], s[:, :1]), "expected shape"),
            (lambda: ops.linear_attention_step(x[0].requires_grad_(), x[0], x[0], g[0], s), "inference only")):
        with pytest.raises(RuntimeError, match=word):
            bad()
