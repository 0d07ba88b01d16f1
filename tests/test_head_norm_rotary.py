"""RMS norm and multi-axis rotation of query and key heads (ops.head_norm_rotary) against the formulas in 64 bits.

Bounds, for rows of at most 256 elements.  1/rms: the squares' sum passes at most E - 1 + 6 additions (E = 8 elements a lane,
then 6 exchanges) and its root halves the error: below 8 steps of 2^-24 with the root itself (1 ulp).  Two products more.  The
angle in turns is rounded to fp32 at most 1/2 from 0: 2^-26 turns, 2^-23.3 radians; sine and cosine are right to 2 ulp, 2^-22.
An output is the sum of two products: |error| <= 2^-20 (|a| + |b|) + eps/2 |y|, a and b the normalised pair.  Positions reach
2^24, where the 64-bit angle itself is right to 2^-28.  A gradient of x joins two such sums and a mean over the row: 2^-18 of
the sum of the absolute values.  A weight's gradient adds at most 128 rows in one chain: 2^-17 more, 2^-16.
"""
import math

import pytest
import torch

from dms_amd import _lib, ops

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def angles(pos, sections, pairs, base):
    """(T, B, 1, pairs) float64 angles from (T, B, axes) positions."""
    out = torch.zeros(pos.shape[:2] + (1, pairs), dtype=torch.float64)
    at = 0
    for axis, n in enumerate(sections):
        for j in range(n):
            out[:, :, 0, at] = pos[..., axis].double() * base ** (-j / n)
            at += 1
    return out


def turned(x, angle, sign=1, absolute=False):
    D = x.shape[-1]
    z = torch.nn.functional.pad(x, (0, D % 2)).unflatten(-1, (-1, 2))
    co, si = angle.cos(), sign * angle.sin()
    a, b = z[..., 0], z[..., 1]
    if absolute:
        turns = (angle != 0).double()
        y = torch.stack([a + b * turns, b + a * turns], -1)
    else:
        y = torch.stack([a * co - b * si, a * si + b * co], -1)
    return y.flatten(-2)[..., :D]


def plain(x, w, angle, eps, dy=None):
    """y and its magnitude; with dy also dx, dw and theirs."""
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    out = [turned(x * r * w, angle), turned((x * r * w).abs(), angle, absolute=True)]
    if dy is not None:
        u, um = turned(dy, angle, -1), turned(dy.abs(), angle, absolute=True)
        n = x * r
        out += [r * (u * w - n * (n * u * w).mean(-1, keepdim=True)),
                r * (um * w.abs() + n.abs() * (n.abs() * um * w.abs()).mean(-1, keepdim=True)),
                (u * n).sum((0, 1, 2)), (um * n.abs()).sum((0, 1, 2))]
    return out


def make(dtype, T, B, Hq, Hk, D, axes, weights, seed=0, far=1 << 24):
    gen = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    row = lambda h: (torch.randn(T, B, h, D, generator=gen) * torch.rand(T, B, h, 1, generator=gen)).to(dt)  # noqa: E731
    q, k, dq, dk = row(Hq), row(Hk), row(Hq), row(Hk)
    wt = {"fp32": torch.float32, "same": dt}.get(weights)
    w = [None if wt is None else (1 + 0.3 * torch.randn(D, generator=gen)).to(wt) for _ in range(2)]
    pos = torch.randint(-far, far, (T, B, axes), generator=gen)
    return q, k, w[0], w[1], pos, dq, dk


def bounded(got, want, mag, delta):
    got = got.detach().cpu()
    half, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).tiny
    assert got.shape == want.shape and torch.isfinite(got).all()
    over = (got.double() - want).abs() - (delta * mag + half * want.abs() + tiny)
    assert float(over.max()) <= 0.0, "off by %g beyond its bound" % float(over.max())


CASES = [
    # dtype, T, B, Hq, Hk, D, sections, weights
    ("fp32", 1, 1, 1, 1, 1, (), None),
    ("fp32", 20, 1, 8, 8, 125, (62,), "fp32"),
    ("bf16", 7, 3, 4, 2, 64, (8, 12, 12), "fp32"),
    ("bf16", 33, 2, 16, 4, 128, (16, 24, 24), "same"),
    ("fp16", 5, 2, 3, 1, 100, (10, 20, 20), "same"),
    ("fp32", 40, 2, 10, 2, 100, (10, 20, 20), "fp32"),
    ("bf16", 9, 1, 2, 2, 33, (3, 0, 5, 8), "fp32"),
    ("fp16", 3, 2, 2, 6, 256, (100,), None),
    ("fp32", 4, 1, 1, 3, 256, (64, 64), "fp32"),
    ("bf16", 3, 2, 2, 2, 2, (1,), "same"),
    ("fp32", 300, 1, 1, 1, 7, (1, 2), "fp32"),
    ("bf16", 11, 2, 3, 2, 36, (2, 2), "fp32"),
]


def _id(c):
    return "%s-T%d-B%d-H%d.%d-D%d-%s-%s" % (c[:6] + ("x".join(map(str, c[6])) or "none", c[7]))


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_forward_and_backward(case):
    dtype, T, B, Hq, Hk, D, sections, weights = case
    q, k, wq, wk, pos, dq, dk = make(dtype, T, B, Hq, Hk, D, len(sections), weights, seed=D)
    dev = [None if x is None else x.to(DEV).requires_grad_() for x in (q, k, wq, wk)]
    p = pos.to(DEV)
    with torch.no_grad():
        y = ops.head_norm_rotary(*dev, p, sections, base=500.0, eps=1e-5)
    z = ops.head_norm_rotary(*dev, p, sections, base=500.0, eps=1e-5)
    assert torch.equal(y[0], z[0]) and torch.equal(y[1], z[1])
    leaves = [x for x in dev if x is not None]
    grads = list(torch.autograd.grad(z, leaves, [dq.to(DEV), dk.to(DEV)]))
    again = torch.autograd.grad(ops.head_norm_rotary(*dev, p, sections, base=500.0, eps=1e-5), leaves, [dq.to(DEV), dk.to(DEV)])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    angle = angles(pos, sections, (D + 1) // 2, 500.0)
    for m, (x, w, d) in enumerate(((q, wq, dq), (k, wk, dk))):
        ww = torch.ones(D, dtype=torch.float64) if w is None else w.double()
        want = plain(x.double(), ww, angle, 1e-5, d.double())
        assert y[m].dtype == x.dtype and y[m].is_contiguous()
        bounded(y[m], want[0], want[1], 2.0 ** -20)
        bounded(grads[m], want[2], want[3], 2.0 ** -18)
        if w is not None:
            assert grads[2 + m].dtype == w.dtype
            bounded(grads[2 + m], want[4], want[5], 2.0 ** -16)


def test_plain_gradients_are_differences():
    q, _, wq, _, pos, dq, _ = make("fp32", 3, 2, 2, 1, 9, 2, "fp32", seed=1, far=50)
    angle = angles(pos, (2, 1), 5, 100.0)
    x, w, d = q.double(), wq.double(), dq.double()
    _, _, dx, _, dw, _ = plain(x, w, angle, 1e-6, d)
    gen = torch.Generator().manual_seed(0)
    for arg, gr in ((0, dx), (1, dw)):
        way = torch.randn(gr.shape, dtype=torch.float64, generator=gen)
        ends = []
        for h in (1e-6, -1e-6):
            xs = [x, w]
            xs[arg] = xs[arg] + h * way
            ends.append(float((plain(*xs, angle, 1e-6)[0] * d).sum()))
        assert abs((ends[0] - ends[1]) / 2e-6 - float((gr * way).sum())) <= 1e-6 * float((gr * way).abs().sum() + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("fp32", 100), ("fp16", 36), ("bf16", 33)])
def test_strides_and_position_forms_give_the_same_bits(dtype, D):
    T, B, Hq, Hk = 12, 3, 4, 2
    gen = torch.Generator().manual_seed(2)
    fused = torch.randn(T, B, (Hq + Hk) * D, generator=gen).to(DTYPES[dtype]).to(DEV)
    q, k = fused[..., :Hq * D].view(T, B, Hq, D), fused[..., Hq * D:].view(T, B, Hk, D)
    pos = ops.map_positions(2, 2, 3, DEV)
    assert pos.tolist()[:4] == [[0, 0, 0], [1, 0, 0], [2, 0, 0], [0, 0, 1]] and pos.tolist()[-1] == [2, 1, 1]
    sec = (D // 2 - 8, 4, 4)
    with torch.no_grad():
        want = ops.head_norm_rotary(q.contiguous(), k.contiguous(), None, None, pos, sec)
        batch_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k)]
        shifted = []
        for x in (q, k):
            room = torch.full((x.numel() + 1,), float("nan"), dtype=x.dtype, device=DEV)
            shifted.append(room[1:].view(x.shape).copy_(x))
        wide = pos.long().unsqueeze(1).expand(T, B, 3)
        for a, p in (((q, k), pos), (batch_first, wide), (shifted, wide.contiguous()), ((q, k), pos.t().contiguous().t())):
            got = ops.head_norm_rotary(*a, None, None, p, sec)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    dy = [torch.randn(x.shape, generator=gen).to(x.dtype).to(DEV) for x in (q, k)]
    leaves = [x.detach().requires_grad_() for x in (q.contiguous(), k.contiguous())]
    y = ops.head_norm_rotary(*leaves, None, None, pos, sec)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    got = torch.autograd.grad(y, leaves, [d.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0) for d in dy], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = torch.autograd.grad(y, leaves, [d[:1].expand_as(d) for d in dy], retain_graph=True)
    want = torch.autograd.grad(y, leaves, [d[:1].expand_as(d).contiguous() for d in dy], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(torch.autograd.grad(y[0], leaves[0], dy[0])[0], torch.autograd.grad(
        ops.head_norm_rotary(*leaves, None, None, pos, sec), leaves, dy)[0])


@pytest.mark.gpu
def test_empty_rows_far_positions_and_spoilt_rows():
    q, k, wq, wk, pos, dq, dk = make("fp32", 6, 2, 2, 2, 64, 2, "fp32", seed=5, far=1 << 31)
    q[1], q[2, 0, 0, 5], k[3, 1, 1, 7] = 0.0, float("nan"), float("inf")
    dev = [x.to(DEV).requires_grad_() for x in (q, k, wq, wk)]
    y = ops.head_norm_rotary(*dev, pos.to(DEV), (20, 12))
    gq, gk = torch.autograd.grad(y, dev[:2], [dq.to(DEV), dk.to(DEV)])
    angle = angles(pos, (20, 12), 32, 10000.0)
    want = plain(q.double(), wq.double(), angle, 1e-6, dq.double())
    good = torch.ones(6, 2, 2, dtype=torch.bool)
    good[2, 0, 0] = False
    assert not y[0][1].any() and torch.isnan(y[0][2, 0, 0]).all()
    # at 2^31 both sides' angles are right to 2^-21 only
    bounded(y[0].cpu()[good], want[0][good], want[1][good], 2.0 ** -19)
    bounded(gq.cpu()[good], want[2][good], want[3][good], 2.0 ** -17)
    other = torch.ones(6, 2, 2, dtype=torch.bool)
    other[3, 1, 1] = False
    assert torch.isfinite(y[1].cpu()[other]).all() and torch.isfinite(gk.cpu()[other]).all()


@pytest.mark.gpu
def test_empty_sizes():
    for T, B in ((0, 2), (3, 0)):
        q = torch.zeros(T, B, 2, 8, device=DEV, requires_grad=True)
        w = torch.ones(8, device=DEV, requires_grad=True)
        y = ops.head_norm_rotary(q, q, w, w, torch.zeros(T, B, 1, dtype=torch.int64, device=DEV), (4,))
        assert y[0].shape == q.shape
        gq, gw = torch.autograd.grad(y, [q, w], [torch.ones_like(t) for t in y])
        assert gq.shape == q.shape and not gw.any()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    T, H, D, gap = 260, 2, 64, (1 << 24) + 8
    gen = torch.Generator().manual_seed(2)
    small = [torch.randn(T, 1, H, D, generator=gen).bfloat16().to(DEV) for _ in range(2)]
    room = torch.empty((T - 1) * gap + 2 * H * D, dtype=torch.bfloat16, device=DEV)
    far = [torch.as_strided(room, (T, 1, H, D), (gap, H * D, D, 1), i * H * D) for i in range(2)]
    for x, y in zip(far, small):
        x.copy_(y)
    pos = torch.arange(T, device=DEV).view(T, 1)
    with torch.no_grad():
        want, got = (ops.head_norm_rotary(*x, None, None, pos, (32,)) for x in (small, far))
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.gpu
def test_capture_and_replay_and_another_stream():
    q, k, wq, wk, pos, dq, dk = (x.to(DEV) for x in make("bf16", 50, 2, 4, 2, 64, 3, "fp32", seed=6))

    def run():
        leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk)]
        y = ops.head_norm_rotary(*leaves, pos, (8, 12, 12))
        return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, [dq, dk]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


# ------------------------------------------------------------------------------------ refusals
def test_entry_points_refuse_bad_arguments_without_a_gpu():
    import ctypes
    lib = _lib.load()
    st = ops._strides([64, 64, 8] * 5)
    sec = lambda *n: (ctypes.c_int * max(len(n), 1))(*n)  # noqa: E731

    rates = (ctypes.c_double * 2)(1.0, 0.5)

    def fwd(dtype=0, q=16, sections=(2,), rates=rates, T=1, B=1, Hq=1, Hk=1, D=8, pos=16, strides=st):
        _lib.call("dmn_head_norm_rotary_fwd", dtype, q, 16, None, None, 1, pos, 1, sec(*sections), len(sections), rates, 1e-6, 16, 16,
                  strides, T, B, Hq, Hk, D, None)

    for bad, word in ((dict(dtype=3), "dtype"), (dict(T=-1), "bad sizes"), (dict(Hq=0), "bad sizes"), (dict(D=0), "widths"),
                      (dict(D=257), "widths"), (dict(sections=(3, 2)), "pairs turn"), (dict(sections=(-1, 2)), "bad section"),
                      (dict(sections=(0,) * 5), "axes"), (dict(rates=None), "null"), (dict(q=None), "null"),
                      (dict(pos=None), "null"), (dict(strides=None), "null")):
        with pytest.raises(RuntimeError, match=word):
            fwd(**bad)
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.call("dmn_head_norm_rotary_bwd", 0, 16, 16, 16, 16, 1, 16, 1, sec(2), 1, rates, 1e-6, 16, 16, 16, 16, 16, 16, st, None,
                  1, 1, 1, 1, 8, None)
    assert lib.dmn_head_norm_rotary_workspace_floats(0, 1, 8) == -1 and lib.dmn_head_norm_rotary_workspace_floats(4, 1, 64) > 0
    x = torch.zeros(2, 1, 1, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.head_norm_rotary(x, x, None, None, None, ())


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros(3, 2, 2, 8, device=DEV)
    p = torch.zeros(3, 2, 1, dtype=torch.int64, device=DEV)
    w = torch.ones(8, device=DEV)
    call = ops.head_norm_rotary
    for bad, word in (
            (lambda: call(x.double(), x, w, w, p, (4,)), "float32, bfloat16 or float16"),
            (lambda: call(x, x.half(), w, w, p, (4,)), "expected torch.float32 for k"),
            (lambda: call(x, x[..., :4], w, w, p, (2,)), "expected shape"),
            (lambda: call(x, x[:2], w, w, p, (2,)), "expected shape"),
            (lambda: call(x[..., ::2], x[..., ::2], None, None, p, (2,)), "unit stride"),
            (lambda: call(x, x[0], w, w, p, (4,)), "4 axes"),
            (lambda: call(x, x, w[:4], w, p, (4,)), "expected shape"),
            (lambda: call(x, x, w.double(), w, p, (4,)), "q_weight must be"),
            (lambda: call(x.half(), x.half(), w.half(), w, p, (4,)), "same type"),
            (lambda: call(x, x, w, w, p, (5,)), "sections"),
            (lambda: call(x, x, w, w, p, (2, 2)), "positions must be"),
            (lambda: call(x, x, w, w, p.float(), (4,)), "positions must be"),
            (lambda: call(x, x, w, w, p.cpu(), (4,)), "positions must be"),
            (lambda: call(x, x, w, w, None, (4,)), "positions must be"),
            (lambda: call(x, x, w, w, p, (4,), base=0.0), "base"),
            (lambda: call(x, x, w, w, p, (4,), base=math.nan), "base"),
            (lambda: call(x[:, :, :0], x, w, w, p, (4,)), "at least one head"),
            (lambda: call(torch.zeros(1, 1, 1, 300, device=DEV), torch.zeros(1, 1, 1, 300, device=DEV), None, None, None, ()), "width")):
        with pytest.raises(RuntimeError, match=word):
            bad()
