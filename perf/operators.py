# -*- coding: utf-8 -*-
"""Measured cases of the linear-attention operators, with their plain forms.

Three operators, each through ``dms_amd.ops``:

* ``attention``: ``linear_attention`` -- S_t = exp(g_t) S_{t-1} + k_t^T v_t, o_t = scale * q_t S_t -- at inference, and
  with ``train`` its backward too;
* ``step``: ``linear_attention_step``, one token of the same recurrence with the state updated in place;
* ``rotary``: ``head_norm_rotary``, the RMS norm of every query and key head and its rotation by positions on several
  axes in one pass, at inference and with ``train`` its backward too.

``run`` with ``own`` false computes the same thing with elementary torch operations in 32 bits (angles and sums of
log decays in 64): the recurrence in its chunked form, with the states between chunks from one masked product.
``exact`` computes it token by token in 64 bits.
"""
import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
BASE = 10000.0
EPS = 1e-6
CHUNK = 64


def listed():
    return [
        # the query's words through a 1000-wide language encoder of 8 heads: one sample, latency only
        attention("words of one query", "fp32", T=20, B=1, H=8, dk=125, dv=125),
        # the (pixel, word) sequence of one 512 px image, 16 * 16 * 20 tokens: few heads, a long axis
        attention("512 px map, one sample", "bf16", T=5120, B=1, H=16, dk=64, dv=64),
        # the same for a batch of 32: the largest call, bound by memory
        attention("512 px map, batch", "bf16", T=5120, B=32, H=16, dk=64, dv=64),
        # 320 px maps of different lengths that go on from a state, 1000 = 10 heads of 100, in full precision
        attention("320 px maps, ragged", "fp32", T=2000, B=16, H=10, dk=100, dv=100, ragged=True, state=True),
        # a training step's mixer at 320 px and batch 64
        attention("training, 320 px map", "bf16", T=2000, B=64, H=16, dk=64, dv=64, train=True),
        # a training step's language encoder: short sequences, one learnt decay for each head
        attention("training, words", "fp32", T=20, B=64, H=8, dk=125, dv=125, train=True, fixed=True),
        # packed sequences with resets between them, queries and keys shared by two value heads, a state carried over
        attention("training, packed, shared heads", "fp32", T=1999, B=4, H=8, Hq=4, Hk=4, dk=64, dv=128, train=True, resets=9,
                  state=True),
        # one token of one stream: latency only
        step("token, one stream", "fp32", B=1, H=8, dk=125, dv=125),
        # one token of 256 streams: bound by the states' memory
        step("token, 256 streams", "bf16", B=256, H=16, dk=128, dv=128),
        # the words of one query
        rotary("rotation, words of one query", "fp32", T=20, B=1, Hq=8, Hk=8, D=125, sections="62"),
        # queries and keys of a batch of 512 px maps: word, row and column positions
        rotary("rotation, 512 px map, batch", "bf16", T=5120, B=32, Hq=16, Hk=16, D=64, sections="8,12,12"),
        # the same in a training step at 320 px, keys shared, heads of 100
        rotary("rotation, training, 320 px map", "fp32", T=2000, B=64, Hq=10, Hk=2, D=100, sections="10,20,20", train=True),
    ]


def attention(name, dtype, T, B, H, dk, dv, Hq=None, Hk=None, Hv=None, train=False, fixed=False, ragged=False, state=False, resets=0):
    return dict(name=name, op="attention", dtype=dtype, T=T, B=B, H=H, Hq=Hq or H, Hk=Hk or H, Hv=Hv or H, dk=dk, dv=dv, train=train,
                fixed=fixed, ragged=ragged, state=state, resets=resets)


def step(name, dtype, B, H, dk, dv):
    return dict(name=name, op="step", dtype=dtype, B=B, H=H, dk=dk, dv=dv)


def rotary(name, dtype, T, B, Hq, Hk, D, sections, train=False):
    return dict(name=name, op="rotary", dtype=dtype, T=T, B=B, Hq=Hq, Hk=Hk, D=D, sections=sections, train=train)


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention train", "step", "rotary", "rotary train"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    train = op.endswith("train")
    H = rng.choice([1, 2, 4, 6, 8, 10, 16])
    width = lambda: rng.choice([16, 32, 64, 64, 128, rng.randint(9, 128)])  # noqa: E731
    if op == "step":
        c = step("", dtype, _log_int(rng, 1, 256), H, width(), width())
    elif op.startswith("rotary"):
        T, B, D = _log_int(rng, 1, 5120), _log_int(rng, 1, 64), width()
        while B * T * H * D > 64 * 2000 * 10 * 100:
            B = (B + 1) // 2
        axes = rng.randint(1, 3)
        n = [max(1, D // 2 // axes - rng.randint(0, 1)) for _ in range(axes)]
        Hk = rng.choice([h for h in (1, 2, 4, 5, 8, 16) if H % h == 0])
        c = rotary("", dtype, T, B, H, Hk, D, ",".join(map(str, n)), train)
    else:
        T, B = _log_int(rng, 1, 5120), _log_int(rng, 1, 64)
        dk, dv = width(), width()
        while B * T * H * max(dk + dv, dk * dv // 32) > (2 if not train else 1) * 64 * 2000 * 16 * 64:
            B = (B + 1) // 2
        share = [rng.choice([H, H, H, 1, max(1, H // 2)]) for _ in range(3)]
        share = [h if H % h == 0 else H for h in share]
        c = attention("", dtype, T, B, H, dk, dv, share[0], share[1], share[2], train, rng.random() < 0.25, rng.random() < 0.4,
                      rng.random() < 0.5, rng.choice([0, 0, 3]))
    del c["name"]
    return c


def work(case):
    c, es = case, SIZE[case["dtype"]]
    if c["op"] == "rotary":
        n = c["T"] * c["B"] * (c["Hq"] + c["Hk"]) * c["D"]
        weights = (4 if c["train"] else 2) * c["D"] * 4
        return {"bytes": n * es * (4 if c["train"] else 2) + c["T"] * c["B"] * len(c["sections"].split(",")) * 8 + weights,
                "flops": n * (22 if c["train"] else 7)}
    state = c["B"] * c["H"] * c["dk"] * c["dv"] * 4
    if c["op"] == "step":
        n = c["B"] * c["H"] * (2 * c["dk"] + 2 * c["dv"])
        return {"bytes": n * es + c["B"] * c["H"] * 4 + 2 * state, "flops": 5 * state // 4}
    rows = c["T"] * c["B"]
    once = rows * (c["Hq"] * c["dk"] + c["Hk"] * c["dk"] + c["Hv"] * c["dv"]) * es      # q, k, v, and again their gradients
    out = rows * c["H"] * c["dv"] * es
    decay = 4 * (c["H"] if c["fixed"] else rows * c["H"])
    flops = 4 * rows * c["H"] * c["dk"] * c["dv"]
    if not c["train"]:
        return {"bytes": once + out + decay + state * (2 if c["state"] else 1), "flops": flops}
    return {"bytes": 2 * once + 2 * out + 2 * decay + state * (4 if c["state"] else 1), "flops": 4 * flops}


# ------------------------------------------------------------------------------------------ inputs

def _rows(gen, shape, dtype):
    """Activations as a projection leaves them: normal, every row at a scale of its own."""
    x = torch.randn(shape, generator=gen, device=DEV)
    return (x * (0.6 + 0.8 * torch.rand(shape[:-1] + (1,), generator=gen, device=DEV))).to(dtype)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    B = c["B"]
    if c["op"] == "rotary":
        sections = tuple(int(n) for n in c["sections"].split(","))
        T, D = c["T"], c["D"]
        n = torch.arange(T, device=DEV)
        s = dict(case=c, q=_rows(gen, (T, B, c["Hq"], D), dt), k=_rows(gen, (T, B, c["Hk"], D), dt),
                 wq=1 + 0.1 * torch.randn(D, generator=gen, device=DEV), wk=1 + 0.1 * torch.randn(D, generator=gen, device=DEV),
                 sections=sections,
                 # word, row and column of the (pixel, word) sequence, every sample somewhere in a long stream: many digits
                 pos=torch.stack([n % 20, n // 320, n // 20 % 16][:len(sections)], -1).unsqueeze(1)
                 + torch.randint(0, 1 << 20, (1, B, len(sections)), generator=gen, device=DEV))
        if c["train"]:
            s["dq"], s["dk"] = _rows(gen, s["q"].shape, dt), _rows(gen, s["k"].shape, dt)
        return s
    H, dk, dv = c["H"], c["dk"], c["dv"]
    gate = lambda *shape: F.logsigmoid(2 + 2 * torch.randn(shape, generator=gen, device=DEV)) / 4  # noqa: E731
    state = lambda: torch.randn((B, H, dk, dv), generator=gen, device=DEV)  # noqa: E731
    if c["op"] == "step":
        return dict(case=c, q=_rows(gen, (B, H, dk), dt), k=_rows(gen, (B, H, dk), dt), v=_rows(gen, (B, H, dv), dt), g=gate(B, H),
                    state=state())
    T = c["T"]
    s = dict(case=c, q=_rows(gen, (T, B, c["Hq"], dk), dt), k=_rows(gen, (T, B, c["Hk"], dk), dt), v=_rows(gen, (T, B, c["Hv"], dv), dt),
             g=gate(H) / 8 if c["fixed"] else gate(T, B, H), state=state() if c["state"] else None, lengths=None)
    if c["ragged"]:
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
    if c["resets"] and not c["fixed"]:
        at = torch.randint(0, T, (c["resets"],), generator=gen, device=DEV)
        s["g"][at] = -math.inf
    if c["train"]:
        s["do"], s["ds"] = _rows(gen, (T, B, H, dv), dt), state() / 8
        for name in ("q", "k", "v", "g", "state"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------ the passes

def run(s):
    if own:
        return _own(s)
    c = s["case"]
    if c["op"] == "rotary":
        return _plain_rotary_train(s) if c["train"] else _plain_rotary(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["sections"])
    if c["op"] == "step":
        return _plain_step(s)
    if not c["train"]:
        with torch.no_grad():
            return _plain_attention(s["q"], s["k"], s["v"], s["g"], s["state"], s["lengths"])
    leaves = [s[n] for n in ("q", "k", "v", "g", "state") if s[n] is not None]
    o, last = _plain_attention(s["q"], s["k"], s["v"], s["g"], s["state"], s["lengths"])
    return [o.detach(), last.detach()] + list(torch.autograd.grad([o, last], leaves, [s["do"], s["ds"]]))


def _own(s):
    from dms_amd import ops
    c = s["case"]
    if c["op"] == "step":
        return ops.linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["state"]), s["state"]
    if c["op"] == "rotary":
        if not c["train"]:
            return ops.head_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["sections"], base=BASE, eps=EPS)
        leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk")]
        y = ops.head_norm_rotary(*leaves, s["pos"], s["sections"], base=BASE, eps=EPS)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, [s["dq"], s["dk"]]))
    if not c["train"]:
        with torch.no_grad():
            return ops.linear_attention(s["q"], s["k"], s["v"], s["g"], s["state"], lengths=s["lengths"])
    leaves = [s[n] for n in ("q", "k", "v", "g", "state") if s[n] is not None]
    o, last = ops.linear_attention(s["q"], s["k"], s["v"], s["g"], s["state"], lengths=s["lengths"])
    return [o.detach(), last.detach()] + list(torch.autograd.grad([o, last], leaves, [s["do"], s["ds"]]))


def _chunks(x, heads, n):
    """(T, B, h, d) -> (B * heads, n, CHUNK, d) in 32 bits, shared heads repeated, zero rows behind the last."""
    x = x.float().repeat_interleave(heads // x.shape[2], 2)
    x = F.pad(x, (0, 0, 0, 0, 0, 0, 0, n * CHUNK - x.shape[0]))
    return x.permute(1, 2, 0, 3).reshape(x.shape[1] * heads, n, CHUNK, x.shape[3])


def _plain_attention(q, k, v, g, state, lengths):
    """The chunked form: products inside a chunk, one product over the chunks for the states between them."""
    T, B, dk, dtype = q.shape[0], q.shape[1], q.shape[3], q.dtype
    H, dv = g.shape[-1], v.shape[3]
    n = -(-T // CHUNK)
    gd = g.expand(T, B, H).double().clamp(min=-128.0)             # exp(-128) is 0 in 32 bits
    if lengths is not None:
        live = (torch.arange(T, device=g.device).view(T, 1) < lengths.view(1, B)).view(T, B, 1)
        gd = torch.where(live, gd, 0.0)
        k, v, q = (torch.where(live.unsqueeze(-1), x, 0.0) for x in (k, v, q))
    gd = F.pad(gd, (0, 0, 0, 0, 0, n * CHUNK - T)).permute(1, 2, 0).reshape(B * H, n, CHUNK)
    inside = gd.cumsum(-1)                                        # G_i
    total = inside[..., -1]
    q, k, v = (_chunks(x, H, n) for x in (q, k, v))
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=g.device).tril()
    d = (inside.unsqueeze(-1) - inside.unsqueeze(-2)).masked_fill(~low, -math.inf).exp().float()
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * d, v)
    left = (total.unsqueeze(-1) - inside).exp().float().unsqueeze(-1)
    s = torch.matmul((k * left).transpose(-1, -2), v).view(B * H, n, dk * dv)         # what each chunk adds
    upto = F.pad(total.cumsum(-1), (1, 0))                        # log decay from the start to each chunk's start
    first = torch.zeros(B * H, 1, dk * dv, device=g.device) if state is None else state.float().reshape(B * H, 1, dk * dv)
    s = torch.cat([first, s], 1)
    below = torch.ones(n + 1, n + 1, dtype=torch.bool, device=g.device).tril()
    mix = (upto.unsqueeze(-1) - upto.unsqueeze(-2)).masked_fill(~below, -math.inf).exp().float()
    s = torch.matmul(mix, s).view(B * H, n + 1, dk, dv)           # the state before every chunk, and after the last
    o = o + torch.matmul(q * inside.exp().float().unsqueeze(-1), s[:, :-1])
    o = (o * dk ** -0.5).view(B, H, n * CHUNK, dv)[:, :, :T].permute(2, 0, 1, 3)
    return o.to(dtype), s[:, -1].reshape(B, H, dk, dv)


def _plain_step(s):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    state = s["state"]
    state.copy_(state * s["g"].exp().unsqueeze(-1).unsqueeze(-1) + k.unsqueeze(-1) * v.unsqueeze(-2))
    o = (q.unsqueeze(-1) * state).sum(-2) * q.shape[-1] ** -0.5
    return o.to(s["q"].dtype), state


def _angles(pos, sections, pairs):
    """cos and sin (T, B, 1, pairs) of every pair's angle, in 64 bits before they are rounded; 0 where nothing turns."""
    freq = torch.cat([BASE ** (-torch.arange(n, device=DEV, dtype=torch.float64) / n) for n in sections])
    axis = torch.cat([torch.full((n,), a, device=DEV) for a, n in enumerate(sections)])
    angle = F.pad(pos.double()[..., axis] * freq, (0, pairs - freq.numel())).unsqueeze(2)
    return angle.cos(), angle.sin()


def _norm_turn(x, w, cos, sin):
    y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w
    even = F.pad(y, (0, y.shape[-1] % 2)).unflatten(-1, (-1, 2))
    a, b = even[..., 0], even[..., 1]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)[..., :x.shape[-1]]


def _plain_rotary(q, k, wq, wk, pos, sections):
    cos, sin = (t.float() for t in _angles(pos, sections, (q.shape[-1] + 1) // 2))
    return _norm_turn(q.float(), wq, cos, sin).to(q.dtype), _norm_turn(k.float(), wk, cos, sin).to(k.dtype)


def _plain_rotary_train(s):
    leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk")]
    y = _plain_rotary(*leaves, s["pos"], s["sections"])
    return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, [s["dq"], s["dk"]]))


# ------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    """Token by token in 64 bits, from the definition."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "step": _exact_step, "attention": _exact_attention}[case["op"]](s)


def _exact_step(s):
    q, k, v, S = (s[n].double() for n in ("q", "k", "v", "state"))
    S = torch.exp(s["g"].double())[..., None, None] * S + k[..., :, None] * v[..., None, :]
    return torch.einsum("bhc,bhcz->bhz", q, S) / math.sqrt(q.shape[-1]), S


def _exact_attention(s):
    c = s["case"]
    T, B, H = c["T"], c["B"], c["H"]
    scale = 1.0 / math.sqrt(c["dk"])
    heads = {n: torch.arange(H, device=DEV) // (H // c[m]) for n, m in (("q", "Hq"), ("k", "Hk"), ("v", "Hv"))}
    live = torch.ones(T, B, dtype=torch.bool, device=DEV)
    if s["lengths"] is not None:
        live = torch.arange(T, device=DEV)[:, None] < s["lengths"][None, :]
    row = {n: (lambda t, n=n: s[n][t].double()[:, heads[n]] * live[t][:, None, None]) for n in heads}
    a = torch.where(live[:, :, None], s["g"].expand(T, B, H).double().exp(), 1.0)
    S0 = torch.zeros(B, H, c["dk"], c["dv"], dtype=torch.float64, device=DEV) if s["state"] is None else s["state"].double()
    S = S0.clone()
    o = torch.empty(T, B, H, c["dv"], device=DEV, dtype=torch.float64)
    train = c["train"]
    if train:
        do = lambda t: s["do"][t].double() * live[t][:, None, None]  # noqa: E731
        dq = torch.empty(T, B, H, c["dk"], device=DEV, dtype=torch.float64)
    for t in range(T):
        S.mul_(a[t][..., None, None]).addcmul_(row["k"](t)[..., :, None], row["v"](t)[..., None, :])
        o[t] = torch.matmul(row["q"](t)[..., None, :], S)[..., 0, :] * scale
        if train:
            dq[t] = torch.matmul(S, do(t)[..., :, None])[..., 0] * scale
    if not train:
        return o, S
    dk, dv = torch.empty_like(dq), torch.empty_like(o)
    R = s["ds"].double().clone()
    for t in range(T - 1, -1, -1):
        R.addcmul_(row["q"](t)[..., :, None], do(t)[..., None, :], value=scale)
        dk[t] = torch.matmul(R, row["v"](t)[..., :, None])[..., 0] * live[t][:, None, None]
        dv[t] = torch.matmul(row["k"](t)[..., None, :], R)[..., 0, :] * live[t][:, None, None]
        R.mul_(a[t][..., None, None])
    # the decay at t acts on every path over the border before t: the flow into the queries from t on less that out of the keys from t on,
    # which is what came in with the first state less the difference of the tokens before t
    flow = torch.stack([(row["q"](t) * dq[t]).sum(-1) - (row["k"](t) * dk[t]).sum(-1) for t in range(T)])
    dg = (S0 * R).sum((-1, -2))[None] - (flow.cumsum(0) - flow)
    dg = torch.where(live[:, :, None] & (a > 0), dg, 0.0)
    if c["fixed"]:
        dg = dg.sum((0, 1))
    grouped = lambda d, h: d.view(T, B, h, H // h, -1).sum(3)  # noqa: E731
    grads = [grouped(dq, c["Hq"]), grouped(dk, c["Hk"]), grouped(dv, c["Hv"]), dg] + ([R] if s["state"] is not None else [])
    return [o, S] + grads


def _exact_rotary(s):
    sections, out = s["sections"], []
    D = s["q"].shape[-1]
    turn = torch.ones(s["pos"].shape[:2] + (1, (D + 1) // 2), dtype=torch.complex128, device=DEV)
    at = 0
    for axis, n in enumerate(sections):
        for i in range(n):
            angle = s["pos"][..., axis].double() * math.pow(BASE, -i / n)
            turn[:, :, 0, at] = torch.polar(torch.ones_like(angle), angle)
            at += 1

    def turned(x, by):
        z = torch.view_as_complex(F.pad(x, (0, D % 2)).unflatten(-1, (-1, 2)).contiguous()) * by
        return torch.view_as_real(z).flatten(-2)[..., :D]

    grads, weights = [], []
    for x, w, dy in ((s["q"], s["wq"], s.get("dq")), (s["k"], s["wk"], s.get("dk"))):
        x, w = x.double(), w.double()
        r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
        out.append(turned(x * r * w, turn))
        if dy is not None:
            back = turned(dy.double(), turn.conj())
            weights.append((back * x * r).sum((0, 1, 2)))
            back = back * w
            grads.append(r * back - x * r ** 3 * (back * x).sum(-1, keepdim=True) / D)
    return out + grads + weights
