"""Measured cases of the attention operators for video and text tokens: rotary positions on several axes (`functional.rope`), the
per-head norm of queries and keys with the rotation in the same pass (`functional.qk_norm_rope`), and attention with capped scores,
a distance bias, document and prefix masks (`functional.attention_mod`).

Every case runs one call of one operator on bf16 / fp16 / fp32 token matrices [rows, heads * dim]; a case with `train` runs the
forward and the backward pass and returns the gradients beside the output.  `own = False` computes the same with elementary torch
operations in 32 bits (angles in 64), rounded once at the end.
"""
import math
import random

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token for each of eight sequences, deep into a long text: the rotation of a serving step (launch latency)
        dict(name="rope step", op="rope", t=8, h=1, w=1, far=100000, heads=16, dim=128, sections="128", style="half", dtype="bf16",
             train=False),
        # the spatio-temporal tokens of a 16-frame clip at 256 x 256 pixels (32 x 32 latents), five heads of 64, with gradients
        dict(name="rope clip train", op="rope", t=16, h=32, w=32, far=0, heads=5, dim=64, sections="16,24,24", style="interleaved",
             dtype="bf16", train=True),
        # a clip of odd size in fp32, heads of 88 of which 72 columns turn
        dict(name="rope odd fp32", op="rope", t=13, h=19, w=27, far=0, heads=5, dim=88, sections="24,24,24", style="interleaved",
             dtype="fp32", train=False),
        # norm + rotation of one new token for each of four sequences, grouped heads
        dict(name="norm rope step", op="norm", t=4, h=1, w=1, far=30000, heads=16, kv_heads=4, dim=128, sections="128", style="half",
             norm="rms", dtype="bf16", train=False),
        # training step of the 16-frame clip, ten heads of 64
        dict(name="norm rope clip train", op="norm", t=16, h=32, w=32, far=0, heads=10, kv_heads=10, dim=64, sections="16,24,24",
             style="interleaved", norm="rms", dtype="bf16", train=True),
        # training step of a 24-frame clip at 576 x 320 pixels (72 x 40 latents), layer norm, twenty heads of 64: the largest rows
        dict(name="norm rope large train", op="norm", t=24, h=40, w=72, far=0, heads=20, kv_heads=20, dim=64, sections="16,24,24",
             style="half", norm="layer", dtype="bf16", train=True),
        # single-token step of eight sequences over a ragged cache, grouped heads, linear distance bias
        dict(name="attn step", op="attn", batch=8, sq=1, sk=16384, heads=16, kv_heads=4, dim=128, causal=True, ragged=True, prefix=0,
             docs=0, cap=0.0, bias="slopes", radius=0, dtype="bf16", train=False),
        # the text tower's rows (77 tokens, 16 heads of 64), causal, with a learned distance table, trained
        dict(name="attn text train", op="attn", batch=4, sq=77, sk=77, heads=16, kv_heads=16, dim=64, causal=True, ragged=False,
             prefix=0, docs=0, cap=0.0, bias="table", radius=32, dtype="bf16", train=True),
        # clips of different sizes packed behind one another, each attending to itself, trained
        dict(name="attn packed train", op="attn", batch=1, sq=8200, sk=8200, heads=10, kv_heads=10, dim=64, causal=False, ragged=False,
             prefix=0, docs=9, cap=0.0, bias="none", radius=0, dtype="bf16", train=True),
        # a prompt read in both directions and a continuation read forwards, capped scores, grouped heads, odd length, trained
        dict(name="attn prefix cap train", op="attn", batch=2, sq=2011, sk=2011, heads=16, kv_heads=4, dim=128, causal=True,
             ragged=False, prefix=300, docs=0, cap=30.0, bias="none", radius=0, dtype="bf16", train=True),
        # a chunk of new tokens over a long context, capped scores, fp16: few rows, long axis
        dict(name="attn chunk", op="attn", batch=1, sq=200, sk=12000, heads=16, kv_heads=4, dim=128, causal=True, ragged=False,
             prefix=0, docs=0, cap=50.0, bias="none", radius=0, dtype="fp16", train=False),
        # all tokens of a 16-frame clip at 32 x 32 latents in one sequence, causal with a distance bias: the largest products
        dict(name="attn clip", op="attn", batch=1, sq=16384, sk=16384, heads=8, kv_heads=8, dim=128, causal=True, ragged=False,
             prefix=1024, docs=0, cap=0.0, bias="slopes", radius=0, dtype="bf16", train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "norm", "attn", "attn"])
    if op != "attn":
        step = rng.random() < 0.3
        t = _log(rng, 1, 300) if step else rng.randint(1, 32)
        h, w = (1, 1) if step else (rng.randint(5, 40), rng.randint(5, 72))
        dim, sections = rng.choice([(64, "16,24,24"), (64, "64"), (88, "24,24,24"), (80, "16,32,32"), (128, "32,48,48"), (128, "128"),
                                    (128, "16,56,56"), (96, "64"), (40, "8,16,16")])
        heads = rng.choice([1, 2, 4, 5, 8, 10, 16])
        c = dict(op=op, t=t, h=h, w=w, far=rng.choice([0, _log(rng, 100, 1000000)]), heads=heads, dim=dim, sections=sections,
                 style=rng.choice(["interleaved", "half"]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                 train=rng.random() < 0.5)
        if op == "norm":
            c.update(kv_heads=rng.choice([k for k in (1, 2, 4, 5, 8, 10, 16) if heads % k == 0]), norm=rng.choice(["rms", "layer"]))
        return c
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4])
    dim = rng.choice([64, 64, 128, 128, 40, 80, 88])
    c = dict(op="attn", heads=heads, kv_heads=kv, dim=dim, prefix=0, docs=0, cap=rng.choice([0.0, 0.0, 20.0, 50.0]), radius=0,
             bias=rng.choice(["none", "slopes", "table"]), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    kind = rng.choice(["step", "chunk", "train", "train"])
    if kind == "step":
        c.update(batch=rng.randint(1, 16), sq=rng.randint(1, 4), sk=_log(rng, 5, 20000), causal=True, ragged=True, train=False)
        c["sk"] = max(c["sk"], c["sq"])
    elif kind == "chunk":
        c.update(batch=rng.randint(1, 3), sq=_log(rng, 16, 900), sk=_log(rng, 1000, 9000), causal=rng.random() < 0.7, ragged=True,
                 train=False)
    else:
        s = _log(rng, 30, 2600)
        c.update(batch=rng.randint(1, 3), sq=s, sk=s, causal=rng.random() < 0.6, ragged=False, train=True)
        c["docs"] = rng.choice([0, rng.randint(2, 8)])
        if c["causal"] and not c["docs"]:
            c["prefix"] = rng.choice([0, rng.randint(1, s)])
    if c["bias"] == "table":
        c["radius"] = rng.choice([8, 32, 128, 500])
    return c


# ------------------------------------------------------------------------------------------------ what a case's structure is
def _kv_lens(c):
    """Keys each sequence holds: ragged from nearly nothing to the whole cache."""
    if not c["ragged"]:
        return [c["sk"]] * c["batch"]
    r = random.Random(c["sk"] * 31 + c["batch"])
    return [max(min(c["sq"], c["sk"]), r.randint(c["sk"] // 3, c["sk"])) for _ in range(c["batch"])]


def _doc_ids(c):
    """One document number per token, -1 in the padding behind the last: clips of unequal sizes."""
    r = random.Random(c["sq"] * 17 + c["docs"])
    cuts = sorted(r.sample(range(1, c["sq"]), min(c["docs"], c["sq"] - 1)))        # the piece behind the last cut is padding
    ids, at = [], 0
    for n, cut in enumerate(cuts):
        ids += [n] * (cut - at)
        at = cut
    return ids + [-1] * (c["sq"] - at)


def _pairs(c):
    """Query / key pairs that may see each other, of one head over the whole batch."""
    if c["docs"]:
        ids = _doc_ids(c)
        n = 0
        for d in set(ids) - {-1}:
            s = ids.count(d)
            n += s * (s + 1) // 2 if c["causal"] else s * s
        return n * c["batch"]
    n = 0
    for L in _kv_lens(c):
        if not c["causal"]:
            n += c["sq"] * L
            continue
        for i in range(c["sq"]):
            n += min(L, max(0, i + L - c["sq"] + 1, c["prefix"]))
    return n


def work(c):
    es = 4 if c["dtype"] == "fp32" else 2
    if c["op"] != "attn":
        rows = c["t"] * c["h"] * c["w"]
        n = rows * (c["heads"] + c.get("kv_heads", 0)) * c["dim"]
        # forward: each element read and written; backward: the upstream gradient read and the input's written (the norm reads its
        # input there too, which one pass over both directions would not need again)
        return {"bytes": n * es * (4 if c["train"] else 2) + rows * 12, "flops": n * (20 if c["train"] else 8)}
    q, kv = c["batch"] * c["sq"] * c["heads"] * c["dim"] * es, sum(_kv_lens(c)) * c["kv_heads"] * c["dim"] * es
    pairs = _pairs(c) * c["heads"]
    if c["train"]:      # q, k, v, do read; o, dq, dk, dv written; two products forward, five backward
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * c["dim"]}
    return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * c["dim"]}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(c, seed):
    g = _gen(seed)
    dt = _DTYPE[c["dtype"]]

    def rand(*shape, mul=1.0, to=dt, leaf=c["train"]):
        x = (torch.randn(*shape, generator=g, device="cuda") * mul).to(to)
        return x.requires_grad_(leaf)

    s = {"case": c}
    if c["op"] != "attn":
        rows, width = c["t"] * c["h"] * c["w"], c["heads"] * c["dim"]
        axes = len(c["sections"].split(","))
        grid = torch.stack(torch.meshgrid(*[torch.arange(n, device="cuda") for n in (c["t"], c["h"], c["w"])], indexing="ij"), -1)
        pos = grid.reshape(rows, 3)[:, :axes]
        if c["far"]:        # sequences stand anywhere up to `far`
            pos = pos + torch.randint(0, c["far"], (rows, axes), generator=g, device="cuda")
        s["pos"] = pos.to(torch.int32).contiguous()
        if c["op"] == "rope":
            s["x"] = rand(rows, width, mul=2.0)
            s["dy"] = [rand(rows, width, leaf=False)] if c["train"] else None
            s["leaves"] = [s["x"]]
        else:
            kw = c["kv_heads"] * c["dim"]
            s["q"], s["k"] = rand(rows, width, mul=2.0), rand(rows, kw, mul=0.5)
            s["qw"] = (1 + rand(c["dim"], mul=0.1, to=torch.float32, leaf=False)).requires_grad_(c["train"])
            s["kw"] = (1 + rand(c["dim"], mul=0.1, to=torch.float32, leaf=False)).requires_grad_(c["train"])
            s["qb"] = s["kb"] = None
            if c["norm"] == "layer":
                s["qb"], s["kb"] = rand(c["dim"], mul=0.1, to=torch.float32), rand(c["dim"], mul=0.1, to=torch.float32)
            s["dy"] = [rand(rows, width, leaf=False), rand(rows, kw, leaf=False)] if c["train"] else None
            s["leaves"] = [x for x in (s["q"], s["k"], s["qw"], s["kw"], s["qb"], s["kb"]) if x is not None]
        return s
    B, D = c["batch"], c["dim"]
    s["q"] = rand(B * c["sq"], c["heads"] * D, mul=1.5 if not c["cap"] else 4.0)
    s["k"], s["v"] = rand(B * c["sk"], c["kv_heads"] * D), rand(B * c["sk"], c["kv_heads"] * D)
    s["leaves"] = [s["q"], s["k"], s["v"]]
    s["kv_len"] = torch.tensor(_kv_lens(c), dtype=torch.int32, device="cuda") if c["ragged"] else None
    s["prefix"] = torch.full((B,), c["prefix"], dtype=torch.int32, device="cuda") if c["prefix"] else None
    s["docs"] = torch.tensor([_doc_ids(c)] * B, dtype=torch.int32, device="cuda") if c["docs"] else None
    s["slopes"] = s["bias"] = None
    if c["bias"] == "slopes":
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (n + 1) / c["heads"]) for n in range(c["heads"])], device="cuda")
    elif c["bias"] == "table":
        s["bias"] = rand(c["heads"], 2 * c["radius"] + 1)
        s["leaves"].append(s["bias"])
    s["dy"] = [rand(B * c["sq"], c["heads"] * D, leaf=False)] if c["train"] else None
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        outs = _own(s, c) if own else _plain(s, c)
        if not c["train"]:
            return list(outs)
        return list(outs) + list(torch.autograd.grad(outs, s["leaves"], s["dy"]))


def _own(s, c):
    import t2v_amd  # noqa: F401
    import t2v_amd.functional as F
    if c["op"] != "attn":
        axes = F.RopeAxes(tuple(map(int, c["sections"].split(","))), style=c["style"])
        if c["op"] == "rope":
            return (F.rope(s["x"], c["heads"], s["pos"], axes),)
        return F.qk_norm_rope(s["q"], s["k"], c["heads"], c["kv_heads"], s["pos"], axes, s["qw"], s["kw"], q_bias=s["qb"],
                              k_bias=s["kb"], norm=c["norm"], eps=1e-6)
    qlay, klay = F.SeqLayout(c["batch"], c["sq"], c["sq"], 0, 1), F.SeqLayout(c["batch"], c["sk"], c["sk"], 0, 1)
    return (F.attention_mod(s["q"], s["k"], s["v"], c["heads"], qlay, klay, kv_heads=c["kv_heads"], causal=c["causal"],
                            prefix=s["prefix"], kv_len=s["kv_len"], q_docs=s["docs"], kv_docs=s["docs"], softcap=c["cap"],
                            slopes=s["slopes"], bias=s["bias"]),)


def _turned(x, pos, c):
    """x: fp32 [rows, heads, dim], its first sum(sections) columns turned pair by pair."""
    dims = [int(d) for d in c["sections"].split(",")]
    R = sum(dims)
    angle = torch.cat([pos[:, a:a + 1].double() * 10000.0 ** (-torch.arange(0, d, 2, device=x.device, dtype=torch.float64) / d)
                       for a, d in enumerate(dims)], 1)                                        # [rows, R / 2]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    r, rest = x[..., :R], x[..., R:]
    if c["style"] == "half":
        a, b = r[..., :R // 2], r[..., R // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = r[..., 0::2], r[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _normed(x, weight, bias, c):
    if c["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
    return y if bias is None else y + bias


def _plain(s, c):
    if c["op"] == "rope":
        x = s["x"]
        return (_turned(x.float().view(x.shape[0], c["heads"], c["dim"]), s["pos"], c).reshape(x.shape).to(x.dtype),)
    if c["op"] == "norm":
        outs = []
        for x, h, w, b in ((s["q"], c["heads"], s["qw"], s["qb"]), (s["k"], c["kv_heads"], s["kw"], s["kb"])):
            y = _normed(x.float().view(x.shape[0], h, c["dim"]), w, b, c)
            outs.append(_turned(y, s["pos"], c).reshape(x.shape).to(x.dtype))
        return tuple(outs)
    B, Sq, Sk, H, KV, D = c["batch"], c["sq"], c["sk"], c["heads"], c["kv_heads"], c["dim"]
    q = s["q"].float().view(B, Sq, H, D).transpose(1, 2)
    k = s["k"].float().view(B, Sk, KV, D).transpose(1, 2).repeat_interleave(H // KV, 1)
    v = s["v"].float().view(B, Sk, KV, D).transpose(1, 2).repeat_interleave(H // KV, 1)
    t = q @ k.transpose(2, 3) * D ** -0.5                                                         # [B, H, Sq, Sk]
    if c["cap"]:
        t = c["cap"] * torch.tanh(t / c["cap"])
    j = torch.arange(Sk, device=q.device)[None, None]
    L = (s["kv_len"] if s["kv_len"] is not None else torch.full((B,), Sk, device=q.device))[:, None, None]
    i = torch.arange(Sq, device=q.device)[None, :, None] + L - Sq                                 # the query's place among the keys
    if s["slopes"] is not None:
        t = t - s["slopes"].view(1, H, 1, 1) * (j - i).abs()[:, None]
    if s["bias"] is not None:
        R = c["radius"]
        at = ((j - i).clamp(-R, R) + R).expand(B, Sq, Sk)
        t = t + s["bias"].float().index_select(1, at.reshape(-1)).view(H, B, Sq, Sk).transpose(0, 1)
    seen = (j < L).expand(B, Sq, Sk)
    if c["causal"]:
        ahead = j <= i
        if s["prefix"] is not None:
            ahead = ahead | (j < s["prefix"][:, None, None])
        seen = seen & ahead
    if s["docs"] is not None:
        seen = seen & (s["docs"][:, :, None] == s["docs"][:, None]) & (s["docs"][:, :, None] >= 0)
    t = t.masked_fill(~seen[:, None], float("-inf"))
    top = t.detach().amax(-1, keepdim=True)
    p = torch.exp(t - torch.where(torch.isinf(top), 0.0, top))
    o = p @ v / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return (o.transpose(1, 2).reshape(B * Sq, H * D).to(s["q"].dtype),)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_rotation(pos, c):
    """The rotation of one row's columns as complex factors [rows, R / 2]."""
    cols = []
    for a, d in enumerate(int(n) for n in c["sections"].split(",")):
        inv = torch.exp(torch.arange(d // 2, dtype=torch.float64, device=pos.device) * (-2.0 * math.log(10000.0) / d))
        cols.append(torch.outer(pos[:, a].to(torch.float64), inv))
    phase = torch.cat(cols, -1)
    return torch.polar(torch.ones_like(phase), phase)


def _exact_turn(x, z, c):
    """x [rows, heads, dim] (64 bits) times the rotation z (its conjugate turns back)."""
    n = z.shape[1]
    y = x.clone()
    first = torch.arange(n, device=x.device) * (1 if c["style"] == "half" else 2)
    second = first + (n if c["style"] == "half" else 1)
    turned = torch.complex(x[:, :, first], x[:, :, second]) * z[:, None]
    y[:, :, first], y[:, :, second] = turned.real, turned.imag
    return y


def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        return _exact_attention(s, c) if c["op"] == "attn" else _exact_rope(s, c)


def _exact_rope(s, c):
    z = _exact_rotation(s["pos"], c)
    D, dy = c["dim"], s["dy"]
    if c["op"] == "rope":
        shape = s["x"].shape
        outs = [_exact_turn(s["x"].double().view(shape[0], -1, D), z, c).reshape(shape)]
        if c["train"]:
            outs.append(_exact_turn(dy[0].double().view(shape[0], -1, D), z.conj(), c).reshape(shape))
        return outs
    outs, dxs, dws, dbs = [], [], [], []
    for n, (x, w, b) in enumerate(((s["q"], s["qw"], s["qb"]), (s["k"], s["kw"], s["kb"]))):
        shape = x.shape
        x, w = x.double().view(shape[0], -1, D), w.double()
        mid = x.mean(-1, keepdim=True) if c["norm"] == "layer" else torch.zeros_like(x[..., :1])
        r = 1.0 / torch.sqrt(((x - mid) ** 2).mean(-1, keepdim=True) + 1e-6)
        hat = (x - mid) * r
        outs.append(_exact_turn(hat * w + (0.0 if b is None else b.double()), z, c).reshape(shape))
        if c["train"]:
            d = _exact_turn(dy[n].double().view(shape[0], -1, D), z.conj(), c)
            dws.append((d * hat).sum((0, 1)))
            if b is not None:
                dbs.append(d.sum((0, 1)))
            e = d * w
            dx = e - hat * (e * hat).mean(-1, keepdim=True)
            if c["norm"] == "layer":
                dx = dx - e.mean(-1, keepdim=True)
            dxs.append((dx * r).reshape(shape))
    return outs + dxs + dws + dbs


def _exact_attention(s, c):
    B, Sq, Sk, H, KV, D = c["batch"], c["sq"], c["sk"], c["heads"], c["kv_heads"], c["dim"]
    dev, G, scale = s["q"].device, H // KV, D ** -0.5
    q, k, v = s["q"].view(B, Sq, H, D), s["k"].view(B, Sk, KV, D), s["v"].view(B, Sk, KV, D)
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device=dev)
    if c["train"]:
        dq, dk, dv = torch.zeros_like(out), torch.zeros(B, Sk, KV, D, dtype=torch.float64, device=dev), \
            torch.zeros(B, Sk, KV, D, dtype=torch.float64, device=dev)
        dtable = torch.zeros(H, 2 * c["radius"] + 1, dtype=torch.float64, device=dev)
        do = s["dy"][0].view(B, Sq, H, D)
    lens = _kv_lens(c)
    for b in range(B):
        L = lens[b]
        col = torch.arange(L, device=dev)
        row = torch.arange(Sq, device=dev) + (L - Sq)
        gap = col[None, :] - row[:, None]
        hidden = torch.zeros(Sq, L, dtype=torch.bool, device=dev)
        if c["causal"]:
            hidden |= (gap > 0) & (col[None, :] >= c["prefix"])
        if c["docs"]:
            ids = s["docs"][b]
            hidden |= (ids[:, None] != ids[None, :]) | (ids[:, None] < 0)
        for h in range(H):
            Q, K, V = q[b, :, h].double(), k[b, :L, h // G].double(), v[b, :L, h // G].double()
            raw = torch.mm(Q, K.t()).mul_(scale)
            bent = None
            if c["cap"]:
                bent = torch.tanh(raw / c["cap"])
                raw = bent * c["cap"]
            if s["slopes"] is not None:
                raw = raw - float(s["slopes"][h]) * gap.abs()
            if s["bias"] is not None:
                place = gap.clamp(-c["radius"], c["radius"]) + c["radius"]
                raw = raw + s["bias"][h].double()[place]
            raw[hidden] = -math.inf
            P = torch.nan_to_num(torch.softmax(raw, -1), nan=0.0)
            del raw
            O = torch.mm(P, V)
            out[b, :, h] = O
            if not c["train"]:
                continue
            G_o = do[b, :, h].double()
            dv[b, :L, h // G] += torch.mm(P.t(), G_o)
            dS = P * (torch.mm(G_o, V.t()) - (G_o * O).sum(-1, keepdim=True))
            if s["bias"] is not None:
                dtable[h].index_add_(0, place.reshape(-1), dS.reshape(-1))
            if bent is not None:
                dS = dS * (1.0 - bent * bent)
            dq[b, :, h] = torch.mm(dS, K) * scale
            dk[b, :L, h // G] += torch.mm(dS.t(), Q) * scale
    outs = [out.reshape(B * Sq, H * D)]
    if c["train"]:
        outs += [dq.reshape(B * Sq, H * D), dk.reshape(B * Sk, KV * D), dv.reshape(B * Sk, KV * D)]
        if s["bias"] is not None:
            outs.append(dtable)
    return outs
