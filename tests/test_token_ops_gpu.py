"""Rotary positions, per-head norms with rotation, and attention with modified scores on the GPU against plain 64-bit forms
(tests/token_ops_ref.py).  Tolerances are elementwise bounds derived there: one half step of the type per rounding."""
import math

import pytest
import torch
import torch.utils.checkpoint

import token_ops_ref as ref

pytestmark = pytest.mark.gpu
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def _f():
    import t2v_amd  # noqa: F401
    import t2v_amd.functional as F
    return F


def _within(name, got, want, bound):
    got = got.detach().cpu().to(F64).reshape(want.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = ((got - want).abs() - bound).max() if want.numel() else torch.tensor(0.0)
    at = ((got - want).abs() / bound).max() if want.numel() else 0.0
    assert over <= 0, f"{name}: {float(at):.2f} times the bound"


# ------------------------------------------------------------------------------------------------ rotary positions
ROPE = [  # rows, heads, dim, dims, style, shared, dtype, pos dtype, far
    (1, 1, 8, (8,), "interleaved", False, BF, torch.int32, 0),
    (3, 2, 64, (16, 24, 24), "interleaved", False, BF, torch.int32, 1000),
    (257, 5, 88, (24, 24, 24), "half", False, F32, torch.int64, 100000),
    (130, 3, 128, (32, 48, 48), "half", True, HF, torch.int32, 2000000),
    (77, 16, 64, (64,), "half", False, BF, torch.float32, 500),
    (19, 9, 40, (8, 16), "interleaved", True, F32, torch.float32, 50),
    (33, 1, 256, (64, 64, 64, 64), "interleaved", False, BF, torch.int32, 300),
    (5, 7, 96, (8,), "half", False, BF, torch.int32, 10),
]


def _half_step(want, dt, mag, fp32=3e-6):
    """Half a step of the stored type, and the fp32 error of the two products (and of a sine to one unit in the last place)."""
    return torch.finfo(dt).eps / 2 * want.abs() + fp32 * mag + (2.0 ** -25 if dt == HF else 1e-30)


@pytest.mark.parametrize("rows,heads,dim,dims,style,shared,dt,pdt,far", ROPE)
def test_rope_matches_the_64_bit_form(rows, heads, dim, dims, style, shared, dt, pdt, far):
    F = _f()
    g = torch.Generator().manual_seed(rows + dim)
    x = (torch.randn(rows, heads * dim, generator=g) * 3).to(dt)
    dy = torch.randn(rows, heads * dim, generator=g).to(dt)
    pos = torch.randint(0, far + 1, (rows, len(dims)), generator=g).to(pdt)
    if pdt == F32:
        pos = pos + 0.25
    scale = tuple(1.0 + 0.5 * n for n in range(len(dims)))
    axes = F.RopeAxes(dims, theta=5000.0, style=style, shared=shared, scale=scale)
    xd = x.cuda().requires_grad_()
    y = F.rope(xd, heads, pos.cuda(), axes)
    y.backward(dy.cuda())
    kw = dict(theta=5000.0, style=style, shared=shared, scale=scale)
    for name, got, src, back in (("y", y, x, False), ("dx", xd.grad, dy, True)):
        s = src.to(F64).view(rows, heads, dim)
        want = ref.turn(s, pos, dims, back=back, **kw)
        mag = s.abs().amax(-1, keepdim=True).expand_as(s)
        assert got.dtype == dt
        _within(name, got, want, _half_step(want, dt, mag))
    with torch.no_grad():
        assert torch.equal(F.rope(x.cuda(), heads, pos.cuda(), axes), y)


def test_rope_strided_rows_and_given_frequencies():
    F = _f()
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(50, 3 * 128, generator=g).to(BF)
    pos = torch.randint(0, 90, (50, 4), generator=g).int()
    fr = torch.rand(32, generator=g, dtype=F64)
    x = wide[:, 128:256]
    y = F.rope(wide.cuda()[:, 128:256], 2, pos.cuda()[:, :2], F.RopeAxes((32, 32), style="half"), freqs=fr.cuda())
    s = x.to(F64).reshape(50, 2, 64)
    want = ref.turn(s, pos, (32, 32), style="half", freqs=fr)
    _within("y", y, want, _half_step(want, BF, s.abs().amax(-1, keepdim=True).expand_as(s)))


NORM = [  # rows, heads, kv_heads, dim, dims, style, norm, bias, dtype
    (1, 1, 1, 64, (64,), "half", "rms", False, BF),
    (4, 16, 4, 128, (128,), "half", "rms", False, BF),
    (301, 5, 5, 64, (16, 24, 24), "interleaved", "rms", True, BF),
    (77, 6, 2, 88, (24, 24, 24), "interleaved", "layer", True, F32),
    (1030, 3, 1, 40, (8, 16, 16), "half", "layer", False, HF),
    (9, 2, 2, 256, (64, 96, 96), "half", "layer", True, F32),
    (130, 20, 20, 64, None, "half", "rms", False, BF),
    (2100, 9, 3, 8, (8,), "half", "rms", True, BF),
]


@pytest.mark.parametrize("rows,heads,kv,dim,dims,style,norm,bias,dt", NORM)
def test_qk_norm_rope_matches_the_64_bit_form(rows, heads, kv, dim, dims, style, norm, bias, dt):
    F = _f()
    g = torch.Generator().manual_seed(rows + dim + heads)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = (r(rows, heads * dim) * 2 + 0.3).to(dt), (r(rows, kv * dim) * 0.5).to(dt)
    dq, dk = r(rows, heads * dim).to(dt), r(rows, kv * dim).to(dt)
    ws = [1 + 0.2 * r(dim), 1 + 0.2 * r(dim)]
    bs = [0.3 * r(dim), 0.3 * r(dim)] if bias else [None, None]
    pos = torch.randint(0, 5000, (rows, len(dims or ())), generator=g).int() if dims else None
    axes = F.RopeAxes(dims, style=style) if dims else None
    leaves = [t.cuda().requires_grad_() if t is not None else None for t in (q, k, *ws, *bs)]
    yq, yk = F.qk_norm_rope(leaves[0], leaves[1], heads, kv, pos.cuda() if dims else None, axes, leaves[2], leaves[3], leaves[4], leaves[5],
                            eps=1e-5, norm=norm)
    torch.autograd.backward((yq, yk), (dq.cuda(), dk.cuda()))
    with torch.no_grad():
        nq, nk = F.qk_norm_rope(leaves[0], leaves[1], heads, kv, pos.cuda() if dims else None, axes, *leaves[2:], eps=1e-5, norm=norm)
    assert torch.equal(nq, yq) and torch.equal(nk, yk)
    for n, (x, up, y, h, w, b) in enumerate(((q, dq, yq, heads, ws[0], bs[0]), (k, dk, yk, kv, ws[1], bs[1]))):
        x, up, w = x.to(F64).view(rows, h, dim), up.to(F64).view(rows, h, dim), w.to(F64)
        hat, rs = ref.norm_stats(x, norm, 1e-5)
        z = hat * w + (0 if b is None else b.to(F64))
        want = ref.turn(z, pos, dims, style=style) if dims else z
        mag = z.abs().amax(-1, keepdim=True).expand_as(z) + 1
        _within(f"y{n}", y, want, _half_step(want, dt, mag, 1e-5))
        d = ref.turn(up, pos, dims, style=style, back=True) if dims else up
        dx, dw, db = ref.norm_backward(x, w, d, norm, 1e-5)
        mag = (d.abs().amax(-1, keepdim=True) * rs * (1 + hat.abs())) * 2
        _within(f"dx{n}", leaves[n].grad, dx, _half_step(dx, dt, mag.expand_as(dx), 1e-5))
        # fp32 sums of rows * heads products whose factors carry an error of ~1e-6 of the row's magnitude
        _within(f"dw{n}", leaves[2 + n].grad, dw, 1e-5 * (d * hat).abs().sum((0, 1)) + 1e-5)
        if b is not None:
            _within(f"db{n}", leaves[4 + n].grad, db, 1e-5 * d.abs().sum((0, 1)) + 1e-5)


def test_qk_norm_rope_gradient_against_differences():
    F = _f()
    g = torch.Generator().manual_seed(5)
    x = [torch.randn(6, 2 * 16, generator=g).cuda().requires_grad_(), torch.randn(6, 16, generator=g).cuda().requires_grad_(),
         (1 + 0.1 * torch.randn(16, generator=g)).cuda().requires_grad_(), (1 + 0.1 * torch.randn(16, generator=g)).cuda().requires_grad_()]
    pos = torch.arange(6).view(6, 1).cuda()
    up = [torch.randn(6, 32, generator=g).cuda(), torch.randn(6, 16, generator=g).cuda()]
    f = lambda: sum((o.double() * w).sum() for o, w in  # noqa: E731
                    zip(F.qk_norm_rope(x[0], x[1], 2, 1, pos, F.RopeAxes((16,)), x[2], x[3], norm="layer"), up))
    f().backward()
    h = 2.0 ** -6
    for t in x:
        for at in (0, t.numel() // 2, t.numel() - 1):
            with torch.no_grad():
                v = t.view(-1)[at].item()
                t.view(-1)[at] = v + h
                hi = f().item()
                t.view(-1)[at] = v - h
                lo = f().item()
                t.view(-1)[at] = v
            # central difference: third derivatives of the norm (about 6 here) times h^2 / 6, and fp32 noise of ~40 sums over 2 h
            assert abs((hi - lo) / (2 * h) - t.grad.view(-1)[at].item()) < 4 * h * h + 1e-3


def test_rope_and_norm_of_nothing_and_broadcast_gradients():
    F = _f()
    e = torch.empty(0, 128, dtype=BF, device="cuda", requires_grad=True)
    y = F.rope(e, 2, torch.empty(0, 1, dtype=torch.int32, device="cuda"), F.RopeAxes((64,)))
    y.sum().backward()
    assert y.shape == (0, 128) and e.grad.shape == (0, 128)
    w = torch.ones(64, device="cuda", requires_grad=True)
    a, b = F.qk_norm_rope(e, e[:, :64], 2, 1, None, None, w, w)
    (a.float().sum() + b.float().sum()).backward()
    assert a.shape == (0, 128) and b.shape == (0, 64) and torch.equal(w.grad, torch.zeros_like(w))
    # an expanded upstream gradient, and ONE weight for both sides: its gradient is the sum
    x = torch.randn(10, 128, device="cuda").to(BF).requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    a, b = F.qk_norm_rope(x, x, 2, 2, None, None, w, w)
    (a.sum() + b.sum()).backward()
    hat, _ = ref.norm_stats(x.detach().cpu().to(F64).view(10, 2, 64), "rms", 1e-6)
    _within("dw", w.grad, 2 * hat.sum((0, 1)), 1e-4 * hat.abs().sum((0, 1)) + 1e-4)


# ------------------------------------------------------------------------------------------------ attention
def _docs(n, cuts, pad):
    d, at = torch.full((n,), -1, dtype=torch.int32), 0
    for k, c in enumerate(cuts):
        d[at:at + c] = k
        at += c
    assert at + pad == n
    return d


ATTN = {  # B, Sq, Sk, H, KV, D, dtype, options
    "one": (1, 1, 1, 1, 1, 64, BF, {}),
    "one row": (2, 1, 70, 4, 2, 64, BF, dict(causal=True)),
    "plain odd": (2, 37, 91, 2, 2, 64, BF, {}),
    "plain 128": (1, 200, 200, 2, 1, 128, HF, {}),
    "dim 8": (1, 33, 65, 2, 2, 8, BF, dict(causal=True)),
    "dim 88": (1, 65, 130, 3, 1, 88, HF, dict(causal=True, softcap=5.0)),
    "dim 40 groups of 3": (2, 129, 129, 6, 2, 40, BF, dict(causal=True, slopes=True)),
    "causal tile edges": (1, 128, 128, 2, 2, 64, BF, dict(causal=True)),
    "causal short keys": (1, 70, 20, 2, 1, 64, BF, dict(causal=True)),
    "cap": (1, 150, 150, 2, 2, 64, BF, dict(softcap=2.0)),
    "cap 128 groups": (2, 140, 140, 4, 1, 128, BF, dict(softcap=8.0, causal=True, prefix=[10, 133])),
    "slopes both ways": (1, 100, 140, 4, 4, 64, HF, dict(slopes=True)),
    "table": (2, 77, 77, 4, 4, 64, BF, dict(causal=True, bias=32)),
    "table fp32 groups": (1, 90, 150, 4, 2, 128, BF, dict(bias=16, bias_f32=True, softcap=10.0)),
    "table of one entry": (1, 40, 40, 2, 2, 64, BF, dict(bias=0)),
    "table wide": (1, 130, 130, 2, 1, 64, HF, dict(bias=1024, slopes=True)),
    "table wide of 128": (1, 150, 190, 2, 2, 128, BF, dict(bias=1024, slopes=True, softcap=11.0, causal=True)),
    "many query heads of one key head": (2, 37, 130, 70, 1, 24, HF, dict(causal=True, kv_len=[130, 64])),
    "lengths": (4, 50, 150, 2, 2, 64, BF, dict(kv_len=[150, 1, 0, 77], causal=True)),
    "lengths two ways": (3, 40, 100, 2, 1, 128, BF, dict(kv_len=[100, 3, 64])),
    "prefix per query": (2, 90, 90, 2, 2, 64, BF, dict(causal=True, prefix="query")),
    "documents": (1, 300, 300, 2, 2, 64, BF, dict(docs=((100, 28, 64, 70), 38))),
    "documents causal": (2, 200, 200, 4, 2, 128, BF, dict(docs=((1, 63, 64, 65), 7), causal=True, softcap=20.0)),
    "documents shuffled": (1, 150, 150, 2, 2, 64, HF, dict(docs="shuffled", slopes=True)),
    "documents, table": (1, 160, 160, 2, 2, 64, BF, dict(docs=((80, 70), 10), bias=8, causal=True)),
    "all at once": (2, 130, 200, 4, 2, 88, BF, dict(docs="shuffled", bias=20, softcap=6.0, slopes=True, causal=True, prefix=[30, 199],
                                                     kv_len=[200, 131])),
    # enough workgroups for the sorted work lists of packed documents (row tiles * heads above 256), with and without a table
    "many documents": (2, 2070, 2070, 9, 9, 8, BF, dict(docs=((300, 1, 500, 77, 128, 640, 390), 34), softcap=9.0)),
    "many documents, table": (1, 2070, 2070, 16, 16, 16, BF, dict(docs=((300, 1, 500, 77, 128, 640, 390), 34), bias=12, causal=True)),
    "many documents of 128": (1, 1100, 1100, 32, 32, 72, HF, dict(docs=((200, 333, 5, 400), 162))),
    "many documents shuffled": (2, 1100, 1100, 16, 16, 8, BF, dict(docs="shuffled")),
    "long": (1, 1100, 1100, 2, 1, 64, BF, dict(causal=True, softcap=15.0)),
    "long keys": (1, 5, 4000, 4, 2, 128, BF, dict(causal=True, slopes=True)),
    "rows for a little more than one workgroup per CU": (1, 2100, 2110, 16, 16, 16, HF, dict(causal=True, prefix=[100], softcap=9.0)),
    "documents in splits": (1, 1100, 1100, 2, 2, 64, BF, dict(docs=((200, 333, 5, 400), 162), causal=True, bias=20)),
    "documents shuffled in splits": (2, 700, 5000, 2, 1, 40, HF, dict(docs="shuffled", softcap=7.0)),
    "very long keys": (1, 3, 40000, 2, 1, 64, HF, dict(causal=True, slopes=True)),
    "steps of long and short keys": (2, 1, 20000, 8, 2, 128, BF, dict(causal=True, softcap=12.0, kv_len=[20000, 777])),
    "few keys, many rows": (1, 1500, 30, 2, 2, 64, BF, {}),
}


def _attn_case(name, seed=0):
    B, Sq, Sk, H, KV, D, dt, opt = ATTN[name]
    opt = dict(opt)
    g = torch.Generator().manual_seed(sum(map(ord, name)) + seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, do = (r(B, Sq, H, D) * 2).to(dt), r(B, Sk, KV, D).to(dt), r(B, Sk, KV, D).to(dt), r(B, Sq, H, D).to(dt)
    kw = dict(causal=opt.get("causal", False), softcap=opt.get("softcap", 0.0))
    if opt.get("slopes"):
        kw["slopes"] = torch.rand(H, generator=g) * 0.3
    if "bias" in opt:
        kw["bias"] = r(H, 2 * opt["bias"] + 1).to(F32 if opt.get("bias_f32") else dt)
    if "kv_len" in opt:
        kw["kv_len"] = torch.tensor(opt["kv_len"], dtype=torch.int32)
    if "prefix" in opt:
        kw["prefix"] = torch.randint(0, Sk + 1, (B, Sq), generator=g).int() if opt["prefix"] == "query" else torch.tensor(opt["prefix"]).int()
    if "docs" in opt:
        if opt["docs"] == "shuffled":
            kw["q_docs"], kw["kv_docs"] = (torch.randint(-1, 4, (B, n), generator=g).int() for n in (Sq, Sk))
        else:
            kw["q_docs"] = kw["kv_docs"] = _docs(Sq, *opt["docs"])[None].repeat(B, 1).contiguous()
    return q, k, v, do, kw


def _dev(t):
    return t.cuda() if torch.is_tensor(t) else t


@pytest.mark.parametrize("name", list(ATTN))
def test_attention_mod_matches_the_64_bit_form(name):
    F = _f()
    q, k, v, do, kw = _attn_case(name)
    B, Sq, H, D = q.shape
    Sk, KV = k.shape[1:3]
    want = ref.attention(q, k, v, D ** -0.5, q.dtype, do=do, **kw)
    flat = [t.reshape(t.shape[0] * t.shape[1], -1).cuda().requires_grad_() for t in (q, k, v)]
    dkw = {n: _dev(t) for n, t in kw.items()}
    if "bias" in dkw:
        dkw["bias"].requires_grad_()
    lays = F.SeqLayout(B, Sq, Sq, 0, 1), F.SeqLayout(B, Sk, Sk, 0, 1)
    o = F.attention_mod(*flat, H, *lays, kv_heads=KV, **dkw)
    _within("o", o, want["o"][0], want["o"][1])
    o.backward(do.reshape(B * Sq, -1).cuda())
    for n, t in zip(("dq", "dk", "dv"), flat):
        _within(n, t.grad, *want[n])
    if "bias" in dkw:
        assert dkw["bias"].grad.dtype == dkw["bias"].dtype
        _within("dbias", dkw["bias"].grad, *want["dbias"])
    # the same again is bit-equal, with and without what the backward pass keeps
    with torch.no_grad():
        o2 = F.attention_mod(*flat, H, *lays, kv_heads=KV, **dkw)
    _within("o (no grad)", o2, want["o"][0], want["o"][1])
    grads = [t.grad.clone() for t in flat]
    for t in flat:
        t.grad = None
    o3 = F.attention_mod(*flat, H, *lays, kv_heads=KV, **dkw)
    assert torch.equal(o3, o)
    o3.backward(do.reshape(B * Sq, -1).cuda())
    assert all(torch.equal(a, t.grad) for a, t in zip(grads, flat))


def test_attention_mod_rows_that_nobody_sees_may_hold_anything():
    F = _f()
    for name in ("lengths", "documents", "documents causal", "lengths two ways", "causal short keys"):
        q, k, v, do, kw = _attn_case(name, 7)
        B, Sq, H, D = q.shape
        Sk, KV = k.shape[1:3]
        want = ref.attention(q, k, v, D ** -0.5, q.dtype, do=do, **kw)
        for b in range(B):
            L = Sk if "kv_len" not in kw else int(kw["kv_len"][b])
            seen = ref.visible(Sq, Sk, L, kw["causal"], None, kw["q_docs"][b] if "q_docs" in kw else None, kw["kv_docs"][b] if "kv_docs" in kw else None)
            hid = torch.arange(Sk) >= L
            if "kv_docs" in kw:
                hid |= kw["kv_docs"][b] < 0
            k[b, hid], v[b, hid] = math.nan, math.inf
            none = ~seen.any(1)
            if "q_docs" in kw:
                none = kw["q_docs"][b] < 0
            q[b, none], do[b, none] = math.inf, math.nan
        flat = [t.reshape(t.shape[0] * t.shape[1], -1).cuda().requires_grad_() for t in (q, k, v)]
        o = F.attention_mod(*flat, H, F.SeqLayout(B, Sq, Sq, 0, 1), F.SeqLayout(B, Sk, Sk, 0, 1), kv_heads=KV, **{n: _dev(t) for n, t in kw.items()})
        o.backward(do.reshape(B * Sq, -1).cuda())
        _within(name + " o", o, *want["o"])
        for n, t in zip(("dq", "dk", "dv"), flat):
            _within(f"{name} {n}", t.grad, *want[n])


def test_attention_mod_table_entries_that_hide_their_distance():
    F = _f()
    g = torch.Generator().manual_seed(1)
    for dt, low in ((BF, -math.inf), (BF, torch.finfo(BF).min), (HF, torch.finfo(HF).min), (F32, torch.finfo(F32).min)):
        x = HF if dt == HF else BF
        q, k, v, do = (torch.randn(1, 90, 2, 64, generator=g).to(x) for _ in range(4))
        bias = torch.randn(2, 41, generator=g).to(dt)
        bias[0, :15] = low         # a window of five keys back
        bias[1] = low              # nothing left for head 1
        want = ref.attention(q, k, v, 0.125, x, causal=True, bias=bias, do=do)
        flat = [t.reshape(90, -1).cuda().requires_grad_() for t in (q, k, v)]
        bd = bias.cuda().requires_grad_()
        lay = F.SeqLayout(1, 90, 90, 0, 1)
        o = F.attention_mod(*flat, 2, lay, lay, causal=True, bias=bd)
        o.backward(do.reshape(90, -1).cuda())
        _within("o", o, *want["o"])
        assert (o.view(90, 2, 64)[:, 1] == 0).all()
        for n, t in zip(("dq", "dk", "dv"), flat):
            _within(n, t.grad, *want[n])
        _within("dbias", bd.grad, *want["dbias"])


def test_attention_mod_strided_layouts_and_uncovered_rows():
    """Frames of a video as sequences (row stride HW), operands as column blocks of one wide matrix, and rows that no sequence owns."""
    F = _f()
    g = torch.Generator().manual_seed(2)
    Fr, HW, H, D = 7, 6, 2, 64
    wide = torch.randn(Fr * HW + 3, 3 * H * D, generator=g).to(BF)
    do = torch.randn(Fr * HW + 3, H * D, generator=g).to(BF)
    x = wide.cuda().requires_grad_()
    lay = F.SeqLayout(HW, Fr, Fr * HW, 1, HW, HW)         # batch = pixel, position = frame
    o = F.attention_mod(x[:, :128], x[:, 128:256], x[:, 256:], H, lay, lay, causal=True, softcap=4.0)
    o.backward(do.cuda())
    n = Fr * HW
    pick = lambda t, c: t[:n, c * 128:(c + 1) * 128].reshape(Fr, HW, H, D).transpose(0, 1)  # noqa: E731
    want = ref.attention(pick(wide, 0), pick(wide, 1), pick(wide, 2), 0.125, BF, causal=True, softcap=4.0, do=pick(do, 0))
    back = lambda t: t.detach().cpu()[:n].reshape(Fr, HW, H, D).transpose(0, 1)  # noqa: E731
    _within("o", back(o), *want["o"])
    assert (o[n:] == 0).all() and (x.grad[n:] == 0).all()
    for c, name in enumerate(("dq", "dk", "dv")):
        _within(name, back(x.grad[:, c * 128:(c + 1) * 128]), *want[name])


@pytest.mark.parametrize("dt", [BF, HF])
def test_attention_mod_shared_keys_get_the_sum_of_their_gradients(dt):
    """Text states shared by the frames of a video (lo = 0): three frames each for two videos."""
    F = _f()
    g = torch.Generator().manual_seed(4)
    q, do = torch.randn(6, 40, 4, 64, generator=g).to(dt), torch.randn(6, 40, 4, 64, generator=g).to(dt)
    k, v = torch.randn(2, 21, 2, 64, generator=g).to(dt), torch.randn(2, 21, 2, 64, generator=g).to(dt)
    want = ref.attention(q, k.repeat_interleave(3, 0), v.repeat_interleave(3, 0), 0.125, dt, softcap=3.0, do=do)
    flat = [t.reshape(t.shape[0] * t.shape[1], -1).cuda().requires_grad_() for t in (q, k, v)]
    o = F.attention_mod(*flat, 4, F.SeqLayout(6, 40, 40, 0, 1), F.SeqLayout(6, 21, 21, 0, 1, 3), kv_heads=2, softcap=3.0)
    o.backward(do.reshape(240, -1).cuda())
    _within("o", o, *want["o"])
    _within("dq", flat[0].grad, *want["dq"])
    for n, t in zip(("dk", "dv"), flat[1:]):
        _within(n, t.grad, *(w.view(2, 3, 21, 2, 64).sum(1) for w in want[n]))


@pytest.mark.parametrize("mask", ["lengths", "documents", "prefix per query", "documents, long"])
def test_attention_mod_keys_shared_by_uneven_groups_under_masks(mask):
    """Five batches, three to a K / V: the second group has two.  Each batch has masks of its own over the shared keys."""
    F = _f()
    g = torch.Generator().manual_seed(len(mask))
    B, Sq, Sk, H, KV, D = 5, 50, 90, 2, 1, 72
    if mask.endswith("long"):
        Sq, Sk, H = 700, 333, 4
    r = lambda *s: torch.randn(*s, generator=g).to(BF)  # noqa: E731
    q, do, k, v = r(B, Sq, H, D), r(B, Sq, H, D), r(2, Sk, KV, D), r(2, Sk, KV, D)
    kw = dict(causal=True)
    if mask == "lengths":
        kw["kv_len"] = torch.tensor([90, 0, 17, 64, 65], dtype=torch.int32)
    elif mask == "prefix per query":
        kw["prefix"] = torch.randint(0, Sk + 20, (B, Sq), generator=g).int()
    else:
        kw["q_docs"], kw["kv_docs"] = (torch.randint(-1, 3, (B, n), generator=g).int() for n in (Sq, Sk))
    at = torch.tensor([0, 0, 0, 1, 1])
    want = ref.attention(q, k[at], v[at], D ** -0.5, BF, do=do, **kw)
    flat = [t.reshape(t.shape[0] * t.shape[1], -1).cuda().requires_grad_() for t in (q, k, v)]
    o = F.attention_mod(*flat, H, F.SeqLayout(B, Sq, Sq, 0, 1), F.SeqLayout(B, Sk, Sk, 0, 1, 3), kv_heads=KV, **{n: _dev(t) for n, t in kw.items()})
    o.backward(do.reshape(B * Sq, -1).cuda())
    _within("o", o, *want["o"])
    _within("dq", flat[0].grad, *want["dq"])
    for n, t in zip(("dk", "dv"), flat[1:]):
        _within(n, t.grad, *(torch.stack([w[at == i].sum(0) for i in (0, 1)]) for w in want[n]))


def test_gradients_of_gradients_are_refused():
    F = _f()
    x = torch.randn(16, 64, device="cuda").to(BF).requires_grad_()
    lay, pos = F.SeqLayout(1, 16, 16, 0, 1), torch.arange(16, dtype=torch.int32, device="cuda")[:, None]
    for y in (F.rope(x, 1, pos, F.RopeAxes((64,))), F.qk_norm_rope(x, x, 1, 1, pos, F.RopeAxes((64,)))[0], F.attention_mod(x, x, x, 1, lay, lay)):
        up = torch.ones_like(y, requires_grad=True)
        gx, = torch.autograd.grad(y, x, up, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            gx.float().sum().backward()


def test_attention_mod_of_nothing():
    F = _f()
    e, k = torch.empty(0, 128, dtype=BF, device="cuda"), torch.randn(8, 128, device="cuda").to(BF)
    assert F.attention_mod(e, k, k, 2, F.SeqLayout(1, 0, 0, 0, 1), F.SeqLayout(1, 8, 8, 0, 1)).shape == (0, 128)
    q = torch.randn(4, 128, device="cuda").to(BF).requires_grad_()
    kk = e.clone().requires_grad_()
    o = F.attention_mod(q, kk, kk, 2, F.SeqLayout(1, 4, 4, 0, 1), F.SeqLayout(1, 0, 0, 0, 1))
    o.sum().backward()
    assert (o == 0).all() and (q.grad == 0).all() and kk.grad.shape == (0, 128)
    # every sequence has no keys
    o = F.attention_mod(q, k, k, 2, F.SeqLayout(2, 2, 2, 0, 1), F.SeqLayout(2, 4, 4, 0, 1), kv_len=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert (o == 0).all()


def test_attention_mod_gradient_against_differences():
    F = _f()
    g = torch.Generator().manual_seed(9)
    H, S = 2, 24
    leaves = [torch.randn(S, H * 64, generator=g).to(HF).cuda().requires_grad_() for _ in range(3)]
    bias = torch.randn(H, 9, generator=g).cuda().requires_grad_()
    up = torch.randn(S, H * 64, generator=g).to(HF).cuda()
    lay = F.SeqLayout(1, S, S, 0, 1)
    f = lambda: (F.attention_mod(*leaves, H, lay, lay, causal=True, softcap=3.0, bias=bias).double() * up.double()).sum()  # noqa: E731
    f().backward()
    for t in leaves + [bias]:
        d = torch.randn(t.shape, generator=g).to(t.dtype).cuda()
        d = d / d.double().norm().to(t.dtype)
        h = 0.25
        with torch.no_grad():
            t0 = t.detach().clone()
            t.copy_(t0 + h * d)
            hi, step = f().item(), (t.double() - t0.double())
            t.copy_(t0 - h * d)
            lo, back = f().item(), (t0.double() - t.double())
            t.copy_(t0)
        want = (t.grad.double() * (step + back)).sum().item() / 2
        # half steps of fp16 in some thousand outputs of size ~1 add up like their root (2^-11 * 60 = 0.03); the curvature adds O(h^3)
        assert abs((hi - lo) / 2 - want) < 0.06 + 0.05 * abs(want), (hi, lo, want)


# ------------------------------------------------------------------------------------------------ use
def _block(F, x, w, heads, kv, pos, axes, lay, docs, pq=None):
    """norm + rotation of the projected rows, then attention: the two calls of a transformer block."""
    qkv = F.conv_linear(x, w)
    D = 64
    q, k, v = qkv[:, :heads * D], qkv[:, heads * D:(heads + kv) * D], qkv[:, (heads + kv) * D:]
    q, k = F.qk_norm_rope(q, k, heads, kv, pos, axes, *(pq or ()))
    return F.attention_mod(q, k, v, heads, lay, lay, kv_heads=kv, q_docs=docs, kv_docs=docs, softcap=20.0)


def test_block_of_packed_clips_matches_the_clips_one_by_one():
    F = _f()
    g = torch.Generator().manual_seed(11)
    heads, kv, C = 4, 2, 256
    sizes = [(3, 5, 7), (2, 4, 4), (1, 9, 6)]
    w = (torch.randn((heads + 2 * kv) * 64, C, generator=g) * C ** -0.5).cuda().requires_grad_()
    pq = [(1 + 0.1 * torch.randn(64, generator=g)).cuda().requires_grad_() for _ in range(2)]
    axes = F.RopeAxes((16, 24, 24))
    xs, ps = [], []
    for t, h, ww in sizes:
        xs.append(torch.randn(t * h * ww, C, generator=g).to(BF).cuda())
        ps.append(torch.stack(torch.meshgrid(torch.arange(t), torch.arange(h), torch.arange(ww), indexing="ij"), -1).reshape(-1, 3).int().cuda())
    n = sum(len(x) for x in xs)
    docs = torch.cat([torch.full((len(x),), i, dtype=torch.int32) for i, x in enumerate(xs)])[None].cuda()
    up = torch.randn(n, heads * 64, generator=g).to(BF).cuda()
    o = _block(F, torch.cat(xs), w, heads, kv, torch.cat(ps), axes, F.SeqLayout(1, n, n, 0, 1), docs, pq)
    o.backward(up)
    packed = [o.detach().float()] + [t.grad.clone() for t in (w, *pq)]
    for t in (w, *pq):
        t.grad = None
    at, single = 0, []
    for x, p in zip(xs, ps):
        s = _block(F, x, w, heads, kv, p, axes, F.SeqLayout(1, len(x), len(x), 0, 1), None, pq)
        s.backward(up[at:at + len(x)])
        single.append(s.detach().float())
        at += len(x)
    for a, b in zip(packed, [torch.cat(single)] + [t.grad for t in (w, *pq)]):
        # both sides round the same values at the same places; only the order of fp32 sums (and a step of bf16 where it tips one) differs
        assert float((a - b).norm() / b.norm()) < 4e-3


def test_steps_over_a_growing_cache_match_the_whole_sequence():
    F = _f()
    g = torch.Generator().manual_seed(12)
    H, KV, D, S, n0 = 8, 2, 128, 200, 150
    q, k, v = torch.randn(S, H * D, generator=g).to(BF).cuda(), torch.randn(S, KV * D, generator=g).to(BF).cuda(), torch.randn(S, KV * D, generator=g).to(BF).cuda()
    slopes = (2.0 ** -torch.arange(1, H + 1).float()).cuda()
    axes = F.RopeAxes((128,), style="half")
    pos = torch.arange(S, device="cuda").view(S, 1)
    with torch.no_grad():
        qr, kr = F.qk_norm_rope(q, k, H, KV, pos, axes)
        lay = F.SeqLayout(1, S, S, 0, 1)
        whole = F.attention_mod(qr, kr, v, H, lay, lay, kv_heads=KV, causal=True, slopes=slopes)
        kc, vc = torch.full((S, KV * D), math.nan, dtype=BF, device="cuda"), torch.full((S, KV * D), math.inf, dtype=BF, device="cuda")
        kc[:n0], vc[:n0] = kr[:n0], v[:n0]
        for i in range(n0, S):
            a, b = F.qk_norm_rope(q[i:i + 1], k[i:i + 1], H, KV, pos[i:i + 1], axes)
            kc[i], vc[i] = b[0], v[i]
            o = F.attention_mod(a, kc, vc, H, F.SeqLayout(1, 1, 1, 0, 1), F.SeqLayout(1, S, S, 0, 1), kv_heads=KV, causal=True, slopes=slopes,
                                kv_len=torch.tensor([i + 1], dtype=torch.int32, device="cuda"))
            assert float((o[0].float() - whole[i].float()).norm() / whole[i].float().norm()) < 6e-3


@pytest.mark.parametrize("dim,splits", [(64, False), (128, False), (128, True)])
def test_delta_is_formed_from_more_of_o_than_its_type_holds(dim, splits):
    """Values with a large common part: delta = dO . O is large and cancels against dP.  With q = 0 every P is 2^-6 (2^-12), exactly, so the
    products' fp32 sums, o and its rest (2^-8 of 2^-8), and dS's one rounding are all that dq may be off."""
    F = _f()
    n, rows = (4096, 64) if splits else (64, 64)
    g = torch.Generator().manual_seed(dim + n)
    v, k = 8 + 0.3 * torch.randn(n, dim, generator=g), 1 + torch.randn(n, dim, generator=g)
    do = torch.randn(rows, dim, generator=g)
    k, v, do = (t.to(BF) for t in (k, v, do))
    q = torch.zeros(rows, dim, dtype=BF, device="cuda", requires_grad=True)
    kd, vd = k.cuda(), v.cuda()
    F.attention_mod(q, kd, vd, 1, F.SeqLayout(1, rows, rows, 0, 1), F.SeqLayout(1, n, n, 0, 1)).backward(do.cuda())
    K, V, G = (t.to(F64) for t in (k, v, do))
    dP = G @ V.T
    dS = (dP - dP.mean(1, keepdim=True)) / n
    want = dS @ K * dim ** -0.5
    size = (G.abs() @ V.abs().amax(0).unsqueeze(1))                      # >= sum_d |dO||V|, |dO||O|
    e = 2.0 ** -16 * size + (3 * dim + n // 64) * 2.0 ** -23 * size      # o and its rest; fp32 sums of dP, delta and (over tiles and splits) o
    bound = ((2.0 ** -8 * dS.abs() + (1 + 2.0 ** -8) * e / n) @ K.abs() + n * 2.0 ** -23 * dS.abs() @ K.abs()) * dim ** -0.5 * (1 + 2.0 ** -8)
    _within("dq", q.grad, want, bound + 2.0 ** -8 * want.abs())


def test_captured_steps_replay_with_new_lengths_and_positions():
    F = _f()
    g = torch.Generator().manual_seed(13)
    H, KV, D, B, S = 8, 2, 64, 3, 700
    q, k, v = (torch.randn(n, h * D, generator=g).to(BF).cuda() for n, h in ((B, H), (B * S, KV), (B * S, KV)))
    kv_len, pos = torch.tensor([5, 600, 1], dtype=torch.int32, device="cuda"), torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    axes = F.RopeAxes((64,), style="half")
    docs = torch.zeros(B, 1, dtype=torch.int32, device="cuda"), torch.zeros(B, S, dtype=torch.int32, device="cuda")

    def step():
        a = F.rope(q, H, pos, axes)
        return F.attention_mod(a, k, v, H, F.SeqLayout(B, 1, 1, 0, 1), F.SeqLayout(B, S, S, 0, 1), kv_heads=KV, causal=True, kv_len=kv_len,
                               q_docs=docs[0], kv_docs=docs[1], softcap=30.0)

    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        other = torch.cuda.CUDAGraph()         # a second captured call of another size: its workspace is its own
        with torch.cuda.graph(other):
            out2 = F.attention_mod(q[:1], k[:S], v[:S], H, F.SeqLayout(1, 1, 1, 0, 1), F.SeqLayout(1, S, S, 0, 1), kv_heads=KV)
        for n in range(4):
            kv_len.copy_(torch.tensor([5 + 200 * n, 700 - n, 1 + n], dtype=torch.int32))
            pos.fill_(n * 1000)
            docs[1][:, :n * 3] = -1
            graph.replay()
            other.replay()
            want, want2 = step(), F.attention_mod(q[:1], k[:S], v[:S], H, F.SeqLayout(1, 1, 1, 0, 1), F.SeqLayout(1, S, S, 0, 1), kv_heads=KV)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(out2, want2), n


def test_captured_training_step_replays_bit_equal():
    F = _f()
    g = torch.Generator().manual_seed(14)
    H, S = 4, 150
    x = [torch.randn(S, H * 64, generator=g).to(BF).cuda().requires_grad_() for _ in range(3)]
    bias = torch.randn(H, 17, generator=g).to(BF).cuda().requires_grad_()
    w = [torch.ones(64, device="cuda", requires_grad=True) for _ in range(2)]
    up = torch.randn(S, H * 64, generator=g).to(BF).cuda()
    pos = torch.arange(S, dtype=torch.int32, device="cuda").view(S, 1)
    lay = F.SeqLayout(1, S, S, 0, 1)

    def step():
        a, b = F.qk_norm_rope(x[0], x[1], H, H, pos, F.RopeAxes((64,)), *w)
        o = F.attention_mod(a, b, x[2], H, lay, lay, causal=True, bias=bias)
        return [o.detach()] + list(torch.autograd.grad(o, x + w + [bias], up))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for n in range(3):
        with torch.no_grad():
            x[0].mul_(1.5)
            up.neg_()
        graph.replay()
        got = [t.clone() for t in outs]
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n


def test_a_captured_backward_pass_is_refused_while_an_eager_graph_holds_its_leaves():
    """The leaf's accumulation belongs to the eager graph's stream: refused before it is reached.  Once that graph is gone the same pass is captured."""
    F = _f()
    x = torch.randn(64, 128, device="cuda").to(BF).requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    up, lay = torch.randn(64, 128, device="cuda").to(BF), F.SeqLayout(1, 64, 64, 0, 1)
    pos = torch.arange(64, dtype=torch.int32, device="cuda").view(64, 1)
    calls = {
        "rope": (lambda: F.rope(x, 2, pos, F.RopeAxes((64,))), (x,)),
        "norm": (lambda: F.qk_norm_rope(x, x, 2, 2, pos, F.RopeAxes((64,)), w, w)[0], (x, w)),
        "attention": (lambda: F.attention_mod(x, x, x, 2, lay, lay, causal=True), (x,)),
    }
    for name, (f, leaves) in calls.items():
        eager = f()
        want = [t.clone() for t in torch.autograd.grad(eager, leaves, up, retain_graph=True)]
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="holds one of its leaves"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(f(), leaves, up)
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            f()                                                          # without a backward pass there is nothing to refuse
        del eager
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            first = f()                                                  # (a graph of the capture's own that holds the leaves is no hindrance)
            got = torch.autograd.grad(f(), leaves, up)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), name
        del first


def test_another_stream_than_the_operands_own():
    F = _f()
    g = torch.Generator().manual_seed(15)
    x = torch.randn(300, 3 * 128, generator=g).to(BF).cuda()
    lay = F.SeqLayout(1, 300, 300, 0, 1)
    want = F.attention_mod(x[:, :128], x[:, 128:256], x[:, 256:], 2, lay, lay, softcap=9.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = F.attention_mod(x[:, :128], x[:, 128:256], x[:, 256:], 2, lay, lay, softcap=9.0)
        both = F.rope(got, 2, torch.arange(300, device="cuda").view(300, 1), F.RopeAxes((64,)))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and torch.equal(both, F.rope(want, 2, torch.arange(300, device="cuda").view(300, 1), F.RopeAxes((64,))))


def _train_call(F, S=700, H=4, KV=2, D=72, seed=21):
    """One pass with every kind of saved tensor, as a function of how its gradients are asked for."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda().requires_grad_()  # noqa: E731
    q, k, v, bias = r(S, H * D), r(S, KV * D), r(S, KV * D), r(H, 41)
    w = torch.ones(D, device="cuda", requires_grad=True)
    docs = torch.randint(0, 3, (1, S), generator=g).int().cuda()
    pos = torch.arange(S, dtype=torch.int32, device="cuda").view(S, 1)
    lay = F.SeqLayout(1, S, S, 0, 1)

    def f(q, k, v, bias, w):
        a, b = F.qk_norm_rope(q, k, H, KV, pos, F.RopeAxes((64,), style="half"), w, w)
        return F.attention_mod(F.rope(a, H, pos, F.RopeAxes((32,))), b, v, H, lay, lay, kv_heads=KV, causal=True, bias=bias, q_docs=docs, kv_docs=docs, softcap=9.0)

    return f, (q, k, v, bias, w)


def test_upstream_gradients_of_any_layout():
    F = _f()
    f, leaves = _train_call(F)
    for up in (torch.ones(1, 288, device="cuda").to(BF).expand(700, 288), torch.randn(288, 700, device="cuda").to(BF).t(),
               torch.randn(700, 300, device="cuda").to(BF)[:, 5:293], torch.randn(700, 320, device="cuda").to(BF)[:, 8:296]):
        got = torch.autograd.grad(f(*leaves), leaves, up)
        want = torch.autograd.grad(f(*leaves), leaves, up.contiguous().clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # the rotary calls alone, one side's upstream gradient dense and the other's a slice
    x, w = torch.randn(300, 256, device="cuda").to(BF).requires_grad_(), torch.rand(64, device="cuda").requires_grad_()
    pos = torch.arange(300, dtype=torch.int32, device="cuda").view(300, 1)
    wide, dense = torch.randn(300, 400, device="cuda").to(BF)[:, 16:144], torch.randn(300, 128, device="cuda").to(BF)
    for ups in ((wide, dense), (dense, wide), (wide, wide)):
        call = lambda: F.qk_norm_rope(x[:, :128], x[:, 128:], 2, 2, pos, F.RopeAxes((64,)), w, w)  # noqa: E731
        got = torch.autograd.grad(call(), (x, w), ups)
        want = torch.autograd.grad(call(), (x, w), [u.contiguous().clone() for u in ups])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got, want = (torch.autograd.grad(F.rope(x[:, 128:], 2, pos, F.RopeAxes((64,))), x, u)[0] for u in (wide, wide.contiguous().clone()))
    assert torch.equal(got, want)


def test_saved_tensors_may_travel_and_calls_may_be_recomputed():
    """Saved tensors moved to the host and back, and a recomputed forward pass, give the bits of the plain pass."""
    F = _f()
    f, leaves = _train_call(F)
    up = torch.randn(700, 288, device="cuda").to(BF)
    want = torch.autograd.grad(f(*leaves), leaves, up)
    with torch.autograd.graph.save_on_cpu():
        o = f(*leaves)
    got = torch.autograd.grad(o, leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = torch.utils.checkpoint.checkpoint(f, *leaves, use_reentrant=False)
    got = torch.autograd.grad(again, leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # slices of one matrix come back with other strides
    x = torch.randn(200, 640, device="cuda").to(BF).requires_grad_()
    lay, pos = F.SeqLayout(2, 100, 100, 0, 1), torch.arange(200, dtype=torch.int32, device="cuda").view(200, 1)
    up = torch.randn(200, 256, device="cuda").to(BF)

    def g(x):
        o = F.attention_mod(x[:, :256], x[:, 256:384], x[:, 384:512], 4, lay, lay, kv_heads=2, causal=True)
        return o + F.qk_norm_rope(x[:, 256:512], x[:, 512:], 4, 2, pos, F.RopeAxes((64,)))[0]

    want, = torch.autograd.grad(g(x), x, up)
    with torch.autograd.graph.save_on_cpu():
        o = g(x)
    got, = torch.autograd.grad(o, x, up)
    assert torch.equal(got, want)


def test_parameters_of_other_types_and_gradients_of_some_inputs_only():
    F = _f()
    x = torch.randn(130, 256, device="cuda").to(BF).requires_grad_()
    pos, axes = torch.arange(130, dtype=torch.int32, device="cuda").view(130, 1), F.RopeAxes((32,))
    w32 = torch.rand(128, device="cuda").to(BF).float()
    ups = [torch.randn(130, 128, device="cuda").to(BF) for _ in range(2)]

    def grads(w, b, wrt):
        return torch.autograd.grad(F.qk_norm_rope(x[:, :128], x[:, 128:], 2, 2, pos, axes, w, None, None, b, norm="layer"), wrt, ups)

    w, b = w32[:64].clone().requires_grad_(), w32[64:].clone().requires_grad_()
    want = grads(w, b, (x, w, b))
    for dt in (BF, torch.float64):                                       # (values of bf16: fp32 holds them too)
        v, c = w.detach().to(dt).requires_grad_(), b.detach().to(dt).requires_grad_()
        got = grads(v, c, (x, v, c))
        assert torch.equal(got[0], want[0]) and all(g.dtype == dt and torch.equal(g, u.to(dt)) for g, u in zip(got[1:], want[1:]))
    two = torch.stack([w32[:64], w32[64:]], 1).requires_grad_()           # columns of a matrix
    got = grads(two[:, 0], two[:, 1], (x, two))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], torch.stack(want[1:], 1))
    assert torch.equal(grads(w, b.detach(), (w,))[0], want[1]) and torch.equal(grads(w.detach(), b, (b,))[0], want[2])
    f, leaves = _train_call(F, S=150)
    up = torch.randn(150, 288, device="cuda").to(BF)
    want = torch.autograd.grad(f(*leaves), leaves, up)
    for n in range(5):
        only = [t if i == n else t.detach() for i, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(f(*only), only[n], up)[0], want[n]), n


def test_sequences_across_the_rows():
    """Temporal layouts: sequence b = (clip, pixel), its rows a frame apart; keys of every second frame only."""
    F = _f()
    C, T, P, H, D = 2, 7, 9, 2, 64
    q, k, v = (torch.randn(C * T * P, H * D, device="cuda").to(BF).requires_grad_() for _ in range(3))
    up = torch.randn(C * T * P, H * D, device="cuda").to(BF)
    o = F.attention_mod(q, k, v, H, F.SeqLayout(C * P, T, T * P, 1, P, P), F.SeqLayout(C * P, 4, T * P, 1, 2 * P, P), causal=True, softcap=5.0)
    got = torch.autograd.grad(o, (q, k, v), up)
    turn = lambda t: t.detach().view(C, T, P, H * D).transpose(1, 2).reshape(C * P * T, H * D).contiguous()  # noqa: E731
    qs, us = turn(q).requires_grad_(), turn(up)
    ks, vs = (turn(t).view(C * P, T, H * D)[:, ::2].reshape(-1, H * D).contiguous().requires_grad_() for t in (k, v))
    p = F.attention_mod(qs, ks, vs, H, F.SeqLayout(C * P, T, T, 0, 1), F.SeqLayout(C * P, 4, 4, 0, 1), causal=True, softcap=5.0)
    want = torch.autograd.grad(p, (qs, ks, vs), us)
    assert torch.equal(turn(o), p) and torch.equal(turn(got[0]), want[0])
    for a, b in zip(got[1:], want[1:]):
        a = turn(a).view(C * P, T, H * D)
        assert torch.equal(a[:, ::2].reshape(-1, H * D), b) and (a[:, 1::2] == 0).all()


def test_two_calls_at_once():
    """Passes with workspaces of their own on two streams, interleaved."""
    F = _f()
    jobs = [_train_call(F, seed=n) for n in (31, 32)]
    up = torch.randn(700, 288, device="cuda").to(BF)
    want = [torch.autograd.grad(f(*leaves), leaves, up) for f, leaves in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for n, ((f, leaves), s) in enumerate(zip(jobs, streams)):
            with torch.cuda.stream(s):
                got[n] = torch.autograd.grad(f(*leaves), leaves, up)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_keys_that_all_batches_read():
    """A key layout that names the same rows for every batch is read, but has no gradients of its own."""
    F = _f()
    q, k = torch.randn(40, 128, device="cuda").to(BF), torch.randn(33, 128, device="cuda").to(BF)
    lay = F.SeqLayout(4, 10, 10, 0, 1)
    a = F.attention_mod(q, k, k, 2, lay, F.SeqLayout(4, 33, 0, 0, 1))
    b = F.attention_mod(q, k.repeat(4, 1), k.repeat(4, 1), 2, lay, F.SeqLayout(4, 33, 33, 0, 1))
    assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """The last sequences of a cache of more than 2^31 elements (and more than 4 GiB) per operand."""
    F = _f()
    H, D, S, B = 2, 128, 8192, 1100                 # B * S * H * D = 2.3e9 elements
    k = torch.zeros(B * S, H * D, dtype=BF, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(16)
    k[-S:] = torch.randn(S, H * D, generator=g, device="cuda").to(BF)
    q = torch.randn(B, H * D, generator=g, device="cuda").to(BF)
    with torch.no_grad():
        o = F.attention_mod(q, k, k, H, F.SeqLayout(B, 1, 1, 0, 1), F.SeqLayout(B, S, S, 0, 1))
        one = F.attention_mod(q[-1:], k[-S:], k[-S:], H, F.SeqLayout(1, 1, 1, 0, 1), F.SeqLayout(1, S, S, 0, 1))
    assert (o[:-1] == 0).all() and o[-1].abs().max() > 0
    assert float((o[-1].float() - one[0].float()).norm() / one.float().norm()) < 6e-3
    del o, one
    with torch.no_grad():
        y = F.rope(k, H, torch.zeros(1, 1, dtype=torch.int32, device="cuda").expand(B * S, 1).contiguous(), F.RopeAxes((128,)))
        assert torch.equal(y[-S:], k[-S:]) and (y[:1000] == 0).all()


def test_refusals():
    F = _f()
    x = torch.zeros(16, 128, dtype=BF, device="cuda")
    lay = F.SeqLayout(1, 16, 16, 0, 1)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    pos = i32(16, 1)
    bad = [
        lambda: F.rope(x.double(), 2, pos, F.RopeAxes((64,))),
        lambda: F.rope(x.t(), 2, pos, F.RopeAxes((64,))),
        lambda: F.rope(x, 3, pos, F.RopeAxes((64,))),
        lambda: F.rope(x, 2, pos, F.RopeAxes((128,))),
        lambda: F.rope(x, 2, pos, F.RopeAxes((12,))),
        lambda: F.rope(x, 2, pos, F.RopeAxes((7, 9))),
        lambda: F.rope(x, 2, pos, F.RopeAxes((64,), style="quarter")),
        lambda: F.rope(x, 2, pos, F.RopeAxes((64,), theta=-1.0)),
        lambda: F.rope(x, 2, pos, F.RopeAxes((64,), scale=(1.0, 2.0))),
        lambda: F.rope(x, 2, pos[:15], F.RopeAxes((64,))),
        lambda: F.rope(x, 2, pos, F.RopeAxes((32, 32))),
        lambda: F.rope(x, 2, pos.double(), F.RopeAxes((64,))),
        lambda: F.rope(x, 2, pos.cpu(), F.RopeAxes((64,))),
        lambda: F.rope(x, 2, pos, None),
        lambda: F.rope(x, 2, pos, F.RopeAxes((64,)), freqs=torch.zeros(31, dtype=F64, device="cuda")),
        lambda: F.rope(x[:, 4:68], 1, pos, F.RopeAxes((64,))),                                  # rows not 16-byte aligned
        lambda: F.rope(torch.zeros(16, 12, dtype=BF, device="cuda"), 1, pos, F.RopeAxes((8,))),   # head dim 12
        lambda: F.rope(x, 2, pos.float().requires_grad_(), F.RopeAxes((64,))),
        lambda: F.rope(x, 2, pos, F.RopeAxes((64,)), freqs=torch.ones(32, dtype=F64, device="cuda", requires_grad=True)),
        lambda: F.qk_norm_rope(x, x.half(), 2, 2, pos, F.RopeAxes((64,))),
        lambda: F.qk_norm_rope(x, x[:8], 2, 2, pos, F.RopeAxes((64,))),
        lambda: F.qk_norm_rope(x, x, 2, 4, pos, F.RopeAxes((64,))),
        lambda: F.qk_norm_rope(x, x, 2, 2, pos, F.RopeAxes((64,)), norm="batch"),
        lambda: F.qk_norm_rope(x, x, 2, 2, pos, F.RopeAxes((64,)), eps=-1.0),
        lambda: F.qk_norm_rope(x, x, 2, 2, pos, F.RopeAxes((64,)), torch.ones(128, device="cuda")),
        lambda: F.qk_norm_rope(x, x, 2, 2, pos, F.RopeAxes((64,)), torch.ones(64)),
        lambda: F.attention_mod(x.float(), x.float(), x.float(), 2, lay, lay),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, kv_heads=3),
        lambda: F.attention_mod(x, x[:, :64], x, 2, lay, lay),
        lambda: F.attention_mod(x, x.half(), x.half(), 2, lay, lay),
        lambda: F.attention_mod(torch.zeros(16, 272, dtype=BF, device="cuda"), *[torch.zeros(16, 272, dtype=BF, device="cuda")] * 2, 2, lay, lay),
        lambda: F.attention_mod(x, x, x, 2, lay, F.SeqLayout(2, 8, 8, 0, 1)),
        lambda: F.attention_mod(x, x, x, 2, F.SeqLayout(1, 17, 17, 0, 1), lay),
        lambda: F.attention_mod(x, x, x, 2, lay, F.SeqLayout(1, 17, 17, 0, 1)),
        lambda: F.attention_mod(x, x, x, 2, F.SeqLayout(2, 8, 0, 0, 1), F.SeqLayout(2, 8, 8, 0, 1)),
        lambda: F.attention_mod(x, x.clone().requires_grad_(), x, 2, F.SeqLayout(2, 8, 8, 0, 1), F.SeqLayout(2, 8, 0, 0, 1)),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, softcap=-1.0),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, scale=math.nan),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, scale=0.0),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, softcap=1e9),
        lambda: F.attention_mod(x[:, :0], x[:, :0], x[:, :0], 2, lay, lay),
        lambda: F.attention_mod(x[:, :1], x[:, :1], x[:, :1], 2, lay, lay),
        lambda: F.rope(x[:, :0], 2, pos, F.RopeAxes((64,))),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, prefix=i32(1)),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, causal=True, prefix=i32(2)),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, kv_len=i32(1).long()),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, q_docs=i32(1, 16)),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, q_docs=i32(1, 16), kv_docs=i32(1, 15)),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, q_docs=i32(1, 16), kv_docs=i32(1, 16).cpu()),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, slopes=torch.zeros(3, device="cuda")),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, slopes=torch.zeros(2, device="cuda", requires_grad=True)),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, bias=torch.zeros(2, 4, device="cuda")),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, bias=torch.zeros(2, 2051, device="cuda")),
        lambda: F.attention_mod(x, x, x, 2, lay, lay, bias=torch.zeros(2, 5, device="cuda", dtype=HF)),
        lambda: F.attention_mod(x[:, 4:68], x[:, :64], x[:, :64], 1, lay, lay),
    ]
    for n, f in enumerate(bad):
        with pytest.raises(RuntimeError, match="t2v_amd"):
            f()
            pytest.fail(f"call {n} was not refused")
    torch.cuda.synchronize()
