"""Calls of the transformer-block operators at the edges of what they document: rows that a sorted work list must not lose, extreme table entries,
large caps, forward-mode derivatives, operands that need no gradient.  Plain 64-bit forms and derived bounds as in tests/token_ops_ref.py."""
import contextlib
import math

import pytest
import torch

import token_ops_ref as ref

pytestmark = pytest.mark.gpu
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def _f():
    import t2v_amd  # noqa: F401
    import t2v_amd.functional as F
    return F


def _within(name, got, want, bound):
    got = got.detach().cpu().to(F64).reshape(want.shape)
    assert torch.isfinite(got).all(), f"{name}: {int((~torch.isfinite(got)).sum())} values are not finite"
    at, inside = float(((got - want).abs() / bound).max()), bool(((got - want).abs() <= bound).all())
    assert inside, f"{name}: {at:.2f} times the bound"


@contextlib.contextmanager
def _empty_is_nan():
    """New tensors start as NaN (bytes: 255), so that what a call leaves unwritten shows."""
    before = torch.are_deterministic_algorithms_enabled(), torch.is_deterministic_algorithms_warn_only_enabled()
    torch.use_deterministic_algorithms(True, warn_only=True)
    try:
        assert torch.empty(8, dtype=BF, device="cuda").isnan().all()
        yield
    finally:
        torch.use_deterministic_algorithms(before[0], warn_only=before[1])


# ------------------------------------------------------------------------------------------------ rows that see nothing, sorted documents
def _falling(n, *runs):
    """Documents of falling number, one run behind the other."""
    return torch.cat([torch.full((c,), len(runs) - k, dtype=torch.int32) for k, c in enumerate(runs)])[None].expand(n, -1).contiguous()


UNSEEN = {  # B, Sq, Sk, H, KV, D, dtype, masks.  Enough workgroups for the sorted work list (rows * heads above 32768)
    "short keys, falling documents": (1, 400, 400, 96, 96, 64, BF, dict(kv_len=[350], q=(50, 350), k=(50, 350))),
    "fewer keys than queries": (1, 400, 330, 96, 96, 72, HF, dict(q=(60, 230, 110), k=(20, 200, 110))),
    "grouped heads, two lengths": (2, 300, 300, 64, 8, 40, BF, dict(kv_len=[300, 170], q=(130, 100, 70), k=(130, 100, 70))),
    "a table": (1, 400, 400, 96, 48, 16, BF, dict(kv_len=[290], q=(100, 60, 240), k=(100, 60, 240), bias=9)),
    "a prefix per query": (1, 512, 512, 80, 80, 24, BF, dict(kv_len=[250], q="rising", k="rising", prefix=True)),
    "no keys": (2, 300, 300, 64, 64, 8, BF, dict(kv_len=[0, 300], q=(100, 200), k=(100, 200))),
}


@pytest.mark.parametrize("name", list(UNSEEN))
def test_rows_that_see_nothing_are_written_under_the_sorted_work_list(name):
    F = _f()
    B, Sq, Sk, H, KV, D, dt, opt = UNSEEN[name]
    assert Sq * H * B > 32768
    g = torch.Generator().manual_seed(len(name))
    r = lambda *s: torch.randn(*s, generator=g).to(dt)  # noqa: E731
    q, k, v, do = r(B, Sq, H, D), r(B, Sk, KV, D), r(B, Sk, KV, D), r(B, Sq, H, D)
    docs = [(torch.arange(n) // 64).int()[None].repeat(B, 1) if opt[s] == "rising" else _falling(B, *opt[s]) for s, n in (("q", Sq), ("k", Sk))]
    kw = dict(causal=True, q_docs=docs[0], kv_docs=docs[1])
    if "kv_len" in opt:
        kw["kv_len"] = torch.tensor(opt["kv_len"], dtype=torch.int32)
    if "bias" in opt:
        kw["bias"] = r(H, 2 * opt["bias"] + 1)
    if "prefix" in opt:
        kw["prefix"] = (10 * (torch.arange(Sq) // 64 % 2 == 0)).int()[None].repeat(B, 1)
    want = ref.attention(q, k, v, D ** -0.5, dt, do=do, **kw)
    flat = [t.reshape(t.shape[0] * t.shape[1], -1).cuda().requires_grad_() for t in (q, k, v)]
    dkw = {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
    if "bias" in dkw:
        dkw["bias"].requires_grad_()
    lays = F.SeqLayout(B, Sq, Sq, 0, 1), F.SeqLayout(B, Sk, Sk, 0, 1)
    with _empty_is_nan():
        o = F.attention_mod(*flat, H, *lays, kv_heads=KV, **dkw)
        o.backward(do.reshape(B * Sq, -1).cuda())
        with torch.no_grad():
            o2 = F.attention_mod(*flat, H, *lays, kv_heads=KV, **dkw)
    none = torch.stack([~ref.visible(Sq, Sk, Sk if "kv_len" not in opt else opt["kv_len"][b], True, kw["prefix"][b] if "prefix" in kw else None,
                                     docs[0][b], docs[1][b]).any(1) for b in range(B)]).view(-1)
    assert none.any()
    for t in (o, o2, flat[0].grad):
        assert (t[none.cuda()] == 0).all()
    _within("o", o, *want["o"])
    _within("o (no grad)", o2, *want["o"])
    for n, t in zip(("dq", "dk", "dv"), flat):
        _within(n, t.grad, *want[n])
    if "bias" in dkw:
        _within("dbias", dkw["bias"].grad, *want["dbias"])


# ------------------------------------------------------------------------------------------------ table entries far outside of the scores
FAR = {  # B, Sq, Sk, H, KV, D, dtype, far entry, table's type, rest.  "away": the documents of rows below 60 and above 89 lie at the other end
    "low, bf16": (1, 150, 150, 2, 2, 64, BF, -1e30, BF, dict(away=True)),
    "low, fp32, groups": (2, 150, 150, 4, 2, 128, BF, -1e30, F32, dict(away=True, softcap=9.0)),
    "low, with slopes": (1, 150, 150, 2, 1, 72, HF, -1e30, F32, dict(away=True, slopes=True)),
    "lowest but one": (1, 150, 150, 2, 2, 64, BF, -3.3e38, F32, dict(away=True)),
    "lowest but one, bf16": (1, 150, 150, 2, 2, 128, BF, -3.3e38, BF, dict(away=True)),
    "high": (1, 150, 150, 2, 2, 64, BF, 1e30, F32, dict(away=True)),
    "highest": (1, 150, 150, 2, 2, 128, BF, 3.3e38, BF, dict(away=True)),
    "a mask of -1e9": (1, 150, 150, 2, 2, 64, BF, -1e9, F32, dict(away=True, zero=True)),
    "a mask of -60000 in fp16": (2, 150, 150, 2, 2, 128, HF, -60000.0, HF, dict(away=True, zero=True)),
    "one far score for all keys": (1, 70, 200, 2, 2, 64, BF, 1e9, F32, dict(all=True, zero=True)),
    "splits": (1, 3, 4000, 4, 2, 64, BF, -1e30, F32, dict(hide=100)),
    "splits, some near": (1, 3, 4000, 4, 2, 128, HF, -1e30, F32, dict(causal=True)),
    "no table: large negative products": (1, 40, 300, 2, 1, 64, BF, None, None, dict(huge=True)),
}


@pytest.mark.parametrize("name", list(FAR))
def test_entries_far_outside_of_the_scores_are_scores(name):
    """Only an entry at or below its type's lowest value hides its distance.  A row whose keys all carry -1e30 (or +1e30) is their mean: at that size a
    score of ordinary size is lost in 64 bits too.  Entries that leave ordinary scores in 64 bits but not in 32 are tested with queries of zero."""
    F = _f()
    B, Sq, Sk, H, KV, D, dt, far, tdt, opt = FAR[name]
    g = torch.Generator().manual_seed(len(name) + D)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, do = r(B, Sq, H, D).to(dt), r(B, Sk, KV, D).to(dt), r(B, Sk, KV, D).to(dt), r(B, Sq, H, D).to(dt)
    kw = dict(causal=opt.get("causal", False), softcap=opt.get("softcap", 0.0))
    if opt.get("zero"):
        q.zero_()
    if opt.get("slopes"):
        kw["slopes"] = 0.1 + 0.2 * torch.rand(H, generator=g)
    if tdt is not None:
        bias = r(H, 9).to(tdt)
        bias[:, 0] = bias[:, -1] = far
        if opt.get("all"):
            bias[:] = far
        kw["bias"] = bias
    if opt.get("away"):
        i = torch.arange(150).int()
        kw["q_docs"] = ((i >= 60).int() + (i >= 90).int())[None].repeat(B, 1)
        kw["kv_docs"] = (2 - kw["q_docs"]).contiguous()
    if "hide" in opt:
        kw["q_docs"], kw["kv_docs"] = torch.zeros(B, Sq, dtype=torch.int32), torch.zeros(B, Sk, dtype=torch.int32)
        kw["kv_docs"][:, -opt["hide"]:] = -1
    if opt.get("huge"):       # every product is -64 * 2^100, below -1e30, exactly: the weights are equal, and scores' gradients times keys cancel to 0
        q[:], k[:] = 2.0 ** 50, -2.0 ** 50
    want = ref.attention(q, k, v, D ** -0.5, dt, do=do, **kw)
    flat = [t.reshape(t.shape[0] * t.shape[1], -1).cuda().requires_grad_() for t in (q, k, v)]
    dkw = {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
    if tdt is not None:
        dkw["bias"].requires_grad_()
    lays = F.SeqLayout(B, Sq, Sq, 0, 1), F.SeqLayout(B, Sk, Sk, 0, 1)
    o = F.attention_mod(*flat, H, *lays, kv_heads=KV, **dkw)
    o.backward(do.reshape(B * Sq, -1).cuda())
    with torch.no_grad():
        o2 = F.attention_mod(*flat, H, *lays, kv_heads=KV, **dkw)
    _within("o", o, *want["o"])
    _within("o (no grad)", o2, *want["o"])
    if opt.get("huge"):
        return                # (the backward pass's fp32 log-sum-exp cannot hold the logarithm of the count beside 2^106: no claim there)
    for n, t in zip(("dq", "dk", "dv"), flat):
        _within(n, t.grad, *want[n])
    if tdt is not None:
        _within("dbias", dkw["bias"].grad, *want["dbias"])


# ------------------------------------------------------------------------------------------------ forward-mode derivatives
def test_tangents_are_refused_forward_and_backward():
    F = _f()
    import torch.autograd.forward_ad as fwd
    x = torch.randn(16, 64, device="cuda").to(BF)
    leaf = x.clone().requires_grad_()
    lay, pos = F.SeqLayout(1, 16, 16, 0, 1), torch.arange(16, dtype=torch.int32, device="cuda")[:, None]
    calls = (lambda t: F.rope(t, 1, pos, F.RopeAxes((64,))), lambda t: F.qk_norm_rope(t, t, 1, 1, pos, F.RopeAxes((64,)))[0],
             lambda t: F.attention_mod(t, t, t, 1, lay, lay))
    for f in calls:
        plain, y = f(x), f(leaf)
        want, = torch.autograd.grad(y, leaf, x, retain_graph=True)
        with fwd.dual_level():
            for t in (x, leaf):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(fwd.make_dual(t, torch.ones_like(t)))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, fwd.make_dual(x, torch.ones_like(x)), retain_graph=True)
            assert torch.equal(f(x), plain) and torch.equal(torch.autograd.grad(y, leaf, x)[0], want)
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))


# ------------------------------------------------------------------------------------------------ operands that need no gradient
def test_parameters_as_slopes_positions_and_frequencies_without_gradients():
    """They are not trained; where nothing is recorded that makes no difference."""
    F = _f()
    x = torch.randn(16, 128, device="cuda").to(BF)
    lay = F.SeqLayout(1, 16, 16, 0, 1)
    pos, fr = torch.arange(16.0, device="cuda")[:, None], torch.rand(32, dtype=F64, device="cuda")
    slopes = torch.tensor([0.5, 0.25], device="cuda")
    P = torch.nn.Parameter
    calls = (lambda s, p, f: F.attention_mod(x, x, x, 2, lay, lay, slopes=s), lambda s, p, f: F.rope(x, 2, p, F.RopeAxes((64,)), freqs=f),
             lambda s, p, f: F.qk_norm_rope(x, x, 2, 2, p, F.RopeAxes((64,)), freqs=f)[1])
    for call in calls:
        want = call(slopes, pos, fr)
        for guard in (torch.no_grad, torch.inference_mode):
            with guard():
                assert torch.equal(call(P(slopes.clone()), P(pos.clone()), P(fr.clone())), want)
        with pytest.raises(RuntimeError, match="not trained"):
            call(P(slopes.clone()), P(pos.clone()), P(fr.clone()))


def test_queries_alone_are_trained_over_keys_that_sequences_share():
    """Key layouts that name a row for several sequences have no gradients of their own; queries and the table do."""
    F = _f()
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    q, up, k, v, bias = r(4 * 70, 256), r(4 * 70, 256), r(48, 128), r(48, 128), r(4, 21)
    lay = F.SeqLayout(4, 70, 70, 0, 1)
    for step in (0, 5):                                                   # one set of keys for all, windows five rows apart
        rows = torch.cat([torch.arange(33) + b * step for b in range(4)]).cuda()
        for with_bias in (False, True):
            def grads(klay, k, v):
                leaves = [t.detach().clone().requires_grad_() for t in ((q, bias) if with_bias else (q,))]
                o = F.attention_mod(leaves[0], k, v, 4, lay, klay, kv_heads=2, softcap=9.0, bias=leaves[1] if with_bias else None)
                return [o] + list(torch.autograd.grad(o, leaves, up))
            got = grads(F.SeqLayout(4, 33, step, 0, 1), k, v)
            want = grads(F.SeqLayout(4, 33, 33, 0, 1), k[rows].contiguous(), v[rows].contiguous())
            full = grads(F.SeqLayout(4, 33, 33, 0, 1), k[rows].contiguous().requires_grad_(), v[rows].contiguous())
            assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(got, want, full))
        with pytest.raises(RuntimeError, match="names a row twice"):
            F.attention_mod(q, k, v.clone().requires_grad_(), 4, lay, F.SeqLayout(4, 33, step, 0, 1), kv_heads=2)


# ------------------------------------------------------------------------------------------------ large caps
@pytest.mark.parametrize("cap", [0.5, 30.0, 100.0, 101.0, 1000.0, 10000.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_capped_scores_lose_nothing_to_a_large_cap(cap, dim):
    """One key, so a row's log-sum-exp is its score.  Up to a cap of 100 the exponential's form is good to 4e-7 of the cap; above, fp32 products
    and a polynomial (six half steps of 2^-24, 4e-7) hold scores below a quarter of the cap, and the exponential's 4e-7 of the cap is 1.7e-6 of the others."""
    F = _f()
    a = torch.logspace(-3, math.log10(6e4), 3000, dtype=F64).to(HF)
    a = torch.cat([-a.flip(0), torch.zeros(1, dtype=HF), a])
    q, k = torch.zeros(len(a), dim, dtype=HF), torch.zeros(1, dim, dtype=HF)
    q[:, 3], k[0, 3] = a, 1.0
    qd = q.cuda().requires_grad_()
    o = F.attention_mod(qd, k.cuda(), k.cuda(), 1, F.SeqLayout(1, len(a), len(a), 0, 1), F.SeqLayout(1, 1, 1, 0, 1), scale=1.0, softcap=cap)
    kept, = [t for t in o.grad_fn.saved_tensors if t is not None and t.dtype == torch.uint8]
    got = kept[o.grad_fn.plan.rest:].view(F32).cpu().to(F64) * math.log(2.0)
    want = cap * torch.tanh(a.to(F64) / cap)
    bound = 4e-7 * cap + 1e-12 if cap <= 100 else 2e-6 * want.abs() + 1e-12
    at, inside = float(((got - want).abs() / bound).max()), bool(((got - want).abs() <= bound).all())
    assert inside, f"{at:.1f} times the bound"


WIDE = {  # B, Sq, Sk, H, KV, D, dtype, factor of the queries, options
    "small scores": (2, 150, 150, 4, 2, 64, HF, 2.0, dict(softcap=10000.0, causal=True)),
    "across the border": (1, 150, 200, 2, 2, 128, HF, 20.0, dict(softcap=101.0)),
    "table": (1, 150, 150, 2, 2, 128, BF, 10.0, dict(softcap=120.0, bias=16, causal=True)),
    "slopes": (1, 150, 150, 4, 2, 72, HF, 10.0, dict(softcap=500.0, slopes=True)),
    "table, 64": (1, 150, 150, 2, 1, 64, BF, 10.0, dict(softcap=300.0, bias=5)),
    "splits": (1, 4, 3000, 4, 2, 128, BF, 10.0, dict(softcap=150.0, causal=True)),
}


@pytest.mark.parametrize("name", list(WIDE))
def test_large_caps_match_the_64_bit_form(name):
    F = _f()
    B, Sq, Sk, H, KV, D, dt, mul, opt = WIDE[name]
    g = torch.Generator().manual_seed(len(name))
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, do = (r(B, Sq, H, D) * mul).to(dt), r(B, Sk, KV, D).to(dt), r(B, Sk, KV, D).to(dt), r(B, Sq, H, D).to(dt)
    kw = dict(causal=opt.get("causal", False), softcap=opt["softcap"])
    if "bias" in opt:
        kw["bias"] = r(H, 2 * opt["bias"] + 1)
    if opt.get("slopes"):
        kw["slopes"] = 0.3 * torch.rand(H, generator=g)
    want = ref.attention(q, k, v, D ** -0.5, dt, do=do, **kw)
    flat = [t.reshape(t.shape[0] * t.shape[1], -1).cuda().requires_grad_() for t in (q, k, v)]
    dkw = {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
    if "bias" in dkw:
        dkw["bias"].requires_grad_()
    o = F.attention_mod(*flat, H, F.SeqLayout(B, Sq, Sq, 0, 1), F.SeqLayout(B, Sk, Sk, 0, 1), kv_heads=KV, **dkw)
    o.backward(do.reshape(B * Sq, -1).cuda())
    _within("o", o, *want["o"])
    for n, t in zip(("dq", "dk", "dv"), flat):
        _within(n, t.grad, *want[n])
    if "bias" in dkw:
        _within("dbias", dkw["bias"].grad, *want["dbias"])
