"""Descriptors, refusals and host rules of the transformer-block operators that need no GPU: the C entry points check before they launch."""
import ctypes as C

import pytest
import torch

import token_ops_ref as ref


def _nv():
    import t2v_amd  # noqa: F401
    import t2v_amd.native as nv
    return nv


def test_descriptor_sizes_match_the_header(tmp_path):
    import os
    import subprocess
    nv = _nv()
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "p.c").write_text('#include <stdio.h>\n#include "t2v_abi.h"\nint main(){ printf("%zu %zu\\n", sizeof(T2VQkRope), sizeof(T2VAttnMod)); return 0; }')
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "p.c"), "-o", str(tmp_path / "p")])
    assert list(map(int, subprocess.check_output([str(tmp_path / "p")]).split())) == [C.sizeof(nv.QkRope), C.sizeof(nv.AttnMod)]


def _mod(**kw):
    nv = _nv()
    a = nv.AttnMod()
    op = lambda: nv.AttnOperand(1 << 20, 128 * 64, 0, 128, 1)  # noqa: E731
    a.nbatch, a.heads, a.kv_heads, a.Sq, a.Sk, a.D, a.scale, a.kv_share = 2, 2, 2, 64, 64, 64, 0.125, 1
    a.q, a.k, a.v, a.o = op(), op(), op(), op()
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("bad", [dict(nbatch=0), dict(heads=3), dict(kv_heads=0), dict(D=60), dict(D=136), dict(dtype=2), dict(softcap=-1.0),
                                 dict(q_docs=256), dict(prefix=256), dict(bias=256, radius=1025), dict(Sq=1 << 26), dict(scale=float("nan")),
                                 dict(scale=0.0), dict(scale=-1.0), dict(softcap=1e5),
                                 dict(o_rest=264), dict(nbatch=1 << 18, Sq=1 << 16), dict(heads=1 << 16, kv_heads=1, Sq=4)])
def test_attention_descriptors_that_are_refused(bad):
    nv = _nv()
    l = nv.lib()
    assert l.t2v_attn_mod_workspace(C.byref(_mod()), 0) >= 0
    a = _mod(**bad)
    assert l.t2v_attn_mod_workspace(C.byref(a), 0) < 0 and l.t2v_last_error()
    assert l.t2v_attn_mod_fwd(C.byref(a), None) == -1
    assert l.t2v_attn_mod_bwd(C.byref(a), None) == -1


def test_attention_operands_and_workspaces_that_are_refused():
    nv = _nv()
    l = nv.lib()
    for field, op in (("q", (0, 0, 0, 128, 1)), ("k", (1 << 20, 0, 0, 129, 1)), ("v", ((1 << 20) + 2, 0, 0, 128, 1)), ("o", (1 << 20, 0, 0, 128, 0))):
        a = _mod()
        setattr(a, field, nv.AttnOperand(*op))
        assert l.t2v_attn_mod_fwd(C.byref(a), None) == -1 and b"operand" in l.t2v_last_error()
    assert l.t2v_attn_mod_bwd(C.byref(_mod()), None) == -1           # no gradients named
    a = _mod(q_docs=256, kv_docs=256)
    need = l.t2v_attn_mod_meta_bytes(C.byref(a))
    assert need > 0 and l.t2v_attn_mod_fwd(C.byref(a), None) == -1 and b"meta" in l.t2v_last_error()
    a.meta, a.meta_bytes = 1 << 20, need - 1
    assert l.t2v_attn_mod_fwd(C.byref(a), None) == -1
    a = _mod(nbatch=1, Sq=1, Sk=4096)                                # few rows, many keys: the keys are split
    need = l.t2v_attn_mod_workspace(C.byref(a), 0)
    assert need > 0 and l.t2v_attn_mod_fwd(C.byref(a), None) == -1 and b"workspace" in l.t2v_last_error()
    a.workspace, a.workspace_bytes = 1 << 20, need - 1
    assert l.t2v_attn_mod_fwd(C.byref(a), None) == -1


@pytest.mark.parametrize("bad", [dict(rows=0), dict(D=12), dict(D=264), dict(dtype=3), dict(norm=3), dict(naxes=5), dict(theta=0.0), dict(pos=None),
                                 dict(ldpos=0), dict(style=2)])
def test_rope_descriptors_that_are_refused(bad):
    nv = _nv()
    d = nv.QkRope()
    d.x[0], d.ldx[0], d.y[0], d.ldy[0], d.heads[0] = 1 << 20, 128, 1 << 20, 128, 2
    d.rows, d.D, d.naxes, d.theta, d.pos, d.ldpos = 4, 64, 1, 10000.0, 1 << 20, 1
    d.dims[0], d.scale[0] = 64, 1.0
    assert nv.lib().t2v_qk_rope_bwd_floats(C.byref(d)) == -1          # no upstream gradient named
    for n, v in bad.items():
        setattr(d, n, v)
    assert nv.lib().t2v_qk_rope_fwd(C.byref(d), None) == -1 and nv.lib().t2v_last_error()


def test_rope_columns_that_are_refused():
    nv = _nv()
    for dims in ((63,), (12,), (64, 8), (-8,)):
        d = nv.QkRope()
        d.x[0], d.ldx[0], d.y[0], d.ldy[0], d.heads[0] = 1 << 20, 128, 1 << 20, 128, 2
        d.rows, d.D, d.naxes, d.theta, d.pos, d.ldpos = 4, 64, len(dims), 10000.0, 1 << 20, 2
        for n, v in enumerate(dims):
            d.dims[n], d.scale[n] = v, 1.0
        assert nv.lib().t2v_qk_rope_fwd(C.byref(d), None) == -1


def test_layout_rules():
    from t2v_amd.functional import SeqLayout
    from t2v_amd.token_ops import _layout_facts
    assert _layout_facts(SeqLayout(2, 8, 8, 0, 1), 16) == (True, True, True)
    assert _layout_facts(SeqLayout(2, 8, 8, 0, 1), 17) == (True, True, False)
    assert _layout_facts(SeqLayout(2, 8, 9, 0, 1), 16)[0] is False
    assert _layout_facts(SeqLayout(6, 7, 42, 1, 6, 6), 42) == (True, True, True)         # frames of pixels
    assert _layout_facts(SeqLayout(6, 8, 8, 0, 1, 3), 16)[:2] == (True, False)            # three batches share their rows
    assert _layout_facts(SeqLayout(2, 8, 7, 0, 1), 16)[1] is False                         # the last row of one is the first of the next
    assert _layout_facts(SeqLayout(0, 8, 8, 0, 1), 0) == (True, True, True)
    assert _layout_facts(SeqLayout(2, 8, -8, 0, 1), 16)[0] is False


def test_cpu_tensors_are_refused():
    import t2v_amd.functional as F
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    lay = F.SeqLayout(1, 4, 4, 0, 1)
    for f in (lambda: F.rope(x, 1, torch.zeros(4, 1), F.RopeAxes((64,))), lambda: F.qk_norm_rope(x, x, 1, 1, None, None),
              lambda: F.attention_mod(x, x, x, 1, lay, lay)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            f()


def test_the_oracle_finds_a_mistake():
    """A wrong mask, a dropped cap or a shifted table leaves the derived bounds by far: they are not so wide that anything passes."""
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(1, 40, 2, 64, generator=g).to(torch.bfloat16) for _ in range(4))
    bias = torch.randn(2, 9, generator=g).to(torch.bfloat16)
    kw = dict(causal=True, softcap=3.0, bias=bias, do=do)
    good = ref.attention(q, k, v, 0.125, torch.bfloat16, **kw)
    for wrong in (dict(causal=False), dict(softcap=0.0), dict(bias=bias.roll(1, 1))):
        other = ref.attention(q, k, v, 0.125, torch.bfloat16, **{**kw, **wrong})
        out = [n for n in ("o", "dq", "dk", "dv", "dbias") if ((good[n][0] - other[n][0]).abs() > good[n][1]).float().mean() > 0.1]
        assert len(out) >= 3 and "o" in out, (wrong, out)
    # and the gradients of the 64-bit form are those of its forward (autograd through an independent softmax)
    Q, K, V = (t.double().squeeze(0).transpose(0, 1).clone().requires_grad_() for t in (q, k, v))
    B = bias.double().requires_grad_()
    gap = torch.arange(40)[None] - torch.arange(40)[:, None]
    t = 3.0 * torch.tanh(Q @ K.transpose(1, 2) * 0.125 / 3.0) + B[:, gap.clamp(-4, 4) + 4]
    o = torch.softmax(t.masked_fill(gap > 0, float("-inf")), -1) @ V
    o.backward(do.double().squeeze(0).transpose(0, 1))
    for n, x in (("o", o), ("dq", Q.grad), ("dk", K.grad), ("dv", V.grad)):
        torch.testing.assert_close(good[n][0][0].transpose(0, 1), x.detach(), rtol=1e-9, atol=1e-9)
    torch.testing.assert_close(good["dbias"][0], B.grad, rtol=1e-9, atol=1e-9)


def test_flat_descriptors_have_the_pointers_where_the_header_has_them():
    import t2v_amd.token_ops as T
    nv = _nv()
    d = T._AttnFlat()
    for n, name in enumerate(("q", "k", "v", "o", "lse", "prefix", "kv_len", "q_docs", "kv_docs", "slopes", "bias", "d_o", "dq", "dk", "dv", "delta",
                              "dbias", "workspace", "meta")):
        setattr(d, name, 100 + n)
    a = nv.AttnMod.from_buffer_copy(d)
    got = [getattr(a, n).ptr if k is nv.AttnOperand else getattr(a, n) for n, k in nv.AttnMod._fields_]
    assert [v for v in got if v and v >= 100] == list(range(100, 119))
    d = T._AttnFlat()
    d.d_o, d.d_o_bstride_hi, d.d_o_bstride_lo, d.d_o_sstride, d.d_o_bdiv, d.dq = 1, 1 << 40, 256, 768, 3, 5
    a = nv.AttnMod.from_buffer_copy(d)
    assert (a.d_o.ptr, a.d_o.bstride_hi, a.d_o.bstride_lo, a.d_o.sstride, a.d_o.bdiv, a.dq.ptr) == (1, 1 << 40, 256, 768, 3, 5)
    d = T._RopeFlat()
    for n, name in enumerate(("x", "ldx", "dy", "lddy", "y", "ldy", "heads", "w", "b", "dw", "db")):
        setattr(d, name + "0", 10 + 2 * n)
        setattr(d, name + "1", 11 + 2 * n)
    a = nv.QkRope.from_buffer_copy(d)
    assert [x for n in ("x", "ldx", "dy", "lddy", "y", "ldy", "heads", "w", "b", "dw", "db") for x in getattr(a, n)] == list(range(10, 32))


def test_plans_hold_no_addresses():
    """A plan is made from shapes, strides, types and flags; the pointers of the call it was made for are not in it."""
    import t2v_amd.token_ops as T
    from t2v_amd.functional import SeqLayout
    nv = _nv()
    sig = lambda *s: (torch.Size(s), (s[-1], 1) if len(s) == 2 else (1,), torch.bfloat16, torch.device("cuda", 0))  # noqa: E731
    i32 = lambda *s: (torch.Size(s), (s[-1], 1) if len(s) == 2 else (1,), torch.int32, torch.device("cuda", 0))  # noqa: E731
    lay = SeqLayout(2, 8, 8, 0, 1)
    p = T._plan_of((sig(16, 128),) * 3 + (2, 2, lay, lay, 0.125, 1, 0.0, i32(2), i32(2), i32(2, 8), i32(2, 8), None, sig(2, 5)))
    a = nv.AttnMod.from_buffer_copy(p.raw)
    assert (a.nbatch, a.heads, a.Sq, a.D, a.causal, a.radius, a.q.sstride, a.o.sstride) == (2, 2, 8, 64, 1, 2, 128, 128)
    assert not any((a.q.ptr, a.k.ptr, a.v.ptr, a.o.ptr, a.lse, a.workspace, a.meta)) and a.kv_docs == 1 and p.meta > 0
    b = nv.AttnMod.from_buffer_copy(p.bwd(True)[0])
    assert b.kv_share == 1 and b.dq.sstride == 128 and not b.dq.ptr and p.bwd(True)[1] > p.bwd(False)[1]
    r = T._rope_plan((sig(16, 128), sig(16, 64)), (2, 1), T.RopeAxes((16, 24), style="half", shared=True, scale=(2.0, 3.0), theta=7.0), "layer", 0.5, i32(16, 2),
                     None, (None,) * 4)
    d = nv.QkRope.from_buffer_copy(r[0])
    assert (list(d.heads), list(d.ldx), list(d.lddy), d.rows, d.D, d.norm, d.eps, d.ldpos, d.pos_type, d.naxes, list(d.dims), list(d.scale), d.theta, d.shared,
            d.style) == ([2, 1], [128, 64], [128, 64], 16, 64, 2, 0.5, 2, 0, 2, [16, 24, 0, 0], [2.0, 3.0, 0.0, 0.0], 7.0, 1, 1)
    assert not any(d.x) and not any(d.y) and not d.pos and r[-1] > 0
