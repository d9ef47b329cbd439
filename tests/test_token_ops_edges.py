"""Refusals and host rules of the transformer-block operators at the edges, without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

BF = torch.bfloat16


def test_tensors_with_a_tangent_are_refused():
    """The kernels have no forward-mode derivative: a tangent must not get lost."""
    import t2v_amd.functional as F
    lay, axes = F.SeqLayout(1, 4, 4, 0, 1), F.RopeAxes((64,))
    x, pos, w = torch.zeros(4, 64, dtype=BF), torch.zeros(4, 1), torch.ones(64)
    with fwd.dual_level():
        d = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [
            lambda: F.rope(d(x), 1, pos, axes),
            lambda: F.rope(x, 1, d(pos), axes),
            lambda: F.qk_norm_rope(x, d(x), 1, 1, pos, axes),
            lambda: F.qk_norm_rope(x, x, 1, 1, pos, axes, w, w, None, d(w)),
            lambda: F.attention_mod(d(x), x, x, 1, lay, lay),
            lambda: F.attention_mod(x, x, d(x), 1, lay, lay),
            lambda: F.attention_mod(x, x, x, 1, lay, lay, slopes=d(torch.zeros(1))),
            lambda: F.attention_mod(x, x, x, 1, lay, lay, bias=d(torch.zeros(1, 3))),
        ]
        for n, f in enumerate(calls):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()
                pytest.fail(f"call {n} was not refused")
        with pytest.raises(RuntimeError, match="ROCm device"):
            F.rope(x, 1, pos, axes)                       # (a level that is open does not matter by itself)


def test_gradients_of_keys_and_values_are_named_together_or_not_at_all():
    import ctypes as C

    from test_token_ops import _mod, _nv
    nv = _nv()
    op = nv.AttnOperand(1 << 20, 128 * 64, 0, 128, 1)
    bwd = nv.lib().t2v_attn_mod_bwd
    for named, word in (((), b"lse and delta"), (("dk",), b"operand dv"), (("dv",), b"operand dk"), (("dk", "dv"), b"lse and delta")):
        a = _mod(d_o=op, dq=op, **{n: op for n in named})
        assert bwd(C.byref(a), None) == -1 and word in nv.lib().t2v_last_error(), named
