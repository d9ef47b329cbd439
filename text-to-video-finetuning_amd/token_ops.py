"""Operators of transformer blocks over video and text tokens: rotary positions with several axes, the per-head norm of queries
and keys with the rotation in the same pass, and attention with capped scores, distance biases, document and prefix masks.

They work on the token matrices of `functional` ([rows, heads * dim], unit inner stride, any row stride that keeps rows 16-byte
aligned) and are re-exported there.  Every one launches hand-written HIP kernels (csrc/rope.hip, csrc/attn_mod.hip) on the current
stream of its operands' device, forward and backward; nothing falls back to torch math, and a call the kernels do not take raises.

Host side: what a call's arguments look like (shapes, strides, types, flags: never addresses or contents) is checked once and kept as
a plan, the descriptor's bytes with the pointers left open and the sizes of its buffers; a call fills in the pointers, and the entry point works
out the launches again from the descriptor (a search over run lengths in the backward pass: 0.2 ms at 130000 keys of one head).  Small calls are as
long as their host code.

Calls and their backward passes can be captured into a graph; a captured backward pass whose leaves a graph from outside the capture still
holds is refused (see _foreign_leaves).  Neither second derivatives nor forward-mode derivatives exist; both are refused.
"""
import ctypes as C
import functools
import math
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import native as nv

_TYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_NORM = {"rms": 1, "layer": 2}


# --------------------------------------------------------------------------- helpers
def _fail(text):
    raise RuntimeError("t2v_amd: " + text)


def _check_tokens(shape, stride, dtype, dev, name, types):
    if len(shape) != 2 or dtype not in types or (shape[1] > 1 and stride[1] != 1):
        _fail(f"{name} must be a 2-D token matrix with unit inner stride in {[str(x)[6:] for x in types]}, got {tuple(shape)} {dtype} "
              f"strides {stride}")
    if dev.type != "cuda":
        nv.require_cuda(torch.empty(0, device=dev))


def _ld(shape, stride):
    return stride[0] if shape[0] > 1 else shape[1]


def _upstream(dy):
    """A gradient as autograd hands it over (it may be expanded, transposed or a narrow view): rows the kernels can read."""
    if dy.is_contiguous():
        return dy if dy.data_ptr() % 16 == 0 else dy.clone()
    ld = _ld(dy.shape, dy.stride())
    if dy.stride(1) != 1 or dy.data_ptr() % 16 or (ld * dy.element_size()) % 16 or ld < dy.shape[1]:
        return dy.contiguous()
    return dy


def _no_tangents(*tensors):
    """A dual tensor needs no gradient in the sense of the tape: its tangent would be dropped by the launch."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any([t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors]):
        _fail("no forward-mode derivative: pass tensors without a tangent")


def _sig(t):
    """What a plan needs to know of an optional operand."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _flat(cls):
    """A structure laid out like `cls` whose pointers are plain fields: operands become name (the pointer), name_sstride, .., pairs name0 and name1."""
    fields = []
    for name, kind in cls._fields_:
        if kind is nv.AttnOperand:
            fields += [(name if n == "ptr" else f"{name}_{n}", k) for n, k in kind._fields_] + [(name + "_pad", C.c_int)]
        elif isinstance(kind, type) and issubclass(kind, C.Array) and kind._length_ == 2:
            fields += [(name + "0", kind._type_), (name + "1", kind._type_)]
        else:
            fields.append((name, kind))
    flat = type(cls.__name__ + "Flat", (C.Structure,), {"_fields_": fields})
    assert C.sizeof(flat) == C.sizeof(cls)
    return flat


_RopeFlat, _AttnFlat = _flat(nv.QkRope), _flat(nv.AttnMod)
_capturing = torch.cuda.is_current_stream_capturing
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _launch(name, desc, dev):
    """The entry point `name` on the current stream of the operands' device (made the current device where it is not)."""
    index = dev.index
    if index == torch._C._cuda_getDevice():
        rc = getattr(nv.lib(), name)(C.byref(desc), _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            rc = getattr(nv.lib(), name)(C.byref(desc), _raw_stream(index))
    if rc:
        nv.check(rc, name)


def _foreign_leaves(tensors, dev):
    """During a capture: (whether a graph from outside of it holds one of the leaves among `tensors`, what keeps the answer true until the call).

    A leaf's accumulation node belongs to the stream on which the first living graph made it.  A captured backward pass that meets such a node of
    another stream would join that stream to the capture, which ends the process.  Whether somebody holds the node shows by a mark that
    outlives our own reference to it (an entry "t2v_stream" in the node's metadata, which nothing else reads); nodes that a captured call has made carry
    the capture's stream.  torch does not tell the stream of a node that was there before: it counts as foreign even if it is the capture's own, because
    the other guess would end the process."""
    stream, kept, foreign = _raw_stream(dev.index), [], False
    for t in tensors:
        if t is None or not t.requires_grad or not t.is_leaf:
            continue
        node = torch.autograd.graph.get_gradient_edge(t).node
        mark = node.metadata.get("t2v_stream")
        if mark is None:
            node.metadata["t2v_stream"] = "?"
            del node
            node = torch.autograd.graph.get_gradient_edge(t).node
            if node.metadata.pop("t2v_stream", None) == "?":
                foreign = True
                continue
            node.metadata["t2v_stream"] = stream
        elif mark != stream:
            foreign = True
        kept.append(node)
    return foreign, kept


def _no_foreign_leaves(foreign):
    if foreign and _capturing():
        _fail("a backward pass cannot be captured while a graph from outside of the capture holds one of its leaves (the gradient would go "
              "through that graph's stream): drop that graph, its outputs and losses, first")


def _size(name, *args):
    n = getattr(nv.lib(), name)(*args)
    if n < 0:
        nv.check(int(n), name)
    return int(n)


# --------------------------------------------------------------------------- rotary positions
@dataclass(frozen=True)
class RopeAxes:
    """Which columns of a head turn, by which coordinate, how fast.

    dims: columns per axis, in order (time, height, width, ...; even numbers, at most four axes, their sum a multiple of 8 and at
    most the head dim; columns behind them pass through).  An axis of d columns owns d / 2 pairs; pair i turns by
    pos[axis] * scale[axis] * theta^(-2 i / d), or, with `shared`, by the frequency its number among ALL pairs gives
    (theta^(-2 p / sum(dims)): one ladder, the axes take turns along it).
    style: "interleaved" pairs columns (2p, 2p + 1), "half" pairs (p, p + sum(dims) / 2)."""
    dims: tuple
    theta: float = 10000.0
    style: str = "interleaved"
    shared: bool = False
    scale: tuple = None

    def __post_init__(self):
        object.__setattr__(self, "dims", tuple(int(n) for n in self.dims))
        if self.scale is not None:
            object.__setattr__(self, "scale", tuple(float(s) for s in self.scale))


_SOMEWHERE = 1 << 20            # an aligned address that is never read: sizes are asked for with it


def _vector(t):
    """fp32, dense form of a per-column parameter (checked by the plan)."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.detach().float().contiguous()


def _fixed(pos, freqs):
    if torch.is_grad_enabled() and ((pos is not None and pos.requires_grad) or (freqs is not None and freqs.requires_grad)):
        _fail("positions and frequencies are not trained: pass them detached")


def _addr(t):
    return 0 if t is None else t.data_ptr()


@functools.lru_cache(maxsize=512)
def _rope_plan(xs, heads, axes, norm, eps, pos, freqs, params):
    """xs: one or two operand signatures; params: signatures of (q_weight, k_weight, q_bias, k_bias).  Returns (forward bytes, backward bytes,
    rows, columns of the sides, dtype, device, D, floats of the backward workspace for parameter gradients)."""
    shape, stride, dtype, dev = xs[0]
    for (sh, st, dt, dv), name in zip(xs, ("x",) if len(xs) == 1 else ("q", "k")):
        _check_tokens(sh, st, dt, dv, name, tuple(_TYPE))
    if heads[0] <= 0 or shape[1] % heads[0]:
        _fail(f"{shape[1]} columns are not a multiple of {heads[0]} heads")
    rows, D = shape[0], shape[1] // heads[0]
    if len(xs) == 2:
        sh, st, dt, dv = xs[1]
        if dt != dtype or dv != dev or sh[0] != rows or heads[1] <= 0 or sh[1] != heads[1] * D:
            _fail(f"q {tuple(shape)} {dtype} with {heads[0]} heads and k {tuple(sh)} {dt} with {heads[1]} must have the same rows, type, device and "
                  f"head dim")
    d = _RopeFlat()
    d.heads0, d.heads1, d.rows, d.D, d.dtype, d.eps = heads[0], heads[1], rows, D, _TYPE[dtype], eps
    if norm is not None:
        if norm not in _NORM or not (eps >= 0 and math.isfinite(eps)):
            _fail(f"norm {norm!r}, eps {eps}: 'rms' or 'layer' and a number that is not negative are wanted")
        d.norm = _NORM[norm]
    for t, name in zip(params or (), ("q_weight", "k_weight", "q_bias", "k_bias")):
        if t is not None and (tuple(t[0]) != (D,) or t[3] != dev or not t[2].is_floating_point):
            _fail(f"{name} must be a floating vector of {D} elements on {dev}, got {tuple(t[0])} {t[2]} on {t[3]}")
    if axes is not None:
        dims = axes.dims
        if not 1 <= len(dims) <= 4 or any(n <= 0 or n % 2 for n in dims) or sum(dims) % 8 or sum(dims) > D:
            _fail(f"RopeAxes.dims {axes.dims}: one to four even numbers whose sum is a multiple of 8 and at most the head dim {D}")
        if axes.style not in ("interleaved", "half"):
            _fail(f"RopeAxes.style {axes.style!r}: 'interleaved' or 'half'")
        if not (axes.theta > 0 and math.isfinite(axes.theta)):
            _fail(f"RopeAxes.theta {axes.theta}: a positive number is wanted")
        scale = (1.0,) * len(dims) if axes.scale is None else axes.scale
        if len(scale) != len(dims) or not all(math.isfinite(s) for s in scale):
            _fail(f"RopeAxes.scale {axes.scale}: one finite number per axis")
        d.naxes, d.theta, d.shared, d.style = len(dims), axes.theta, int(axes.shared), int(axes.style == "half")
        for n, (k, s) in enumerate(zip(dims, scale)):
            d.dims[n], d.scale[n] = k, s
        if pos is None or len(pos[0]) != 2 or pos[0][0] != rows or pos[0][1] < len(dims) or pos[2] not in _POS or pos[3] != dev:
            _fail(f"pos must be an int32, int64 or fp32 [{rows}, {len(dims)}] tensor on {dev}, got {None if pos is None else (tuple(pos[0]), *pos[2:])}")
        ld = _ld(pos[0], pos[1])
        if (pos[0][1] > 1 and pos[1][1] != 1) or ld < len(dims):
            _fail(f"pos must have unit inner stride and rows that do not overlap, got strides {pos[1]}")
        d.ldpos, d.pos_type = ld, _POS[pos[2]]
        if freqs is not None and (tuple(freqs[0]) != (sum(dims) // 2,) or freqs[2] != torch.float64 or freqs[3] != dev or
                                  (freqs[0][0] > 1 and freqs[1] != (1,))):
            _fail(f"freqs must be a contiguous fp64 tensor of {sum(dims) // 2} frequencies on {dev}")
    elif pos is not None or freqs is not None:
        _fail("positions need RopeAxes that say what they turn")
    widths = tuple(sh[1] for sh, _, _, _ in xs)
    d.ldx0, d.ldy0, d.lddy0 = _ld(shape, stride), widths[0], widths[0]
    if len(xs) == 2:
        d.ldx1, d.ldy1, d.lddy1 = _ld(xs[1][0], xs[1][1]), widths[1], widths[1]
    floats = 0
    if norm is not None and rows:
        e = _RopeFlat.from_buffer_copy(d)
        for n in ("x0", "x1", "dy0", "dy1", "y0", "y1", "dw0", "pos"):
            setattr(e, n, _SOMEWHERE)
        floats = _size("t2v_qk_rope_bwd_floats", C.byref(e))
    return bytes(d), rows, widths, dtype, dev, D, floats


def _rope_fwd(plan, xs, pos, freqs, ws, bs):
    raw, rows, widths, dtype, dev = plan[:5]
    d = _RopeFlat.from_buffer_copy(raw)
    y = torch.empty((rows, widths[0]), dtype=dtype, device=dev)
    d.x0, d.y0, d.pos, d.freqs = xs[0].data_ptr(), y.data_ptr(), _addr(pos), _addr(freqs)
    ys = (y,)
    if len(xs) == 2:
        y = torch.empty((rows, widths[1]), dtype=dtype, device=dev)
        d.x1, d.y1, d.w0, d.w1, d.b0, d.b1 = xs[1].data_ptr(), y.data_ptr(), _addr(ws[0]), _addr(ws[1]), _addr(bs[0]), _addr(bs[1])
        ys += (y,)
    if rows:
        _launch("t2v_qk_rope_fwd", d, dev)
    return ys


def _rope_bwd(plan, xs, dys, pos, freqs, ws, want):
    """want: (dw0, dw1, db0, db1) wanted, or None.  Returns dxs and the four parameter gradients (fp32 or None)."""
    raw, rows, widths, dtype, dev, D, floats = plan
    d = _RopeFlat.from_buffer_copy(raw)
    dx = torch.empty((rows, widths[0]), dtype=dtype, device=dev)
    d.dy0, d.y0, d.pos, d.freqs = dys[0].data_ptr(), dx.data_ptr(), _addr(pos), _addr(freqs)
    if not dys[0].is_contiguous():
        d.lddy0 = _ld(dys[0].shape, dys[0].stride())
    dxs, grads = (dx,), [None] * 4
    if len(dys) == 2:
        dx = torch.empty((rows, widths[1]), dtype=dtype, device=dev)
        d.dy1, d.y1 = dys[1].data_ptr(), dx.data_ptr()
        if not dys[1].is_contiguous():
            d.lddy1 = _ld(dys[1].shape, dys[1].stride())
        d.x0, d.x1, d.w0, d.w1 = xs[0].data_ptr(), xs[1].data_ptr(), _addr(ws[0]), _addr(ws[1])
        dxs += (dx,)
        if any(want):
            new = torch.empty if rows else torch.zeros
            grads = [new(D, dtype=torch.float32, device=dev) if w else None for w in want]
            work = torch.empty(floats, dtype=torch.float32, device=dev)
            d.dw0, d.dw1, d.db0, d.db1, d.workspace = _addr(grads[0]), _addr(grads[1]), _addr(grads[2]), _addr(grads[3]), work.data_ptr()
    if rows:
        _launch("t2v_qk_rope_bwd", d, dev)
    return dxs, grads


# (The differentiable tensors are the Functions' arguments, the rest travels in one tuple: apply() spends about a microsecond per argument.)
class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rest):
        ctx.plan, pos, freqs, ctx.foreign = rest
        ctx.save_for_backward(pos, freqs)
        return _rope_fwd(ctx.plan, (x,), pos, freqs, None, None)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _no_tangents(dy)
        _no_foreign_leaves(ctx.foreign)
        pos, freqs = ctx.saved_tensors
        return _rope_bwd(ctx.plan, None, (_upstream(dy),), pos, freqs, None, None)[0][0], None


def rope(x, heads, pos, axes, freqs=None):
    """Rotary positions: x [rows, heads * dim] (bf16, fp16 or fp32) with the columns `axes` (RopeAxes) names turned by pos [rows, number
    of axes] (int32, int64 or fp32).  Angles are formed in 64 bits.  freqs: fp64 [sum(dims) / 2] radians per unit of position, in the place of the
    ladder theta gives.  Returns a dense matrix of x's shape; differentiable in x."""
    _no_tangents(x, pos, freqs)
    _fixed(pos, freqs)
    plan = _rope_plan((_sig(x),), (int(heads), 0), axes, None, 0.0, _sig(pos), _sig(freqs), None)
    if torch.is_grad_enabled() and x.requires_grad:
        foreign, _kept = _foreign_leaves((x,), x.device) if _capturing() else (False, None)
        return _Rope.apply(x, (plan, pos, freqs, foreign))
    return _rope_fwd(plan, (x,), pos, freqs, None, None)[0]


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, qb, kb, rest):
        ctx.plan, ctx.key, pos, freqs, ctx.foreign = rest
        ctx.types = [None if t is None else t.dtype for t in (qw, kw, qb, kb)]
        ctx.save_for_backward(q, k, qw, kw, pos, freqs)
        return _rope_fwd(ctx.plan, (q, k), pos, freqs, (_vector(qw), _vector(kw)), (_vector(qb), _vector(kb)))

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        _no_tangents(dq, dk)
        _no_foreign_leaves(ctx.foreign)
        q, k, qw, kw, pos, freqs = ctx.saved_tensors
        plan, sigs = ctx.plan, (_sig(q), _sig(k))
        if sigs != ctx.key[0]:                      # (a saved tensor may come back with other strides)
            plan = _rope_plan(sigs, *ctx.key[1:])
        dxs, grads = _rope_bwd(plan, (q, k), (_upstream(dq), _upstream(dk)), pos, freqs, (_vector(qw), _vector(kw)), ctx.needs_input_grad[2:6])
        return (*dxs, *[g if g is None or g.dtype == t else g.to(t) for g, t in zip(grads, ctx.types)], None)


def qk_norm_rope(q, k, heads, kv_heads, pos, axes, q_weight=None, k_weight=None, q_bias=None, k_bias=None, eps=1e-6, norm="rms",
                 freqs=None):
    """Queries [rows, heads * dim] and keys [rows, kv_heads * dim] normed per head and turned, in one launch: returns (q', k').

    norm: "rms" (x * rsqrt(mean x^2 + eps)) or "layer" (centred first); q_weight, k_weight, q_bias, k_bias: [dim] vectors shared by the
    heads, or None.  pos, axes, freqs: as in `rope`; both None: the norm alone.  Differentiable in q, k and the four vectors; the
    statistics are recomputed in the backward pass from the saved inputs."""
    if norm is None:
        _fail("norm None: 'rms' or 'layer' (`rope` turns without a norm)")
    _no_tangents(q, k, pos, freqs, q_weight, k_weight, q_bias, k_bias)
    _fixed(pos, freqs)
    key = ((_sig(q), _sig(k)), (int(heads), int(kv_heads)), axes, norm, float(eps), _sig(pos), _sig(freqs),
           (_sig(q_weight), _sig(k_weight), _sig(q_bias), _sig(k_bias)))
    plan = _rope_plan(*key)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or
                                    any([t is not None and t.requires_grad for t in (q_weight, k_weight, q_bias, k_bias)])):
        foreign, _kept = _foreign_leaves((q, k, q_weight, k_weight, q_bias, k_bias), q.device) if _capturing() else (False, None)
        return _QkNormRope.apply(q, k, q_weight, k_weight, q_bias, k_bias, (plan, key, pos, freqs, foreign))
    return _rope_fwd(plan, (q, k), pos, freqs, (_vector(q_weight), _vector(k_weight)), (_vector(q_bias), _vector(k_bias)))


# --------------------------------------------------------------------------- attention with modified scores
@functools.lru_cache(maxsize=1024)
def _layout_facts(lay, rows):
    """(inside, own, covered) of a SeqLayout over a matrix of `rows` rows: every row it names exists; no row is named twice; every row is named."""
    if min(lay.nbatch, lay.S, lay.hi, lay.lo, lay.ss) < 0 or lay.bdiv < 1:
        return False, False, False
    if lay.nbatch * lay.S == 0:
        return True, True, rows == 0
    sizes = [(-(-lay.nbatch // lay.bdiv), lay.hi), (min(lay.nbatch, lay.bdiv), lay.lo), (lay.S, lay.ss)]
    last = sum((n - 1) * s for n, s in sizes)
    own, reach = True, 0
    for n, s in sorted((p for p in sizes if p[0] > 1), key=lambda p: p[1]):
        own = own and s > reach
        reach += (n - 1) * s
    return last < rows, own, own and lay.nbatch * lay.S == rows


def _operand(ld, lay):
    """A T2VAttnOperand without its pointer."""
    return nv.AttnOperand(0, lay.hi * ld, lay.lo * ld, lay.ss * ld, lay.bdiv)


def _check_ints(t, shapes, dev, name):
    if t is not None and (t[2] != torch.int32 or tuple(t[0]) not in shapes or t[3] != dev or not _dense(t)):
        _fail(f"{name} must be a contiguous int32 tensor of shape {' or '.join(map(str, shapes))} on {dev}, got {tuple(t[0])} {t[2]} on {t[3]}")


def _dense(t):
    expect = 1
    for n, s in zip(reversed(t[0]), reversed(t[1])):
        if n != 1 and s != expect:
            return False
        expect *= n
    return True


class _AttnPlan:
    """raw: descriptor of the forward; work, meta: bytes of its buffers; bwd: (descriptor, workspace bytes, with dense gradients), made on first use."""
    __slots__ = ("key", "raw", "work", "meta", "empty", "covered", "kv_covered", "share", "dtype", "dev", "lse", "delta", "rest", "shared_ok", "_bwd", "lays")

    def bwd(self, with_bias):
        if self._bwd.get(with_bias) is None:
            qlay, klay, width, kwidth = self.lays
            d = nv.AttnMod.from_buffer_copy(self.raw)
            d.d_o, d.dq, d.dk, d.dv = _operand(width, qlay), _operand(width, qlay), _operand(kwidth, klay), _operand(kwidth, klay)
            d.kv_share = self.share
            e = nv.AttnMod.from_buffer_copy(d)
            for n in ("q", "k", "v", "o"):
                getattr(e, n).ptr = _SOMEWHERE
            e.dbias = _SOMEWHERE if with_bias else None
            _somewhere(e)
            self._bwd[with_bias] = (bytes(d), _size("t2v_attn_mod_workspace", C.byref(e), 1))
        return self._bwd[with_bias]


def _somewhere(e):
    """Pointers that only have to be there: which masks and biases a call has is part of its plan (flagged in the open pointers by 1)."""
    for n in ("prefix", "kv_len", "q_docs", "kv_docs", "slopes", "bias"):
        if getattr(e, n):
            setattr(e, n, _SOMEWHERE)


@functools.lru_cache(maxsize=512)
def _attn_plan(qs, ks, vs, heads, kv_heads, qlay, klay, scale, causal, softcap, prefix, kv_len, q_docs, kv_docs, slopes, bias):
    types = (torch.bfloat16, torch.float16)
    for (sh, st, dt, dv), name in ((qs, "q"), (ks, "k"), (vs, "v")):
        _check_tokens(sh, st, dt, dv, name, types)
    (qsh, qst, dtype, dev), (ksh, kst, _, _), (vsh, vst, _, _) = qs, ks, vs
    if heads <= 0 or qsh[1] % heads:
        _fail(f"q has {qsh[1]} columns: not a multiple of {heads} heads")
    D = qsh[1] // heads
    if kv_heads <= 0 or heads % kv_heads:
        _fail(f"{heads} query heads cannot share {kv_heads} key / value heads evenly")
    if ksh != vsh or ksh[1] != kv_heads * D or not dtype == ks[2] == vs[2] or not dev == ks[3] == vs[3]:
        _fail(f"q {tuple(qsh)} {dtype}, k {tuple(ksh)} {ks[2]}, v {tuple(vsh)} {vs[2]}: one type, one device, {kv_heads} key / value heads of {D} "
              f"columns are wanted")
    if D % 8 or not 8 <= D <= 128:
        _fail(f"attention_mod takes head dims that are multiples of 8 up to 128, got {D}")
    scale = D ** -0.5 if scale is None else scale
    nb, Sq, Sk = qlay.nbatch, qlay.S, klay.S
    qf, kf = _layout_facts(qlay, qsh[0]), _layout_facts(klay, ksh[0])
    if nb != klay.nbatch or not qf[0] or not kf[0]:
        _fail(f"layouts {qlay} over {qsh[0]} rows and {klay} over {ksh[0]} rows: as many batches on both sides, rows that exist")
    if not qf[1]:
        _fail(f"query layout {qlay} names a row twice")
    if not 1e-15 <= scale <= 1e6 or not (softcap == 0.0 or 1e-6 <= softcap <= 1e4):
        _fail(f"softcap {softcap}, scale {scale}: a scale between 1e-15 and 1e6 and a cap of 0 (none) or between 1e-6 and 1e4 are wanted")
    if prefix is not None and not causal:
        _fail("prefix opens a causal mask: pass causal=True with it")
    if (q_docs is None) != (kv_docs is None):
        _fail("q_docs and kv_docs come together")
    _check_ints(prefix, ((nb,), (nb, Sq)), dev, "prefix")
    _check_ints(kv_len, ((nb,),), dev, "kv_len")
    _check_ints(q_docs, ((nb, Sq),), dev, "q_docs")
    _check_ints(kv_docs, ((nb, Sk),), dev, "kv_docs")
    if slopes is not None and (slopes[2] != torch.float32 or tuple(slopes[0]) != (heads,) or slopes[3] != dev or not _dense(slopes)):
        _fail(f"slopes must be a contiguous fp32 tensor of {heads} elements on {dev}")
    if bias is not None and (bias[2] not in (dtype, torch.float32) or len(bias[0]) != 2 or bias[0][0] != heads or bias[0][1] % 2 == 0 or
                             bias[0][1] > 2049 or bias[3] != dev or not _dense(bias)):
        _fail(f"bias must be a contiguous [{heads}, 2R + 1] table with R <= 1024 in {dtype} or fp32 on {dev}, got {tuple(bias[0])} {bias[2]}")
    p = _AttnPlan()
    p.empty = nb * Sq == 0 or Sk == 0                   # nothing is asked, or there is nothing to see
    p.dtype, p.dev, p.delta, p.rest = dtype, dev, nb * heads * Sq, qsh[0] * heads * D * 2    # elements of delta, bytes of o's rest (a multiple of 16)
    p.lse = p.delta * (1 if slopes is None and bias is None else 2)
    p.covered = qf[2]
    p.share = klay.bdiv if klay.bdiv > 1 and klay.lo == 0 else 1
    p.kv_covered = kf[2] or (p.share > 1 and nb % p.share == 0 and nb // p.share * Sk == ksh[0] and klay.ss == 1 and klay.hi == Sk)
    p.shared_ok = kf[1] or (p.share > 1 and klay.ss > 0 and klay.hi >= (Sk - 1) * klay.ss + 1)
    p._bwd, p.lays, p.work, p.meta, p.raw = {}, (qlay, klay, heads * D, kv_heads * D), 0, 0, b""
    if p.empty:
        return p
    a = nv.AttnMod()
    a.nbatch, a.heads, a.kv_heads, a.Sq, a.Sk, a.D = nb, heads, kv_heads, Sq, Sk, D
    a.dtype, a.causal, a.scale, a.softcap = _TYPE[dtype], causal, scale, softcap
    a.q, a.k, a.v, a.o = _operand(_ld(qsh, qst), qlay), _operand(_ld(ksh, kst), klay), _operand(_ld(vsh, vst), klay), _operand(heads * D, qlay)
    a.prefix_per_query = int(prefix is not None and len(prefix[0]) == 2)
    if bias is not None:
        a.bias_f32, a.radius = int(bias[2] == torch.float32), bias[0][1] // 2
    for name, t in (("prefix", prefix), ("kv_len", kv_len), ("q_docs", q_docs), ("kv_docs", kv_docs), ("slopes", slopes), ("bias", bias)):
        setattr(a, name, None if t is None else 1)      # (there: the address comes with the call)
    p.raw = bytes(a)
    for n in ("q", "k", "v", "o"):
        getattr(a, n).ptr = _SOMEWHERE
    _somewhere(a)
    p.work, p.meta = _size("t2v_attn_mod_workspace", C.byref(a), 0), _size("t2v_attn_mod_meta_bytes", C.byref(a))
    return p


def _fill(d, q, k, v, o, prefix, kv_len, q_docs, kv_docs, slopes, bias):
    d.q, d.k, d.v, d.o = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr()
    if prefix is not None:
        d.prefix = prefix.data_ptr()
    if kv_len is not None:
        d.kv_len = kv_len.data_ptr()
    if q_docs is not None:
        d.q_docs, d.kv_docs = q_docs.data_ptr(), kv_docs.data_ptr()
    if slopes is not None:
        d.slopes = slopes.data_ptr()
    if bias is not None:
        d.bias = bias.data_ptr()


def _bytes(n, dev):
    return torch.empty(n, dtype=torch.uint8, device=dev)      # (the caching allocator's blocks are 512-byte aligned)


def _attn_fwd(p, q, k, v, masks, bias, keep):
    """o, and with `keep` what the backward pass wants: what o's rounding left behind with lse behind it, and the tile data of the masks."""
    dev = p.dev
    if p.empty:
        return torch.zeros(q.shape, dtype=p.dtype, device=dev), None, None
    o = (torch.empty if p.covered else torch.zeros)(q.shape, dtype=p.dtype, device=dev)      # rows that no sequence owns: zeros
    d = _AttnFlat.from_buffer_copy(p.raw)
    _fill(d, q, k, v, o, *masks, bias)
    kept = tiles = None
    if keep:
        kept = _bytes(p.rest + 4 * p.lse, dev)
        d.o_rest = at = kept.data_ptr()
        d.lse = at + p.rest
    if p.meta:
        tiles = _bytes(p.meta, dev)
        d.meta, d.meta_bytes = tiles.data_ptr(), p.meta
    if p.work:
        work = _bytes(p.work, dev)
        d.workspace, d.workspace_bytes = work.data_ptr(), p.work
    _launch("t2v_attn_mod_fwd", d, dev)
    return o, kept, tiles


class _AttentionMod(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, rest):
        ctx.plan, masks, ctx.foreign = rest
        o, kept, tiles = _attn_fwd(ctx.plan, q, k, v, masks, bias, True)
        ctx.save_for_backward(q, k, v, bias, o, kept, tiles, *masks)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        _no_tangents(do)
        _no_foreign_leaves(ctx.foreign)
        q, k, v, bias, o, kept, tiles, *masks = ctx.saved_tensors
        p = ctx.plan
        dev, dtype = p.dev, p.dtype
        with_bias = bias is not None and ctx.needs_input_grad[3]
        with_kv = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        if p.empty:
            return (*[torch.zeros(t.shape, dtype=dtype, device=dev) for t in (q, k, v)], torch.zeros_like(bias) if with_bias else None, None)
        if (_sig(q), _sig(k), _sig(v)) != p.key[:3]:            # (a saved tensor may come back with other strides)
            p = _plan_of((_sig(q), _sig(k), _sig(v)) + p.key[3:])
        raw, work_bytes = p.bwd(with_bias)
        dq = (torch.empty if p.covered else torch.zeros)(q.shape, dtype=dtype, device=dev)
        dk = dv = None
        if with_kv:
            new = torch.empty if p.kv_covered else torch.zeros
            dk, dv = new(k.shape, dtype=dtype, device=dev), new(v.shape, dtype=dtype, device=dev)
        do, o = _upstream(do), o.contiguous()
        work = _bytes(work_bytes + 4 * p.delta, dev)            # and delta behind it
        d = _AttnFlat.from_buffer_copy(raw)
        _fill(d, q, k, v, o, *masks, bias)
        d.o_rest = at = kept.data_ptr()
        d.lse = at + p.rest
        d.workspace = at = work.data_ptr()
        d.workspace_bytes, d.delta = work_bytes, at + work_bytes
        d.d_o, d.dq, d.dk, d.dv = do.data_ptr(), dq.data_ptr(), _addr(dk), _addr(dv)
        if not do.is_contiguous():
            ld, lay = _ld(do.shape, do.stride()), p.lays[0]
            d.d_o_bstride_hi, d.d_o_bstride_lo, d.d_o_sstride = lay.hi * ld, lay.lo * ld, lay.ss * ld
        dbias = None
        if with_bias:
            dbias = torch.empty(bias.shape, dtype=bias.dtype, device=dev)
            d.dbias = dbias.data_ptr()
        if tiles is not None:
            d.meta, d.meta_bytes, d.meta_ready = tiles.data_ptr(), tiles.numel(), 1
        _launch("t2v_attn_mod_bwd", d, dev)
        return dq, dk, dv, dbias, None


def _plan_of(key):
    p = _attn_plan(*key)
    p.key = key
    return p


def attention_mod(q, k, v, heads, qlay, klay, kv_heads=None, scale=None, causal=False, prefix=None, kv_len=None, q_docs=None, kv_docs=None,
                  softcap=0.0, slopes=None, bias=None):
    """Attention whose scores may be capped, biased by distance and masked by position and document.

    q: [rows_q, heads * dim]; k, v: [rows_kv, kv_heads * dim] token matrices in bf16 or fp16 (dim a multiple of 8 up to 128; heads a
    multiple of kv_heads, which defaults to heads); qlay, klay: SeqLayout of the sequences.  With t = scale * q.k (scale defaults to
    dim^-0.5):
      softcap > 0    t <- softcap * tanh(t / softcap)                                             (1e-6 to 1e4; scale: 1e-15 to 1e6)
      slopes         fp32 [heads]: t <- t - slopes[h] * |j - i'|                                  (not trained)
      bias           [heads, 2R + 1] (R <= 1024, the operands' type or fp32): t <- t + bias[h, clip(j - i', -R, R) + R]; trained when it
                     requires a gradient; an entry at or below its type's lowest finite value hides its distance (finite ones beyond 2e38
                     count as 2e38; scores are held in 32 bits: beside an entry of 1e6 the rest of a score is rounded to 0.1)
      kv_len         int32 [nbatch]: keys 0 .. kv_len - 1 exist (default: all)
      causal         keys j <= i';  prefix (int32 [nbatch] or [nbatch, Sq], with causal): and all keys j < prefix
      q_docs, kv_docs  int32 [nbatch, Sq], [nbatch, Sk]: only keys of the query's document; numbers below 0 mark padding
    i' = i + kv_len - Sq is the query's place among the keys: the queries are the last positions.  A row that may see nothing is zero.
    Keys and values behind kv_len and of documents below 0 may hold anything; all others must be finite, also where the masks happen to
    leave no query that sees them: masked weights of a tile are exact zeros that multiply its rows.
    Weights and the gradients of scores are rounded once to the operands' type for the matrix cores: in fp16 a score's gradient has that type's range
    (bits are lost below 6e-5, infinite above 65504), so a small loss wants scaling there.
    Few query rows over many keys (serving steps, chunks of new tokens) split the keys over workgroups and join them.
    Returns [rows_q, heads * dim]; rows that no sequence owns are zero.  Differentiable in q, k, v and bias; K / V shared by the bdiv batches
    of a layout with lo = 0 get the sum of their gradients; other layouts that name a key row twice train q and bias alone.  The order of all sums is
    fixed: repeated runs are bit-equal."""
    heads = int(heads)
    _no_tangents(q, k, v, slopes, bias)
    p = _plan_of((_sig(q), _sig(k), _sig(v), heads, heads if kv_heads is None else int(kv_heads), qlay, klay,
                  None if scale is None else float(scale), int(bool(causal)), float(softcap), _sig(prefix), _sig(kv_len),
                  _sig(q_docs), _sig(kv_docs), _sig(slopes), _sig(bias)))
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        _fail("slopes are not trained: pass slopes.detach(), or a bias table for a learned distance bias")
    masks = (prefix, kv_len, q_docs, kv_docs, slopes)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad)):
        if not p.shared_ok and (k.requires_grad or v.requires_grad):
            _fail(f"key layout {klay} names a row twice: gradients are defined for rows of their own, or shared by the bdiv batches (lo = 0)")
        foreign, _kept = _foreign_leaves((q, k, v, bias), p.dev) if _capturing() else (False, None)
        return _AttentionMod.apply(q, k, v, bias, (p, masks, foreign))
    return _attn_fwd(p, q, k, v, masks, bias, False)[0]
