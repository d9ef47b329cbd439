"""Operators of transformer blocks over video and text tokens: rotary positions with several axes, the per-head norm of queries
and keys with the rotation in the same pass, and attention with capped scores, distance biases, document and prefix masks.

They work on the token matrices of `functional` ([rows, heads * dim], unit inner stride, any row stride that keeps rows 16-byte
aligned) and are re-exported there.  Every one launches hand-written HIP kernels (csrc/rope.hip, csrc/attn_mod.hip) on the current
stream of its operands' device, forward and backward; nothing falls back to torch math, and a call the kernels do not take raises.
"""
import ctypes as C
import functools
import math
import struct
from dataclasses import dataclass

import torch

from . import native as nv

_TYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_NORM = {"rms": 1, "layer": 2}


# --------------------------------------------------------------------------- helpers
def _fail(text):
    raise RuntimeError("t2v_amd: " + text)


def _tokens(t, name, types=(torch.bfloat16, torch.float16, torch.float32)):
    if t.dim() != 2 or t.dtype not in types or (t.shape[1] > 1 and t.stride(1) != 1):
        _fail(f"{name} must be a 2-D token matrix with unit inner stride in {[str(x)[6:] for x in types]}, got {tuple(t.shape)} {t.dtype} "
              f"strides {t.stride()}")
    if not t.is_cuda:
        nv.require_cuda(t)
    return t


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _upstream(dy):
    """A gradient as autograd hands it over (it may be expanded, transposed or a narrow view): rows the kernels can read."""
    if dy.stride(1) != 1 or dy.data_ptr() % 16 or (_ld(dy) * dy.element_size()) % 16 or _ld(dy) < dy.shape[1]:
        return dy.contiguous()
    return dy


def _vector(t, n, dev, name):
    """fp32 copy / view of a per-column parameter."""
    if t is None:
        return None
    if tuple(t.shape) != (n,) or t.device != dev or not t.is_floating_point():
        _fail(f"{name} must be a floating vector of {n} elements on {dev}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    t = t.detach()
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _launch(name, desc, dev):
    """The entry point `name` on the current stream of the operands' device (made the current device where it is not)."""
    index = dev.index
    if index == torch.cuda.current_device():
        rc = getattr(nv.lib(), name)(C.byref(desc), _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            rc = getattr(nv.lib(), name)(C.byref(desc), _raw_stream(index))
    if rc:
        nv.check(rc, name)


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


# T2VQkRope in three pieces, packed in one go (a ctypes structure filled field by field costs several microseconds of a call that takes ten)
_SIDES = struct.Struct("@12Q2i8QQq")        # x, ldx, dy, lddy, y, ldy (both sides each); heads; w, b, dw, db; workspace; rows
_WHERE = struct.Struct("@Qqi")              # pos, ldpos, pos_type


@functools.lru_cache(maxsize=256)
def _rope_fixed(axes, D, dtype, norm, eps):
    """(number of axes, bytes in front of the positions, bytes behind them but for `freqs`): fixed by values, nothing of a call's tensors."""
    d = nv.QkRope()
    d.D, d.dtype, d.norm, d.eps = D, _TYPE[dtype], _NORM[norm] if norm else 0, eps
    if axes is not None:
        dims = tuple(int(n) for n in axes.dims)
        if not 1 <= len(dims) <= 4 or any(n <= 0 or n % 2 for n in dims) or sum(dims) % 8 or sum(dims) > D:
            _fail(f"RopeAxes.dims {axes.dims}: one to four even numbers whose sum is a multiple of 8 and at most the head dim {D}")
        if axes.style not in ("interleaved", "half"):
            _fail(f"RopeAxes.style {axes.style!r}: 'interleaved' or 'half'")
        if not (axes.theta > 0 and math.isfinite(axes.theta)):
            _fail(f"RopeAxes.theta {axes.theta}: a positive number is wanted")
        scale = (1.0,) * len(dims) if axes.scale is None else tuple(float(s) for s in axes.scale)
        if len(scale) != len(dims) or not all(math.isfinite(s) for s in scale):
            _fail(f"RopeAxes.scale {axes.scale}: one finite number per axis")
        d.naxes, d.theta, d.shared, d.style = len(dims), axes.theta, int(axes.shared), int(axes.style == "half")
        for n, (k, s) in enumerate(zip(dims, scale)):
            d.dims[n], d.scale[n] = k, s
    raw, q = bytes(d), nv.QkRope
    return d.naxes, raw[q.D.offset:q.pos.offset], raw[q.naxes.offset:q.freqs.offset]


def _rope_desc(axes, D, dtype, norm, eps, rows, pos, freqs, dev, heads, x, dy, y, w, b, dw, db, work):
    """x, dy, y: two (pointer, row stride); w, b, dw, db: two pointers; 0: not there."""
    naxes, mid, tail = _rope_fixed(axes, D, dtype, norm, eps)
    fr = 0
    where = (0, 0, 0)
    if axes is not None:
        if pos is None or pos.dim() != 2 or pos.shape[0] != rows or pos.shape[1] < naxes or pos.dtype not in _POS or pos.device != dev:
            _fail(f"pos must be an int32, int64 or fp32 [{rows}, {naxes}] tensor on {dev}, got "
                  f"{None if pos is None else (tuple(pos.shape), pos.dtype, pos.device)}")
        ld = pos.stride(0) if rows > 1 else pos.shape[1]
        if (pos.shape[1] > 1 and pos.stride(1) != 1) or ld < naxes:
            _fail(f"pos must have unit inner stride and rows that do not overlap, got strides {pos.stride()}")
        where = (pos.data_ptr(), ld, _POS[pos.dtype])
        if freqs is not None:
            rot = sum(axes.dims)
            if tuple(freqs.shape) != (rot // 2,) or freqs.dtype != torch.float64 or freqs.device != dev or not freqs.is_contiguous():
                _fail(f"freqs must be a contiguous fp64 tensor of {rot // 2} frequencies on {dev}")
            fr = freqs.data_ptr()
    elif pos is not None or freqs is not None:
        _fail("positions need RopeAxes that say what they turn")
    (x0, lx0), (x1, lx1) = x
    (g0, lg0), (g1, lg1) = dy
    (y0, ly0), (y1, ly1) = y
    sides = _SIDES.pack(x0, x1, lx0, lx1, g0, g1, lg0, lg1, y0, y1, ly0, ly1, *heads, *w, *b, *dw, *db, work, rows)
    return nv.QkRope.from_buffer_copy(sides + mid + _WHERE.pack(*where) + tail + fr.to_bytes(8, "little"))


_NO = ((0, 0), (0, 0))
_ZZ = (0, 0)


def _head_dim(x, heads, name):
    if heads <= 0 or x.shape[1] % heads:
        _fail(f"{name} has {x.shape[1]} columns: not a multiple of {heads} heads")
    return x.shape[1] // heads


def _ptrs(ts):
    """(pointer, row stride) of one or two matrices."""
    a = (ts[0].data_ptr(), _ld(ts[0]))
    return (a, (ts[1].data_ptr(), _ld(ts[1]))) if len(ts) > 1 else (a, (0, 0))


def _vptrs(ts):
    return tuple(0 if t is None else t.data_ptr() for t in ts) if ts is not None else _ZZ


def _rope_fwd(xs, heads, pos, axes, freqs, norm, eps, ws, bs):
    x0 = xs[0]
    dev, rows = x0.device, x0.shape[0]
    ys = tuple([torch.empty(x.shape, dtype=x.dtype, device=dev) for x in xs])
    d = _rope_desc(axes, _head_dim(x0, heads[0], "q"), x0.dtype, norm, eps, rows, pos, freqs, dev, heads, _ptrs(xs), _NO, _ptrs(ys),
                   _vptrs(ws), _vptrs(bs), _ZZ, _ZZ, 0)
    if rows:
        _launch("t2v_qk_rope_fwd", d, dev)
    return ys


def _rope_bwd(xs, dys, heads, pos, axes, freqs, norm, eps, ws, want):
    """want: per side (dw, db) wanted.  Returns dxs and the parameter gradients (fp32)."""
    dy0 = dys[0]
    dev, rows, D = dy0.device, dy0.shape[0], _head_dim(dy0, heads[0], "dy")
    dxs = [torch.empty(dy.shape, dtype=dy.dtype, device=dev) for dy in dys]
    dws, dbs = [None, None], [None, None]
    if norm:
        new = torch.empty if rows else torch.zeros
        for i in range(2):
            if want[i][0]:
                dws[i] = new(D, dtype=torch.float32, device=dev)
            if want[i][1]:
                dbs[i] = new(D, dtype=torch.float32, device=dev)
    d = _rope_desc(axes, D, dy0.dtype, norm, eps, rows, pos, freqs, dev, heads, _ptrs(xs) if norm else _NO, _ptrs(dys), _ptrs(dxs),
                   _vptrs(ws), _ZZ, _vptrs(dws), _vptrs(dbs), 0)
    if rows:
        if norm and (want[0][0] or want[0][1] or want[1][0] or want[1][1]):
            n = nv.lib().t2v_qk_rope_bwd_floats(C.byref(d))
            if n < 0:
                nv.check(int(n), "t2v_qk_rope_bwd_floats")
            work = torch.empty(int(n), dtype=torch.float32, device=dev)
            d.workspace = work.data_ptr()
        _launch("t2v_qk_rope_bwd", d, dev)
    return dxs, dws, dbs


# (The differentiable tensors are the Functions' arguments, the rest travels in one tuple: apply() spends about a microsecond per argument.)
class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rest):
        heads, pos, axes, freqs = rest
        ctx.heads, ctx.axes = heads, axes
        ctx.save_for_backward(pos, freqs)
        return _rope_fwd((x,), (heads, 0), pos, axes, freqs, None, 0.0, None, None)[0]

    @staticmethod
    def backward(ctx, dy):
        pos, freqs = ctx.saved_tensors
        return _rope_bwd(None, (_upstream(dy),), (ctx.heads, 0), pos, ctx.axes, freqs, None, 0.0, None, None)[0][0], None


def rope(x, heads, pos, axes, freqs=None):
    """Rotary positions: x [rows, heads * dim] (bf16, fp16 or fp32) with the columns `axes` (RopeAxes) names turned by pos [rows, number
    of axes] (int32, int64 or fp32).  Angles are formed in 64 bits.  freqs: fp64 [sum(dims) / 2] radians per unit of position, in the place of the
    ladder theta gives.  Returns a dense matrix of x's shape; differentiable in x."""
    x = _tokens(x, "x")
    heads = int(heads)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Rope.apply(x, (heads, pos, axes, freqs))
    return _rope_fwd((x,), (heads, 0), pos, axes, freqs, None, 0.0, None, None)[0]


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, qb, kb, rest):
        heads, pos, axes, freqs, norm, eps, ws, bs = rest
        ctx.meta = (heads, axes, norm, eps)
        ctx.types = [None if t is None else t.dtype for t in (qw, kw, qb, kb)]
        ctx.save_for_backward(q, k, qw, kw, pos, freqs)
        return _rope_fwd((q, k), heads, pos, axes, freqs, norm, eps, ws, bs)

    @staticmethod
    def backward(ctx, dq, dk):
        q, k, qw, kw, pos, freqs = ctx.saved_tensors
        heads, axes, norm, eps = ctx.meta
        D, dev, need = q.shape[1] // heads[0], q.device, ctx.needs_input_grad
        ws = (_vector(qw, D, dev, "q_weight"), _vector(kw, D, dev, "k_weight"))
        dxs, dws, dbs = _rope_bwd((q, k), (_upstream(dq), _upstream(dk)), heads, pos, axes, freqs, norm, eps, ws,
                                  ((need[2], need[4]), (need[3], need[5])))
        g = [None if t is None else t.to(y) for t, y in zip(dws + dbs, ctx.types)]
        return (dxs[0], dxs[1], *g, None)


def qk_norm_rope(q, k, heads, kv_heads, pos, axes, q_weight=None, k_weight=None, q_bias=None, k_bias=None, eps=1e-6, norm="rms",
                 freqs=None):
    """Queries [rows, heads * dim] and keys [rows, kv_heads * dim] normed per head and turned, in one launch: returns (q', k').

    norm: "rms" (x * rsqrt(mean x^2 + eps)) or "layer" (centred first); q_weight, k_weight, q_bias, k_bias: [dim] vectors shared by the
    heads, or None.  pos, axes, freqs: as in `rope`; both None: the norm alone.  Differentiable in q, k and the four vectors; the
    statistics are recomputed in the backward pass from the saved inputs."""
    q, k = _tokens(q, "q"), _tokens(k, "k")
    heads, kv_heads = int(heads), int(kv_heads)
    if norm not in _NORM:
        _fail(f"norm {norm!r}: 'rms' or 'layer'")
    if k.dtype != q.dtype or k.device != q.device or k.shape[0] != q.shape[0] or _head_dim(q, heads, "q") != _head_dim(k, kv_heads, "k"):
        _fail(f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} must have the same rows, type, device and head dim")
    D, dev = q.shape[1] // heads, q.device
    params = (q_weight, k_weight, q_bias, k_bias)
    ws = (_vector(q_weight, D, dev, "q_weight"), _vector(k_weight, D, dev, "k_weight"))
    bs = (_vector(q_bias, D, dev, "q_bias"), _vector(k_bias, D, dev, "k_bias"))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or any([t is not None and t.requires_grad for t in params])):
        return _QkNormRope.apply(q, k, *params, ((heads, kv_heads), pos, axes, freqs, norm, float(eps), ws, bs))
    return _rope_fwd((q, k), (heads, kv_heads), pos, axes, freqs, norm, float(eps), ws, bs)


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


def _op(t, lay):
    """The five fields of a T2VAttnOperand."""
    ld = _ld(t)
    return t.data_ptr(), lay.hi * ld, lay.lo * ld, lay.ss * ld, lay.bdiv


def _ints(t, shapes, dev, name):
    if t is None:
        return None
    if t.dtype != torch.int32 or tuple(t.shape) not in shapes or t.device != dev or not t.is_contiguous():
        _fail(f"{name} must be a contiguous int32 tensor of shape {' or '.join(map(str, shapes))} on {dev}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


# T2VAttnMod field by field, packed in one go (see _SIDES); _FWD ends where the fields of the backward pass begin
_OP = "Qqqqi4x"
_FWD = struct.Struct("@8i2f" + 4 * _OP + "QQi4xQQQQQii")
_BWD = struct.Struct("@" + 4 * _OP + "QQi4xQqQqi4x")
_NO_BWD = bytes(_BWD.size)


def _attn_desc(q, k, v, o, meta, lse, prefix, kv_len, q_docs, kv_docs, slopes, bias, bwd=None):
    heads, kv_heads, qlay, klay, scale, causal, softcap = meta
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    fwd = _FWD.pack(qlay.nbatch, heads, kv_heads, qlay.S, klay.S, q.shape[1] // heads, _TYPE[q.dtype], causal, scale, softcap,
                    *_op(q, qlay), *_op(k, klay), *_op(v, klay), *_op(o, qlay), ptr(lse), ptr(prefix), 0 if prefix is None else prefix.dim() - 1,
                    ptr(kv_len), ptr(q_docs), ptr(kv_docs), ptr(slopes), ptr(bias), 0 if bias is None else bias.dtype == torch.float32,
                    0 if bias is None else bias.shape[1] // 2)
    return nv.AttnMod.from_buffer_copy(fwd + (_NO_BWD if bwd is None else _BWD.pack(*bwd, 0, 0, 0, 0, 0)))


def _workspace(a, backward, dev):
    n = nv.lib().t2v_attn_mod_workspace(C.byref(a), backward)
    if n < 0:
        nv.check(int(n), "t2v_attn_mod_workspace")
    if n == 0:
        return None
    w = torch.empty(int(n), dtype=torch.uint8, device=dev)      # (the caching allocator's blocks are 512-byte aligned)
    a.workspace, a.workspace_bytes = w.data_ptr(), int(n)
    return w


def _meta(a, dev):
    """The buffer for what a call derives from documents and prefixes per query, tile by tile (None where there are none)."""
    if not a.q_docs and not (a.prefix and a.prefix_per_query):
        return None
    n = nv.lib().t2v_attn_mod_meta_bytes(C.byref(a))
    if n < 0:
        nv.check(int(n), "t2v_attn_mod_meta_bytes")
    m = torch.empty(int(n), dtype=torch.uint8, device=dev)
    a.meta, a.meta_bytes = m.data_ptr(), int(n)
    return m


def _attn_fwd(q, k, v, meta, prefix, kv_len, q_docs, kv_docs, slopes, bias, keep):
    heads, _, qlay, klay = meta[:4]
    dev = q.device
    if qlay.nbatch * qlay.S == 0 or klay.S == 0:        # nothing is asked, or there is nothing to see
        o = torch.zeros(q.shape, dtype=q.dtype, device=dev)
        return o, (torch.full((qlay.nbatch * heads * qlay.S,), math.inf, device=dev) if keep else None), None
    covered = _layout_facts(qlay, q.shape[0])[2]
    o = (torch.empty if covered else torch.zeros)(q.shape, dtype=q.dtype, device=dev)      # rows that no sequence owns: zeros
    lse = torch.empty(qlay.nbatch * heads * qlay.S, dtype=torch.float32, device=dev) if keep else None
    a = _attn_desc(q, k, v, o, meta, lse, prefix, kv_len, q_docs, kv_docs, slopes, bias)
    tiles = _meta(a, dev)
    work = _workspace(a, 0, dev)      # noqa: F841 (kept until the launch is issued)
    _launch("t2v_attn_mod_fwd", a, dev)
    return o, lse, tiles


class _AttentionMod(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, rest):
        meta, prefix, kv_len, q_docs, kv_docs, slopes = rest
        o, lse, tiles = _attn_fwd(q, k, v, meta, prefix, kv_len, q_docs, kv_docs, slopes, bias, True)
        ctx.meta = meta
        ctx.save_for_backward(q, k, v, bias, prefix, kv_len, q_docs, kv_docs, slopes, o, lse, tiles)
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, bias, prefix, kv_len, q_docs, kv_docs, slopes, o, lse, tiles = ctx.saved_tensors
        qlay, klay = ctx.meta[2:4]
        dev = q.device
        do = _upstream(do)
        empty = qlay.nbatch * qlay.S == 0 or klay.S == 0
        share = klay.bdiv if klay.bdiv > 1 and klay.lo == 0 else 1
        kfacts = _layout_facts(klay, k.shape[0])
        kall = kfacts[2] or (share > 1 and klay.nbatch % share == 0 and klay.nbatch // share * klay.S == k.shape[0])
        new = lambda t, full: (torch.empty if full and not empty else torch.zeros)(t.shape, dtype=t.dtype, device=dev)  # noqa: E731
        dq, dk, dv = new(q, _layout_facts(qlay, q.shape[0])[2]), new(k, kall), new(v, kall)
        dbias = new(bias, True) if bias is not None and ctx.needs_input_grad[3] else None
        if not empty:
            delta = torch.empty_like(lse)
            a = _attn_desc(q, k, v, o, ctx.meta, lse, prefix, kv_len, q_docs, kv_docs, slopes, bias,
                           (*_op(do, qlay), *_op(dq, qlay), *_op(dk, klay), *_op(dv, klay), delta.data_ptr(),
                            0 if dbias is None else dbias.data_ptr(), share))
            if tiles is not None:
                a.meta, a.meta_bytes, a.meta_ready = tiles.data_ptr(), tiles.numel(), 1
            work = _workspace(a, 1, dev)      # noqa: F841 (kept until the launches are issued)
            _launch("t2v_attn_mod_bwd", a, dev)
        return dq, dk, dv, dbias, None


def attention_mod(q, k, v, heads, qlay, klay, kv_heads=None, scale=None, causal=False, prefix=None, kv_len=None, q_docs=None, kv_docs=None,
                  softcap=0.0, slopes=None, bias=None):
    """Attention whose scores may be capped, biased by distance and masked by position and document.

    q: [rows_q, heads * dim]; k, v: [rows_kv, kv_heads * dim] token matrices in bf16 or fp16 (dim a multiple of 8 up to 128; heads a
    multiple of kv_heads, which defaults to heads); qlay, klay: SeqLayout of the sequences.  With t = scale * q.k (scale defaults to
    dim^-0.5):
      softcap > 0    t <- softcap * tanh(t / softcap)
      slopes         fp32 [heads]: t <- t - slopes[h] * |j - i'|                                  (not trained)
      bias           [heads, 2R + 1] (R <= 1024, the operands' type or fp32): t <- t + bias[h, clip(j - i', -R, R) + R]; trained when it
                     requires a gradient; an entry at or below its type's lowest finite value hides its distance
      kv_len         int32 [nbatch]: keys 0 .. kv_len - 1 exist (default: all)
      causal         keys j <= i';  prefix (int32 [nbatch] or [nbatch, Sq], with causal): and all keys j < prefix
      q_docs, kv_docs  int32 [nbatch, Sq], [nbatch, Sk]: only keys of the query's document; numbers below 0 mark padding
    i' = i + kv_len - Sq is the query's place among the keys: the queries are the last positions.  A row that may see nothing is zero.
    Keys and values that no query may see (behind kv_len, padding) may hold anything; a key or value that is visible to one query of a
    sequence must be finite, since masked weights of its tile are exact zeros that multiply it.
    Few query rows over many keys (serving steps, chunks of new tokens) split the keys over workgroups and join them.
    Returns [rows_q, heads * dim]; rows that no sequence owns are zero.  Differentiable in q, k, v and bias; K / V shared by the bdiv batches
    of a layout with lo = 0 get the sum of their gradients.  The order of all sums is fixed: repeated runs are bit-equal."""
    types = (torch.bfloat16, torch.float16)
    q, k, v = _tokens(q, "q", types), _tokens(k, "k", types), _tokens(v, "v", types)
    heads = int(heads)
    kv_heads = heads if kv_heads is None else int(kv_heads)
    dev, D = q.device, _head_dim(q, heads, "q")
    if kv_heads <= 0 or heads % kv_heads:
        _fail(f"{heads} query heads cannot share {kv_heads} key / value heads evenly")
    if k.shape != v.shape or k.shape[1] != kv_heads * D or not q.dtype == k.dtype == v.dtype or not dev == k.device == v.device:
        _fail(f"q {tuple(q.shape)} {q.dtype}, k {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype}: one type, one device, {kv_heads} "
              f"key / value heads of {D} columns are wanted")
    if D % 8 or D > 128:
        _fail(f"attention_mod takes head dims that are multiples of 8 up to 128, got {D}")
    nb, Sq, Sk = qlay.nbatch, qlay.S, klay.S
    qf, kf = _layout_facts(qlay, q.shape[0]), _layout_facts(klay, k.shape[0])
    if nb != klay.nbatch or not qf[0] or not kf[0]:
        _fail(f"layouts {qlay} over {q.shape[0]} rows and {klay} over {k.shape[0]} rows: as many batches on both sides, rows that exist")
    if not qf[1]:
        _fail(f"query layout {qlay} names a row twice")
    softcap, scale = float(softcap), float(D ** -0.5 if scale is None else scale)
    if not 0.0 <= softcap < 1e30 or not math.isfinite(scale):
        _fail(f"softcap {softcap}, scale {scale}: a finite scale and a cap of 0 (none) or more are wanted")
    if prefix is not None and not causal:
        _fail("prefix opens a causal mask: pass causal=True with it")
    if (q_docs is None) != (kv_docs is None):
        _fail("q_docs and kv_docs come together")
    _ints(prefix, ((nb,), (nb, Sq)), dev, "prefix")
    _ints(kv_len, ((nb,),), dev, "kv_len")
    _ints(q_docs, ((nb, Sq),), dev, "q_docs")
    _ints(kv_docs, ((nb, Sk),), dev, "kv_docs")
    if slopes is not None:
        if slopes.dtype != torch.float32 or tuple(slopes.shape) != (heads,) or slopes.device != dev or not slopes.is_contiguous():
            _fail(f"slopes must be a contiguous fp32 tensor of {heads} elements on {dev}")
        if slopes.requires_grad:
            _fail("slopes are not trained: pass slopes.detach(), or a bias table for a learned distance bias")
    if bias is not None:
        if bias.dtype not in (q.dtype, torch.float32) or bias.dim() != 2 or bias.shape[0] != heads or bias.shape[1] % 2 == 0 or \
                bias.shape[1] > 2049 or bias.device != dev or not bias.is_contiguous():
            _fail(f"bias must be a contiguous [{heads}, 2R + 1] table with R <= 1024 in {q.dtype} or fp32 on {dev}, got {tuple(bias.shape)} {bias.dtype}")
    meta = (heads, kv_heads, qlay, klay, scale, int(bool(causal)), softcap)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad)):
        if not kf[1] and not (klay.bdiv > 1 and klay.lo == 0 and klay.hi >= (klay.S - 1) * klay.ss + 1 and klay.ss > 0):
            _fail(f"key layout {klay} names a row twice: gradients are defined for rows of their own, or shared by the bdiv batches (lo = 0)")
        return _AttentionMod.apply(q, k, v, bias, (meta, prefix, kv_len, q_docs, kv_docs, slopes))
    return _attn_fwd(q, k, v, meta, prefix, kv_len, q_docs, kv_docs, slopes, bias, False)[0]
