"""Plain 64-bit forms of the transformer-block operators (rotary positions, per-head norms, attention with modified scores) on the CPU, with the
elementwise error that one rounding of each intermediate the kernels hold in 16 bits can cause."""
import math

import torch

F64 = torch.float64


def turn(x, pos, dims, theta=10000.0, style="interleaved", shared=False, scale=None, freqs=None, back=False):
    """x [rows, heads, D] in 64 bits, turned (or turned back)."""
    x = x.clone()
    R, rows = sum(dims), x.shape[0]
    p, first = 0, 0
    for a, d in enumerate(dims):
        for i in range(d // 2):
            f = float(freqs[p]) if freqs is not None else theta ** (-2.0 * (p / R if shared else i / d))
            ang = pos[:, a].to(F64) * f * (1.0 if scale is None else scale[a])
            c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None] * (-1.0 if back else 1.0)
            m, n = (2 * p, 2 * p + 1) if style == "interleaved" else (p, p + R // 2)
            u, v = x[:, :, m].clone(), x[:, :, n].clone()
            x[:, :, m], x[:, :, n] = u * c - v * s, v * c + u * s
            p += 1
        first += d
    return x


def norm_stats(x, kind, eps):
    mid = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    r = ((x - mid) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    return (x - mid) * r, r


def norm_backward(x, w, d, kind, eps):
    """dx, dw, db of y = w * xhat + b for upstream d, all [rows, heads, D] in 64 bits."""
    hat, r = norm_stats(x, kind, eps)
    e = d * w
    dx = e - hat * (e * hat).mean(-1, keepdim=True)
    if kind == "layer":
        dx = dx - e.mean(-1, keepdim=True)
    return dx * r, (d * hat).sum((0, 1)), d.sum((0, 1))


def visible(Sq, Sk, L, causal, prefix, qd, kd):
    """[Sq, Sk] of what query i may see, from plain loops over the definition."""
    i, j = torch.arange(Sq)[:, None] + (L - Sq), torch.arange(Sk)[None]
    m = (j < L).expand(Sq, Sk).clone()
    if causal:
        open_ = torch.zeros(Sq, 1, dtype=torch.long) if prefix is None else prefix.long().reshape(-1, 1).expand(Sq, 1)
        m &= (j <= i) | (j < open_)
    if qd is not None:
        m &= (qd[:, None] == kd[None]) & (qd[:, None] >= 0)
    return m


def attention(q, k, v, scale, dt, causal=False, prefix=None, kv_len=None, q_docs=None, kv_docs=None, softcap=0.0, slopes=None, bias=None,
              do=None):
    """q [B, Sq, H, D], k, v [B, Sk, KV, D], bias [H, 2R + 1], do like q: any dtype, computed in 64 bits.
    Returns {name: (value, bound)} for o (and dq, dk, dv, dbias): `bound` is the elementwise error that the kernels' roundings to `dt`
    (half a step each: the output, P, dS, and O inside delta) and fp32 sums can cause."""
    u = torch.finfo(dt).eps / 2
    tiny = float(torch.finfo(dt).smallest_normal) * u * 2 if dt == torch.float16 else 0.0      # half a step among the subnormals
    B, Sq, H, D = q.shape
    Sk, KV = k.shape[1], k.shape[2]
    G = H // KV
    z = lambda *s: torch.zeros(*s, dtype=F64)  # noqa: E731
    out = {"o": (z(B, Sq, H, D), z(B, Sq, H, D))}
    if do is not None:
        out.update(dq=(z(B, Sq, H, D), z(B, Sq, H, D)), dk=(z(B, Sk, KV, D), z(B, Sk, KV, D)), dv=(z(B, Sk, KV, D), z(B, Sk, KV, D)))
        if bias is not None:
            out["dbias"] = (z(*bias.shape), z(*bias.shape))
    S = 2e-4          # fp32 slack, relative to the sums of magnitudes: scores up to ~1e2 in fp32, exp2 / rcp of one unit in the last place
    for b in range(B):
        L = Sk if kv_len is None else max(0, min(int(kv_len[b]), Sk))
        seen = visible(Sq, Sk, L, causal, None if prefix is None else prefix[b], None if q_docs is None else q_docs[b],
                       None if kv_docs is None else kv_docs[b])
        anyq, anyk = seen.any(1), seen.any(0)
        gap = torch.arange(Sk)[None] - (torch.arange(Sq)[:, None] + (L - Sq))
        for h in range(H):
            Q = torch.where(anyq[:, None], q[b, :, h].to(F64), 0.0)
            K, V = (torch.where(anyk[:, None], t[b, :, h // G].to(F64), 0.0) for t in (k, v))
            t = Q @ K.T * scale
            w = torch.ones_like(t)
            if softcap:
                th = torch.tanh(t / softcap)
                t, w = softcap * th, 1 - th * th
            if slopes is not None:
                t = t - float(slopes[h]) * gap.abs()
            if bias is not None:
                R = bias.shape[1] // 2
                at = gap.clamp(-R, R) + R
                low = torch.finfo(bias.dtype).min
                t = t + torch.where(bias[h] <= low, -math.inf, bias[h].to(F64))[at]
            t = torch.where(seen, t, -math.inf)
            top = t.amax(1, keepdim=True) if Sk else z(Sq, 1)
            p = torch.exp(t - torch.where(torch.isinf(top), 0.0, top))
            P = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            O = P @ V
            A = P @ V.abs()
            eo = u * O.abs() + (u + S) * A + tiny * (V.abs().sum(0)[None] + 1)
            out["o"][0][b, :, h], out["o"][1][b, :, h] = O, eo
            if do is None:
                continue
            g = torch.where(anyq[:, None], do[b, :, h].to(F64), 0.0)
            dP = g @ V.T
            dS = P * (dP - (g * O).sum(1, keepdim=True))
            ed = (g.abs() * eo).sum(1, keepdim=True)                                # error of delta through the rounded O
            eds = P * (ed + S * (g.abs() @ V.abs().T + (g.abs() * O.abs()).sum(1, keepdim=True))) + 4 * S * dS.abs()
            for name, val, err in (("dv", P.T @ g, (u + S) * (P.T @ g.abs()) + tiny * g.abs().sum(0)[None]),
                                   ("dk", (dS * w).T @ Q * scale, (u * (dS * w).abs() + eds + tiny).T @ Q.abs() * abs(scale))):
                out[name][0][b, :, h // G] += val
                out[name][1][b, :, h // G] += err
            out["dq"][0][b, :, h] = (dS * w) @ K * scale
            out["dq"][1][b, :, h] = (u * (dS * w).abs() + eds + tiny) @ K.abs() * abs(scale)
            if bias is not None:
                out["dbias"][0][h].index_add_(0, at.reshape(-1), torch.where(seen, dS, 0.0).reshape(-1))
                out["dbias"][1][h].index_add_(0, at.reshape(-1), torch.where(seen, eds, 0.0).reshape(-1))
    for name, (val, err) in out.items():
        if name != "o":
            err += (0.0 if name == "dbias" and bias.dtype == torch.float32 else u) * val.abs() + tiny
        err += 1e-9
    return out
