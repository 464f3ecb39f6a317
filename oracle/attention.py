"""Packed attention and norm + rotation of query / key heads from their formulas, in float64 on the CPU, with error bounds.

The bounds are sums of what each rounding can do: `u` is half a step of the 16-bit type (operands p and dS of the second products, the
result), the 32-bit part counts the length of the accumulations.  Nothing here calls the code under test."""
import math

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def keys_seen(q_len, k_len, block):
    """how many of its first keys each token sees"""
    if block == 0:
        return torch.full((q_len,), k_len)
    at = torch.arange(q_len) + (k_len - q_len)
    return torch.clamp((torch.div(at, block, rounding_mode="floor") + 1) * block, 0, k_len)


def attention(q, k, v, lengths, key_lengths=None, key_starts=None, block=0, scale=None, grad=None):
    """{o, lse, dq, dk, dv} in float64 for any inputs, and a bound of each one's error ("o_err", ...) for results computed with 16-bit
    operands of q's type and 32-bit sums.  Rows of no sequence: 0 / -inf."""
    u = half_step(q.dtype) if q.dtype in (torch.float16, torch.bfloat16) else U32
    # p and dS of a key: half a step of fp16's smallest numbers (2^-25) after the lift by 2^4 is 2^-29, two operands' worth 2^-28; in bf16 and
    # in 32 bits what lies below the smallest normal number 2^-126 may count as zero, which is off by 2^-126 at most
    tiny = 2.0 ** -28 if q.dtype == torch.float16 else 2.0 ** -126
    sub = 2.0 ** -25 if q.dtype == torch.float16 else 0.0                  # the same for results
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    heads, kv_heads, d = q.shape[1], k.shape[1], q.shape[2]
    group = heads // kv_heads
    key_lengths = lengths if key_lengths is None else key_lengths
    scale = 1 / math.sqrt(d) if scale is None else scale
    r = {"o": torch.zeros_like(q), "lse": torch.full(q.shape[:2], -math.inf, dtype=torch.float64)}
    names = ["o", "lse"]
    if grad is not None:
        g = grad.double().cpu()
        r.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
        names += ["dq", "dk", "dv"]
    for n in names:
        r[n + "_err"] = torch.zeros_like(r[n])
    q0 = k0 = 0
    for i, (m, l) in enumerate(zip(lengths, key_lengths)):
        ks = k0 if key_starts is None else key_starts[i]
        seen = torch.arange(l)[None] < keys_seen(m, l, block)[:, None]
        rows, keys = slice(q0, q0 + m), slice(ks, ks + l)
        for h in range(heads if m and l else 0):
            hk = h // group
            Q, K, V = q[rows, h], k[keys, hk], v[keys, hk]
            s = torch.where(seen, scale * (Q @ K.T), -math.inf)
            lse = torch.logsumexp(s, 1)
            p = torch.where(seen, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None]), 0.0)
            V = torch.where(seen.any(0)[:, None], V, 0.0)                  # what nobody sees has no part
            K = torch.where(seen.any(0)[:, None], K, 0.0)
            o = p @ V
            # a score is a sum of d products (and the exponent's rounding grows with its size); p inherits it, and so does the row's sum
            ds = (d + 4) * U32 * scale * (Q.abs() @ K.abs().T).amax(1, keepdim=True) + 8 * U32
            e = u + 2 * ds + (l + 8) * U32                                 # relative error of p as an operand, and of the sums
            po = p @ V.abs()
            r["o"][rows, h], r["lse"][rows, h] = o, lse
            r["o_err"][rows, h] = u * o.abs() + e * po + sub + tiny * V.abs().sum(0)
            r["lse_err"][rows, h] = (ds + (l + 8) * U32)[:, 0] + 4 * U32 * torch.where(lse == -math.inf, 0.0, lse.abs())
            if grad is None:
                continue
            G = g[rows, h]
            dp = G @ V.T
            delta = (G * o).sum(1, keepdim=True)
            dS = p * (dp - delta)
            # |dP| and |delta| as sums of absolute values; o's own error (before its rounding, known to u^2) enters delta
            size = G.abs() @ V.abs().T + (G.abs() * (po + r["o"][rows, h].abs())).sum(1, keepdim=True)
            e2 = e - u + (2 * d + 8) * U32 + u * u
            derr = (G.abs() * ((e - 0.0) * po)).sum(1, keepdim=True)       # delta from an o that is off by e * po
            dS_err = p * (u * (dp - delta).abs() + e2 * size + derr)
            r["dq"][rows, h] = scale * (dS @ K)
            r["dq_err"][rows, h] = scale * (dS_err @ K.abs() + (l + 8) * U32 * (dS.abs() @ K.abs()) + tiny * K.abs().sum(0)) + u * r["dq"][rows, h].abs() + sub
            r["dk"][keys, hk] += scale * (dS.T @ Q)
            r["dk_err"][keys, hk] += scale * (dS_err.T @ Q.abs() + (m * group + 8) * U32 * (dS.abs().T @ Q.abs()) + tiny * Q.abs().sum(0))
            r["dv"][keys, hk] += p.T @ G
            r["dv_err"][keys, hk] += (p * e).T @ G.abs() + (m * group + 8) * U32 * (p.T @ G.abs()) + tiny * G.abs().sum(0)
        q0, k0 = q0 + m, k0 + l
    if grad is not None:
        for n in ("dk", "dv"):
            r[n + "_err"] += u * r[n].abs() + sub
    return r


def _turn(x, cos, sin, pairs, interleaved):
    y = x.clone()
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., a] * sin + x[..., b] * cos
    return y


def qk_norm_rope(x, positions, inv_freq, sections, weight=None, normalize=True, eps=1e-6, interleaved=False, grad=None):
    """{y, dx, dw} of one of the two tensors in float64, and bounds of their errors"""
    u = half_step(x.dtype) if x.dtype != torch.float32 else U32
    uw = u if weight is None else half_step(weight.dtype) if weight.dtype != torch.float32 else U32
    sub = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    x = x.double().cpu()
    n, heads, d = x.shape
    w = torch.ones(d, dtype=torch.float64) if weight is None else weight.double().cpu()
    pairs = sum(sections)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angle = positions.double().cpu().view(n, -1)[:, axis] * inv_freq.double().cpu()
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    s = (x.square().mean(-1, keepdim=True) + eps).rsqrt() if normalize else torch.ones(n, heads, 1, dtype=torch.float64)
    z = x * s * w
    y = _turn(z, cos, sin, pairs, interleaved)
    # sines and cosines are off by a few 2^-24 (argument reduced to half a turn, then 32 bits); the mean of squares is a sum of d
    c = (16 + (d if normalize else 0)) * U32
    mag = _turn(z.abs(), torch.ones_like(cos), torch.ones_like(sin), pairs, interleaved).abs()       # |b| + |a| (and |a| - |b|: made a sum below)
    both = torch.maximum(mag, _turn(z.abs(), torch.ones_like(cos), -torch.ones_like(sin), pairs, interleaved).abs())
    r = {"y": y, "y_err": u * y.abs() + c * both + sub}
    if grad is None:
        return r
    g = grad.double().cpu()
    dz = _turn(g, cos, -sin, pairs, interleaved)
    ga = torch.maximum(_turn(g.abs(), torch.ones_like(cos), torch.ones_like(sin), pairs, interleaved).abs(),
                       _turn(g.abs(), torch.ones_like(cos), -torch.ones_like(sin), pairs, interleaved).abs())
    if not normalize:
        r.update(dx=dz, dx_err=u * dz.abs() + c * ga + sub)
        return r
    m = (w * dz * x).mean(-1, keepdim=True)
    r["dx"] = s * w * dz - x * s ** 3 * m
    size = s * w.abs() * ga + x.abs() * s ** 3 * (w.abs() * ga * x.abs()).mean(-1, keepdim=True)
    r["dx_err"] = u * r["dx"].abs() + (32 + 3 * d) * U32 * size + sub
    r["dw"] = (dz * x * s).sum((0, 1))
    total = (ga * x.abs() * s).sum((0, 1))
    r["dw_err"] = uw * r["dw"].abs() + (32 + d + min(n * heads, 4096)) * U32 * total
    return r
