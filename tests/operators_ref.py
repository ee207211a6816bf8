"""Plain f64 references of the operators, with the bounds their results keep.

u is half a step of the rows' type (2^-8 bf16, 2^-11 f16, 2^-24 f32, relative).
"""
import numpy as np

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
U32 = 2.0 ** -24
TINY = {"bf16": 2.0 ** -133, "f16": 2.0 ** -25, "f32": 2.0 ** -149}   # half the smallest step


def rounded(a, dtype):
    """Values of `dtype` nearest to a, as f64."""
    from mlk2_amd.backend import bf16_bits, bf16_values
    if dtype == "bf16":
        return bf16_values(bf16_bits(a)).astype(np.float64)
    return np.asarray(a).astype({"f16": np.float16, "f32": np.float32}[dtype]).astype(np.float64)


def norm_rope(x, weight, positions, *, rot, theta, eps, interleaved, sections, dtype):
    """(y, bound) of heads x [tokens, heads, dim]; weight or positions may be
    None.

    Bound: the mean of dim squares, its root and two products in f32 are within
    (dim / 2 + 8) U32 relatively; cosine and sine each within 2^-22 of the exact
    ones (angle reduced in f64, f32 polynomial); two products and a sum; then
    one rounding to the type."""
    t, h, d = x.shape
    y = x.copy()
    if weight is not None:
        y = x / np.sqrt((x * x).sum(-1, keepdims=True) / d + eps) * weight
    rel = (d / 2 + 8) * U32 if weight is not None else 0.0
    size = np.abs(y)
    z, slack = y.copy(), rel * size
    if positions is not None:
        half, ends = rot // 2, np.cumsum(sections)
        for i in range(half):
            axis = int(np.searchsorted(ends, i, side="right"))
            angle = positions[axis].astype(np.float64) * theta ** (-2.0 * i / rot)
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
            z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
            both = size[..., a] + size[..., b]
            slack[..., a] = slack[..., b] = both * (rel + 2.0 ** -22 + 3 * U32)
    return z, slack * (1 + 2 * U[dtype]) + U[dtype] * np.abs(z) + TINY[dtype]


def attention(q, k, v, q_offsets, kv_start, kv_len, *, scale, causal, dtype, prefix_k=None, prefix_v=None):
    """(out, bound, lse, lse bound, rows written) of rows q [tokens, heads,
    dim], keys k, v [rows, kv_heads, dim]. Only visible keys are read.

    Bound: a score (a sum of dim products, the scale, log2 e) is within e = U32
    (2 dim + 32) sum |q k| scale of the exact one, a weight relative to the
    row's largest within 2 e + n U32 (its exponential, the running sum of n,
    rescaled as the maximum grows), then rounded to the type: out is within
    (u + 4 max e + 4 (n + 64) U32) sum w |v|, and one rounding of itself. f16
    weights below 2^-14 are within 2^-25 of a largest weight of 1: n 2^-25 |v|
    over a sum of at least 1."""
    tokens, heads, dim = q.shape
    group = heads // k.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    lse, lse_bound = np.full((tokens, heads), -np.inf), np.zeros((tokens, heads))
    written = np.zeros(tokens, dtype=bool)
    for b in range(len(q_offsets) - 1):
        q0, q1 = int(q_offsets[b]), int(q_offsets[b + 1])
        n, k0, nk = q1 - q0, int(kv_start[b]), int(kv_len[b])
        written[q0:q1] = True
        for i in range(n):
            own = max(0, min(nk, i + nk - n + 1)) if causal else nk
            for g in range(k.shape[1]):
                kk, vv = k[k0:k0 + own, g], v[k0:k0 + own, g]
                if prefix_k is not None:
                    kk, vv = np.concatenate([prefix_k[:, g], kk]), np.concatenate([prefix_v[:, g], vv])
                if len(kk) == 0:
                    continue
                qq = q[q0 + i, g * group:(g + 1) * group]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = qq @ kk.T * scale
                    top = s.max(-1, keepdims=True)
                    w = np.exp(s - np.where(np.isfinite(top), top, 0.0))
                    total = w.sum(-1, keepdims=True)
                    o = (w @ vv) / total
                    e = U32 * (2 * dim + 32) * (np.abs(qq) @ np.abs(kk).T).max(-1, keepdims=True) * abs(scale)
                    spread = (w / total) @ np.abs(vv)
                    cut = len(kk) * 2.0 ** -25 * np.abs(vv).max(0) if dtype == "f16" else 0.0
                    hi = slice(g * group, (g + 1) * group)
                    out[q0 + i, hi] = o
                    u = U[dtype]
                    bound[q0 + i, hi] = ((u + 4 * e + 4 * (len(kk) + 64) * U32) * spread + cut) * (1 + u) + u * np.abs(o) + TINY[dtype]
                    lse[q0 + i, hi] = (top + np.log(total))[:, 0]
                    lse_bound[q0 + i, hi] = (2 * e[:, 0] + (len(kk) + 64) * U32) + 8 * U32 * (1 + np.abs(lse[q0 + i, hi]))
    return out, bound, lse, lse_bound, written
