"""Calls of the operators that the headers allow at the ends of their ranges:
magnitudes, long tails, rows that no sequence holds, many tokens to a wave."""
import numpy as np
import pytest

from attention_abi import Attention
from mlk2_amd import operators as op
from mlk2_amd.backend import DeviceBuffer
from operators_ref import TINY, U, U32, attention, norm_rope, rounded
from test_operators_gpu import KEEP, TYPES, close, run

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------- qk_norm_rope --
# Elements whose squares f32 does not hold, or loses bits of: below 1e-19, past 1e19.
SMALL, LARGE = [1e-20, 1e-24, 1e-30, 1e-38], [1e19, 1e25, 3e36]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [8, 64, 128, 256, 36, 20])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-6])
@pytest.mark.parametrize("magnitudes", [SMALL, LARGE, SMALL + [1.0] + LARGE])
def test_norm_of_heads_far_from_one(hip, dtype, d, eps, magnitudes):
    # Heads of different magnitudes side by side, so that one wave has several.
    t, h, g = 9, 6, 3
    rng = np.random.default_rng(d)
    x = rng.standard_normal((t, h + 2 * g, d)) * rng.choice(magnitudes, (t, h + 2 * g, 1))
    x = rounded(x, dtype)
    weights = {w: rounded(1 + 0.2 * rng.standard_normal(d), dtype) for w in ("q_weight", "k_weight")}
    pos = np.arange(t)[None]
    km = op.qk_norm_rope_module(t, heads=h, kv_heads=g, dim=d, dtype=dtype, eps=eps)
    got = run(hip, km, {"qkv": x, "positions": pos, **weights})
    args = dict(rot=d, theta=1e4, eps=eps, interleaved=False, sections=[d // 2], dtype=dtype)
    for name, heads in (("q", slice(0, h)), ("k", slice(h, h + g))):
        want, bound = norm_rope(x[:, heads], weights[f"{name}_weight"], pos, **args)
        close(got[name], want, bound, name)
    assert (got["v"] == x[:, h + g:]).all()


# ---------------------------------------------------------------- attention --
# Row blocks and key ranges: (heads, key/value heads, queries, keys).
TAILS = {"narrow": (4, 2, 1, 300), "ranges": (4, 1, 1, 20000), "halves": (32, 16, 200, 5000), "halves_ranges": (4, 1, 300, 20000),
         "wide": (132, 132, 130, 601)}


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("name,hidden", [(n, b) for n in TAILS for b in (False, True) if not b or TAILS[n][2] > 1])
def test_f16_tail_behind_one_key(hip, d, name, hidden):
    """One key with the largest score and no value, all others 2^-26 of it, with
    values about 1: what is left of a tail in f16 weights. `hidden`: a NaN that
    the first queries do not see, so that keys are taken one by one.

    Bound, scores being exact products: a weight relative to the largest is
    within 2^-11 of itself or 2^-25 2^-7, its exponential and the running sums
    within (n + 64) 2^-24, and out is rounded once."""
    h, g, nq, nk = TAILS[name]
    rng = np.random.default_rng(nk)
    q, k = np.zeros((nq, h, d)), np.zeros((nk, g, d))
    q[..., 0], k[..., 0], k[nk // 3, :, 0] = 1.0, -18.0, 0.0
    v = rounded(0.5 + rng.random((nk, g, d)), "f16")
    v[nk // 3] = 0.0
    if hidden:
        v[nk - 1, :, 0] = np.nan
    km = op.attention_module(nq, kv_rows=nk, sequences=1, heads=h, kv_heads=g, dim=d, dtype="f16", causal=hidden, scale=1.0, lse=True)
    got = run(hip, km, {"q": q, "k": k, "v": v, "q_offsets": [0, nq], "kv_start": [0], "kv_len": [nk]})
    rows = nq - 1 if hidden else nq
    seen = nk - nq + 1 + np.arange(rows) if hidden else np.full(rows, nk)
    w = np.exp(k[:, 0, 0])
    total, sums = np.cumsum(w)[seen - 1], np.cumsum(w[:, None, None] * np.where(np.isnan(v), 0.0, v), 0)[seen - 1]
    top = np.cumsum(np.where(np.isnan(v), 0.0, v), 0)[seen - 1]   # sums of the tail's values
    want = np.repeat(sums / total[:, None, None], h // g, 1)
    sum_error = (nk + 64) * 2.0 ** -24
    bound = want * (2.0 ** -11 + sum_error) * 2 + np.repeat(top, h // g, 1) * 2.0 ** -32 + 2.0 ** -25
    close(got["out"][:rows], want, bound)
    close(got["lse"][:rows], np.repeat(np.log(total)[:, None], h, 1), sum_error + 2.0 ** -22)


SHAPES = {"narrow": (4, 2, 1, 300), "ranges": (4, 1, 1, 5000), "halves": (32, 16, 200, 500), "halves_ranges": (4, 1, 300, 3000),
          "wide": (132, 132, 130, 601)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 256, 20])
@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [23, 26, 31, 40, 60])
def test_scores_far_from_zero(hip, dtype, d, name, sign, size):
    """Scores of about 2^size: the keys with the largest share the weight.

    Scores are one product, the same for the same operands, and an eighth and
    more apart, which is 2^20 and more; so the result is a mean of n values,
    each product and sum within 2^-24 n, the weights and out rounded once."""
    h, g, nq, nk = SHAPES[name]
    rng = np.random.default_rng(nk)
    q, k = np.zeros((nq, h, d)), np.zeros((nk, g, d))
    q[..., 1] = 1.37 * 2.0 ** 8
    k[..., 1] = sign * rng.choice([1.25, 1.3828125, 1.5] if sign > 0 else [1.8671875, 1.99], (nk, g)) * 2.0 ** 8
    best = sorted(rng.choice(nk, 7, replace=False))
    k[best, :, 1] = sign * 1.7109375 * 2.0 ** 8
    q, k = rounded(q, dtype), rounded(k, dtype)
    v = rounded(rng.standard_normal((nk, g, d)), dtype)
    scale = 2.0 ** (size - 17)
    km = op.attention_module(nq, kv_rows=nk, sequences=1, heads=h, kv_heads=g, dim=d, dtype=dtype, causal=False, scale=scale, lse=True)
    got = run(hip, km, {"q": q, "k": k, "v": v, "q_offsets": [0, nq], "kv_start": [0], "kv_len": [nk]})
    want = np.repeat(v[best].mean(0), h // g, 0)
    size_of = np.repeat(np.abs(v[best]).mean(0), h // g, 0)
    close(got["out"], np.broadcast_to(want, got["out"].shape), (U[dtype] + 64 * U32) * size_of + U[dtype] * np.abs(want) + TINY[dtype])
    lse = q[0, 0, 1] * k[best[0], 0, 1] * scale + np.log(len(best))
    close(got["lse"], np.full(got["lse"].shape, lse), 8 * U32 * abs(lse))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offsets", [[10] + list(range(11, 51)), [0] * 20 + list(range(21)), [300] * 41, [0] * 41, [5, 50] + [7] * 38 + [40]])
def test_rows_of_no_sequence_take_no_part_behind_a_prefix(hip, dtype, offsets):
    # Rows before, behind and past the sequences hold NaN and infinities: neither
    # partial results nor outputs are written for them, and the others are whole.
    h, g, d, rows, prefix, keys = 4, 1, 64, 300, 700, 3
    n = len(offsets) - 1
    rng = np.random.default_rng(3)
    first, end = min(offsets), min(max(offsets), rows)
    q = rng.standard_normal((rows, h, d))
    q[:first], q[end:] = np.nan, np.inf
    q = rounded(q, dtype)
    k, v = (rounded(rng.standard_normal((n * keys, g, d)), dtype) for _ in range(2))
    pk, pv = (rounded(rng.standard_normal((prefix, g, d)), dtype) for _ in range(2))
    start, lens = np.arange(n) * keys, np.full(n, keys)
    p = Attention.of(heads=h, kv_heads=g, dim=d, sequences=n, q_rows=rows, kv_rows=n * keys, prefix_rows=prefix, dtype=dtype)
    parts = p.ranges()
    assert parts > 1
    bufs = {name: DeviceBuffer.from_array(np.asarray(a), dtype) for name, a in
            {"q": q, "k": k, "v": v, "prefix_k": pk, "prefix_v": pv, "out": np.full((rows, h, d), KEEP)}.items()}
    bufs.update({name: DeviceBuffer.from_array(np.asarray(a), "i32") for name, a in
                 {"q_offsets": offsets, "kv_start": start, "kv_len": lens}.items()})
    bufs["lse"] = DeviceBuffer.from_array(np.full((rows, h), KEEP), "f32")
    bufs["work"] = DeviceBuffer.from_array(np.full(p.work_needed() // 4, KEEP), "f32")
    for name, b in bufs.items():
        setattr(p, name, b.ptr)
    p.work_bytes = bufs["work"].nbytes
    p.launch()
    work = bufs["work"].to_numpy()
    sums = work[:parts * rows * h * d].reshape(parts, rows, h * d)
    stats = work[parts * rows * h * d:].reshape(parts, rows, 2 * h)
    for part in (sums, stats):
        assert (part[:, :first] == KEEP).all() and (part[:, end:] == KEEP).all()
    out, lse = bufs["out"].to_numpy().reshape(rows, h, d), bufs["lse"].to_numpy().reshape(rows, h)
    assert (out[:first] == KEEP).all() and (out[end:] == KEEP).all() and (lse[:first] == KEEP).all() and (lse[end:] == KEEP).all()
    if list(offsets) != sorted(offsets):
        assert np.isfinite(out[first:end]).all()   # rows in two sequences: either's keys
        return
    want, bound, want_lse, lse_bound, written = attention(q, k, v, np.minimum(offsets, rows), start, lens, scale=d ** -0.5, causal=True,
                                                          dtype=dtype, prefix_k=pk, prefix_v=pv)
    close(out[written], want[written], bound[written], "out")
    close(lse[written], want_lse[written], lse_bound[written], "lse")
