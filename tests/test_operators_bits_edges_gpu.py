"""Calls of the operators in 8 and 4 bits at the ends of their ranges:
magnitudes of queries, keys, values and scales, scores far from zero, long tails."""
import numpy as np
import pytest

from mlk2_amd import operators as op
from mlk2_amd.kernel_ir import KernelBuffer, KernelModule
from operators_bits_ref import load_bound, load_kv4, store_kv4
from operators_ref import TINY, U, U32, attention, rounded
from test_operators_gpu import KEEP, TYPES, close, run

pytestmark = pytest.mark.gpu

# Row blocks of 16 and 32 rows, one key range and several, a wave to a row:
# (heads, key/value heads, queries, keys).
SHAPES = {"token": (4, 2, [1, 1], [70, 33]), "ranges": (4, 1, [1, 1], [9000, 40]), "prompt": (4, 2, [40, 3], [90, 3])}


def heads_of(values):
    """A cache of these heads: codes and scales, and the numbers they stand for."""
    codes, scale = store_kv4(values)
    return codes, scale, load_kv4(codes, scale)


# ------------------------------------------------------------ attention_kv4 --
# Queries and keys whose products are about 1 while one of them is far from it.
FAR = {"large": (1e37, 1e-37), "largest": (2e38, 1e-38), "small": (1e-37, 1e37), "smallest": (1e-40, 1e38), "f16 large": (4e4, 1e-4),
       "f16 small": (1e-6, 1e6), "f16 smallest": (1e-7, 1e30)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256, 34])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", FAR)
def test_queries_far_from_one(hip, dtype, d, shape, name):
    # Every other row of a block has queries of the magnitude that makes scores of
    # about 1 with these keys, the others of about 1 (f16: of a tenth).
    if dtype == "f16" and not name.startswith("f16"):
        return
    size_q, size_k = FAR[name]
    h, g, q_lens, k_lens = SHAPES[shape]
    rng = np.random.default_rng(d)
    t, rows = sum(q_lens), sum(k_lens)
    size = np.where(np.arange(t * h).reshape(t, h, 1) % 2 == 0, size_q, min(1.0, 0.1 * size_q))
    q = rounded(rng.standard_normal((t, h, d)).clip(-1.5, 1.5) * size, dtype)
    k_codes, k_scale, k = heads_of((rng.standard_normal((rows, g, d)).clip(-3, 3) * size_k).astype(np.float32).astype(np.float64))
    v_codes, v_scale, v = heads_of(rounded(rng.standard_normal((rows, g, d)), "bf16"))
    offsets, start = np.concatenate([[0], np.cumsum(q_lens)]), np.concatenate([[0], np.cumsum(k_lens)[:-1]])
    km = op.attention_kv4_module(t, kv_rows=rows, sequences=len(q_lens), heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True)
    got = run(hip, km, {"q": q, "k_codes": k_codes, "k_scale": k_scale, "v_codes": v_codes, "v_scale": v_scale, "q_offsets": offsets,
                        "kv_start": start, "kv_len": k_lens})
    out, bound, lse, lse_bound, _ = attention(q, k, v, offsets, start, k_lens, scale=d ** -0.5, causal=True, dtype=dtype)
    close(got["out"], out, bound, "out")
    close(got["lse"], lse, lse_bound, "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 34])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale,size_q,size_k", [(1e20, 1e-18, 1e-2), (1e20, 1e-36, 1e16), (-1e3, 1e-5, 1e1), (5e2, 1e4, 1e-7), (1e2, 1.0, 1e-2),
                                                 (1e3, 1e-4, 1e37), (1e-20, 1e3, 1e17), (1e-20, 1e36, 1e-16)])
def test_scales_far_from_one(hip, dtype, d, shape, scale, size_q, size_k):
    # A scale of any size, where scale q k^T is about 1, or one key's is far the largest.
    if dtype == "f16" and not 6e-6 <= size_q <= 1e4:
        return
    h, g, q_lens, k_lens = SHAPES[shape]
    rng = np.random.default_rng(d)
    t, rows = sum(q_lens), sum(k_lens)
    q = rounded(rng.standard_normal((t, h, d)) * size_q, dtype)
    q[0] = 0.0
    k_codes, k_scale, k = heads_of((rng.standard_normal((rows, g, d)).clip(-3, 3) * size_k).astype(np.float32).astype(np.float64))
    v_codes, v_scale, v = heads_of(rounded(rng.standard_normal((rows, g, d)), "bf16"))
    offsets, start = np.concatenate([[0], np.cumsum(q_lens)]), np.concatenate([[0], np.cumsum(k_lens)[:-1]])
    km = op.attention_kv4_module(t, kv_rows=rows, sequences=len(q_lens), heads=h, kv_heads=g, dim=d, dtype=dtype, scale=scale, lse=True)
    got = run(hip, km, {"q": q, "k_codes": k_codes, "k_scale": k_scale, "v_codes": v_codes, "v_scale": v_scale, "q_offsets": offsets,
                        "kv_start": start, "kv_len": k_lens})
    out, bound, lse, lse_bound, _ = attention(q, k, v, offsets, start, k_lens, scale=scale, causal=True, dtype=dtype)
    close(got["lse"], lse, lse_bound, "lse")
    # Scores so large that a rounding of one decides who has the weight are left to the lse.
    sure = np.abs(scale) * size_q * size_k * d < 1e5
    assert np.isfinite(got["out"]).all()
    if sure:
        close(got["out"], out, bound, "out")
    else:
        close(got["out"][0], out[0], bound[0], "out")


def scores_about_one(hip, dtype, d, shape, scale, size_q, size_k, seed):
    h, g, q_lens, k_lens = SHAPES[shape]
    rng = np.random.default_rng(seed)
    t, rows = sum(q_lens), sum(k_lens)
    q = rounded(rng.standard_normal((t, h, d)).clip(-1.9, 1.9) * size_q, dtype)
    k_codes, k_scale, k = heads_of((rng.standard_normal((rows, g, d)).clip(-3, 3) * size_k).astype(np.float32).astype(np.float64))
    v_codes, v_scale, v = heads_of(rounded(rng.standard_normal((rows, g, d)), "bf16"))
    offsets, start = np.concatenate([[0], np.cumsum(q_lens)]), np.concatenate([[0], np.cumsum(k_lens)[:-1]])
    km = op.attention_kv4_module(t, kv_rows=rows, sequences=len(q_lens), heads=h, kv_heads=g, dim=d, dtype=dtype, scale=scale, lse=True)
    got = run(hip, km, {"q": q, "k_codes": k_codes, "k_scale": k_scale, "v_codes": v_codes, "v_scale": v_scale, "q_offsets": offsets,
                        "kv_start": start, "kv_len": k_lens})
    out, bound, lse, lse_bound, _ = attention(q, k, v, offsets, start, k_lens, scale=scale, causal=True, dtype=dtype)
    close(got["out"], out, bound, "out")
    close(got["lse"], lse, lse_bound, "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 256, 34])
@pytest.mark.parametrize("shape", ["token", "prompt"])
def test_every_power_of_a_scale(hip, dtype, d, shape):
    # Past 2^13 / log2 e the codes' factor ends and the queries take the rest.
    for n in list(range(-2, 16)) + [20, 40, 60]:
        scale = 1.3 * 2.0 ** n * (-1) ** n
        size_q = 2.0 ** -(n // 2) if dtype == "f16" else 1.0
        scores_about_one(hip, dtype, d, shape, scale, size_q if n < 20 else 0.01, 1 / (abs(scale) * d ** 0.5 * (size_q if n < 20 else 0.01)), n + 9)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("shape", ["token", "prompt"])
@pytest.mark.parametrize("scale", [None, 8000.0, 30000.0])
def test_queries_of_every_size(hip, dtype, d, shape, scale):
    # Sizes around those from which a row is taken times a power of two.
    scale = scale or d ** -0.5
    for e in (-125, -100, -65, -61, -60, -59, -30, 30, 55, 57, 59, 60, 61, 99, 100, 101, 103, 104, 105, 115, 117, 125):
        size_k = 2.0 ** -e / (scale * d ** 0.5)
        if 1e-43 < size_k < 1e37:
            scores_about_one(hip, dtype, d, shape, scale, 2.0 ** e, size_k, e + 200)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256, 34])
@pytest.mark.parametrize("shape", ["token", "ranges", "prompt"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [23, 26, 31, 40, 60])
def test_scores_far_from_zero(hip, dtype, d, shape, sign, size):
    """Scores of about 2^size: the keys with the largest share the weight.

    Scores are one product, the same for the same operands, and a sixteenth and
    more apart, which is 2^19 and more; so the result is a mean of n values, each
    product and sum within 2^-24 n, the weights and out rounded once."""
    h, g, q_lens, k_lens = SHAPES[shape]
    rng = np.random.default_rng(d)
    t, rows = sum(q_lens), sum(k_lens)
    q = np.zeros((t, h, d))
    q[..., 1] = 1.375 * 2.0 ** 8
    k_scale = rng.choice([1.25, 1.3828125, 1.5] if sign > 0 else [1.8671875, 1.99], (rows, g)).astype(np.float32).astype(np.float64)
    best, start = [], np.concatenate([[0], np.cumsum(k_lens)[:-1]])
    for s, n, m in zip(start, k_lens, q_lens):
        best.append(s + np.sort(rng.choice(n - m + 1, min(7, n - m + 1), replace=False)))
        k_scale[best[-1]] = 1.7109375
    k_codes = np.zeros((rows, g, d // 2))
    k_codes[..., 0] = (7 if sign > 0 else 15) << 4   # element 1: 6, the others 0
    v_codes, v_scale, v = heads_of(rounded(rng.standard_normal((rows, g, d)), "bf16"))
    scale = 2.0 ** (size - 12)
    offsets = np.concatenate([[0], np.cumsum(q_lens)])
    km = op.attention_kv4_module(t, kv_rows=rows, sequences=len(q_lens), heads=h, kv_heads=g, dim=d, dtype=dtype, scale=scale, lse=True)
    got = run(hip, km, {"q": q, "k_codes": k_codes, "k_scale": k_scale, "v_codes": v_codes, "v_scale": v_scale, "q_offsets": offsets,
                        "kv_start": start, "kv_len": k_lens})
    for i, at in enumerate(best):
        rows_of = slice(offsets[i], offsets[i + 1])
        want, size_of = (np.repeat(x.mean(0), h // g, 0) for x in (v[at], np.abs(v[at])))
        close(got["out"][rows_of], np.broadcast_to(want, got["out"][rows_of].shape),
              (U[dtype] + 64 * U32) * size_of + U[dtype] * np.abs(want) + TINY[dtype], "out")
        lse = sign * 1.375 * 2.0 ** 8 * 6 * 1.7109375 * scale + np.log(len(at))
        close(got["lse"][rows_of], np.full(got["lse"][rows_of].shape, lse), 8 * U32 * abs(lse), "lse")


TAILS = {"token": (4, 2, 1, 300), "ranges": (4, 1, 1, 20000), "prompt": (4, 2, 40, 900)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("name", TAILS)
def test_tail_behind_one_key(hip, dtype, d, name):
    """One key with the largest score and no value, all others 2^-26 of it, with
    values about 1: what is left of a tail in rounded weights.

    Bound, scores being exact products: a weight times its value's scale is within
    half a step of the type's of itself, its exponential and the running sums
    within (n + 64) 2^-24, and out is rounded once."""
    h, g, nq, nk = TAILS[name]
    rng = np.random.default_rng(nk)
    q = np.zeros((nq, h, d))
    q[..., 0] = 1.0
    k_codes, k_scale = np.zeros((nk, g, d // 2)), np.full((nk, g), 3.0)
    k_codes[..., 0] = 15   # -6 * 3
    k_codes[nk // 3] = 0
    v = 0.5 + rng.random((nk, g, d))
    v[nk // 3] = 0.0
    v_codes, v_scale, v = heads_of(rounded(v, "bf16"))
    km = op.attention_kv4_module(nq, kv_rows=nk, sequences=1, heads=h, kv_heads=g, dim=d, dtype=dtype, causal=False, scale=1.0, lse=True)
    got = run(hip, km, {"q": q, "k_codes": k_codes, "k_scale": k_scale, "v_codes": v_codes, "v_scale": v_scale, "q_offsets": [0, nq],
                        "kv_start": [0], "kv_len": [nk]})
    w = np.full(nk, np.exp(-18.0))
    w[nk // 3] = 1.0
    want = np.repeat((w[:, None, None] * v).sum(0) / w.sum(), h // g, 0)
    sum_error = (nk + 64) * U32
    close(got["out"], np.broadcast_to(want, got["out"].shape), want * (2 * U[dtype] + 2 * sum_error) + TINY[dtype], "out")
    close(got["lse"], np.full((nq, h), np.log(w.sum())), sum_error + 2.0 ** -22, "lse")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256, 34])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [1e-20, 1e-26, 1e-32, 1e-36, 1e20, 1e32, 1e35])
def test_values_far_from_one(hip, dtype, d, shape, size):
    # Values all of one magnitude. A weight times its value's scale is off by half a
    # step of bf16's least, 2^-134, where it is that small: 6 times that for a key's
    # largest code, over a sum of weights of 1 at least.
    h, g, q_lens, k_lens = SHAPES[shape]
    rng = np.random.default_rng(d)
    t, rows = sum(q_lens), sum(k_lens)
    q = rounded(rng.standard_normal((t, h, d)), dtype)
    k_codes, k_scale, k = heads_of(rounded(rng.standard_normal((rows, g, d)), "bf16"))
    v_codes, v_scale, v = heads_of((rng.standard_normal((rows, g, d)).clip(-3, 3) * size).astype(np.float32).astype(np.float64))
    offsets, start = np.concatenate([[0], np.cumsum(q_lens)]), np.concatenate([[0], np.cumsum(k_lens)[:-1]])
    km = op.attention_kv4_module(t, kv_rows=rows, sequences=len(q_lens), heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True)
    got = run(hip, km, {"q": q, "k_codes": k_codes, "k_scale": k_scale, "v_codes": v_codes, "v_scale": v_scale, "q_offsets": offsets,
                        "kv_start": start, "kv_len": k_lens})
    out, bound, *_ = attention(q, k, v, offsets, start, k_lens, scale=d ** -0.5, causal=True, dtype=dtype)
    close(got["out"], out, bound + max(k_lens) * 6 * 2.0 ** -134, "out")


# ---------------------------------------------------------------- matmul_i8 --
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(3, 40, 256), (40, 90, 512), (70, 130, 4096), (70, 130, 8192), (300, 260, 320)])
@pytest.mark.parametrize("size_a,size_b", [(1e36, 1e-30), (1e-30, 1e36), (1e-40, 1e37), (1e37, 1e-40), (1e-20, 1e-10), (1e10, 1e15)])
def test_matmul_scales_far_from_one(hip, dtype, m, n, k, size_a, size_b):
    # Rows of about 1e38, or 1e-38, whose products with the other operand's are in
    # range. Three roundings of f32, then one to the type.
    rng = np.random.default_rng(m + k)
    a, b = rng.integers(-127, 128, (m, k)), rng.integers(-127, 128, (n, k))
    a[0] = 0
    sa, sb = ((size * (0.5 + rng.random(x))).astype(np.float32).astype(np.float64) for size, x in ((size_a, m), (size_b, n)))
    got = run(hip, op.matmul_i8_module(m, n, k, dtype=dtype), {"a": a, "b": b, "a_scale": sa, "b_scale": sb})["out"]
    want = (a.astype(np.float64) @ b.T.astype(np.float64)) * sa[:, None] * sb
    close(got, want, (3 * U32 * (1 + U[dtype]) + U[dtype]) * (1 + 4 * U32) * np.abs(want) + TINY["f32"] + TINY[dtype], "out")


@pytest.mark.parametrize("m,n,k", [(3, 40, 256), (70, 130, 4096), (300, 260, 320)])
def test_matmul_sums_of_zero_under_any_scale(hip, m, n, k):
    a, b = np.zeros((m, k)), np.ones((n, k))
    for size in (3e38, 1e-45):
        got = run(hip, op.matmul_i8_module(m, n, k, dtype="f32"), {"a": a, "b": b, "a_scale": np.full(m, size), "b_scale": np.full(n, 3e38)})["out"]
        assert (got == 0).all()


# ---------------------------------------------------------- buffers, lengths --
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 34])
@pytest.mark.parametrize("rows", [300, 9000])
def test_offsets_and_lengths_are_clipped(hip, dtype, d, rows):
    # Offsets and lengths outside the buffers, and below 0: what lies in them counts.
    h, g, t = 4, 2, 50
    offsets = [-5, 20, 21, 21, 45, 2 ** 31 - 1]
    start, lens = [rows - 100, -1, 7, rows, 0], [2 ** 31 - 1, 50, 40, 3, -9]
    for offsets, start, lens in ((offsets, start, lens), ([0, 10, 20, 30, 40, 50], [0, rows - 1, 2 ** 31 - 1, -2 ** 31, 5], [rows + 1, 2, 1, 2 ** 31 - 1, 1])):
        rng = np.random.default_rng(d)
        q = rounded(rng.standard_normal((t, h, d)), dtype)
        k_codes, k_scale, k = heads_of(rounded(rng.standard_normal((rows, g, d)), "bf16"))
        v_codes, v_scale, v = heads_of(rounded(rng.standard_normal((rows, g, d)), "bf16"))
        km = op.attention_kv4_module(t, kv_rows=rows, sequences=5, heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True)
        got = run(hip, km, {"q": q, "k_codes": k_codes, "k_scale": k_scale, "v_codes": v_codes, "v_scale": v_scale, "q_offsets": offsets,
                            "kv_start": start, "kv_len": lens})
        held = [max(0, min(rows - s, n)) if 0 <= s < rows else 0 for s, n in zip(start, lens)]
        out, bound, lse, lse_bound, written = attention(q, k, v, np.clip(offsets, 0, t), [s if n > 0 else 0 for s, n in zip(start, held)], held,
                                                        scale=d ** -0.5, causal=True, dtype=dtype)
        assert written.all()
        close(got["out"], out, bound, "out")
        real = np.isfinite(lse)
        close(got["lse"][real], lse[real], lse_bound[real], "lse")
        assert (got["lse"][~real] == -np.inf).all() and not real.all()


@pytest.mark.parametrize("build", [lambda: op.quantize_rows_module(0, 8), lambda: op.matmul_i8_module(0, 8, 16), lambda: op.linear_i8_module(0, 8, 16),
                                   lambda: op.store_load_kv4_module(0, cache_rows=9, kv_heads=2, dim=64), lambda: op.store_kv4_module(0, kv_heads=2, dim=64),
                                   lambda: op.attention_kv4_module(0, kv_rows=4000, sequences=1, heads=4, kv_heads=2, dim=64, lse=True)])
def test_no_rows(hip, build):
    km = build()
    host = {b.name: np.zeros(b.dims) for b in km.buffers if b.is_input}
    got = run(hip, km, {**host, **{b.name: np.full(b.dims, 9) for b in km.buffers if b.name.endswith("codes")}})
    for name, a in got.items():
        assert (a == (9 if name.endswith("codes") else KEEP)).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_an_empty_cache(hip, dtype):
    # A cache of no rows: nothing is stored or loaded, and queries see no keys.
    t, h, g, d = 5, 4, 2, 64
    x = np.ones((t, g, d))
    got = run(hip, op.store_load_kv4_module(t, cache_rows=0, kv_heads=g, dim=d, dtype=dtype), {"k": x, "v": x, "slots": np.arange(t)})
    assert (got["k_read"] == KEEP).all() and (got["v_read"] == KEEP).all()
    empty = {f"{p}_{w}": np.zeros((0, g, d // 2) if w == "codes" else (0, g)) for p in "kv" for w in ("codes", "scale")}
    km = op.attention_kv4_module(t, kv_rows=0, sequences=2, heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True)
    got = run(hip, km, {"q": np.ones((t, h, d)), "q_offsets": [0, 2, 4], "kv_start": [0, 0], "kv_len": [3, 0], **empty})
    assert (got["out"][:4] == 0).all() and (got["lse"][:4] == -np.inf).all() and (got["out"][4:] == KEEP).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,extra", [(64, 0), (64, 8), (80, 8), (128, 3)])
def test_keys_and_values_in_one_buffer(hip, dtype, d, extra):
    # Codes of k and v as columns of one buffer's rows, `extra` bytes behind them;
    # attended, and read back.
    h, g, rows, lens = 4, 2, 500, [90, 400]
    rng = np.random.default_rng(d + extra)
    q = rounded(rng.standard_normal((41, h, d)), dtype)
    both = [heads_of(rounded(rng.standard_normal((rows, g, d)), "bf16")) for _ in "kv"]
    part, width = g * d // 2, g * d + extra
    codes = np.full((rows, width), 255)
    codes[:, :part], codes[:, part:2 * part] = (b[0].reshape(rows, part) for b in both)
    km = KernelModule(name="one buffer")

    def buf(name, kind, dims, out=False):
        return km.add_buffer(KernelBuffer(name, kind, is_input=not out, is_output=out, elements=int(np.prod(dims)), dims=list(dims)))

    cache = buf("codes", "u8", [rows, width])
    ids = {"k_codes": cache, "v_codes": cache, "k_scale": buf("k_scale", "f32", [rows, g]), "v_scale": buf("v_scale", "f32", [rows, g])}
    at = {"v_codes": part}
    sides = {"q": buf("q", dtype, [41, h, d]), "q_offsets": buf("q_offsets", "i32", [3]), "kv_start": buf("kv_start", "i32", [2]),
             "kv_len": buf("kv_len", "i32", [2]), "out": buf("out", dtype, [41, h, d], True)}
    op.add_attention_kv4(km, {**ids, **sides}, heads=h, kv_heads=g, dim=d, columns=at)
    op.add_load_kv4(km, {**ids, "k_out": buf("k", dtype, [rows, g, d], True), "v_out": buf("v", dtype, [rows, g, d], True)}, kv_heads=g, dim=d, columns=at)
    got = run(hip, km, {"codes": codes, "k_scale": both[0][1], "v_scale": both[1][1], "q": q, "q_offsets": [0, 40, 41], "kv_start": [3, 100], "kv_len": lens})
    out, bound, *_ = attention(q, both[0][2], both[1][2], [0, 40, 41], [3, 100], lens, scale=d ** -0.5, causal=True, dtype=dtype)
    close(got["out"], out, bound, "out")
    for name, (_, _, want) in zip("kv", both):
        close(got[name], want, load_bound(want, dtype), name)
