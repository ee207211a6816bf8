"""The operators in 8 and 4 bits on the GPU against plain f64 references, at the
sizes, masks, strides and values where they could go wrong."""
import numpy as np
import pytest

from mlk2_amd import operators as op
from mlk2_amd.backend import DeviceBuffer
from mlk2_amd.kernel_ir import KernelBuffer, KernelModule
from operators_bits_ref import load_bound, load_kv4, matmul_i8, quantize_rows, store_kv4
from operators_ref import attention, rounded
from test_operators_gpu import KEEP, TYPES, close, run
from test_score_two_pass_gpu import _Capture

pytestmark = pytest.mark.gpu
LIMIT = {"bf16": 3.3e38, "f16": 65504.0, "f32": 3.4e38}
SMALL = {"bf16": 2.0 ** -133, "f16": 2.0 ** -24, "f32": 2.0 ** -149}


def same(got, want, what=""):
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} differ, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}"


def rows_of(rng, shape, dtype):
    """Rows of unlike sizes; some elements half way between two codes."""
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:-1]))[..., None]
    return rounded(x, dtype)


# ------------------------------------------------------------ quantize_rows --
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (1, 4096), (64, 4096), (7, 1000), (2, 8191), (33, 2056), (3, 40000),
                                       (1030, 512), (4, 16384), (3, 8), (2, 24)])
def test_quantize_rows(hip, dtype, rows, cols):
    x = rows_of(np.random.default_rng(rows * 31 + cols), (rows, cols), dtype)
    codes, scale = quantize_rows(x)
    got = run(hip, op.quantize_rows_module(rows, cols, dtype=dtype), {"x": x, "codes": np.zeros((rows, cols))})
    same(got["scale"], scale, "scale")
    same(got["codes"], codes, "codes")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [127, 128, 4096])
def test_quantize_rows_at_the_borders(hip, dtype, cols):
    # Values on and next to every border of scales that are powers of two and not.
    x = np.zeros((40, cols))
    rng = np.random.default_rng(5)
    for r in range(40):
        top = rounded(np.array([127.0 * 2.0 ** (r % 7 - 3) if r % 2 else 1 + rng.random()]), dtype)[0]
        half = (rng.integers(-127, 127, cols) + 0.5) * top / 127
        x[r] = np.clip(half, -top, top)
        x[r, r % cols] = top if r % 3 else -top
    x = rounded(x, dtype)
    codes, scale = quantize_rows(x)
    got = run(hip, op.quantize_rows_module(40, cols, dtype=dtype), {"x": x, "codes": np.zeros((40, cols))})
    same(got["scale"], scale, "scale")
    same(got["codes"], codes, "codes")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [9, 512])
def test_quantize_rows_far_values(hip, dtype, cols):
    x = np.zeros((12, cols))
    x[1, 0], x[2, 1], x[3, cols - 1], x[4, 2] = np.nan, np.inf, -np.inf, -0.0
    x[5] = LIMIT[dtype]
    x[6] = SMALL[dtype] * np.arange(cols)
    x[7] = SMALL[dtype]
    x[8, :3] = SMALL[dtype] * np.array([1, 127, 63])
    x[9] = rounded(LIMIT[dtype] * np.linspace(-1, 1, cols), dtype)
    x[10, 0], x[10, 1] = LIMIT[dtype], SMALL[dtype]
    x[11] = 1e-30 * np.linspace(-1, 1, cols)
    x = rounded(x, dtype)
    codes, scale = quantize_rows(x)
    got = run(hip, op.quantize_rows_module(12, cols, dtype=dtype), {"x": x, "codes": np.ones((12, cols))})
    same(got["scale"], scale, "scale")
    same(got["codes"], codes, "codes")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at,width,cols,codes_at,codes_width", [(3, 200, 128, 5, 150), (8, 256, 128, 16, 256), (0, 129, 128, 0, 131), (16, 4200, 4096, 1, 4100)])
def test_quantize_rows_columns_of_wider_rows(hip, dtype, at, width, cols, codes_at, codes_width):
    rng = np.random.default_rng(at + width)
    x = rows_of(rng, (6, width), dtype)
    x[:, :at] = np.nan
    x[:, at + cols:] = np.inf
    km = KernelModule(name="wide")
    ids = {"x": km.add_buffer(KernelBuffer("x", dtype, is_input=True, elements=6 * width, dims=[6, width])),
           "codes_out": km.add_buffer(KernelBuffer("codes", "i8", is_output=True, elements=6 * codes_width, dims=[6, codes_width])),
           "scale_out": km.add_buffer(KernelBuffer("scale", "f32", is_output=True, elements=6, dims=[6]))}
    op.add_quantize_rows(km, ids, cols=cols, columns={"x": at, "codes_out": codes_at})
    got = run(hip, km, {"x": x})
    codes, scale = quantize_rows(x[:, at:at + cols])
    same(got["scale"], scale)
    same(got["codes"][:, codes_at:codes_at + cols], codes)
    rest = np.delete(got["codes"], np.s_[codes_at:codes_at + cols], axis=1)
    assert (rest == KEEP).all()


# ---------------------------------------------------------------- matmul_i8 --
def matmul_case(hip, m, n, k, dtype, *, bias=False, at=None, width=None, noalloc=False, extreme=False):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a, b = rng.integers(-127, 128, (m, k)), rng.integers(-127, 128, (n, k))
    if extreme:   # the largest sums there are
        a, b = np.full((m, k), -128), np.full((n, k), -128)
        b[n // 2:] = 127
    sa, sb = (np.exp(rng.standard_normal(x)).astype(np.float32).astype(np.float64) * 1e-3 for x in (m, n))
    sa, sb = sa.astype(np.float32).astype(np.float64), sb.astype(np.float32).astype(np.float64)
    bs = rng.standard_normal(n).astype(np.float32).astype(np.float64) if bias else None
    host = {"a_scale": sa, "b_scale": sb, "bias": bs}
    out, bound = matmul_i8(a, sa, b, sb, bs, dtype)
    if at is None:
        host.update(a=a, b=b)
        got = run(hip, op.matmul_i8_module(m, n, k, dtype=dtype, bias=bias), {x: y for x, y in host.items() if y is not None}, noalloc)
        close(got["out"], out, bound, "out")
        return
    km = KernelModule(name="wide")
    ids = {}
    for name, r, code, part in (("a", m, "i8", a), ("b", n, "i8", b)):
        full = rng.integers(-128, 128, (r, width[name]))
        full[:, at[name]:at[name] + k] = part
        host[name] = full
        ids[name] = km.add_buffer(KernelBuffer(name, code, is_input=True, elements=full.size, dims=list(full.shape)))
    for name, r in (("a_scale", m), ("b_scale", n)) + ((("bias", n),) if bias else ()):
        ids[name] = km.add_buffer(KernelBuffer(name, "f32", is_input=True, elements=r, dims=[r]))
    ids["out"] = km.add_buffer(KernelBuffer("out", dtype, is_output=True, elements=m * width["out"], dims=[m, width["out"]]))
    op.add_matmul_i8(km, ids, cols=n, inner=k, columns=at)
    got = run(hip, km, {x: y for x, y in host.items() if y is not None}, noalloc)["out"]
    close(got[:, at["out"]:at["out"] + n], out, bound, "out")
    assert (np.delete(got, np.s_[at["out"]:at["out"] + n], axis=1) == KEEP).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 1, 16), (2, 3, 5), (1, 64, 64), (16, 16, 64), (17, 33, 65), (1, 1000, 4096), (3, 500, 1040),
                                   (32, 260, 777), (33, 128, 128), (64, 300, 2000), (65, 130, 200), (100, 100, 4000), (128, 128, 64),
                                   (129, 257, 192), (200, 400, 1008), (256, 256, 256), (300, 600, 500), (260, 1030, 640), (700, 900, 96)])
def test_matmul_sizes(hip, dtype, m, n, k):
    matmul_case(hip, m, n, k, dtype, bias=(m + n) % 2 == 0)


@pytest.mark.parametrize("m,n,k", [(1, 20, 131071), (70, 65, 131071), (5, 40, 131064), (300, 300, 20000), (8, 8, 100000), (130, 140, 65536)])
def test_matmul_largest_sums(hip, m, n, k):
    matmul_case(hip, m, n, k, "f32", extreme=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1100, 1100, 128), (520, 2050, 448), (2049, 300, 320)])
def test_matmul_many_tiles(hip, dtype, m, n, k):
    matmul_case(hip, m, n, k, dtype, bias=True)


@pytest.mark.parametrize("m,n,k", [(33, 64, 2048), (64, 130, 2064), (32, 70, 8208), (17, 70, 16384), (40, 8200, 64), (32, 6500, 48), (16, 6400, 80),
                                   (256, 5120, 80), (250, 5100, 96), (640, 5120, 72), (600, 5100, 144), (2040, 4090, 400), (2560, 4096, 64), (2500, 4000, 80)])
def test_matmul_each_tile(hip, m, n, k):
    matmul_case(hip, m, n, k, "bf16", bias=True)


@pytest.mark.parametrize("n", [66, 5120, 9000])
@pytest.mark.parametrize("m", [66, 250])
def test_matmul_every_count_of_steps(hip, m, n):
    for steps in list(range(1, 24)) if n == 66 else (1, 2, 5, 6, 7, 8, 9, 13):
        matmul_case(hip, m, n, 64 * steps - (16 if steps % 2 else 0), "f32")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(5, 70, 100), (40, 90, 256), (150, 140, 130), (300, 270, 320)])
@pytest.mark.parametrize("at,extra", [(dict(a=1, b=3, out=5), 11), (dict(a=16, b=32, out=8), 48), (dict(a=0, b=0, out=0), 16), (dict(a=4, b=8, out=2), 12)])
def test_matmul_columns_of_wider_rows(hip, dtype, m, n, k, at, extra):
    width = dict(a=at["a"] + k + extra, b=at["b"] + k + extra, out=at["out"] + n + extra)
    matmul_case(hip, m, n, k, dtype, bias=True, at=at, width=width)


@pytest.mark.parametrize("m,n,k", [(4, 40, 4096), (100, 100, 8000), (300, 300, 640)])
def test_matmul_without_allocation(hip, m, n, k):
    matmul_case(hip, m, n, k, "f16", noalloc=True)


def test_matmul_scales_that_are_not_finite(hip):
    a, b = np.ones((20, 64)), np.ones((24, 64))
    sa, sb = np.ones(20), np.ones(24)
    sa[3], sa[5], sb[7], sa[6] = np.nan, np.inf, -np.inf, 0.0
    a[5] = 0
    got = run(hip, op.matmul_i8_module(20, 24, 64, dtype="f32"), {"a": a, "b": b, "a_scale": sa, "b_scale": sb})["out"]
    with np.errstate(invalid="ignore"):
        want = (a @ b.T) * sa[:, None] * sb
    same(got, want)


@pytest.mark.parametrize("rows", [0, 1])
def test_matmul_no_rows(hip, rows):
    got = run(hip, op.linear_i8_module(rows, 8, 32), {"x": np.ones((rows, 32)), "b": np.ones((8, 32)), "b_scale": np.ones(8)})
    assert got["out"].shape == (rows, 8) and (got["out"] == 32).all()


# ------------------------------------------------------- store_kv4, load_kv4 --
def cache_of(rng, rows, g, d, dtype="bf16"):
    """A cache's codes and scales, and the numbers they stand for, of k and v."""
    host, values = {}, []
    for part in "kv":
        codes, scale = store_kv4(rounded(rng.standard_normal((rows, g, d)), dtype))
        host[f"{part}_codes"], host[f"{part}_scale"] = codes, scale
        values.append(load_kv4(codes, scale))
    return host, values


def store_case(hip, t, g, d, dtype, cache=None, valid=None, x=None):
    rng = np.random.default_rng(t + d)
    x = rows_of(rng, (2, t, g, d), dtype) if x is None else x
    rows = t if cache is None else cache
    km = op.store_kv4_module(t, kv_heads=g, dim=d, dtype=dtype, cache_rows=cache, sequences=2 if valid is not None else None)
    host = {"k": x[0], "v": x[1], "q_offsets": [0, 0, valid]}
    slots = np.arange(t)
    if cache is not None:
        slots = rng.permutation(cache)[:t]
        slots[t // 2] = cache
        if t > 3:
            slots[0], slots[1] = -1, -2 ** 31
        host["slots"] = slots
    old = {}
    for part in "kv":
        old[f"{part}_codes"] = host[f"{part}_codes"] = rng.integers(0, 256, (rows, g, d // 2))
        old[f"{part}_scale"] = host[f"{part}_scale"] = np.full((rows, g), KEEP)
    got = run(hip, km, host)
    n = t if valid is None else max(0, min(t, valid))
    for i, part in enumerate("kv"):
        codes, scale = store_kv4(x[i])
        want_codes, want_scale = old[f"{part}_codes"].copy(), old[f"{part}_scale"].copy()
        for j in range(n):
            if 0 <= slots[j] < rows:
                want_codes[slots[j]], want_scale[slots[j]] = codes[j], scale[j]
        same(got[f"{part}_scale"], want_scale, part + " scale")
        same(got[f"{part}_codes"], want_codes, part + " codes")
    # And back, over what the cache holds now.
    km = op.load_kv4_module(t, kv_heads=g, dim=d, dtype=dtype, cache_rows=cache, sequences=2 if valid is not None else None)
    cached = {f"{part}_{what}": got[f"{part}_{what}"] for part in "kv" for what in ("codes", "scale")}
    read = run(hip, km, {**host, **cached, "k": np.full((t, g, d), KEEP), "v": np.full((t, g, d), KEEP)})
    for i, part in enumerate("kv"):
        numbers = load_kv4(cached[f"{part}_codes"], cached[f"{part}_scale"])
        want, bound = np.full((t, g, d), KEEP), np.zeros((t, g, d))
        for j in range(n):
            if 0 <= slots[j] < rows:
                want[j] = numbers[slots[j]]
                bound[j] = load_bound(want[j], dtype)
        nan = np.isnan(want)
        assert (np.isnan(read[part]) == nan).all()
        close(read[part][~nan], want[~nan], bound[~nan], part + " read")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [2, 8, 10, 20, 64, 80, 96, 128, 130, 200, 256])
def test_store_dims(hip, dtype, d):
    store_case(hip, 5, 3, d, dtype, cache=11)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,g,d", [(1, 1, 128), (1, 8, 128), (64, 8, 128), (1031, 2, 64), (3, 40, 96), (77, 5, 256)])
def test_store_sizes(hip, dtype, t, g, d):
    store_case(hip, t, g, d, dtype, cache=t + 9)


@pytest.mark.parametrize("kw", [dict(), dict(valid=17), dict(valid=0), dict(valid=9, cache=31), dict(valid=20, cache=20),
                                dict(valid=-5), dict(valid=99, cache=30), dict(valid=-2 ** 31)])
@pytest.mark.parametrize("d", [64, 36])
def test_store_options(hip, kw, d):
    store_case(hip, 20, 2, d, "f16", **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 34])
def test_store_at_the_borders_and_far_values(hip, dtype, d):
    rng = np.random.default_rng(d)
    x = np.zeros((2, 40, 2, d))
    for r in range(30):   # on and next to every border
        top = rounded(np.array([6.0 * 2.0 ** (r % 7 - 3) if r % 2 else 1 + rng.random()]), dtype)[0]
        size = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], (2, 2, d)) * top / 6
        x[:, r] = size * rng.choice([-1, 1], (2, 2, d))
        x[:, r, :, r % d] = top if r % 3 else -top
    x[0, 30, 0, 1], x[0, 31, 1, 0], x[1, 32, 0, d - 1] = np.nan, np.inf, -np.inf
    x[0, 33] = -0.0
    x[0, 34] = LIMIT[dtype]
    x[1, 35] = SMALL[dtype] * np.arange(d)
    x[1, 36] = SMALL[dtype]
    x[0, 37] = SMALL[dtype] * (np.arange(d) % 7 - 3)
    x[0, 38] = 1e-30 * np.linspace(-1, 1, d)
    store_case(hip, 40, 2, d, dtype, x=rounded(x, dtype))


def test_store_columns_of_a_fused_projection(hip):
    t, h, g, d = 9, 4, 2, 64
    rng = np.random.default_rng(8)
    qkv = rounded(rng.standard_normal((t, (h + 2 * g) * d)), "bf16")
    km = KernelModule(name="fused")
    x = km.add_buffer(KernelBuffer("qkv", "bf16", is_input=True, elements=qkv.size, dims=list(qkv.shape)))
    ids = {"k": x, "v": x}
    for part in "kv":   # codes of both in one buffer's rows
        ids[f"{part}_scale_out"] = km.add_buffer(KernelBuffer(f"{part}_scale", "f32", is_output=True, elements=t * g, dims=[t, g]))
    ids["k_codes_out"] = ids["v_codes_out"] = km.add_buffer(KernelBuffer("codes", "u8", is_output=True, elements=t * 2 * g * d // 2, dims=[t, g * d]))
    op.add_store_kv4(km, ids, kv_heads=g, dim=d, columns={"k": h * d, "v": (h + g) * d, "v_codes_out": g * d // 2})
    got = run(hip, km, {"qkv": qkv, "codes": np.zeros((t, g * d))})
    heads = qkv.reshape(t, h + 2 * g, d)
    for i, part in enumerate("kv"):
        codes, scale = store_kv4(heads[:, h + i * g:h + (i + 1) * g])
        same(got[f"{part}_scale"], scale)
        same(got["codes"][:, i * g * d // 2:(i + 1) * g * d // 2], codes.reshape(t, -1))


# ------------------------------------------------------------ attention_kv4 --
def attention_case(hip, q_lens, k_lens, h, g, d, dtype, *, causal=True, spare=0, scale=None, gap=0, noalloc=False, magnitude=1.0,
                   poison=False, rows=None):
    """Sequences in a cache whose rows have `gap` others between them."""
    rng = np.random.default_rng(sum(q_lens) * 7 + sum(k_lens) + d)
    n, t = len(q_lens), sum(q_lens) + spare
    start = np.concatenate([[0], np.cumsum(np.asarray(k_lens) + gap)[:-1]]).astype(int) + gap
    rows = rows or int(sum(k_lens) + gap * (n + 1))
    q = rounded(magnitude * rng.standard_normal((t, h, d)), dtype)
    host, (k, v) = cache_of(rng, rows, g, d)
    if poison:   # rows that no sequence holds
        held = np.zeros(rows, dtype=bool)
        for s, m in zip(start, k_lens):
            held[s:s + m] = True
        host["k_scale"][~held], host["v_scale"][~held] = np.nan, np.inf
    host.update(q=q, q_offsets=np.concatenate([[0], np.cumsum(q_lens)]), kv_start=start, kv_len=k_lens)
    km = op.attention_kv4_module(t, kv_rows=rows, sequences=n, heads=h, kv_heads=g, dim=d, dtype=dtype, causal=causal, scale=scale, lse=True)
    got = run(hip, km, host, noalloc)
    out, bound, lse, lse_bound, written = attention(q, k, v, host["q_offsets"], start, k_lens, scale=scale or d ** -0.5, causal=causal,
                                                    dtype=dtype)
    close(got["out"][written], out[written], bound[written], "out")
    real = np.isfinite(lse) & written[:, None]
    close(got["lse"][real], lse[real], lse_bound[real], "lse")
    assert (got["lse"][~np.isfinite(lse) & written[:, None]] == -np.inf).all()
    assert (got["out"][~written] == KEEP).all() and (got["lse"][~written] == KEEP).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [2, 8, 34, 32, 64, 80, 96, 128, 160, 192, 256])
def test_attention_dims(hip, dtype, causal, d):
    attention_case(hip, [70, 3], [70, 3], 4, 2, d, dtype, causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_lens,k_lens", [
    ([1], [1]), ([1], [2]), ([2], [1]), ([1, 1, 1], [0, 5, 1]), ([0, 3, 0], [4, 3, 0]), ([5, 0], [0, 0]),
    ([130], [130]), ([129], [300]), ([64], [64]), ([63, 65, 1], [63, 65, 1]), ([40], [17]), ([7, 19, 1, 33], [64, 128, 65, 191]),
    ([257], [257]), ([1] * 9, [1, 31, 32, 33, 63, 64, 65, 500, 127]), ([3] * 5, [700, 3, 2, 64, 1])])
def test_attention_lengths(hip, dtype, q_lens, k_lens):
    attention_case(hip, q_lens, k_lens, 4, 2, 64, dtype, spare=3)
    attention_case(hip, q_lens, k_lens, 4, 1, 128, dtype, causal=False, spare=1)


@pytest.mark.parametrize("h,g", [(1, 1), (3, 3), (3, 1), (6, 2), (8, 1), (12, 4), (40, 8), (17, 1), (33, 1)])
def test_attention_heads(hip, h, g):
    attention_case(hip, [33, 1, 0, 5], [50, 200, 3, 5], h, g, 64, "bf16")
    attention_case(hip, [1, 1], [333, 40], h, g, 128, "f16", causal=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 72, 34])
def test_attention_rows_of_no_sequence_reach_nothing(hip, dtype, d):
    attention_case(hip, [1, 40, 3], [70, 45, 129], 4, 2, d, dtype, gap=5, poison=True, spare=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.5, -0.125, 3.0])
def test_attention_scales(hip, dtype, scale):
    attention_case(hip, [20, 1], [40, 300], 4, 2, 64, dtype, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_long(hip, dtype):
    attention_case(hip, [1], [20000], 8, 2, 64, dtype)
    attention_case(hip, [1, 2], [9000, 31], 4, 1, 128, dtype, noalloc=True)
    attention_case(hip, [300], [2100], 4, 2, 128, dtype)


def test_attention_hidden_keys_that_are_not_numbers(hip):
    # A causal mask hides keys whose scales are NaN or infinite.
    rng = np.random.default_rng(2)
    for dtype in TYPES:
        host, (k, v) = cache_of(rng, 100, 2, 64)
        host["k_scale"][60:] = np.nan
        host["v_scale"][60:] = np.inf
        q = rounded(rng.standard_normal((100, 4, 64)), dtype)
        host.update(q=q, q_offsets=[0, 100])
        km = op.attention_kv4_module(100, sequences=1, heads=4, kv_heads=2, dim=64, dtype=dtype)
        got = run(hip, km, host)["out"]
        out, bound, *_ = attention(q[:60], k, v, [0, 60], [0], [60], scale=0.125, causal=True, dtype=dtype)
        close(got[:60], out, bound, dtype)
        assert np.isnan(got[60:]).all()


# ------------------------------------------------------------ run of them all --
def layer(t, h, g, d, hidden, cache, seqs, dtype):
    """A decoder layer's attention: x in, the cache's rows written and read, y out."""
    km = KernelModule(name="layer")

    def buf(name, dt, dims, out=False):
        return km.add_buffer(KernelBuffer(name, dt, is_input=not out, is_output=out, elements=int(np.prod(dims)), dims=list(dims)))

    width = (h + 2 * g) * d
    x, w1, s1 = buf("x", dtype, [t, hidden]), buf("w1", "i8", [width, hidden]), buf("s1", "f32", [width])
    w2, s2 = buf("w2", "i8", [hidden, h * d]), buf("s2", "f32", [hidden])
    pos, slots, offs = buf("positions", "i32", [1, t]), buf("slots", "i32", [t]), buf("q_offsets", "i32", [seqs + 1])
    start, lens = buf("kv_start", "i32", [seqs]), buf("kv_len", "i32", [seqs])
    a, sa = buf("a", "i8", [t, hidden], True), buf("sa", "f32", [t], True)
    qkv, k = buf("qkv", dtype, [t, width], True), buf("k", dtype, [t, g, d], True)
    c = {f"{p}_{w}": buf(f"{p}_{w}", "u8" if w == "codes" else "f32", [cache, g, d // 2] if w == "codes" else [cache, g], True)
         for p in "kv" for w in ("codes", "scale")}
    o, b, sb, y = buf("o", dtype, [t, h, d], True), buf("b", "i8", [t, h * d], True), buf("sb", "f32", [t], True), buf("y", dtype, [t, hidden], True)
    op.add_quantize_rows(km, dict(x=x, codes_out=a, scale_out=sa), cols=hidden)
    op.add_matmul_i8(km, dict(a=a, a_scale=sa, b=w1, b_scale=s1, out=qkv), cols=width, inner=hidden)
    op.add_qk_norm_rope(km, dict(q=qkv, k=qkv, positions=pos, q_out=qkv, k_out=k), heads=h, kv_heads=g, dim=d, columns={"k": h * d})
    op.add_store_kv4(km, dict(k=k, v=qkv, slots=slots, **{f"{n}_out": i for n, i in c.items()}), kv_heads=g, dim=d, columns={"v": (h + g) * d})
    op.add_attention_kv4(km, dict(q=qkv, q_offsets=offs, kv_start=start, kv_len=lens, out=o, **c), heads=h, kv_heads=g, dim=d)
    op.add_quantize_rows(km, dict(x=o, codes_out=b, scale_out=sb), cols=h * d)
    op.add_matmul_i8(km, dict(a=b, a_scale=sb, b=w2, b_scale=s2, out=y), cols=hidden, inner=h * d)
    return km


@pytest.mark.parametrize("dtype,t,d", [("bf16", 3, 64), ("f16", 40, 128), ("f32", 17, 64)])
def test_layer(hip, dtype, t, d):
    # Each step against its reference on what the step before it wrote.
    h, g, hidden, seqs, cache = 4, 2, 320, 1, 200
    rng = np.random.default_rng(t)
    km = layer(t, h, g, d, hidden, cache, seqs, dtype)
    before, _ = cache_of(rng, cache, g, d)
    n = 100 + t
    w1, s1 = quantize_rows(rng.standard_normal(((h + 2 * g) * d, hidden)).astype(np.float32).astype(np.float64) * 0.05)
    w2, s2 = quantize_rows(rng.standard_normal((hidden, h * d)).astype(np.float32).astype(np.float64) * 0.05)
    host = dict(x=rounded(rng.standard_normal((t, hidden)), dtype), w1=w1, s1=s1, w2=w2, s2=s2, positions=np.arange(100, n)[None],
                slots=np.arange(103, n + 3), q_offsets=[0, t], kv_start=[3], kv_len=[n], a=np.zeros((t, hidden)), b=np.zeros((t, h * d)), **before)
    got = run(hip, km, host)
    a, sa = quantize_rows(host["x"])
    same(got["a"], a)
    same(got["sa"], sa)
    want, bound = matmul_i8(a, sa, w1, s1, None, dtype)
    v = np.s_[:, (h + g) * d:]
    close(got["qkv"][v], want[v], bound[v], "v")
    for part, x in (("k", got["k"]), ("v", got["qkv"][v].reshape(t, g, d))):
        codes, scale = store_kv4(x)
        before[f"{part}_codes"][103:n + 3], before[f"{part}_scale"][103:n + 3] = codes, scale
        same(got[f"{part}_codes"], before[f"{part}_codes"])
        same(got[f"{part}_scale"], before[f"{part}_scale"])
    k, vv = (load_kv4(before[f"{p}_codes"], before[f"{p}_scale"]) for p in "kv")
    q = got["qkv"][:, :h * d].reshape(t, h, d)
    out, bound, *_ = attention(q, k, vv, [0, t], [3], [n], scale=d ** -0.5, causal=True, dtype=dtype)
    close(got["o"], out, bound, "o")
    b, sb = quantize_rows(got["o"].reshape(t, h * d))
    same(got["b"], b)
    y, bound = matmul_i8(b, sb, w2, s2, None, dtype)
    close(got["y"], y, bound, "y")


@pytest.mark.parametrize("t", [1, 40])
def test_layer_captured(hip, t):
    # Every replay gives the eager run's bits, with the eager run between them.
    h, g, d, hidden, cache = 4, 2, 64, 512, 3000
    rng = np.random.default_rng(t)
    km = layer(t, h, g, d, hidden, cache, 1, "bf16")
    before, _ = cache_of(rng, cache, g, d)
    host = dict(x=rounded(rng.standard_normal((t, hidden)), "bf16"), w1=rng.integers(-127, 128, ((h + 2 * g) * d, hidden)), s1=np.full((h + 2 * g) * d, 1e-3),
                w2=rng.integers(-127, 128, (hidden, h * d)), s2=np.full(hidden, 1e-3), positions=np.arange(t)[None] + 2000, slots=np.arange(t) + 2000,
                q_offsets=[0, t], kv_start=[0], kv_len=[2000 + t], a=np.zeros((t, hidden)), b=np.zeros((t, h * d)), **before)
    art = hip.build(km)
    bufs = {i: DeviceBuffer.from_array(np.asarray(host.get(km.buffers[i].name, np.zeros(km.buffers[i].dims))), km.buffers[i].dtype) for i in km.bindable_ids()}
    y = [i for i in km.output_ids() if km.buffers[i].name == "y"][0]
    art.run_device(bufs)
    want = bufs[y].to_numpy()
    cap = _Capture(mode=2)
    art.run_device(bufs, stream=cap.stream.value)   # the stream's workspaces
    with cap as stream:
        art.run_device(bufs, stream=stream, sync=False)
    for _ in range(4):
        bufs[y].fill_zero()
        cap.replay()
        assert np.array_equal(bufs[y].to_numpy(), want)
        art.run_device(bufs)
        assert np.array_equal(bufs[y].to_numpy(), want)
    cap.close()
