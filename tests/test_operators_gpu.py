"""The operators on the GPU against plain f64 references (operators_ref), at the
sizes, masks, strides and lengths where they could go wrong."""
import numpy as np
import pytest

from mlk2_amd import operators as op
from mlk2_amd.backend import DeviceBuffer, lib
from mlk2_amd.kernel_ir import KernelBuffer, KernelModule
from operators_ref import attention, norm_rope, rounded
from test_score_two_pass_gpu import _Capture

pytestmark = pytest.mark.gpu
KEEP = -77.0   # in every type; what a run must leave alone
TYPES = ["bf16", "f16", "f32"]


def device(km, host):
    """Device buffers by id from host arrays by buffer name; outputs hold KEEP."""
    bufs = {}
    for i in km.bindable_ids():
        b = km.buffers[i]
        a = host[b.name] if b.name in host else np.full(b.dims, KEEP)
        bufs[i] = DeviceBuffer.from_array(np.asarray(a), b.dtype)
    return bufs


def outputs(km, bufs):
    return {km.buffers[i].name: bufs[i].to_numpy().astype(np.float64).reshape(km.buffers[i].dims) for i in km.output_ids()}


def run(hip, km, host, noalloc=False):
    art, bufs = hip.build(km), device(km, host)
    (art.run_device_noalloc if noalloc else art.run_device)(bufs)
    return outputs(km, bufs)


def close(got, want, bound, what=""):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.where(bad, np.abs(got - want) / bound, 0)):.3g} bounds"


# ------------------------------------------------------------- qk_norm_rope --
def norm_rope_case(hip, t, h, g, d, dtype, *, rot=None, inter=False, sections=None, norm=True, wt=None, positions=True,
                   cache=None, valid=None, theta=1e4, first=0, eps=1e-6):
    rng = np.random.default_rng(t * 131 + d)
    rot = d if rot is None else rot
    km = op.qk_norm_rope_module(t, heads=h, kv_heads=g, dim=d, dtype=dtype, cache_rows=cache, norm=norm, weight_dtype=wt,
                                positions=positions, theta=theta, rot=rot, interleaved=inter, sections=sections, eps=eps,
                                sequences=2 if valid is not None else None)
    x = rounded(rng.standard_normal((t, (h + 2 * g) * d)), dtype)
    host = {"qkv": x}
    weights = {}
    for n in ("q_weight", "k_weight"):
        weights[n] = host[n] = rounded(1 + 0.2 * rng.standard_normal(d), wt or dtype)
    secs = sections or [rot // 2]
    pos = rng.integers(first, first + 1000, (len(secs), t))
    host["positions"] = pos
    slots = np.arange(t)
    if cache is not None:
        slots = rng.permutation(cache)[:t]
        slots[t // 2] = cache + 5       # outside the rows: nothing stored
        if t > 3:
            slots[0], slots[1] = -1, -2 ** 31
        host["slots"] = slots
    n = t if valid is None else valid
    host["q_offsets"] = [0, n // 2, n]
    got = run(hip, km, host)
    x = x.reshape(t, h + 2 * g, d)
    args = dict(rot=rot, theta=theta, eps=eps, interleaved=inter, sections=secs, dtype=dtype)
    where = pos if positions else None
    q, qb = norm_rope(x[:, :h], weights["q_weight"] if norm else None, where, **args)
    k, kb = norm_rope(x[:, h:h + g], weights["k_weight"] if norm else None, where, **args)
    close(got["q"][:n], q[:n], qb[:n], "q")
    assert (got["q"][n:] == KEEP).all()
    rows = t if cache is None else cache
    want_k, want_v, bound = np.full((rows, g, d), KEEP), np.full((rows, g, d), KEEP), np.zeros((rows, g, d))
    for i in range(n):
        if 0 <= slots[i] < rows:
            want_k[slots[i]], bound[slots[i]], want_v[slots[i]] = k[i], kb[i], x[i, h + g:]
    close(got["k"], want_k, bound, "k")
    assert (got["v"] == want_v).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [8, 20, 40, 64, 80, 96, 128, 200, 256])
def test_norm_rope_dims(hip, dtype, d):
    norm_rope_case(hip, 5, 6, 2, d, dtype, cache=11)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rot,inter,sections", [(64, False, None), (32, True, None), (40, False, None), (16, False, None),
                                                (128, False, [24, 20, 20]), (128, True, [30, 34]), (96, False, [48, 0, 0])])
def test_norm_rope_rotations(hip, dtype, rot, inter, sections):
    norm_rope_case(hip, 7, 3, 1, 128, dtype, rot=rot, inter=inter, sections=sections)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,h,g", [(1, 1, 1), (1, 32, 8), (3, 5, 5), (130, 12, 4), (67, 40, 8), (33, 16, 1)])
def test_norm_rope_sizes(hip, dtype, t, h, g):
    norm_rope_case(hip, t, h, g, 64, dtype, cache=t + 9, wt="f32")


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_rope_far_positions(hip, dtype):
    norm_rope_case(hip, 9, 2, 2, 128, dtype, theta=1e6, first=1_000_000)
    norm_rope_case(hip, 9, 2, 2, 128, dtype, theta=5e5, first=-3000)


@pytest.mark.parametrize("kw", [dict(norm=False), dict(positions=False), dict(valid=17), dict(valid=0), dict(norm=False, positions=False),
                                dict(eps=0.5)])
@pytest.mark.parametrize("d", [64, 36])
def test_norm_rope_options(hip, kw, d):
    norm_rope_case(hip, 20, 4, 2, d, "bf16", cache=31, **kw)


@pytest.mark.parametrize("d", [64, 128, 36])
def test_norm_rope_in_place(hip, d):
    # The fused rows' q, k and v in their own places equal those of the copy.
    t, h, g = 21, 4, 2
    rng = np.random.default_rng(3)
    host = {"qkv": rounded(rng.standard_normal((t, (h + 2 * g) * d)), "bf16"), "q_weight": rounded(rng.standard_normal(d), "bf16"),
            "k_weight": rounded(rng.standard_normal(d), "bf16"), "positions": np.arange(t)}
    want = run(hip, op.qk_norm_rope_module(t, heads=h, kv_heads=g, dim=d), host)
    km = KernelModule(name="in_place")
    ids = {}
    for name, dt, dims in (("q_weight", "bf16", [d]), ("k_weight", "bf16", [d]), ("positions", "i32", [1, t])):
        ids[name] = km.add_buffer(KernelBuffer(name, dt, is_input=True, elements=int(np.prod(dims)), dims=dims))
    x = km.add_buffer(KernelBuffer("qkv", "bf16", is_output=True, elements=t * (h + 2 * g) * d, dims=[t, (h + 2 * g) * d]))
    at = {"q": 0, "k": h * d, "v": (h + g) * d}
    ids.update({p + o: x for p in at for o in ("", "_out")})
    op.add_qk_norm_rope(km, ids, heads=h, kv_heads=g, dim=d, columns={p + o: c for p, c in at.items() for o in ("", "_out")})
    got = run(hip, km, host)["qkv"].reshape(t, h + 2 * g, d)
    assert (got[:, :h] == want["q"]).all() and (got[:, h:h + g] == want["k"]).all() and (got[:, h + g:] == want["v"]).all()


def test_norm_rope_non_finite_stays_in_its_head(hip):
    t, h, g, d = 4, 4, 2, 64
    x = np.ones((t, h + 2 * g, d))
    x[1, 0, 5], x[2, h, 7] = np.nan, np.inf
    host = {"qkv": x, "q_weight": np.ones(d), "k_weight": np.ones(d), "positions": np.arange(t)}
    got = run(hip, op.qk_norm_rope_module(t, heads=h, kv_heads=g, dim=d), host)
    assert np.isnan(got["q"][1, 0]).all() and np.isfinite(np.delete(got["q"].reshape(t * h, d), h, 0)).all()
    assert np.isfinite(np.delete(got["k"].reshape(t * g, d), 2 * g, 0)).all()


# ---------------------------------------------------------------- attention --
def attention_case(hip, q_lens, k_lens, h, g, d, dtype, *, causal=True, spare=0, scale=None, prefix=0, prefix_rows=None, gap=0,
                   noalloc=False, magnitude=1.0, poison=False):
    """Sequences in a cache whose rows have `gap` others between them."""
    rng = np.random.default_rng(sum(q_lens) * 7 + sum(k_lens) + d)
    n, t = len(q_lens), sum(q_lens) + spare
    start = np.concatenate([[0], np.cumsum(np.asarray(k_lens) + gap)[:-1]]).astype(int) + gap
    rows = int(sum(k_lens) + gap * (n + 1))
    q = rounded(magnitude * rng.standard_normal((t, h, d)), dtype)
    k, v = (rounded(rng.standard_normal((rows, g, d)), dtype) for _ in range(2))
    if poison:   # rows that no sequence holds
        held = np.zeros(rows, dtype=bool)
        for s, m in zip(start, k_lens):
            held[s:s + m] = True
        k[~held], v[~held] = np.nan, np.inf
    host = {"q": q, "k": k, "v": v, "q_offsets": np.concatenate([[0], np.cumsum(q_lens)]), "kv_start": start, "kv_len": k_lens}
    args = dict(kv_rows=rows, sequences=n, heads=h, kv_heads=g, dim=d, dtype=dtype, causal=causal, scale=scale, lse=True)
    extra = {}
    if prefix_rows is not None:
        pk, pv = (rounded(rng.standard_normal((prefix_rows, g, d)), dtype) for _ in range(2))
        if poison:
            pk[prefix:], pv[prefix:] = np.nan, np.inf
        host.update(prefix_k=pk, prefix_v=pv, prefix_len=[prefix])
        extra = dict(prefix_k=pk[:prefix], prefix_v=pv[:prefix])
        km = op.shared_prefix_attention_module(t, prefix_rows=prefix_rows, prefix_len=True, **args)
    else:
        km = op.attention_module(t, **args)
    got = run(hip, km, host, noalloc)
    out, bound, lse, lse_bound, written = attention(q, k, v, host["q_offsets"], start, k_lens, scale=scale or d ** -0.5, causal=causal,
                                                    dtype=dtype, **extra)
    close(got["out"][written], out[written], bound[written], "out")
    real = np.isfinite(lse) & written[:, None]
    close(got["lse"][real], lse[real], lse_bound[real], "lse")
    assert (got["lse"][~np.isfinite(lse) & written[:, None]] == -np.inf).all()
    assert (got["out"][~written] == KEEP).all() and (got["lse"][~written] == KEEP).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [8, 33, 64, 80, 96, 128, 192, 256])
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
@pytest.mark.parametrize("q_lens,k_lens", [([1, 1], [90, 33]), ([50], [80])])
def test_attention_heads(hip, h, g, q_lens, k_lens):
    attention_case(hip, q_lens, k_lens, h, g, 64, "bf16")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_lens,k_lens", [([90, 31], [90, 31]), ([1, 1, 2], [70, 1, 129])])
@pytest.mark.parametrize("prefix", [None, 37])
def test_attention_keys_behind_the_sequences_reach_nothing(hip, dtype, q_lens, k_lens, prefix):
    rows = None if prefix is None else prefix + 60
    attention_case(hip, q_lens, k_lens, 4, 2, 128, dtype, gap=5, poison=True, prefix=prefix or 0, prefix_rows=rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [100, 200])
@pytest.mark.parametrize("g", [1, 4])
def test_attention_hidden_keys_reach_nothing(hip, dtype, n, g):
    # Infinities and NaN in keys and values that the earlier queries do not see.
    h, d, at = 4, 64, n - 30
    rng = np.random.default_rng(n)
    q, k, v = (rounded(rng.standard_normal((n, m, d)), dtype) for m in (h, g, g))
    v[at, 0, 3], v[at + 2, g - 1, 7], k[at + 5, 0, 1] = np.inf, np.nan, np.nan
    km = op.attention_module(n, sequences=1, heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True)
    got = run(hip, km, {"q": q, "k": k, "v": v, "q_offsets": [0, n]})
    out, bound, lse, lse_bound, _ = attention(q, k, v, [0, n], [0], [n], scale=d ** -0.5, causal=True, dtype=dtype)
    fine = np.isfinite(out)
    assert fine[:at].all() and not fine[at:].all()
    assert (np.isfinite(got["out"]) == fine).all()
    assert (got["out"][np.isinf(out)] == out[np.isinf(out)]).all()
    close(got["out"][fine], out[fine], bound[fine])
    assert (np.isnan(got["lse"]) == np.isnan(lse)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 150])
def test_attention_infinite_scores(hip, dtype, n):
    # Keys whose scores are -inf carry nothing; a row of nothing else is zero.
    h, g, d = 2, 1, 64
    big = 6e4 if dtype == "f16" else 3e38
    rng = np.random.default_rng(n)
    q, v = (rounded(rng.standard_normal((n, m, d)), dtype) for m in (h, g))
    k = rounded(rng.standard_normal((n, g, d)), dtype)
    q[:, :, 0] = rounded(big, dtype)
    k[:, 0, 0] = 0.0
    k[0, 0], k[n // 2, 0] = 0.0, 0.0
    k[0, 0, 0] = k[n // 2, 0, 0] = -np.inf
    km = op.attention_module(n, sequences=1, heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True)
    got = run(hip, km, {"q": q, "k": k, "v": v, "q_offsets": [0, n]})
    seen = np.delete(np.arange(n), [0, n // 2])
    assert (got["out"][0] == 0).all() and (got["lse"][0] == -np.inf).all()
    for i in range(1, n):
        kk = seen[seen <= i]
        if len(kk) == 0:
            assert (got["out"][i] == 0).all()
            continue
        o, b, _, _, _ = attention(q[i:i + 1], k[kk], v[kk], [0, 1], [0], [len(kk)], scale=d ** -0.5, causal=False, dtype=dtype)
        # The first element times 0 is an exact 0: the bound's sum goes without it.
        _, b, _, _, _ = attention(np.where(np.arange(d) == 0, 0.0, q[i:i + 1]), k[kk], v[kk], [0, 1], [0], [len(kk)], scale=d ** -0.5,
                                  causal=False, dtype=dtype)
        close(got["out"][i], o[0], b[0], i)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_large_scores(hip, dtype):
    attention_case(hip, [150, 1], [150, 300], 4, 2, 64, dtype, magnitude=30.0)
    attention_case(hip, [60], [60], 2, 2, 64, dtype, scale=-0.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,pad,at", [(64, 0, 0), (64, 8, 8), (64, 3, 1), (128, 5, 0), (40, 1, 1)])
def test_attention_columns_of_fused_rows(hip, dtype, d, pad, at):
    # q, k and v in one buffer's rows, at columns on and off 16 bytes; out in wider rows.
    t, h, g = 45, 4, 2
    rng = np.random.default_rng(d + pad)
    width, wide = (h + 2 * g) * d + pad, h * d + pad
    x = rounded(rng.standard_normal((t, width)), dtype)
    km = KernelModule(name="fused")
    b = km.add_buffer(KernelBuffer("x", dtype, is_input=True, elements=t * width, dims=[t, width]))
    offs = km.add_buffer(KernelBuffer("q_offsets", "i32", is_input=True, elements=3, dims=[3]))
    out = km.add_buffer(KernelBuffer("out", dtype, is_output=True, elements=t * wide, dims=[t, wide]))
    op.add_attention(km, dict(q=b, k=b, v=b, q_offsets=offs, out=out), heads=h, kv_heads=g, dim=d,
                     columns=dict(q=at, k=at + h * d, v=at + (h + g) * d, out=at))
    got = run(hip, km, {"x": x, "q_offsets": [0, 30, t]})["out"]
    parts = [x[:, a:a + m * d].reshape(t, m, d) for a, m in ((at, h), (at + h * d, g), (at + (h + g) * d, g))]
    want, bound, _, _, _ = attention(*parts, [0, 30, t], [0, 30], [30, t - 30], scale=d ** -0.5, causal=True, dtype=dtype)
    close(got[:, at:at + h * d].reshape(want.shape), want, bound)
    assert (got[:, :at] == KEEP).all() and (got[:, at + h * d:] == KEEP).all()


@pytest.mark.parametrize("queries", [1, 40])
def test_attention_clips_offsets_and_lengths(hip, queries):
    # Offsets and lengths past the buffers are clipped; starts outside hold no keys.
    t, rows, h, g, d = 3 * queries, 60, 4, 2, 64
    rng = np.random.default_rng(9)
    q = rounded(rng.standard_normal((t, h, d)), "bf16")
    k, v = (rounded(rng.standard_normal((rows, g, d)), "bf16") for _ in range(2))
    km = op.attention_module(t, kv_rows=rows, sequences=3, heads=h, kv_heads=g, dim=d, causal=False, lse=True)
    offs, start, lens = [0, queries, 2 * queries, t + 1000], [30, -4, 59], [2 ** 31 - 1, 20, 5]
    got = run(hip, km, {"q": q, "k": k, "v": v, "q_offsets": offs, "kv_start": start, "kv_len": lens})
    want, bound, _, _, _ = attention(q, k, v, [0, queries, 2 * queries, t], [30, 0, 59], [30, 0, 1], scale=d ** -0.5, causal=False, dtype="bf16")
    close(got["out"], want, bound)
    # Out of order, below zero: only the rows they name, each once written or left.
    for offs in ([0, t, queries, t], [-5, queries, queries, -1], [t, 0, 0, 0], [2 ** 31 - 1, -2 ** 31, 5, 7]):
        host = {"q": q, "k": k, "v": v, "q_offsets": offs, "kv_start": [0, 2 ** 31 - 1, -2 ** 31], "kv_len": [-3, 9, 9]}
        got = run(hip, km, host)
        assert (np.isin(got["out"], [0.0, KEEP])).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("q_lens,k_lens", [([1], [20000]), ([1, 1], [9000, 40]), ([300], [5000])])
def test_attention_long(hip, dtype, q_lens, k_lens):
    attention_case(hip, q_lens, k_lens, 4, 1, 64, dtype)


def test_attention_offsets_past_32_bits(hip):
    # Keys whose elements start past 2^32 in the cache.
    h, g, d, rows = 8, 8, 128, (1 << 22) + 300
    n = 260
    km = op.attention_module(2, kv_rows=rows, sequences=2, heads=h, kv_heads=g, dim=d, dtype="bf16")
    rng = np.random.default_rng(1)
    q = rounded(rng.standard_normal((2, h, d)), "bf16")
    k, v = (rounded(rng.standard_normal((n, g, d)), "bf16") for _ in range(2))
    art = hip.build(km)
    bufs = {i: DeviceBuffer(int(np.prod(km.buffers[i].dims)), km.buffers[i].dtype) for i in km.bindable_ids()}
    at = (rows - n) * g * d * 2
    for i, a in ((1, k), (2, v)):
        tail = DeviceBuffer.from_array(a, "bf16").to_numpy()   # the same bits through the host
        from mlk2_amd.backend import bf16_bits
        bits = bf16_bits(tail)
        assert lib().mlkhip_memcpy_h2d(bufs[i].ptr + at, bits.ctypes.data, bits.nbytes) == 0
    for i, a in ((0, q), (3, [0, 1, 2]), (4, [rows - n, rows - 7]), (5, [n, 7])):
        bufs[i] = DeviceBuffer.from_array(np.asarray(a), km.buffers[i].dtype)
    art.run_device(bufs)
    want, bound, _, _, _ = attention(q, k, v, [0, 1, 2], [0, n - 7], [n, 7], scale=d ** -0.5, causal=True, dtype="bf16")
    close(bufs[6].to_numpy().reshape(want.shape), want, bound)


@pytest.mark.parametrize("q_lens,k_lens", [([1] * 4, [600, 30, 1200, 1]), ([90, 20], [90, 200])])
def test_attention_without_allocation(hip, q_lens, k_lens):
    attention_case(hip, q_lens, k_lens, 8, 2, 128, "bf16", noalloc=True)
    attention_case(hip, q_lens, k_lens, 8, 2, 128, "bf16", noalloc=True, prefix=150, prefix_rows=150)


# Row blocks of 32 rows, of eight waves in two groups with 128 rows, and the
# widest, by the rows and heads at hand: (heads, key/value heads, tokens, keys).
BLOCKS = {"narrow": (4, 2, [70, 0, 9], [70, 4, 9]), "halves": (80, 40, [129, 70, 0], [200, 70, 5]),
          "wide": (120, 120, [129, 70, 0], [200, 70, 5]), "halves_long": (32, 16, [200], [777]), "wide_long": (132, 132, [130], [601]),
          "halves_ranges": (8, 4, [150, 3, 110], [1500, 40, 1101])}


def block_of(name, dtype):
    return "narrow" if name == "narrow" or (dtype == "f32" and name.startswith("halves")) else name.split("_")[0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("name", BLOCKS)
def test_attention_row_blocks(hip, dtype, d, name):
    h, g, q_lens, k_lens = BLOCKS[name]
    km = op.attention_module(sum(q_lens) + 2, kv_rows=sum(k_lens), sequences=len(q_lens), heads=h, kv_heads=g, dim=d, dtype=dtype)
    waves, groups = {"narrow": (1, 1), "halves": (8, 2), "wide": (8, 1)}[block_of(name, dtype)]
    if dtype == "f32" or d == 256:
        waves, groups = (1, 1) if waves == 1 else (4, 1)
    step = hip.build(km).step_kernel_name(0)
    assert f"{max(d, 64) if d != 80 else 96}, {waves}, {groups}, " in step, step
    attention_case(hip, q_lens, k_lens, h, g, d, dtype, spare=2, causal=d != 64, gap=3, poison=True)


@pytest.mark.parametrize("n,q,k", [(64, 1, 9), (65, 1, 9), (150, 5, 40), (200, 40, 70), (4096, 1, 2), (4097, 1, 2)])
@pytest.mark.parametrize("prefix", [None, 50])
def test_attention_many_sequences(hip, n, q, k, prefix):
    # Lengths from none to q and k, found 64 sequences at a time up to 4096.
    rng = np.random.default_rng(n)
    q_lens, k_lens = [int(x) for x in rng.integers(0, q + 1, n)], [int(x) for x in rng.integers(0, k + 1, n)]
    attention_case(hip, q_lens, k_lens, 4, 2, 64, "bf16", spare=3, prefix=prefix or 0, prefix_rows=prefix, gap=1, poison=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["halves", "wide"])
def test_attention_row_blocks_options(hip, dtype, name):
    # A negative scale; scores far apart, so that the running maximum grows; a
    # prefix in front of every sequence's keys, its tiles before theirs.
    h, g, q_lens, k_lens = BLOCKS[name]
    attention_case(hip, q_lens, k_lens, h, g, 64, dtype, scale=-0.2)
    attention_case(hip, q_lens, k_lens, h, g, 128, dtype, magnitude=30.0)
    attention_case(hip, q_lens, k_lens, h, g, 96, dtype, prefix=70, prefix_rows=90, poison=True, gap=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,g", [(80, 40), (120, 120)])
def test_attention_row_blocks_hidden_and_infinite(hip, dtype, h, g):
    # NaN and infinities that the earlier queries do not see, in either group's
    # keys of a tile, and a key whose scores are -inf before all others.
    n, d = 150, 64
    rng = np.random.default_rng(g)
    q, k, v = (rounded(rng.standard_normal((n, m, d)), dtype) for m in (h, g, g))
    v[70, 0, 3], v[100, g - 1, 7], k[140, 5, 1] = np.inf, np.nan, np.nan
    q[:, :, 0] = np.abs(q[:, :, 0]) + 1
    k[0, 3, 0] = -np.inf
    got = run(hip, op.attention_module(n, sequences=1, heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True), {"q": q, "k": k, "v": v, "q_offsets": [0, n]})
    group = h // g
    for head, first in ((0, 70), ((g - 1) * group, 100), (5 * group, 140)):
        assert np.isfinite(got["out"][:first, head]).all() and not np.isfinite(got["out"][first:, head]).all()
    three = slice(3 * group, 4 * group)
    assert (got["out"][0, three] == 0).all() and (got["lse"][0, three] == -np.inf).all() and np.isfinite(got["out"][1:, three]).all()
    # Where nothing is seen that is not finite: as without it.
    clean = {"q": q, "k": np.where(np.isfinite(k), k, 0.0), "v": np.where(np.isfinite(v), v, 0.0)}
    out, bound, _, _, _ = attention(clean["q"], clean["k"], clean["v"], [0, n], [0], [n], scale=d ** -0.5, causal=True, dtype=dtype)
    close(got["out"][:70, :3 * group], out[:70, :3 * group], bound[:70, :3 * group])


# ---------------------------------------------------------- shared prefixes --
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_lens,k_lens", [([1], [1]), ([1, 1, 1], [0, 1, 70]), ([1] * 20, [3] * 20), ([5, 0, 40], [5, 9, 40]),
                                           ([60, 130], [60, 131]), ([3], [1])])
@pytest.mark.parametrize("prefix,rows", [(0, 5), (1, 1), (64, 64), (200, 201), (513, 600)])
def test_prefix_lengths(hip, dtype, q_lens, k_lens, prefix, rows):
    attention_case(hip, q_lens, k_lens, 4, 2, 64, dtype, prefix=prefix, prefix_rows=rows, spare=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [40, 80, 128, 256])
@pytest.mark.parametrize("q_lens", [[1] * 6, [33, 2]])
def test_prefix_dims(hip, dtype, d, q_lens):
    attention_case(hip, q_lens, [n + 9 for n in q_lens], 6, 2, d, dtype, prefix=100, prefix_rows=100)
    attention_case(hip, q_lens, [n + 9 for n in q_lens], 6, 2, d, dtype, prefix=100, prefix_rows=100, causal=False)


def test_prefix_equals_attention_over_copies(hip):
    # One shared prefix against the same prefix copied before each sequence's keys.
    h, g, d, prefix, lens = 8, 2, 128, 300, [1, 1, 1, 1, 1]
    attention_case(hip, lens, [9, 1, 70, 33, 2], h, g, d, "bf16", prefix=prefix, prefix_rows=prefix)


# ------------------------------------------------------------- used together --
def _serving_module(t, rows, n, h, g, d, dtype):
    """qk_norm_rope into a cache, then attention over it, as one module."""
    km = op.qk_norm_rope_module(t, heads=h, kv_heads=g, dim=d, dtype=dtype, cache_rows=rows, sequences=n, theta=1e4)
    q, k, v = km.output_ids()
    ids = {b.name: i for i, b in enumerate(km.buffers)}
    start = km.add_buffer(KernelBuffer("kv_start", "i32", is_input=True, elements=n, dims=[n]))
    lens = km.add_buffer(KernelBuffer("kv_len", "i32", is_input=True, elements=n, dims=[n]))
    out = km.add_buffer(KernelBuffer("out", dtype, is_output=True, elements=t * h * d, dims=[t, h, d]))
    op.add_attention(km, dict(q=q, k=k, v=v, q_offsets=ids["q_offsets"], kv_start=start, kv_len=lens, out=out), heads=h,
                     kv_heads=g, dim=d)
    return km


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_then_single_tokens(hip, dtype):
    # A prompt and then token after token on its cache equals the whole sequence at once.
    h, g, d, rows, prompts, steps = 4, 2, 64, 128, [37, 20], 6
    rng = np.random.default_rng(11)
    full = [rounded(rng.standard_normal((p + steps, (h + 2 * g) * d)), dtype) for p in prompts]
    weights = {w: rounded(1 + 0.1 * rng.standard_normal(d), dtype) for w in ("q_weight", "k_weight")}
    base = [0, 64]
    whole = _serving_module(sum(p + steps for p in prompts), rows, 2, h, g, d, dtype)

    def host(parts, firsts):
        pos = np.concatenate([np.arange(f, f + len(x)) for x, f in zip(parts, firsts)])
        slots = np.concatenate([np.arange(f, f + len(x)) + b for x, f, b in zip(parts, firsts, base)])
        return {"qkv": np.concatenate(parts), "positions": pos, "slots": slots, "kv_start": base, **weights,
                "q_offsets": np.concatenate([[0], np.cumsum([len(x) for x in parts])]),
                "kv_len": [f + len(x) for x, f in zip(parts, firsts)]}

    want = run(hip, whole, host(full, [0, 0]))
    at = np.concatenate([[0], np.cumsum([p + steps for p in prompts])])
    first = _serving_module(sum(prompts), rows, 2, h, g, d, dtype)
    art, bufs = hip.build(first), device(first, host([x[:p] for x, p in zip(full, prompts)], [0, 0]))
    art.run_device(bufs)
    cache = [bufs[i] for i in first.output_ids()[1:3]]
    step = _serving_module(2, rows, 2, h, g, d, dtype)
    art = hip.build(step)
    u = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}[dtype]
    for s in range(steps):
        now = [p + s for p in prompts]
        bufs = device(step, host([x[n:n + 1] for x, n in zip(full, now)], now))
        for i, c in zip(step.output_ids()[1:3], cache):
            bufs[i] = c
        art.run_device(bufs)
        got = outputs(step, bufs)
        rows_of = [at[b] + now[b] for b in range(2)]
        assert (got["q"] == want["q"][rows_of]).all()
        # The same q and cache rows; weights rounded relative to another
        # running maximum, sums of at most 43 in another order.
        close(got["out"], want["out"][rows_of], 8 * u + 400 * 2.0 ** -24)
    for c, name in zip(cache, "kv"):
        held = [base[b] + i for b in range(2) for i in range(prompts[b] + steps)]
        assert (c.to_numpy().reshape(rows, g, d)[held] == want[name][held]).all()


def test_host_entry_runs_the_operators(hip):
    # The f64 host ABI converts bf16 and i32 buffers and returns whole outputs.
    t, h, g, d = 12, 2, 1, 64
    km = op.attention_module(t, sequences=2, heads=h, kv_heads=g, dim=d, lse=True)
    rng = np.random.default_rng(2)
    q, k, v = (rounded(rng.standard_normal((t, m, d)), "bf16") for m in (h, g, g))
    got = hip.build(km).run({0: q, 1: k, 2: v, 3: np.array([0, 5, 9]), 4: np.full(t * h * d, KEEP), 5: np.full(t * h, KEEP)})
    want, bound, _, _, _ = attention(q, k, v, [0, 5, 9], [0, 5], [5, 4], scale=d ** -0.5, causal=True, dtype="bf16")
    out = got[4].reshape(t, h, d)
    close(out[:9], want[:9], bound[:9])
    assert (out[9:] == KEEP).all() and (got[5].reshape(t, h)[9:] == KEEP).all()


CAPTURED = [("decode", [1] * 4, [700, 30, 1500, 1], None), ("prompt", [60, 90], [60, 120], None), ("prefix", [1] * 5, [4, 9, 1, 70, 3], 400),
            ("ranges", [100, 50], [1500, 1000], None)]


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("name,q_lens,k_lens,prefix", CAPTURED)
def test_captured_and_replayed(hip, mode, name, q_lens, k_lens, prefix):
    # A run under capture (the stream's first, then one with a workspace) replays
    # to the eager result, with eager runs between, and reads lengths anew.
    h, g, d, n, t, rows = 8, 2, 128, len(q_lens), sum(q_lens), sum(k_lens)
    rng = np.random.default_rng(4)
    args = dict(kv_rows=rows, sequences=n, heads=h, kv_heads=g, dim=d, dtype="bf16", lse=True)
    km = op.attention_module(t, **args) if prefix is None else op.shared_prefix_attention_module(t, prefix_rows=prefix, **args)
    host = {"q": rng.standard_normal((t, h, d)), "k": rng.standard_normal((rows, g, d)), "v": rng.standard_normal((rows, g, d)),
            "q_offsets": np.concatenate([[0], np.cumsum(q_lens)]), "kv_start": np.concatenate([[0], np.cumsum(k_lens)[:-1]]), "kv_len": k_lens}
    if prefix is not None:
        host.update(prefix_k=rng.standard_normal((prefix, g, d)), prefix_v=rng.standard_normal((prefix, g, d)))
    host = {name: a if np.asarray(a).dtype.kind == "i" or isinstance(a, list) else rounded(a, "bf16") for name, a in host.items()}
    art, bufs = hip.build(km), device(km, host)
    keys = {"prefix_k": host.get("prefix_k"), "prefix_v": host.get("prefix_v")} if prefix is not None else {}
    lens_id = [i for i, b in enumerate(km.buffers) if b.name == "kv_len"][0]
    cap = _Capture(mode=mode)
    for warm in (False, True):
        if warm:
            art.run_device(bufs, stream=cap.stream.value)
        with cap as stream:
            art.run_device(bufs, stream=stream, sync=False)
        for lens in (k_lens, [max(1, m // 2) for m in k_lens], k_lens):
            q_lens_host = np.asarray(lens, dtype=np.int32)
            assert lib().mlkhip_memcpy_h2d(bufs[lens_id].ptr, q_lens_host.ctypes.data, q_lens_host.nbytes) == 0
            cap.replay()
            got = outputs(km, bufs)
            want, bound, lse, lse_bound, _ = attention(host["q"], host["k"], host["v"], host["q_offsets"], host["kv_start"], lens,
                                                       scale=d ** -0.5, causal=True, dtype="bf16", **keys)
            close(got["out"], want, bound, name)
            real = np.isfinite(lse)
            close(got["lse"][real], lse[real], lse_bound[real], name)
            art.run_device(bufs)
            close(outputs(km, bufs)["out"], want, bound, name)
    cap.close()


def test_two_streams_at_once(hip):
    # Runs of one artifact on two streams, each with its own workspace.
    h, g, d, n, keys = 8, 2, 128, 4, 3000
    km = op.attention_module(n, kv_rows=n * keys, sequences=n, heads=h, kv_heads=g, dim=d, dtype="bf16")
    art = hip.build(km)
    rng = np.random.default_rng(6)
    sets, streams = [], [_Capture().stream.value for _ in range(2)]
    for _ in range(2):
        host = {"q": rng.standard_normal((n, h, d)), "k": rng.standard_normal((n * keys, g, d)), "v": rng.standard_normal((n * keys, g, d)),
                "q_offsets": np.arange(n + 1), "kv_start": np.arange(n) * keys, "kv_len": [keys] * n}
        sets.append(device(km, host))
    want = []
    for bufs in sets:
        art.run_device(bufs)
        want.append(outputs(km, bufs)["out"])
    for _ in range(5):
        for bufs, stream in zip(sets, streams):
            art.run_device(bufs, stream=stream, sync=False)
    assert lib().mlkhip_synchronize() == 0
    for bufs, w in zip(sets, want):
        assert (outputs(km, bufs)["out"] == w).all()


@pytest.mark.parametrize("build", ["attention", "prefix", "norm_rope"])
def test_no_tokens(hip, build):
    if build == "norm_rope":
        km = op.qk_norm_rope_module(0, heads=4, kv_heads=2, dim=64, cache_rows=3)
        got = run(hip, km, {})
        assert (got["k"] == KEEP).all()
        return
    args = dict(kv_rows=0, sequences=1, heads=4, kv_heads=2, dim=64)
    for t in (0, 2):
        km = op.attention_module(t, **args) if build == "attention" else op.shared_prefix_attention_module(t, prefix_rows=0, **args)
        got = run(hip, km, {"q": np.ones((t, 4, 64)), "q_offsets": [0, t], "kv_start": [0], "kv_len": [9]})
        assert (got["out"] == 0).all()
