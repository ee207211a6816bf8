"""The operators in 8 and 4 bits as programs use them: captured and replayed with
other lengths, on two streams at once, through every entry, at addresses off 16
bytes, in rows past 2^32 bytes, with many sequences and with unlike ones."""
import numpy as np
import pytest

from mlk2_amd import operators as op
from mlk2_amd.backend import NP_OF_CODE, DeviceBuffer, bf16_bits, execute_kernel_on_buffers, lib
from operators_bits_ref import load_kv4, matmul_i8, quantize_rows, store_kv4
from operators_ref import attention, rounded
from test_operators_bits_gpu import attention_case, cache_of, same
from test_operators_gpu import KEEP, TYPES, close, device, outputs
from test_operators_uses_gpu import _Shifted
from test_score_two_pass_gpu import _Capture

pytestmark = pytest.mark.gpu


def put(km, bufs, host):
    for i in km.bindable_ids():
        name = km.buffers[i].name
        if name in host:
            buf, a = bufs[i], host[name]
            raw = bf16_bits(a) if buf.dtype == "bf16" else np.ascontiguousarray(np.asarray(a).astype(NP_OF_CODE[buf.code]))
            assert lib().mlkhip_memcpy_h2d(buf.ptr, raw.ctypes.data, buf.nbytes) == 0


def attention_host(rng, q_lens, start, k_lens, rows, h, g, d, dtype):
    host, (k, v) = cache_of(rng, rows, g, d)
    host.update(q=rounded(rng.standard_normal((sum(q_lens), h, d)), dtype), q_offsets=np.concatenate([[0], np.cumsum(q_lens)]),
                kv_start=np.asarray(start), kv_len=np.asarray(k_lens))
    return host, k, v


def close_f16(got, want, bound):
    """Values past 65520, half a step past the largest, round to infinity."""
    past = np.abs(want) - bound >= 65520
    assert (got[past] == np.sign(want[past]) * np.inf).all()
    edge = np.isinf(got) & (np.abs(want) + bound >= 65520)   # may round either way
    close(got[~past & ~edge], want[~past & ~edge], bound[~past & ~edge])


# ------------------------------------------------------------------ lengths --
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_lens,k_lens", [
    ([1] * 8, [9000] + [5] * 7), ([1] * 8, [5] * 7 + [12000]), ([1] * 3, [0, 9001, 0]), ([1, 0, 1], [8000, 70, 33]),
    ([129, 1, 40], [9000, 200, 8000]), ([33, 64], [4097, 6001]), ([5] * 12, [3000 + 37 * i for i in range(12)]), ([1] * 64, [1700 + i for i in range(64)])])
def test_unlike_lengths(hip, dtype, q_lens, k_lens):
    attention_case(hip, q_lens, k_lens, 4, 1, 64, dtype, spare=2)


@pytest.mark.parametrize("n", [63, 64, 65, 130, 700, 5000])
def test_many_sequences(hip, n):
    rng = np.random.default_rng(n)
    attention_case(hip, [1] * n, rng.integers(0, 90, n).tolist(), 4, 2, 64, "bf16")
    attention_case(hip, rng.integers(0, 4, n).tolist(), rng.integers(1, 40, n).tolist(), 2, 2, 32, "f32", spare=3)


@pytest.mark.parametrize("d", [64, 72])
def test_sequences_that_share_rows(hip, d):
    # Two sequences in the same rows, and one in a part of them.
    rng = np.random.default_rng(d)
    lens, start, k_lens = [1, 30, 2], [10, 10, 50], [2500, 2500, 900]
    host, k, v = attention_host(rng, lens, start, k_lens, 2600, 4, 2, d, "bf16")
    km = op.attention_kv4_module(33, kv_rows=2600, sequences=3, heads=4, kv_heads=2, dim=d)
    bufs = device(km, host)
    hip.build(km).run_device(bufs)
    want, bound, *_ = attention(host["q"], k, v, host["q_offsets"], start, k_lens, scale=d ** -0.5, causal=True, dtype="bf16")
    close(outputs(km, bufs)["out"], want, bound)


def test_a_cache_that_both_halves_share(hip):
    # k and v from the same codes and scales.
    rng = np.random.default_rng(11)
    host, k, _ = attention_host(rng, [40], [0], [300], 300, 4, 2, 64, "f16")
    host["v_codes"], host["v_scale"] = host["k_codes"], host["k_scale"]
    km = op.attention_kv4_module(40, kv_rows=300, sequences=1, heads=4, kv_heads=2, dim=64, dtype="f16")
    bufs = device(km, host)
    ids = {km.buffers[i].name: i for i in km.bindable_ids()}
    bufs[ids["v_codes"]], bufs[ids["v_scale"]] = bufs[ids["k_codes"]], bufs[ids["k_scale"]]
    hip.build(km).run_device(bufs)
    want, bound, *_ = attention(host["q"], k, k, [0, 40], [0], [300], scale=0.125, causal=True, dtype="f16")
    close(outputs(km, bufs)["out"], want, bound)


# ------------------------------------------------------- graphs and streams --
LENGTHS = [[9000] + [5] * 7, [2500] * 8, [0] * 8, [1, 2, 3, 40, 500, 6000, 7, 8]]


@pytest.mark.parametrize("dtype", TYPES)
def test_replays_read_lengths_anew(hip, dtype):
    # Lengths that the ranges of keys are dealt by change between the replays.
    n, h, g, d, rows = 8, 8, 2, 128, 24000
    rng = np.random.default_rng(1)
    km = op.attention_kv4_module(n, kv_rows=rows, sequences=n, heads=h, kv_heads=g, dim=d, dtype=dtype)
    host, k, v = attention_host(rng, [1] * n, np.zeros(n), LENGTHS[0], rows, h, g, d, dtype)
    art, bufs, other = hip.build(km), device(km, host), device(km, host)
    cap = _Capture(mode=2)
    art.run_device(bufs, stream=cap.stream.value)   # the stream's workspace
    with cap as stream:
        art.run_device(bufs, stream=stream, sync=False)
    for lens in LENGTHS + LENGTHS[::-1]:
        host["kv_len"], host["kv_start"] = np.asarray(lens), rng.integers(0, rows - max(lens), n)
        put(km, bufs, host)
        put(km, other, host)
        cap.replay()
        art.run_device(other)
        got = outputs(km, bufs)["out"]
        assert np.array_equal(got, outputs(km, other)["out"])
        want, bound, *_ = attention(host["q"], k, v, host["q_offsets"], host["kv_start"], lens, scale=d ** -0.5, causal=True, dtype=dtype)
        close(got, want, bound)
    cap.close()


def serving_step(rng, m, n, k, dtype):
    """A product whose rows are copied and whose k is split, and its operands."""
    a, b = rng.integers(-127, 128, (m, k)), rng.integers(-127, 128, (n, k))
    sa, sb = (np.exp(rng.standard_normal(x)).astype(np.float32).astype(np.float64) for x in (m, n))
    return op.matmul_i8_module(m, n, k, dtype=dtype), {"a": a, "b": b, "a_scale": sa, "b_scale": sb}, matmul_i8(a, sa, b, sb, None, dtype)


@pytest.mark.parametrize("m,n,k", [(70, 130, 8191), (70, 130, 8192), (200, 70, 5000)])
def test_matmul_on_two_streams_and_in_two_graphs(hip, m, n, k):
    # Each stream has a workspace of its own; graphs replayed side by side.
    rng = np.random.default_rng(k)
    parts = [serving_step(rng, m, n, k, "bf16") for _ in range(2)]
    arts = [hip.build(km) for km, *_ in parts]
    bufs = [device(km, host) for km, host, _ in parts]
    caps = [_Capture(mode=2) for _ in parts]
    for art, buf, cap in zip(arts, bufs, caps):
        art.run_device(buf, stream=cap.stream.value)
    for _ in range(10):
        for art, buf, cap in zip(arts, bufs, caps):
            art.run_device(buf, stream=cap.stream.value, sync=False)
    for cap in caps:
        cap("hipStreamSynchronize", cap.stream)
    for (km, _, (want, bound)), buf in zip(parts, bufs):
        close(outputs(km, buf)["out"], want, bound)
    for art, buf, cap in zip(arts, bufs, caps):
        with cap as stream:
            art.run_device(buf, stream=stream, sync=False)
    for buf, (km, *_) in zip(bufs, parts):
        for i in km.output_ids():
            buf[i].fill_zero()
    for _ in range(5):
        for cap in caps:
            cap("hipGraphLaunch", cap.exec, cap.stream)
    for cap in caps:
        cap("hipStreamSynchronize", cap.stream)
    for (km, _, (want, bound)), buf in zip(parts, bufs):
        close(outputs(km, buf)["out"], want, bound)
    for cap in caps:
        cap.close()


def test_attention_on_two_streams(hip):
    h, g, d, rows, lens = 8, 2, 64, 20000, [9000, 300, 10000]
    rng = np.random.default_rng(6)
    km = op.attention_kv4_module(3, kv_rows=rows, sequences=3, heads=h, kv_heads=g, dim=d)
    hosts = [attention_host(rng, [1] * 3, [0, 9000, 9300], lens, rows, h, g, d, "bf16") for _ in range(2)]
    art, caps = hip.build(km), [_Capture(mode=2) for _ in hosts]
    bufs = [device(km, host) for host, *_ in hosts]
    for _ in range(10):
        for buf, cap in zip(bufs, caps):
            art.run_device(buf, stream=cap.stream.value, sync=False)
    for cap in caps:
        cap("hipStreamSynchronize", cap.stream)
    for buf, (host, k, v) in zip(bufs, hosts):
        want, bound, *_ = attention(host["q"], k, v, [0, 1, 2, 3], host["kv_start"], lens, scale=0.125, causal=True, dtype="bf16")
        close(outputs(km, buf)["out"], want, bound)


def test_captured_without_a_workspace(hip):
    # A stream's first run, under capture: nothing is allocated, and forms that
    # need no workspace give the results.
    rng = np.random.default_rng(3)
    h, g, d, rows, lens = 8, 2, 64, 12000, [9000, 3000]
    km = op.attention_kv4_module(2, kv_rows=rows, sequences=2, heads=h, kv_heads=g, dim=d)
    host, k, v = attention_host(rng, [1, 1], [0, 9000], lens, rows, h, g, d, "bf16")
    want, bound, *_ = attention(host["q"], k, v, [0, 1, 2], [0, 9000], lens, scale=0.125, causal=True, dtype="bf16")
    cases = [(km, host, (want, bound))] + [serving_step(rng, *size, "f16") for size in ((70, 130, 8191), (70, 130, 8192))]
    for km, host, (want, bound) in cases:
        art, bufs, cap = hip.build(km), device(km, host), _Capture()
        with cap as stream:
            art.run_device(bufs, stream=stream, sync=False)
        for _ in range(3):
            bufs[km.output_ids()[0]].fill_zero()
            cap.replay()
            (close if km is cases[0][0] else close_f16)(outputs(km, bufs)["out"], want, bound)
        cap.close()


# ------------------------------------------------------------------ entries --
def entries(rng):
    h, g, d = 4, 2, 64
    x = rounded(rng.standard_normal((70, 136)), "bf16")
    codes, scale = quantize_rows(x)
    yield op.quantize_rows_module(70, 136), {"x": x}, {"codes": codes, "scale": scale}
    km, host, (want, _) = serving_step(rng, 70, 130, 8191, "f32")
    yield km, host, None
    y = rounded(rng.standard_normal((2, 9, g, d)), "f16")
    kv = [store_kv4(p) for p in y]
    yield (op.store_kv4_module(9, kv_heads=g, dim=d, dtype="f16"), {"k": y[0], "v": y[1]},
           {f"{p}_{w}": kv[i][j] for i, p in enumerate("kv") for j, w in enumerate(("codes", "scale"))})
    host, _, _ = attention_host(rng, [40, 1], [0, 40], [40, 9000], 9040, h, g, d, "bf16")
    yield op.attention_kv4_module(41, kv_rows=9040, sequences=2, heads=h, kv_heads=g, dim=d, lse=True), host, None
    cache = {f"{p}_{w}": kv[i][j] for i, p in enumerate("kv") for j, w in enumerate(("codes", "scale"))}
    yield op.load_kv4_module(9, kv_heads=g, dim=d, dtype="f32"), cache, {p: load_kv4(*kv[i]) for i, p in enumerate("kv")}


@pytest.mark.parametrize("which", range(5))
def test_every_entry_runs_the_operators(hip, which):
    # Timing, the search, runs that allocate nothing and the one-shot host entry
    # leave or give the results of a run.
    km, host, want = list(entries(np.random.default_rng(0)))[which]
    art, bufs = hip.build(km), device(km, host)
    art.run_device(bufs)
    got = outputs(km, bufs)
    for name, a in (want or {}).items():
        if name in ("k", "v"):
            close(got[name].reshape(a.shape), a, np.abs(a) * 2.0 ** -24)
        else:
            same(got[name].reshape(a.shape), a, name)
    assert art.num_steps() == 1 and art.step_variants(0) == []
    assert (art.time_device(bufs, 3, warmup=1) > 0).all() and art.time_device_span(bufs, 3, warmup=1) > 0
    assert art.autotune(bufs, reps=2)
    art.run_device_noalloc(bufs)
    for name, a in outputs(km, bufs).items():
        same(a, got[name], name)
    ids = km.bindable_ids()
    outs = [np.full(got[km.buffers[i].name].size, KEEP if km.buffers[i].dtype not in ("i8", "u8") else 0.0) for i in km.output_ids()]
    execute_kernel_on_buffers(km, [np.asarray(host[km.buffers[i].name], dtype=np.float64) for i in ids if i not in km.output_ids()], outs)
    for i, a in zip(km.output_ids(), outs):
        same(a, got[km.buffers[i].name].reshape(-1), km.buffers[i].name)
    art.release_stream_scratch()


# ---------------------------------------------------------------- addresses --
def shift(km, bufs, host, shifted):
    for i in km.bindable_ids():
        b = km.buffers[i]
        if shifted in (b.name, "all"):
            keep = 7.0 if b.dtype in ("i8", "u8") else KEEP
            bufs[i] = ShiftedBytes(host.get(b.name, np.zeros(b.dims)), b.dtype) if keep == 7.0 else _Shifted(host.get(b.name, np.full(b.dims, KEEP)), b.dtype)


class ShiftedBytes(_Shifted):
    def __init__(self, a, dtype):
        flat = np.asarray(a, dtype=np.float64).reshape(-1)
        self.whole = DeviceBuffer.from_array(np.concatenate([[7], flat]), dtype)
        self.elements = flat.size

    def to_numpy(self):
        a = self.whole.to_numpy()
        assert a[0] == 7
        return a[1:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shifted", ["q", "k_codes", "k_scale", "v_codes", "v_scale", "out", "lse", "q_offsets", "all"])
def test_attention_at_addresses_off_16_bytes(hip, dtype, shifted):
    h, g, d, q_lens, k_lens = 4, 2, 64, [40, 1, 3], [40, 900, 3]
    rng = np.random.default_rng(2)
    host, k, v = attention_host(rng, q_lens, [0, 40, 940], k_lens, 943, h, g, d, dtype)
    km = op.attention_kv4_module(44, kv_rows=943, sequences=3, heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True)
    bufs = device(km, host)
    shift(km, bufs, host, shifted)
    hip.build(km).run_device(bufs)
    got = outputs(km, bufs)
    want, bound, lse, lse_bound, _ = attention(host["q"], k, v, host["q_offsets"], host["kv_start"], k_lens, scale=d ** -0.5, causal=True, dtype=dtype)
    close(got["out"], want, bound, "out")
    close(got["lse"], lse, lse_bound, "lse")


@pytest.mark.parametrize("m,n,k", [(1, 40, 512), (20, 40, 256), (48, 40, 4096), (70, 70, 4096), (300, 700, 320)])
@pytest.mark.parametrize("shifted", ["a", "b", "a_scale", "b_scale", "out", "all"])
def test_matmul_at_addresses_off_16_bytes(hip, m, n, k, shifted):
    km, host, (want, bound) = serving_step(np.random.default_rng(m), m, n, k, "f16")
    host["a_scale"], host["b_scale"] = host["a_scale"] * 2.0 ** -12, host["b_scale"]
    bufs = device(km, host)
    shift(km, bufs, host, shifted)
    hip.build(km).run_device(bufs)
    close_f16(outputs(km, bufs)["out"], want * 2.0 ** -12, bound * 2.0 ** -12 + 2.0 ** -25)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shifted", ["x", "codes", "scale", "all"])
def test_quantize_rows_at_addresses_off_16_bytes(hip, dtype, shifted):
    x = rounded(np.random.default_rng(5).standard_normal((9, 264)), dtype)
    codes, scale = quantize_rows(x)
    km = op.quantize_rows_module(9, 264, dtype=dtype)
    bufs = device(km, {"x": x, "codes": np.zeros((9, 264))})
    shift(km, bufs, {"x": x}, shifted)
    hip.build(km).run_device(bufs)
    got = outputs(km, bufs)
    same(got["codes"], codes)
    same(got["scale"], scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shifted", ["k", "v", "k_codes", "v_scale", "slots", "all"])
def test_store_at_addresses_off_16_bytes(hip, dtype, shifted):
    t, g, d = 9, 2, 64
    y = rounded(np.random.default_rng(7).standard_normal((2, t, g, d)), dtype)
    host = {"k": y[0], "v": y[1], "slots": np.random.default_rng(8).permutation(t)}
    for p in "kv":
        host[f"{p}_codes"], host[f"{p}_scale"] = np.zeros((t, g, d // 2)), np.zeros((t, g))
    km = op.store_kv4_module(t, kv_heads=g, dim=d, dtype=dtype, cache_rows=t)
    bufs = device(km, host)
    shift(km, bufs, host, shifted)
    hip.build(km).run_device(bufs)
    got = outputs(km, bufs)
    for i, p in enumerate("kv"):
        codes, scale = store_kv4(y[i])
        same(got[f"{p}_codes"].reshape(t, g, -1)[host["slots"]], codes)
        same(got[f"{p}_scale"].reshape(t, g)[host["slots"]], scale)


# ------------------------------------------------------------- past 32 bits --
def _put(buf, byte, a):
    a = np.ascontiguousarray(a)
    assert lib().mlkhip_memcpy_h2d(buf.ptr + byte, a.ctypes.data, a.nbytes) == 0


def _take(buf, byte, shape, dtype):
    a = np.empty(shape, dtype)
    assert lib().mlkhip_memcpy_d2h(a.ctypes.data, buf.ptr + byte, a.nbytes) == 0
    return a


def _bf16(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def _buffers(km):
    bufs = {i: DeviceBuffer(int(np.prod(km.buffers[i].dims)), km.buffers[i].dtype) for i in km.bindable_ids()}
    return bufs, {km.buffers[i].name: bufs[i] for i in bufs}


@pytest.mark.parametrize("d", [128, 130])
def test_a_cache_past_32_bits(hip, d):
    # Tokens stored to the last rows of a cache of more than 2^32 bytes, attended
    # there and read back.
    h, g, t, n = 16, 8, 5, 900
    rows = (1 << 32) // (g * d // 2) + 2 * n
    rng = np.random.default_rng(d)
    last = rows - n
    y = rounded(rng.standard_normal((2, n, g, d)), "bf16")
    km = op.store_kv4_module(n, kv_heads=g, dim=d, cache_rows=rows)
    store, by = _buffers(km)
    slots = (rows - 1 - rng.permutation(n)).astype(np.int32)
    for i, p in enumerate("kv"):
        _put(by[p], 0, bf16_bits(y[i]))
    _put(by["slots"], 0, slots)
    hip.build(km).run_device(store)
    cache = {}
    for i, p in enumerate("kv"):
        codes, scale = store_kv4(y[i])
        order = slots - last
        cache[p] = np.empty((n, g, d))
        cache[p][order] = load_kv4(codes, scale)
        assert np.array_equal(_take(by[f"{p}_codes"], last * g * d // 2, (n, g, d // 2), np.uint8)[order], codes)
        assert np.array_equal(_take(by[f"{p}_scale"], last * g * 4, (n, g), np.float32)[order], scale.astype(np.float32))
    km = op.attention_kv4_module(t, kv_rows=rows, sequences=1, heads=h, kv_heads=g, dim=d)
    bufs, ids = _buffers(op.attention_kv4_module(t, kv_rows=n, sequences=1, heads=h, kv_heads=g, dim=d))
    names = {km.buffers[i].name: i for i in km.bindable_ids()}
    bufs = {names[m]: by[m] if m in by and m.endswith(("codes", "scale")) else ids[m] for m in names}
    q = rounded(rng.standard_normal((t, h, d)), "bf16")
    _put(ids["q"], 0, bf16_bits(q))
    for m, a in (("q_offsets", [0, t]), ("kv_start", [last]), ("kv_len", [n])):
        _put(ids[m], 0, np.asarray(a, np.int32))
    hip.build(km).run_device(bufs)
    want, bound, *_ = attention(q, cache["k"], cache["v"], [0, t], [0], [n], scale=d ** -0.5, causal=True, dtype="bf16")
    close(_bf16(_take(ids["out"], 0, (t, h, d), np.uint16)), want, bound)


def test_rows_of_a_product_past_32_bits(hip):
    m, n, k, few = (1 << 20) + 300, 66, 4096, 200
    rng = np.random.default_rng(4)
    x = rounded(rng.standard_normal((few, k)), "bf16")
    km = op.quantize_rows_module(m, k)
    bufs, ids = _buffers(km)
    first = m - few
    _put(ids["x"], first * k * 2, bf16_bits(x))
    hip.build(km).run_device(bufs)
    codes, scale = quantize_rows(x)
    assert np.array_equal(_take(ids["codes"], first * k, (few, k), np.int8), codes.astype(np.int8))
    assert np.array_equal(_take(ids["scale"], first * 4, few, np.float32), scale.astype(np.float32))
    b, sb = rng.integers(-127, 128, (n, k)), np.exp(rng.standard_normal(n)).astype(np.float32).astype(np.float64)
    km = op.matmul_i8_module(m, n, k)
    names = {km.buffers[i].name: i for i in km.bindable_ids()}
    product = {names["a"]: ids["codes"], names["a_scale"]: ids["scale"], names["b"]: DeviceBuffer.from_array(b, "i8"),
               names["b_scale"]: DeviceBuffer.from_array(sb, "f32"), names["out"]: DeviceBuffer(m * n, "bf16")}
    hip.build(km).run_device(product)
    want, bound = matmul_i8(codes, scale, b, sb, None, "bf16")
    close(_bf16(_take(product[names["out"]], first * n * 2, (few, n), np.uint16)), want, bound)
