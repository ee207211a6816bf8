"""The operators as programs use them: captured together and replayed, through
every entry, at addresses off 16 bytes, and in rows past 2^32 elements."""
import numpy as np
import pytest

from mlk2_amd import fixtures as fx
from mlk2_amd import operators as op
from mlk2_amd.backend import NP_OF_CODE, DeviceBuffer, bf16_bits, execute_kernel_on_buffers, lib
from mlk2_amd.kernel_ir import KernelBuffer
from operators_ref import attention, norm_rope, rounded
from test_operators_gpu import KEEP, TYPES, _serving_module, close, device, outputs, run
from test_score_two_pass_gpu import _Capture

pytestmark = pytest.mark.gpu


def _serving_host(rng, t, rows, n, h, g, d, dtype, lens):
    q_lens = [t // n] * n
    return {"qkv": rounded(rng.standard_normal((t, (h + 2 * g) * d)), dtype), "positions": rng.integers(0, 5000, t),
            "slots": np.concatenate([np.arange(m) + i * (rows // n) + lens[i] - m for i, m in enumerate(q_lens)]),
            "kv_start": np.arange(n) * (rows // n), "kv_len": lens, "q_offsets": np.arange(n + 1) * (t // n),
            **{w: rounded(1 + 0.1 * rng.standard_normal(d), dtype) for w in ("q_weight", "k_weight")}}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n", [(4, 4), (160, 2)])
def test_norm_and_attention_captured_together(hip, dtype, t, n):
    # One graph of both Calls: replays equal eager runs, with eager work on the
    # same buffers between, and read slots and lengths anew.
    h, g, d, rows = 8, 2, 128, 4096
    rng = np.random.default_rng(t)
    km = _serving_module(t, rows, n, h, g, d, dtype)
    art = hip.build(km)
    sets = [_serving_host(rng, t, rows, n, h, g, d, dtype, [rows // n - 5 * i for i in range(n)]),
            _serving_host(rng, t, rows, n, h, g, d, dtype, [t // n + 3 * i for i in range(n)])]
    bufs, other = device(km, sets[0]), device(km, sets[0])
    cache = rounded(rng.standard_normal((rows, g, d)), dtype)
    ids = {km.buffers[i].name: i for i in km.bindable_ids()}

    def put(where, host):
        for name, a in {**host, "k": cache, "v": cache}.items():
            buf = where[ids[name]]
            raw = bf16_bits(a) if buf.dtype == "bf16" else np.asarray(a).astype(NP_OF_CODE[buf.code])
            assert lib().mlkhip_memcpy_h2d(buf.ptr, np.ascontiguousarray(raw).ctypes.data, buf.nbytes) == 0

    cap = _Capture(mode=2)
    put(bufs, sets[0])
    art.run_device(bufs, stream=cap.stream.value)   # the stream's workspace
    with cap as stream:
        art.run_device(bufs, stream=stream, sync=False)
    for turn in (0, 1, 1, 0):
        put(bufs, sets[turn])
        cap.replay()
        got = outputs(km, bufs)
        put(other, sets[turn])
        art.run_device(other)
        want = outputs(km, other)
        for name in got:
            assert np.array_equal(got[name], want[name]), (turn, name)
    cap.close()


def _attention_host(rng, q_lens, k_lens, h, g, d, dtype):
    rows = sum(k_lens)
    return {"q": rounded(rng.standard_normal((sum(q_lens), h, d)), dtype), "k": rounded(rng.standard_normal((rows, g, d)), dtype),
            "v": rounded(rng.standard_normal((rows, g, d)), dtype), "q_offsets": np.concatenate([[0], np.cumsum(q_lens)]),
            "kv_start": np.concatenate([[0], np.cumsum(k_lens)[:-1]]), "kv_len": np.asarray(k_lens)}


def test_every_entry_runs_the_operators(hip):
    # Timing, the search and the one-shot host entry leave or give the results of a run.
    h, g, d = 4, 2, 64
    rng = np.random.default_rng(0)
    host = _attention_host(rng, [40, 1], [40, 90], h, g, d, "bf16")
    km = op.attention_module(41, kv_rows=130, sequences=2, heads=h, kv_heads=g, dim=d, lse=True)
    art, bufs = hip.build(km), device(km, host)
    art.run_device(bufs)
    want = outputs(km, bufs)
    assert art.num_steps() == 1 and art.step_variants(0) == []
    assert (art.time_device(bufs, 3, warmup=1) > 0).all() and art.time_device_span(bufs, 3, warmup=1) > 0
    report = art.autotune(bufs, reps=2)
    assert report
    art.run_device_noalloc(bufs)
    for name, a in outputs(km, bufs).items():
        assert np.array_equal(a, want[name]), name
    names = [km.buffers[i].name for i in km.bindable_ids()]
    outs = [np.full(want[n].size, KEEP) for n in ("out", "lse")]
    execute_kernel_on_buffers(km, [host[n] for n in names if n in host], outs)
    assert np.array_equal(outs[0], want["out"].reshape(-1)) and np.array_equal(outs[1], want["lse"].reshape(-1))
    art.release_stream_scratch()


def test_beside_other_steps(hip):
    # An f32 attention's output as the operand of a softmax Call in the same module.
    h, g, d, t = 2, 1, 64, 33
    rng = np.random.default_rng(1)
    host = _attention_host(rng, [t], [t], h, g, d, "f32")
    km = op.attention_module(t, sequences=1, heads=h, kv_heads=g, dim=d, dtype="f32")
    soft = fx.softmax_call_module(t, h * d, "f32")
    out = km.output_ids()[0]
    km.buffers[out].dims = [t, h * d]
    y = km.add_buffer(KernelBuffer("y", "f32", is_output=True, elements=t * h * d, dims=[t, h * d]))
    node = soft.nodes[-1]
    node.a, node.out = out, y
    km.add_node(node)
    art, bufs = hip.build(km), device(km, host)
    assert art.num_steps() == 2
    art.run_device(bufs)
    got = outputs(km, bufs)
    want, bound, _, _, _ = attention(host["q"], host["k"], host["v"], [0, t], [0], [t], scale=d ** -0.5, causal=True, dtype="f32")
    close(got["out"].reshape(want.shape), want, bound)
    x = got["out"]
    e = np.exp(x - x.max(-1, keepdims=True))
    assert np.abs(got["y"] - e / e.sum(-1, keepdims=True)).max() < 1e-6
    report = art.autotune(bufs, reps=2)
    assert report


class _Shifted:
    """A buffer whose elements start one element past a 256-byte boundary."""

    def __init__(self, a, dtype):
        flat = np.asarray(a, dtype=np.float64).reshape(-1)
        self.whole = DeviceBuffer.from_array(np.concatenate([[KEEP], flat]), dtype)
        self.elements = flat.size

    def binding(self):
        b = self.whole.binding()
        b.ptr += self.whole.nbytes // self.whole.elements
        b.elements -= 1
        return b

    def to_numpy(self):
        a = self.whole.to_numpy()
        assert a[0] == KEEP
        return a[1:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shifted", ["q", "k", "v", "out", "lse", "q_offsets", "prefix_k", "all"])
def test_attention_at_addresses_off_16_bytes(hip, dtype, shifted):
    h, g, d, prefix, q_lens, k_lens = 4, 2, 64, 70, [40, 1, 3], [40, 90, 3]
    rng = np.random.default_rng(2)
    host = _attention_host(rng, q_lens, k_lens, h, g, d, dtype)
    host.update({n: rounded(rng.standard_normal((prefix, g, d)), dtype) for n in ("prefix_k", "prefix_v")})
    km = op.shared_prefix_attention_module(44, prefix_rows=prefix, kv_rows=133, sequences=3, heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True)
    bufs = device(km, host)
    for i in km.bindable_ids():
        b = km.buffers[i]
        if shifted in (b.name, "all"):
            bufs[i] = _Shifted(host.get(b.name, np.full(b.dims, KEEP)), b.dtype)
    hip.build(km).run_device(bufs)
    got = outputs(km, bufs)
    want, bound, lse, lse_bound, _ = attention(host["q"], host["k"], host["v"], host["q_offsets"], host["kv_start"], k_lens, scale=d ** -0.5,
                                               causal=True, dtype=dtype, prefix_k=host["prefix_k"], prefix_v=host["prefix_v"])
    close(got["out"], want, bound, "out")
    close(got["lse"], lse, lse_bound, "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shifted", ["qkv", "q_weight", "k_weight", "positions", "slots", "q", "k", "v", "all"])
def test_norm_rope_at_addresses_off_16_bytes(hip, dtype, shifted):
    t, h, g, d, rows = 9, 4, 2, 64, 20
    rng = np.random.default_rng(4)
    km = op.qk_norm_rope_module(t, heads=h, kv_heads=g, dim=d, dtype=dtype, cache_rows=rows)
    host = {"qkv": rounded(rng.standard_normal((t, (h + 2 * g) * d)), dtype), "positions": rng.integers(0, 999, (1, t)),
            "slots": rng.permutation(rows)[:t], **{w: rounded(1 + 0.1 * rng.standard_normal(d), dtype) for w in ("q_weight", "k_weight")}}
    bufs = device(km, host)
    for i in km.bindable_ids():
        b = km.buffers[i]
        if shifted in (b.name, "all"):
            bufs[i] = _Shifted(host.get(b.name, np.full(b.dims, KEEP)), b.dtype)
    hip.build(km).run_device(bufs)
    got = outputs(km, bufs)
    x = host["qkv"].reshape(t, h + 2 * g, d)
    args = dict(rot=d, theta=1e4, eps=1e-6, interleaved=False, sections=[d // 2], dtype=dtype)
    q, qb = norm_rope(x[:, :h], host["q_weight"], host["positions"], **args)
    k, kb = norm_rope(x[:, h:h + g], host["k_weight"], host["positions"], **args)
    close(got["q"], q, qb, "q")
    close(got["k"][host["slots"]], k, kb, "k")
    assert (got["v"][host["slots"]] == x[:, h + g:]).all()
    free = np.setdiff1d(np.arange(rows), host["slots"])
    assert (got["k"][free] == KEEP).all() and (got["v"][free] == KEEP).all()


def _put(buf, at, a):
    """bf16 values at an element of a device buffer."""
    bits = bf16_bits(a).reshape(-1)
    assert lib().mlkhip_memcpy_h2d(buf.ptr + at * 2, bits.ctypes.data, bits.nbytes) == 0


def _take(buf, at, shape):
    bits = np.empty(int(np.prod(shape)), np.uint16)
    assert lib().mlkhip_memcpy_d2h(bits.ctypes.data, buf.ptr + at * 2, bits.nbytes) == 0
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(shape)


def test_queries_and_results_past_32_bits(hip):
    # Rows of q and out that start past 2^32 elements, one sequence row by row
    # and one of several row blocks.
    h, g, d, rows, lens = 32, 8, 128, (1 << 20) + 400, [300, 1]
    n = sum(lens)
    km = op.attention_module(rows, kv_rows=n, sequences=2, heads=h, kv_heads=g, dim=d, lse=True)
    rng = np.random.default_rng(8)
    q, k, v = (rounded(rng.standard_normal((n, m, d)), "bf16") for m in (h, g, g))
    bufs = {i: DeviceBuffer(int(np.prod(km.buffers[i].dims)), km.buffers[i].dtype) for i in km.bindable_ids()}
    ids = {km.buffers[i].name: i for i in bufs}
    first = rows - n
    _put(bufs[ids["q"]], first * h * d, q)
    for name, a in (("k", k), ("v", v)):
        _put(bufs[ids[name]], 0, a)
    offsets, start = np.array([first, first + 300, rows]), np.array([0, 300])
    for name, a in (("q_offsets", offsets), ("kv_start", start), ("kv_len", lens)):
        bufs[ids[name]] = DeviceBuffer.from_array(np.asarray(a), "i32")
    hip.build(km).run_device(bufs)
    want, bound, lse, lse_bound, _ = attention(q, k, v, offsets - first, start, lens, scale=d ** -0.5, causal=True, dtype="bf16")
    close(_take(bufs[ids["out"]], first * h * d, (n, h, d)), want, bound, "out")
    close(bufs[ids["lse"]].to_numpy().reshape(rows, h)[first:], lse, lse_bound, "lse")


@pytest.mark.parametrize("d", [128, 130])
def test_norm_rope_rows_past_32_bits(hip, d):
    h, g, n = 32, 4, 200
    rows = (1 << 32) // ((h + 2 * g) * d) + 2 * n
    cache = (1 << 32) // (g * d) + 50
    km = op.qk_norm_rope_module(rows, heads=h, kv_heads=g, dim=d, cache_rows=cache)
    rng = np.random.default_rng(9)
    bufs = {i: DeviceBuffer(int(np.prod(km.buffers[i].dims)), km.buffers[i].dtype) for i in km.bindable_ids()}
    ids = {km.buffers[i].name: i for i in bufs}
    x = rounded(rng.standard_normal((n, h + 2 * g, d)), "bf16")
    first = rows - n
    _put(bufs[ids["qkv"]], first * (h + 2 * g) * d, x)
    slots = np.full(rows, -1)
    slots[first:] = cache - 1 - rng.permutation(n // 2 + n)[:n]
    pos = rng.integers(0, 9000, (1, rows))
    weights = {w: rounded(1 + 0.1 * rng.standard_normal(d), "bf16") for w in ("q_weight", "k_weight")}
    for name, a, dt in (("slots", slots, "i32"), ("positions", pos, "i32"), *((w, a, "bf16") for w, a in weights.items())):
        bufs[ids[name]] = DeviceBuffer.from_array(a, dt)
    hip.build(km).run_device(bufs)
    args = dict(rot=d, theta=1e4, eps=1e-6, interleaved=False, sections=[d // 2], dtype="bf16")
    q, qb = norm_rope(x[:, :h], weights["q_weight"], pos[:, first:], **args)
    k, kb = norm_rope(x[:, h:h + g], weights["k_weight"], pos[:, first:], **args)
    close(_take(bufs[ids["q"]], first * h * d, (n, h, d)), q, qb, "q")
    low = int(slots[first:].min())
    got_k, got_v = (_take(bufs[ids[name]], low * g * d, (cache - low, g, d)) for name in ("k", "v"))
    close(got_k[slots[first:] - low], k, kb, "k")
    assert (got_v[slots[first:] - low] == x[:, h + g:]).all()
