"""The forms that the operators in 8 and 4 bits choose by sizes and alignment: each
is named by the step and gives the f64 references' results."""
import ctypes

import numpy as np
import pytest

from mlk2_amd import operators as op
from mlk2_amd.backend import DeviceBuffer
from operators_bits_ref import matmul_i8
from operators_ref import attention
from test_operators_bits_gpu import attention_case, matmul_case
from test_operators_bits_uses_gpu import attention_host
from test_operators_gpu import TYPES, close, device, outputs
from test_score_two_pass_gpu import _Capture

pytestmark = pytest.mark.gpu
NAMES = {"bf16": "__bf16", "f16": "_Float16", "f32": "float"}


def width(d):
    """The columns that a kernel's sums are held for."""
    return 64 if d <= 64 else 96 if d <= 96 else 128 if d <= 128 else 256


def attention_form(hip, q_lens, k_lens, h, g, d, dtype, spare=0, rows=None):
    km = op.attention_kv4_module(sum(q_lens) + spare, kv_rows=rows or sum(k_lens), sequences=len(q_lens), heads=h, kv_heads=g, dim=d, dtype=dtype)
    return hip.build(km).step_kernel_name(0)


def tiles(dtype, d, rows, waves):
    return f"attentionKv4Tiles<{NAMES[dtype]}, {width(d)}, {rows}, {waves}>"


# ------------------------------------------------------------ attention_kv4 --
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [48, 80, 112, 144, 176, 208, 240])
@pytest.mark.parametrize("g", [1, 3])
def test_cache_rows_of_8_bytes(hip, dtype, d, g):
    # Rows of the cache are 8 bytes past whole sixteens.
    assert g * d // 2 % 16 == 8
    for q_lens, k_lens, rows in (([1, 1], [70, 333], 16), ([40, 3], [90, 3], 32)):
        assert attention_form(hip, q_lens, k_lens, 2 * g, g, d, dtype) == tiles(dtype, d, rows, 4)
        attention_case(hip, q_lens, k_lens, 2 * g, g, d, dtype, spare=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 80])
@pytest.mark.parametrize("which", ["k_codes", "v_codes", "both"])
def test_cache_at_8_bytes(hip, dtype, d, which):
    # Codes whose buffers start 8 bytes past sixteen, as columns of wider rows do.
    h, g, q_lens, k_lens = 4, 2, [20, 1], [50, 900]
    rng = np.random.default_rng(d)
    host, k, v = attention_host(rng, q_lens, [0, 50], k_lens, 950, h, g, d, dtype)
    km = op.attention_kv4_module(21, kv_rows=950, sequences=2, heads=h, kv_heads=g, dim=d, dtype=dtype)
    bufs = device(km, host)
    for i in km.bindable_ids():
        name = km.buffers[i].name
        if name == which or (which == "both" and name.endswith("_codes")):
            bufs[i] = _Past8(host[name])
    hip.build(km).run_device(bufs)
    want, bound, *_ = attention(host["q"], k, v, host["q_offsets"], host["kv_start"], k_lens, scale=d ** -0.5, causal=True, dtype=dtype)
    close(outputs(km, bufs)["out"], want, bound)


class _Past8:
    """Codes that start 8 bytes past a 256-byte boundary."""

    def __init__(self, codes):
        codes = np.asarray(codes).reshape(-1)
        self.whole, self.elements = DeviceBuffer.from_array(np.concatenate([np.full(8, 255), codes]), "u8"), codes.size

    def binding(self):
        b = self.whole.binding()
        b.ptr += 8
        b.elements -= 8
        return b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 80, 96, 128, 160, 192, 256])
def test_single_tokens_by_16_rows(hip, dtype, d):
    q_lens, k_lens, h, g = [1, 1, 1], [70, 3, 333], 6, 2
    assert attention_form(hip, q_lens, k_lens, h, g, d, dtype, spare=1) == tiles(dtype, d, 16, 4)
    attention_case(hip, q_lens, k_lens, h, g, d, dtype, spare=1)
    attention_case(hip, q_lens, k_lens, h, g, d, dtype, causal=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 80, 96, 128, 160, 256])
@pytest.mark.parametrize("q_lens,k_lens,rows", [([1], [2500], 16), ([1, 1, 2], [9000, 40, 33], 16), ([40], [2300], 32), ([70, 1], [4500, 900], 32)])
def test_keys_dealt_out(hip, dtype, d, q_lens, k_lens, rows):
    join = f"attentionJoin<{NAMES[dtype]}, {16 if d <= 64 else 32 if d <= 128 else 64}>"
    assert attention_form(hip, q_lens, k_lens, 4, 2, d, dtype) == f"{tiles(dtype, d, rows, 4)}+{join}"
    attention_case(hip, q_lens, k_lens, 4, 2, d, dtype)
    attention_case(hip, q_lens, k_lens, 4, 2, d, dtype, causal=False, gap=3, poison=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 80, 128, 256])
def test_one_wave_to_a_row_block(hip, dtype, d):
    # From 4096 row blocks of 32 on: 64 kv heads, sequences of one to three rows of
    # blocks (nine heads a group; 5 tokens are 45 rows).
    h, g, q_lens = 576, 64, [2, 1, 3, 2, 5, 0, 2, 1] * 8
    k_lens = [2 + i % 70 if i % 5 else q for i, q in enumerate(q_lens)]
    assert attention_form(hip, q_lens, k_lens, h, g, d, dtype) == tiles(dtype, d, 32, 1)
    attention_case(hip, q_lens, k_lens, h, g, d, dtype, causal=d != 128)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_prompts_by_one_wave(hip, dtype):
    # As many blocks of whole prompts, whose tiles fill the ring.
    h, g, d, q_lens = 32, 32, 64, [700, 1, 900, 300, 800, 500, 600, 300]
    assert attention_form(hip, q_lens, q_lens, h, g, d, dtype) == tiles(dtype, d, 32, 1)
    rng = np.random.default_rng(9)
    start = np.concatenate([[0], np.cumsum(q_lens)[:-1]])
    host, k, v = attention_host(rng, q_lens, start, q_lens, sum(q_lens), h, g, d, dtype)
    km = op.attention_kv4_module(sum(q_lens), kv_rows=sum(q_lens), sequences=len(q_lens), heads=h, kv_heads=g, dim=d, dtype=dtype)
    bufs = device(km, host)
    hip.build(km).run_device(bufs)
    got = outputs(km, bufs)["out"]
    # Some heads of some rows: a reference of all takes minutes.
    for b, n in enumerate(q_lens):
        for i in sorted({0, n // 3, n - 1}):
            kk, vv = (x[start[b]:start[b] + i + 1, 5:8] for x in (k, v))
            q = host["q"][start[b] + i, 5:8]
            want, bound, *_ = attention(q[None], kk, vv, [0, 1], [0], [i + 1], scale=d ** -0.5, causal=True, dtype=dtype)
            close(got[start[b] + i, 5:8], want[0], bound[0], f"row {i} of {b}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_lens,k_lens", [([1], [100]), ([1] * 8, [9000 - 1000 * i for i in range(8)]), ([70, 3], [2500, 900])])
def test_runs_repeat_their_bits(hip, dtype, q_lens, k_lens):
    rng = np.random.default_rng(4)
    start = np.concatenate([[0], np.cumsum(k_lens)[:-1]])
    host, *_ = attention_host(rng, q_lens, start, k_lens, sum(k_lens), 8, 2, 128, dtype)
    km = op.attention_kv4_module(sum(q_lens), kv_rows=sum(k_lens), sequences=len(q_lens), heads=8, kv_heads=2, dim=128, dtype=dtype, lse=True)
    art, bufs = hip.build(km), device(km, host)
    art.run_device(bufs)
    first = outputs(km, bufs)
    for _ in range(5):
        art.run_device(bufs)
        for name, a in outputs(km, bufs).items():
            assert np.array_equal(a, first[name])


# ---------------------------------------------------------------- matmul_i8 --
FORMS = [(1, 300, 512, "Few", "1, 1, true"), (16, 6500, 512, "Few", "1, 2, true"), (16, 6500, 511, "Few", "1, 2, false"), (20, 300, 257, "Few", "2, 1, false"),
         (32, 6500, 256, "Few", "2, 2, true"), (48, 300, 256, "Few", "4, 1, true"), (48, 6500, 256, "Few", "4, 2, true"), (64, 6401, 255, "Few", "4, 2, false"),
         (33, 8200, 256, "Tiles", "2, 2, 2, 2, 8"), (250, 5100, 96, "Tiles", "2, 2, 4, 2, 6"), (640, 5100, 528, "Tiles", "2, 2, 4, 4, 6"),
         (2040, 4090, 400, "Tiles", "2, 2, 4, 4, 4"), (2500, 4000, 511, "Tiles", "4, 2, 4, 8, 4"),
         (2560, 4096, 512, "Tiles", "4, 2, 4, 8, 4"), (2500, 4000, 576, "Tiles", "4, 2, 4, 8, 4"), (2560, 4096, 752, "Tiles", "4, 2, 4, 8, 4"),
         (2560, 4096, 832, "Tiles", "4, 2, 4, 8, 4"), (2500, 4000, 1040, "Tiles", "4, 2, 4, 8, 4")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,kernel,parameters", FORMS)
def test_product_forms(hip, dtype, m, n, k, kernel, parameters):
    pack = "matmulI8Pack+" if kernel == "Tiles" and k % 16 else ""
    assert hip.build(op.matmul_i8_module(m, n, k, dtype=dtype)).step_kernel_name(0) == f"{pack}matmulI8{kernel}<{NAMES[dtype]}, {parameters}>"
    matmul_case(hip, m, n, k, dtype, bias=m % 2 == 0)


@pytest.mark.parametrize("m,n,k", [(70, 130, 8192), (200, 70, 5000), (64, 64, 4096), (40, 200, 16384)])
def test_product_in_ranges_of_k(hip, m, n, k):
    for dtype in TYPES:
        assert hip.build(op.matmul_i8_module(m, n, k, dtype=dtype)).step_kernel_name(0).endswith(f"matmulI8Join<{NAMES[dtype]}>")
        matmul_case(hip, m, n, k, dtype, bias=True)


# -------------------------------------------------------- without workspace --
def _nodes(cap):
    n = ctypes.c_size_t(0)
    cap("hipGraphGetNodes", cap.graph, None, ctypes.byref(n))
    return n.value


@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("k,launches", [(8191, 3), (8192, 2)])
def test_products_captured_with_and_without_a_workspace(hip, room, k, launches):
    # A stream's first run, under capture, has no workspace: one launch, in the form
    # that needs none; after a run on the stream, its copies, tiles and join.
    rng = np.random.default_rng(k)
    m, n = 70, 130
    a, b = rng.integers(-127, 128, (m, k)), rng.integers(-127, 128, (n, k))
    sa, sb = (np.exp(rng.standard_normal(x)).astype(np.float32).astype(np.float64) * 2.0 ** -9 for x in (m, n))
    want, bound = matmul_i8(a, sa, b, sb, None, "f16")
    assert np.abs(want).max() < 65504
    km = op.matmul_i8_module(m, n, k, dtype="f16")
    art, bufs, cap = hip.build(km), device(km, {"a": a, "b": b, "a_scale": sa, "b_scale": sb}), _Capture()
    if room:
        art.run_device(bufs, stream=cap.stream.value)
    with cap as stream:
        art.run_device(bufs, stream=stream, sync=False)
    assert _nodes(cap) == (launches if room else 1)
    for _ in range(3):
        bufs[km.output_ids()[0]].fill_zero()
        cap.replay()
        close(outputs(km, bufs)["out"], want, bound)
    cap.close()


@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_captured_with_and_without_a_workspace(hip, dtype, room):
    h, g, d, rows, lens = 8, 2, 64, 12000, [9000, 3000]
    rng = np.random.default_rng(3)
    km = op.attention_kv4_module(2, kv_rows=rows, sequences=2, heads=h, kv_heads=g, dim=d, dtype=dtype)
    host, k, v = attention_host(rng, [1, 1], [0, 9000], lens, rows, h, g, d, dtype)
    want, bound, *_ = attention(host["q"], k, v, [0, 1, 2], [0, 9000], lens, scale=0.125, causal=True, dtype=dtype)
    art, bufs, cap = hip.build(km), device(km, host), _Capture()
    if room:
        art.run_device(bufs, stream=cap.stream.value)
    with cap as stream:
        art.run_device(bufs, stream=stream, sync=False)
    assert _nodes(cap) == (2 if room else 1)
    for _ in range(3):
        bufs[km.output_ids()[0]].fill_zero()
        cap.replay()
        close(outputs(km, bufs)["out"], want, bound)
    cap.close()


# ------------------------------------------------------------------- search --
def test_the_search_prices_them_and_claims_no_grid(hip):
    # The declared rate is that of the fastest matrix instructions a plan runs on.
    for km, rate in ((op.linear_i8_module(20, 30, 48, dtype="f32"), 5e15), (op.matmul_i8_module(20, 30, 48), 5e15),
                     (op.attention_kv4_module(4, sequences=1, heads=2, kv_heads=1, dim=64, dtype="f32"), 2.5e15),
                     (op.quantize_rows_module(20, 48), 157.3e12), (op.store_load_kv4_module(4, cache_rows=9, kv_heads=1, dim=64), 157.3e12)):
        art = hip.build(km)
        report = art.autotune({i: DeviceBuffer.from_array(np.zeros(km.buffers[i].dims), km.buffers[i].dtype) for i in km.bindable_ids()}, reps=2)
        assert report["environment"]["declared_ops_per_sec"] == rate
        for step in report["steps"]:
            assert step["launch"]["covered"] and step["launch"]["instances"] > 0 and "workgroups" not in step["launch"], step["launch"]
