"""The forms that the operators in 8 and 4 bits choose by sizes and alignment: each
is named by the step and gives the f64 references' results."""
import numpy as np
import pytest

from mlk2_amd import operators as op
from mlk2_amd.backend import DeviceBuffer
from operators_ref import attention
from test_operators_bits_gpu import attention_case
from test_operators_bits_uses_gpu import attention_host
from test_operators_gpu import TYPES, close, device, outputs

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
