"""qk_norm_rope where a wave takes several tokens in turn, reads units of heads
ahead, and holds units of q, k and v together: what prompts run on.

The launch has 4096 waves at most. Past 4096 tokens a wave takes tokens 4096
apart, all their units; below, a token's units are spread over 4096 / tokens
waves. A unit is 64 lanes of 8 columns; 4 units (f32: 2) are read at a time."""
import numpy as np
import pytest

from mlk2_amd import operators as op
from mlk2_amd.kernel_ir import KernelBuffer, KernelModule
from operators_ref import rounded
from test_operators_gpu import TYPES, norm_rope_case, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inter", [False, True])
def test_several_tokens_to_a_wave(hip, dtype, inter):
    norm_rope_case(hip, 8200, 3, 1, 16, dtype, inter=inter, cache=8300)
    norm_rope_case(hip, 4099, 10, 2, 64, dtype, inter=inter)
    norm_rope_case(hip, 9001, 1, 1, 24, dtype, inter=inter, rot=16, norm=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("valid", [8200, 6000, 4097, 4096, 100])
def test_several_tokens_to_a_wave_and_rows_behind_the_last(hip, dtype, valid):
    norm_rope_case(hip, 8200, 2, 1, 32, dtype, sections=[6, 5, 5], cache=8250, valid=valid)


# 40 + 8 + 8 heads of 128 are 10, 2 and 2 units; of f32 too.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,h,g,d", [(1500, 40, 8, 128), (2050, 40, 8, 128), (1300, 15, 3, 64), (4097, 6, 2, 256), (700, 33, 11, 80)])
def test_several_units_to_a_wave(hip, dtype, t, h, g, d):
    norm_rope_case(hip, t, h, g, d, dtype, cache=t + 7, wt="f32")
    norm_rope_case(hip, t, h, g, d, dtype, sections=[d // 2 - 2 * (d // 8), d // 8, d // 8], valid=t - t // 3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,d", [(5000, 32), (8193, 64)])
def test_several_tokens_in_place(hip, dtype, t, d):
    # The fused rows' q, k and v in their own places equal those of the copy.
    h, g = 3, 1
    rng = np.random.default_rng(t)
    host = {"qkv": rounded(rng.standard_normal((t, (h + 2 * g) * d)), dtype), "positions": rng.integers(0, 9000, t)}
    for w in ("q_weight", "k_weight"):
        host[w] = rounded(rng.standard_normal(d), dtype)
    want = run(hip, op.qk_norm_rope_module(t, heads=h, kv_heads=g, dim=d, dtype=dtype), host)
    km = KernelModule(name="in_place")
    ids = {}
    for name, dt, dims in (("q_weight", dtype, [d]), ("k_weight", dtype, [d]), ("positions", "i32", [1, t])):
        ids[name] = km.add_buffer(KernelBuffer(name, dt, is_input=True, elements=int(np.prod(dims)), dims=dims))
    x = km.add_buffer(KernelBuffer("qkv", dtype, is_output=True, elements=t * (h + 2 * g) * d, dims=[t, (h + 2 * g) * d]))
    at = {"q": 0, "k": h * d, "v": (h + g) * d}
    ids.update({p + o: x for p in at for o in ("", "_out")})
    op.add_qk_norm_rope(km, ids, heads=h, kv_heads=g, dim=d, columns={p + o: c for p, c in at.items() for o in ("", "_out")})
    got = run(hip, km, host)["qkv"].reshape(t, h + 2 * g, d)
    assert (got[:, :h] == want["q"]).all() and (got[:, h:h + g] == want["k"]).all() and (got[:, h + g:] == want["v"]).all()
