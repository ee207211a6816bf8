"""Calls of the operators that the headers allow at the ends of their ranges:
magnitudes, long tails, rows that no sequence holds, many tokens to a wave."""
import numpy as np
import pytest

from mlk2_amd import operators as op
from operators_ref import norm_rope, rounded
from test_operators_gpu import close, run

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
