"""shared_prefix_attention where its launches branch: more key ranges than a
wave has lanes, the widest row blocks, prefix columns of wider rows, and the
same keys copied in front of each sequence's."""
import numpy as np
import pytest

from attention_abi import Attention
from mlk2_amd import operators as op
from mlk2_amd.kernel_ir import KernelBuffer, KernelModule
from operators_ref import attention, rounded
from test_operators_gpu import TYPES, attention_case, close, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("own,prefix,least", [(512, 8192, 65), (8200, 8200, 100)])
def test_more_than_64_ranges(hip, dtype, d, own, prefix, least):
    # The join reads its ranges' weights from two registers of 64 lanes.
    assert Attention.of(heads=8, kv_heads=1, dim=d, sequences=1, q_rows=1, kv_rows=own, prefix_rows=prefix, dtype=dtype).ranges() >= least
    attention_case(hip, [1], [own], 8, 1, d, dtype, prefix=prefix, prefix_rows=prefix)
    attention_case(hip, [1], [own // 3], 8, 1, d, dtype, prefix=prefix // 5, prefix_rows=prefix, gap=own // 3, poison=True)


# 400 rows of 40 heads and 40 key/value heads are 160 blocks of 256 rows.
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_widest_blocks_over_the_prefix(hip, dtype, d):
    h, g, n, each, prefix = 80, 40, 16, 25, 150
    km = op.shared_prefix_attention_module(n * each, prefix_rows=prefix, kv_rows=n * each, sequences=n, heads=h, kv_heads=g, dim=d, dtype=dtype)
    name = hip.build(km).step_kernel_name(0)
    assert f", {d}, 8, 1, 64, " in name.split("+")[0], name
    attention_case(hip, [each] * n, [each] * n, h, g, d, dtype, prefix=prefix, prefix_rows=prefix)
    attention_case(hip, [each + (-1) ** i * (i % 7) for i in range(n)], [each + 7] * n, h, g, d, dtype, prefix=prefix - 21, prefix_rows=prefix,
                   gap=1, poison=True, spare=9)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,prefix", [([1] * 5, 300), ([20, 1, 0, 9], 77), ([100, 130], 200)])
def test_equals_attention_over_copied_prefixes(hip, dtype, lens, prefix):
    # The same queries over a cache that holds the prefix before each sequence's
    # own keys: each side within the reference's bound.
    h, g, d, n, t = 8, 2, 128, len(lens), sum(lens)
    rng = np.random.default_rng(prefix)
    own = [m + i for i, m in enumerate(lens)]
    q, k, v, pk, pv = (rounded(rng.standard_normal((rows, m, d)), dtype)
                       for rows, m in ((t, h), (sum(own), g), (sum(own), g), (prefix, g), (prefix, g)))
    offsets, start = np.concatenate([[0], np.cumsum(lens)]), np.concatenate([[0], np.cumsum(own)[:-1]])
    args = dict(sequences=n, heads=h, kv_heads=g, dim=d, dtype=dtype, lse=True)
    shared = run(hip, op.shared_prefix_attention_module(t, prefix_rows=prefix, kv_rows=sum(own), **args),
                 {"q": q, "k": k, "v": v, "prefix_k": pk, "prefix_v": pv, "q_offsets": offsets, "kv_start": start, "kv_len": own})
    whole = [np.concatenate([np.concatenate([p, x[s:s + m]]) for s, m in zip(start, own)]) for p, x in ((pk, k), (pv, v))]
    longer = [prefix + m for m in own]
    copied = run(hip, op.attention_module(t, kv_rows=sum(longer), **args),
                 {"q": q, "k": whole[0], "v": whole[1], "q_offsets": offsets, "kv_start": np.concatenate([[0], np.cumsum(longer)[:-1]]),
                  "kv_len": longer})
    _, bound, _, lse_bound, _ = attention(q, k, v, offsets, start, own, scale=d ** -0.5, causal=True, dtype=dtype, prefix_k=pk, prefix_v=pv)
    close(shared["out"], copied["out"], 2 * bound)
    close(shared["lse"], copied["lse"], 2 * lse_bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,pad,at", [(64, 8, 8), (64, 3, 1), (128, 16, 0), (40, 8, 8)])
@pytest.mark.parametrize("lens", [[1] * 6, [70, 41]])
def test_columns_of_wider_prefix_rows(hip, dtype, d, pad, at, lens):
    # Keys and values of the prefix in one buffer's rows, on and off 16 bytes.
    h, g, prefix, t = 4, 2, 130, sum(lens)
    rng = np.random.default_rng(d + pad)
    width = 2 * g * d + pad
    x = rounded(rng.standard_normal((prefix, width)), dtype)
    x[:, :at], x[:, at + 2 * g * d:] = np.nan, np.nan
    q, k, v = (rounded(rng.standard_normal((t, m, d)), dtype) for m in (h, g, g))
    km = KernelModule(name="prefix_columns")
    ids = {}
    for name, dt, dims in (("x", dtype, [prefix, width]), ("q", dtype, [t, h, d]), ("k", dtype, [t, g, d]), ("v", dtype, [t, g, d]),
                           ("q_offsets", "i32", [len(lens) + 1])):
        ids[name] = km.add_buffer(KernelBuffer(name, dt, is_input=True, elements=int(np.prod(dims)), dims=dims))
    out = km.add_buffer(KernelBuffer("out", dtype, is_output=True, elements=t * h * d, dims=[t, h, d]))
    op.add_attention(km, dict(q=ids["q"], k=ids["k"], v=ids["v"], prefix_k=ids["x"], prefix_v=ids["x"], q_offsets=ids["q_offsets"], out=out),
                     heads=h, kv_heads=g, dim=d, columns=dict(prefix_k=at, prefix_v=at + g * d))
    offsets = np.concatenate([[0], np.cumsum(lens)])
    got = run(hip, km, {"x": x, "q": q, "k": k, "v": v, "q_offsets": offsets})["out"]
    pk, pv = (x[:, c:c + g * d].reshape(prefix, g, d) for c in (at, at + g * d))
    want, bound, _, _, _ = attention(q, k, v, offsets, offsets[:-1], lens, scale=d ** -0.5, causal=True, dtype=dtype, prefix_k=pk, prefix_v=pv)
    close(got, want, bound)
