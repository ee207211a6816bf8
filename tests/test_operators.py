"""Operator Calls on the CPU: planning, what a Call may not hold, the host's
bf16 conversion, and the modules' documents."""
import numpy as np
import pytest

from mlk2_amd import backend as be
from mlk2_amd import fixtures as fx
from mlk2_amd import operators as op
from mlk2_amd.kernel_ir import KernelBuffer, KernelNode


def norm_rope(**kw):
    args = dict(heads=4, kv_heads=2, dim=64, cache_rows=40, sequences=3)
    args.update(kw)
    return op.qk_norm_rope_module(20, **args)


def attention(**kw):
    args = dict(kv_rows=50, sequences=3, heads=4, kv_heads=2, dim=64, lse=True)
    args.update(kw)
    return op.attention_module(20, **args)


def prefix(**kw):
    args = dict(prefix_rows=9, kv_rows=50, sequences=3, heads=4, kv_heads=2, dim=64, lse=True, prefix_len=True)
    args.update(kw)
    return op.shared_prefix_attention_module(20, **args)


@pytest.mark.parametrize("build,name", [(norm_rope, "qk-norm-rope"), (attention, "attention"), (prefix, "shared-prefix-attention")])
@pytest.mark.parametrize("dtype,policy", [("bf16", "tol-rel1e-2-gfx950-v1"), ("f16", "tol-rel1e-2-gfx950-v1"),
                                          ("f32", "tol-rel1e-5sqrtk-gfx950-v1")])
def test_plans(build, name, dtype, policy):
    assert be.plan(build(dtype=dtype)) == (name, policy, 1)
    assert be.plan_variants(build(dtype=dtype)) == []
    work = be.essential_work(build(dtype=dtype))
    assert not work["bytes_known"] and not work["ops_known"] and work["roofline_lower_sec"] == 0.0


def test_several_calls_in_one_module():
    km = norm_rope()
    q, k, v = km.output_ids()
    offs = [i for i, b in enumerate(km.buffers) if b.name == "q_offsets"][0]
    start = km.add_buffer(KernelBuffer("kv_start", "i32", is_input=True, elements=3, dims=[3]))
    lens = km.add_buffer(KernelBuffer("kv_len", "i32", is_input=True, elements=3, dims=[3]))
    out = km.add_buffer(KernelBuffer("out", "bf16", is_output=True, elements=20 * 256, dims=[20, 4, 64]))
    op.add_attention(km, dict(q=q, k=k, v=v, q_offsets=offs, kv_start=start, kv_len=lens, out=out), heads=4, kv_heads=2, dim=64)
    assert be.plan(km) == ("qk-norm-rope+attention", "tol-rel1e-2-gfx950-v1", 2)


def _operand(name, **buffer):
    def change(km):
        b = km.buffers[km.nodes[-1].operands[name]]
        for key, value in buffer.items():
            setattr(b, key, value)
    return change


def _attr(name, value):
    return lambda km: km.nodes[-1].attrs.__setitem__(name, value)


def _drop(*names):
    return lambda km: [km.nodes[-1].operands.pop(n) for n in names]


def _same(a, b):
    return lambda km: km.nodes[-1].operands.__setitem__(a, km.nodes[-1].operands[b])


def _nest(km):
    km.add_node(KernelNode(op="loop", var="i", end=2, children=[len(km.nodes) - 1]))


@pytest.mark.parametrize("build,change,message", [
    (attention, _attr("heads", 5), "multiple of kv_heads"),
    (attention, _attr("heads", 0), "heads must be a whole number"),
    (attention, _attr("heads", 2.5), "heads must be a whole number"),
    (attention, _attr("dim", 257), "dim must be a whole number"),
    (attention, _attr("dim", 65), "elements, columns 0 .. 260 are needed"),
    (attention, _attr("scale", float("nan")), "scale is not a finite number"),
    (attention, _attr("scale", 0.0), "scale must be"),
    (attention, _attr("causal", 2), "causal must be"),
    (attention, _attr("window", 4), "unknown attribute 'window'"),
    (attention, _attr("q_at", 1), "columns 1 .. 257 are needed"),
    (attention, _attr("q_at", -1), "q_at must be"),
    (attention, _drop("q"), "operand 'q' is missing"),
    (attention, _drop("v"), "operand 'v' is missing"),
    (attention, _drop("out"), "operand 'out' is missing"),
    (attention, _drop("q_offsets"), "operand 'q_offsets' is missing"),
    (attention, _drop("kv_start"), "'kv_start' and 'kv_len' come together"),
    (attention, _drop("kv_start", "kv_len"), "must have the rows of 'q'"),
    (attention, _operand("q", dtype="f64"), "'q' must be f16, bf16 or f32"),
    (attention, _operand("k", dtype="f16"), "'k' has another dtype"),
    (attention, _operand("out", dtype="f32"), "'out' has another dtype"),
    (attention, _operand("lse", dtype="bf16"), "'lse' must be f32"),
    (attention, _operand("lse", dims=[20, 3]), "'lse' must hold 80 elements"),
    (attention, _operand("q_offsets", dtype="f32"), "'q_offsets' must be i32"),
    (attention, _operand("q_offsets", dims=[1]), "'q_offsets' must hold"),
    (attention, _operand("kv_len", dims=[4]), "'kv_len' must hold 3 elements"),
    (attention, _operand("v", dims=[49, 2, 64]), "'k' and 'v' must have the same rows"),
    (attention, _operand("out", dims=[19, 4, 64]), "'q' and 'out' must have the same rows"),
    (attention, _operand("k", dims=[]), "has no dims"),
    (attention, _operand("k", dims=[1 << 31, 2, 64]), "2^31 rows"),
    (attention, _operand("k", dims=[1 << 62, 2, 64]), "too large"),
    (attention, _operand("out", is_output=False, is_temp=True), "neither an input nor an output"),
    (attention, _same("out", "q"), "'out' overlaps 'q'"),
    (attention, lambda km: km.nodes[-1].operands.__setitem__("q", 99), "names no buffer"),
    (attention, lambda km: km.nodes[-1].operands.__setitem__("prefix_k", 1), "unknown operand 'prefix_k'"),
    (attention, _nest, "stands by itself"),
    (prefix, _drop("prefix_k"), "operand 'prefix_k' is missing"),
    (prefix, _operand("prefix_v", dims=[8, 2, 64]), "'prefix_k' and 'prefix_v' must have the same rows"),
    (prefix, _operand("prefix_len", dims=[3]), "'prefix_len' must hold 1 elements"),
    (norm_rope, _attr("rot", 66), "rot must be"),
    (norm_rope, _attr("rot", 31), "rot must be even"),
    (norm_rope, _attr("eps", -1.0), "eps must be"),
    (norm_rope, _attr("theta", 0.5), "theta must be"),
    (norm_rope, _attr("section_1", 3), "sections must add up"),
    (norm_rope, _operand("positions", dims=[2, 20]), "'positions' must hold 20 elements"),
    (norm_rope, _operand("slots", dims=[21]), "'slots' must hold 20 elements"),
    (norm_rope, _drop("slots"), "must have the rows of 'k'"),
    (norm_rope, _drop("v"), "'v' and 'v_out' come together"),
    (norm_rope, _drop("q_weight"), "'q_weight' and 'k_weight' come together"),
    (norm_rope, _operand("q_weight", dims=[63]), "'q_weight' must hold 64 elements"),
    (norm_rope, _operand("q_weight", dtype="f16"), "weights must be f32"),
    (norm_rope, _operand("k_weight", dtype="f32"), "'k_weight' must be"),
    (norm_rope, _operand("v_out", dims=[41, 2, 64]), "'k_out' and 'v_out' must have the same rows"),
    (norm_rope, _same("v_out", "k_out"), "overlaps"),
])
def test_refused(build, change, message):
    km = build()
    change(km)
    with pytest.raises(be.MlkHipError) as e:
        be.plan(km)
    assert e.value.code == be.REFUSED and message in e.value.message


def test_in_place_rows_are_taken():
    # q, k and v of the fused rows in their own places, without a cache.
    km = op.qk_norm_rope_module(20, heads=4, kv_heads=2, dim=64)
    ops, attrs = km.nodes[0].operands, km.nodes[0].attrs
    for part in "qkv":
        ops[f"{part}_out"] = ops[part]
        if part != "q":
            attrs[f"{part}_out_at"] = attrs[f"{part}_at"]
    assert be.plan(km)[0] == "qk-norm-rope"
    attrs["k_out_at"] = attrs["k_at"] - 64
    with pytest.raises(be.MlkHipError, match="overlaps"):
        be.plan(km)


@pytest.mark.parametrize("dtype", ["bf16", "i32"])
def test_other_steps_refuse_the_operators_types(dtype):
    for km in (fx.softmax_call_module(8, 8, "f32"), fx.config1_module(n=64), fx.synth_softmax(fx.softmax_call_module(8, 8, "f32"))):
        km.buffers[0].dtype = dtype
        with pytest.raises(be.MlkHipError, match="dtype outside f16/f32/f64"):
            be.plan(km)


def test_bf16_conversion_rounds_once():
    # Around each tie of bf16, by f64 steps that f32 does not hold.
    v = np.array([1.0, 1.5, 3.0e38, 1e-40, 65504.0])
    up = 2.0 ** (np.floor(np.log2(v)) - 8)
    for near in (0.0, 2.0 ** -40, -2.0 ** -40):
        x = v + up + near * v
        got = be.bf16_values(be.bf16_bits(x)).astype(np.float64)
        step = 2.0 ** np.maximum(np.floor(np.log2(x)) - 7, -133)
        lo = np.floor(x / step) * step
        want = np.where(x - lo > step / 2, lo + step, np.where(x - lo < step / 2, lo, np.where((lo / step) % 2 == 0, lo, lo + step)))
        assert np.array_equal(got, want)
    special = be.bf16_values(be.bf16_bits([np.inf, -np.inf, np.nan, 1e300, -0.0]))
    assert special[0] == np.inf and special[1] == -np.inf and np.isnan(special[2]) and special[3] == np.inf
    assert special[4] == 0 and np.signbit(special[4])


def test_document_round_trip_keeps_the_call():
    km = attention(scale=0.1)
    doc = km.to_dict()["nodes"][0]
    assert doc["operands"]["q"] == 0 and doc["attrs"]["scale"] == 0.1
