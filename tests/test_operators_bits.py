"""The operators in 8 and 4 bits on the CPU: planning, what a Call may not hold,
the host's conversions, and the artifact's source."""
import numpy as np
import pytest

from mlk2_amd import backend as be
from mlk2_amd import fixtures as fx
from mlk2_amd import operators as op
from mlk2_amd.kernel_ir import KernelBuffer
from operators_bits_ref import load_kv4, quantize_rows, store_kv4


def quantize(**kw):
    return op.quantize_rows_module(20, 48, **kw)


def matmul(**kw):
    return op.matmul_i8_module(20, 30, 48, bias=True, **kw)


def linear(**kw):
    return op.linear_i8_module(20, 30, 48, **kw)


def store(**kw):
    return op.store_kv4_module(20, kv_heads=2, dim=64, cache_rows=40, sequences=3, **kw)


def load(**kw):
    return op.load_kv4_module(20, kv_heads=2, dim=64, cache_rows=40, sequences=3, **kw)


def both(**kw):
    return op.store_load_kv4_module(20, kv_heads=2, dim=64, cache_rows=40, **kw)


def attention(**kw):
    return op.attention_kv4_module(20, kv_rows=50, sequences=3, heads=4, kv_heads=2, dim=64, lse=True, **kw)


@pytest.mark.parametrize("build,name,steps", [(quantize, "quantize-rows", 1), (matmul, "matmul-i8", 1), (linear, "quantize-rows+matmul-i8", 2),
                                              (store, "store-kv4", 1), (load, "load-kv4", 1), (both, "store-kv4+load-kv4", 2),
                                              (attention, "attention-kv4", 1)])
@pytest.mark.parametrize("dtype,policy", [("bf16", "tol-rel1e-2-gfx950-v1"), ("f16", "tol-rel1e-2-gfx950-v1"),
                                          ("f32", "tol-rel1e-5sqrtk-gfx950-v1")])
def test_plans(build, name, steps, dtype, policy):
    assert be.plan(build(dtype=dtype)) == (name, policy, steps)
    assert be.plan_variants(build(dtype=dtype)) == []
    work = be.essential_work(build(dtype=dtype))
    assert not work["bytes_known"] and not work["ops_known"] and work["roofline_lower_sec"] == 0.0


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


@pytest.mark.parametrize("build,change,message", [
    (quantize, _drop("x"), "operand 'x' is missing"),
    (quantize, _drop("codes_out"), "operand 'codes_out' is missing"),
    (quantize, _drop("scale_out"), "operand 'scale_out' is missing"),
    (quantize, _attr("cols", 0), "cols must be a whole number"),
    (quantize, _attr("cols", 49), "columns 0 .. 49 are needed"),
    (quantize, _attr("x_at", 1), "columns 1 .. 49 are needed"),
    (quantize, _attr("scale_out_at", 0), "unknown attribute 'scale_out_at'"),
    (quantize, _attr("heads", 1), "unknown attribute 'heads'"),
    (quantize, _operand("x", dtype="f64"), "'x' must be f16, bf16 or f32"),
    (quantize, _operand("x", dtype="i8"), "'x' must be f16, bf16 or f32"),
    (quantize, _operand("codes_out", dtype="u8"), "'codes_out' must be i8"),
    (quantize, _operand("codes_out", dims=[19, 48]), "'x' and 'codes_out' must have the same rows"),
    (quantize, _operand("scale_out", dims=[21]), "'scale_out' must hold 20 elements"),
    (quantize, _operand("scale_out", dtype="f16"), "'scale_out' must be f32"),
    (quantize, _operand("x", dims=[1 << 31, 48]), "2^31 rows"),
    (matmul, _drop("a"), "operand 'a' is missing"),
    (matmul, _drop("b"), "operand 'b' is missing"),
    (matmul, _drop("a_scale"), "operand 'a_scale' is missing"),
    (matmul, _drop("b_scale"), "operand 'b_scale' is missing"),
    (matmul, _drop("out"), "operand 'out' is missing"),
    (matmul, _attr("inner", 1 << 17), "inner must be a whole number of 1 .. 131071"),
    (matmul, _attr("inner", 49), "columns 0 .. 49 are needed"),
    (matmul, _attr("cols", 31), "columns 0 .. 31 are needed"),
    (matmul, _attr("cols", 29), "'b' must have 29 rows"),
    (matmul, _operand("a", dtype="u8"), "'a' must be i8"),
    (matmul, _operand("b", dtype="f16"), "'b' must be i8"),
    (matmul, _operand("out", dtype="i32"), "'out' must be f16, bf16 or f32"),
    (matmul, _operand("out", dims=[19, 30]), "'a' and 'out' must have the same rows"),
    (matmul, _operand("a_scale", dims=[30]), "'a_scale' must hold 20 elements"),
    (matmul, _operand("b_scale", dims=[20]), "'b_scale' must hold 30 elements"),
    (matmul, _operand("bias", dims=[20]), "'bias' must hold 30 elements"),
    (matmul, _operand("bias", dtype="bf16"), "'bias' must be f32"),
    (matmul, _operand("b", dims=[1 << 32, 48]), "2^31 rows"),
    (linear, _same("b", "a"), "'b' must have 30 rows"),
    (store, _drop("k"), "operand 'k' is missing"),
    (store, _drop("v"), "operand 'v' is missing"),
    (store, _drop("v_codes_out"), "operand 'v_codes_out' is missing"),
    (store, _drop("k_scale_out"), "operand 'k_scale_out' is missing"),
    (store, _drop("slots"), "the codes must have the rows of k"),
    (store, _attr("dim", 63), "dim must be even"),
    (store, _attr("dim", 258), "dim must be a whole number of 2 .. 256"),
    (store, _attr("kv_heads", 3), "columns 0 .. 192 are needed"),
    (store, _attr("kv_heads", 0), "kv_heads must be a whole number"),
    (store, _operand("k", dtype="u8"), "'k' must be f16, bf16 or f32"),
    (store, _operand("v", dtype="f32"), "k and v must be of one dtype"),
    (store, _operand("v", dims=[21, 2, 64]), "k and v must have the same rows"),
    (store, _operand("k_codes_out", dtype="i8"), "'k_codes_out' must be u8"),
    (store, _operand("k_codes_out", dims=[40, 2, 31]), "columns 0 .. 64 are needed"),
    (store, _operand("v_codes_out", dims=[41, 2, 32]), "'v_scale_out' must hold 82 elements"),
    (store, _operand("slots", dims=[40]), "'slots' must hold 20 elements"),
    (store, _operand("q_offsets", dims=[1]), "'q_offsets' must hold"),
    (store, _same("v_codes_out", "k_codes_out"), "overlaps"),
    (store, _same("v_scale_out", "k_scale_out"), "overlaps"),
    (load, _drop("k_out"), "operand 'k_out' is missing"),
    (load, _drop("v_scale"), "operand 'v_scale' is missing"),
    (load, _operand("v_out", dtype="f16"), "k and v must be of one dtype"),
    (load, _operand("k_scale", dims=[40]), "'k_scale' must hold 80 elements"),
    (load, _same("v_out", "k_out"), "overlaps"),
    (attention, _drop("k_codes"), "operand 'k_codes' is missing"),
    (attention, _drop("v_scale"), "operand 'v_scale' is missing"),
    (attention, _drop("q_offsets"), "operand 'q_offsets' is missing"),
    (attention, _drop("out"), "operand 'out' is missing"),
    (attention, _drop("kv_len"), "'kv_start' and 'kv_len' come together"),
    (attention, _drop("kv_start", "kv_len"), "'k_codes' must have the rows of 'q'"),
    (attention, _attr("dim", 33), "dim must be even"),
    (attention, _attr("heads", 5), "multiple of kv_heads"),
    (attention, _attr("scale", 0.0), "scale must be"),
    (attention, _attr("causal", 2), "causal must be"),
    (attention, _operand("k_codes", dtype="i8"), "'k_codes' must be u8"),
    (attention, _operand("k_scale", dtype="bf16"), "'k_scale' must be f32"),
    (attention, _operand("v_codes", dims=[49, 2, 32]), "'v_scale' must hold 98 elements"),
    (attention, _operand("out", dims=[19, 4, 64]), "'q' and 'out' must have the same rows"),
    (attention, _operand("lse", dims=[20, 3]), "'lse' must hold 80 elements"),
    (attention, lambda km: km.nodes[-1].operands.__setitem__("prefix_k", 1), "unknown operand 'prefix_k'"),
])
def test_refused(build, change, message):
    km = build()
    change(km)
    with pytest.raises(be.MlkHipError) as e:
        be.plan(km)
    assert e.value.code == be.REFUSED and message in e.value.message


def test_cache_rows_that_differ():
    km = store()
    _operand("v_codes_out", dims=[41, 2, 32])(km)
    _operand("v_scale_out", dims=[41, 2])(km)
    with pytest.raises(be.MlkHipError, match="the codes of k and v must have the same rows"):
        be.plan(km)


@pytest.mark.parametrize("dtype", ["i8", "u8"])
def test_other_steps_refuse_these_types(dtype):
    for km in (fx.softmax_call_module(8, 8, "f32"), fx.config1_module(n=64), fx.synth_softmax(fx.softmax_call_module(8, 8, "f32"))):
        km.buffers[0].dtype = dtype
        with pytest.raises(be.MlkHipError, match="dtype outside f16/f32/f64"):
            be.plan(km)


def test_the_other_operators_refuse_them():
    km = op.attention_module(20, kv_rows=50, sequences=3, heads=4, kv_heads=2, dim=64)
    km.buffers[km.nodes[0].operands["k"]].dtype = "u8"
    with pytest.raises(be.MlkHipError, match="'k' has another dtype"):
        be.plan(km)


def test_a_cache_is_written_then_read_in_one_module():
    km = store()
    ids = {k[:-4]: v for k, v in km.nodes[0].operands.items() if k.endswith("_out")}
    ids["q"] = km.add_buffer(KernelBuffer("q", "bf16", is_input=True, elements=20 * 256, dims=[20, 4, 64]))
    ids["q_offsets"] = km.nodes[0].operands["q_offsets"]
    for name in ("kv_start", "kv_len"):
        ids[name] = km.add_buffer(KernelBuffer(name, "i32", is_input=True, elements=3, dims=[3]))
    ids["out"] = km.add_buffer(KernelBuffer("out", "bf16", is_output=True, elements=20 * 256, dims=[20, 4, 64]))
    op.add_attention_kv4(km, ids, heads=4, kv_heads=2, dim=64)
    assert be.plan(km) == ("store-kv4+attention-kv4", "tol-rel1e-2-gfx950-v1", 2)


def test_references_on_known_values():
    codes, scale = store_kv4(np.array([[6.0, -0.25, 0.75, 5.0, -3.5, 2.5, 1.25, -0.0]]))
    assert scale[0] == 1 and (load_kv4(codes, scale)[0] == [6, 0, 1, 4, -4, 2, 1, 0]).all()
    codes, scale = quantize_rows(np.array([[127.0, -0.5, 1.5, 2.5, -127.0], [0.0] * 5, [np.inf, 1, 1, 1, 1]]))
    assert (codes == [[127, 0, 2, 2, -127], [0] * 5, [0] * 5]).all() and scale[0] == 1 and scale[1] == 0 and np.isnan(scale[2])


@pytest.mark.parametrize("build", [linear, both, attention])
def test_artifact_source_writes_the_outputs(build, tmp_path):
    km = build()
    data = km.to_json().encode()
    import ctypes
    path = ctypes.create_string_buffer(4096)
    assert be.lib().mlkhip_emit_artifact(data, len(data), b"gfx950", b"", str(tmp_path).encode(), path, 4096) == 0, be.last_error()
    source = (tmp_path / "mlk_kernel.cpp").read_text()
    params = source[source.index("mlk_kernel("):]
    ids = km.bindable_ids()
    for i in ids:
        at = params.index(f"p{ids.index(i)}")
        const = "const double*" in params[max(0, at - 16):at]
        assert const == (not km.buffers[i].is_output), km.buffers[i].name
