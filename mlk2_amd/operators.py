"""KernelModule builders for the operators around attention.

Each builder returns a module of one Call node whose operands are buffers by
name; ``add_*`` appends the Call to a module that already holds the buffers,
so that several run as one module. Bind the buffers in table order
(``KernelModule.bindable_ids``): inputs first, as the builders list them, then
the outputs. The operators and their operands:

``qk_norm_rope``
    Rows of q, k (and v): ``heads`` (``kv_heads``) heads of ``dim`` elements.
    Each head of q and k becomes x / sqrt(mean(x^2) + eps) * weight, its first
    ``rot`` elements then turned in pairs by the angles positions[axis, t] *
    theta^(-2 i / rot) (pair i is elements i and i + rot/2, or 2i and 2i + 1
    with ``interleaved``; ``sections`` counts the pairs of each position axis).
    k_out and v_out take token t at row ``slots[t]`` (row t without slots); a
    slot outside the rows stores nothing, one that names a row again leaves
    pieces of either token there. With ``q_offsets`` the tokens from
    q_offsets[-1] on are left alone.
``attention``
    out = softmax(scale q k^T) v over packed sequences: sequence b has the
    query rows q_offsets[b] .. q_offsets[b + 1] and the keys kv_start[b] ..
    kv_start[b] + kv_len[b] (without those, the rows of its queries). Causal:
    the last query sees every key, the one before it one key less, and so on.
    A query that sees no key gets zeros, and -inf in ``lse``. Rows behind the
    last sequence are left alone; lengths are clipped to the buffers.
``shared_prefix_attention``
    The same with every sequence's keys behind the rows of prefix_k, prefix_v
    (the first ``prefix_len`` of them).

``quantize_rows``
    Rows of x as 8-bit integers: scale_out[t] = max |x[t]| / 127, codes_out[t]
    = x[t] / scale_out[t] rounded (half way to even).
``matmul_i8``
    out[t, n] = (sum of a[t, k] b[n, k]) a_scale[t] b_scale[n] + bias[n]: rows
    a and b of 8-bit integers (b a row for each output channel), exact sums.
``store_kv4``, ``load_kv4``
    Heads of k and v to the rows ``slots`` of a cache in 4 bits, and back: a
    scale for each row and head, its largest magnitude over 6, and 4-bit
    floating-point numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte.
``attention_kv4``
    ``attention`` whose keys and values are such a cache's rows.

Types: f16, bf16 or f32, the same for all rows; sums are held in f32 and each
output is rounded once. Attention's weights are rounded to the type of v before
they meet it, so that f16 and bf16 run on the matrix cores; their sum is of the
f32 values. Codes are i8 (``quantize_rows``, ``matmul_i8``) and u8 (the cache's), scales
f32; a row or head with a value that is not finite has scale NaN and codes 0.
Buffers' sizes decide how an attention runs, not the lengths in them,
and rows off 16 bytes (codes: 8) or more than 4096 sequences run a wave to a row (see
include/mlk_hip.h).
"""
from __future__ import annotations

from typing import Optional, Sequence

from .kernel_ir import KernelBuffer, KernelModule, KernelNode


def _buffer(km: KernelModule, name: str, dtype: str, dims: Sequence[int], output: bool = False) -> int:
    n = 1
    for d in dims:
        n *= int(d)
    return km.add_buffer(KernelBuffer(name=name, dtype=dtype, is_input=not output, is_output=output, elements=n,
                                      dims=[int(d) for d in dims]))


def _call(km: KernelModule, math: str, operands: dict, attrs: dict) -> int:
    return km.add_node(KernelNode(op="call", math=math, operands={k: v for k, v in operands.items() if v is not None},
                                  attrs={k: v for k, v in attrs.items() if v is not None}))


def add_qk_norm_rope(km: KernelModule, operands: dict, *, heads: int, kv_heads: int, dim: int, eps: float = 1e-6,
                     theta: float = 10000.0, rot: Optional[int] = None, interleaved: bool = False,
                     sections: Optional[Sequence[int]] = None, columns: Optional[dict] = None) -> int:
    """Appends a qk_norm_rope Call. ``operands`` maps q, k, v, q_weight,
    k_weight, positions, slots, q_offsets, q_out, k_out and v_out to buffer
    ids (None or absent: without it); ``columns`` gives the first column of
    rows that start further in, by operand."""
    attrs = dict(heads=heads, kv_heads=kv_heads, dim=dim, eps=eps, theta=theta, rot=rot, interleaved=int(interleaved))
    for i, s in enumerate(sections or ()):
        attrs[f"section_{i}"] = s
    attrs.update({f"{k}_at": v for k, v in (columns or {}).items()})
    return _call(km, "qk_norm_rope", operands, attrs)


def add_attention(km: KernelModule, operands: dict, *, heads: int, kv_heads: int, dim: int, causal: bool = True,
                  scale: Optional[float] = None, columns: Optional[dict] = None) -> int:
    """Appends an attention Call, or a shared_prefix_attention Call where
    ``operands`` holds prefix_k. ``operands`` maps q, k, v, q_offsets,
    kv_start, kv_len, prefix_k, prefix_v, prefix_len, out and lse to buffer
    ids (None or absent: without it). ``scale`` is 1 / sqrt(dim) by default."""
    attrs = dict(heads=heads, kv_heads=kv_heads, dim=dim, causal=int(causal), scale=scale)
    attrs.update({f"{k}_at": v for k, v in (columns or {}).items()})
    shared = operands.get("prefix_k") is not None
    return _call(km, "shared_prefix_attention" if shared else "attention", operands, attrs)


def qk_norm_rope_module(tokens: int, *, heads: int, kv_heads: int, dim: int, dtype: str = "bf16",
                        cache_rows: Optional[int] = None, norm: bool = True, weight_dtype: Optional[str] = None,
                        positions: bool = True, eps: float = 1e-6, theta: float = 10000.0, rot: Optional[int] = None,
                        interleaved: bool = False, sections: Optional[Sequence[int]] = None,
                        sequences: Optional[int] = None) -> KernelModule:
    """Over a fused projection's rows. Buffers: qkv [tokens, (heads + 2
    kv_heads) dim], q_weight and k_weight [dim] (with ``norm``), positions
    [axes, tokens] (with ``positions``), slots [tokens] (with ``cache_rows``),
    q_offsets [sequences + 1] (with ``sequences``); outputs q [tokens, heads,
    dim], k and v [cache_rows or tokens, kv_heads, dim]."""
    km = KernelModule(name="qk_norm_rope")
    width = (heads + 2 * kv_heads) * dim
    op = {}
    op["q"] = op["k"] = op["v"] = _buffer(km, "qkv", dtype, [tokens, width])
    if norm:
        op["q_weight"] = _buffer(km, "q_weight", weight_dtype or dtype, [dim])
        op["k_weight"] = _buffer(km, "k_weight", weight_dtype or dtype, [dim])
    if positions:
        axes = max((i + 1 for i, s in enumerate(sections or ()) if s > 0), default=1)
        op["positions"] = _buffer(km, "positions", "i32", [axes, tokens])
    if cache_rows is not None:
        op["slots"] = _buffer(km, "slots", "i32", [tokens])
    if sequences is not None:
        op["q_offsets"] = _buffer(km, "q_offsets", "i32", [sequences + 1])
    rows = tokens if cache_rows is None else cache_rows
    op["q_out"] = _buffer(km, "q", dtype, [tokens, heads, dim], output=True)
    op["k_out"] = _buffer(km, "k", dtype, [rows, kv_heads, dim], output=True)
    op["v_out"] = _buffer(km, "v", dtype, [rows, kv_heads, dim], output=True)
    add_qk_norm_rope(km, op, heads=heads, kv_heads=kv_heads, dim=dim, eps=eps, theta=theta, rot=rot,
                     interleaved=interleaved, sections=sections,
                     columns={"k": heads * dim, "v": (heads + kv_heads) * dim})
    return km


def _attention(km: KernelModule, op: dict, tokens: int, kv_rows: Optional[int], sequences: int, heads: int, kv_heads: int,
               dim: int, dtype: str, causal: bool, scale: Optional[float], lse: bool) -> KernelModule:
    rows = tokens if kv_rows is None else kv_rows
    op["k"] = _buffer(km, "k", dtype, [rows, kv_heads, dim])
    op["v"] = _buffer(km, "v", dtype, [rows, kv_heads, dim])
    op["q_offsets"] = _buffer(km, "q_offsets", "i32", [sequences + 1])
    if kv_rows is not None:
        op["kv_start"] = _buffer(km, "kv_start", "i32", [sequences])
        op["kv_len"] = _buffer(km, "kv_len", "i32", [sequences])
    op["out"] = _buffer(km, "out", dtype, [tokens, heads, dim], output=True)
    if lse:
        op["lse"] = _buffer(km, "lse", "f32", [tokens, heads], output=True)
    add_attention(km, op, heads=heads, kv_heads=kv_heads, dim=dim, causal=causal, scale=scale)
    return km


def attention_module(tokens: int, *, kv_rows: Optional[int] = None, sequences: int, heads: int, kv_heads: int, dim: int,
                     dtype: str = "bf16", causal: bool = True, scale: Optional[float] = None,
                     lse: bool = False) -> KernelModule:
    """Buffers: q [tokens, heads, dim], k and v [kv_rows or tokens, kv_heads,
    dim], q_offsets [sequences + 1], kv_start and kv_len [sequences] (with
    ``kv_rows``); outputs out like q, lse [tokens, heads] (with ``lse``)."""
    km = KernelModule(name="attention")
    op = {"q": _buffer(km, "q", dtype, [tokens, heads, dim])}
    return _attention(km, op, tokens, kv_rows, sequences, heads, kv_heads, dim, dtype, causal, scale, lse)


def shared_prefix_attention_module(tokens: int, *, prefix_rows: int, kv_rows: Optional[int] = None, sequences: int,
                                   heads: int, kv_heads: int, dim: int, dtype: str = "bf16", causal: bool = True,
                                   scale: Optional[float] = None, lse: bool = False,
                                   prefix_len: bool = False) -> KernelModule:
    """Buffers: q, prefix_k and prefix_v [prefix_rows, kv_heads, dim],
    prefix_len [1] (with ``prefix_len``), then as ``attention_module``."""
    km = KernelModule(name="shared_prefix_attention")
    op = {"q": _buffer(km, "q", dtype, [tokens, heads, dim]),
          "prefix_k": _buffer(km, "prefix_k", dtype, [prefix_rows, kv_heads, dim]),
          "prefix_v": _buffer(km, "prefix_v", dtype, [prefix_rows, kv_heads, dim])}
    if prefix_len:
        op["prefix_len"] = _buffer(km, "prefix_len", "i32", [1])
    return _attention(km, op, tokens, kv_rows, sequences, heads, kv_heads, dim, dtype, causal, scale, lse)


def add_quantize_rows(km: KernelModule, operands: dict, *, cols: int, columns: Optional[dict] = None) -> int:
    """Appends a quantize_rows Call. ``operands`` maps x, codes_out and
    scale_out to buffer ids."""
    attrs = dict(cols=cols)
    attrs.update({f"{k}_at": v for k, v in (columns or {}).items()})
    return _call(km, "quantize_rows", operands, attrs)


def add_matmul_i8(km: KernelModule, operands: dict, *, cols: int, inner: int, columns: Optional[dict] = None) -> int:
    """Appends a matmul_i8 Call. ``operands`` maps a, a_scale, b, b_scale, bias
    and out to buffer ids (bias None or absent: without it)."""
    attrs = dict(cols=cols, inner=inner)
    attrs.update({f"{k}_at": v for k, v in (columns or {}).items()})
    return _call(km, "matmul_i8", operands, attrs)


def add_store_kv4(km: KernelModule, operands: dict, *, kv_heads: int, dim: int, columns: Optional[dict] = None) -> int:
    """Appends a store_kv4 Call. ``operands`` maps k, v, slots, q_offsets,
    k_codes_out, k_scale_out, v_codes_out and v_scale_out to buffer ids (slots
    and q_offsets None or absent: without them)."""
    attrs = dict(kv_heads=kv_heads, dim=dim)
    attrs.update({f"{k}_at": v for k, v in (columns or {}).items()})
    return _call(km, "store_kv4", operands, attrs)


def add_load_kv4(km: KernelModule, operands: dict, *, kv_heads: int, dim: int, columns: Optional[dict] = None) -> int:
    """Appends a load_kv4 Call. ``operands`` maps k_codes, k_scale, v_codes,
    v_scale, slots, q_offsets, k_out and v_out to buffer ids."""
    attrs = dict(kv_heads=kv_heads, dim=dim)
    attrs.update({f"{k}_at": v for k, v in (columns or {}).items()})
    return _call(km, "load_kv4", operands, attrs)


def add_attention_kv4(km: KernelModule, operands: dict, *, heads: int, kv_heads: int, dim: int, causal: bool = True,
                      scale: Optional[float] = None, columns: Optional[dict] = None) -> int:
    """Appends an attention_kv4 Call. ``operands`` maps q, k_codes, k_scale,
    v_codes, v_scale, q_offsets, kv_start, kv_len, out and lse to buffer ids."""
    attrs = dict(heads=heads, kv_heads=kv_heads, dim=dim, causal=int(causal), scale=scale)
    attrs.update({f"{k}_at": v for k, v in (columns or {}).items()})
    return _call(km, "attention_kv4", operands, attrs)


def quantize_rows_module(rows: int, cols: int, *, dtype: str = "bf16") -> KernelModule:
    """Buffers: x [rows, cols]; outputs codes [rows, cols] i8, scale [rows]."""
    km = KernelModule(name="quantize_rows")
    op = {"x": _buffer(km, "x", dtype, [rows, cols])}
    op["codes_out"] = _buffer(km, "codes", "i8", [rows, cols], output=True)
    op["scale_out"] = _buffer(km, "scale", "f32", [rows], output=True)
    add_quantize_rows(km, op, cols=cols)
    return km


def _weights(km: KernelModule, cols: int, inner: int, bias: bool) -> dict:
    op = {"b": _buffer(km, "b", "i8", [cols, inner]), "b_scale": _buffer(km, "b_scale", "f32", [cols])}
    if bias:
        op["bias"] = _buffer(km, "bias", "f32", [cols])
    return op


def matmul_i8_module(rows: int, cols: int, inner: int, *, dtype: str = "bf16", bias: bool = False) -> KernelModule:
    """Buffers: a [rows, inner] i8, a_scale [rows], b [cols, inner] i8, b_scale
    [cols], bias [cols] (with ``bias``); output out [rows, cols]."""
    km = KernelModule(name="matmul_i8")
    op = {"a": _buffer(km, "a", "i8", [rows, inner]), "a_scale": _buffer(km, "a_scale", "f32", [rows])}
    op.update(_weights(km, cols, inner, bias))
    op["out"] = _buffer(km, "out", dtype, [rows, cols], output=True)
    add_matmul_i8(km, op, cols=cols, inner=inner)
    return km


def linear_i8_module(rows: int, cols: int, inner: int, *, dtype: str = "bf16", bias: bool = False) -> KernelModule:
    """quantize_rows, then matmul_i8 of its rows. Buffers: x [rows, inner], b
    [cols, inner] i8, b_scale [cols], bias [cols] (with ``bias``); outputs codes
    [rows, inner] i8, scale [rows], out [rows, cols]."""
    km = KernelModule(name="linear_i8")
    x = _buffer(km, "x", dtype, [rows, inner])
    op = _weights(km, cols, inner, bias)
    op["a"] = _buffer(km, "codes", "i8", [rows, inner], output=True)
    op["a_scale"] = _buffer(km, "scale", "f32", [rows], output=True)
    op["out"] = _buffer(km, "out", dtype, [rows, cols], output=True)
    add_quantize_rows(km, {"x": x, "codes_out": op["a"], "scale_out": op["a_scale"]}, cols=inner)
    add_matmul_i8(km, op, cols=cols, inner=inner)
    return km


def _cache_kv4(km: KernelModule, rows: int, kv_heads: int, dim: int, output: bool) -> dict:
    op = {}
    for part in "kv":
        op[f"{part}_codes"] = _buffer(km, f"{part}_codes", "u8", [rows, kv_heads, dim // 2], output)
        op[f"{part}_scale"] = _buffer(km, f"{part}_scale", "f32", [rows, kv_heads], output)
    return op


def _tokens(km: KernelModule, tokens: int, cache_rows: Optional[int], sequences: Optional[int]) -> dict:
    op = {}
    if cache_rows is not None:
        op["slots"] = _buffer(km, "slots", "i32", [tokens])
    if sequences is not None:
        op["q_offsets"] = _buffer(km, "q_offsets", "i32", [sequences + 1])
    return op


def store_kv4_module(tokens: int, *, kv_heads: int, dim: int, dtype: str = "bf16", cache_rows: Optional[int] = None,
                     sequences: Optional[int] = None) -> KernelModule:
    """Buffers: k and v [tokens, kv_heads, dim], slots [tokens] (with
    ``cache_rows``), q_offsets [sequences + 1] (with ``sequences``); outputs
    k_codes [cache_rows or tokens, kv_heads, dim / 2] u8, k_scale [.., kv_heads],
    v_codes, v_scale."""
    km = KernelModule(name="store_kv4")
    op = {p: _buffer(km, p, dtype, [tokens, kv_heads, dim]) for p in "kv"}
    op.update(_tokens(km, tokens, cache_rows, sequences))
    cache = _cache_kv4(km, tokens if cache_rows is None else cache_rows, kv_heads, dim, True)
    op.update({f"{name}_out": b for name, b in cache.items()})
    add_store_kv4(km, op, kv_heads=kv_heads, dim=dim)
    return km


def load_kv4_module(tokens: int, *, kv_heads: int, dim: int, dtype: str = "bf16", cache_rows: Optional[int] = None,
                    sequences: Optional[int] = None) -> KernelModule:
    """Buffers: k_codes, k_scale, v_codes and v_scale as ``store_kv4_module``
    has them, slots, q_offsets; outputs k and v [tokens, kv_heads, dim]."""
    km = KernelModule(name="load_kv4")
    op = _cache_kv4(km, tokens if cache_rows is None else cache_rows, kv_heads, dim, False)
    op.update(_tokens(km, tokens, cache_rows, sequences))
    op.update({f"{p}_out": _buffer(km, p, dtype, [tokens, kv_heads, dim], output=True) for p in "kv"})
    add_load_kv4(km, op, kv_heads=kv_heads, dim=dim)
    return km


def store_load_kv4_module(tokens: int, *, cache_rows: int, kv_heads: int, dim: int, dtype: str = "bf16",
                          read_dtype: Optional[str] = None) -> KernelModule:
    """store_kv4, then load_kv4 of the same rows. Buffers: k, v, slots; outputs
    k_codes, k_scale, v_codes, v_scale, and k_read and v_read [tokens, kv_heads,
    dim] of ``read_dtype`` (``dtype``)."""
    km = store_kv4_module(tokens, kv_heads=kv_heads, dim=dim, dtype=dtype, cache_rows=cache_rows)
    km.name = "store_load_kv4"
    stored = km.nodes[-1].operands
    op = {name[:-4]: b for name, b in stored.items() if name.endswith("_out")}
    op["slots"] = stored["slots"]
    op.update({f"{p}_out": _buffer(km, f"{p}_read", read_dtype or dtype, [tokens, kv_heads, dim], output=True) for p in "kv"})
    add_load_kv4(km, op, kv_heads=kv_heads, dim=dim)
    return km


def attention_kv4_module(tokens: int, *, kv_rows: Optional[int] = None, sequences: int, heads: int, kv_heads: int, dim: int,
                         dtype: str = "bf16", causal: bool = True, scale: Optional[float] = None,
                         lse: bool = False) -> KernelModule:
    """Buffers: q [tokens, heads, dim], k_codes [kv_rows or tokens, kv_heads, dim
    / 2] u8, k_scale [.., kv_heads], v_codes, v_scale, q_offsets [sequences + 1],
    kv_start and kv_len [sequences] (with ``kv_rows``); outputs out like q, lse
    [tokens, heads] (with ``lse``)."""
    km = KernelModule(name="attention_kv4")
    op = {"q": _buffer(km, "q", dtype, [tokens, heads, dim])}
    op.update(_cache_kv4(km, tokens if kv_rows is None else kv_rows, kv_heads, dim, False))
    op["q_offsets"] = _buffer(km, "q_offsets", "i32", [sequences + 1])
    if kv_rows is not None:
        op["kv_start"] = _buffer(km, "kv_start", "i32", [sequences])
        op["kv_len"] = _buffer(km, "kv_len", "i32", [sequences])
    op["out"] = _buffer(km, "out", dtype, [tokens, heads, dim], output=True)
    if lse:
        op["lse"] = _buffer(km, "lse", "f32", [tokens, heads], output=True)
    add_attention_kv4(km, op, heads=heads, kv_heads=kv_heads, dim=dim, causal=causal, scale=scale)
    return km
