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

Types: f16, bf16 or f32, the same for all rows; sums are held in f32 and each
output is rounded once. Attention's weights are rounded to the type of v before
they meet it, so that f16 and bf16 run on the matrix cores; their sum is of the
f32 values. Buffers' sizes decide how an attention runs, not the lengths in them,
and rows off 16 bytes or more than 4096 sequences run a wave to a row (see
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
