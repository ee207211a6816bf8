"""The operators around attention, as timed cases: head norms with the position
rotation, attention over packed sequences, attention behind a shared prefix.

A case is a dict: "kind", its sizes, its types and its lengths, all plain
values. `listed` holds the named ones, `draw` gives others of the same ranges.
`run` computes a case in plain torch operations; with `own` it runs the
framework's operator through mlkhip_build and mlkhip_run_device, on artifacts
and binding arrays that are made once and kept, as a serving loop keeps them.

The three kinds, for T tokens of H query heads and G key/value heads of dim D:

norm_rope  rows of a fused projection [T, (H + 2 G) D]: each head of q and k is
           divided by its root mean square, weighted and rotated by its token's
           position; k and v go to their tokens' rows of a cache.
attention  softmax(scale q k^T) v, each query over its own sequence's keys in a
           cache (causal: its last key is its own position), grouped heads.
prefix     the same where every sequence's keys continue one shared prefix.
"""
from __future__ import annotations

import ctypes
import itertools
import math

import torch

own = False

TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6


def listed():
    return [
        # One decode step of 64 requests: a launch and little else.
        dict(name="norm_rope_64", kind="norm_rope", tokens=64, heads=32, kv_heads=8, dim=128, dtype="bf16", cache=16384,
             rot=128, interleaved=False, axes=1, theta=1e6, first=100000),
        # A whole prompt of ordinary length.
        dict(name="norm_rope_8192", kind="norm_rope", tokens=8192, heads=32, kv_heads=8, dim=128, dtype="bf16", cache=9000,
             rot=128, interleaved=False, axes=1, theta=1e6, first=0),
        # Patches of a video: three axes, an odd count, smaller heads.
        dict(name="norm_rope_video_4099", kind="norm_rope", tokens=4099, heads=16, kv_heads=16, dim=64, dtype="f16",
             cache=4099, rot=64, interleaved=False, axes=3, theta=1e4, first=0),
        # Single precision, a part of each head rotated, neighbours paired.
        dict(name="norm_rope_f32_777", kind="norm_rope", tokens=777, heads=12, kv_heads=4, dim=96, dtype="f32", cache=1000,
             rot=48, interleaved=True, axes=1, theta=1e4, first=5000),
        # A chat turn of a few words: latency.
        dict(name="attention_1x19", kind="attention", sequences=1, queries=19, keys=19, even=True, heads=32, kv_heads=8,
             dim=128, dtype="bf16", causal=True, spare=0),
        # One prompt of ordinary length.
        dict(name="attention_1x2048", kind="attention", sequences=1, queries=2048, keys=2048, even=True, heads=32, kv_heads=8,
             dim=128, dtype="bf16", causal=True, spare=0),
        # Prompts of different lengths packed into one batch, the buffer not full.
        dict(name="attention_packed_8x4096", kind="attention", sequences=8, queries=4096, keys=4096, even=False, heads=32,
             kv_heads=8, dim=128, dtype="bf16", causal=True, spare=100),
        # An encoder's sequences: every key seen, a head for each query head.
        dict(name="attention_f16_16x1024", kind="attention", sequences=16, queries=1024, keys=1024, even=False, heads=16,
             kv_heads=16, dim=64, dtype="f16", causal=False, spare=0),
        # One decode step of 32 requests over caches of different lengths.
        dict(name="attention_decode_32x8192", kind="attention", sequences=32, queries=1, keys=8192, even=False, heads=32,
             kv_heads=8, dim=128, dtype="bf16", causal=True, spare=0),
        # Single precision, an odd length.
        dict(name="attention_f32_2x1001", kind="attention", sequences=2, queries=1001, keys=1001, even=False, heads=8,
             kv_heads=8, dim=64, dtype="f32", causal=True, spare=0),
        # 64 requests decode behind one long system prompt.
        dict(name="prefix_decode_64x8192", kind="prefix", sequences=64, prefix=8192, queries=1, keys=256, even=False, heads=32,
             kv_heads=8, dim=128, dtype="bf16", causal=True, spare=0),
        # Short questions about one document, in one batch.
        dict(name="prefix_16x128_2000", kind="prefix", sequences=16, prefix=2000, queries=128, keys=128, even=False, heads=16,
             kv_heads=4, dim=128, dtype="f16", causal=True, spare=3),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm_rope", "attention", "attention", "prefix"])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    if kind == "norm_rope":
        tokens = _log(rng, 1, 8192)
        axes = rng.choice([1, 1, 3])
        return dict(kind=kind, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["bf16", "f16", "f32"]),
                    cache=tokens + rng.randint(0, 500), rot=dim if axes == 3 else rng.choice([dim, dim, dim // 2]),
                    interleaved=rng.random() < 0.3, axes=axes, theta=rng.choice([1e4, 1e6]),
                    first=0 if axes == 3 else rng.choice([0, 1000, 100000]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    even, spare = rng.random() < 0.3, rng.choice([0, 0, 1, 50])
    while True:
        sequences = _log(rng, 1, 64)
        form = rng.choice(["prompt", "continued", "decode"])
        if form == "decode":
            queries, keys = rng.choice([1, 1, 1, 2, 4]), _log(rng, 16, 8192 if kind == "attention" else 512)
        else:
            queries = _log(rng, 4, 2048)
            keys = queries + (_log(rng, 16, 4096) if form == "continued" else 0)
        prefix = _log(rng, 64, 8192)
        pairs = sequences * queries * (keys + (prefix if kind == "prefix" else 0)) * heads * dim
        limit = (1 << 36) if dtype != "f32" else (1 << 33)
        if pairs <= limit and sequences * keys * kv_heads * dim <= 1 << 27:
            break
    case = dict(kind=kind, sequences=sequences, queries=queries, keys=keys, even=even, heads=heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype, causal=kind == "prefix" or rng.random() < 0.7, spare=spare)
    if kind == "prefix":
        case["prefix"] = prefix
    return case


def _lengths(c):
    """(queries, keys) of each sequence: all the largest, or spread from about
    an eighth of that up to it, keys at least the queries."""
    n, q, k = c["sequences"], c["queries"], c["keys"]
    if c["even"]:
        return [q] * n, [k] * n
    part = [1.0 - 0.875 * ((0.6180339887 * i) % 1.0) for i in range(n)]
    qs = [max(1, round(q * p)) for p in part]
    return qs, [max(a, round(k * p)) for a, p in zip(qs, part)]


def _sections(c):
    """Frequency pairs of each axis."""
    pairs = c["rot"] // 2
    if c["axes"] == 1:
        return [pairs]
    side = 3 * pairs // 8
    return [pairs - 2 * side, side, side]


class _State:
    pass


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, s = case, _State()
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)

    def normal(shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std + mean).to(TORCH[c["dtype"]])

    s.case, s.bound = c, None
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "norm_rope":
        t = c["tokens"]
        s.qkv = normal((t, (heads + 2 * kv) * dim))
        s.q_weight, s.k_weight = normal((dim,), 0.1, 1.0), normal((dim,), 0.1, 1.0)
        if c["axes"] == 1:
            s.positions = (torch.arange(t, device="cuda", dtype=torch.int32) + c["first"]).reshape(1, t)
        else:  # frames of 16 x 16 patches
            i = torch.arange(t, device="cuda", dtype=torch.int32)
            s.positions = torch.stack([i // 256, i // 16 % 16, i % 16]).contiguous()
        s.slots = torch.randperm(c["cache"], generator=g, device="cuda")[:t].to(torch.int32)
        s.q_out = torch.zeros((t, heads, dim), device="cuda", dtype=TORCH[c["dtype"]])
        s.k_cache, s.v_cache = normal((c["cache"], kv, dim)), normal((c["cache"], kv, dim))
        return s
    s.q_lens, s.k_lens = _lengths(c)
    t, rows = sum(s.q_lens) + c["spare"], sum(s.k_lens)
    s.q, s.k, s.v = normal((t, heads, dim)), normal((rows, kv, dim)), normal((rows, kv, dim))
    if c["kind"] == "prefix":
        s.prefix_k, s.prefix_v = normal((c["prefix"], kv, dim)), normal((c["prefix"], kv, dim))
    s.q_offsets = _ints([0] + list(itertools.accumulate(s.q_lens)))
    s.kv_start, s.kv_len = _ints([0] + list(itertools.accumulate(s.k_lens[:-1]))), _ints(s.k_lens)
    s.out = torch.zeros_like(s.q)
    s.lse = torch.zeros((t, heads), device="cuda", dtype=torch.float32)
    return s


# ------------------------------------------------- the framework's operators --
_artifacts = {}


def _artifact(c):
    """The artifact of a case's module, built once."""
    key = tuple(sorted((k, v) for k, v in c.items() if k != "name"))
    if key not in _artifacts:
        from mlk2_amd import operators as op
        from mlk2_amd.backend import last_error, lib
        heads = dict(heads=c["heads"], kv_heads=c["kv_heads"], dim=c["dim"], dtype=c["dtype"])
        if c["kind"] == "norm_rope":
            km = op.qk_norm_rope_module(c["tokens"], cache_rows=c["cache"], eps=EPS, theta=c["theta"], rot=c["rot"],
                                        interleaved=c["interleaved"], sections=_sections(c), **heads)
        else:
            qs, ks = _lengths(c)
            sizes = dict(tokens=sum(qs) + c["spare"], kv_rows=sum(ks), sequences=c["sequences"], causal=c["causal"], lse=True)
            if c["kind"] == "attention":
                km = op.attention_module(**sizes, **heads)
            else:
                km = op.shared_prefix_attention_module(prefix_rows=c["prefix"], **sizes, **heads)
        doc, handle = km.to_json().encode(), ctypes.c_void_p()
        if lib().mlkhip_build(doc, len(doc), b"gfx950", b"", ctypes.byref(handle)) != 0:
            raise RuntimeError(last_error())
        _artifacts[key] = handle
    return _artifacts[key]


def _bind(s):
    """A state's arguments of mlkhip_run_device."""
    from mlk2_amd.backend import DTYPE_CODE, Binding
    codes = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32", torch.int32: "i32"}
    if s.case["kind"] == "norm_rope":
        bufs = [s.qkv, s.q_weight, s.k_weight, s.positions, s.slots, s.q_out, s.k_cache, s.v_cache]
    else:
        prefix = [s.prefix_k, s.prefix_v] if s.case["kind"] == "prefix" else []
        bufs = [s.q] + prefix + [s.k, s.v, s.q_offsets, s.kv_start, s.kv_len, s.out, s.lse]
    binds = (Binding * len(bufs))(*[Binding(b.data_ptr(), b.numel(), DTYPE_CODE[codes[b.dtype]], 0) for b in bufs])
    s.bound = (_artifact(s.case), binds, len(bufs), (ctypes.c_double * 1)(0.0), 0, 0, None)


def _run_own(s):
    from mlk2_amd.backend import last_error, lib
    if s.bound is None:
        _bind(s)
    if lib().mlkhip_run_device(*s.bound) != 0:
        raise RuntimeError(last_error())


# --------------------------------------------------------------- plain forms --
def _norm_rope(s):
    c = s.case
    heads, kv, dim, rot = c["heads"], c["kv_heads"], c["dim"], c["rot"]
    x = s.qkv.float().reshape(-1, heads + 2 * kv, dim)
    qk, v = x[:, : heads + kv], x[:, heads + kv:]
    w = torch.cat([s.q_weight.float().expand(heads, dim), s.k_weight.float().expand(kv, dim)])
    y = qk * torch.rsqrt((qk * qk).mean(dim=-1, keepdim=True) + EPS) * w
    pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    axis = torch.repeat_interleave(torch.arange(c["axes"], device="cuda"), torch.tensor(_sections(c), device="cuda"))
    angle = s.positions.double()[axis].t() * c["theta"] ** (-2.0 * pair / rot)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if c["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    y = torch.cat([turned, y[..., rot:]], dim=-1).to(s.q_out.dtype)
    at = s.slots.long()
    s.q_out.copy_(y[:, :heads])
    s.k_cache[at] = y[:, heads:]
    s.v_cache[at] = v.to(s.v_cache.dtype)


def _padded(rows, starts, lens, longest):
    """Rows of each sequence, padded to the longest, and where they are real."""
    j = torch.arange(longest, device="cuda")
    real = j[None] < lens[:, None]
    return rows[torch.where(real, starts[:, None] + j[None], 0)].float(), real


def _attention(s):
    c = s.case
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    n, group, lq, lk = c["sequences"], heads // kv, max(s.q_lens), max(s.k_lens)
    q_start, q_len = s.q_offsets[:-1].long(), (s.q_offsets[1:] - s.q_offsets[:-1]).long()
    k_len = s.kv_len.long()
    q, real_q = _padded(s.q, q_start, q_len, lq)
    k, real_k = _padded(s.k, s.kv_start.long(), k_len, lk)
    v, _ = _padded(s.v, s.kv_start.long(), k_len, lk)
    seen = real_k[:, None, :].expand(n, lq, lk)
    if c["causal"]:
        i, j = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
        seen = seen & (j[None, None] <= i[None, :, None] + (k_len - q_len)[:, None, None])
    if c["kind"] == "prefix":
        p = c["prefix"]
        k = torch.cat([s.prefix_k.float().expand(n, p, kv, dim), k], dim=1)
        v = torch.cat([s.prefix_v.float().expand(n, p, kv, dim), v], dim=1)
        seen = torch.cat([torch.ones((n, lq, p), dtype=torch.bool, device="cuda"), seen], dim=2)
        lk += p
    q = q.reshape(n, lq, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n * kv, group * lq, dim)
    k = k.permute(0, 2, 3, 1).reshape(n * kv, dim, lk)
    v = v.permute(0, 2, 1, 3).reshape(n * kv, lk, dim)
    scores = (torch.bmm(q, k) / math.sqrt(dim)).reshape(n, kv, group, lq, lk)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores.sub_(top.clamp_min(torch.finfo(torch.float32).min)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.bmm(scores.reshape(n * kv, group * lq, lk), v).reshape(n, kv, group, lq, dim)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n, lq, heads, dim)
    lse = (top + torch.log(total)).permute(0, 3, 1, 2, 4).reshape(n, lq, heads)
    at = (q_start[:, None] + torch.arange(lq, device="cuda")[None])[real_q]
    s.out[at] = out[real_q].to(s.out.dtype)
    s.lse[at] = lse[real_q]


def run(state):
    if own:
        _run_own(state)
    elif state.case["kind"] == "norm_rope":
        _norm_rope(state)
    else:
        _attention(state)
    if state.case["kind"] == "norm_rope":
        return {"q": state.q_out, "k": state.k_cache, "v": state.v_cache}
    return {"out": state.out, "lse": state.lse}


def work(case):
    c = case
    heads, kv, dim, size = c["heads"], c["kv_heads"], c["dim"], BYTES[c["dtype"]]
    if c["kind"] == "norm_rope":
        t = c["tokens"]
        values = t * (heads + 2 * kv) * dim
        return {"bytes": 2 * values * size + 4 * t * (c["axes"] + 1) + 2 * dim * size, "flops": 10 * t * (heads + kv) * dim}
    qs, ks = _lengths(c)
    p = c.get("prefix", 0)
    pairs = sum(q * k - (q * (q - 1) // 2 if c["causal"] else 0) + q * p for q, k in zip(qs, ks))
    return {"bytes": (2 * sum(qs) * heads + 2 * (sum(ks) + p) * kv) * dim * size + 4 * sum(qs) * heads + 12 * len(qs),
            "flops": 4 * pairs * heads * dim}


# --------------------------------------------------------------- in 64 bits --
def _exact_norm_rope(s):
    c = s.case
    heads, kv, dim, half = c["heads"], c["kv_heads"], c["dim"], c["rot"] // 2
    x = s.qkv.double().reshape(c["tokens"], heads + 2 * kv, dim)
    found = []
    for part, weight in ((x[:, :heads], s.q_weight), (x[:, heads:heads + kv], s.k_weight)):
        y = part / torch.sqrt(part.pow(2).sum(-1, keepdim=True) / dim + EPS) * weight.double()
        z = y.clone()
        pair = 0
        for axis, count in enumerate(_sections(c)):
            for _ in range(count):
                angle = s.positions[axis].double() / c["theta"] ** (2.0 * pair / c["rot"])
                turn = torch.polar(torch.ones_like(angle), angle)[:, None]
                a, b = (2 * pair, 2 * pair + 1) if c["interleaved"] else (pair, pair + half)
                w = torch.complex(y[..., a], y[..., b]) * turn
                z[..., a], z[..., b] = w.real, w.imag
                pair += 1
        found.append(z)
    k, v = s.k_cache.double(), s.v_cache.double()
    k[s.slots.long()], v[s.slots.long()] = found[1], x[:, heads + kv:]
    return {"q": found[0], "k": k, "v": v}


def _exact_attention(s):
    c = s.case
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    group = heads // kv
    out, lse = torch.zeros(s.out.shape, device="cuda", dtype=torch.float64), s.lse.double()
    q0 = k0 = 0
    for nq, nk in zip(s.q_lens, s.k_lens):
        for h in range(kv):
            k, v = s.k[k0:k0 + nk, h].double(), s.v[k0:k0 + nk, h].double()
            if c["kind"] == "prefix":
                k, v = torch.cat([s.prefix_k[:, h].double(), k]), torch.cat([s.prefix_v[:, h].double(), v])
            q = s.q[q0:q0 + nq, h * group:(h + 1) * group].double().reshape(nq * group, dim)
            w = torch.mm(q, k.t().contiguous()) * dim ** -0.5
            if c["causal"]:
                last = torch.arange(nq, device="cuda").repeat_interleave(group) + len(k) - nq
                w[torch.arange(len(k), device="cuda")[None] > last[:, None]] = -math.inf
            sums = torch.logsumexp(w, dim=1)
            out[q0:q0 + nq, h * group:(h + 1) * group] = torch.mm(torch.exp(w - sums[:, None]), v).reshape(nq, group, dim)
            lse[q0:q0 + nq, h * group:(h + 1) * group] = sums.reshape(nq, group)
        q0, k0 = q0 + nq, k0 + nk
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm_rope(s) if case["kind"] == "norm_rope" else _exact_attention(s)
