"""Plain f64 references of the operators in 8 and 4 bits.

Codes and scales are exact: a scale is an f32 quotient rounded once, a code the
whole number (the 4-bit number) nearest to a quotient of two f32 values, which
64 bits hold apart from every border: x / s and a border of 8 bits differ by
2^-33 of themselves or not at all.
"""
import numpy as np

from operators_ref import TINY, U, U32

NUMBERS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
BORDERS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])


def _scale(x, largest):
    """f32 scales of the last axis, NaN where a value is not finite."""
    with np.errstate(invalid="ignore", over="ignore"):
        s = (np.abs(x).max(-1) / largest).astype(np.float32)
    return np.where(np.isfinite(x).all(-1), s, np.float32(np.nan)).astype(np.float64)


def quantize_rows(x):
    """(codes, scale) of rows x."""
    s = _scale(x, 127.0)
    good = (s > 0)[..., None]
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.clip(np.rint(x / s[..., None]), -127, 127)
    return np.where(good, q, 0.0), s


def store_kv4(x):
    """(packed codes, scale) of heads x [..., dim]."""
    s = _scale(x, 6.0)
    with np.errstate(invalid="ignore", divide="ignore"):
        y = np.abs(x) / s[..., None]
    code = np.zeros(x.shape, dtype=np.int64)
    for i, border in enumerate(BORDERS):
        code += (y >= border) if i % 2 else (y > border)
    code = np.where((s > 0)[..., None], code, 0) | np.signbit(x).astype(np.int64) << 3
    code = np.where(np.isnan(s)[..., None], 0, code)
    return code[..., 0::2] | code[..., 1::2] << 4, s


def load_kv4(codes, scale):
    """The numbers of packed codes."""
    codes = np.asarray(codes).astype(np.int64)
    four = np.stack([codes & 15, codes >> 4], axis=-1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    return np.where(four >= 8, -1.0, 1.0) * NUMBERS[four & 7] * np.asarray(scale, dtype=np.float64)[..., None]


def load_bound(x, dtype):
    """A number times its scale in f32, then one rounding to the type."""
    return (U32 + U[dtype] * (1 + U32)) * np.abs(x) + TINY[dtype]


def matmul_i8(a, a_scale, b, b_scale, bias, dtype):
    """(out, bound): the sum is exact; turned to f32 and taken times two scales
    it is off by half a step three times, the bias's sum once more, and it is
    rounded to the type once. Products below f32's steps are off by half of one."""
    total = (a.astype(np.float64) @ b.astype(np.float64).T)
    y = total * a_scale[:, None] * b_scale[None, :]
    out = y if bias is None else y + bias[None, :]
    slack = 3 * U32 * np.abs(y) * (1 + 3 * U32) + TINY["f32"] * (2 + np.abs(b_scale[None, :])) + (0 if bias is None else U32 * (np.abs(out) + 4 * U32 * np.abs(y)))
    return out, slack * (1 + U[dtype]) + U[dtype] * np.abs(out) + TINY[dtype]
