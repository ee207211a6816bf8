"""mlkd_attention of csrc/device_abi.h: the launch itself, and its workspace."""
import ctypes

from mlk2_amd.backend import DTYPE_CODE, lib


class Attention(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "prefix_k", "prefix_v", "out", "lse", "q_offsets", "kv_start", "kv_len",
                                                "prefix_len")] +
                [(n, ctypes.c_int32) for n in ("dtype", "causal", "heads", "kv_heads", "dim", "sequences")] +
                [(n, ctypes.c_int64) for n in ("q_rows", "kv_rows", "prefix_rows", "q_stride", "k_stride", "v_stride", "prefix_k_stride",
                                               "prefix_v_stride", "out_stride")] +
                [("scale", ctypes.c_double), ("work", ctypes.c_void_p), ("work_bytes", ctypes.c_int64)])

    @classmethod
    def of(cls, *, heads, kv_heads, dim, sequences, q_rows, kv_rows, prefix_rows=None, dtype="bf16", causal=True):
        """Whole buffers of these sizes, at addresses that a plan may look at."""
        p = cls(dtype=DTYPE_CODE[dtype], causal=int(causal), heads=heads, kv_heads=kv_heads, dim=dim, sequences=sequences, q_rows=q_rows,
                kv_rows=kv_rows, prefix_rows=prefix_rows or 0, scale=dim ** -0.5)
        for name in ("q", "k", "v", "out", "q_offsets", "kv_start", "kv_len") + (("prefix_k", "prefix_v") if prefix_rows is not None else ()):
            setattr(p, name, 1 << 20)
        p.q_stride = p.out_stride = heads * dim
        p.k_stride = p.v_stride = p.prefix_k_stride = p.prefix_v_stride = kv_heads * dim
        return p

    def work_needed(self):
        f = lib().mlkd_attention_work_bytes
        f.restype = ctypes.c_int64
        return f(ctypes.byref(self))

    def ranges(self):
        """Key ranges with partial results (0: none)."""
        return self.work_needed() // (self.q_rows * self.heads * (self.dim * 4 + 8))

    def launch(self):
        assert lib().mlkd_launch_attention(ctypes.byref(self), None) == 0
        assert lib().mlkhip_synchronize() == 0
