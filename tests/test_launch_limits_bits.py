"""Products in 8-bit integers too large for one grid of some tiles: HIP launches
fewer than 2^32 threads, and the form that is chosen stays below (no device needed)."""
import ctypes

import pytest

from mlk2_amd.backend import DTYPE_CODE, lib

# Rows and columns of a tile, and its threads, by the kernel's parameters.
TILES = {"4, 2, 4, 8": (256, 256, 512), "2, 2, 4, 4": (128, 128, 256), "2, 2, 4, 2": (128, 64, 256), "2, 2, 2, 2": (64, 64, 256)}


class MatmulI8(ctypes.Structure):
    """mlkd_matmul_i8 of csrc/device_abi.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("a", "b", "a_scale", "b_scale", "bias", "out")] +
                [(n, ctypes.c_int32) for n in ("dtype", "pad")] + [(n, ctypes.c_int64) for n in ("m", "n", "k", "lda", "ldb", "ldo")] +
                [("work", ctypes.c_void_p), ("work_bytes", ctypes.c_int64)])

    @classmethod
    def of(cls, m, n, k, dtype="bf16", room=True):
        """Whole buffers at addresses that a plan may look at."""
        p = cls(*(i << 20 for i in range(1, 7)), DTYPE_CODE[dtype], 0, m, n, k, k, k, n)
        p.bias = None
        f = lib().mlkd_matmul_i8_work_bytes
        f.restype = ctypes.c_int64
        if room and f(ctypes.byref(p)) > 0:
            p.work, p.work_bytes = 7 << 20, f(ctypes.byref(p))
        return p

    def names(self):
        f = lib().mlkd_matmul_i8_kernel_names
        f.restype = ctypes.c_char_p
        return f(ctypes.byref(self)).decode()


# Rows and cols are 2^30 at most.
@pytest.mark.parametrize("m,n", [(64, 1 << 30), (33, (1 << 30) - 63), (33, (1 << 30) - 64), (40, 1 << 29), (1 << 30, 64), (1 << 30, 1), (1 << 30, 200),
                                 (100, 1 << 30), (1 << 30, 257), (1 << 29, 512), (1 << 30, 1 << 30), (1 << 20, 1 << 20), (70000, 70000)])
@pytest.mark.parametrize("k", [16, 100, 4096])
@pytest.mark.parametrize("room", [True, False])
def test_products_past_one_grid(m, n, k, room):
    names = MatmulI8.of(m, n, k, room=room).names().split("+")
    tiles = [x for x in names if x.startswith("matmulI8Tiles")]
    if not tiles:
        assert names[0].startswith("matmulI8Few") and len(names) == 1   # a grid of its own, at most 2^20 by 2^15
        return
    rows, cols, threads = TILES[tiles[0].split("<__bf16, ")[1].rsplit(",", 1)[0]]
    assert -(-m // rows) * -(-n // cols) * threads < 1 << 32
