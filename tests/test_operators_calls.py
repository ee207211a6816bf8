"""Operator Calls on the CPU: documents that no builder writes."""
import pytest

from mlk2_amd import backend as be
from test_operators import attention


@pytest.mark.parametrize("buffer", [-1, 2 ** 32, 2 ** 32 + 1, -(2 ** 32), 2 ** 32 - 1, 2 ** 63 - 1])
@pytest.mark.parametrize("operand", ["q", "k", "lse"])
def test_ids_past_32_bits_name_no_buffer(operand, buffer):
    # Cut to 32 bits they would be buffers 0 and 1.
    km = attention()
    km.nodes[-1].operands[operand] = buffer
    with pytest.raises(be.MlkHipError) as e:
        be.plan(km)
    assert e.value.code == be.REFUSED and f"'{operand}' names no buffer" in e.value.message


@pytest.mark.parametrize("dims", [[0, 1 << 62, 1 << 62], [0, 1 << 45], [1 << 40, 0, 1 << 40], [0, 1 << 32, 1 << 32]])
@pytest.mark.parametrize("operand", ["k", "v", "out", "q_offsets"])
def test_rows_too_wide_of_buffers_without_elements(operand, dims):
    # A dim of 0 hides nothing: the width of a row has to fit 64 bits.
    km = attention()
    km.buffers[km.nodes[-1].operands[operand]].dims = dims
    with pytest.raises(be.MlkHipError) as e:
        be.plan(km)
    assert e.value.code == be.REFUSED and f"'{operand}' is too large" in e.value.message
