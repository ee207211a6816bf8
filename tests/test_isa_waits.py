"""Wait states that gfx9-family hardware leaves to software, checked in the
built library's device code. The compiler keeps them between its own
instructions, but puts none inside inline assembly or for its sake:

- a scalar write of M0, then a load to LDS that takes its place from M0: one;
- a vector write of a scalar register, then a memory access that reads it: five.
"""
import os

import pytest

import isa
from mlk2_amd.backend import LIB_PATH

CODE = list(isa.code_objects(LIB_PATH)) if os.path.exists(LIB_PATH) else []


@pytest.mark.parametrize("n", range(len(CODE)))
def test_waits(n):
    ins, before = isa.disassembled(CODE[n])
    assert ins
    missing = []
    for i, (kernel, op, args) in enumerate(ins):
        if not op.startswith(("global_", "buffer_", "flat_", "scratch_")):
            continue
        if "_lds_" in op:
            if any(w.op.startswith("s_") and "m0" in isa.scalars(w.args.split(",")[0]) for w in isa.writers(ins, before, i, 1)):
                missing.append((kernel, op, "m0"))
        reads = isa.scalars(args)
        if reads and any(w.op.startswith("v_") and reads & isa.scalars(",".join(w.args.split(",")[:2 if "_co_" in w.op else 1]))
                         for w in isa.writers(ins, before, i, 5)):
            missing.append((kernel, op, args))
    assert not missing, (len(missing), missing[:5])


def test_direct_loads_are_there():
    # What the first rule is about: the library is built and does load to LDS.
    assert sum("_lds_" in i.op for code in CODE for i in isa.disassembled(code)[0]) > 100
