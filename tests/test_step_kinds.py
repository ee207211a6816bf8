"""Every place that goes by a step's kind names all kinds, so that the compiler
stops a kind added later where it is not handled (no device needed)."""
import os
import shutil
import subprocess

import pytest

from mlk2_amd import build as mb


@pytest.mark.parametrize("added", [False, True])
@pytest.mark.parametrize("source,switches", [("planner.cpp", 3), ("operators.cpp", 1)])
def test_a_new_kind_is_handled_everywhere(tmp_path, source, switches, added):
    csrc = shutil.copytree(mb.CSRC, tmp_path / "csrc")
    header = csrc / "host" / "planner.h"
    text = header.read_text()
    last = "StoreKv4, LoadKv4, AttentionKv4\n"
    assert text.count(last) == 1
    if added:
        header.write_text(text.replace(last, last.rstrip() + ", Later\n"))
    r = subprocess.run([mb.CLANG] + mb.HOST_FLAGS + ["-I", os.path.join(mb.BUILD, "gen"), "-fsyntax-only", str(csrc / "host" / source)],
                       stderr=subprocess.PIPE, text=True)
    assert r.stderr.count("'Later' not handled in switch") == (switches if added else 0), r.stderr
    assert (r.returncode != 0) == added
