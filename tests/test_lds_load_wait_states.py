"""A load from memory straight into LDS takes its place there from M0.  Where a scalar instruction writes M0, one wait state has to
lie in front of such a load; the compiler leaves it for loads that it issues itself and does not look into inline assembly.  Runs on
the disassembly of the libraries' own gfx950 code objects; no GPU."""
import os
import re
from concurrent.futures import ThreadPoolExecutor

import pytest

import test_mfma_wait_states as scan
from cldnn_amd import hip, ops

WRITES_M0 = re.compile(r"m0\b")


def into_lds(op, operands):
    return op.startswith(("buffer_load", "global_load")) and ("lds" in operands.split() or "_lds_" in op)


def too_near(ins):
    """the loads into LDS directly behind a write of M0.  What lies between the two on any path is an instruction, and each is a wait
    state at least: a branch too, so the order of addresses is all that there is to look at."""
    return [(ins[i - 1][:2], ins[i][:2]) for i in range(1, len(ins))
            if into_lds(*ins[i][:2]) and ins[i - 1][0].startswith("s_") and WRITES_M0.match(ins[i - 1][1])]


def test_pairs_are_found():
    """the scan itself"""
    write, load = ("s_mov_b32", "m0, s4", 0), ("buffer_load_dwordx4", "v1, s[0:3], s5 offen lds", 4)
    assert too_near([write, load]) and too_near([("s_add_i32", "m0, s4, s5", 0), load])
    assert too_near([write, ("global_load_lds_dwordx4", "v[0:1], off", 4)])
    assert not too_near([write, ("s_nop", "0", 4), load]) and not too_near([("s_mov_b32", "s4, m0", 0), load])
    assert not too_near([write, ("buffer_load_dwordx4", "v[0:3], v1, s[0:3], 0 offen", 4)])


@pytest.mark.skipif(not os.path.exists(scan.OBJDUMP), reason="needs the ROCm disassembler")
@pytest.mark.parametrize("library", [hip.LIB_PATH, ops.LIB_PATH], ids=os.path.basename)
def test_a_wait_state_behind_m0(tmp_path, monkeypatch, library):
    monkeypatch.setattr(hip, "LIB_PATH", library)
    paths, loads = [], 0
    for n, elf in enumerate(scan.code_objects()):
        paths.append(str(tmp_path / ("%d.elf" % n)))
        with open(paths[-1], "wb") as f:
            f.write(elf)
    with ThreadPoolExecutor(4) as pool:
        for found in pool.map(scan.kernels, paths):
            for name, ins in found.items():
                loads += sum(into_lds(*i[:2]) for i in ins)
                bad = too_near(ins)
                assert not bad, "%s: %d, the first %s" % (name, len(bad), bad[0])
    assert loads > 100  # the libraries' loads were found
