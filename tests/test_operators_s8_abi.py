"""CPU-side checks of the int8 operators' library: it exports what include/cldnn_hip_ops_s8.h declares, the binding has the header's
structures, entry points refuse null handles, matrix results get their wait states, loads into LDS theirs, and no kernel of rows that
fit its registers spills."""
import ctypes as C
import os
import re
import subprocess

import pytest

import test_kernel_registers as registers
import test_lds_load_wait_states as lds
import test_mfma_wait_states as waits
from cldnn_amd import hip, ops, ops_s8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "cldnn_hip_ops_s8.h")
DESCRIPTIONS = {"quantize": ops_s8.QuantizeDesc, "matmul_s8": ops_s8.MatmulS8Desc, "block_norm": ops_s8.BlockNormDesc}
needs_tools = pytest.mark.skipif(not os.path.exists(waits.OBJDUMP), reason="needs the ROCm disassembler")


def test_binding_covers_the_header():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(cldnn_hip_[a-z0-9_]+)\s*\(", text))
    assert set(ops_s8.SIGNATURES) == declared and len(declared) == 6
    L = C.CDLL(ops_s8.LIB_PATH)
    for n in declared:
        assert hasattr(L, n), "missing export: " + n
        arguments = re.search(r"\b%s\s*\(([^)]*)\)" % n, text).group(1).count(",") + 1
        assert len(ops_s8.SIGNATURES[n][1]) == arguments, n


def test_structures_and_values_match_the_header(tmp_path):
    names = {"cldnn_hip_%s_desc" % k: s for k, s in DESCRIPTIONS.items()}
    values = {"CLDNN_HIP_SCALES_NONE": ops_s8.SCALES_NAME[None], "CLDNN_HIP_SCALES_ONE": ops_s8.SCALES_NAME["one"], "CLDNN_HIP_SCALES_EACH": ops_s8.SCALES_NAME["each"],
              "CLDNN_HIP_TOKEN_NORM_NONE": ops_s8.NORM_NAME["none"], "CLDNN_HIP_TOKEN_NORM_LAYER": ops_s8.NORM_NAME["layer"], "CLDNN_HIP_TOKEN_NORM_RMS": ops_s8.NORM_NAME["rms"],
              "CLDNN_HIP_S8": ops.DT_NAME["s8"]}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "cldnn_hip_ops_s8.h"', "int main(void) {"]
    for n, s in names.items():
        lines += ['printf("%%zu ", sizeof(%s));' % n] + ['printf("%%zu ", offsetof(%s, %s));' % (n, f[0]) for f in s._fields_]
    lines += ['printf("%%d ", (int)%s);' % v for v in values]
    src = tmp_path / "offsets.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "offsets")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "offsets")], stdout=subprocess.PIPE, check=True, text=True).stdout.split()]
    want = []
    for s in names.values():
        want += [C.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want + list(values.values())


def test_null_handles_are_refused():
    L = ops_s8.lib()
    for kind, desc in DESCRIPTIONS.items():
        h = C.c_void_p()
        assert getattr(L, "cldnn_hip_%s_create" % kind)(None, C.byref(desc()), C.byref(h)) == -2
        enqueue = getattr(L, "cldnn_hip_%s_enqueue" % kind)
        assert enqueue(*[None] * len(enqueue.argtypes)) == -2
    assert hip.lib().cldnn_hip_last_error()


@pytest.fixture
def built(monkeypatch):
    """the scans of built code look into this library"""
    monkeypatch.setattr(hip, "LIB_PATH", ops_s8.LIB_PATH)


@needs_tools
def test_wait_states(tmp_path, built):
    products, loads = 0, 0
    for n, elf in enumerate(waits.code_objects()):
        path = tmp_path / ("%d.elf" % n)
        path.write_bytes(elf)
        for name, ins in waits.kernels(str(path)).items():
            products += sum(op in waits.NEED for op, _, _ in ins)
            loads += sum(lds.into_lds(*i[:2]) for i in ins)
            bad = waits.too_early(ins) + lds.too_near(ins)
            assert not bad, "%s: %s" % (name, bad[:3])
            assert not any(re.match(r"v_pk_(add|mul|fma)_f32", op) for op, _, _ in ins), name
    assert products > 200 and loads > 50


@needs_tools
def test_kernels_keep_their_values_in_registers(tmp_path, built):
    table = registers.resources.__wrapped__(tmp_path)
    assert len(table) > 20
    for name, (count, scratch) in table.items():
        assert scratch == 0, "%s: %d registers, %d bytes of scratch" % (name, count, scratch)
