"""CPU-side checks of the float operators' library: it exports what include/cldnn_hip_ops.h declares, the binding has the
header's structures, entry points refuse null handles, and matrix results get their wait states."""
import ctypes as C
import os
import re
import subprocess

import pytest

import test_mfma_wait_states as waits
from cldnn_amd import hip, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def header():
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "cldnn_hip_ops.h")).read(), flags=re.S)


def test_binding_covers_the_header():
    declared = set(re.findall(r"\b(cldnn_hip_[a-z0-9_]+)\s*\(", header()))
    assert set(ops.SIGNATURES) == declared and len(declared) == 12
    L = C.CDLL(ops.LIB_PATH)
    for n in declared:
        assert hasattr(L, n), "missing export: " + n


def test_structures_match_the_header(tmp_path):
    names = {"cldnn_hip_group_norm_desc": ops.GroupNormDesc, "cldnn_hip_matmul_desc": ops.MatmulDesc, "cldnn_hip_rotary_desc": ops.RotaryDesc,
             "cldnn_hip_attention_desc": ops.AttentionDesc, "cldnn_hip_operator_info": ops.OperatorInfo}
    lines = ["#include <stdio.h>", '#include "cldnn_hip_ops.h"', "int main(void) {"]
    for n, s in names.items():
        lines += ['printf("%%zu ", sizeof(%s));' % n] + ['printf("%%zu ", offsetof(%s, %s));' % (n, f[0]) for f in s._fields_]
    src = tmp_path / "offsets.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "offsets")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "offsets")], stdout=subprocess.PIPE, check=True, text=True).stdout.split()]
    want = []
    for s in names.values():
        want += [C.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want


def test_null_handles_are_refused():
    L = ops.lib()
    for create, desc in (("group_norm", ops.GroupNormDesc), ("matmul", ops.MatmulDesc), ("rotary", ops.RotaryDesc), ("attention", ops.AttentionDesc)):
        h = C.c_void_p()
        assert getattr(L, "cldnn_hip_%s_create" % create)(None, C.byref(desc()), C.byref(h)) == -2
        enqueue = getattr(L, "cldnn_hip_%s_enqueue" % create)
        assert enqueue(*[None] * len(enqueue.argtypes)) == -2
    assert L.cldnn_hip_operator_release(None) == L.cldnn_hip_operator_retain(None) == L.cldnn_hip_operator_get_info(None, None) == -2
    assert hip.lib().cldnn_hip_last_error()


def test_tensor_bytes():
    assert ops.tensor_bytes(ops.map_tensor("bf16", 2, 3, 5, 7, 1, 2, 4)) == 2 * 5 * 9 * 11 * 2
    assert ops.tensor_bytes(ops.map_tensor("f32", 1, 1, 1, 3)) == 12
    t = ops.map_tensor("f16", 1, 1, 1, 3)
    assert hip.lib().cldnn_hip_tensor_bytes(C.byref(t)) == 0  # the convolution path does not take the type
    t.dtype = 77
    assert ops.tensor_bytes(t) == 0


@pytest.mark.skipif(not os.path.exists(waits.OBJDUMP), reason="needs the ROCm disassembler")
def test_no_result_is_read_before_its_wait_states(tmp_path, monkeypatch):
    # 16x16x32 takes 4 passes, 32x32x16 takes 8
    monkeypatch.setattr(waits, "NEED", {"v_mfma_f32_%s_%s" % (shape, t): states for shape, states in (("16x16x32", 8), ("32x32x16", 12)) for t in ("f16", "bf16")})
    monkeypatch.setattr(hip, "LIB_PATH", ops.LIB_PATH)
    products = 0
    for n, elf in enumerate(waits.code_objects()):
        path = tmp_path / ("%d.elf" % n)
        path.write_bytes(elf)
        for name, ins in waits.kernels(str(path)).items():
            products += sum(op in waits.NEED for op, _, _ in ins)
            bad = waits.too_early(ins)
            assert not bad, "%s: %s" % (name, bad[:3])
            assert not any(re.match(r"v_pk_(add|mul|fma)_f32", op) for op, _, _ in ins), name
    assert products > 200
