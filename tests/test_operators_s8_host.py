"""What the int8 operators' library does on the host, with the runtime that only writes launches down (tests/cpp/host_runtime.cpp):
refusals, infos, checks of operands, threads and recordings.  No GPU: each test is a process of its own."""
import ctypes as C
import math
import os
import subprocess
import sys
import threading

import pytest

import test_operators_host as host
from cldnn_amd import hip, ops, ops_s8
from test_operators_host import AT, a_refusal, launches, memory, runtime  # noqa: F401

pytestmark = host.pytestmark


@pytest.fixture
def on_host(runtime):  # noqa: F811
    """runs a function of this module in a process whose runtime is the host's"""
    def run(function, *args):
        code = "import sys; sys.path[:0] = %r; import test_operators_s8_host as t; t.%s(*%r)" % ([host.ROOT, host.HERE], function.__name__, args)
        env = dict(os.environ, LD_PRELOAD=":".join(x for x in (runtime, os.environ.get("LD_PRELOAD")) if x))
        p = subprocess.run([sys.executable, "-c", code], env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
        assert p.returncode == 0, p.stdout
    return run


# ---------------------------------------------------------------------------------------------------- in the other process
def calls_of_two_kernels(e):
    made = {"packed": ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(1001, 1000, 255)), "joined": ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(7, 250, 30000))}
    for op in made.values():
        assert op.info().launches == 2 and op.info().workspace_bytes
    return {k: (op, lambda op=op: op.enqueue(AT, AT, AT, AT, AT)) for k, op in made.items()}


def two_threads(name):
    e = hip.Engine()
    op, call = calls_of_two_kernels(e)[name]
    call()
    pair = [l[1] for l in launches()]
    assert len(pair) == 2 and pair[0] != pair[1]
    host.host().host_pause(300)
    threads = [threading.Thread(target=lambda: [call() for _ in range(30)]) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    found = launches()[2:]
    assert len(found) == 120
    for first, second in zip(found[::2], found[1::2]):
        assert [first[1], second[1]] == pair and first[0] == second[0], "a launch of the other thread between the kernels of a call"


@pytest.mark.parametrize("name", ["packed", "joined"])
def test_threads_that_enqueue_one_operator(on_host, name):
    on_host(two_threads, name)


def a_recording_outlives_its_operators():
    e = hip.Engine()
    L, rec, before = hip.lib(), C.c_void_p(), memory()
    calls = calls_of_two_kernels(e)
    scratch = sum(op.info().workspace_bytes for op, _ in calls.values())
    assert memory() - before == scratch
    hip.check(L.cldnn_hip_engine_record_begin(e.h))
    for _, call in calls.values():
        call()
    hip.check(L.cldnn_hip_engine_record_end(e.h, C.byref(rec)))
    for op, _ in calls.values():
        op.close()
    assert memory() - before == scratch
    e.close()
    hip.check(L.cldnn_hip_recording_enqueue(rec))
    hip.check(L.cldnn_hip_recording_release(rec))
    assert memory() == 0


def test_a_recording_holds_the_operators_in_it(on_host):
    on_host(a_recording_outlives_its_operators)


def infos_describe_the_launches(directory):
    e = hip.Engine()
    made = []
    for rows, features in ((3, 100), (17, 512), (300, 1000), (5, 2048), (9, 4096), (2, 8192), (3, 16000), (1, 32768), (7, 32769)):
        made.append((ops_s8.Quantize(e, ops_s8.quantize_desc(rows, features, "f16")), 4))
        if features <= 32768:
            made.append((ops_s8.BlockNorm(e, ops_s8.block_norm_desc(rows, features, "f32", branch_dtype="f16", out_dtype="s8")), 12))
    for m, n, k in ((4090, 4093, 144), (7160, 2042, 272), (6130, 2046, 64), (4090, 4092, 144), (7160, 2040, 272), (6130, 2044, 64), (3100, 1537, 208), (1601, 1000, 112), (1001, 1000, 272), (190, 2000, 528), (30, 1000, 1000), (7, 250, 30000),
                    (600, 500, 63), (1601, 1400, 61), (1001, 1000, 255), (1, 1, 1)):
        made.append((ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(m, n, k)), 7))
    hip_path = hip.LIB_PATH
    ops.LIB_PATH, kept = ops_s8.LIB_PATH, ops.LIB_PATH  # where static_lds looks
    lds = host.static_lds(directory)
    ops.LIB_PATH, hip.LIB_PATH = kept, hip_path
    for op, pointers in made:
        before = len(launches())
        assert op._enqueue(op.h, *[AT] * pointers) == 0
        found, i = launches()[before:], op.info()
        name = i.kernel_name.decode()
        assert i.launches == len(found), name
        assert (i.grid, i.block) == found[0][2:4], "%s: %r, launched %r" % (name, (i.grid, i.block), found[0])
        assert i.lds_bytes == max(lds[l[1]] + l[4] for l in found), "%s: %d bytes of LDS" % (name, i.lds_bytes)
        for part in ("matmul_pack", "matmul_join", "quantize", "block_norm"):
            assert (part in name) == any(part in l[1] for l in found), "%s: %r" % (name, [l[1] for l in found])
        assert ("split" in name) == any("matmul_split" in l[1] for l in found) and ("tile" in name) == any("matmul_tile" in l[1] for l in found)
        assert ("walk" in name) == any("matmul_s8_walk" in l[1] for l in found)


@pytest.mark.skipif(not os.path.exists(host.READELF), reason="needs the kernels' metadata")
def test_infos_describe_the_launches(on_host, tmp_path):
    on_host(infos_describe_the_launches, str(tmp_path))


def operands_are_checked():
    import torch

    class OnDevice(torch.Tensor):  # host memory that says it is the device's: nothing reads it
        def get_device(self):
            return 0

    def dev(*shape, dtype=torch.float16):
        return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)

    e, s8, f32 = hip.Engine(), torch.int8, torch.float32

    def checks(call, good, bad, fine=()):
        before = len(launches())
        call(**good)
        for other in fine:
            call(**dict(good, **other))
        assert len(launches()) == before + 1 + len(fine)
        for other, words in bad:
            a_refusal(lambda: call(**dict(good, **other)), words)

    op = ops_s8.Quantize(e, ops_s8.quantize_desc(5, 24, "f16", gated=True, factors=True, out_stride=32))
    checks(op.enqueue, dict(src=dev(5, 48), dst=dev(5, 32, dtype=s8), scales=dev(5, dtype=f32), factors=dev(24, dtype=f32)),
           [(dict(src=dev(5, 47)), "input: 470 bytes, described are 480"), (dict(src=dev(5, 48, dtype=f32)), "input: a tensor of torch.float32"), (dict(dst=dev(5, 24, dtype=s8)), "output: 120 bytes, described are 152"),
            (dict(dst=dev(5, 32)), "output: a tensor of torch.float16"), (dict(scales=dev(4, dtype=f32)), "scales: 16 bytes, described are 20"), (dict(factors=dev(23, dtype=f32)), "factors: 92 bytes"),
            (dict(factors=None), "null"), (dict(src=torch.zeros(5, 48, dtype=torch.float16)), "input: a tensor on cpu")],
           [dict(dst=dev(5, 32, dtype=s8)[:, :24]), dict(dst=dev(152, dtype=torch.uint8))])

    op = ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(5, 24, 16, out_dtype="f16", weights_scales="one", bias=True, residual=True, residual_dtype="bf16", a_stride=20))
    checks(op.enqueue, dict(a=dev(5, 20, dtype=s8), weights=dev(24, 16, dtype=s8), out=dev(5, 24), a_scales=dev(5, dtype=f32), weights_scales=dev(1, dtype=f32), bias=dev(24, dtype=f32),
                            residual=dev(5, 24, dtype=torch.bfloat16)),
           [(dict(a=dev(5, 20)), "a: a tensor of torch.float16"), (dict(a=dev(5, 16, dtype=s8)[:, :15]), "a: a tensor of shape"), (dict(a_scales=dev(4, dtype=f32)), "a_scales: 16 bytes"),
            (dict(a_scales=None), "null"), (dict(weights_scales=None), "null"), (dict(bias=None), "null"), (dict(residual=None), "null"), (dict(residual=dev(5, 24)), "residual: a tensor of torch.float16"),
            (dict(out=dev(5, 23)), "output: 230 bytes, described are 240"), (dict(weights=dev(24, 15, dtype=s8)), "weights: 360 bytes")],
           [dict(a=dev(5, 20, dtype=s8)[:, :16])])

    op = ops_s8.BlockNorm(e, ops_s8.block_norm_desc(6, 24, "bf16", branch_dtype="f16", out_dtype="s8", tokens_per_image=4, modulation_dtype="f16", gate_stride=72))
    modulation, b16 = dev(2, 72), torch.bfloat16
    checks(op.enqueue, dict(x=dev(6, 24, dtype=b16), y=dev(6, 24, dtype=b16), out=dev(6, 24, dtype=s8), branch=dev(6, 24), post_weight=dev(24, dtype=f32), post_bias=dev(24, dtype=f32),
                            gate=modulation[:, :24], weight=dev(24, dtype=f32), bias=dev(24, dtype=f32), scale=dev(2, 24), shift=dev(2, 24), out_scales=dev(6, dtype=f32)),
           [(dict(x=dev(6, 24)), "x: a tensor of torch.float16"), (dict(y=dev(5, 24, dtype=b16)), "y: 240 bytes, described are 288"), (dict(branch=None), "null"), (dict(out=None), "null"), (dict(out_scales=None), "null"),
            (dict(out_scales=dev(5, dtype=f32)), "out_scales: 20 bytes"), (dict(gate=dev(1, 72)), "gate: 144 bytes"), (dict(scale=modulation[:, 24:48]), "scale: a tensor of shape"), (dict(shift=dev(2, 24, dtype=f32)), "shift: a tensor"),
            (dict(weight=dev(23, dtype=f32)), "weight: 92 bytes"), (dict(post_bias=dev(24)), "post_bias: a tensor of torch.float16"), (dict(out=dev(6, 24)), "output: a tensor of torch.float16")],
           [dict(y=None), dict(gate=None, scale=None, shift=None, weight=None, bias=None, post_weight=None, post_bias=None)])
    x = dev(6, 24, dtype=b16)
    op.enqueue(x, x, dev(6, 24, dtype=s8), branch=dev(6, 24), out_scales=dev(6, dtype=f32))


def test_operands_are_checked(on_host):
    on_host(operands_are_checked)


def entry_points_refuse():
    """the C entry points themselves, given addresses"""
    e = hip.Engine()
    made = [  # operator, the alignment of each pointer in bytes, those that may be null
        (ops_s8.Quantize(e, ops_s8.quantize_desc(4, 12, "f16", factors=True)), (2, 4, 1, 4), ()),
        (ops_s8.Quantize(e, ops_s8.quantize_desc(4, 12, "f32")), (4, 1, 1, 4), (1,)),
        (ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(4, 4, 4, out_dtype="f16", bias=True, residual=True, residual_dtype="f32")), (1, 1, 4, 4, 4, 4, 2), ()),
        (ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(4, 4, 4, a_scales=None, weights_scales=None)), (1, 1, 1, 1, 1, 1, 4), (2, 3, 4, 5)),
        (ops_s8.BlockNorm(e, ops_s8.block_norm_desc(4, 12, "f32", branch_dtype="f16", out_dtype="s8", modulation_dtype="bf16")), (4, 2, 4, 4, 2, 4, 4, 2, 2, 4, 1, 4), (2, 3, 4, 5, 6, 7, 8, 9)),
        (ops_s8.BlockNorm(e, ops_s8.block_norm_desc(4, 12, "f16", out_dtype="f32")), (2, 1, 1, 1, 1, 4, 4, 1, 1, 1, 4, 1), (1, 2, 3, 4, 5, 6, 7, 8, 9, 11)),
        (ops_s8.BlockNorm(e, ops_s8.block_norm_desc(4, 12, "f16", branch_dtype="f32", norm="none")), (2, 4, 4, 4, 1, 1, 1, 1, 1, 2, 1, 1), (2, 3, 4, 5, 6, 7, 8, 10, 11)),
    ]
    for op, aligned, optional in made:
        assert op._enqueue(op.h, *[AT] * len(aligned)) == 0
        for i, to in enumerate(aligned):
            pointers = [AT] * len(aligned)
            pointers[i] = None
            assert (op._enqueue(op.h, *pointers) == 0) == (i in optional), (type(op), i)
            pointers[i] = AT + 4096 + to // 2
            if to > 1:
                assert op._enqueue(op.h, *pointers) == -2 and b"aligned" in hip.lib().cldnn_hip_last_error(), (type(op), i)
            else:
                assert op._enqueue(op.h, *pointers) == 0
    # an operator of another kind, in each library
    quantize, product = made[0][0], ops.Matmul(e, ops.matmul_desc(4, 4, 4, "f16"))
    assert product._enqueue(quantize.h, *[AT] * 5) == quantize._enqueue(product.h, *[AT] * 4) == -2
    # the stream in its own place has one stride
    op = ops_s8.BlockNorm(e, ops_s8.block_norm_desc(4, 12, "f16", branch_dtype="f16", norm="none", y_stride=16))
    pointers = [AT, AT + 4096] + [None] * 7 + [AT, None, None]
    assert op._enqueue(op.h, *pointers) == -2 and op._enqueue(op.h, *pointers[:9], AT + 8192, None, None) == 0


def test_entry_points_refuse(on_host):
    on_host(entry_points_refuse)


def descriptions_are_checked():
    """the refusals of the GPU tests, where no device is"""
    import test_block_norm_gpu as block_norm
    import test_matmul_s8_gpu as matmul
    import test_quantize_gpu as quantize

    e = hip.Engine()
    for module in (quantize, matmul, block_norm):
        module.test_refusals(e)
    assert math.isfinite(ops_s8.Quantize(e, ops_s8.quantize_desc(4, 4, "f16")).info().ops)


def test_descriptions_are_checked(on_host):
    on_host(descriptions_are_checked)


def grids_hold_what_they_launch():
    """The runtime counts the threads of a grid in 32 bits: the largest that are left are launched whole."""
    e = hip.Engine()
    most = (1 << 32) // 256 - 1
    made = [(ops_s8.Quantize(e, ops_s8.quantize_desc(16 * most, 128, "f16")), 4, most), (ops_s8.Quantize(e, ops_s8.quantize_desc(4 * most, 500, "f32")), 4, most),
            (ops_s8.BlockNorm(e, ops_s8.block_norm_desc(16 * most, 8, "f16", out_dtype="s8")), 12, most), (ops_s8.Quantize(e, ops_s8.quantize_desc((1 << 22) - 1, 40000, "f32")), 4, (1 << 22) - 1),
            (ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(1 << 30, 64, 16)), 7, (1 << 30) // 128)]
    for op, pointers, workgroups in made:
        before = len(launches())
        assert op._enqueue(op.h, *[AT] * pointers) == 0
        grid = launches()[before][2:4]
        assert grid[0] == workgroups and grid[0] * grid[1] < 1 << 32, (op.info().kernel_name, grid, workgroups)
    for kind, desc in ((ops_s8.Quantize, ops_s8.quantize_desc(16 * most + 1, 128, "f16")), (ops_s8.BlockNorm, ops_s8.block_norm_desc(4 * most + 1, 500, "f16", out_dtype="f16")),
                       (ops_s8.Quantize, ops_s8.quantize_desc(1 << 22, 40000, "f32"))):
        try:
            kind(e, desc).close()
            raise AssertionError("taken")
        except hip.HipError as x:
            assert x.status == -5 and "too large" in str(x)


def test_grids_hold_what_they_launch(on_host):
    on_host(grids_hold_what_they_launch)
