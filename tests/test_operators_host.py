"""What the float operators' library does on the host, with a runtime that only writes launches down (tests/cpp/host_runtime.cpp):
the order of launches from several threads.  No GPU: each test is a process of its own."""
import ctypes as C
import os
import subprocess
import sys
import threading

import pytest

from cldnn_amd import hip, ops

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
ROCM = "/opt/rocm/include"
pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(ROCM, "hip")), reason="needs the runtime's headers")


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("host") / "runtime.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I", ROCM, os.path.join(HERE, "cpp", "host_runtime.cpp"), "-o", path],
                   check=True)
    return path


@pytest.fixture
def on_host(runtime):
    """runs a function of this module in a process whose runtime is the host's"""
    def run(function, *args):
        code = "import sys; sys.path[:0] = %r; import test_operators_host as t; t.%s(*%r)" % ([ROOT, HERE], function.__name__, args)
        env = dict(os.environ, LD_PRELOAD=":".join(x for x in (runtime, os.environ.get("LD_PRELOAD")) if x))
        p = subprocess.run([sys.executable, "-c", code], env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
        assert p.returncode == 0, p.stdout
    return run


# ---------------------------------------------------------------------------------------------------- in the other process
AT = 1 << 20  # stands for device memory: nothing reads it


def host():
    return C.CDLL(None)


def launches():
    """[(thread, kernel, workgroups, threads of one, bytes of dynamic LDS)] since the start"""
    h, name, shape, found = host(), C.create_string_buffer(1024), (C.c_uint * 3)(), []
    h.host_launch.restype = C.c_size_t
    for i in range(h.host_launches()):
        thread = h.host_launch(i, name, len(name), shape)
        found.append((thread, name.value.decode(), *shape))
    return found


def calls_of_two_kernels(e):
    """name -> (operator, a call of it)"""
    made = {
        "norm": (ops.GroupNorm(e, ops.group_norm_desc(ops.map_tensor("f16", 1, 90, 80, 64), 8)), (AT, AT)),
        "packed": (ops.Matmul(e, ops.matmul_desc(1001, 1000, 255, "f16")), (AT, AT, AT)),
        "joined": (ops.Matmul(e, ops.matmul_desc(7, 250, 9000, "f16")), (AT, AT, AT)),
        "attention": (ops.Attention(e, ops.attention_desc(1, 1, 5000, 8, 2, 64, "f16")), (AT, AT, AT, AT)),
    }
    for op, _ in made.values():
        assert op.info().launches == 2 and op.info().workspace_bytes
    return {k: (op, lambda op=op, args=args: op.enqueue(*args)) for k, (op, args) in made.items()}


def two_threads(name):
    e = hip.Engine()
    op, call = calls_of_two_kernels(e)[name]
    call()
    pair = [l[1] for l in launches()]
    assert len(pair) == 2 and pair[0] != pair[1]
    host().host_pause(300)

    def work():
        for _ in range(30):
            call()

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    found = launches()[2:]
    assert len(found) == 120
    # the second kernel of a call reads what its first one left in the object's memory
    for first, second in zip(found[::2], found[1::2]):
        assert [first[1], second[1]] == pair and first[0] == second[0], "a launch of the other thread between the kernels of a call"


@pytest.mark.parametrize("name", ["norm", "packed", "joined", "attention"])
def test_threads_that_enqueue_one_operator(on_host, name):
    on_host(two_threads, name)


def a_thread_and_a_recording():
    e = hip.Engine()
    op, call = calls_of_two_kernels(e)["attention"]
    L, rec = hip.lib(), C.c_void_p()
    hip.check(L.cldnn_hip_engine_record_begin(e.h))
    call()
    hip.check(L.cldnn_hip_engine_record_end(e.h, C.byref(rec)))
    host().host_pause(300)
    thread = threading.Thread(target=lambda: [hip.check(L.cldnn_hip_recording_enqueue(rec)) for _ in range(40)])
    thread.start()
    for _ in range(40):
        call()
    thread.join()
    found = [l[1] for l in launches()]
    assert len(found) == 120 and found.count("graph") == 40
    for i, name in enumerate(found):
        if "attention_join" in name:
            assert found[i - 1] != "graph", "a recording between the kernels of a call"


def test_a_thread_enqueues_and_another_a_recording(on_host):
    on_host(a_thread_and_a_recording)


def memory():
    host().host_memory.restype = C.c_size_t
    return host().host_memory()


def a_recording_outlives_its_operators(kept):
    e = hip.Engine()
    L, rec, before = hip.lib(), C.c_void_p(), memory()
    calls = calls_of_two_kernels(e)
    scratch = sum(op.info().workspace_bytes for op, _ in calls.values())
    assert memory() - before == scratch
    hip.check(L.cldnn_hip_engine_record_begin(e.h))
    for _, call in calls.values():
        call()
        call()
    hip.check(L.cldnn_hip_engine_record_end(e.h, C.byref(rec) if kept else None))
    for op, _ in calls.values():
        op.close()
    assert memory() - before == (scratch if kept else 0), "the scratch memory of a recording's kernels"
    if kept:
        e.close()
        hip.check(L.cldnn_hip_recording_enqueue(rec))
        hip.check(L.cldnn_hip_recording_release(rec))
        assert memory() == 0  # the engine's, too
    else:
        e.close()
        assert memory() == 0


@pytest.mark.parametrize("kept", [True, False])
def test_a_recording_holds_the_operators_in_it(on_host, kept):
    on_host(a_recording_outlives_its_operators, kept)


READELF = "/opt/rocm/llvm/bin/llvm-readelf"


def static_lds(directory):
    """mangled name -> bytes of LDS that a kernel of the operators' library has by itself"""
    import re

    import test_mfma_wait_states as scan

    found, hip.LIB_PATH = {}, ops.LIB_PATH
    for n, image in enumerate(scan.code_objects()):
        path = os.path.join(directory, "%d.elf" % n)
        with open(path, "wb") as f:
            f.write(image)
        notes = subprocess.run([READELF, "--notes", path], stdout=subprocess.PIPE, check=True, text=True).stdout
        for kernel in notes.split("  - .agpr_count:")[1:]:
            value = {k: re.search(r"\.%s:\s+(\S+)" % k, kernel).group(1) for k in ("name", "group_segment_fixed_size")}
            found[value["name"]] = int(value["group_segment_fixed_size"])
    return found


def infos_describe_the_launches(directory):
    e = hip.Engine()
    made = []
    for b, y, x, f, groups, dtype, out in ((1, 7, 7, 2048, 32, "bf16", "bf16"), (3, 31, 45, 84, 12, "f32", "f16"), (16, 224, 224, 64, 32, "f16", "f16"), (2, 200, 200, 21, 7, "f32", "f32")):
        made.append((ops.GroupNorm(e, ops.group_norm_desc(ops.map_tensor(dtype, b, y, x, f), groups, out_dtype=out)), 2))
    for m, n, k in ((4090, 4093, 72), (7160, 2040, 136), (6130, 2046, 64), (3100, 1537, 200), (1601, 1000, 104), (1001, 1000, 264), (190, 2000, 520), (30, 1000, 1000), (7, 250, 9000),
                    (600, 500, 63), (1601, 1400, 61), (1001, 1000, 255), (3101, 1500, 263), (3101, 1700, 263), (1, 1, 1)):
        made.append((ops.Matmul(e, ops.matmul_desc(m, n, k, "f16")), 3))
    for tokens, q, k, size, pairs, pairing in ((196, 16, 16, 64, (16, 16), "halves"), (25088, 16, 4, 128, (16, 24, 24), "interleaved"), (5, 1, 1, 33, (7, 3), "halves_per_axis")):
        made.append((ops.Rotary(e, ops.rotary_desc(tokens, q, k, size, pairs, "bf16", pairing=pairing)), 5))
    for b, lq, lk, h, kv, d in ((64, 49, 49, 4, 4, 32), (4, 3136, 3136, 8, 8, 64), (2, 1, 50176, 8, 2, 128), (4, 1030, 130, 4, 4, 104), (2, 1030, 65, 8, 8, 160), (1, 30, 1000, 2, 2, 200)):
        made.append((ops.Attention(e, ops.attention_desc(b, lq, lk, h, kv, d, "bf16")), 4))
    lds = static_lds(directory)
    for op, pointers in made:
        before = len(launches())
        op.enqueue(*[AT] * pointers)
        found, i = launches()[before:], op.info()
        name = i.kernel_name.decode()
        assert i.launches == len(found), name
        assert (i.grid, i.block) == found[0][2:4], "%s: %r, launched %r" % (name, (i.grid, i.block), found[0])
        assert i.lds_bytes == max(lds[l[1]] + l[4] for l in found), "%s: %d bytes of LDS" % (name, i.lds_bytes)
        # every kernel is named
        for part in ("matmul_pack", "matmul_split", "matmul_tile", "matmul_join", "norm_whole", "norm_stats", "norm_apply", "rotary"):
            assert (part in name) == any(part in l[1] for l in found), "%s: %r" % (name, [l[1] for l in found])


@pytest.mark.skipif(not os.path.exists(READELF), reason="needs the kernels' metadata")
def test_infos_describe_the_launches(on_host, tmp_path):
    on_host(infos_describe_the_launches, str(tmp_path))


def a_refusal(call, word):
    before = len(launches())
    try:
        call()
    except hip.HipError as e:
        assert e.status == -2 and word in str(e), e
    else:
        raise AssertionError("taken: " + word)
    assert len(launches()) == before


def operands_are_checked():
    import torch

    class OnDevice(torch.Tensor):  # host memory that says it is the device's: nothing reads it
        def get_device(self):
            return 0

    def dev(*shape, dtype=torch.float16):
        return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice)

    e = hip.Engine()
    op = ops.Matmul(e, ops.matmul_desc(5, 24, 16, "f16", bias=True, residual=True, out_stride=32))
    good = dict(a=dev(5, 16), weights=dev(24, 16), out=dev(5, 32), bias=dev(24, dtype=torch.float32), residual=dev(5, 24))

    def call(**other):
        op.enqueue(**dict(good, **other))

    def taken(**other):
        before = len(launches())
        call(**other)
        assert len(launches()) == before + 1

    taken()
    # memory, an address, a buffer, a view that is laid out as described
    taken(a=dev(80), weights=dev(24 * 16 * 2, dtype=torch.uint8), out=dev(5 * 32)[:152], residual=AT)
    taken(out=dev(5, 32)[:, :24])
    buffer = ops.Buffer(e, 2 * 5 * 16)
    taken(a=buffer)
    a_refusal(lambda: call(a=torch.zeros(5, 16, dtype=torch.float16)), "a: a tensor on cpu")
    a_refusal(lambda: call(a=dev(16, 5).t()), "a: a tensor of shape (5, 16) and strides (1, 5)")
    a_refusal(lambda: call(weights=dev(24, 32)[:, :16]), "weights: a tensor of shape (24, 16) and strides (32, 1)")
    a_refusal(lambda: call(out=dev(5, 32, dtype=torch.uint8)[:, :24]), "output: a tensor of shape")
    a_refusal(lambda: call(out=dev(5, 24)), "output: 240 bytes, described are 304")
    a_refusal(lambda: call(residual=dev(5, 24, dtype=torch.bfloat16)), "residual: a tensor of torch.bfloat16")
    a_refusal(lambda: call(bias=dev(24)), "bias: a tensor of torch.float16")
    a_refusal(lambda: call(weights=buffer), "weights: a buffer of 160 bytes, described are 768")

    op = ops.Attention(e, ops.attention_desc(2, 3, 70, 4, 2, 32, "bf16", key_lengths=True, bias_shape=(1, 4, 1, 70), k_strides=(70 * 64, 32, 70 * 32)))
    b16 = torch.bfloat16
    good = dict(q=dev(2, 3, 4, 32, dtype=b16), k=dev(2, 2, 70, 32, dtype=b16), v=dev(2, 70, 2, 32, dtype=b16), out=dev(2, 3, 4, 32, dtype=b16), key_lengths=dev(2, dtype=torch.int32),
                bias=dev(1, 4, 1, 70, dtype=b16))
    taken()
    taken(k=good["k"].transpose(1, 2))
    a_refusal(lambda: call(v=good["k"].transpose(1, 2)), "v: a tensor of shape")
    a_refusal(lambda: call(q=good["q"][:, :2]), "q: a tensor of shape")
    a_refusal(lambda: call(q=dev(2, 2, 4, 32, dtype=b16)), "q: 1024 bytes, described are 1536")
    a_refusal(lambda: call(key_lengths=dev(2, dtype=torch.int64)), "key_lengths: a tensor of torch.int64")
    a_refusal(lambda: call(bias=dev(4, 69, dtype=b16)), "bias: 552 bytes, described are 560")

    op = ops.GroupNorm(e, ops.group_norm_desc(ops.map_tensor("f16", 2, 3, 5, 8, 1, 2, 4), 4, out_dtype="f32"))
    whole = dev(2, 5, 9, 12)
    good = dict(src=whole, dst=dev(2, 3, 5, 8, dtype=torch.float32))
    taken()
    a_refusal(lambda: call(src=whole[:, 1:4, 2:7, :8]), "input: a tensor of shape")  # the description counts from the padding on
    a_refusal(lambda: call(dst=dev(2, 3, 5, 8)), "output: a tensor of torch.float16")
    a_refusal(lambda: call(scale=dev(7, dtype=torch.float32)), "scale: 28 bytes, described are 32")

    op = ops.Rotary(e, ops.rotary_desc(7, 2, 1, 16, (4, 4), "f16", q_strides=(48, 16)))
    qkv = dev(7, 3, 16)
    good = dict(q=qkv[:, :2], k=dev(7, 1, 16), positions=dev(7, 2, dtype=torch.int32), q_out=dev(7, 2, 16), k_out=dev(7, 1, 16))
    taken()
    taken(q=qkv)
    a_refusal(lambda: call(k=qkv[:, 2:]), "k: a tensor of shape")
    a_refusal(lambda: call(positions=dev(7, 2, dtype=torch.float32)), "positions: a tensor of torch.float32")


def test_operands_are_checked(on_host):
    on_host(operands_are_checked)


def entry_points_refuse():
    """the C entry points themselves, given addresses"""
    e = hip.Engine()
    made = [  # operator, how many pointers, the alignment of each in bytes, those that may be null
        (ops.GroupNorm(e, ops.group_norm_desc(ops.map_tensor("f16", 1, 4, 4, 12), 4, out_dtype="f32")), (2, 4, 4, 4), (1, 2)),
        (ops.Matmul(e, ops.matmul_desc(4, 4, 4, "f16", bias=True, residual=True, residual_dtype="f32")), (2, 2, 4, 4, 2), ()),
        (ops.Matmul(e, ops.matmul_desc(4, 4, 4, "f16", out_dtype="f32")), (2, 2, 1, 1, 4), (2, 3)),
        (ops.Rotary(e, ops.rotary_desc(4, 2, 2, 16, (4, 4), "f16")), (2, 2, 4, 2, 2), ()),
        (ops.Attention(e, ops.attention_desc(1, 4, 4, 2, 2, 32, "f16", key_lengths=True, bias_shape=(1, 1, 4, 4))), (16, 16, 16, 4, 2, 16), ()),
    ]
    for op, aligned, optional in made:
        assert op._enqueue(op.h, *[AT] * len(aligned)) == 0
        for i, to in enumerate(aligned):
            pointers = [AT] * len(aligned)
            pointers[i] = None
            assert (op._enqueue(op.h, *pointers) == 0) == (i in optional), (type(op), i)
            if to > 1:
                pointers[i] = AT + to // 2
                assert op._enqueue(op.h, *pointers) == -2 and b"aligned" in hip.lib().cldnn_hip_last_error(), (type(op), i)


def test_entry_points_refuse(on_host):
    on_host(entry_points_refuse)


def grids_hold_what_they_launch():
    """The runtime counts the threads of a grid in 32 bits, and the kernels rows and features in 31: a size beyond is refused when the
    object is made, whatever memory there is."""
    e = hip.Engine()
    most = (1 << 31) - 1

    def status(kind, desc):
        try:
            kind(e, desc).close()
            return 0
        except hip.HipError as x:
            assert "too" in str(x), x
            return x.status

    for m, n, k in ((most, 8, 8), (most - 200, 8, 8), (8, most, 8), (most, 1, 1), (1, most, 3), (1, 1, most), (2, 2, most - 8), (most - 300, 1 << 17, 8), (1 << 30, 1 << 13, 9)):
        assert status(ops.Matmul, ops.matmul_desc(m, n, k, "f16")) == -5, (m, n, k)
    for size in ((65535, 1, 1, 512, 512, 32), (65535, 300, 300, 128, 128, 64)):
        assert status(ops.Attention, ops.attention_desc(*size, "f16")) == -5, size
    for tokens, heads in ((1 << 30, 1), (1 << 41, 1), (4, most)):
        assert status(ops.Rotary, ops.rotary_desc(tokens, heads, heads if heads > 1 else 0, 64, (32,), "f32")) == -5, (tokens, heads)
    # the largest that are left
    made = [(ops.Matmul(e, ops.matmul_desc(m, n, k, "f16")), 3, -(-m // rows) * -(-n // columns)) for m, n, k, rows, columns in (
        (1 << 30, 64, 8, 128, 128), (1 << 28, 8, 129, 64, 64), (1, (1 << 30) - 7, 8, 128, 128), (7, 3, most - 300, 16, 16))]
    made += [(ops.Rotary(e, ops.rotary_desc((1 << 28) - 1, 1, 0, 64, (32,), "f16")), 5, -(-((1 << 28) - 1) * 8 // 256))]
    made += [(ops.Attention(e, ops.attention_desc(65535, 1, 1, 255, 255, 32, "f16")), 4, 65535 * 255)]
    for op, pointers, workgroups in made:
        before = len(launches())
        op.enqueue(*[AT] * pointers)
        grid = launches()[before][2:4]
        assert grid[0] % workgroups == 0 and grid[0] * grid[1] < 1 << 32, (op.info().kernel_name, grid, workgroups)


def test_grids_hold_what_they_launch(on_host):
    on_host(grids_hold_what_they_launch)
