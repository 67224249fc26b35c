"""One operator of two kernels, enqueued by two threads with data of their own: each result is that of the call alone.  A recording
that outlives its operator.  Operands in pinned host memory."""
import threading

import pytest
import torch

from cldnn_amd import hip, ops
from operator_cases import *

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = hip.Engine()
    yield e
    e.close()


def operators(eng):
    def rand(*shape):
        return random(generator(sum(shape)), *shape, dtype="f16").cuda()

    k, v, w, far = rand(1, 5000, 2, 64), rand(1, 5000, 2, 64), rand(250, 9000), rand(1000, 255)
    return {
        "norm": (ops.GroupNorm(eng, ops.group_norm_desc(ops.map_tensor("f16", 1, 90, 80, 64), 8)), (1, 90, 80, 64), (1, 90, 80, 64), lambda op, x, y: op.enqueue(x, y)),
        "packed": (ops.Matmul(eng, ops.matmul_desc(1001, 1000, 255, "f16")), (1001, 255), (1001, 1000), lambda op, x, y: op.enqueue(x, far, y)),
        "joined": (ops.Matmul(eng, ops.matmul_desc(7, 250, 9000, "f16")), (7, 9000), (7, 250), lambda op, x, y: op.enqueue(x, w, y)),
        "attention": (ops.Attention(eng, ops.attention_desc(1, 1, 5000, 8, 2, 64, "f16")), (1, 1, 8, 64), (1, 1, 8, 64), lambda op, x, y: op.enqueue(x, k, v, y)),
    }


@pytest.mark.parametrize("name", ["norm", "packed", "joined", "attention"])
def test_threads_that_enqueue_one_operator(eng, name):
    op, inner, outer, call = operators(eng)[name]
    assert op.info().launches == 2
    x = [random(generator(n), *inner, dtype="f16").cuda() for n in range(2)]
    want = [torch.empty(outer, dtype=torch.float16, device="cuda") for _ in x]
    got = [[torch.zeros(outer, dtype=torch.float16, device="cuda") for _ in range(50)] for _ in x]
    torch.cuda.synchronize()
    for a, b in zip(x, want):
        call(op, a, b)
        eng.finish()
    start = threading.Barrier(2)

    def work(n):
        start.wait()
        for y in got[n]:
            call(op, x[n], y)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    eng.finish()
    for n in range(2):
        assert all(torch.equal(y, want[n]) for y in got[n])
    op.close()


@pytest.mark.parametrize("name", ["norm", "packed", "joined", "attention"])
def test_a_recording_outlives_its_operator(eng, name):
    op, inner, outer, call = operators(eng)[name]
    x = random(generator(7), *inner, dtype="f16").cuda()
    want, got = (torch.zeros(outer, dtype=torch.float16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    call(op, x, want)
    L, rec = hip.lib(), hip.C.c_void_p()
    hip.check(L.cldnn_hip_engine_record_begin(eng.h))
    call(op, x, got)
    hip.check(L.cldnn_hip_engine_record_end(eng.h, hip.C.byref(rec)))
    scratch = op.info().workspace_bytes
    used = L.cldnn_hip_engine_used_memory(eng.h)
    op.close()
    assert L.cldnn_hip_engine_used_memory(eng.h) == used
    # memory of the size that would have been given back, taken by others
    others = [ops.Buffer(eng, scratch) for _ in range(4)]
    for _ in range(3):
        got.zero_()
        torch.cuda.synchronize()
        hip.check(L.cldnn_hip_recording_enqueue(rec))
        eng.finish()
        assert torch.equal(got, want)
    for b in others:
        assert (b.read((scratch // 4,), "i32") == 0).all()
        b.close()
    used = L.cldnn_hip_engine_used_memory(eng.h)
    hip.check(L.cldnn_hip_recording_release(rec))
    assert L.cldnn_hip_engine_used_memory(eng.h) == used - scratch


def test_operands_in_pinned_memory(eng):
    a, w = (random(generator(n), n, 64, dtype="f16") for n in (3, 40))
    out, far = torch.empty(3, 40, dtype=torch.float16).pin_memory(), torch.empty(3, 40, dtype=torch.float16, device="cuda")
    op = ops.Matmul(eng, ops.matmul_desc(3, 40, 64, "f16"))
    run(eng, op, a.pin_memory(), w.cuda(), out)
    run(eng, op, a.cuda(), w.cuda(), far)
    assert torch.equal(out, far.cpu())
    with pytest.raises(hip.HipError) as err:
        op.enqueue(a, w.cuda(), far)
    assert err.value.status == INVALID_ARG
    op.close()
