"""One operator of two kernels, enqueued by two threads with data of their own: each result is that of the call alone."""
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
