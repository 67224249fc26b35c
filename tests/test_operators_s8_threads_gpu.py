"""Int8 operators of two kernels, enqueued by two threads with data of their own; a recording that outlives its operators, replayed with
other calls between; operands in pinned host memory; two engines."""
import threading

import pytest
import torch

from cldnn_amd import hip, ops, ops_s8
from operator_s8_cases import *

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = hip.Engine()
    yield e
    e.close()


def integers(seed, *shape):
    return torch.randint(-128, 128, shape, generator=generator(seed)).to(torch.int8).cuda()


def operators(eng):
    def product(m, n, k):
        w, s = integers(n, n, k), random(generator(k), n).exp().cuda()
        op = ops_s8.MatmulS8(eng, ops_s8.matmul_s8_desc(m, n, k, a_scales=None))
        return op, (m, k), (m, n), lambda x, y: op.enqueue(x, w, y, None, s)

    return {"packed": product(1001, 1000, 255), "joined": product(7, 250, 30000), "walk": product(4000, 4096, 256)}


@pytest.mark.parametrize("name", ["packed", "joined", "walk"])
def test_threads_that_enqueue_one_operator(eng, name):
    op, inner, outer, call = operators(eng)[name]
    assert op.info().launches == (1 if name == "walk" else 2)
    x = [integers(n, *inner) for n in range(2)]
    want = [torch.empty(outer, device="cuda") for _ in x]
    got = [[torch.zeros(outer, device="cuda") for _ in range(20)] for _ in x]
    torch.cuda.synchronize()
    for a, b in zip(x, want):
        call(a, b)
        eng.finish()
    start = threading.Barrier(2)

    def work(n):
        start.wait()
        for y in got[n]:
            call(x[n], y)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    eng.finish()
    for n in range(2):
        assert all(torch.equal(y, want[n]) for y in got[n])
    op.close()


def test_a_recorded_block_outlives_its_operators(eng):
    """norm -> int8 -> product -> gelu -> int8 -> product with a long K, recorded once and replayed on other values in the same memory"""
    rows, c, wide = 9, 640, 16400
    g = generator(3)
    x, branch = (torch.empty(rows, c, device="cuda") for _ in range(2))
    q, s, wide_q = torch.empty(rows, c, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, wide, dtype=torch.int8, device="cuda")
    up, out = torch.empty(rows, wide, dtype=torch.float16, device="cuda"), torch.empty(rows, c, device="cuda")
    w1, w2, s1, s2 = integers(1, wide, c), integers(2, c, wide), (random(g, wide).exp() / 2000).cuda(), (random(g, c).exp() / 9000).cuda()
    made = [ops_s8.BlockNorm(eng, ops_s8.block_norm_desc(rows, c, "f32", branch_dtype="f32", out_dtype="s8", norm="rms")), ops_s8.MatmulS8(eng, ops_s8.matmul_s8_desc(rows, wide, c, out_dtype="f16")),
            ops_s8.Quantize(eng, ops_s8.quantize_desc(rows, wide, "f16", act="gelu")), ops_s8.MatmulS8(eng, ops_s8.matmul_s8_desc(rows, c, wide, residual=True))]
    assert made[3].info().launches == 2

    def block():
        made[0].enqueue(x, x, q, branch=branch, out_scales=s)
        made[1].enqueue(q, w1, up, s, s1)
        made[2].enqueue(up, wide_q, s)
        made[3].enqueue(wide_q, w2, out, s, s2, residual=x)

    values = [[random(generator(n), rows, c).cuda() for n in (k, 100 + k)] for k in range(3)]

    def load(pair):
        x.copy_(pair[0]), branch.copy_(pair[1]), out.zero_()
        torch.cuda.synchronize()

    want = []
    for pair in values:
        load(pair)
        block()
        eng.finish()
        want.append((x.clone(), out.clone()))
    assert not torch.equal(want[0][1], want[1][1])
    L, rec = hip.lib(), hip.C.c_void_p()
    hip.check(L.cldnn_hip_engine_record_begin(eng.h))
    block()
    hip.check(L.cldnn_hip_engine_record_end(eng.h, hip.C.byref(rec)))
    scratch = made[3].info().workspace_bytes
    # the operators' own calls and synchronizations lie between the replays
    for k, pair in enumerate(values):
        load(pair)
        hip.check(L.cldnn_hip_recording_enqueue(rec))
        eng.finish()
        assert torch.equal(x, want[k][0]) and torch.equal(out, want[k][1])
        load(values[0])
        block()
        eng.finish()
        assert torch.equal(out, want[0][1])
    for op in made:
        op.close()
    others = [ops.Buffer(eng, scratch) for _ in range(4)]
    for k, pair in enumerate(values):
        load(pair)
        hip.check(L.cldnn_hip_recording_enqueue(rec))
        eng.finish()
        assert torch.equal(out, want[k][1])
    for b in others:
        assert (b.read((scratch // 4,), "i32") == 0).all()
        b.close()
    hip.check(L.cldnn_hip_recording_release(rec))


def test_two_engines(eng):
    """objects of the same shapes on two queues, at the same time"""
    other = hip.Engine()
    made = [operators(e)["joined"] for e in (eng, other)]
    x = [integers(n, *made[0][1]) for n in range(2)]
    got = [[torch.zeros(made[0][2], device="cuda") for _ in range(20)] for _ in x]
    torch.cuda.synchronize()
    for k in range(20):
        for n in range(2):
            made[n][3](x[n], got[n][k])
    eng.finish(), other.finish()
    alone = [torch.zeros(made[0][2], device="cuda") for _ in x]
    torch.cuda.synchronize()
    for n in range(2):
        made[0][3](x[n], alone[n])
    eng.finish()
    for n in range(2):
        assert all(torch.equal(y, alone[n]) for y in got[n])
        made[n][0].close()
    other.close()


def test_operands_in_pinned_memory(eng):
    x = random(generator(1), 5, 200, dtype="f16")
    q, s = torch.empty(5, 200, dtype=torch.int8).pin_memory(), torch.empty(5).pin_memory()
    op = ops_s8.Quantize(eng, ops_s8.quantize_desc(5, 200, "f16"))
    run(eng, op, x.pin_memory(), q, s)
    same_rows(q, s, x.float())
    with pytest.raises(hip.HipError) as err:
        op.enqueue(x, q, s)
    assert err.value.status == INVALID_ARG
    op.close()
