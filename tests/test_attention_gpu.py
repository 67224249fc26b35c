"""Attention over image tokens against the formula in 64 bits."""
import math

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


def reference(q, k, v, scale, lengths, bias, dtype):
    """values and what one rounding of each probability, 32-bit scores and one rounding of the result may be off"""
    b, lq, h, d = q.shape
    lk, kv = k.shape[1], k.shape[2]
    want, bound = torch.zeros(b, lq, h, d, dtype=torch.float64), torch.zeros(b, lq, h, d, dtype=torch.float64)
    for i in range(b):
        n = lk if lengths is None else max(0, min(lk, int(lengths[i])))
        for j in range(h if n else 0):
            g = j // (h // kv)
            qd, kd, vd = q[i, :, j].double(), k[i, :n, g].double(), v[i, :n, g].double()
            s = qd @ kd.T * scale
            size = qd.abs() @ kd.abs().T * abs(scale)
            if bias is not None:
                at = bias[i if bias.shape[0] > 1 else 0, j if bias.shape[1] > 1 else 0].double()
                s = s + at[:, :n]
                size = size + torch.where(torch.isinf(at[:, :n]), torch.zeros_like(size), at[:, :n].abs())
            top = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
            total = p.sum(1, keepdim=True)
            p = p / torch.where(total == 0, torch.ones_like(total), total)
            # a score's own roundings, and that of its distance from the maximum, shift its probability and all the others
            score = (d + 4) * EPS * size.amax(1, keepdim=True) + 4 * EPS * (1 + size.amax(1, keepdim=True))
            each = HALF_ULP[dtype] + 4 * score + (n + 8) * EPS
            want[i, :, j] = p @ vd
            bound[i, :, j] = each * (p @ vd.abs()) * 1.1
    return want, bound + HALF_ULP[dtype] * want.abs() * (1 + 2 ** -8) + SMALLEST[dtype]


def check(eng, b, lq, lk, h, kv, d, dtype, *, lengths=None, bias=None, bias_dtype=None, scale=0.0, spare=0, seed=0, spread=1.0, behind=math.nan):
    """spare: elements behind each head, token and batch; `behind`: what lies in memory at and behind the lengths"""
    g = generator(seed + lq + lk + d)
    x = [random(g, b, n, heads, d, dtype=dtype, scale=s) for n, heads, s in ((lq, h, spread), (lk, kv, spread), (lk, kv, 1.0))]
    dev, strides = [], []
    for n, (t, length, heads) in enumerate(zip(x + [x[0]], (lq, lk, lk, lq), (h, kv, kv, h))):
        head = d + spare
        token = heads * head + spare
        batch = length * token + spare
        full = torch.full((b, batch), math.nan, dtype=t.dtype)
        inner = torch.as_strided(full, (b, length, heads, d), (batch, token, head, 1))
        if n < 3:
            inner.copy_(t)
        if n in (1, 2) and lengths is not None:
            for i in range(b):
                inner[i, max(0, min(lk, int(lengths[i]))):] = behind
        whole, view = framed(full, 8)
        dev.append((whole, view, torch.as_strided(view, (b, length, heads, d), (batch, token, head, 1), view.storage_offset())))
        strides.append((batch, token, head))
    dl = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    op = ops.Attention(eng, ops.attention_desc(b, lq, lk, h, kv, d, dtype, scale=scale, key_lengths=lengths is not None, bias_dtype=bias_dtype,
                                               bias_shape=None if bias is None else tuple(bias.shape), q_strides=strides[0], k_strides=strides[1], v_strides=strides[2],
                                               out_strides=strides[3]))
    db = None if bias is None else bias.cuda()
    run(eng, op, dev[0][2], dev[1][2], dev[2][2], dev[3][2], dl, db)
    got = dev[3][2].cpu()
    want, bound = reference(*x, scale if scale else d ** -0.5, lengths, bias, dtype)
    close(got, want, bound, op.info().kernel_name.decode())
    assert int(torch.isnan(dev[3][0]).sum()) == dev[3][0].numel() - got.numel(), "written outside the rows"
    again = dev[3][2].clone()
    run(eng, op, dev[0][2], dev[1][2], dev[2][2], dev[3][2], dl, db)
    assert torch.equal(again, dev[3][2]), "the same call gives other bits"
    op.close()
    return got


SIZES = [  # batch, queries, keys, query heads, key heads
    (1, 1, 1, 1, 1), (2, 1, 7, 4, 1), (1, 49, 49, 4, 4), (2, 33, 65, 3, 3), (1, 196, 196, 2, 2), (3, 5, 1000, 8, 2), (1, 1, 5000, 8, 2), (1, 130, 64, 2, 1), (2, 64, 63, 6, 2),
    (1, 257, 300, 1, 1), (70, 9, 9, 2, 2), (1, 3, 129, 64, 1), (1, 20, 3000, 2, 2),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("head", [32, 64, 80, 128])
def test_sizes(eng, size, head, dtype):
    check(eng, *size, head, dtype)


@pytest.mark.parametrize("head", [8, 16, 24, 40, 48, 56, 72, 88, 96, 104, 112, 120, 136, 152, 160, 168, 192, 200, 248, 256])
@pytest.mark.parametrize("lq,lk", [(37, 70), (1, 260)])
def test_head_sizes(eng, head, lq, lk):
    check(eng, 2, lq, lk, 2, 1, head, "bf16", spare=8)
    check(eng, 1, lq, lk, 2, 2, head, "f16", lengths=[lk - 5])


@pytest.mark.parametrize("lq,lk,h,kv", [(1, 200, 4, 2), (40, 200, 4, 2), (150, 130, 2, 2), (2, 3000, 4, 1)])
@pytest.mark.parametrize("behind", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("head", [64, 72])
def test_lengths(eng, lq, lk, h, kv, behind, head):
    lengths = [0, 1, 63, 64, 65, lk - 1, lk, lk + 5, -3, lk // 2]
    got = check(eng, len(lengths), lq, lk, h, kv, head, "f16", lengths=lengths, behind=behind)
    assert (got[0] == 0).all() and (got[8] == 0).all()


@pytest.mark.parametrize("bias_dtype", ["f16", "f32"])
@pytest.mark.parametrize("shape", [(1, 4, 50, 70), (3, 1, 1, 70), (3, 4, 50, 70), (1, 1, 50, 70), (1, 1, 1, 70)], ids=str)
@pytest.mark.parametrize("ragged", [False, True])
def test_bias(eng, shape, bias_dtype, ragged):
    g = generator(3)
    bias = random(g, *shape, scale=2.0, dtype=bias_dtype)
    check(eng, 3, 50, 70, 4, 2, 64, "f16", bias=bias, bias_dtype=bias_dtype, lengths=[70, 0, 33] if ragged else None)


@pytest.mark.parametrize("lq,lk", [(40, 150), (1, 2000), (3, 64)])
def test_masks_that_leave_rows_empty(eng, lq, lk):
    g = generator(4)
    bias = random(g, 2, 2, lq, lk, dtype="bf16")
    bias[0, 0, 0] = -math.inf                              # no key at all
    bias[0, 1, :, 1:] = -math.inf                          # one key
    bias[1, 0, lq // 2:, :lk // 2 + 1] = -math.inf         # the first tiles empty
    bias[1, 1] = torch.finfo(torch.bfloat16).min           # the lowest value: all the same
    got = check(eng, 2, lq, lk, 2, 2, 32, "bf16", bias=bias, bias_dtype="bf16")
    assert (got[0, 0, 0] == 0).all()


def test_lowest_values_in_f16_and_f32(eng):
    for dt in ("f16", "f32"):
        bias = torch.zeros(1, 1, 9, 80, dtype=TYPES[dt])
        bias[..., 40:] = torch.finfo(TYPES[dt]).min
        bias[0, 0, 3] = torch.finfo(TYPES[dt]).min
        q, k, v = (random(generator(n), 1, 9 if n == 0 else 80, 1, 64, dtype="f16") for n in range(3))
        op = ops.Attention(eng, ops.attention_desc(1, 9, 80, 1, 1, 64, "f16", bias_dtype=dt, bias_shape=tuple(bias.shape)))
        out = torch.empty(1, 9, 1, 64, dtype=torch.float16, device="cuda")
        run(eng, op, q.cuda(), k.cuda(), v.cuda(), out, None, bias.cuda())
        op.close()
        # the softmax of the scores in 32 bits, as the formula has them: in row 3 an f32 bias swallows every score
        s = q[0, :, 0].double() @ k[0, :, 0].double().T / 8 + bias[0, 0].double()
        p = torch.softmax(s if dt == "f16" else s.float().double(), 1)
        want = p @ v[0, :, 0].double()
        # at -65504 a score is a multiple of 2^-8
        slack = 2.0 ** -8 if dt == "f16" else 0.0
        rows = torch.ones(9, 1).double()
        rows[3] = 1 + slack / HALF_ULP["f16"]
        close(out[0, :, 0], want, rows * (4 * HALF_ULP["f16"] + 100 * EPS) * (p @ v[0, :, 0].double().abs()))


@pytest.mark.parametrize("scale", [3.0, -0.5, 1e-3])
@pytest.mark.parametrize("lq", [40, 1])
def test_scales_and_sharp_rows(eng, scale, lq):
    check(eng, 1, lq, 300, 2, 2, 64, "f16", scale=scale, spread=2.0)


@pytest.mark.parametrize("scale", [1e-39, -1e-44, 3e-38, 1e30])
@pytest.mark.parametrize("size", [(1, 40, 300, 2, 2), (1, 1, 2000, 2, 2), (2, 1, 3, 2, 1)], ids=str)
def test_scales_at_the_ends_of_their_range(eng, scale, size):
    # next to nothing: the mean of the values; next to infinite: the value of the largest score
    b, lq, lk, h, kv = size
    g = generator(12)
    q, k, v = (random(g, b, n, heads, 64, dtype="f16") for n, heads in ((lq, h), (lk, kv), (lk, kv)))
    out = torch.empty(b, lq, h, 64, dtype=torch.float16, device="cuda")
    op = ops.Attention(eng, ops.attention_desc(b, lq, lk, h, kv, 64, "f16", scale=scale))
    run(eng, op, q.cuda(), k.cuda(), v.cuda(), out)
    op.close()
    for i in range(b):
        for j in range(h):
            vd = v[i, :, j * kv // h].double()
            if abs(scale) < 1:
                want, size = vd.mean(0).expand(lq, 64), vd.abs().mean(0)
            else:
                want = vd[(q[i, :, j].double() @ k[i, :, j * kv // h].double().T).argmax(1)]
                size = want.abs()
            close(out[i, :, j], want, 2 * HALF_ULP["f16"] * size + (lk + 8) * EPS * size + SMALLEST["f16"], "scale %g" % scale)


def test_scales_that_32_bits_cannot_turn_into_powers_of_two(eng):
    assert refused(eng, ops.Attention, ops.attention_desc(1, 4, 4, 2, 2, 32, "f16", scale=3e38)) == INVALID_ARG
    assert refused(eng, ops.Attention, ops.attention_desc(1, 4, 4, 2, 2, 32, "f16", scale=-3e38)) == INVALID_ARG
    assert refused(eng, ops.Attention, ops.attention_desc(1, 4, 4, 2, 2, 32, "f16", scale=3e38, bias_shape=(1, 1, 4, 4))) == 0


@pytest.mark.parametrize("lq", [33, 1])
def test_nan_and_infinity_within_the_lengths_count(eng, lq):
    g = generator(8)
    q, k, v = (random(g, 1, n, 2, 64, dtype="f16") for n in (lq, 90, 90))
    v[0, 40, 0, 5] = math.nan
    k[0, 41, 1, 0] = math.nan
    out = torch.empty(1, lq, 2, 64, dtype=torch.float16, device="cuda")
    op = ops.Attention(eng, ops.attention_desc(1, lq, 90, 2, 2, 64, "f16"))
    run(eng, op, q.cuda(), k.cuda(), v.cuda(), out)
    op.close()
    bad = torch.isnan(out.cpu())
    want = torch.zeros_like(bad)
    want[0, :, 0, 5] = True
    want[0, :, 1] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("size,head,kernel", [
    ((6, 512, 100, 16, 16), 64, "<64,8 waves>"), ((6, 512, 70, 16, 8), 128, "<128,8 waves>"), ((4, 1030, 130, 4, 4), 104, "<128,4 waves>"), ((6, 512, 70, 16, 16), 120, "<128,8 waves>"), ((4, 1030, 130, 4, 4), 32, "<32,4 waves>"),
    ((2, 1030, 65, 8, 8), 160, "<160,4 waves>"), ((1, 30, 1000, 2, 2), 200, "<256,4 waves,split keys>"), ((1, 30, 1000, 2, 2), 96, "<96,1 wave,split keys>"), ((1, 1, 200, 2, 2), 64, "<64,1 wave>")], ids=str)
def test_every_kernel(eng, size, head, kernel):
    b, lq, lk, h, kv = size
    op = ops.Attention(eng, ops.attention_desc(b, lq, lk, h, kv, head, "bf16", key_lengths=True))
    assert op.info().kernel_name.decode() == "attention" + kernel
    op.close()
    check(eng, *size, head, "bf16", lengths=[lk - 7 * i for i in range(b)])


def test_keys_too_far_apart_for_32_bits_within_a_tile(eng):
    # 2^24 elements from key to key, as many rows as share tiles between four waves
    lq, lk, d, pitch = 16400, 70, 32, 1 << 24
    g = generator(19)
    q, k, v = (random(g, 1, n, 1, d, dtype="bf16") for n in (lq, lk, lk))
    far = torch.empty(2, (lk - 1) * pitch + 64, dtype=torch.bfloat16, device="cuda")
    for i in range(lk):
        far[0, i * pitch:i * pitch + d], far[1, i * pitch:i * pitch + d] = k[0, i, 0].cuda(), v[0, i, 0].cuda()
    out = torch.empty(1, lq, 1, d, dtype=torch.bfloat16, device="cuda")
    op = ops.Attention(eng, ops.attention_desc(1, lq, lk, 1, 1, d, "bf16", k_strides=(0, pitch, d), v_strides=(0, pitch, d)))
    assert "4 waves,far" in op.info().kernel_name.decode()
    run(eng, op, q.cuda(), far[0], far[1], out)
    op.close()
    close(out, *reference(q, k, v, d ** -0.5, None, None, "bf16"))


@pytest.mark.parametrize("lq", [2, 40])
def test_offsets_past_32_bits(eng, lq):
    # tokens 2^30 elements apart: the last of 5 starts 8 GiB in
    lk, d, pitch = 5, 32, 1 << 30
    g = generator(9)
    q, k, v = random(g, 1, lq, 1, d, dtype="f16"), random(g, 1, lk, 1, d, dtype="f16"), random(g, 1, lk, 1, d, dtype="f16")
    far = torch.empty(2, (lk - 1) * pitch + 64, dtype=torch.float16, device="cuda")
    for i in range(lk):
        far[0, i * pitch:i * pitch + d], far[1, i * pitch:i * pitch + d] = k[0, i, 0].cuda(), v[0, i, 0].cuda()
    out = torch.empty(1, lq, 1, d, dtype=torch.float16, device="cuda")
    op = ops.Attention(eng, ops.attention_desc(1, lq, lk, 1, 1, d, "f16", k_strides=(0, pitch, d), v_strides=(0, pitch, d)))
    run(eng, op, q.cuda(), far[0], far[1], out)
    op.close()
    close(out, *reference(q, k, v, d ** -0.5, None, None, "f16"))


def test_a_recording_is_replayed(eng):
    g = generator(10)
    q, k, v = (random(g, 1, n, 4, 64, dtype="bf16").cuda() for n in (1, 4000, 4000))
    want, got = torch.empty_like(q), torch.zeros_like(q)
    op = ops.Attention(eng, ops.attention_desc(1, 1, 4000, 4, 4, 64, "bf16"))
    run(eng, op, q, k, v, want)
    L, rec = hip.lib(), hip.C.c_void_p()
    hip.check(L.cldnn_hip_engine_record_begin(eng.h))
    op.enqueue(q, k, v, got)
    hip.check(L.cldnn_hip_engine_record_end(eng.h, hip.C.byref(rec)))
    for _ in range(3):
        got.zero_()
        torch.cuda.synchronize()
        hip.check(L.cldnn_hip_recording_enqueue(rec))
        eng.finish()
        assert torch.equal(got, want)
    hip.check(L.cldnn_hip_recording_release(rec))
    op.close()


def test_refusals(eng):
    def status(*args, **kw):
        return refused(eng, ops.Attention, ops.attention_desc(*args, **kw))

    assert status(1, 4, 4, 2, 2, 32, "f16") == 0
    for i in range(6):
        sizes = [1, 4, 4, 2, 2, 32]
        sizes[i] = 0
        assert status(*sizes, "f16") == INVALID_ARG
    assert status(1, 4, 4, 3, 2, 32, "f16") == DIMENSION_MISMATCH
    assert status(1, 4, 4, 2, 2, 32, "f32") == INVALID_ARG
    assert status(1, 4, 4, 2, 2, 36, "f16") == status(1, 4, 4, 2, 2, 264, "f16") == UNSUPPORTED_SIZE
    assert status(1, 4, 4, 2, 2, 32, "f16", k_strides=(0, 68, 0)) == UNSUPPORTED_FORMAT
    assert status(1, 4, 4, 2, 2, 32, "f16", v_strides=(0, -64, 0)) == INVALID_ARG
    assert status(1, 4, 4, 2, 2, 32, "f16", scale=math.inf) == status(1, 4, 4, 2, 2, 32, "f16", scale=math.nan) == INVALID_ARG
    assert status(1, 4, 4, 2, 2, 32, "f16", bias_dtype="bf16", bias_shape=(1, 1, 4, 4)) == INVALID_ARG
    with pytest.raises(ValueError):
        ops.attention_desc(1, 4, 4, 2, 2, 32, "f16", bias_shape=(1, 2, 3, 4))
    op = ops.Attention(eng, ops.attention_desc(1, 4, 4, 2, 2, 32, "f16", key_lengths=True, bias_shape=(1, 1, 4, 4)))
    x = torch.zeros(256, dtype=torch.float16, device="cuda")
    for i in range(6):
        args = [x] * 6
        args[i] = None
        with pytest.raises(hip.HipError) as err:
            op.enqueue(*args)
        assert err.value.status == INVALID_ARG
    for i in range(4):
        args = [x] * 6
        args[i] = x.data_ptr() + 8
        with pytest.raises(hip.HipError) as err:
            op.enqueue(*args)
        assert err.value.status == INVALID_ARG
    op.close()
