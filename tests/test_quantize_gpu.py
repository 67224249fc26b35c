"""Rows to int8 with a scale each: the bits that the definition gives where 32 bits hold the values, and against the formula in 64
bits where an activation comes first."""
import math

import pytest
import torch

from cldnn_amd import hip, ops_s8
from operator_s8_cases import *

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = hip.Engine()
    yield e
    e.close()


def quantize(eng, x, features, *, act="none", am=0.0, an=0.0, gated=False, factors=None, in_spare=0, out_spare=0, in_offset=0, out_offset=0):
    """x: CPU rows, as they are in memory"""
    rows, width = x.shape
    dtype = {v: k for k, v in TYPES.items()}[x.dtype]
    full = torch.full((rows, width + in_spare), math.nan, dtype=x.dtype)
    full[:, :width] = x
    _, src = framed(full, in_offset)
    keep, dst = framed(torch.full((rows, features + out_spare), 77, dtype=torch.int8), out_offset, fill=77)
    keep_s, scales = framed(torch.zeros(rows))
    op = ops_s8.Quantize(eng, ops_s8.quantize_desc(rows, features, dtype, act=act, act_m=am, act_n=an, gated=gated, factors=factors is not None,
                                                   in_stride=width + in_spare, out_stride=features + out_spare))
    df = None if factors is None else factors.float().cuda()
    run(eng, op, src, dst, scales, df)
    assert untouched(keep, out_offset, dst.numel(), 77) and (dst[:, features:] == 77).all() and untouched(keep_s, 0, rows, math.nan)
    first = dst.clone()
    run(eng, op, src, dst, scales, df)
    assert torch.equal(first, dst), "the same call gives other bits"
    name = op.info().kernel_name.decode()
    op.close()
    return dst[:, :features], scales, name


ROWS = [(1, 1), (1, 7), (3, 8), (17, 84), (5, 127), (64, 128), (33, 129), (9, 500), (12, 512), (7, 513), (130, 1000), (300, 1024), (4, 1500), (3, 2047), (2, 2048), (5, 3000), (2, 4096),
        (3, 5000), (2, 8192), (2, 9001), (1, 16384), (2, 20001), (1, 25088), (1, 32768), (3, 32769), (2, 40000), (1, 131071)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", ROWS, ids=str)
def test_rows(eng, size, dtype):
    rows, features = size
    x = random(generator(features), rows, features, dtype=dtype)
    q, scales, name = quantize(eng, x, features)
    assert ("far" in name) == (features > 32768)
    same_rows(q, scales, x.float(), name)


@pytest.mark.parametrize("spare,offset", [((0, 0), (1, 1)), ((3, 1), (0, 0)), ((8, 16), (8, 8)), ((1, 5), (3, 7))])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [(37, 84), (6, 640), (3, 2500), (2, 33000)], ids=str)
def test_strides_and_alignment(eng, size, dtype, spare, offset):
    x = random(generator(3), *size, dtype=dtype)
    q, scales, name = quantize(eng, x, size[1], in_spare=spare[0], out_spare=spare[1], in_offset=offset[0], out_offset=offset[1])
    same_rows(q, scales, x.float(), name)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("size", [(21, 90), (5, 777), (3, 3100), (2, 10001), (2, 33333)], ids=str)
def test_factors_and_gates(eng, size, dtype):
    rows, features = size
    g = generator(5)
    factors = random(g, features).abs() + 0.1
    x, gate = random(g, rows, features, dtype=dtype), random(g, rows, features, dtype=dtype)
    q, scales, name = quantize(eng, x, features, factors=factors)
    same_rows(q, scales, (x.float() * factors), name)
    both = torch.cat([x, gate], 1)
    q, scales, name = quantize(eng, both, features, gated=True)
    same_rows(q, scales, x.float() * gate.float(), name)
    q, scales, name = quantize(eng, both, features, gated=True, factors=factors, in_spare=5)
    same_rows(q, scales, x.float() * gate.float() * factors, name)


@pytest.mark.parametrize("act,m,n", [("relu", 0, 0), ("relu_slope", 0.1, 0), ("clamp", 0.5, 0.75), ("silu", 0, 0), ("gelu", 0, 0), ("gelu_tanh", 0, 0)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("size", [(40, 84), (7, 1111), (3, 33001)], ids=str)
def test_activations(eng, size, act, m, n, gated):
    rows, features = size
    g = generator(7)
    x = random(g, rows, features * (2 if gated else 1), dtype="bf16")
    q, scales, name = quantize(eng, x, features, act=act, am=m, an=n, gated=gated)
    v = x[:, :features].double()
    y, error = act64(v, act, m, n), act_error(v)
    if gated:
        other = x[:, features:].double()
        y, error = y * other, error * other.abs() + U * (y * other).abs()
    near_rows(q, scales, y, error, name)


def test_rows_of_no_value_and_of_what_is_no_number(eng):
    big, tiny = 3.3e38, 2.0 ** -119
    rows = torch.zeros(12, 200)
    rows[1, 5], rows[2, 5], rows[3, 199], rows[4, 0] = math.nan, math.inf, -math.inf, big
    rows[5, 7], rows[6, 7], rows[7, 7] = tiny, 2.0 ** -121, 1e-44
    rows[8], rows[9], rows[10, 3] = -0.0, -1.0, -5.5
    rows[11] = torch.arange(200) - 100.0
    rows[1, 6] = 3.0
    q, scales, _ = quantize(eng, rows, 200)
    same_rows(q, scales, rows)
    assert scales[0] == 0 and not q[0].any() and torch.isnan(scales[1:4]).all() and not q[1:4].any() and not q[6:8].any() and q[9].eq(-127).all()
    far = torch.zeros(4, 33000)
    far[0, 32999], far[1, 1], far[2, 5] = math.nan, 7.0, 2.0 ** -121
    q, scales, _ = quantize(eng, far, 33000)
    same_rows(q, scales, far)


def test_ties_go_to_even(eng):
    # most = 127: a step is 1, and its halves are ties
    x = torch.cat([torch.tensor([127.0]), torch.arange(-126, 127) + 0.5])[None].repeat(3, 1)
    q, scales, _ = quantize(eng, x, x.shape[1])
    assert torch.equal(q.cpu().float(), torch.round(x)) and (scales == 1).all()
    same_rows(q, scales, x)


@pytest.mark.parametrize("features", [40, 2100])
def test_offsets_past_32_bits(eng, features):
    rows, pitch = 3, 1 << 31
    x = random(generator(9), rows, features, dtype="f16")
    src = torch.empty((rows - 1) * pitch + features, dtype=torch.float16, device="cuda")
    dst = torch.empty((rows - 1) * pitch + features, dtype=torch.int8, device="cuda")
    for i in range(rows):
        src[i * pitch:i * pitch + features] = x[i].cuda()
    scales = torch.zeros(rows, device="cuda")
    op = ops_s8.Quantize(eng, ops_s8.quantize_desc(rows, features, "f16", in_stride=pitch, out_stride=pitch))
    run(eng, op, src, dst, scales)
    same_rows(torch.stack([dst[i * pitch:i * pitch + features] for i in range(rows)]), scales, x.float())
    op.close()


def test_refusals(eng):
    def status(*args, **kw):
        return refused(eng, ops_s8.Quantize, ops_s8.quantize_desc(*args, **kw))

    assert status(4, 4, "f16") == 0
    assert status(0, 4, "f16") == status(4, 0, "f16") == status(-1, 4, "f16") == INVALID_ARG
    assert status(4, 4, "i32") == status(4, 4, "s8") == status(4, 4, 77) == INVALID_ARG
    assert status(4, 4, "f16", in_stride=3) == status(4, 4, "f16", out_stride=3) == status(4, 4, "f16", gated=True, in_stride=7) == status(4, 4, "f16", out_stride=-8) == INVALID_ARG
    assert status(4, 4, "f16", act=77) == status(4, 4, "f16", act="clamp", act_m=1.0, act_n=0.0) == INVALID_ARG
    assert status(4, (1 << 31) - 1, "f16") == status(1 << 40, 4, "f16") == status(1 << 30, 5000, "f16") == UNSUPPORTED_SIZE
