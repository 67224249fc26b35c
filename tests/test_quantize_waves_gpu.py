"""Rows to int8 where there are enough of them for a wave to each: 16-bit rows of 2049 to 4096 values, in six and in eight vectors a lane."""
import pytest
import torch

from cldnn_amd import hip
from operator_s8_cases import *
from test_quantize_gpu import quantize

pytestmark = pytest.mark.gpu

# the least and the most of each shape, and last vectors that lie over the one before them
WIDTHS = [(2049, "quantize<64x6>"), (2500, "quantize<64x6>"), (3071, "quantize<64x6>"), (3073, "quantize<64x8>"), (3588, "quantize<64x8>"), (4093, "quantize<64x8>"), (4096, "quantize<64x8>")]


@pytest.fixture(scope="module")
def eng():
    e = hip.Engine()
    yield e
    e.close()


@pytest.fixture(scope="module")
def rows():
    """more than 16 to a CU, and no whole workgroups of four"""
    return 16 * torch.cuda.get_device_properties(0).multi_processor_count + 3


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("features,kernel", WIDTHS)
def test_rows(eng, rows, features, kernel, dtype):
    x = random(generator(features), rows, features, dtype=dtype)
    q, scales, name = quantize(eng, x, features)
    assert name == kernel
    same_rows(q, scales, x.float(), name)
    q, scales, name = quantize(eng, x, features, in_spare=3, out_spare=5, in_offset=1, out_offset=3)
    assert name == kernel
    same_rows(q, scales, x.float(), name)


@pytest.mark.parametrize("features,kernel", WIDTHS)
def test_factors_and_gates(eng, rows, features, kernel):
    g = generator(features)
    factors = random(g, features).abs() + 0.1
    both = random(g, rows, 2 * features, dtype="f16")
    x, gate = both[:, :features], both[:, features:]
    q, scales, name = quantize(eng, x, features, factors=factors)
    assert name == kernel
    same_rows(q, scales, x.float() * factors, name)
    q, scales, name = quantize(eng, both, features, gated=True, factors=factors, out_spare=1)
    assert name == kernel
    same_rows(q, scales, x.float() * gate.float() * factors, name)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("features,kernel", WIDTHS)
def test_activations(eng, rows, features, kernel, act):
    x = random(generator(features + 1), rows, features, dtype="f16")
    q, scales, name = quantize(eng, x, features, act=act)
    assert name == kernel
    v = x.double()
    near_rows(q, scales, act64(v, act), act_error(v), name)


def test_rows_of_no_value_and_of_what_is_no_number(eng, rows):
    for features, kernel in WIDTHS[1::3]:
        x = random(generator(1), rows, features, dtype="bf16")
        x[0], x[5, features - 1], x[rows - 1, 7], x[rows - 2, 2048] = 0, float("nan"), float("inf"), 60000.0
        q, scales, name = quantize(eng, x, features)
        assert name == kernel
        same_rows(q, scales, x.float(), name)
