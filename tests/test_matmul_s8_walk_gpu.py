"""Int8 products whose workgroups go through several tiles, against the formula in 64 bits: more tiles than CUs, a last round that not all
workgroups have, last rows and features that do not fill their tile, results that go past the caches."""
import math
import re

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


def integers(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def check(eng, m, n, k, kernel, *, out="f32", residual=None, act="none", act2="none", a_scales="each", w_scales="each", bias=True, spare=0, in_place=False):
    """spare: elements between rows of the output and the residual"""
    g = torch.Generator("cuda")
    g.manual_seed(m + 3 * n + 7 * k)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    a, w = integers(g, m, k), integers(g, n, k)
    sa = None if a_scales is None else normal(m if a_scales == "each" else 1).exp() / 73
    sw = None if w_scales is None else normal(n if w_scales == "each" else 1).exp() * k ** -0.5 / 73
    b = normal(n) * 0.5 if bias else None
    op = ops_s8.MatmulS8(eng, ops_s8.matmul_s8_desc(m, n, k, out_dtype=out, a_scales=a_scales, weights_scales=w_scales, bias=bias, residual=bool(residual), residual_dtype=residual,
                                                    act=act, residual_act=act2, out_stride=n + spare, residual_stride=n + spare))
    name, workgroups = op.info().kernel_name.decode(), op.info().grid
    rows, features = map(int, re.match(r"matmul_s8_walk<(\d+)x(\d+)>$", name).groups())
    tiles = -(-m // rows) * -(-n // features)
    assert kernel in name and workgroups < tiles, "%s: %d tiles, %d workgroups" % (name, tiles, workgroups)
    assert tiles % workgroups and m % rows and n % features

    pitch = n + spare
    whole = torch.full((m * pitch + 64,), math.nan, dtype=TYPES[out], device="cuda")
    dst = whole[:m * pitch].view(m, pitch)
    r = dr = None
    if residual:
        r = normal(m, n).to(TYPES[residual])
        dr = dst if in_place else torch.full((m, pitch), math.nan, dtype=TYPES[residual], device="cuda")
        dr[:, :n] = r
    run(eng, op, a, w, dst, sa, sw, b, dr)
    assert torch.isnan(whole[m * pitch:]).all() and torch.isnan(dst[:, n:]).all(), "written outside the rows"

    v = a.double() @ w.double().T
    v *= torch.ones((), device="cuda").double() if sa is None else sa.double()[:, None]
    v *= torch.ones((), device="cuda").double() if sw is None else sw.double()
    # the sum is exact; it, two products and the sum with the bias are rounded once each
    bound = 3 * U * v.abs()
    if b is not None:
        v += b.double()
        bound += U * v.abs()
    want = act64(v, act)
    bound = STEEPEST * bound * (1 + U * 8) + act_error(v)
    if r is not None:
        v = want + r.double()
        want = act64(v, act2)
        bound = STEEPEST * (bound + EPS * v.abs()) + act_error(v)
    bound += HALF_ULP[out] * want.abs() * (1 + 2 ** -8) + SMALLEST[out]
    off = (dst[:, :n].double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d off, the first at %r" % (name, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist())
    first = dst[:, :n].clone()
    if in_place:
        dst[:, :n] = r
    run(eng, op, a, w, dst, sa, sw, b, dr)
    assert torch.equal(dst[:, :n], first), "the same call gives other bits"
    op.close()


# two and three tiles to a workgroup; a step of K, and several; results of 16 bits and of 32 on either side of the 64 MiB from which they
# go past the caches
SIZES = [((12545, 2056, 144), "<256x256>"), ((12545, 2056, 64), "<256x256>"), ((10799, 2056, 272), "<224x256>"), ((7695, 2056, 144), "<192x256>"), ((8180, 2056, 144), "<192x256>"),
         ((7695, 2056, 16), "<192x256>"), ((16401, 2056, 80), "<224x256>")]


@pytest.mark.parametrize("size,kernel", SIZES, ids=str)
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_several_tiles_to_a_workgroup(eng, size, kernel, out):
    check(eng, *size, kernel, out=out, act="gelu")
    check(eng, *size, kernel, out=out, residual=out, act2="relu", in_place=True)
    check(eng, *size, kernel, out=out, residual="f16" if out == "f32" else "f32", act="silu", a_scales="one", w_scales=None, bias=False, spare=8)

