"""Matrix product of int8 operands with scales against the formula in 64 bits, where the sums are exact."""
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


def integers(g, *shape):
    return torch.randint(-128, 128, shape, generator=g).to(torch.int8)


def check(eng, m, n, k, *, out="f32", bias=True, residual=None, act="none", am=0.0, an=0.0, act2="none", a2m=0.0, a2n=0.0, a_scales="each", w_scales="each", spare=(0, 0, 0, 0),
          offsets=(0, 0, 0, 0), in_place=False, seed=0):
    """spare: elements between rows of a, weights, output and residual; offsets: of their starts"""
    g = generator(seed + m + 3 * n + 7 * k)

    def matrix(values, extra, offset, fill):
        full = torch.full((values.shape[0], values.shape[1] + extra), fill, dtype=values.dtype)
        full[:, :values.shape[1]] = values
        return framed(full, offset, fill=fill)

    a, w = integers(g, m, k), integers(g, n, k)

    def scales(kind, rows, size):
        if kind is None:
            return None, torch.ones(1)
        s = (random(g, rows if kind == "each" else 1).exp() * size).float()
        return s.cuda(), s

    dsa, sa = scales(a_scales, m, 1 / 73)
    dsw, sw = scales(w_scales, n, k ** -0.5 / 73)
    b = random(g, n, scale=0.5) if bias else None
    r = random(g, m, n, dtype=residual) if residual else None
    _, da = matrix(a, spare[0], offsets[0], 55)
    _, dw = matrix(w, spare[1], offsets[1], -77)
    if in_place:
        assert residual == out
        keep_o, do = matrix(r, spare[2], offsets[2], math.nan)
        dr, spare = do, (spare[0], spare[1], spare[2], spare[2])
    else:
        keep_o, do = matrix(torch.zeros(m, n, dtype=TYPES[out]), spare[2], offsets[2], math.nan)
        dr = matrix(r, spare[3], offsets[3], math.nan)[1] if residual else None
    before = do.clone()
    op = ops_s8.MatmulS8(eng, ops_s8.matmul_s8_desc(m, n, k, out_dtype=out, a_scales=a_scales, weights_scales=w_scales, bias=bias, residual=bool(residual), residual_dtype=residual,
                                                    act=act, act_m=am, act_n=an, residual_act=act2, residual_act_m=a2m, residual_act_n=a2n, a_stride=k + spare[0],
                                                    weights_stride=k + spare[1], out_stride=n + spare[2], residual_stride=n + spare[3]))
    db = None if b is None else b.cuda()
    run(eng, op, da, dw, do, dsa, dsw, db, dr)
    # between the rows and around the matrix nothing is written
    assert torch.isnan(do[:, n:]).all() and untouched(keep_o, offsets[2], do.numel(), math.nan)
    v = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    # the sum is exact; it, two products and the sum with the bias are rounded once each
    bound = 3 * U * v.abs()
    if b is not None:
        v = v + b.double()
        bound = bound + U * v.abs()
    want = act64(v, act, am, an)
    bound = STEEPEST * max(1.0, abs(am)) * bound * (1 + U * 8) + act_error(v)
    if r is not None:
        v = want + r.double()
        want = act64(v, act2, a2m, a2n)
        bound = STEEPEST * (bound + EPS * v.abs()) + act_error(v)
    close(do[:, :n], want, bound + HALF_ULP[out] * want.abs() * (1 + 2 ** -8) + SMALLEST[out], info(op))
    first = do.clone()
    do.copy_(before)
    run(eng, op, da, dw, do, dsa, dsw, db, dr)
    assert torch.equal(first[:, :n], do[:, :n]), "the same call gives other bits"
    op.close()


def info(op):
    return op.info().kernel_name.decode()


SIZES = [  # m, n, k
    (1, 1, 1), (1, 1000, 2048), (2, 3, 5), (1, 33, 4100), (16, 512, 1600), (17, 64, 8), (33, 100, 72), (49, 108, 84), (64, 64, 64), (65, 65, 65), (100, 1000, 528),
    (128, 128, 128), (129, 257, 136), (196, 1024, 272), (255, 255, 255), (256, 256, 256), (300, 700, 96), (512, 256, 1040), (1395, 108, 84), (2000, 40, 32),
    (784, 520, 48), (1000, 1000, 200), (40, 40, 16384), (1300, 1300, 80), (3, 20, 131071), (70, 300, 15), (70, 300, 17),
]


@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(eng, size, out):
    check(eng, *size, out=out, act="relu", residual=out)


@pytest.mark.parametrize("out,residual", [("f32", None), ("f32", "f16"), ("f16", "f32"), ("bf16", "f16"), ("f16", "bf16"), ("bf16", "f32"), ("bf16", None)])
@pytest.mark.parametrize("size", [(5, 70, 96), (150, 300, 128), (600, 520, 192), (9, 30, 20000)], ids=str)
def test_types(eng, size, out, residual):
    check(eng, *size, out=out, residual=residual, bias=False)


@pytest.mark.parametrize("a_scales", [None, "one", "each"])
@pytest.mark.parametrize("w_scales", [None, "one", "each"])
@pytest.mark.parametrize("size", [(5, 70, 96), (150, 300, 128), (1100, 1030, 64), (9, 30, 20000)], ids=str)
def test_scales(eng, size, a_scales, w_scales):
    check(eng, *size, a_scales=a_scales, w_scales=w_scales, bias=False)


@pytest.mark.parametrize("act,m,n", [("none", 0, 0), ("relu", 0, 0), ("relu_slope", 0.1, 0), ("clamp", -0.5, 0.75), ("silu", 0, 0), ("gelu", 0, 0), ("gelu_tanh", 0, 0)])
@pytest.mark.parametrize("size", [(3, 50, 40), (300, 280, 64)], ids=str)
def test_activations(eng, size, act, m, n):
    check(eng, *size, act=act, am=m, an=n)
    check(eng, *size, out="bf16", act="none", residual="bf16", act2=act, a2m=m, a2n=n)


@pytest.mark.parametrize("spare,offsets", [((16, 16, 8, 8), (16, 16, 8, 8)), ((1, 3, 5, 7), (0, 0, 0, 0)), ((0, 0, 0, 0), (1, 3, 5, 7)), ((4, 8, 1, 4), (8, 4, 1, 1))])
@pytest.mark.parametrize("size", [(7, 90, 104), (200, 168, 80), (520, 640, 272), (24, 40, 1040)], ids=str)
def test_strides_and_alignment(eng, size, spare, offsets):
    check(eng, *size, out="bf16", act="silu", residual="bf16", spare=spare, offsets=offsets)


@pytest.mark.parametrize("size", [(7, 90, 104), (300, 280, 64), (16, 256, 2048)], ids=str)
def test_residual_in_the_output(eng, size):
    check(eng, *size, out="f16", residual="f16", act2="relu", in_place=True)
    check(eng, *size, out="f32", residual="f32", in_place=True, spare=(0, 0, 3, 0))


@pytest.mark.parametrize("size", [(4, 40, 64), (300, 300, 96)], ids=str)
def test_scales_that_are_no_number_stay_in_their_rows(eng, size):
    m, n, k = size
    g = generator(3)
    sa, sw = torch.ones(m), torch.ones(n)
    sa[1], sw[7] = math.nan, math.nan
    out = torch.empty(m, n, dtype=torch.float16, device="cuda")
    op = ops_s8.MatmulS8(eng, ops_s8.matmul_s8_desc(m, n, k, out_dtype="f16"))
    run(eng, op, (integers(g, m, k) // 64).cuda(), (integers(g, n, k) // 64).cuda(), out, sa.cuda(), sw.cuda())
    want = torch.zeros(m, n, dtype=torch.bool)
    want[1], want[:, 7] = True, True
    assert torch.equal(torch.isnan(out.cpu()), want) and torch.isfinite(out.cpu()[~want]).all()
    op.close()


KERNELS = [
    ((4090, 4093, 144), "tile<256x256>"), ((7160, 2042, 272), "tile<224x256>"), ((6130, 2046, 64), "tile<192x256>"), ((4090, 4092, 144), "walk<256x256>"), ((7160, 2040, 272), "walk<224x256>"), ((6130, 2044, 64), "walk<192x256>"), ((3100, 1537, 208), "tile<128x128>"),
    ((1601, 1000, 112), "tile<64x128>"), ((1001, 1000, 272), "tile<64x64,k2>"), ((190, 2000, 528), "tile<32x64,k4>"), ((30, 1000, 1000), "split<16x16>"),
    ((16, 4200, 4096), "tile<32x64,k4>"), ((8, 4200, 4096), "split<16x16>"), ((13, 4200, 4160), "tile<32x64,k4>"), ((16, 4200, 2112), "split<16x16>"),
    ((7, 250, 18000), "split<16x16> + matmul_join"), ((1, 31, 16383), "split<16x16> + matmul_join"), ((20, 65, 18200), "split<16x16> + matmul_join"),
    ((1001, 1000, 255), "tile<64x64,k2>"), ((600, 500, 63), "split<32x32>"), ((1601, 1400, 61), "split<64x64>"), ((1601, 1000, 263), "tile<64x128>"), ((3101, 1700, 263), "tile<128x128>")]


@pytest.mark.parametrize("size,kernel", KERNELS, ids=str)
def test_every_kernel(eng, size, kernel):
    m, n, k = size
    op = ops_s8.MatmulS8(eng, ops_s8.matmul_s8_desc(m, n, k, bias=True, residual=True))
    assert kernel in info(op) and op.info().launches == (2 if k % 16 and ("tile" in kernel or "walk" in kernel) or "join" in kernel else 1), info(op)
    op.close()
    half = "f16" if m % 2 else "bf16"
    if "walk" in kernel:  # several tiles to a workgroup, each with its last rows and features; f32 results of runs of 4, others of 8
        check(eng, m, n, k, out="f32", act="gelu", bias=False)
        check(eng, m, n, k, out="f32", act="silu", residual=half, act2="relu")
        check(eng, m, n // 8 * 8, k, out=half, act="gelu")
        check(eng, m, n // 8 * 8, k, out=half, residual="f32", spare=(0, 0, 8, 8), a_scales="one", w_scales=None, in_place=False)
        check(eng, m, n // 8 * 8, k, out=half, act="relu", residual=half, in_place=True)
        check(eng, m, n // 8 * 8, k, out=half, act="relu", offsets=(0, 0, 1, 0))
    check(eng, m, n, k, out=half, act="gelu", residual=half)
    if "join" in kernel:
        check(eng, m, n, k, out="f32", act="relu", residual="f32", act2="silu", in_place=True)
        check(eng, m, n, k, out="bf16", bias=False, spare=(1, 0, 3, 0), offsets=(1, 3, 0, 0))


def test_pointers_that_are_not_aligned(eng):
    # the description allows the tile kernels, the pointers do not
    for size in ((300, 280, 64), (700, 600, 80)):
        check(eng, *size, out="f16", act="silu", offsets=(1, 0, 0, 0))
        check(eng, *size, out="f16", act="silu", offsets=(16, 3, 1, 0))


def test_offsets_past_32_bits(eng):
    m, n, k, pitch = 3, 33, 48, (1 << 32) + 48
    g = generator(4)
    a, w = integers(g, m, k), integers(g, n, k)
    far = torch.empty((m - 1) * pitch + 64, dtype=torch.int8, device="cuda")
    out = torch.empty((m - 1) * (1 << 31) + 64, dtype=torch.float32, device="cuda")
    for i in range(m):
        far[i * pitch:i * pitch + k] = a[i].cuda()
    op = ops_s8.MatmulS8(eng, ops_s8.matmul_s8_desc(m, n, k, a_scales=None, weights_scales=None, a_stride=pitch, out_stride=1 << 31))
    run(eng, op, far, w.cuda(), out)
    got = torch.stack([out[i << 31:(i << 31) + n] for i in range(m)])
    assert torch.equal(got.cpu().double(), a.double() @ w.double().T)
    op.close()


@pytest.mark.parametrize("size", [s for s, _ in KERNELS] + [(1, 40, 131071), (16, 128, 131056), (300, 300, 65536)], ids=str)
def test_sums_are_exact(eng, size):
    """the largest that 8 bits give, of one sign: no sum may be held in fewer than 32 bits; and any, at any length of K"""
    m, n, k = size
    g = generator(sum(size))
    op = ops_s8.MatmulS8(eng, ops_s8.matmul_s8_desc(m, n, k, a_scales=None, weights_scales=None))
    out = torch.full((m, n), math.nan, device="cuda")
    for a, w in ((torch.full((m, k), -128, dtype=torch.int8), torch.full((n, k), -128, dtype=torch.int8)), (integers(g, m, k), integers(g, n, k))):
        a, w = a.cuda(), w.cuda()
        run(eng, op, a, w, out)
        want = a.double() @ w.double().T  # at most 2^31: exact
        assert torch.equal(out, want.float())
    op.close()


def test_refusals(eng):
    def status(*args, **kw):
        return refused(eng, ops_s8.MatmulS8, ops_s8.matmul_s8_desc(*args, **kw))

    assert status(4, 4, 4) == status(1, 1, 131071) == 0
    for sizes in ((0, 4, 4), (4, -1, 4), (4, 4, 0)):
        assert status(*sizes) == INVALID_ARG
    assert status(1, 1, 131072) == status((1 << 31) - 1, 8, 8) == status(8, (1 << 31) - 200, 8) == UNSUPPORTED_SIZE
    assert status(4, 4, 4, out_dtype="s8") == status(4, 4, 4, out_dtype="i32") == status(4, 4, 4, residual=True, residual_dtype="s8") == INVALID_ARG
    assert status(4, 4, 4, residual_act="relu") == INVALID_ARG
    assert status(4, 4, 4, a_scales=3) == status(4, 4, 4, weights_scales=-1) == INVALID_ARG
    assert status(4, 4, 4, act=77) == status(4, 4, 4, act=-1) == INVALID_ARG
    for stride in ("a_stride", "weights_stride", "out_stride", "residual_stride"):
        assert status(4, 4, 4, **{stride: 3}) == status(4, 4, 4, **{stride: -8}) == INVALID_ARG
