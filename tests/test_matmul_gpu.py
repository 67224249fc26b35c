"""Matrix product with bias, activation and residual against the formula in 64 bits."""
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


def check(eng, m, n, k, dtype, *, out=None, bias=True, residual=None, act="none", am=0.0, an=0.0, act2="none", a2m=0.0, a2n=0.0, spare=(0, 0, 0, 0),
          offsets=(0, 0, 0, 0), in_place=False, seed=0):
    """spare: elements between rows of a, weights, output and residual; offsets: of their starts"""
    g = generator(seed + m + 3 * n + 7 * k)
    out = out or dtype

    def matrix(rows, cols, extra, offset, values):
        full = torch.full((rows, cols + extra), math.nan, dtype=values.dtype)
        full[:, :cols] = values
        whole, view = framed(full, offset)
        return whole, view

    a, w = random(g, m, k, dtype=dtype), random(g, n, k, scale=k ** -0.5, dtype=dtype)
    b = random(g, n, scale=0.5) if bias else None
    r = random(g, m, n, dtype=residual) if residual else None
    keep_a, da = matrix(m, k, spare[0], offsets[0], a)
    keep_w, dw = matrix(n, k, spare[1], offsets[1], w)
    if in_place:
        assert residual == out
        keep_o, do = matrix(m, n, spare[2], offsets[2], r)
        dr, spare = do, (spare[0], spare[1], spare[2], spare[2])
    else:
        keep_o, do = matrix(m, n, spare[2], offsets[2], torch.zeros(m, n, dtype=TYPES[out]))
        dr = matrix(m, n, spare[3], offsets[3], r)[1] if residual else None
    before = do.clone()
    op = ops.Matmul(eng, ops.matmul_desc(m, n, k, dtype, out_dtype=out, bias=bias, residual=bool(residual), residual_dtype=residual, act=act, act_m=am, act_n=an,
                                         residual_act=act2, residual_act_m=a2m, residual_act_n=a2n, a_stride=k + spare[0], weights_stride=k + spare[1],
                                         out_stride=n + spare[2], residual_stride=n + spare[3]))
    db = None if b is None else b.cuda()
    run(eng, op, da, dw, do, db, dr)
    # between the rows and around the matrix nothing is written
    assert torch.isnan(do[:, n:]).all() and untouched(keep_o, offsets[2], do.numel(), math.nan)
    v = a.double() @ w.double().T
    # every one of k sums and of the epilogue's is rounded once, at most at the size of all terms together
    size = a.double().abs() @ w.double().abs().T
    if b is not None:
        v, size = v + b.double(), size + b.double().abs()
    bound = (k + 2) * EPS * size
    want = act64(v, act, am, an)
    bound = STEEPEST * max(1.0, abs(am)) * bound + act_error(v)
    if r is not None:
        v = want + r.double()
        want = act64(v, act2, a2m, a2n)
        bound = STEEPEST * (bound + EPS * v.abs()) + act_error(v)
    close(do[:, :n], want, bound + HALF_ULP[out] * want.abs() * (1 + 2 ** -8) + SMALLEST[out], info(op))
    first = do.clone()
    do.copy_(before)
    run(eng, op, da, dw, do, db, dr)
    assert torch.equal(first[:, :n], do[:, :n]), "the same call gives other bits"
    op.close()


def info(op):
    return op.info().kernel_name.decode()


SIZES = [  # m, n, k
    (1, 1, 1), (1, 1000, 2048), (2, 3, 5), (1, 33, 4100), (16, 512, 1600), (17, 64, 8), (33, 100, 72), (49, 108, 84), (64, 64, 64), (65, 65, 65), (100, 1000, 520),
    (128, 128, 128), (129, 257, 136), (196, 1024, 264), (255, 255, 255), (256, 256, 256), (300, 700, 96), (512, 256, 1032), (1395, 108, 84), (2000, 40, 32),
    (784, 520, 40), (1000, 1000, 200), (40, 40, 16384), (1300, 1300, 72),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(eng, size, dtype):
    check(eng, *size, dtype, act="relu", residual=dtype)


@pytest.mark.parametrize("dtype,out,residual", [("f16", "f32", None), ("bf16", "f32", "f32"), ("f16", "f32", "f16"), ("bf16", "bf16", "f32"), ("f16", "f16", None)])
@pytest.mark.parametrize("size", [(5, 70, 96), (150, 300, 128), (600, 520, 192)], ids=str)
def test_types(eng, size, dtype, out, residual):
    check(eng, *size, dtype, out=out, residual=residual, bias=False)


@pytest.mark.parametrize("act,m,n", [("none", 0, 0), ("relu", 0, 0), ("relu_slope", 0.1, 0), ("clamp", -0.5, 0.75), ("silu", 0, 0), ("gelu", 0, 0), ("gelu_tanh", 0, 0)])
@pytest.mark.parametrize("size", [(3, 50, 40), (300, 280, 64)], ids=str)
def test_activations(eng, size, act, m, n):
    check(eng, *size, "f16", out="f32", act=act, am=m, an=n)
    check(eng, *size, "bf16", act="none", residual="bf16", act2=act, a2m=m, a2n=n)


@pytest.mark.parametrize("spare,offsets", [((8, 8, 8, 8), (8, 8, 8, 8)), ((1, 3, 5, 7), (0, 0, 0, 0)), ((0, 0, 0, 0), (1, 3, 5, 7)), ((4, 2, 1, 4), (2, 4, 1, 1))])
@pytest.mark.parametrize("size", [(7, 90, 104), (200, 168, 80), (520, 640, 264), (24, 40, 1040)], ids=str)
def test_strides_and_alignment(eng, size, spare, offsets):
    check(eng, *size, "bf16", act="silu", residual="bf16", spare=spare, offsets=offsets)


@pytest.mark.parametrize("size", [(7, 90, 104), (300, 280, 64), (16, 256, 2048)], ids=str)
def test_residual_in_the_output(eng, size):
    check(eng, *size, "f16", residual="f16", act2="relu", in_place=True)
    check(eng, *size, "f16", out="f32", residual="f32", in_place=True, spare=(0, 0, 3, 0))


@pytest.mark.parametrize("size", [(4, 40, 64), (300, 300, 96)], ids=str)
def test_nan_and_infinity_stay_in_their_rows(eng, size):
    m, n, k = size
    g = generator(3)
    a, w = random(g, m, k, dtype="f16"), random(g, n, k, dtype="f16")
    a[1, 5], w[7, 3], w[n - 1, k - 1] = math.nan, math.inf, math.nan
    out = torch.empty(m, n, dtype=torch.float16, device="cuda")
    op = ops.Matmul(eng, ops.matmul_desc(m, n, k, "f16"))
    run(eng, op, a.cuda(), w.cuda(), out)
    bad = ~torch.isfinite(out.cpu())
    want = torch.zeros_like(bad)
    want[1], want[:, 7], want[:, n - 1] = True, True, True
    assert torch.equal(bad, want)
    op.close()


@pytest.mark.parametrize("size,kernel", [
    ((4090, 4093, 72), "tile<256x256>"), ((7160, 2040, 136), "tile<224x256>"), ((6130, 2046, 64), "tile<192x256>"), ((3100, 1537, 200), "tile<128x128>"),
    ((1601, 1000, 104), "tile<64x128>"), ((1001, 1000, 264), "tile<64x64,k2>"), ((190, 2000, 520), "tile<32x64,k4>"), ((30, 1000, 1000), "split<16x16>"),
    ((7, 250, 9000), "split<16x16> + matmul_join"), ((1, 31, 16383), "split<16x16> + matmul_join"), ((20, 65, 8200), "split<16x16> + matmul_join"),
    ((1001, 1000, 255), "tile<64x64,k2>"), ((600, 500, 63), "split<32x32>"), ((1601, 1400, 61), "split<64x64>"), ((3101, 1500, 263), "tile<64x128>"), ((3101, 1700, 263), "tile<128x128>")], ids=str)
def test_every_kernel(eng, size, kernel):
    m, n, k = size
    dtype = "f16" if m % 2 else "bf16"
    op = ops.Matmul(eng, ops.matmul_desc(m, n, k, dtype, bias=True, residual=True))
    assert kernel in info(op) and op.info().launches == (2 if k % 8 and "tile" in kernel or "join" in kernel else 1)
    op.close()
    check(eng, m, n, k, dtype, act="gelu", residual=dtype)
    if "join" in kernel:
        check(eng, m, n, k, dtype, out="f32", act="relu", residual="f32", act2="silu", in_place=True)
        check(eng, m, n, k, dtype, bias=False, spare=(1, 0, 3, 0), offsets=(1, 3, 0, 0))


def test_pointers_that_are_not_aligned(eng):
    # the description allows the tile kernels, the pointers do not
    for size in ((300, 280, 64), (700, 600, 72)):
        check(eng, *size, "f16", act="silu", offsets=(1, 0, 0, 0))
        check(eng, *size, "f16", act="silu", offsets=(8, 3, 1, 0))


def test_offsets_past_32_bits(eng):
    # rows 2^31 elements apart: the last of a starts 8 GiB in, that of the output 16 GiB
    m, n, k, pitch = 3, 33, 40, 1 << 31
    g = generator(4)
    a, w = random(g, m, k, dtype="bf16"), random(g, n, k, dtype="bf16")
    far = torch.empty((m - 1) * pitch + 64, dtype=torch.bfloat16, device="cuda")
    out = torch.empty((m - 1) * pitch + 64, dtype=torch.float32, device="cuda")
    for i in range(m):
        far[i * pitch:i * pitch + k] = a[i].cuda()
    op = ops.Matmul(eng, ops.matmul_desc(m, n, k, "bf16", out_dtype="f32", a_stride=pitch, out_stride=pitch))
    run(eng, op, far, w.cuda(), out)
    got = torch.stack([out[i * pitch:i * pitch + n] for i in range(m)])
    want = a.double() @ w.double().T
    close(got, want, (k + 2) * EPS * (a.double().abs() @ w.double().abs().T))
    op.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size,kernel", [
    ((1, 1000, 2048), "split<16x16>"), ((1, 33, 4100), "split<16x16>"), ((3, 40, 1031), "split<16x16>"), ((16, 4096, 25088), "split<16x16>"), ((40, 40, 16384), "join"), ((1, 31, 16383), "join"),
    ((20, 65, 8200), "join"), ((7, 250, 9001), "join"), ((9, 100, 20480), "join"), ((600, 500, 63), "split<32x32>"), ((190, 2000, 2056), "tile<32x64,k4>"), ((1001, 1000, 1992), "tile<64x64,k2>"),
    ((1001, 1000, 2055), "matmul_tile<64x64,k2>"), ((1601, 1000, 1096), "tile<64x128>"), ((3100, 1537, 1064), "tile<128x128>"), ((4090, 4093, 1032), "tile<256x256>"), ((6130, 2046, 1000), "tile<192x256>"),
    ((7160, 2040, 1160), "tile<224x256>")], ids=str)
def test_sums_of_whole_numbers_are_exact(eng, size, kernel, dtype):
    """Whose partial sums all fit 32 bits and do not fit 16: no value of K may be lost, and no sum held in fewer bits, at any length.
    No value is zero, so every k counts."""
    m, n, k = size
    g = generator(sum(size))
    a = torch.randint(1, 4, (m, k), generator=g).to(TYPES[dtype])
    w = torch.tensor([-1, 1, 2, 3])[torch.randint(0, 4, (n, k), generator=g)].to(TYPES[dtype])
    want = a.double() @ w.double().T  # at most 9 k, exact in any order
    assert 9 * k < 1 << 24
    op = ops.Matmul(eng, ops.matmul_desc(m, n, k, dtype, out_dtype="f32"))
    assert kernel in info(op)
    out = torch.full((m, n), math.nan, device="cuda")
    run(eng, op, a.cuda(), w.cuda(), out)
    assert torch.equal(out.cpu().double(), want)
    op.close()
    if k % 8 == 0:  # the kernel for any rows
        op = ops.Matmul(eng, ops.matmul_desc(m, n, k, dtype, out_dtype="f32", a_stride=k + 1))
        far = torch.full((m, k + 1), math.nan, dtype=a.dtype)
        far[:, :k] = a
        out.fill_(math.nan)
        run(eng, op, far.cuda(), w.cuda(), out)
        assert torch.equal(out.cpu().double(), want)
        op.close()


def test_refusals(eng):
    def status(*args, **kw):
        return refused(eng, ops.Matmul, ops.matmul_desc(*args, **kw))

    assert status(4, 4, 4, "f16") == 0
    for sizes in ((0, 4, 4), (4, -1, 4), (4, 4, 0)):
        assert status(*sizes, "f16") == INVALID_ARG
    assert status(4, 4, 4, "f32") == status(4, 4, 4, hip.S8) == INVALID_ARG
    assert status(4, 4, 4, "f16", out_dtype="bf16") == INVALID_ARG
    assert status(4, 4, 4, "f16", residual=True, residual_dtype="bf16") == INVALID_ARG
    assert status(4, 4, 4, "f16", residual_act="relu") == INVALID_ARG
    assert status(4, 4, 4, "f16", act=77) == status(4, 4, 4, "f16", act=-1) == INVALID_ARG
    for stride in ("a_stride", "weights_stride", "out_stride"):
        assert status(4, 4, 4, "f16", **{stride: 3}) == status(4, 4, 4, "f16", **{stride: -8}) == INVALID_ARG
    op = ops.Matmul(eng, ops.matmul_desc(4, 4, 4, "f16", bias=True, residual=True))
    x = torch.zeros(64, dtype=torch.float32, device="cuda")
    for args in ((None, x, x, x, x), (x, None, x, x, x), (x, x, None, x, x), (x, x, x, None, x), (x, x, x, x, None), (x.data_ptr() + 1, x, x, x, x),
                 (x, x, x, x.data_ptr() + 2, x)):
        with pytest.raises(hip.HipError) as err:
            op.enqueue(*args)
        assert err.value.status == INVALID_ARG
    other = ops.GroupNorm(eng, ops.group_norm_desc(ops.map_tensor("f16", 1, 1, 1, 4), 1))
    with pytest.raises(hip.HipError):
        hip.check(ops.lib().cldnn_hip_matmul_enqueue(other.h, *[x.data_ptr()] * 5))
    other.close()
    op.close()
