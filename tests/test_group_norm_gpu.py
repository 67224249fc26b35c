"""Group norm with an activation against the formula in 64 bits."""
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


def reference(x, groups, scale, shift, eps, act, m, n):
    """values and what 32-bit arithmetic may be off them: (value before the activation, value, bound)"""
    b, y, w, f = x.shape
    g = x.double().reshape(b, y * w, groups, f // groups)
    mean = g.mean((1, 3), keepdim=True)
    var = ((g - mean) ** 2).mean((1, 3), keepdim=True)
    z = ((g - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    scale = torch.ones(f).double() if scale is None else scale.double()
    shift = torch.zeros(f).double() if shift is None else shift.double()
    v = z * scale + shift
    # A mean or variance joins values of at most a few hundred to a thread, then rows, features and parts: within 64 + values / 256
    # roundings of its size.  Values are held around one of themselves: the mean's size counts by its own rounding, once.
    roundings = 64 + g.shape[1] * g.shape[3] / 256
    spread = (mean.abs() / torch.sqrt(var + eps)).expand_as(g).reshape(x.shape)
    bound = EPS * (roundings * (z.abs() + 1) * scale.abs() + 2 * spread * scale.abs() + 2 * shift.abs())
    return v, act64(v, act, m, n), bound


def check(eng, x, groups, dtype, out, act="none", m=0.0, n=0.0, scale=None, shift=None, eps=1e-5, pads=(0, 0, 0), out_pads=(0, 0, 0), offset=0):
    b, h, w, f = x.shape
    x = x.to(TYPES[dtype])
    tin, tout = ops.map_tensor(dtype, b, h, w, f, *pads), ops.map_tensor(out, b, h, w, f, *out_pads)

    def shape(p):
        return (b, h + 2 * p[0], w + 2 * p[1], f + p[2])

    inside = (slice(None), slice(pads[0], pads[0] + h), slice(pads[1], pads[1] + w), slice(0, f))
    outside = (slice(None), slice(out_pads[0], out_pads[0] + h), slice(out_pads[1], out_pads[1] + w), slice(0, f))
    full = torch.full(shape(pads), math.nan, dtype=TYPES[dtype])  # padding is neither read ...
    full[inside] = x
    _, src = framed(full, offset)
    whole, dst = framed(torch.full(shape(out_pads), 7.0, dtype=TYPES[out]), offset, 7.0)  # ... nor written
    op = ops.GroupNorm(eng, ops.group_norm_desc(tin, groups, output=tout, epsilon=eps, act=act, act_m=m, act_n=n))
    dev = [None if t is None else t.float().cuda() for t in (scale, shift)]
    run(eng, op, src, dst, *dev)
    got, rest = dst.cpu(), dst.cpu().clone()
    rest[outside] = 7.0
    assert (rest == 7.0).all() and untouched(whole, offset, dst.numel(), 7.0)
    v, want, bound = reference(x, groups, None if scale is None else scale.float(), None if shift is None else shift.float(), eps, act, m, n)
    bound = STEEPEST * max(1.0, abs(m)) * bound + act_error(v) + HALF_ULP[out] * want.abs() * (1 + 2 ** -8) + SMALLEST[out]
    close(got[outside], want, bound)
    again = dst.clone()
    run(eng, op, src, dst, *dev)
    assert torch.equal(again, dst), "the same call gives other bits"
    op.close()
    return got[outside]


SIZES = [  # b, y, x, f, groups
    (1, 1, 1, 8, 8), (1, 1, 1, 1, 1), (2, 1, 1, 64, 32), (1, 7, 7, 2048, 32), (3, 31, 45, 84, 12), (2, 56, 56, 64, 32), (1, 13, 9, 1369, 37),
    (5, 3, 2, 24, 1), (1, 112, 97, 16, 2), (2, 5, 3, 4160, 5), (1, 2, 3, 6144, 1), (1, 40, 40, 320, 32), (2, 17, 4, 26, 13), (33, 2, 2, 40, 4), (1, 4, 4, 3075, 3),
    (1, 60, 60, 32, 32), (1, 130, 130, 32, 32), (2, 30, 20, 40, 40), (1, 70, 60, 16, 16),  # a feature to a group
]


@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "f16"), ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes_and_types(eng, size, dtype, out):
    b, y, x, f, groups = size
    g = generator(f + y)
    data = random(g, b, y, x, f) * torch.exp(random(g, f)) + random(g, f)
    check(eng, data, groups, dtype, out, "silu", scale=1 + random(g, f, scale=0.3), shift=random(g, f))


@pytest.mark.parametrize("act,m,n", [("none", 0, 0), ("relu", 0, 0), ("relu_slope", 0.1, 0), ("clamp", -0.5, 0.75), ("silu", 0, 0), ("gelu", 0, 0), ("gelu_tanh", 0, 0)])
@pytest.mark.parametrize("scaled", [True, False])
def test_activations(eng, act, m, n, scaled):
    g = generator(5)
    data = random(g, 2, 9, 11, 48)
    # factors of up to 12: where the activations are flat as well
    scale, shift = (random(g, 48, scale=4.0), random(g, 48)) if scaled else (None, None)
    check(eng, data, 6, "f32", "f32", act, m, n, scale, shift)


@pytest.mark.parametrize("mean,spread", [(1000.0, 1.0), (-3e4, 0.01), (0.0, 1e-6), (1e-3, 0.0), (5.0, 0.0)])
def test_large_means_and_constant_maps(eng, mean, spread):
    g = generator(7)
    data = mean + spread * random(g, 2, 33, 21, 16)
    data[1, 0, 0] = 0.0 if spread else mean  # a first pixel that is nothing like the rest
    check(eng, data, 4, "f32", "f32", "none", scale=random(g, 16), shift=random(g, 16))


@pytest.mark.parametrize("pads,out_pads,offset", [((1, 2, 0), (0, 0, 0), 0), ((0, 0, 3), (2, 1, 5), 1), ((0, 0, 8), (0, 0, 8), 8), ((1, 1, 1), (1, 1, 1), 3)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("f,groups", [(48, 6), (21, 7)])
def test_padding_is_a_stride(eng, pads, out_pads, offset, dtype, f, groups):
    g = generator(9)
    check(eng, random(g, 2, 6, 5, f), groups, dtype, dtype, "gelu", scale=random(g, f), pads=pads, out_pads=out_pads, offset=offset)


@pytest.mark.parametrize("size", [(2, 9, 7, 64, 8), (1, 90, 80, 64, 8)], ids=str)
def test_in_place(eng, size):
    b, y, x, f, groups = size
    g = generator(11)
    data = random(g, b, y, x, f, dtype="f16").cuda()
    src, want = data.clone(), torch.empty_like(data)
    op = ops.GroupNorm(eng, ops.group_norm_desc(ops.map_tensor("f16", b, y, x, f), groups, act="silu"))
    run(eng, op, src, want)
    run(eng, op, data, data)
    assert torch.equal(data, want) and not torch.equal(data, src)
    op.close()


def test_maps_larger_than_the_caches(eng):
    g = generator(21)
    check(eng, torch.randn((8, 201, 200, 128), generator=g) * 2 + 1, 32, "f16", "f16", "silu", scale=random(g, 128))


def test_offsets_past_32_bits(eng):
    # 2^26 elements from pixel to pixel: the last starts 10 GiB in
    y, x, f, spare = 9, 9, 24, (1 << 26) - 24
    g = generator(23)
    data = random(g, 1, y, x, f, dtype="bf16")
    src, dst = (torch.empty(y * x << 26, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    src.view(y * x, 1 << 26)[:, :f] = data.view(y * x, f).cuda()
    t = ops.map_tensor("bf16", 1, y, x, f, pad_f=spare)
    op = ops.GroupNorm(eng, ops.group_norm_desc(t, 3, output=t))
    run(eng, op, src, dst)
    op.close()
    _, want, bound = reference(data, 3, None, None, 1e-5, "none", 0, 0)
    close(dst.view(y * x, 1 << 26)[:, :f].reshape(1, y, x, f), want, bound + HALF_ULP["bf16"] * want.abs() * (1 + 2 ** -8))


@pytest.mark.parametrize("first", ["one", "rows"])
@pytest.mark.parametrize("batch,y,x,f,groups,dtype,spare", [(256, 40, 50, 1023, 31, "f32", 0), (256, 41, 35, 1023, 31, "f16", 1), (64, 40, 40, 8192, 256, "f16", 0)])
def test_first_pixels_unlike_the_rest_of_many(eng, batch, y, x, f, groups, dtype, spare, first):
    """hundreds of pixels to a thread, the first (or the first rows) far from all others: a border, a corner"""
    g = torch.Generator("cuda")
    g.manual_seed(batch + f)
    data = torch.empty(batch, y, x, f + spare, dtype=TYPES[dtype], device="cuda")
    for image in data:
        image.copy_(10 + 0.1 * torch.randn(y, x, f + spare, generator=g, device="cuda"))
    if first == "one":
        data[:, 0, 0] = 0
    else:
        data[:, :2] = 0
    t = ops.map_tensor(dtype, batch, y, x, f, pad_f=spare)
    op = ops.GroupNorm(eng, ops.group_norm_desc(t, groups, out_dtype="f32"))
    out = torch.empty(batch, y, x, f, device="cuda")
    run(eng, op, data, out)
    op.close()
    for i in (0, batch - 1):
        v, want, bound = reference(data[i:i + 1, :, :, :f].cpu(), groups, None, None, 1e-5, "none", 0, 0)
        close(out[i:i + 1], want, bound + HALF_ULP["f32"] * want.abs())


def test_nan_and_infinity_stay_in_their_group(eng):
    g = generator(13)
    data = random(g, 2, 5, 5, 32)
    clean = check(eng, data, 4, "f32", "f32", scale=random(g, 32))
    data[0, 2, 3, 9] = math.nan
    data[1, 0, 0, 31] = math.inf
    op = ops.GroupNorm(eng, ops.group_norm_desc(ops.map_tensor("f32", 2, 5, 5, 32), 4))
    dst = torch.empty(2, 5, 5, 32, device="cuda")
    run(eng, op, data.float().cuda(), dst)
    bad = torch.isnan(dst.cpu())
    want = torch.zeros_like(bad)
    want[0, :, :, 8:16] = True
    want[1, :, :, 24:] = True
    assert torch.equal(bad, want) and not torch.isnan(clean).any()
    op.close()


def test_many_images_and_a_recording(eng):
    g = generator(15)
    data = random(g, 4, 20, 20, 64, dtype="bf16").cuda()
    op = ops.GroupNorm(eng, ops.group_norm_desc(ops.map_tensor("bf16", 4, 20, 20, 64), 8, act="silu"))
    want, got = torch.empty_like(data), torch.zeros_like(data)
    run(eng, op, data, want)
    L, rec = hip.lib(), hip.C.c_void_p()
    hip.check(L.cldnn_hip_engine_record_begin(eng.h))
    op.enqueue(data, got)
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
    t = ops.map_tensor("f16", 1, 4, 4, 12)
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(t, 4)) == 0
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(t, 5)) == INVALID_ARG
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(t, 0)) == INVALID_ARG
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(t, 4, epsilon=-1e-3)) == INVALID_ARG
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(t, 4, epsilon=math.nan)) == INVALID_ARG
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(t, 4, act=77)) == INVALID_ARG
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(t, 4, act="clamp", act_m=1.0, act_n=-1.0)) == INVALID_ARG
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(t, 4, output=ops.map_tensor("f16", 1, 4, 5, 12))) == DIMENSION_MISMATCH
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(hip.Tensor.make("s8", "byxf", 1, 12, 4, 4), 4)) == INVALID_ARG
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(hip.Tensor.make("f32", "bfyx", 1, 12, 4, 4), 4)) == UNSUPPORTED_FORMAT
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(hip.Tensor.make("f32", "byxf", 1, 12, 0, 4), 4, output=t)) != 0
    assert refused(eng, ops.GroupNorm, ops.group_norm_desc(ops.map_tensor("f16", 1, 1, 1, 6152), 1)) == UNSUPPORTED_SIZE
    op = ops.GroupNorm(eng, ops.group_norm_desc(t, 4))
    x = torch.zeros(4 * 4 * 12, dtype=torch.float16, device="cuda")
    for args in ((None, x), (x, None), (x.data_ptr() + 1, x), (x, x.data_ptr() + 1), (x, x, x.data_ptr() + 2)):
        with pytest.raises(hip.HipError) as err:
            op.enqueue(*args)
        assert err.value.status == INVALID_ARG
    op.close()
