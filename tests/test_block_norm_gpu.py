"""Norms before and after a block, with its gate and residual scale, against the formula in 64 bits."""
import itertools
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


def check(eng, tokens, features, dtype="f32", *, branch=None, out="f32", norm="layer", post="none", epsilon=1e-5, post_epsilon=1e-5, residual_scale=1.0, per_image=0, modulation=None,
          has=("post_weight", "post_bias", "gate", "weight", "bias", "scale", "shift", "y"), spare=0, offset=0, in_place=False, shift_by=0.0, seed=0):
    """spare: elements between the rows of everything; offset: of the starts; shift_by: the mean of all values"""
    g = generator(seed + tokens + 3 * features)
    images = -(-tokens // per_image) if per_image else 1
    keep = {}

    def rows(name, count, kind, scale=1.0, mean=0.0):
        values = (random(g, count, features, scale=scale).double() + mean).to(TYPES[kind])
        full = torch.full((count, features + spare), math.nan, dtype=TYPES[kind])
        full[:, :features] = values
        keep[name] = framed(full, offset)
        return values.double(), keep[name][1]

    def vector(mean):
        v = mean + random(g, features, scale=0.3)
        return v.double(), framed(v, offset)[1]

    x, dx = rows("x", tokens, dtype, mean=shift_by)
    given, host = {}, {}
    if branch:
        host["branch"], given["branch"] = rows("branch", tokens, branch, mean=shift_by)
        for name, mean in (("post_weight", 0.7), ("post_bias", 0.0)):
            if name in has:
                host[name], given[name] = vector(mean)
    for name, mean in (("weight", 1.0), ("bias", 0.0)):
        if out and name in has:
            host[name], given[name] = vector(mean)
    if modulation:
        for name in ("gate", "scale", "shift"):
            if name in has and (branch if name == "gate" else out):
                host[name], given[name] = rows(name, images, modulation, scale=0.5)
    dy = dout = scales = None
    if branch and "y" in has:
        dy = dx if in_place else rows("y", tokens, dtype)[1]
    if out == "s8":
        keep["out"] = framed(torch.full((tokens, features + spare), 99, dtype=torch.int8), offset, fill=99)
        dout, scales = keep["out"][1], torch.zeros(tokens, device="cuda")
    elif out:
        dout = rows("out", tokens, out)[1]
    stride = {n + "_stride": features + spare for n in ("x", "branch", "y", "out", "gate", "scale", "shift")}
    op = ops_s8.BlockNorm(eng, ops_s8.block_norm_desc(tokens, features, dtype, branch_dtype=branch, out_dtype=out, norm=norm if out else "none", post=post if branch else "none", epsilon=epsilon,
                                                      post_epsilon=post_epsilon, residual_scale=residual_scale if branch else 1.0, tokens_per_image=per_image, modulation_dtype=modulation, **stride))
    before = dx.clone()
    run(eng, op, dx, dy, dout, out_scales=scales, **given)
    what = op.info().kernel_name.decode()

    def per_token(name):
        image = torch.arange(tokens) // per_image if per_image else torch.zeros(tokens, dtype=torch.long)
        return host[name][image]

    # each operation rounds once, at the size of its result or of its larger operand
    y, error = x, torch.zeros_like(x)
    if branch:
        z, error = unit(host["branch"], torch.zeros_like(x), post, post_epsilon)
        for name in ("post_weight", "post_bias", "gate"):
            if name in host:
                by = per_token(name) if name == "gate" else host[name]
                error = error if name == "post_bias" else error * by.abs()
                z = z + by if name == "post_bias" else z * by
                error = error + 2 * U * (z.abs() + (by.abs() if name == "post_bias" else 0))
        y = residual_scale * x + z
        error = error + 2 * U * (y.abs() + z.abs() + (residual_scale * x).abs())
        if dy is not None:
            close(dy[:, :features], y, error + HALF_ULP[dtype] * (y.abs() + error) + SMALLEST[dtype], what)
    if out:
        h, error = unit(y, error, norm, epsilon)
        for name in ("weight", "bias", "scale", "shift"):
            if name in host:
                by = 1 + per_token(name) if name == "scale" else per_token(name) if name == "shift" else host[name]
                if name in ("weight", "scale"):
                    h, error = h * by, error * by.abs() + 3 * U * (h * by).abs()
                else:
                    error = error + U * (h.abs() + by.abs())
                    h, error = h + by, error + U * (h + by).abs()
        if out == "s8":
            near_rows(dout[:, :features], scales, h, error, what)
        else:
            close(dout[:, :features], h, error + HALF_ULP[out] * (h.abs() + error) + SMALLEST[out], what)
    for name, (whole, view) in keep.items():
        fill = 99 if name == "out" and out == "s8" else math.nan
        assert untouched(whole, offset, view.numel(), fill), name
        between = view[:, features:]
        assert (between == 99).all() if fill == 99 else torch.isnan(between).all(), name
    first = [None if t is None else t.clone() for t in (dy, dout, scales)]
    dx.copy_(before)
    run(eng, op, dx, dy, dout, out_scales=scales, **given)
    for a, b in zip(first, (dy, dout, scales)):
        assert a is None or torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())), "the same call gives other bits"
    op.close()
    return what


WIDTHS = [1, 2, 7, 8, 9, 84, 127, 128, 129, 500, 512, 513, 1000, 1024, 1025, 1999, 2048, 2050, 4096, 4100, 8192, 8195, 16384, 16400, 32767, 32768]


@pytest.mark.parametrize("norm,post", [("layer", "none"), ("rms", "rms"), ("layer", "layer")])
@pytest.mark.parametrize("features", WIDTHS)
def test_widths(eng, features, norm, post):
    tokens = 37 if features < 600 else 5 if features < 5000 else 2
    check(eng, tokens, features, "f32", branch="f16", out="f32", norm=norm, post=post, modulation="f32", per_image=2)
    check(eng, tokens, features, "bf16", out="s8", norm=norm)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "s8", None])
@pytest.mark.parametrize("branch", ["f32", "f16", "bf16", None])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_types(eng, dtype, branch, out):
    if not branch and not out:
        return
    for modulation, (tokens, features) in zip(("f32", "f16", "bf16", None), ((21, 100), (9, 264), (5, 1500), (3, 9000))):
        check(eng, tokens, features, dtype, branch=branch, out=out, modulation=modulation, per_image=4, norm="rms", post="layer", residual_scale=0.75)


NAMES = ("post_weight", "post_bias", "gate", "weight", "bias", "scale", "shift", "y")


@pytest.mark.parametrize("norm,post", itertools.product(("none", "layer", "rms"), repeat=2))
def test_norms_and_what_may_be_left_out(eng, norm, post):
    for n in range(len(NAMES) + 1):  # each alone left out, and all
        has = NAMES[:n] + NAMES[n + 1:] if n < len(NAMES) else ()
        check(eng, 11, 200, "f32", branch="f32", out="f32" if n % 2 else "s8", norm=norm, post=post, modulation="f16", per_image=3, has=has, seed=n)


@pytest.mark.parametrize("spare,offset", [(0, 1), (3, 0), (8, 8), (5, 3)])
@pytest.mark.parametrize("dtype,out", [("f32", "f16"), ("f16", "s8"), ("bf16", "f32")])
@pytest.mark.parametrize("features", [84, 1000, 2304, 10000])
def test_strides_and_alignment(eng, features, dtype, out, spare, offset):
    check(eng, 7, features, dtype, branch="f16" if dtype == "f32" else dtype, out=out, post="rms", modulation="bf16", per_image=3, spare=spare, offset=offset)


@pytest.mark.parametrize("features", [84, 640, 3000, 20000])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_the_stream_in_place(eng, features, dtype):
    check(eng, 9, features, dtype, branch="f16", out="s8", modulation="f32", per_image=4, in_place=True)
    check(eng, 9, features, dtype, branch="f16", out=None, modulation="f32", per_image=4, in_place=True, spare=2)


@pytest.mark.parametrize("per_image", [0, 1, 2, 49, 50, 51, 1000])
def test_images(eng, per_image):
    for features in (40, 700, 5000):
        check(eng, 50, features, "bf16", branch="bf16", out="bf16", modulation="bf16", per_image=per_image)


def test_many_tokens(eng):
    check(eng, 4099, 96, "f16", branch="f16", out="s8", modulation="f16", per_image=784)
    check(eng, 3001, 1024, "bf16", branch="bf16", out="bf16", modulation="bf16", per_image=1000)


@pytest.mark.parametrize("out", ["f32", "f16", "s8"])
def test_results_that_go_past_the_caches(eng, out):
    # 34 MiB each; a last vector that lies over the one before it; in place
    check(eng, 8501, 1052, "f32", branch="f16", out=out, norm="layer", in_place=out == "s8")


@pytest.mark.parametrize("features", [84, 1024, 4100, 12000])
def test_a_mean_far_from_zero_costs_no_digits(eng, features):
    # the squares are taken around the mean: a deviation of 1 at a mean of 1000 keeps what the mean leaves of 32 bits
    check(eng, 6, features, "f32", branch="f32", out="f32", norm="layer", post="layer", shift_by=1000.0)


def test_rows_of_one_value_and_of_zeros(eng):
    """No deviation: what is left is the rounding of the mean, over the root of epsilon.  A mean is of sums that are rounded at most 64
    times, each at the size of the sum: 66 halves of a step of the value, which is what unit() counts.  Zeros, and whole numbers whose sums
    32 bits hold, leave nothing."""
    for features in (1, 60, 3000):
        x = torch.cat([torch.zeros(1, features), torch.full((1, features), 3.0), torch.full((1, features), -1e-30)])
        want, error = unit(x.double(), torch.zeros(3, features, dtype=torch.float64), "layer", 1e-5)
        x = x.cuda()
        out, q, scales = torch.empty_like(x), torch.ones(3, features, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")
        op = ops_s8.BlockNorm(eng, ops_s8.block_norm_desc(3, features, "f32", out_dtype="f32"))
        run(eng, op, x, None, out)
        close(out, torch.zeros(3, features), want.abs() + error)
        assert not out[:2].any()
        op.close()
        op = ops_s8.BlockNorm(eng, ops_s8.block_norm_desc(3, features, "f32", out_dtype="s8"))
        run(eng, op, x, None, q, out_scales=scales)
        assert not q[:2].any() and not scales[:2].any()
        close(q.cpu() * scales.cpu()[:, None].double(), torch.zeros(3, features), (want.abs() + error) * 1.01)
        op.close()


@pytest.mark.parametrize("features", [100, 3000])
def test_what_is_no_number_stays_in_its_row(eng, features):
    x = random(generator(1), 5, features).cuda()
    x[1, 3], x[3, features - 1] = math.nan, math.inf
    q, scales, h = torch.ones(5, features, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"), torch.ones(5, features, device="cuda")
    op = ops_s8.BlockNorm(eng, ops_s8.block_norm_desc(5, features, "f32", out_dtype="s8", norm="rms"))
    run(eng, op, x, None, q, out_scales=scales)
    assert torch.equal(torch.isnan(scales).cpu(), torch.tensor([False, True, False, True, False])) and not q[1].any() and not q[3].any() and (q[::2].abs().amax(1) == 127).all()
    op.close()
    op = ops_s8.BlockNorm(eng, ops_s8.block_norm_desc(5, features, "f32", out_dtype="f32"))
    run(eng, op, x, None, h)
    assert torch.isfinite(h[::2]).all() and torch.isnan(h[1]).all() and torch.isnan(h[3]).all()
    op.close()


def test_offsets_past_32_bits(eng):
    rows, features, pitch = 3, 72, 1 << 31
    x = random(generator(9), rows, features, dtype="f16")
    far = [torch.empty((rows - 1) * pitch + features, dtype=torch.float16, device="cuda") for _ in range(3)]
    for t in far[:2]:
        for i in range(rows):
            t[i * pitch:i * pitch + features] = x[i].cuda()
    op = ops_s8.BlockNorm(eng, ops_s8.block_norm_desc(rows, features, "f16", branch_dtype="f16", out_dtype="f16", norm="rms", x_stride=pitch, branch_stride=pitch, y_stride=pitch, out_stride=pitch))
    run(eng, op, far[0], far[0], far[2], branch=far[1])
    at = [torch.stack([t[i * pitch:i * pitch + features] for i in range(rows)]) for t in far]
    assert torch.equal(at[0], (x + x).cuda())
    y = 2 * x.double()
    h, error = unit(y, U * y.abs(), "rms", 1e-5)
    close(at[2], h, error + HALF_ULP["f16"] * h.abs() * 1.01 + SMALLEST["f16"])
    op.close()


def test_refusals(eng):
    def status(*args, **kw):
        return refused(eng, ops_s8.BlockNorm, ops_s8.block_norm_desc(*args, **kw))

    assert status(4, 4, "f16", out_dtype="f16") == status(4, 4, "f16", branch_dtype="f32", norm="none") == status(1, 32768, "f32", out_dtype="s8") == 0
    assert status(0, 4, "f16", out_dtype="f16") == status(4, 0, "f16", out_dtype="f16") == status(4, 4, "f16", out_dtype="f16", tokens_per_image=-1) == INVALID_ARG
    assert status(4, 32769, "f16", out_dtype="f16") == status(1 << 40, 8, "f16", out_dtype="f16") == UNSUPPORTED_SIZE
    assert status(4, 4, "s8", out_dtype="f16") == status(4, 4, "f16", out_dtype="i32") == status(4, 4, "f16", branch_dtype="s8", out_dtype="f16") == INVALID_ARG
    assert status(4, 4, "f16", out_dtype="f16", modulation_dtype="s8") == status(4, 4, "f16", norm="none") == status(4, 4, "f16", branch_dtype="f16", norm="rms") == INVALID_ARG
    assert status(4, 4, "f16", out_dtype="f16", post="rms") == status(4, 4, "f16", out_dtype="f16", residual_scale=0.5) == INVALID_ARG
    assert status(4, 4, "f16", out_dtype="f16", norm=3) == status(4, 4, "f16", branch_dtype="f16", out_dtype="f16", post=-1) == INVALID_ARG
    assert status(4, 4, "f16", out_dtype="f16", epsilon=-1e-9) == status(4, 4, "f16", out_dtype="f16", post_epsilon=math.nan) == INVALID_ARG
    for name in ("x", "branch", "y", "out", "gate", "scale", "shift"):
        assert status(4, 4, "f16", branch_dtype="f16", out_dtype="f16", modulation_dtype="f16", **{name + "_stride": 3}) == INVALID_ARG
