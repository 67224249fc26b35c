"""Rotary positions with several axes against the formula in 64 bits; their gradient against the formula's and against
differences."""
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


def reference(x, positions, pairs, pairing, shared, base, inverse=False):
    """x: [tokens][heads][size] -> values and what 32-bit angles may be off"""
    y, bound, total, start = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64), sum(pairs), 0
    for axis, count in enumerate(pairs):
        for j in range(count):
            i = start + j
            frequency = base ** -(i / total if shared else j / count)
            angle = positions[:, axis].double() * frequency * (-1 if inverse else 1)
            lo, hi = {"interleaved": (2 * i, 2 * i + 1), "halves": (i, i + total), "halves_per_axis": (2 * start + j, 2 * start + j + count)}[pairing]
            c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            a, b = x[..., lo].double(), x[..., hi].double()
            y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
            # 2^-24 of a turn, a few units of sine and cosine, and the products' roundings
            bound[..., lo] = bound[..., hi] = (2 * math.pi * 2.0 ** -24 + 4 * EPS) * (a.abs() + b.abs())
        start += count
    return y, bound


def check(eng, tokens, q_heads, k_heads, size, pairs, dtype, *, pairing="interleaved", shared=False, base=10000.0, positions=None, inverse=False, spare=0, in_place=False,
          offset=0):
    """spare: elements behind each head and behind each token"""
    g = generator(tokens + size)
    if positions is None:
        positions = torch.randint(-300, 300, (tokens, len(pairs)), generator=g, dtype=torch.int32)
    heads, views, strides = (q_heads, k_heads), [], []
    for n in heads:
        x = random(g, tokens, n, size, dtype=dtype)
        head, token = size + spare, n * (size + spare) + spare
        strides.append((token, head) if n else (0, 0))
        flat = torch.full((tokens, token), 7.0, dtype=x.dtype)
        flat[:, :n * head].view(tokens, n, head)[..., :size] = x
        views.append((x, *framed(flat, offset, 7.0), head))
    outs = []
    for n, (x, whole, flat, head) in zip(heads, views):
        outs.append((whole, flat) if in_place else framed(torch.full_like(flat.cpu(), 7.0), offset, 7.0))
    op = ops.Rotary(eng, ops.rotary_desc(tokens, q_heads, k_heads, size, pairs, dtype, pairing=pairing, shared_frequencies=shared, base=base, inverse=inverse,
                                         position_dtype="f32" if positions.dtype == torch.float32 else "i32", q_strides=strides[0], k_strides=strides[1],
                                         q_out_strides=strides[0], k_out_strides=strides[1]))
    run(eng, op, views[0][2], views[1][2] if k_heads else None, positions.cuda(), outs[0][1], outs[1][1] if k_heads else None)
    op.close()
    results = []
    for n, (x, _, _, head), (whole, flat) in zip(heads, views, outs):
        if not n:
            continue
        got = flat.cpu()[:, :n * head].reshape(tokens, n, head)
        rest = flat.cpu().clone()
        rest[:, :n * head].view(tokens, n, head)[..., :size] = 7.0
        assert (rest == 7.0).all() and untouched(whole, offset, flat.numel(), 7.0)
        want, bound = reference(x, positions, pairs, pairing, shared, base, inverse)
        close(got[..., :size], want, bound + HALF_ULP[dtype] * want.abs() * (1 + 2 ** -8) + SMALLEST[dtype])
        results.append(got[..., :size])
    return results


PAIRINGS = ["interleaved", "halves", "halves_per_axis"]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("pairing", PAIRINGS)
@pytest.mark.parametrize("shape", [(1, 1, 0, 2, (1,)), (1, 16, 16, 64, (16, 16)), (49, 4, 1, 80, (20, 20)), (37, 3, 3, 128, (16, 24, 24)), (65, 2, 5, 96, (9, 20, 10)),
                                   (200, 1, 2, 40, (5, 0, 3, 4)), (13, 5, 1, 33, (7, 3)), (1000, 2, 2, 32, (8, 8)), (9, 40, 8, 128, (32, 32))], ids=str)
def test_shapes(eng, shape, pairing, dtype):
    tokens, q, k, size, pairs = shape
    check(eng, tokens, q, k, size, pairs, dtype, pairing=pairing)


@pytest.mark.parametrize("pairing", PAIRINGS)
def test_shared_frequencies_and_other_bases(eng, pairing):
    check(eng, 30, 2, 2, 64, (8, 12, 12), "f32", pairing=pairing, shared=True, base=500000.0)
    check(eng, 30, 2, 1, 64, (16, 16), "f32", pairing=pairing, base=100.0)


@pytest.mark.parametrize("pairing", PAIRINGS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("spare,offset", [(8, 8), (1, 3), (2, 1)])
def test_strides_alignment_and_in_place(eng, pairing, dtype, spare, offset):
    for in_place in (False, True):
        check(eng, 21, 3, 2, 48, (12, 12), dtype, pairing=pairing, spare=spare, offset=offset, in_place=in_place)
        check(eng, 21, 3, 2, 48, (9, 12), dtype, pairing=pairing, spare=spare, offset=offset, in_place=in_place)


def test_large_and_fractional_positions(eng):
    g = generator(3)
    large = torch.randint(-(1 << 24), 1 << 24, (64, 2), generator=g, dtype=torch.int32)
    large[0] = torch.tensor([1 << 24, -(1 << 24)])
    check(eng, 64, 2, 2, 64, (16, 16), "f32", positions=large)
    check(eng, 64, 2, 2, 64, (16, 16), "f32", positions=(torch.randn(64, 2, generator=g) * 1000).float())
    check(eng, 64, 2, 2, 64, (16, 16), "f32", positions=torch.zeros(64, 2, dtype=torch.int32))


@pytest.mark.parametrize("base", [0.5, 2.0 ** -7, 2.0 ** -13])
def test_bases_below_one(eng, base):
    # frequencies up to 1 / base, positions up to 2^24 * base
    most = int(2 ** 24 * base)
    positions = torch.randint(-most, most + 1, (64, 2), generator=generator(7), dtype=torch.int32)
    positions[0] = torch.tensor([most, -most])
    check(eng, 64, 2, 2, 64, (16, 16), "f32", positions=positions, base=base)
    check(eng, 64, 2, 2, 64, (12, 20), "f32", positions=positions.float() * 0.75, base=base, shared=True)


def test_gradient(eng):
    """The transpose of a rotation is the rotation back: against automatic differentiation of the formula, and against differences
    (the operator is linear: they are exact but for its roundings)."""
    g = generator(5)
    tokens, heads, size, pairs = 11, 2, 24, (4, 6)
    positions = torch.randint(0, 50, (tokens, 2), generator=g, dtype=torch.int32)
    x, seen = random(g, tokens, heads, size), random(g, tokens, heads, size)

    def turn(v, inverse):
        out = torch.empty(tokens, heads, size, device="cuda")
        op = ops.Rotary(eng, ops.rotary_desc(tokens, heads, 0, size, pairs, "f32", inverse=inverse))
        run(eng, op, v.float().cuda(), None, positions.cuda(), out, None)
        op.close()
        return out.cpu().double()

    got = turn(seen, True)
    leaf = x.double().clone().requires_grad_()
    i, start = 0, 0
    parts = []
    for axis, count in enumerate(pairs):
        for j in range(count):
            angle = positions[:, axis].double()[:, None] * 10000.0 ** -(j / count)
            a, b = leaf[..., 2 * i], leaf[..., 2 * i + 1]
            parts += [a * torch.cos(angle) - b * torch.sin(angle), b * torch.cos(angle) + a * torch.sin(angle)]
            i += 1
    y = torch.cat([torch.stack(parts, -1), leaf[..., 2 * i:]], -1)
    (y * seen.double()).sum().backward()
    close(got, leaf.grad, 16 * EPS * (seen.double().abs().sum(-1, keepdim=True) + 1))
    for t, h, d in ((0, 0, 0), (3, 1, 7), (10, 0, 19), (7, 1, 23)):
        step = torch.zeros_like(x)
        step[t, h, d] = 1.0
        change = ((turn(x + step, False) - turn(x - step, False)) / 2 * seen.double()).sum()
        assert abs(float(change - got[t, h, d])) < 64 * EPS * float(seen.abs().sum(-1).max() * (x.abs().max() + 1))


def test_offsets_past_32_bits(eng):
    tokens, size, pitch = 3, 16, 1 << 31
    g = generator(6)
    x = random(g, tokens, 1, size, dtype="bf16")
    far = torch.empty((tokens - 1) * pitch + 64, dtype=torch.bfloat16, device="cuda")
    for t in range(tokens):
        far[t * pitch:t * pitch + size] = x[t, 0].cuda()
    positions = torch.tensor([[5, 1], [100, 7], [3, 900]], dtype=torch.int32)
    op = ops.Rotary(eng, ops.rotary_desc(tokens, 1, 0, size, (4, 4), "bf16", q_strides=(pitch, size), q_out_strides=(pitch, size)))
    run(eng, op, far, None, positions.cuda(), far, None)
    op.close()
    want, bound = reference(x, positions, (4, 4), "interleaved", False, 10000.0)
    got = torch.stack([far[t * pitch:t * pitch + size] for t in range(tokens)])[:, None]
    close(got, want, bound + HALF_ULP["bf16"] * want.abs() * (1 + 2 ** -8))


def test_refusals(eng):
    def status(*args, **kw):
        return refused(eng, ops.Rotary, ops.rotary_desc(*args, **kw))

    assert status(4, 2, 2, 16, (4, 4), "f16") == 0
    for sizes in ((0, 2, 2, 16), (4, 0, 2, 16), (4, 2, -1, 16), (4, 2, 2, 0)):
        assert status(*sizes, (4, 4), "f16") == INVALID_ARG
    assert status(4, 2, 2, 16, (4, 5), "f16") == DIMENSION_MISMATCH
    assert status(4, 2, 2, 16, (0, 0), "f16") == DIMENSION_MISMATCH
    assert status(4, 2, 2, 16, (4, -1), "f16") == INVALID_ARG
    assert status(4, 2, 2, 16, (4, 4), hip.U8) == INVALID_ARG
    assert status(4, 2, 2, 16, (4, 4), "f16", pairing=3) == INVALID_ARG
    assert status(4, 2, 2, 16, (4, 4), "f16", position_dtype=hip.S8) == INVALID_ARG
    for base in (0.0, -1.0, math.inf, math.nan):
        assert status(4, 2, 2, 16, (4, 4), "f16", base=base) == INVALID_ARG
    assert status(4, 2, 2, 16, (4, 4), "f16", q_strides=(-1, 16)) == INVALID_ARG
    with pytest.raises(ValueError):
        ops.rotary_desc(4, 2, 2, 16, (1,) * 5, "f16")
    op = ops.Rotary(eng, ops.rotary_desc(4, 2, 2, 16, (4, 4), "f16"))
    x = torch.zeros(4 * 2 * 16, dtype=torch.float16, device="cuda")
    for args in ((None, x, x, x, x), (x, None, x, x, x), (x, x, None, x, x), (x, x, x, None, x), (x, x, x, x, None), (x.data_ptr() + 1, x, x, x, x),
                 (x, x, x.data_ptr() + 2, x, x)):
        with pytest.raises(hip.HipError) as err:
            op.enqueue(*args)
        assert err.value.status == INVALID_ARG
    op.close()
