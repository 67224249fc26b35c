"""What the tests of the float operators share: types with their rounding, activations in 64 bits, device tensors with memory
around them that must be neither used nor written."""
import math

import torch

from cldnn_amd import hip, ops

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a unit in the last place of 1, relative to the value: what one rounding may be off
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# results below these are rounded to a grid of their own
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
EPS = 2.0 ** -23


def act64(v, act, m=0.0, n=0.0):
    return {
        "none": lambda: v, "relu": lambda: torch.clamp(v, min=0), "relu_slope": lambda: torch.where(v < 0, v * m, v),
        "clamp": lambda: torch.clamp(v, m, n), "silu": lambda: v * torch.sigmoid(v), "gelu": lambda: v * torch.special.ndtr(v),
        "gelu_tanh": lambda: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))),
    }[act]()


# no activation here is steeper than this
STEEPEST = 1.13


def act_error(v):
    """What the activations' own arithmetic may be off: erfc to 1.5e-7 (its published bound) times half the value, and
    reciprocals and exponentials of 32 bits, whose argument v * log2(e) is rounded: relative errors of |v| units."""
    return v.abs() * (1.0e-7 + 4 * EPS) + v.abs() * act_slope(v) * EPS * v.abs()


def act_slope(v):
    return torch.exp(-v.abs().clamp(max=80))  # where the exponential counts beside 1


def random(g, *shape, scale=1.0, dtype="f32"):
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(TYPES[dtype])


def generator(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def framed(t, offset=0, fill=math.nan):
    """A copy of the dense CPU tensor t on the GPU, `offset` elements behind the start of an allocation that is full of `fill`
    before and behind it."""
    whole = torch.full((offset + t.numel() + 64,), fill, dtype=t.dtype, device="cuda")
    view = whole[offset:offset + t.numel()].view(t.shape)
    view.copy_(t)
    return whole, view


def untouched(whole, offset, count, fill):
    rest = torch.cat([whole[:offset], whole[offset + count:]])
    return bool(torch.isnan(rest).all()) if math.isnan(fill) else bool((rest == fill).all())


def close(got, want, bound, what=""):
    """|got - want| <= bound everywhere, NaN and infinities at the same places"""
    got, want, bound = got.detach().cpu().double(), want.double(), bound.double()
    same = (torch.isnan(got) & torch.isnan(want)) | (got == want)
    off = (got - want).abs()
    bad = ~same & ~(off <= bound)
    assert not bad.any(), "%s: %d of %d off, worst %g for a bound of %g" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(bound.expand_as(off)[bad].min()))


def run(engine, operator, *args, **kw):
    torch.cuda.synchronize()
    operator.enqueue(*args, **kw)
    engine.finish()


def refused(engine, kind, desc):
    """status of a description that create refuses"""
    try:
        kind(engine, desc).close()
    except hip.HipError as e:
        assert str(e).split(": ", 1)[1], "no message"
        return e.status
    return 0


INVALID_ARG, UNSUPPORTED_SIZE, UNSUPPORTED_FORMAT, DIMENSION_MISMATCH = -2, -5, -6, -7
__all__ = [n for n in dir() if not n.startswith("_")]
