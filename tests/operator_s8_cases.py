"""What the tests of the int8 operators share: quantised rows in 32 and 64 bits, unit forms of rows with the error that 32 bits allow."""
import numpy as np
import torch

from operator_cases import *

U = 2.0 ** -24  # half a step of 32 bits, relative to the value


def quantized32(y):
    """What the header defines, in 32 bits step by step: numpy's quotients, products and rint are the ones it names.  y: float32 rows."""
    y = np.asarray(y, np.float32)
    with np.errstate(all="ignore"):
        most = np.abs(y).max(1)
        bad, zero = ~np.isfinite(y).all(1), most < np.float32(2.0 ** -120)
        inverse, scale = np.float32(127) / most, most / np.float32(127)
        q = np.rint(y * inverse[:, None])
    q[bad | zero], scale[zero], scale[bad] = 0, 0, np.nan
    return q.astype(np.int8), scale.astype(np.float32)


def same_rows(q, scales, y, what=""):
    """quantised rows of values that 32 bits hold are the same bits"""
    want, steps = quantized32(y)
    q, scales = q.cpu().numpy(), scales.cpu().numpy()
    assert np.array_equal(scales, steps, equal_nan=True), what
    assert np.array_equal(q, want), "%s: %d values of %d" % (what, (q != want).sum(), q.size)


def near_rows(q, scales, y, error, what=""):
    """Quantised rows of values that the operator has within `error`: each is within half a step of its value and the errors.  The step is
    most / 127, most within the largest error; the quotient, the product and the step are rounded once each, at 127 steps at most."""
    y, error, q, scales = y.double(), error.double().expand(y.shape), q.cpu().double(), scales.cpu().double()
    most, off = y.abs().amax(1), error.amax(1)
    step = most / 127
    assert ((scales - step).abs() <= off / 127 + U * step + 2.0 ** -149).all(), what
    live = most > 0
    away = (q - y / torch.where(live, step, 1.0)[:, None])[live]
    room = (0.5 + 127 * 3 * U + error / step[:, None] + (127 * off / most)[:, None])[live]
    assert (away.abs() <= room).all(), "%s: worst %g of %g" % (what, float((away.abs() - room).max()), float(room.max()))
    assert (q[~live] == 0).all() and q.abs().max() <= 127


def unit(v, error, kind, epsilon):
    """The unit form of the rows of v in 64 bits, and how far 32 bits may be off: sums of C values over lanes that add 32 of theirs and
    meet in trees and runs of 16 are rounded at most 64 times on a value's way, each at the size of all magnitudes together."""
    if kind == "none":
        return v, error
    D = 64
    if kind == "layer":
        off = (D + 2) * U * v.abs().mean(1, keepdim=True) + error.mean(1, keepdim=True)
        v = v - v.mean(1, keepdim=True)
        error = error + off + U * v.abs()
    square = (v * v).mean(1, keepdim=True)
    s = torch.sqrt(square + epsilon)
    off = error.amax(1, keepdim=True) / s  # of a value, in deviations
    # the mean square is off by its sums, and by 2 |v| e + e^2 of each value; its root by half of that; quotient, root and product round
    factor = 0.5 * ((D + 4) * U + 2 * off + off * off) + 4 * U
    return v / s, error / s * (1 + factor) + (v / s).abs() * factor
