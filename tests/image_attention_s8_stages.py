"""The classifier with int8 products taken apart: what each call of a pass leaves, worked out on the CPU (`walk`), read from a model on
the GPU (`record`), and held against the formula of that call alone in 64 bits (`verify`), whose inputs are what the calls before it left.
A call's own roundings are all that is between the two then, and not what a quantisation makes of them later."""
import numpy as np
import torch

import test_attention_gpu
import test_rotary_gpu
from cldnn_amd import hip, ops, ops_s8
from operator_s8_cases import *

PRODUCTS = ("qkv", "project", "expand", "contract")


class Shapes:
    def __init__(self, p, batch, y, x):
        self.c, self.heads, self.kv = p["features"], p["heads"], p["kv_heads"]
        self.d, self.batch, self.n = self.c // self.heads, batch, y * x
        self.rows, self.qkv, self.pair = batch * self.n, (self.heads + 2 * self.kv) * self.d, 2 * self.kv * self.d
        grid = torch.stack(torch.meshgrid(torch.arange(y), torch.arange(x), indexing="ij"), -1).reshape(1, self.n, 2)
        self.positions = grid.expand(batch, self.n, 2).reshape(self.rows, 2)

    def heads_of(self, v, first, count):
        """[batch][tokens][heads][size] of the rows of v"""
        return v[:, first * self.d:(first + count) * self.d].reshape(self.batch, -1, count, self.d)

    def pooled_operands(self, p, kv, dtype):
        query = torch.from_numpy(p["query"]).to(TYPES[dtype]).expand(self.batch, 1, self.heads, self.d)
        return query, self.heads_of(kv, 0, self.kv), self.heads_of(kv, self.kv, self.kv)


def order(blocks):
    """the calls of a pass, and what each leaves"""
    calls = [("patches", ("x",)), ("first", ("q8", "scale"))]
    for _ in range(blocks):
        calls += [("qkv", ("qkv",)), ("rotary", ("qkv",)), ("attention", ("o",)), ("quantize", ("q8", "scale")), ("project", ("branch",)), ("between", ("x", "q8", "scale")),
                  ("expand", ("wide",)), ("quantize_wide", ("wide8", "scale")), ("contract", ("branch",)), ("between", ("x", "q8", "scale"))]
    return calls + [("kv", ("kv",)), ("pool", ("pooled",)), ("head", ("scores",))]


def t64(a):
    return torch.from_numpy(np.asarray(a)).double()


def patches(p, image):
    q = p["patches"]
    m = torch.nn.functional.conv2d(t64(image), t64(q["w"]), stride=p["patch"]) * t64(q["wqf"])[None, :, None, None]
    m = m.permute(0, 2, 3, 1).reshape(-1, p["features"])
    return m, m + t64(q["bias"])


def norms_of(p):
    return [b[k] for b in p["blocks"] for k in ("norm1", "norm2")] + [p["norm"]]


# ---------------------------------------------------------------------------------------------------------------- on the CPU
def quantized(v, mistake=None):
    """rows of v as 32 bits hold them"""
    y = v.float().numpy()
    q, scale = quantized32(y)
    if mistake == "rows of 4 bits":
        q = (np.rint(q / 18.0) * 18).astype(np.int8)
    if mistake == "truncation":
        q = np.trunc(y * (np.float32(127) / np.abs(y).max(1, keepdims=True))).astype(np.int8)
    return torch.from_numpy(q), torch.from_numpy(scale)


def walk(p, image, y, x, dtype, mistake=None):
    """(weights, [what each call of a pass leaves]), from the formulas in 64 bits, rounded where the network rounds.  mistake: one that is
    made on the way."""
    s, half = Shapes(p, len(image), y, x), TYPES[dtype]
    weights = [{k: quantized(t64(b[k][0])) for k in PRODUCTS} for b in p["blocks"]] + [{"kv": quantized(t64(p["kv"][0]))}]
    left, norms = [], norms_of(p)

    def leave(**what):
        left.append(what)

    def norm(i):
        if mistake == "norm2 has norm1's parameters" and i % 2 and i < len(norms):
            i -= 1
        h = unit(m, torch.zeros_like(m), "layer", 1e-5)[0] * t64(norms[i][0]) + t64(norms[i][1])
        return quantized(h, mistake)

    def product(q, scale, name, i, bias):
        w, steps = weights[i][name]
        if mistake == "no row scales":
            scale = torch.ones_like(scale)
        return ((q.double() @ w.double().T) * scale.double()[:, None] * steps.double() + t64(bias)).to(half)

    def attend(q, k, v):
        if mistake == "uniform attention":
            q = q * 0
        return test_attention_gpu.reference(q, k, v, s.d ** -0.5, None, None, dtype)[0].to(half).reshape(-1, s.c)

    m = patches(p, image)[1].float().double()
    leave(x=m.float())
    q, scale = norm(0)
    leave(q8=q, scale=scale)
    for i, b in enumerate(p["blocks"]):
        qkv = product(q, scale, "qkv", i, b["qkv"][1])
        leave(qkv=qkv)
        if mistake != "no rotary":
            positions = s.positions.flip(1) if mistake == "rotary axes swapped" else s.positions
            turned = (s.heads + s.kv) * s.d
            heads = qkv[:, :turned].reshape(s.rows, -1, s.d)
            qkv = torch.cat([test_rotary_gpu.reference(heads, positions, (s.d // 4, s.d // 4), "interleaved", False, 10000.0)[0].to(half).reshape(s.rows, turned), qkv[:, turned:]], 1)
        leave(qkv=qkv)
        o = attend(s.heads_of(qkv, 0, s.heads), s.heads_of(qkv, s.heads, s.kv), s.heads_of(qkv, s.heads + s.kv, s.kv))
        leave(o=o)
        q, scale = quantized(o, mistake)
        leave(q8=q, scale=scale)
        for half_of_block, name in enumerate(("project", "contract")):
            if name == "contract":
                wide = product(q, scale, "expand", i, b["expand"][1])
                leave(wide=wide)
                act = {"relu for gelu": "relu", "no gelu": "none"}.get(mistake, "gelu")
                q, scale = quantized(act64(wide.double(), act), mistake)
                leave(wide8=q, scale=scale)
            branch = product(q, scale, name, i, b[name][1])
            leave(branch=branch)
            factor = t64(b["scale%d" % (2 - half_of_block if mistake == "scales swapped" else 1 + half_of_block)])
            if mistake == "no scale%d" % (1 + half_of_block):
                factor = 1.0
            m = m + factor * branch.double()
            q, scale = norm(2 * i + half_of_block + 1)
            m = m.float().double()
            leave(x=m.float(), q8=q, scale=scale)
    kv = product(q, scale, "kv", -1, p["kv"][1])
    leave(kv=kv)
    pooled = attend(*s.pooled_operands(p, kv, dtype))
    leave(pooled=pooled)
    leave(scores=(pooled.double() @ t64(p["scores"][0]).to(half).double().T + t64(p["scores"][1])).float())
    return weights, left


# ---------------------------------------------------------------------------------------------------------------- on the GPU
def record(model, image):
    """(weights, [what each call of a pass leaves]) of a model; its scores are read behind all of it"""
    p, s, dtype = model.params, Shapes(model.params, model.batch, *_patch_grid(model, image)), model.dtype
    left, names = [], []

    def rows(buffer, width, kind):
        return torch.from_numpy(buffer.read((s.rows, width), kind)).to(TYPES.get(kind, torch.int8))

    where = {
        "x": lambda: torch.from_numpy(np.asarray(model._x.read_raw()).view(np.float32).reshape(s.rows, s.c).copy()), "q8": lambda: rows(model._q8, s.c, "s8"),
        "scale": lambda: rows(model._scale, 1, "f32")[:, 0], "qkv": lambda: rows(model._qkv, s.qkv, dtype), "kv": lambda: rows(model._qkv, s.pair, dtype), "o": lambda: rows(model._o, s.c, dtype),
        "branch": lambda: rows(model._branch, s.c, dtype), "wide": lambda: rows(model._wide, 4 * s.c, dtype), "wide8": lambda: rows(model._wide8, 4 * s.c, "s8"),
        "pooled": lambda: torch.from_numpy(model._pooled.read((s.batch, s.c), dtype)).to(TYPES[dtype]),
        "scores": lambda: torch.from_numpy(model._scores.read((s.batch, p["classes"]), "f32")),
    }
    outputs = dict(order(1))

    def wrap(owner, attribute, name):
        call = getattr(owner, attribute)

        def called(*args, **kw):
            call(*args, **kw)
            names.append(name)
            left.append({k: where[k]() for k in outputs[name]})

        setattr(owner, attribute, called)
        return lambda: delattr(owner, attribute)

    undo = [wrap(model, "_run_patches", "patches")]
    for name in ("first", "between", "quantize", "quantize_wide", "rotary", "attention", "pool", "head"):
        undo.append(wrap(getattr(model, "_" + name), "enqueue", name))
    for name in PRODUCTS + ("kv",):
        undo.append(wrap(model._product[name], "enqueue", name))
    try:
        model.run(image)
    finally:
        for f in undo:
            f()
    assert names == [name for name, _ in order(len(p["blocks"]))]

    def read_weights(of, pair):
        n, k = pair[0].shape
        return torch.from_numpy(of[0].read((n, k), "s8")), torch.from_numpy(of[1].read((n,), "f32"))

    weights = [{k: read_weights(kept[k], b[k]) for k in PRODUCTS} for kept, b in zip(model._blocks, p["blocks"])] + [{"kv": read_weights(model._kv, p["kv"])}]
    return weights, left


def _patch_grid(model, image):
    patch = model.params["patch"]
    return image.shape[2] // patch, image.shape[3] // patch


# ------------------------------------------------------------------------------------------------------------ against 64 bits
def verify(p, image, y, x, dtype, weights, left):
    """Each call against its formula on what the calls before it left."""
    s, norms = Shapes(p, len(image), y, x), norms_of(p)
    for kept, given in zip(weights, p["blocks"] + [{"kv": p["kv"]}]):
        for name, (q, steps) in kept.items():
            same_rows(q, steps, given[name][0], "weights of " + name)
    calls = iter(zip(order(len(p["blocks"])), left))

    def following(name):
        (expected, _), got = next(calls)
        assert expected == name
        return got

    def to_type(want, bound, kind=dtype):
        return bound + HALF_ULP[kind] * (want.abs() + bound) * (1 + 2 ** -8) + SMALLEST[kind]

    def norm(m, error, i, got, what):
        """a layer norm of m with its weight and bias, as quantised rows"""
        h, error = unit(m, error, "layer", 1e-5)
        w, b = t64(norms[i][0]), t64(norms[i][1])
        h, error = h * w, error * w.abs() + 3 * U * (h * w).abs()
        error = error + U * (h.abs() + b.abs())
        h = h + b
        near_rows(got["q8"], got["scale"], h, error + U * h.abs(), what)

    def product(name, i, src, bias, what, key):
        w, steps = weights[i][name]
        q = src["wide8" if name == "contract" else "q8"]
        v = (q.double() @ w.double().T) * src["scale"].double()[:, None] * steps.double()
        want = v + t64(bias)
        got = following(name)[key]
        close(got, want, to_type(want, 3 * U * v.abs() + U * want.abs()), what + name)  # the sum is exact
        return got

    def attention(q, k, v, got, what):
        want, bound = test_attention_gpu.reference(q, k, v, s.d ** -0.5, None, None, dtype)
        close(got.reshape(want.shape), want, bound, what)

    product_of, m = patches(p, image)
    got = following("patches")["x"]
    close(got, m, 4 * EPS * (product_of.abs() + m.abs()), "patches")  # a whole number, exact; a product and a sum
    m = got.double()
    rows = following("first")
    norm(m, torch.zeros_like(m), 0, rows, "first norm")
    for i, b in enumerate(p["blocks"]):
        at = "block %d: " % i
        qkv = product("qkv", i, rows, b["qkv"][1], at, "qkv")
        turned = (s.heads + s.kv) * s.d
        got = following("rotary")["qkv"]
        want, bound = test_rotary_gpu.reference(qkv[:, :turned].reshape(s.rows, -1, s.d), s.positions, (s.d // 4, s.d // 4), "interleaved", False, 10000.0)
        close(got[:, :turned].reshape(want.shape), want, to_type(want, bound), at + "rotary")
        assert torch.equal(got[:, turned:], qkv[:, turned:]), at + "the values changed"
        o = following("attention")["o"]
        attention(s.heads_of(got, 0, s.heads), s.heads_of(got, s.heads, s.kv), s.heads_of(got, s.heads + s.kv, s.kv), o, at + "attention")
        rows = following("quantize")
        same_rows(rows["q8"], rows["scale"], o.float(), at + "quantize")
        for j, name in enumerate(("project", "contract")):
            if name == "contract":
                wide = product("expand", i, rows, b["expand"][1], at, "wide")
                rows = following("quantize_wide")
                near_rows(rows["wide8"], rows["scale"], act64(wide.double(), "gelu"), act_error(wide.double()), at + "gelu")
            branch = product(name, i, rows, b[name][1], at, "branch").double()
            factor = t64(b["scale%d" % (1 + j)])
            z = factor * branch
            want = m + z
            error = 2 * U * z.abs() + 2 * U * (want.abs() + z.abs() + m.abs())
            rows = following("between")
            close(rows["x"], want, to_type(want, error, "f32"), at + "the sum into the map")
            norm(want, error, 2 * i + j + 1, rows, at + "norm %d" % (2 * i + j + 1))
            m = rows["x"].double()
    kv = product("kv", -1, rows, p["kv"][1], "", "kv")
    pooled = following("pool")["pooled"]
    attention(*s.pooled_operands(p, kv, dtype), pooled, "pool")
    classes, bias = t64(p["scores"][0]).to(TYPES[dtype]).double(), t64(p["scores"][1])
    want, size = pooled.double() @ classes.T + bias, pooled.double().abs() @ classes.abs().T + bias.abs()
    close(following("head")["scores"], want, to_type(want, (s.c + 2) * EPS * size, "f32"), "scores")
    assert next(calls, None) is None
