"""Performance cases of the operators that an image network with attention needs beside its convolutions: group norm with an
activation on channels-last maps, the matrix product with bias, activation and residual in its epilogue, rotary positions with
several axes, and attention over image tokens.

`run` computes an operator in its plain form, from elementary torch operations in 32 bits, or (where `own` is true) makes the
calls of the library: an object per operator, made once from a description of the shapes, and one enqueue per pass on tensors
that are on the device.  Outputs go into buffers that the caller owns and are left on the queue.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPSILON = 1e-5
BASE = 10000.0
MOST_VALUES = 16 * 224 * 224 * 64    # of a normalised map
MOST_BYTES = 2 * (25088 * (1024 + 4096) + 1024 * 4096)
MOST_PRODUCT = 2 * 25088 * 1024 * 4096
MOST_ATTENTION = 4 * 4 * 8 * 3136 * 3136 * 64
MOST_SCORES = 4 * 8 * 3136 * 3136    # the plain form holds them all
MOST_ROTARY = 8 * 56 * 56 * 20 * 128


def _norm(name, batch, y, x, features, groups, dtype, act, out=None):
    return dict(name=name, kind="norm", batch=batch, y=y, x=x, features=features, groups=groups, dtype=dtype, out=out or dtype, act=act)


def _product(name, m, k, n, dtype, act="none", bias=True, residual=False, out=None):
    return dict(name=name, kind="product", m=m, k=k, n=n, dtype=dtype, out=out or dtype, act=act, bias=bias, residual=residual)


def _rotary(name, batch, axes, t, y, x, q_heads, k_heads, head, dtype, pairing, shared=False):
    return dict(name=name, kind="rotary", batch=batch, axes=axes, t=t, y=y, x=x, q_heads=q_heads, k_heads=k_heads, head=head, dtype=dtype,
                pairing=pairing, shared=shared)


def _attention(name, batch, q_len, kv_len, q_heads, kv_heads, head, dtype, ragged=False, bias=False):
    return dict(name=name, kind="attention", batch=batch, q_len=q_len, kv_len=kv_len, q_heads=q_heads, kv_heads=kv_heads, head=head, dtype=dtype,
                ragged=ragged, bias=bias)


def listed():
    return [
        # the last map of a ResNet-50-shaped network, one image at a time: the smallest call
        _norm("norm_7x7_b1", 1, 7, 7, 2048, 32, "bf16", "silu"),
        # an image that is not square and widths that are no multiples of a vector: 7 features to a group
        _norm("norm_odd_b3", 3, 31, 45, 84, 12, "f32", "relu", out="f16"),
        # the first maps of a VGG-16-shaped network at its benchmark batch: the largest
        _norm("norm_224_b16", 16, 224, 224, 64, 32, "f16", "silu"),
        # the classifier of one image: latency
        _product("product_scores_m1", 1, 2048, 1000, "bf16", out="f32"),
        # a projection back into a map of odd size, with the residual
        _product("product_odd_residual", 1395, 84, 108, "f16", "relu", residual=True),
        # VGG-16's first classifier layer at its benchmark batch: the weights are the work
        _product("product_fc6_m16", 16, 25088, 4096, "f16", "relu"),
        # the expansion of a transformer block over 32 maps of 28x28 tokens: the matrix cores are the work
        _product("product_expand_28_b32", 25088, 1024, 4096, "bf16", "gelu"),
        # the tokens of one 14x14 map with two axes: latency
        _rotary("rotary_14x14_b1", 1, 2, 1, 14, 14, 16, 16, 64, "bf16", "halves_per_axis"),
        # a clip of eight 56x56 maps with time, height and width, keys shared by four heads
        _rotary("rotary_8x56x56", 1, 3, 8, 56, 56, 16, 4, 128, "f16", "interleaved"),
        # windows of 7x7 tokens with a relative-position bias, some of whose entries separate regions of a shifted window
        _attention("attention_windows_49_b64", 64, 49, 49, 4, 4, 32, "f16", bias=True),
        # every token of a 56x56 map against every other: the matrix cores are the work
        _attention("attention_56x56_b4", 4, 3136, 3136, 8, 8, 64, "bf16"),
        # one query that pools the pixels of images of different sizes, up to 224x224: a single token over long keys
        _attention("attention_pool_224_b2", 2, 1, 50176, 8, 2, 128, "bf16", ragged=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width of a layer: mostly a multiple of 8."""
    n = _log(rng, lo, hi)
    return min(hi, 8 * -(-n // 8)) if rng.random() < 0.7 else n


def draw(rng):
    kind = rng.choice(("norm", "product", "rotary", "attention"))
    half = rng.choice(("f16", "bf16"))
    while True:
        if kind == "norm":
            per, groups = _log(rng, 1, 64), rng.choice((1, 8, 16, 32, rng.randint(1, 40)))
            y = _log(rng, 4, 224)
            x = y if rng.random() < 0.5 else _log(rng, 4, 224)
            dtype = rng.choice(("f16", "bf16", "f32"))
            c = _norm("", _log(rng, 1, 32), y, x, per * groups, groups, dtype, rng.choice(("silu", "silu", "none", "relu", "gelu")),
                      rng.choice((dtype, dtype, half)))
            ok = per * groups >= 8 and c["batch"] * y * x * per * groups <= MOST_VALUES
        elif kind == "product":
            m, k, n = _log(rng, 1, 32768), _width(rng, 32, 16384), _width(rng, 32, 8192)
            c = _product("", m, k, n, half, rng.choice(("none", "relu", "gelu", "silu")), rng.random() < 0.8, rng.random() < 0.4, rng.choice((half, half, "f32")))
            ok = 2 * m * k * n <= MOST_PRODUCT
        elif kind == "rotary":
            axes = rng.choice((1, 2, 2, 3))
            t, y = _log(rng, 1, 16) if axes == 3 else 1, _log(rng, 4, 128)
            x = y if rng.random() < 0.5 else _log(rng, 4, 128)
            kv = _log(rng, 1, 16)
            dtype = rng.choice(("f16", "bf16", "f32"))
            c = _rotary("", _log(rng, 1, 16), axes, t, y, x, kv * rng.choice((1, 1, 2, 4)), kv, rng.choice((32, 64, 80, 96, 128)), dtype,
                        rng.choice(("interleaved", "halves", "halves_per_axis")), rng.random() < 0.3)
            ok = c["batch"] * t * y * x * (c["q_heads"] + kv) * c["head"] <= MOST_ROTARY
        else:
            kv = _log(rng, 1, 16)
            q_len = rng.choice((1, _log(rng, 1, 4096), _log(rng, 1, 4096)))
            kv_len = q_len if q_len > 1 and rng.random() < 0.5 else _log(rng, 1, 50176)
            c = _attention("", _log(rng, 1, 64), q_len, kv_len, kv * rng.choice((1, 1, 1, 4)), kv, rng.choice((32, 40, 64, 64, 72, 80, 96, 128, 128, 160)),
                           half, rng.random() < 0.4, rng.random() < 0.3)
            scores = c["batch"] * c["q_heads"] * q_len * kv_len
            ok = (scores <= MOST_SCORES and 4 * scores * c["head"] <= MOST_ATTENTION and c["batch"] * kv_len * kv * c["head"] <= 1 << 26
                  and c["q_heads"] * q_len * kv_len <= 1 << 26)
        if ok and work(c)["bytes"] <= MOST_BYTES:
            del c["name"]
            return c


# ------------------------------------------------------------------------------------------------------------------ inputs
def _sections(case):
    """Pairs of a head's values that turn with each axis: time has the fewest."""
    pairs = case["head"] // 2
    if case["axes"] == 1:
        return (pairs,)
    if case["axes"] == 2:
        return (pairs // 2, pairs - pairs // 2)
    t = pairs // 4
    return (t, (pairs - t) // 2, pairs - t - (pairs - t) // 2)


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    def empty(*shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    kind, dtype, s = case["kind"], TYPES[case["dtype"]], dict(case)
    if kind == "norm":
        c, shape = case["features"], (case["batch"], case["y"], case["x"], case["features"])
        # a map's features differ in size and have means of their own
        s["input"] = torch.addcmul(normal(c), normal(*shape), normal(c).exp()).to(dtype)
        s["scale"], s["shift"] = 1 + normal(c, scale=0.2), normal(c, scale=0.2)
        s["output"] = empty(*shape, dtype=TYPES[case["out"]])
    elif kind == "product":
        m, k, n = case["m"], case["k"], case["n"]
        s["a"], s["weights"] = normal(m, k, dtype=dtype), normal(n, k, scale=k ** -0.5, dtype=dtype)
        s["bias_values"] = normal(n, scale=0.2) if case["bias"] else None
        s["residual_values"] = normal(m, n, dtype=TYPES[case["out"]]) if case["residual"] else None
        s["output"] = empty(m, n, dtype=TYPES[case["out"]])
    elif kind == "rotary":
        tokens = case["batch"] * case["t"] * case["y"] * case["x"]
        s["q"], s["k"] = (normal(tokens, case[h], case["head"], dtype=dtype) for h in ("q_heads", "k_heads"))
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        # the grid of the tokens, cut from a larger one at a place of its own for each image
        extents = {1: ("x",), 2: ("y", "x"), 3: ("t", "y", "x")}[case["axes"]]
        if case["axes"] == 1:
            grid = torch.arange(case["t"] * case["y"] * case["x"], device="cuda")[:, None]
        else:
            grid = torch.cartesian_prod(*(torch.arange(case[e], device="cuda") for e in extents))
        first = torch.randint(0, 64, (case["batch"], 1, case["axes"]), generator=g, device="cuda")
        s["positions"] = (grid[None] + first).reshape(tokens, case["axes"]).to(torch.int32).contiguous()
    else:
        b, lq, lk, h, kv, d = (case[n] for n in ("batch", "q_len", "kv_len", "q_heads", "kv_heads", "head"))
        s["q"], s["k"], s["v"] = normal(b, lq, h, d, dtype=dtype), normal(b, lk, kv, d, dtype=dtype), normal(b, lk, kv, d, dtype=dtype)
        s["lengths"] = torch.randint(lk // 2, lk + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
        s["bias_values"] = None
        if case["bias"]:
            bias = normal(h, lq, lk)
            region_q, region_k = torch.arange(lq, device="cuda") * 3 // (2 * lq), torch.arange(lk, device="cuda") * 3 // (2 * lk)
            apart = (region_q[:, None] != region_k[None]) & (torch.arange(h, device="cuda") % 2 == 1)[:, None, None]
            s["bias_values"] = bias.masked_fill(apart, -math.inf).to(dtype)
        s["output"] = empty(b, lq, h, d, dtype=dtype)
    if own:
        s["operator"] = _operator(case)
    return s


# ------------------------------------------------------------------------------------------------------- the library's calls
_engines = []


def _operator(case):
    """The object that a program makes once for a shape and keeps."""
    from cldnn_amd import hip, ops

    if not _engines:  # one queue per process, as an application keeps it
        _engines.append(hip.Engine(0))
    e, c = _engines[0], case
    if c["kind"] == "norm":
        return ops.GroupNorm(e, ops.group_norm_desc(ops.map_tensor(c["dtype"], c["batch"], c["y"], c["x"], c["features"]), c["groups"], out_dtype=c["out"],
                                                    epsilon=EPSILON, act=c["act"]))
    if c["kind"] == "product":
        return ops.Matmul(e, ops.matmul_desc(c["m"], c["n"], c["k"], c["dtype"], out_dtype=c["out"], act=c["act"], bias=c["bias"], residual=c["residual"]))
    if c["kind"] == "rotary":
        return ops.Rotary(e, ops.rotary_desc(c["batch"] * c["t"] * c["y"] * c["x"], c["q_heads"], c["k_heads"], c["head"], _sections(c), c["dtype"],
                                             pairing=c["pairing"], shared_frequencies=c["shared"], base=BASE))
    return ops.Attention(e, ops.attention_desc(c["batch"], c["q_len"], c["kv_len"], c["q_heads"], c["kv_heads"], c["head"], c["dtype"],
                                               key_lengths=c["ragged"], bias_shape=(1, c["q_heads"], c["q_len"], c["kv_len"]) if c["bias"] else None))


def _run_own(s):
    op = s["operator"]
    if s["kind"] == "norm":
        op.enqueue(s["input"], s["output"], s["scale"], s["shift"])
        return s["output"]
    if s["kind"] == "product":
        op.enqueue(s["a"], s["weights"], s["output"], s["bias_values"], s["residual_values"])
        return s["output"]
    if s["kind"] == "rotary":
        op.enqueue(s["q"], s["k"], s["positions"], s["q_out"], s["k_out"])
        return s["q_out"], s["k_out"]
    op.enqueue(s["q"], s["k"], s["v"], s["output"], s["lengths"], s["bias_values"])
    return s["output"]


# -------------------------------------------------------------------------------------------------------------- plain forms
def _act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return torch.clamp(v, min=0) if act == "relu" else v


def _plain_norm(s):
    x = s["input"].float().reshape(s["batch"], s["y"] * s["x"], s["groups"], -1)
    mean = x.mean(dim=(1, 3), keepdim=True)
    x = x - mean
    x = x * torch.rsqrt((x * x).mean(dim=(1, 3), keepdim=True) + EPSILON)
    return _act(x.reshape(s["input"].shape) * s["scale"] + s["shift"], s["act"]).to(TYPES[s["out"]])


def _plain_product(s):
    v = torch.matmul(s["a"].float(), s["weights"].float().t())
    if s["bias_values"] is not None:
        v = v + s["bias_values"]
    v = _act(v, s["act"])
    if s["residual_values"] is not None:
        v = v + s["residual_values"].float()
    return v.to(TYPES[s["out"]])


def _pair_index(s, device):
    """For each pair of a head: where its two values lie, which axis turns it and the exponent of its frequency."""
    sections, pairs = _sections(s), s["head"] // 2
    i = torch.arange(pairs, device=device)
    ends = torch.tensor(sections, device=device).cumsum(0)
    axis = (i[:, None] >= ends).sum(1)
    size = torch.tensor(sections, device=device)[axis]
    start = ends[axis] - size
    within = i - start
    first, second = {"interleaved": (2 * i, 2 * i + 1), "halves": (i, i + pairs), "halves_per_axis": (i + start, i + start + size)}[s["pairing"]]
    return first, second, axis, (i / pairs if s["shared"] else within / size)


def _plain_rotary(s):
    first, second, axis, exponent = _pair_index(s, s["q"].device)
    angle = s["positions"].float()[:, axis] * torch.pow(BASE, -exponent.float())
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]

    def turn(v):
        v, out = v.float(), torch.empty(v.shape, device=v.device)
        a, b = v[..., first], v[..., second]
        out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
        return out

    return turn(s["q"]).to(s["q"].dtype), turn(s["k"]).to(s["k"].dtype)


def _plain_attention(s):
    b, lq, lk, h, kv, d = (s[n] for n in ("batch", "q_len", "kv_len", "q_heads", "kv_heads", "head"))
    share = torch.arange(h, device="cuda") // (h // kv)
    q, k, v = s["q"].float().transpose(1, 2), s["k"].float()[:, :, share].transpose(1, 2), s["v"].float()[:, :, share].transpose(1, 2)
    scores = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    if s["bias_values"] is not None:
        scores = scores + s["bias_values"].float()
    if s["lengths"] is not None:
        scores = torch.where(torch.arange(lk, device="cuda") < s["lengths"][:, None, None, None], scores, -math.inf)
    most = scores.amax(dim=3, keepdim=True)
    p = torch.exp(scores - torch.where(most == -math.inf, 0.0, most))
    total = p.sum(dim=3, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return o.transpose(1, 2).to(s["q"].dtype).contiguous()


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "product": _plain_product, "rotary": _plain_rotary, "attention": _plain_attention}[state["kind"]](state)


# --------------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    size = SIZE[c["dtype"]]
    if c["kind"] == "norm":
        n = c["batch"] * c["y"] * c["x"] * c["features"]
        return {"bytes": n * (size + SIZE[c["out"]]) + 8 * c["features"], "flops": 10 * n}
    if c["kind"] == "product":
        m, k, n = c["m"], c["k"], c["n"]
        return {"bytes": (m * k + n * k) * size + (4 * n if c["bias"] else 0) + m * n * SIZE[c["out"]] * (2 if c["residual"] else 1), "flops": 2 * m * n * k}
    if c["kind"] == "rotary":
        tokens = c["batch"] * c["t"] * c["y"] * c["x"]
        n = tokens * (c["q_heads"] + c["k_heads"]) * c["head"]
        return {"bytes": 2 * n * size + 4 * tokens * c["axes"], "flops": 3 * n}
    b, lq, lk, h = (c[n] for n in ("batch", "q_len", "kv_len", "q_heads"))
    keys = lk * 0.75 if c["ragged"] else lk  # lengths are spread evenly over the upper half
    return {"bytes": size * (2 * b * lq * h + 2 * b * keys * c["kv_heads"]) * c["head"] + (size * h * lq * keys if c["bias"] else 0),
            "flops": 4 * b * h * lq * keys * c["head"]}


# --------------------------------------------------------------------------------------------------------- values in 64 bits
def _exact_act(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    return torch.where(v > 0, v, torch.zeros_like(v)) if act == "relu" else v


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        out = torch.empty(s["input"].shape, dtype=torch.float64, device="cuda")
        per = case["features"] // case["groups"]
        for b in range(case["batch"]):
            for f in range(0, case["features"], per):
                x = s["input"][b, :, :, f:f + per].double()
                variance, mean = torch.var_mean(x, correction=0)
                out[b, :, :, f:f + per] = _exact_act((x - mean) / torch.sqrt(variance + EPSILON) * s["scale"][f:f + per].double() + s["shift"][f:f + per].double(), case["act"])
        return out
    if case["kind"] == "product":
        v = s["a"].double() @ s["weights"].double().T
        v = _exact_act(v if s["bias_values"] is None else v + s["bias_values"].double(), case["act"])
        return v if s["residual_values"] is None else v + s["residual_values"].double()
    if case["kind"] == "rotary":
        outs, at, pairs = [s["q"].double(), s["k"].double()], 0, case["head"] // 2
        for axis, count in enumerate(_sections(case)):
            for j in range(count):
                frequency = BASE ** -((at + j) / pairs if case["shared"] else j / count)
                turn = torch.polar(torch.ones(len(s["q"]), dtype=torch.float64, device="cuda"), s["positions"][:, axis].double() * frequency)[:, None]
                lo, hi = {"interleaved": (2 * (at + j), 2 * (at + j) + 1), "halves": (at + j, at + j + pairs),
                          "halves_per_axis": (2 * at + j, 2 * at + j + count)}[case["pairing"]]
                for o in outs:
                    z = torch.complex(o[..., lo].clone(), o[..., hi].clone()) * turn
                    o[..., lo], o[..., hi] = z.real, z.imag
            at += count
        return tuple(outs)
    out = torch.zeros(s["output"].shape, dtype=torch.float64, device="cuda")
    group = case["q_heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        keys = case["kv_len"] if s["lengths"] is None else int(s["lengths"][b])
        for h in range(case["q_heads"] if keys else 0):
            score = s["q"][b, :, h].double() @ s["k"][b, :keys, h // group].double().T / math.sqrt(case["head"])
            if s["bias_values"] is not None:
                score += s["bias_values"][h, :, :keys].double()
            out[b, :, h] = torch.nan_to_num(torch.softmax(score, dim=1), nan=0.0) @ s["v"][b, :keys, h // group].double()
    return out
