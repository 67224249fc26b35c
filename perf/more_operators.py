"""Performance cases of the operators that bring the transformer blocks of an image network into int8: the matrix product of int8
operands with a scale for each token and channel, the quantisation of rows to int8 behind an activation, and the norms before and
after a block with its gate and residual scale, whose result may be int8 too.

`run` computes an operator in its plain form, from elementary torch operations in 32 bits, or (where `own` is true) makes the
calls of the library: an object per operator, made once from a description of the shapes, and one enqueue each per pass on tensors
that are on the device.  Outputs go into buffers that the caller owns and are left on the queue.  The int8 values between two
operators of one pass stay on the device; what comes back are the results and the scales.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4, "s8": 1}
EPSILON = 1e-5
MOST_PRODUCT = 2 * 25088 * 1024 * 4096
MOST_BYTES = 25088 * 4096 * 2 + 4096 * 1024 + 25088 * 1024 * 4


def _product(name, m, k, n, out, act="none", bias=True, residual=False, token_scales=True):
    return dict(name=name, kind="product", m=m, k=k, n=n, out=out, act=act, bias=bias, residual=residual, token_scales=token_scales)


def _linear(name, m, k, n, dtype, out, act="none", gated=False, factors=False, bias=True, residual=False):
    return dict(name=name, kind="linear", m=m, k=k, n=n, dtype=dtype, out=out, act=act, gated=gated, factors=factors, bias=bias, residual=residual)


def _norm(name, batch, tokens, features, dtype, branch, out, norm="layer", post="none", gate=False, modulation=None, residual_scale=1.0):
    return dict(name=name, kind="norm", batch=batch, tokens=tokens, features=features, dtype=dtype, branch=branch, out=out, norm=norm, post=post, gate=gate,
                modulation=modulation, residual_scale=residual_scale)


def _block(name, batch, tokens, features, n, dtype, branch, out, norm="layer", post="none", gate=False, modulation=None, residual_scale=1.0):
    return dict(_norm(name, batch, tokens, features, dtype, branch, "s8", norm, post, gate, modulation, residual_scale), kind="block", n=n, product_out=out)


def listed():
    return [
        # the classifier of 32 images whose features are quantised: latency
        _product("product_scores_b32", 32, 2048, 1000, "f32"),
        # a projection back into a map of odd size, rows of 84 bytes, with the residual
        _product("product_odd_residual", 1395, 84, 108, "f16", "relu", residual=True),
        # VGG-16's first classifier layer at its benchmark batch: the weights are the work
        _product("product_fc6_m16", 16, 25088, 4096, "f16", "relu"),
        # the expansion of a transformer block over 32 maps of 28x28 tokens: the matrix cores are the work
        _product("product_expand_28_b32", 25088, 1024, 4096, "bf16", "gelu"),
        # one pooled token through a quantised layer: two small calls, latency
        _linear("linear_scores_m1", 1, 2048, 1000, "bf16", "bf16"),
        # a gated expansion of odd width, contracted
        _linear("linear_odd_gated", 1395, 84, 108, "f16", "f16", "silu", gated=True, factors=True),
        # the contraction of a transformer block over 32 maps: the wide map behind its activation becomes int8, then the product
        _linear("linear_contract_28_b32", 25088, 4096, 1024, "f16", "f16", "gelu", residual=True),
        # one pooled token: latency
        _norm("norm_token_b1", 1, 1, 2048, "f32", None, "f32"),
        # norms on both sides of a block of odd width and an image that is not square
        _norm("norm_odd_b3", 3, 1395, 84, "f32", "f16", "f32", "rms", "rms", residual_scale=0.5),
        # the residual stream between two blocks that are conditioned per image: gate, scale and shift; bound by memory
        _norm("norm_adaptive_28_b32", 32, 784, 1024, "bf16", "bf16", "bf16", gate=True, modulation="bf16"),
        # wide tokens of one map, norms on both sides, a stream in 32 bits
        _norm("norm_wide_28_b1", 1, 784, 8192, "f32", "f16", "f16", "rms", "rms"),
        # a block's entry in int8: the residual, the norm that writes int8, queries of 8 heads and keys and values of 2
        _block("block_qkv_28_b8", 8, 784, 1024, 1536, "f32", "f16", "f16", gate=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width of a layer: mostly a multiple of 16."""
    n = _log(rng, lo, hi)
    return min(hi, 16 * -(-n // 16)) if rng.random() < 0.7 else n


def _residual(rng, features):
    dtype, half = rng.choice(("f32", "f16", "bf16")), rng.choice(("f16", "bf16"))
    branch = rng.choice((dtype, dtype if dtype != "f32" else half, None))
    tokens = _log(rng, 1, 3136)
    return (_log(rng, 1, 32), tokens, features, dtype, branch), dict(
        norm=rng.choice(("layer", "rms")), post=rng.choice(("none", "none", "layer", "rms")) if branch else "none", gate=bool(branch) and rng.random() < 0.4,
        modulation=rng.choice((None, None, dtype, "f32")), residual_scale=rng.choice((1.0, 1.0, 0.5)) if branch else 1.0)


def draw(rng):
    kind = rng.choice(("product", "linear", "norm", "block"))
    half = rng.choice(("f16", "bf16"))
    while True:
        if kind == "product":
            m, k, n = _log(rng, 1, 32768), _width(rng, 32, 25088), _width(rng, 32, 8192)
            c = _product("", m, k, n, rng.choice((half, half, "f32")), rng.choice(("none", "relu", "gelu", "silu")), rng.random() < 0.8, rng.random() < 0.4, rng.random() < 0.9)
        elif kind == "linear":
            m, k, n = _log(rng, 1, 32768), _width(rng, 32, 16384), _width(rng, 32, 8192)
            c = _linear("", m, k, n, rng.choice((half, half, "f32")), half, rng.choice(("none", "relu", "gelu", "silu")), rng.random() < 0.3, rng.random() < 0.3,
                        rng.random() < 0.8, rng.random() < 0.4)
        elif kind == "norm":
            a, more = _residual(rng, _width(rng, 32, 16384))
            c = _norm("", *a, rng.choice((half, half, "f32")), **more)
        else:
            a, more = _residual(rng, _width(rng, 32, 8192))
            c = _block("", *a[:3], _width(rng, 32, 8192), *a[3:], half, **more)
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_PRODUCT:
            del c["name"]
            return c


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    def empty(*shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    def rows(count, width):
        """rows of their own sizes as int8, and what a step of each stands for"""
        v = torch.randn(count, width, generator=g, device="cuda")
        most = v.abs().amax(1, keepdim=True)
        return torch.round(v * (127 / most)).to(torch.int8), (most[:, 0] / 127 * normal(count, scale=0.5).exp())

    def stream(count, width):
        """tokens of a residual stream: features differ in size and have means of their own"""
        return torch.addcmul(normal(width, scale=0.5), normal(count, width), normal(width, scale=0.5).exp())

    kind, s = case["kind"], dict(case)
    if kind in ("product", "linear"):
        m, k, n = case["m"], case["k"], case["n"]
        if kind == "product":
            s["a"], s["a_scales"] = rows(m, k)
            if not case["token_scales"]:
                s["a_scales"] = s["a_scales"][:1].contiguous()
        else:
            s["input"] = stream(m, k * (2 if case["gated"] else 1)).to(TYPES[case["dtype"]])
            s["channel_factors"] = normal(k, scale=0.3).exp() if case["factors"] else None
            s["quantized"], s["a_scales"] = empty(m, k, dtype=torch.int8), empty(m, dtype=torch.float32)
        s["residual_values"] = normal(m, n, dtype=TYPES[case["out"]]) if case["residual"] else None
        out = case["out"]
    else:
        m, k = case["batch"] * case["tokens"], case["features"]
        s["x"], s["x_out"] = stream(m, k).to(TYPES[case["dtype"]]), None
        s["branch_values"] = s["post_weight"] = s["post_bias"] = s["gate_values"] = s["scale"] = s["shift"] = None
        if case["branch"]:
            s["branch_values"], s["x_out"] = stream(m, k).to(TYPES[case["branch"]]), empty(m, k, dtype=TYPES[case["dtype"]])
            s["post_weight"] = 0.5 + normal(k, scale=0.1)
            s["post_bias"] = normal(k, scale=0.1) if case["post"] == "layer" else None
        modulation = TYPES[case["modulation"] or "f32"]
        if case["gate"]:
            s["gate_values"] = normal(case["batch"], k, dtype=modulation)
        if case["modulation"]:
            s["scale"], s["shift"] = normal(case["batch"], k, scale=0.3, dtype=modulation), normal(case["batch"], k, scale=0.3, dtype=modulation)
        s["weight"], s["bias_values"] = 1 + normal(k, scale=0.2), normal(k, scale=0.2) if case["norm"] == "layer" else None
        if kind == "norm":
            s["output"] = empty(m, k, dtype=TYPES[case["out"]])
        else:
            s["quantized"], s["a_scales"] = empty(m, k, dtype=torch.int8), empty(m, dtype=torch.float32)
            n, out = case["n"], case["product_out"]
    if kind != "norm":
        s["weights"], s["weights_scales"] = rows(n, k)
        s["weights_scales"] = s["weights_scales"] * k ** -0.5
        s["product_bias"] = normal(n, scale=0.2) if case.get("bias", True) else None
        s["output"] = empty(m, n, dtype=TYPES[out])
    if own:
        s["operators"] = _operators(case)
    return s


# ------------------------------------------------------------------------------------------------------- the library's calls
_engines = []


def _operators(c):
    """The objects that a program makes once for a shape and keeps."""
    from cldnn_amd import hip, ops_s8

    if not _engines:  # one queue per process, as an application keeps it
        _engines.append(hip.Engine(0))
    e, made = _engines[0], {}
    m, k = (c["m"], c["k"]) if "m" in c else (c["batch"] * c["tokens"], c["features"])
    if c["kind"] == "linear":
        made["quantize"] = ops_s8.Quantize(e, ops_s8.quantize_desc(m, k, c["dtype"], act=c["act"], gated=c["gated"], factors=c["factors"]))
    if c["kind"] in ("norm", "block"):
        modulation = (c["modulation"] or "f32") if c["gate"] or c["modulation"] else None
        made["norm"] = ops_s8.BlockNorm(e, ops_s8.block_norm_desc(m, k, c["dtype"], branch_dtype=c["branch"], out_dtype=c["out"], norm=c["norm"], post=c["post"], epsilon=EPSILON,
                                                                  post_epsilon=EPSILON, residual_scale=c["residual_scale"], tokens_per_image=c["tokens"],
                                                                  modulation_dtype=modulation))
    if c["kind"] == "product":
        made["product"] = ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(m, c["n"], k, out_dtype=c["out"], a_scales="each" if c["token_scales"] else "one", act=c["act"], bias=c["bias"],
                                                                   residual=c["residual"]))
    elif c["kind"] == "linear":
        made["product"] = ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(m, c["n"], k, out_dtype=c["out"], bias=c["bias"], residual=c["residual"]))
    elif c["kind"] == "block":
        made["product"] = ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(m, c["n"], k, out_dtype=c["product_out"], bias=True))
    return made


def _run_norm(s, out, out_scales=None):
    s["operators"]["norm"].enqueue(s["x"], s["x_out"], out, branch=s["branch_values"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate_values"],
                                   weight=s["weight"], bias=s["bias_values"], scale=s["scale"], shift=s["shift"], out_scales=out_scales)


def _run_own(s):
    made = s["operators"]
    if s["kind"] == "product":
        made["product"].enqueue(s["a"], s["weights"], s["output"], s["a_scales"], s["weights_scales"], s["product_bias"], s["residual_values"])
        return s["output"]
    if s["kind"] == "linear":
        made["quantize"].enqueue(s["input"], s["quantized"], s["a_scales"], s["channel_factors"])
        made["product"].enqueue(s["quantized"], s["weights"], s["output"], s["a_scales"], s["weights_scales"], s["product_bias"], s["residual_values"])
        return {"scales": s["a_scales"], "out": s["output"]}
    if s["kind"] == "norm":
        _run_norm(s, s["output"])
        return {"x": s["x_out"], "out": s["output"]}
    _run_norm(s, s["quantized"], s["a_scales"])
    made["product"].enqueue(s["quantized"], s["weights"], s["output"], s["a_scales"], s["weights_scales"], s["product_bias"])
    return {"x": s["x_out"], "scales": s["a_scales"], "out": s["output"]}


# -------------------------------------------------------------------------------------------------------------- plain forms
def _act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return torch.clamp(v, min=0) if act == "relu" else v


def _plain_quantize(v):
    most = v.abs().amax(1, keepdim=True)
    return torch.round(v * torch.where(most > 0, 127 / most, 0.0)), most[:, 0] / 127


def _plain_product(s, a, a_scales, act, out):
    v = torch.matmul(a, s["weights"].float().t()) * a_scales[:, None] * s["weights_scales"]
    if s["product_bias"] is not None:
        v = v + s["product_bias"]
    v = _act(v, act)
    if s.get("residual_values") is not None:
        v = v + s["residual_values"].float()
    return v.to(TYPES[out])


def _plain_linear(s):
    v = s["input"].float()
    v = _act(v[:, :s["k"]], s["act"]) * v[:, s["k"]:] if s["gated"] else _act(v, s["act"])
    if s["channel_factors"] is not None:
        v = v * s["channel_factors"]
    q, scales = _plain_quantize(v)
    return {"scales": scales, "out": _plain_product(s, q, scales, "none", s["out"])}


def _plain_normalised(v, kind):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    return v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPSILON)


def _per_token(s, v):
    return v.float()[:, None].expand(-1, s["tokens"], -1).reshape(-1, s["features"])


def _plain_norm(s):
    x = s["x"].float()
    if s["branch_values"] is not None:
        z = _plain_normalised(s["branch_values"].float(), s["post"]) * s["post_weight"]
        if s["post_bias"] is not None:
            z = z + s["post_bias"]
        if s["gate_values"] is not None:
            z = z * _per_token(s, s["gate_values"])
        x = s["residual_scale"] * x + z
    h = _plain_normalised(x, s["norm"]) * s["weight"]
    if s["bias_values"] is not None:
        h = h + s["bias_values"]
    if s["scale"] is not None:
        h = h * (1 + _per_token(s, s["scale"])) + _per_token(s, s["shift"])
    stream = None if s["branch_values"] is None else x.to(s["x"].dtype)
    if s["kind"] == "norm":
        return {"x": stream, "out": h.to(TYPES[s["out"]])}
    q, scales = _plain_quantize(h)
    return {"x": stream, "scales": scales, "out": _plain_product(s, q, scales, "none", s["product_out"])}


def run(state):
    if own:
        return _run_own(state)
    if state["kind"] == "product":
        return _plain_product(state, state["a"].float(), state["a_scales"], state["act"], state["out"])
    return _plain_linear(state) if state["kind"] == "linear" else _plain_norm(state)


# --------------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] in ("product", "linear"):
        m, k, n = c["m"], c["k"], c["n"]
        size = 1 if c["kind"] == "product" else SIZE[c["dtype"]] * (2 if c["gated"] else 1)
        return {"bytes": m * k * size + n * k + 4 * (m + n) + (4 * n if c["bias"] else 0) + m * n * SIZE[c["out"]] * (2 if c["residual"] else 1), "flops": 2 * m * n * k}
    m, k = c["batch"] * c["tokens"], c["features"]
    per_image = (SIZE[c["modulation"] or "f32"] * ((2 if c["modulation"] else 0) + c["gate"])) * c["batch"] * k
    moved = m * k * (SIZE[c["dtype"]] + (SIZE[c["branch"]] + SIZE[c["dtype"]] if c["branch"] else 0)) + per_image + 8 * k
    if c["kind"] == "norm":
        return {"bytes": moved + m * k * SIZE[c["out"]], "flops": 20 * m * k}
    return {"bytes": moved + 4 * m + c["n"] * k + m * c["n"] * SIZE[c["product_out"]], "flops": 2 * m * c["n"] * k}


# --------------------------------------------------------------------------------------------------------- values in 64 bits
def _exact_act(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    return torch.where(v > 0, v, torch.zeros_like(v)) if act == "relu" else v


def _exact_rows(v):
    step = torch.linalg.vector_norm(v, math.inf, dim=1) / 127
    return torch.round(v / torch.where(step > 0, step, 1.0)[:, None]), step


def _exact_layer(s, q, step):
    v = (q @ s["weights"].double().T) * torch.outer(step.double().expand(len(q)), s["weights_scales"].double())
    return v if s["product_bias"] is None else v + s["product_bias"].double()


def _exact_unit(v, kind):
    if kind == "none":
        return v
    if kind == "layer":
        variance, mean = torch.var_mean(v, dim=1, correction=0, keepdim=True)
        return (v - mean) / torch.sqrt(variance + EPSILON)
    return v / torch.sqrt(torch.linalg.vector_norm(v, dim=1, keepdim=True) ** 2 / v.shape[1] + EPSILON)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "product":
        v = _exact_act(_exact_layer(s, s["a"].double(), s["a_scales"]), case["act"])
        return v if s["residual_values"] is None else v + s["residual_values"].double()
    if case["kind"] == "linear":
        first, *second = s["input"].double().split(case["k"], dim=1)
        v = _exact_act(first, case["act"])
        for factor in second + ([] if s["channel_factors"] is None else [s["channel_factors"].double()]):
            v = v * factor
        q, step = _exact_rows(v)
        v = _exact_layer(s, q, step)
        return {"scales": step, "out": v if s["residual_values"] is None else v + s["residual_values"].double()}
    image = torch.arange(case["batch"], device="cuda").repeat_interleave(case["tokens"])
    x, stream = s["x"].double(), None
    if case["branch"]:
        z = _exact_unit(s["branch_values"].double(), case["post"]) * s["post_weight"].double()
        z = z if s["post_bias"] is None else z + s["post_bias"].double()
        stream = x = case["residual_scale"] * x + (z if s["gate_values"] is None else z * s["gate_values"].double()[image])
    h = _exact_unit(x, case["norm"]) * s["weight"].double()
    h = h if s["bias_values"] is None else h + s["bias_values"].double()
    h = h if s["scale"] is None else h + h * s["scale"].double()[image] + s["shift"].double()[image]
    if case["kind"] == "norm":
        return {"x": stream, "out": h}
    q, step = _exact_rows(h)
    return {"x": stream, "scales": step, "out": _exact_layer(s, q, step)}
