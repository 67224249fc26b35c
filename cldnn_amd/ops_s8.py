"""ctypes binding of the int8 operators (include/cldnn_hip_ops_s8.h): rows quantised with a scale each, the matrix product of int8
operands with scales for each token and channel, the norms before and after a block with its gate and residual scale.

Only plumbing lives here; objects, operands and what is checked of them are those of the float operators (ops.py).
"""
import ctypes as C
import os

from . import hip, ops

LIB_PATH = os.path.join(os.path.dirname(hip.LIB_PATH), "libcldnn_hip_ops_s8.so")

SCALES_NAME = {None: 0, "one": 1, "each": 2}
NORM_NAME = {"none": 0, "layer": 1, "rms": 2}


class QuantizeDesc(C.Structure):
    _fields_ = [("rows", C.c_int64)] + [(n, C.c_int32) for n in ("features", "dtype", "gated", "has_factors", "activation")] + [
        ("activation_m", C.c_float), ("activation_n", C.c_float), ("in_stride", C.c_int64), ("out_stride", C.c_int64)]


class MatmulS8Desc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("m", "n", "k", "a_scales", "weights_scales", "out_dtype", "residual_dtype", "has_bias")] + [
        (n, C.c_int64) for n in ("a_stride", "weights_stride", "out_stride", "residual_stride")] + [
        ("activation", C.c_int32), ("activation_m", C.c_float), ("activation_n", C.c_float),
        ("residual_activation", C.c_int32), ("residual_activation_m", C.c_float), ("residual_activation_n", C.c_float)]


class BlockNormDesc(C.Structure):
    _fields_ = [("tokens", C.c_int64)] + [(n, C.c_int32) for n in (
        "features", "tokens_per_image", "dtype", "branch_dtype", "out_dtype", "modulation_dtype", "norm", "post")] + [
        (n, C.c_float) for n in ("epsilon", "post_epsilon", "residual_scale")] + [
        (n, C.c_int64) for n in ("x_stride", "branch_stride", "y_stride", "out_stride", "gate_stride", "scale_stride", "shift_stride")]


_P = C.c_void_p
# name -> (restype, argtypes); the single source of truth for what the library must export
SIGNATURES = {
    "cldnn_hip_quantize_create": (C.c_int32, [_P, C.POINTER(QuantizeDesc), C.POINTER(_P)]),
    "cldnn_hip_quantize_enqueue": (C.c_int32, [_P] * 5),
    "cldnn_hip_matmul_s8_create": (C.c_int32, [_P, C.POINTER(MatmulS8Desc), C.POINTER(_P)]),
    "cldnn_hip_matmul_s8_enqueue": (C.c_int32, [_P] * 8),
    "cldnn_hip_block_norm_create": (C.c_int32, [_P, C.POINTER(BlockNormDesc), C.POINTER(_P)]),
    "cldnn_hip_block_norm_enqueue": (C.c_int32, [_P] * 13),
}

_lib = None


def lib():
    """Load libcldnn_hip_ops_s8.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        ops.lib()
        if not os.path.exists(LIB_PATH):
            raise OSError("%s is missing: run `python -c 'import __graft_entry__ as g; g.build()'`" % LIB_PATH)
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _lib = L
    return _lib


class Operator(ops.Operator):
    """An operator whose entry points are in this library."""

    _library = staticmethod(lib)


def _rows(name, dtype, rows, columns, stride):
    return ops.Operand(name, dtype, (rows, columns), (stride or columns, 1))


def quantize_desc(rows, features, dtype, *, act="none", act_m=0.0, act_n=0.0, gated=False, factors=False, in_stride=0, out_stride=0):
    """features: of the output; a gated input has twice as many, the second half the factors of the first."""
    d = QuantizeDesc()
    d.rows, d.features, d.dtype, d.gated, d.has_factors = rows, features, ops._type(dtype), int(gated), int(factors)
    d.activation, d.activation_m, d.activation_n = ops._act(act), act_m, act_n
    d.in_stride, d.out_stride = in_stride, out_stride
    return d


class Quantize(Operator):
    """Rows of act(x) * factors, or act(x) * gate * factors, as int8 with a scale each."""

    def __init__(self, engine, desc):
        super().__init__(engine, "quantize", desc)

    @staticmethod
    def _operands(d):
        return (_rows("input", d.dtype, d.rows, d.features * (2 if d.gated else 1), d.in_stride), ops.Operand.dense("factors", ops.F32, d.features) if d.has_factors else None,
                _rows("output", hip.S8, d.rows, d.features, d.out_stride), ops.Operand.dense("scales", ops.F32, d.rows))

    def enqueue(self, src, dst, scales, factors=None):
        of_src, of_factors, of_dst, of_scales = self._address
        status = self._enqueue(self.h, of_src(src), of_factors(factors), of_dst(dst), of_scales(scales))
        if status:
            hip.check(status)


def matmul_s8_desc(m, n, k, *, out_dtype="f32", a_scales="each", weights_scales="each", bias=False, residual=False, residual_dtype=None, act="none", act_m=0.0, act_n=0.0,
                   residual_act="none", residual_act_m=0.0, residual_act_n=0.0, a_stride=0, weights_stride=0, out_stride=0, residual_stride=0):
    """a_scales, weights_scales: None, "one" or "each" (row); residual_dtype: the output's type unless given."""
    d = MatmulS8Desc()
    d.m, d.n, d.k, d.out_dtype = m, n, k, ops._type(out_dtype)
    d.a_scales, d.weights_scales = (s if type(s) is int else SCALES_NAME[s] for s in (a_scales, weights_scales))
    d.residual_dtype = ops.NO_TYPE if not residual else d.out_dtype if residual_dtype is None else ops._type(residual_dtype)
    d.has_bias = int(bias)
    d.a_stride, d.weights_stride, d.out_stride, d.residual_stride = a_stride, weights_stride, out_stride, residual_stride
    d.activation, d.activation_m, d.activation_n = ops._act(act), act_m, act_n
    d.residual_activation, d.residual_activation_m, d.residual_activation_n = ops._act(residual_act), residual_act_m, residual_act_n
    return d


class MatmulS8(Operator):
    """out = act2(act(a weights^T * a_scales * weights_scales + bias) + residual), a and weights int8."""

    def __init__(self, engine, desc):
        super().__init__(engine, "matmul_s8", desc)

    @staticmethod
    def _operands(d):
        def scales(name, kind, rows):
            return ops.Operand.dense(name, ops.F32, rows if kind == SCALES_NAME["each"] else 1) if kind else None

        return (_rows("a", hip.S8, d.m, d.k, d.a_stride), _rows("weights", hip.S8, d.n, d.k, d.weights_stride), scales("a_scales", d.a_scales, d.m),
                scales("weights_scales", d.weights_scales, d.n), ops.Operand.dense("bias", ops.F32, d.n) if d.has_bias else None,
                _rows("residual", d.residual_dtype, d.m, d.n, d.residual_stride) if d.residual_dtype != ops.NO_TYPE else None,
                _rows("output", d.out_dtype, d.m, d.n, d.out_stride))

    def enqueue(self, a, weights, out, a_scales=None, weights_scales=None, bias=None, residual=None):
        of_a, of_weights, of_a_scales, of_weights_scales, of_bias, of_residual, of_out = self._address
        status = self._enqueue(self.h, of_a(a), of_weights(weights), of_a_scales(a_scales), of_weights_scales(weights_scales), of_bias(bias), of_residual(residual), of_out(out))
        if status:
            hip.check(status)


def block_norm_desc(tokens, features, dtype, *, branch_dtype=None, out_dtype=None, norm="layer", post="none", epsilon=1e-5, post_epsilon=1e-5, residual_scale=1.0,
                    tokens_per_image=0, modulation_dtype=None, x_stride=0, branch_stride=0, y_stride=0, out_stride=0, gate_stride=0, scale_stride=0, shift_stride=0):
    """dtype: the stream's; branch_dtype: None: no branch; out_dtype: a type, "s8", or None: only the stream is wanted (norm="none" then);
    modulation_dtype: of gate, scale and shift, None: none of them.  norm, post: "layer", "rms" or "none"."""
    d = BlockNormDesc()

    def type_of(dt):
        return ops.NO_TYPE if dt is None else ops._type(dt)

    d.tokens, d.features, d.tokens_per_image = tokens, features, tokens_per_image
    d.dtype, d.branch_dtype, d.out_dtype, d.modulation_dtype = type_of(dtype), type_of(branch_dtype), type_of(out_dtype), type_of(modulation_dtype)
    d.norm, d.post = (NORM_NAME[n] if isinstance(n, str) else n for n in (norm, post))
    d.epsilon, d.post_epsilon, d.residual_scale = epsilon, post_epsilon, residual_scale
    d.x_stride, d.branch_stride, d.y_stride, d.out_stride = x_stride, branch_stride, y_stride, out_stride
    d.gate_stride, d.scale_stride, d.shift_stride = gate_stride, scale_stride, shift_stride
    return d


class BlockNorm(Operator):
    """y = residual_scale * x + gate * (post(branch) * post_weight + post_bias);  out = (norm(y) * weight + bias) * (1 + scale) + shift."""

    def __init__(self, engine, desc):
        super().__init__(engine, "block_norm", desc)

    @staticmethod
    def _operands(d):
        branch, out, modulated = d.branch_dtype != ops.NO_TYPE, d.out_dtype != ops.NO_TYPE, d.modulation_dtype != ops.NO_TYPE
        images = -(-d.tokens // d.tokens_per_image) if d.tokens_per_image else 1

        def tokens(name, dtype, stride, has=True):
            return _rows(name, dtype, d.tokens, d.features, stride) if has else None

        def image(name, stride, has):
            return _rows(name, d.modulation_dtype, images, d.features, stride) if modulated and has else None

        def features(name, has):
            return ops.Operand.dense(name, ops.F32, d.features) if has else None

        return (tokens("x", d.dtype, d.x_stride), tokens("branch", d.branch_dtype, d.branch_stride, branch), features("post_weight", branch), features("post_bias", branch),
                image("gate", d.gate_stride, branch), features("weight", out), features("bias", out), image("scale", d.scale_stride, out), image("shift", d.shift_stride, out),
                tokens("y", d.dtype, d.y_stride, branch), tokens("output", d.out_dtype, d.out_stride, out),
                ops.Operand.dense("out_scales", ops.F32, d.tokens) if d.out_dtype == hip.S8 else None)

    def enqueue(self, x, y=None, out=None, *, branch=None, post_weight=None, post_bias=None, gate=None, weight=None, bias=None, scale=None, shift=None, out_scales=None):
        """y: the stream behind the block, which may be x itself; None: not wanted."""
        of = self._address
        # what is not given, most of it in most calls, is not asked for: 0.4 us of 5.2
        status = self._enqueue(
            self.h, of[0](x), None if branch is None else of[1](branch), None if post_weight is None else of[2](post_weight), None if post_bias is None else of[3](post_bias),
            None if gate is None else of[4](gate), None if weight is None else of[5](weight), None if bias is None else of[6](bias), None if scale is None else of[7](scale),
            None if shift is None else of[8](shift), None if y is None else of[9](y), None if out is None else of[10](out), None if out_scales is None else of[11](out_scales))
        if status:
            hip.check(status)
