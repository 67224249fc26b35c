"""ctypes binding of the float operators (include/cldnn_hip_ops.h): group norm with an activation, matrix product with bias,
activation and residual, rotary positions, attention.

Only plumbing lives here.  An operator is made once for a shape and enqueued on its engine's stream; what it reads and writes is
device memory: a hip.Buffer, a torch tensor, anything else with a `ptr` or a `data_ptr()`, or an address.  A tensor has to be on the
engine's device or in pinned memory, of the operand's type (or uint8: plain memory), and either contiguous memory that is large enough, or laid out as the
operator's description says; a buffer has to be large enough; of an address nothing is known.  Work of other streams on that memory
has to be ordered by the caller (Engine.finish, events).
"""
import ctypes as C
import os

import numpy as np

from . import hip

LIB_PATH = os.path.join(os.path.dirname(hip.LIB_PATH), "libcldnn_hip_ops.so")

F32, F16, BF16, I32, NO_TYPE = hip.F32, 4, 5, hip.I32, hip.NO_TYPE
DT_NAME = {"f32": F32, "f16": F16, "bf16": BF16, "i32": I32}
TORCH_NAME = {F32: "torch.float32", F16: "torch.float16", BF16: "torch.bfloat16", I32: "torch.int32"}
SIZE = {F32: 4, F16: 2, BF16: 2, I32: 4}
POSITION_NAME = {"i32": I32, "f32": F32}
ACT_NAME = dict(hip.ACT_NAME, silu=4, gelu=5, gelu_tanh=6)
PAIRING_NAME = {"interleaved": 0, "halves": 1, "halves_per_axis": 2}
MAX_AXES = 4


class GroupNormDesc(C.Structure):
    _fields_ = [("input", hip.Tensor), ("output", hip.Tensor), ("groups", C.c_int32), ("epsilon", C.c_float), ("activation", C.c_int32),
                ("activation_m", C.c_float), ("activation_n", C.c_float)]


class MatmulDesc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("m", "n", "k", "dtype", "out_dtype", "residual_dtype", "has_bias")] + [
        (n, C.c_int64) for n in ("a_stride", "weights_stride", "out_stride", "residual_stride")] + [
        ("activation", C.c_int32), ("activation_m", C.c_float), ("activation_n", C.c_float),
        ("residual_activation", C.c_int32), ("residual_activation_m", C.c_float), ("residual_activation_n", C.c_float)]


class RotaryDesc(C.Structure):
    _fields_ = [("tokens", C.c_int64)] + [(n, C.c_int32) for n in ("q_heads", "k_heads", "head_size", "axes")] + [
        ("pairs", C.c_int32 * MAX_AXES), ("pairing", C.c_int32), ("shared_frequencies", C.c_int32), ("base", C.c_float)] + [
        (n, C.c_int32) for n in ("dtype", "position_dtype", "inverse")] + [(n, C.c_int64) for n in (
            "q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride",
            "q_out_token_stride", "q_out_head_stride", "k_out_token_stride", "k_out_head_stride")]


class AttentionDesc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("batch", "q_len", "kv_len", "q_heads", "kv_heads", "head_size", "dtype")] + [("scale", C.c_float)] + [
        (n, C.c_int32) for n in ("has_key_lengths", "bias_dtype")] + [(n, C.c_int64) for n in (
            "q_batch_stride", "q_token_stride", "q_head_stride", "k_batch_stride", "k_token_stride", "k_head_stride",
            "v_batch_stride", "v_token_stride", "v_head_stride", "out_batch_stride", "out_token_stride", "out_head_stride",
            "bias_batch_stride", "bias_head_stride", "bias_q_stride")]


class OperatorInfo(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("launches", "grid", "block", "lds_bytes")] + [
        (n, C.c_int64) for n in ("workspace_bytes", "ops", "bytes")] + [("kernel_name", C.c_char * 96)]


_P = C.c_void_p
# name -> (restype, argtypes); the single source of truth for what the library must export
SIGNATURES = {
    "cldnn_hip_operator_retain": (C.c_int32, [_P]),
    "cldnn_hip_operator_release": (C.c_int32, [_P]),
    "cldnn_hip_operator_get_info": (C.c_int32, [_P, C.POINTER(OperatorInfo)]),
    "cldnn_hip_operator_tensor_bytes": (C.c_size_t, [C.POINTER(hip.Tensor)]),
    "cldnn_hip_group_norm_create": (C.c_int32, [_P, C.POINTER(GroupNormDesc), C.POINTER(_P)]),
    "cldnn_hip_group_norm_enqueue": (C.c_int32, [_P] * 5),
    "cldnn_hip_matmul_create": (C.c_int32, [_P, C.POINTER(MatmulDesc), C.POINTER(_P)]),
    "cldnn_hip_matmul_enqueue": (C.c_int32, [_P] * 6),
    "cldnn_hip_rotary_create": (C.c_int32, [_P, C.POINTER(RotaryDesc), C.POINTER(_P)]),
    "cldnn_hip_rotary_enqueue": (C.c_int32, [_P] * 6),
    "cldnn_hip_attention_create": (C.c_int32, [_P, C.POINTER(AttentionDesc), C.POINTER(_P)]),
    "cldnn_hip_attention_enqueue": (C.c_int32, [_P] * 7),
}

_lib = None


def lib():
    """Load libcldnn_hip_ops.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        hip.lib()
        if not os.path.exists(LIB_PATH):
            raise OSError("%s is missing: run `python -c 'import __graft_entry__ as g; g.build()'`" % LIB_PATH)
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _lib = L
    return _lib


class Operand:
    """What an operator reads or writes at a pointer: elements of `shape`, `strides` elements apart, the first `offset` behind it."""

    def __init__(self, name, dtype, shape, strides, offset=0):
        self.name, self.dtype, self.shape, self.strides, self.offset = name, dtype, tuple(shape), tuple(strides), offset
        self.nbytes = (offset + sum((n - 1) * step for n, step in zip(shape, strides)) + 1) * SIZE[dtype]

    @staticmethod
    def dense(name, dtype, *shape):
        strides = [1]
        for n in reversed(shape[1:]):
            strides.insert(0, strides[0] * n)
        return Operand(name, dtype, shape, strides)

    def fits(self, t):
        """a strided tensor as the description has it"""
        return str(t.dtype) == TORCH_NAME[self.dtype] and tuple(t.shape) == self.shape and not self.offset and all(n == 1 or a == b for n, a, b in zip(self.shape, t.stride(), self.strides))


def _check_tensor(t, operand, device):
    def refuse(what):
        raise hip.HipError(-2, "%s: %s" % (operand.name, what))

    if t.get_device() != device and not (t.device.type == "cpu" and t.is_pinned()):
        refuse("a tensor on %s, not on the engine's device %d" % (t.device, device))
    if str(t.dtype) not in (TORCH_NAME[operand.dtype], "torch.uint8"):
        refuse("a tensor of %s" % t.dtype)
    if not t.is_contiguous() and not operand.fits(t):
        refuse("a tensor of shape %r and strides %r, described are %r and %r" % (tuple(t.shape), t.stride(), operand.shape, operand.strides))
    if t.is_contiguous() and t.nbytes < operand.nbytes:
        refuse("%d bytes, described are %d" % (t.nbytes, operand.nbytes))


def _address_of(operand, device):
    """The function that takes what is given for an operand and returns its address, or refuses it.  operand: None where the description
    has none, and what is given is not looked at."""
    if operand is None:
        return lambda x: None
    need, kind, dtype = operand.nbytes, None, None  # torch's, once one has come

    def address(x):
        # what is asked of each tensor is little, in the order of a tensor that fits: 0.2 us beside a launch of 3.5
        if x.__class__ is kind and x.dtype is dtype and x.get_device() == device and x.nbytes >= need and x.is_contiguous():
            return x.data_ptr()
        return checked(x)

    def checked(x):
        nonlocal kind, dtype
        if x is None or type(x) is int:
            return x
        if hasattr(x, "get_device"):
            _check_tensor(x, operand, device)
            if str(x.dtype) == TORCH_NAME[operand.dtype]:
                kind, dtype = type(x), x.dtype
            return x.data_ptr()
        if hasattr(x, "data_ptr"):
            return x.data_ptr()
        if getattr(x, "nbytes", need) < need:
            raise hip.HipError(-2, "%s: a buffer of %d bytes, described are %d" % (operand.name, x.nbytes, need))
        return x.ptr

    return address


def _type(dt):
    return DT_NAME[dt] if isinstance(dt, str) else dt


def _act(act):
    return ACT_NAME[act] if isinstance(act, str) else act


class Buffer:
    """Device memory for a tensor of the operators' types, zeros at first (a hip.Buffer knows the convolution path's types only)."""

    def __init__(self, engine, nbytes):
        self.engine, self.nbytes, self.h = engine, nbytes, None
        h = _P()
        hip.check(hip.lib().cldnn_hip_buffer_alloc(engine.h, nbytes, C.byref(h)))
        self.h = h

    @property
    def ptr(self):
        return hip.lib().cldnn_hip_buffer_device_ptr(self.h)

    def write(self, values, dtype):
        """numpy values, rounded to `dtype`; behind what the engine has been given so far"""
        a = to_type(values, dtype)
        assert a.nbytes <= self.nbytes, (a.nbytes, self.nbytes)
        hip.check(hip.lib().cldnn_hip_buffer_write(self.h, 0, a.ctypes.data, a.nbytes))
        return self

    def read(self, shape, dtype):
        """the first values as numpy float32 (i32: int32); waits for the engine"""
        n = {F32: np.float32, I32: np.int32, F16: np.float16, BF16: np.uint16}[_type(dtype)]
        a = np.empty(shape, n)
        assert a.nbytes <= self.nbytes, (a.nbytes, self.nbytes)
        hip.check(hip.lib().cldnn_hip_buffer_read(self.h, 0, a.ctypes.data, a.nbytes))
        if _type(dtype) == BF16:
            return (a.astype(np.uint32) << 16).view(np.float32)
        return a if _type(dtype) == I32 else a.astype(np.float32)

    def close(self):
        if self.h:
            hip.check(hip.lib().cldnn_hip_buffer_release(self.h))
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def to_type(values, dtype):
    """numpy array of the bits of `values` in an operator's type; bf16, which numpy has not, as uint16 rounded to nearest even"""
    dt = _type(dtype)
    if dt == BF16:
        with np.errstate(over="ignore"):
            single = np.ascontiguousarray(values, np.float32)
        bits = single.view(np.uint32)
        if np.asarray(values).dtype == np.float64:  # rounded to odd first, so that what follows is the one rounding
            rest = single != values
            bits = np.where(rest & np.isfinite(single), (bits - (np.abs(single) > np.abs(values))) | 1, bits).astype(np.uint32)
        rounded = ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
        return np.where(np.isnan(values), np.uint16(0x7fc0), rounded)
    return np.ascontiguousarray(values, {F32: np.float32, F16: np.float16, I32: np.int32}[dt])


class Operator:
    """What the operators have in common: the object behind the handle."""

    def __init__(self, engine, kind, desc):
        self.engine, self.desc, self.h = engine, desc, None
        h = _P()
        hip.check(getattr(lib(), "cldnn_hip_%s_create" % kind)(engine.h, C.byref(desc), C.byref(h)))
        self.h = h
        self._enqueue = getattr(lib(), "cldnn_hip_%s_enqueue" % kind)
        self._address = [_address_of(o, engine.device) for o in self._operands(desc)]  # in the entry point's order

    def info(self):
        i = OperatorInfo()
        hip.check(lib().cldnn_hip_operator_get_info(self.h, C.byref(i)))
        return i

    def close(self):
        if self.h:
            hip.check(lib().cldnn_hip_operator_release(self.h))
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def map_tensor(dtype, b, y, x, f, pad_y=0, pad_x=0, pad_f=0):
    """Channels-last map as a hip.Tensor: [b][pad + y + pad][pad + x + pad][f + pad_f] in memory."""
    t = hip.Tensor.make(_type(dtype), hip.BYXF, b, f, y, x, pad_y, pad_x)
    t.pad_hi_f = pad_f
    return t


def tensor_bytes(tensor):
    return lib().cldnn_hip_operator_tensor_bytes(C.byref(tensor))


def group_norm_desc(input, groups, *, out_dtype=None, output=None, epsilon=1e-5, act="none", act_m=0.0, act_n=0.0):
    """input: hip.Tensor in byxf; the output is a dense map of out_dtype (default: the input's type) unless `output` describes it."""
    d = GroupNormDesc()
    d.input = input
    d.output = output if output is not None else map_tensor(input.dtype if out_dtype is None else out_dtype, input.b, input.y, input.x, input.f)
    d.groups, d.epsilon = groups, epsilon
    d.activation, d.activation_m, d.activation_n = _act(act), act_m, act_n
    return d


class GroupNorm(Operator):
    """y = act((x - mean) / sqrt(variance + epsilon) * scale + shift), per image and group of features."""

    def __init__(self, engine, desc):
        super().__init__(engine, "group_norm", desc)

    @staticmethod
    def _operands(d):
        def plane(name, t):
            x = t.pad_lo_f + t.f + t.pad_hi_f
            y = x * (t.pad_lo_x + t.x + t.pad_hi_x)
            b = y * (t.pad_lo_y + t.y + t.pad_hi_y)
            return Operand(name, t.dtype, (t.b, t.y, t.x, t.f), (b, y, x, 1), t.pad_lo_b * b + t.pad_lo_y * y + t.pad_lo_x * x + t.pad_lo_f)

        return plane("input", d.input), Operand.dense("scale", F32, d.input.f), Operand.dense("shift", F32, d.input.f), plane("output", d.output)

    def enqueue(self, src, dst, scale=None, shift=None):
        of_src, of_scale, of_shift, of_dst = self._address
        status = self._enqueue(self.h, of_src(src), of_scale(scale), of_shift(shift), of_dst(dst))
        if status:
            hip.check(status)


def matmul_desc(m, n, k, dtype, *, out_dtype=None, bias=False, residual=False, residual_dtype=None, act="none", act_m=0.0, act_n=0.0,
                residual_act="none", residual_act_m=0.0, residual_act_n=0.0, a_stride=0, weights_stride=0, out_stride=0, residual_stride=0):
    """residual_dtype: the output's type unless given."""
    d = MatmulDesc()
    d.m, d.n, d.k, d.dtype = m, n, k, _type(dtype)
    d.out_dtype = d.dtype if out_dtype is None else _type(out_dtype)
    d.residual_dtype = NO_TYPE if not residual else d.out_dtype if residual_dtype is None else _type(residual_dtype)
    d.has_bias = int(bias)
    d.a_stride, d.weights_stride, d.out_stride, d.residual_stride = a_stride, weights_stride, out_stride, residual_stride
    d.activation, d.activation_m, d.activation_n = _act(act), act_m, act_n
    d.residual_activation, d.residual_activation_m, d.residual_activation_n = _act(residual_act), residual_act_m, residual_act_n
    return d


class Matmul(Operator):
    """out = act2(act(a weights^T + bias) + residual)."""

    def __init__(self, engine, desc):
        super().__init__(engine, "matmul", desc)

    @staticmethod
    def _operands(d):
        def matrix(name, dtype, rows, columns, stride):
            return Operand(name, dtype, (rows, columns), (stride or columns, 1))

        return (matrix("a", d.dtype, d.m, d.k, d.a_stride), matrix("weights", d.dtype, d.n, d.k, d.weights_stride), Operand.dense("bias", F32, d.n) if d.has_bias else None,
                matrix("residual", d.residual_dtype, d.m, d.n, d.residual_stride) if d.residual_dtype != NO_TYPE else None,
                matrix("output", d.out_dtype, d.m, d.n, d.out_stride))

    def enqueue(self, a, weights, out, bias=None, residual=None):
        of_a, of_weights, of_bias, of_residual, of_out = self._address
        status = self._enqueue(self.h, of_a(a), of_weights(weights), of_bias(bias), of_residual(residual), of_out(out))
        if status:
            hip.check(status)


def rotary_desc(tokens, q_heads, k_heads, head_size, pairs, dtype, *, pairing="interleaved", shared_frequencies=False, base=10000.0,
                position_dtype="i32", inverse=False, q_strides=(0, 0), k_strides=(0, 0), q_out_strides=(0, 0), k_out_strides=(0, 0)):
    """pairs: how many pairs of a head's values turn with each axis; strides: elements from (token to token, head to head)."""
    if not 1 <= len(pairs) <= MAX_AXES:
        raise ValueError("rotary: one to %d axes" % MAX_AXES)
    d = RotaryDesc()
    d.tokens, d.q_heads, d.k_heads, d.head_size, d.axes = tokens, q_heads, k_heads, head_size, len(pairs)
    d.pairs[:len(pairs)] = pairs
    d.pairing = PAIRING_NAME[pairing] if isinstance(pairing, str) else pairing
    d.shared_frequencies, d.base, d.dtype, d.inverse = int(shared_frequencies), base, _type(dtype), int(inverse)
    d.position_dtype = POSITION_NAME[position_dtype] if isinstance(position_dtype, str) else position_dtype
    (d.q_token_stride, d.q_head_stride), (d.k_token_stride, d.k_head_stride) = q_strides, k_strides
    (d.q_out_token_stride, d.q_out_head_stride), (d.k_out_token_stride, d.k_out_head_stride) = q_out_strides, k_out_strides
    return d


class Rotary(Operator):
    """Queries and keys turned by their tokens' positions along one axis per pair of values."""

    def __init__(self, engine, desc):
        super().__init__(engine, "rotary", desc)

    @staticmethod
    def _operands(d):
        def heads(name, n, token, head):
            return Operand(name, d.dtype, (d.tokens, n, d.head_size), (token or n * d.head_size, head or d.head_size, 1)) if n else None

        return (heads("q", d.q_heads, d.q_token_stride, d.q_head_stride), heads("k", d.k_heads, d.k_token_stride, d.k_head_stride),
                Operand.dense("positions", d.position_dtype, d.tokens, d.axes), heads("q output", d.q_heads, d.q_out_token_stride, d.q_out_head_stride),
                heads("k output", d.k_heads, d.k_out_token_stride, d.k_out_head_stride))

    def enqueue(self, q, k, positions, q_out, k_out):
        of_q, of_k, of_positions, of_q_out, of_k_out = self._address
        status = self._enqueue(self.h, of_q(q), of_k(k), of_positions(positions), of_q_out(q_out), of_k_out(k_out))
        if status:
            hip.check(status)


def attention_desc(batch, q_len, kv_len, q_heads, kv_heads, head_size, dtype, *, scale=0.0, key_lengths=False, bias_dtype=None, bias_shape=None,
                   q_strides=(0, 0, 0), k_strides=(0, 0, 0), v_strides=(0, 0, 0), out_strides=(0, 0, 0)):
    """bias_shape: (batch or 1, q_heads or 1, q_len or 1, kv_len) of a dense bias of bias_dtype (default: dtype); strides: elements
    from (batch to batch, token to token, head to head)."""
    d = AttentionDesc()
    d.batch, d.q_len, d.kv_len, d.q_heads, d.kv_heads, d.head_size, d.dtype = batch, q_len, kv_len, q_heads, kv_heads, head_size, _type(dtype)
    d.scale, d.has_key_lengths, d.bias_dtype = scale, int(key_lengths), NO_TYPE
    if bias_shape is not None:
        b, h, q, k = bias_shape
        if b not in (1, batch) or h not in (1, q_heads) or q not in (1, q_len) or k != kv_len:
            raise ValueError("attention: a bias of shape %r" % (bias_shape,))
        d.bias_dtype = d.dtype if bias_dtype is None else _type(bias_dtype)
        d.bias_batch_stride, d.bias_head_stride, d.bias_q_stride = h * q * k if b > 1 else 0, q * k if h > 1 else 0, k if q > 1 else 0
    d.q_batch_stride, d.q_token_stride, d.q_head_stride = q_strides
    d.k_batch_stride, d.k_token_stride, d.k_head_stride = k_strides
    d.v_batch_stride, d.v_token_stride, d.v_head_stride = v_strides
    d.out_batch_stride, d.out_token_stride, d.out_head_stride = out_strides
    return d


class Attention(Operator):
    """softmax(scale q k^T + bias) v over the keys below each image's length."""

    def __init__(self, engine, desc):
        super().__init__(engine, "attention", desc)

    @staticmethod
    def _operands(d):
        def tokens(name, length, heads, batch, token, head):
            token = token or heads * d.head_size
            return Operand(name, d.dtype, (d.batch, length, heads, d.head_size), (batch or length * token, token, head or d.head_size, 1))

        bias = (d.batch, d.q_heads, d.q_len, d.kv_len), (d.bias_batch_stride, d.bias_head_stride, d.bias_q_stride, 1)
        return (tokens("q", d.q_len, d.q_heads, d.q_batch_stride, d.q_token_stride, d.q_head_stride),
                tokens("k", d.kv_len, d.kv_heads, d.k_batch_stride, d.k_token_stride, d.k_head_stride),
                tokens("v", d.kv_len, d.kv_heads, d.v_batch_stride, d.v_token_stride, d.v_head_stride),
                Operand.dense("key_lengths", I32, d.batch) if d.has_key_lengths else None,
                Operand("bias", d.bias_dtype, *bias) if d.bias_dtype != NO_TYPE else None,
                tokens("output", d.q_len, d.q_heads, d.out_batch_stride, d.out_token_stride, d.out_head_stride))

    def enqueue(self, q, k, v, out, key_lengths=None, bias=None):
        of_q, of_k, of_v, of_lengths, of_bias, of_out = self._address
        status = self._enqueue(self.h, of_q(q), of_k(k), of_v(v), of_lengths(key_lengths), of_bias(bias), of_out(out))
        if status:
            hip.check(status)
