"""The image classifier with attention in int8 throughout: patches by an int8 convolution, transformer blocks whose products are of int8
tokens and weights, norms that write int8.

    image u8 -> convolution (stride = filter) -> map, f32, channels last
    block:  x += scale1 * project(attention(rotary(product(norm(x)))));  x += scale2 * contract(gelu(expand(norm(x))))
    scores = product(attention(one query, keys and values of norm(x)))

Norms are over a token's features; the sum into the map, its norm and the quantisation of what the next product reads are one call.  Each
token has a scale of its own, worked out on the way; each row of weights has one, worked out when the network is made.  Attention and
the scores, which are of one token to an image, stay in `dtype`.
"""
import numpy as np

from . import ops, ops_s8
from .image_attention_net import ImageAttentionNet


class ImageAttentionS8Net(ImageAttentionNet):
    """The network for one batch and image size, of image_attention_net.parameters(.., layer_scales=True)."""

    def __init__(self, engine, params, batch, height, width, dtype="f16"):
        p, e = params, engine
        self.engine, self.params, self.batch, self.dtype = e, p, batch, dtype
        c, heads, kv, patch = p["features"], p["heads"], p["kv_heads"], p["patch"]
        d, n = c // heads, (height // patch) * (width // patch)
        self.tokens, self._owned = n, []
        rows, qkv, size = batch * n, (heads + 2 * kv) * d, 2
        self._make_patches(height, width)

        # one operator per shape: blocks share them, and the buffers between them
        self._qkv, self._o, self._branch = self._memory(rows * qkv * size), self._memory(rows * c * size), self._memory(rows * c * size)
        self._wide = self._memory(rows * 4 * c * size)
        self._q8, self._wide8, self._scale = self._memory(rows * c), self._memory(rows * 4 * c), self._memory(rows * 4)
        self._first = self._keep(ops_s8.BlockNorm(e, ops_s8.block_norm_desc(rows, c, "f32", out_dtype="s8")))
        self._between = self._keep(ops_s8.BlockNorm(e, ops_s8.block_norm_desc(rows, c, "f32", branch_dtype=dtype, out_dtype="s8")))
        self._quantize = self._keep(ops_s8.Quantize(e, ops_s8.quantize_desc(rows, c, dtype)))
        self._quantize_wide = self._keep(ops_s8.Quantize(e, ops_s8.quantize_desc(rows, 4 * c, dtype, act="gelu")))
        self._product = {name: self._keep(ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(rows, out, k, out_dtype=dtype, bias=True)))
                         for name, out, k in (("qkv", qkv, c), ("project", c, c), ("expand", 4 * c, c), ("contract", c, 4 * c), ("kv", 2 * kv * d, c))}
        # queries, keys and values of a token lie side by side
        self._rotary = self._keep(ops.Rotary(e, ops.rotary_desc(rows, heads, kv, d, (d // 4, d // 4), dtype, q_strides=(qkv, d), k_strides=(qkv, d), q_out_strides=(qkv, d),
                                                                k_out_strides=(qkv, d))))
        self._attention = self._keep(ops.Attention(e, ops.attention_desc(batch, n, n, heads, kv, d, dtype, q_strides=(n * qkv, qkv, d), k_strides=(n * qkv, qkv, d),
                                                                         v_strides=(n * qkv, qkv, d))))
        self._k_at, self._v_at = heads * d * size, (heads + kv) * d * size

        # one query pools the map
        kvd = 2 * kv * d
        self._query = self._upload(np.broadcast_to(p["query"], (batch, heads, d)), dtype)
        self._pool = self._keep(ops.Attention(e, ops.attention_desc(batch, 1, n, heads, kv, d, dtype, k_strides=(n * kvd, kvd, d), v_strides=(n * kvd, kvd, d))))
        self._pooled, self._scores = self._memory(batch * c * size), self._memory(batch * p["classes"] * 4)
        self._head = self._keep(ops.Matmul(e, ops.matmul_desc(batch, p["classes"], c, dtype, out_dtype="f32", bias=True)))
        self._v_pool = kv * d * size

        def vectors(pair):
            return dict(weight=self._upload(pair[0], "f32"), bias=self._upload(pair[1], "f32"))

        self._blocks = [dict({k: vectors(b[k]) for k in ("norm1", "norm2")}, **{k: self._quantized(b[k]) for k in ("qkv", "project", "expand", "contract")},
                             **{k: self._upload(b[k], "f32") for k in ("scale1", "scale2")}) for b in p["blocks"]]
        self._last, self._kv = vectors(p["norm"]), self._quantized(p["kv"])
        self._classes = self._upload(p["scores"][0], dtype), self._upload(p["scores"][1], "f32")
        e.finish()

    def _quantized(self, pair):
        """Weights as int8 rows with a scale each, and their bias."""
        n, k = pair[0].shape
        plain = ops.Buffer(self.engine, n * k * 4).write(pair[0], "f32")
        op = ops_s8.Quantize(self.engine, ops_s8.quantize_desc(n, k, "f32"))
        weights, scales = self._memory(n * k), self._memory(n * 4)
        op.enqueue(plain, weights, scales)
        self.engine.finish()
        op.close()
        plain.close()
        return weights, scales, self._upload(pair[1], "f32")

    def _run_product(self, name, src, weights, dst):
        self._product[name].enqueue(src, weights[0], dst, self._scale, weights[1], weights[2])

    def enqueue(self):
        """One pass over the image that is in place; nothing is waited for."""
        self._run_patches()
        qkv, x = self._qkv.ptr, self._x
        norms = [norm for b in self._blocks for norm in (b["norm1"], b["norm2"])] + [self._last]
        self._first.enqueue(x, None, self._q8, out_scales=self._scale, **norms[0])
        for i, b in enumerate(self._blocks):
            self._run_product("qkv", self._q8, b["qkv"], self._qkv)
            self._rotary.enqueue(qkv, qkv + self._k_at, self._positions, qkv, qkv + self._k_at)
            self._attention.enqueue(qkv, qkv + self._k_at, qkv + self._v_at, self._o)
            self._quantize.enqueue(self._o, self._q8, self._scale)
            self._run_product("project", self._q8, b["project"], self._branch)
            self._between.enqueue(x, x, self._q8, branch=self._branch, post_weight=b["scale1"], out_scales=self._scale, **norms[2 * i + 1])
            self._run_product("expand", self._q8, b["expand"], self._wide)
            self._quantize_wide.enqueue(self._wide, self._wide8, self._scale)
            self._run_product("contract", self._wide8, b["contract"], self._branch)
            self._between.enqueue(x, x, self._q8, branch=self._branch, post_weight=b["scale2"], out_scales=self._scale, **norms[2 * i + 2])
        self._run_product("kv", self._q8, self._kv, self._qkv)
        self._pool.enqueue(self._query, qkv, qkv + self._v_pool, self._pooled)
        self._head.enqueue(self._pooled, self._classes[0], self._scores, self._classes[1])
