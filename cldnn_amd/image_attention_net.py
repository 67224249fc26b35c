"""An image classifier with attention, from the convolution path and the float operators together: patches by one int8
convolution, transformer blocks over their map, one query that pools it, scores.

    image u8 -> convolution (stride = filter) -> map, f32, channels last
    block:  x += project(attention(rotary(product(norm(x)))));  x += contract(gelu(expand(norm(x))))
    scores = product(attention(one query, keys and values of norm(x)))

The map between blocks is f32; what the matrix cores read is of `dtype`.  Positions are the patches' rows and columns.
"""
import numpy as np

from . import hip, ops


def parameters(r, features=64, heads=4, kv_heads=2, blocks=2, patch=8, classes=10, layer_scales=False):
    """Random parameters with the factors that keep a signal alive.  r: numpy Generator.  layer_scales: a block's two branches have a factor
    for each feature."""
    d = features // heads

    def weights(n, k, scale=1.0):
        return (r.standard_normal((n, k)) * scale * k ** -0.5).astype(np.float32)

    def vector(n, mean=0.0):
        return (mean + 0.2 * r.standard_normal(n)).astype(np.float32)

    def norm():
        return vector(features, 1.0), vector(features)

    k = 3 * patch * patch
    p = dict(features=features, heads=heads, kv_heads=kv_heads, patch=patch, classes=classes, patches=dict(
        w=r.integers(-127, 128, (features, 3, patch, patch)).astype(np.int8), bias=vector(features),
        wqf=np.full(features, 1.0 / (np.sqrt(k) * 147.4 * 73.3), np.float32)), blocks=[])
    for _ in range(blocks):
        p["blocks"].append(dict(
            norm1=norm(), qkv=(weights((heads + 2 * kv_heads) * d, features), vector((heads + 2 * kv_heads) * d)), project=(weights(features, features, 0.5), vector(features)),
            norm2=norm(), expand=(weights(4 * features, features), vector(4 * features)), contract=(weights(features, 4 * features, 0.5), vector(features))))
    p.update(norm=norm(), kv=(weights(2 * kv_heads * d, features), vector(2 * kv_heads * d)), query=r.standard_normal((heads, d)).astype(np.float32),
             scores=(weights(classes, features), vector(classes)))
    if layer_scales:
        for b in p["blocks"]:
            b.update(scale1=vector(features, 0.7), scale2=vector(features, 0.7))
    return p


class ImageAttentionNet:
    """The network for one batch and image size: everything is allocated and laid out here, a run only launches."""

    def __init__(self, engine, params, batch, height, width, dtype="f16", groups=8):
        p, e = params, engine
        self.engine, self.params, self.batch, self.dtype = e, p, batch, dtype
        c, heads, kv, patch = p["features"], p["heads"], p["kv_heads"], p["patch"]
        d, y, x = c // heads, height // patch, width // patch
        self.tokens = n = y * x
        rows, qkv = batch * n, (heads + 2 * kv) * d
        self._owned = []

        self._make_patches(height, width)

        # one operator per shape: blocks share them, and the buffers between them
        size = 2
        self._h, self._qkv = self._memory(rows * c * size), self._memory(rows * qkv * size)
        self._o, self._wide = self._memory(rows * c * size), self._memory(rows * 4 * c * size)
        self._norm = self._keep(ops.GroupNorm(e, ops.group_norm_desc(ops.map_tensor("f32", batch, y, x, c), groups, out_dtype=dtype)))
        self._product = {name: self._keep(ops.Matmul(e, ops.matmul_desc(rows, out, k, dtype, bias=True, **more))) for name, out, k, more in (
            ("qkv", qkv, c, {}), ("project", c, c, dict(out_dtype="f32", residual=True)), ("expand", 4 * c, c, dict(act="gelu")),
            ("contract", c, 4 * c, dict(out_dtype="f32", residual=True)), ("kv", 2 * kv * d, c, {}))}
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

        def norm(pair):
            return self._upload(pair[0], "f32"), self._upload(pair[1], "f32")

        def linear(pair):
            return self._upload(pair[0], dtype), self._upload(pair[1], "f32")

        self._blocks = [{k: (norm if k.startswith("norm") else linear)(v) for k, v in b.items()} for b in p["blocks"]]
        self._last, self._kv, self._classes = norm(p["norm"]), linear(p["kv"]), linear(p["scores"])
        e.finish()

    def _make_patches(self, height, width):
        """The int8 convolution from the image to the map, and the patches' positions."""
        e, p, batch = self.engine, self.params, self.batch
        c, patch = p["features"], p["patch"]
        y, x = height // patch, width // patch
        self.image = hip.Tensor.make("u8", "bfyx", batch, 3, height, width)
        self._plain, self._blocked = self._keep(hip.Buffer(e, self.image)), self._keep(hip.Buffer(e, hip.Tensor.make("u8", "fs_b_yx_fsv16", batch, 3, height, width)))
        q = p["patches"]
        desc = hip.conv_desc(self._blocked.tensor, q["w"].shape, "f32", stride=(patch, patch), bias_dt=hip.F32, has_wqf=True)
        self._conv = self._keep(hip.Conv(e, desc, q["w"], q["bias"], q["wqf"]))
        self._patches, self._x = self._keep(hip.Buffer(e, desc.output)), self._keep(hip.Buffer(e, hip.Tensor.make("f32", "byxf", batch, c, y, x)))
        grid = np.stack(np.meshgrid(np.arange(y), np.arange(x), indexing="ij"), -1).reshape(1, y * x, 2)
        self._positions = self._upload(np.broadcast_to(grid, (batch, y * x, 2)), "i32")

    def _run_patches(self):
        hip.reorder(self.engine, self._plain, self._blocked)
        self._conv.enqueue(self._blocked, self._patches)
        hip.reorder(self.engine, self._patches, self._x)

    def _keep(self, x):
        self._owned.append(x)
        return x

    def _memory(self, nbytes):
        return self._keep(ops.Buffer(self.engine, nbytes))

    def _upload(self, values, dtype):
        return self._memory(ops.to_type(values, dtype).nbytes).write(values, dtype)

    def _run_product(self, name, src, weights, dst, residual=None):
        self._product[name].enqueue(src, weights[0], dst, weights[1], residual)

    def enqueue(self):
        """One pass over the image that is in place; nothing is waited for."""
        self._run_patches()
        qkv, x = self._qkv.ptr, self._x
        for b in self._blocks:
            self._norm.enqueue(x, self._h, *b["norm1"])
            self._run_product("qkv", self._h, b["qkv"], self._qkv)
            self._rotary.enqueue(qkv, qkv + self._k_at, self._positions, qkv, qkv + self._k_at)
            self._attention.enqueue(qkv, qkv + self._k_at, qkv + self._v_at, self._o)
            self._run_product("project", self._o, b["project"], x, x)
            self._norm.enqueue(x, self._h, *b["norm2"])
            self._run_product("expand", self._h, b["expand"], self._wide)
            self._run_product("contract", self._wide, b["contract"], x, x)
        self._norm.enqueue(x, self._h, *self._last)
        self._run_product("kv", self._h, self._kv, self._qkv)
        self._pool.enqueue(self._query, qkv, qkv + self._v_pool, self._pooled)
        self._head.enqueue(self._pooled, self._classes[0], self._scores, self._classes[1])

    def run(self, image):
        """image: numpy u8 [batch][3][height][width] -> scores, float32 [batch][classes]"""
        self._plain.write_raw(image)
        self.enqueue()
        return self._scores.read((self.batch, self.params["classes"]), "f32")

    def close(self):
        self.engine.finish()
        for x in reversed(self._owned):
            x.close()
        self._owned = []
