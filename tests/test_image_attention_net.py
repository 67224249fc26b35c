"""A network of the convolution path and the float operators together against its formula in 64 bits."""
import numpy as np
import pytest
import torch

from cldnn_amd import hip, image_attention_net as net, ops


def reference(p, image, y, x, groups=8):
    c, heads, kv = p["features"], p["heads"], p["kv_heads"]
    d, b, n = c // heads, len(image), y * x
    t = lambda a: torch.from_numpy(np.asarray(a)).double()  # noqa: E731
    q = p["patches"]
    m = torch.nn.functional.conv2d(t(image), t(q["w"]), stride=p["patch"]) * t(q["wqf"])[None, :, None, None] + t(q["bias"])[None, :, None, None]
    m = m.permute(0, 2, 3, 1).reshape(b, n, c)

    def norm(v, pair):
        g = v.reshape(b, n, groups, c // groups)
        g = (g - g.mean((1, 3), keepdim=True)) / torch.sqrt(g.var((1, 3), unbiased=False, keepdim=True) + 1e-5)
        return g.reshape(b, n, c) * t(pair[0]) + t(pair[1])

    def linear(v, pair):
        return v @ t(pair[0]).T + t(pair[1])

    def attend(q_, k_, v_):
        k_, v_ = (a.repeat_interleave(heads // kv, 2) for a in (k_, v_))
        s = torch.einsum("bqhd,bkhd->bhqk", q_, k_) / d ** 0.5
        return torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), v_).reshape(b, -1, c)

    rows, cols = torch.arange(n) // x, torch.arange(n) % x

    def turn(v):
        out = v.clone()
        for axis, pos in enumerate((rows, cols)):
            for j in range(d // 4):
                a = pos.double() * 10000.0 ** -(j / (d // 4))
                i = 2 * (axis * (d // 4) + j)
                cos, sin = torch.cos(a)[None, :, None], torch.sin(a)[None, :, None]
                out[..., i], out[..., i + 1] = v[..., i] * cos - v[..., i + 1] * sin, v[..., i + 1] * cos + v[..., i] * sin
        return out

    for blk in p["blocks"]:
        h = linear(norm(m, blk["norm1"]), blk["qkv"]).reshape(b, n, heads + 2 * kv, d)
        m = m + linear(attend(turn(h[:, :, :heads]), turn(h[:, :, heads:heads + kv]), h[:, :, heads + kv:]), blk["project"])
        v = linear(norm(m, blk["norm2"]), blk["expand"])
        m = m + linear(v * torch.special.ndtr(v), blk["contract"])
    h = linear(norm(m, p["norm"]), p["kv"]).reshape(b, n, 2 * kv, d)
    pooled = attend(t(p["query"]).expand(b, 1, heads, d), h[:, :, :kv], h[:, :, kv:])
    return linear(pooled[:, 0], p["scores"]).numpy()


def test_bf16_bits_round_to_nearest_even():
    values = np.array([1.0, 1.00390625, 1.01171875, -1.00390625, 3.4e38, np.inf, -np.inf, 0.0], np.float32)
    want = torch.from_numpy(values).bfloat16().view(torch.int16).numpy().view(np.uint16)
    assert np.array_equal(ops.to_type(values, "bf16"), want)
    assert ops.to_type(np.array([np.nan], np.float32), "bf16")[0] == 0x7fc0


def test_bf16_bits_of_64_bit_values_are_rounded_once():
    # next to the middle of two bf16 values, nearer than 32 bits can tell
    r = np.random.default_rng(3)
    middles = ((r.integers(0x0080, 0x7f00, 500).astype(np.uint32) << 16) | 0x8000).view(np.float32).astype(np.float64)
    for sign in (1, -1):
        for off, up in ((1 + 2.0 ** -40, True), (1 - 2.0 ** -40, False)):
            values = sign * middles * off
            bits = ops.to_type(values, "bf16").astype(np.uint32) << 16
            assert np.array_equal(np.abs(bits.view(np.float32)) > middles, np.full(500, up))
    assert np.array_equal(ops.to_type(middles, "bf16") & 1, np.zeros(500))  # the middle itself: to even
    assert np.array_equal(ops.to_type(np.array([1e300, -1e300, np.inf, np.nan, 0.0, -0.0, 1e-300]), "bf16"), np.array([0x7f80, 0xff80, 0x7f80, 0x7fc0, 0, 0x8000, 0], np.uint16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,half_ulp", [("f16", 2.0 ** -11), ("bf16", 2.0 ** -8)])
@pytest.mark.parametrize("batch,height,width,blocks", [(1, 56, 56, 1), (3, 72, 40, 2)])
def test_scores(batch, height, width, blocks, dtype, half_ulp):
    r = np.random.default_rng(batch)
    p = net.parameters(r, blocks=blocks)
    image = r.integers(0, 256, (batch, 3, height, width)).astype(np.uint8)
    eng = hip.Engine()
    model = net.ImageAttentionNet(eng, p, batch, height, width, dtype)
    got = model.run(image)
    assert np.array_equal(model.run(image), got), "the same image gives other scores"
    other = model.run(255 - image)
    assert not np.array_equal(other, got)
    # the same pass recorded once and enqueued with one call
    L, rec = hip.lib(), hip.C.c_void_p()
    hip.check(L.cldnn_hip_engine_record_begin(eng.h))
    model.enqueue()
    hip.check(L.cldnn_hip_engine_record_end(eng.h, hip.C.byref(rec)))
    for _ in range(3):
        model._plain.write_raw(image)
        hip.check(L.cldnn_hip_recording_enqueue(rec))
        assert np.array_equal(model._scores.read(got.shape, "f32"), got)
    hip.check(L.cldnn_hip_recording_release(rec))
    model.close()
    eng.close()
    want = reference(p, image, height // 8, width // 8)
    # each block rounds to the type six times on the way of a value (and its weights twice more per product), the head four times;
    # norms and sums keep relative errors within twice their size
    roundings = 2 * (10 * blocks + 6)
    assert np.linalg.norm(got - want) <= roundings * half_ulp * np.linalg.norm(want)
