"""The classifier with int8 products against its formula in 64 bits, with and without the quantisation."""
import numpy as np
import pytest
import torch

import test_image_attention_net as float_net
from cldnn_amd import hip, image_attention_net as net, image_attention_s8_net as s8_net


def reference(p, image, y, x, quantize):
    """scores, and the crest (largest over root mean square of a row) of each quantised operand on the way.  quantize: rows of products'
    operands are rounded to 127 steps either way, as the operators do."""
    c, heads, kv = p["features"], p["heads"], p["kv_heads"]
    d, b, n = c // heads, len(image), y * x
    t = lambda a: torch.from_numpy(np.asarray(a)).double()  # noqa: E731
    q = p["patches"]
    m = torch.nn.functional.conv2d(t(image), t(q["w"]), stride=p["patch"]) * t(q["wqf"])[None, :, None, None] + t(q["bias"])[None, :, None, None]
    m = m.permute(0, 2, 3, 1).reshape(b, n, c)
    crests = []

    def rows(v):
        most = v.abs().amax(-1, keepdim=True)
        crests.append(float((most / v.square().mean(-1, keepdim=True).sqrt()).max()))
        return torch.round(v * 127 / most) * most / 127 if quantize else v

    def norm(v, pair):
        return (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-5) * t(pair[0]) + t(pair[1])

    def linear(v, pair):
        return rows(v) @ rows(t(pair[0])).T + t(pair[1])

    def attend(q_, k_, v_):
        k_, v_ = (a.repeat_interleave(heads // kv, 2) for a in (k_, v_))
        s = torch.einsum("bqhd,bkhd->bhqk", q_, k_) / d ** 0.5
        return torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), v_).reshape(b, -1, c)

    cols = torch.arange(n) % x

    def turn(v):
        out = v.clone()
        for axis, pos in enumerate((torch.arange(n) // x, cols)):
            for j in range(d // 4):
                a = pos.double() * 10000.0 ** -(j / (d // 4))
                i = 2 * (axis * (d // 4) + j)
                cos, sin = torch.cos(a)[None, :, None], torch.sin(a)[None, :, None]
                out[..., i], out[..., i + 1] = v[..., i] * cos - v[..., i + 1] * sin, v[..., i + 1] * cos + v[..., i] * sin
        return out

    for blk in p["blocks"]:
        h = linear(norm(m, blk["norm1"]), blk["qkv"]).reshape(b, n, heads + 2 * kv, d)
        m = m + t(blk["scale1"]) * linear(attend(turn(h[:, :, :heads]), turn(h[:, :, heads:heads + kv]), h[:, :, heads + kv:]), blk["project"])
        v = linear(norm(m, blk["norm2"]), blk["expand"])
        m = m + t(blk["scale2"]) * linear(v * torch.special.ndtr(v), blk["contract"])
    h = linear(norm(m, p["norm"]), p["kv"]).reshape(b, n, 2 * kv, d)
    pooled = attend(t(p["query"]).expand(b, 1, heads, d), h[:, :, :kv], h[:, :, kv:])
    return (pooled[:, 0] @ t(p["scores"][0]).T + t(p["scores"][1])).numpy(), crests


def noise(crests):
    """What the quantisation may do to the scores, relative: a rounding is spread evenly over a step, crest / 127 of a row's root mean square,
    which is 1 / sqrt(12) of it; independent ones add by their squares; norms and sums keep relative errors within twice their size."""
    return 2 * np.sqrt(sum((k / 127) ** 2 / 12 for k in crests))


def test_layer_scales_leave_the_other_parameters():
    a, b = net.parameters(np.random.default_rng(4)), net.parameters(np.random.default_rng(4), layer_scales=True)
    assert np.array_equal(a["scores"][0], b["scores"][0]) and np.array_equal(a["blocks"][1]["contract"][0], b["blocks"][1]["contract"][0])
    assert "scale1" not in a["blocks"][0] and b["blocks"][1]["scale2"].shape == (64,)


def test_the_formulas_agree_up_to_the_quantisation():
    r = np.random.default_rng(2)
    p = net.parameters(r, layer_scales=True)
    image = r.integers(0, 256, (2, 3, 48, 40)).astype(np.uint8)
    exact, crests = reference(p, image, 6, 5, False)
    rounded, _ = reference(p, image, 6, 5, True)
    assert len(crests) == 2 * (4 * 2 + 1)
    assert 0 < np.linalg.norm(rounded - exact) <= 2 * noise(crests) * np.linalg.norm(exact)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,half_ulp", [("f16", 2.0 ** -11), ("bf16", 2.0 ** -8)])
@pytest.mark.parametrize("batch,height,width,blocks", [(1, 56, 56, 1), (3, 72, 40, 2)])
def test_scores(batch, height, width, blocks, dtype, half_ulp):
    r = np.random.default_rng(batch)
    p = net.parameters(r, blocks=blocks, layer_scales=True)
    image = r.integers(0, 256, (batch, 3, height, width)).astype(np.uint8)
    eng = hip.Engine()
    model = s8_net.ImageAttentionS8Net(eng, p, batch, height, width, dtype)
    got = model.run(image)
    assert np.array_equal(model.run(image), got), "the same image gives other scores"
    assert not np.array_equal(model.run(255 - image), got)
    # the same pass recorded once and enqueued with one call
    L, rec = hip.lib(), hip.C.c_void_p()
    hip.check(L.cldnn_hip_engine_record_begin(eng.h))
    model.enqueue()
    hip.check(L.cldnn_hip_engine_record_end(eng.h, hip.C.byref(rec)))
    for _ in range(3):
        model._plain.write_raw(image)
        hip.check(L.cldnn_hip_recording_enqueue(rec))
        assert np.array_equal(model._scores.read(got.shape, "f32"), got)
        assert np.array_equal(model.run(image), got)
    hip.check(L.cldnn_hip_recording_release(rec))
    model.close()
    eng.close()
    # roundings to the type on the way of a value: qkv, the turned ones, probabilities, attention, branch, wide, branch; keys and values,
    # probabilities, the pooled query, the scores' weights
    roundings = 2 * (7 * blocks + 4) * half_ulp
    exact, crests = reference(p, image, height // 8, width // 8, False)
    assert np.linalg.norm(got - exact) <= (2 * noise(crests) + roundings) * np.linalg.norm(exact)
    # with the same quantisation: what is left is values that the roundings to the type take over a border of two steps
    rounded, _ = reference(p, image, height // 8, width // 8, True)
    assert np.linalg.norm(got - rounded) <= (2 * noise(crests) + roundings) * np.linalg.norm(rounded)


@pytest.mark.gpu
def test_the_float_network_is_as_it_was():
    r = np.random.default_rng(5)
    p = net.parameters(r)
    image = r.integers(0, 256, (1, 3, 48, 40)).astype(np.uint8)
    eng = hip.Engine()
    model = net.ImageAttentionNet(eng, p, 1, 48, 40)
    got, want = model.run(image), float_net.reference(p, image, 6, 5)
    model.close()
    eng.close()
    assert np.linalg.norm(got - want) <= 2 * 26 * 2.0 ** -11 * np.linalg.norm(want)
