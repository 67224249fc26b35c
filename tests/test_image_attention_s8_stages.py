"""Each call of the classifier with int8 products against its formula in 64 bits, and mistakes that this has to find."""
import numpy as np
import pytest

import image_attention_s8_stages as stages
from cldnn_amd import hip, image_attention_net as net, image_attention_s8_net as s8_net

SIZES = [(1, 56, 56, 1), (3, 72, 40, 2)]


def a_case(batch, height, width, blocks):
    r = np.random.default_rng(batch)
    p = net.parameters(r, blocks=blocks, layer_scales=True)
    return p, r.integers(0, 256, (batch, 3, height, width)).astype(np.uint8), height // p["patch"], width // p["patch"]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_the_formulas_pass(size, dtype):
    p, image, y, x = a_case(*size)
    stages.verify(p, image, y, x, dtype, *stages.walk(p, image, y, x, dtype))


MISTAKES = {"no rotary": "rotary", "rotary axes swapped": "rotary", "uniform attention": "attention", "relu for gelu": "gelu", "no gelu": "gelu", "norm2 has norm1's parameters": "norm 1",
            "no scale1": "the sum into the map", "no scale2": "the sum into the map", "scales swapped": "the sum into the map", "rows of 4 bits": "first norm", "truncation": "first norm",
            "no row scales": "qkv"}


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("mistake", MISTAKES)
def test_mistakes_are_found(mistake, size, dtype):
    p, image, y, x = a_case(*size)
    left = stages.walk(p, image, y, x, dtype, mistake)
    with pytest.raises(AssertionError, match=MISTAKES[mistake]):
        stages.verify(p, image, y, x, dtype, *left)


def test_weights_of_another_scale_are_found():
    p, image, y, x = a_case(*SIZES[0])
    weights, left = stages.walk(p, image, y, x, "f16")
    weights[0]["project"] = weights[0]["project"][0], weights[0]["project"][1] * 1.01
    with pytest.raises(AssertionError, match="weights of project"):
        stages.verify(p, image, y, x, "f16", weights, left)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_every_call_of_a_pass(size, dtype):
    p, image, y, x = a_case(*size)
    eng = hip.Engine()
    model = s8_net.ImageAttentionS8Net(eng, p, *image.shape[:1], *image.shape[2:], dtype)
    weights, left = stages.record(model, image)
    stages.verify(p, image, y, x, dtype, weights, left)
    # a pass that nobody looks into gives the same scores
    assert np.array_equal(model.run(image), left[-1]["scores"].numpy())
    model.close()
    eng.close()
