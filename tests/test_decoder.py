"""The INT8 cross-attention layer over a ResNet's features (spinnv2_b200.decoder): the operators together."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def float_layer(weights, heads, kv_heads, x, residual, features, valid):
    """The layer in 64 bits, without any rounding to 8 bits."""
    w = {k: v.double() for k, v in weights.items()}
    s = x.double() + (0 if residual is None else residual.double())
    h = s * w["norm"] / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    b, lq = x.shape[:2]
    d = w["q"].shape[0] // heads
    q = (h @ w["q"].t()).view(b, lq, heads, d)
    k, v = (features.double() @ w["kv"].t()).view(b, -1, 2, kv_heads, d).unbind(2)
    k, v = (t.repeat_interleave(heads // kv_heads, dim=2) for t in (k, v))
    scores = torch.einsum("bqhd,bkhd->bhqk", q, k) * d**-0.5
    if valid is not None:
        scores = scores.masked_fill(~valid[:, None, None, :], -np.inf)
    o = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(scores, -1), v)
    return o.flatten(2) @ w["out"].t(), s


@pytest.mark.parametrize("tokens", [1, 9, 60])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_against_floats(gpu, tokens, dtype):
    """Codes of 8 bits round each of an operand's values by up to half a step of max / 127, which is about 1 %
    of the values' spread here (the largest of a row is four to five spreads), in both operands of three
    products in a row; 5 % of the answer's norm holds them all."""
    from spinnv2_b200.decoder import CrossAttentionLayer

    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)

    def matrix(n, k):
        return (torch.randn(n, k, generator=g, device="cuda") * k**-0.5).to(dtype)

    heads, kv_heads = 8, 2
    weights = {"norm": (1 + 0.1 * torch.randn(512, generator=g, device="cuda")).to(dtype), "q": matrix(heads * 64, 512),
               "kv": matrix(2 * kv_heads * 64, 300), "out": matrix(512, heads * 64)}
    layer = CrossAttentionLayer(weights, heads, kv_heads)
    features = torch.randn(3, 49, 300, generator=g, device="cuda")
    x = torch.randn(3, tokens, 512, generator=g, device="cuda").to(dtype)
    residual = torch.randn(3, tokens, 512, generator=g, device="cuda").to(dtype)
    valid = torch.ones(3, 49, dtype=torch.bool, device="cuda")
    valid[1, 30:] = False
    for r, mask in ((None, None), (residual, valid)):
        y, stream = layer.step(x, r, layer.states(features), key_mask=mask)
        want, s = float_layer(weights, heads, kv_heads, x, r, features, mask)
        assert float((y.double() - want).norm() / want.norm()) < 0.05
        assert torch.equal(stream, s.to(dtype)) if dtype is torch.float32 else float((stream.double() - s).abs().max()) < 0.04
    lengths = torch.tensor([49, 30, 49], dtype=torch.int32, device="cuda")
    by_length, _ = layer.step(x, residual, layer.states(features), lengths=lengths)
    assert torch.equal(by_length, y)


def test_tokens_do_not_depend_on_their_batch(gpu):
    """Every operator works row by row, so a prompt's token alone gives what it gives in the prompt, up to the
    order in which the attention kernels for few and for many rows add."""
    from spinnv2_b200.decoder import CrossAttentionLayer

    layer = CrossAttentionLayer.random(256, 128, 4, 2, 64, seed=3)
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    states = layer.states(torch.randn(2, 70, 128, generator=g, device="cuda"))
    x = torch.randn(2, 40, 256, generator=g, device="cuda").bfloat16()
    whole, stream = layer.step(x, None, states)
    assert stream is x
    one, _ = layer.step(x[:, 7:8], None, states)
    # One code of the attention's answer may differ where it lies at a rounding edge: a step of 8 bits.
    assert float((one - whole[:, 7:8]).float().norm() / whole[:, 7:8].float().norm()) < 0.02


def test_features_of_the_graph_runtime(gpu):
    """The encoder's features reach the layer in place, and the package's own output stays what it was."""
    from conftest import compile_pair, seeded_input
    from spinnv2_b200 import transformer as T
    from spinnv2_b200.decoder import CrossAttentionLayer, ImageEncoder
    from spinnv2_b200.runtime import Runtime

    images = seeded_input((2, 3, 224, 224))
    encoder = ImageEncoder("resnet50", 2)
    features = encoder(images)
    assert features.shape == (2, 49, 2048) and torch.isfinite(features).all() and float(features.abs().max()) > 0
    probabilities = encoder.rt.get_output(0)
    with Runtime(compile_pair("resnet50", 2, targets=("cuda_b200",))["cuda_b200"], device=0) as rt:
        np.testing.assert_allclose(probabilities, rt.run(images)[0], atol=1e-5)
    layer = CrossAttentionLayer.random(512, 2048, 8, 8, 64)
    x = torch.randn(2, 5, 512, device="cuda").bfloat16()
    y, _ = layer.step(x, None, layer.states(features))
    T.check()
    assert y.shape == x.shape and torch.isfinite(y).all()
    encoder.close()
