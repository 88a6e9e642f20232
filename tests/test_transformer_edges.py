"""Edges of the decoder-layer operators (spinnv2_b200.transformer): values that are not finite or lie at the
ends of their types, empty dimensions, sizes past 32 bits, other streams."""

from __future__ import annotations

import math

import pytest
import torch

from test_transformer import F32, TYPES, U, attention64, check_codes, codes_of, gen, inputs

gpu_test = pytest.mark.gpu


# ------------------------------------------------------------------ attention
@gpu_test
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,hq,hk,d", [(40, 4, 4, 64), (40, 8, 2, 128), (50, 6, 2, 64), (130, 3, 1, 104), (1, 4, 2, 64),
                                        (5, 10, 2, 128), (33, 2, 2, 200)])
def test_query_that_is_not_finite_stays_alone(gpu, lq, hq, hk, d, dtype):
    """A row of queries that holds an infinity or a NaN changes no other row, bit by bit, also where an entry's
    keys are fewer than the parts that they are divided into; and a row without keys is 0 whatever it holds."""
    from spinnv2_b200 import transformer as T

    for keys in (520, 2100):
        lengths = torch.tensor([0, 1, 100, 300, keys, 0], dtype=torch.int32, device="cuda")
        q, k, v = inputs(len(lengths), lq, keys, hq, hk, d, dtype, 21)
        mask = torch.arange(keys, device="cuda")[None, :] < lengths[:, None]
        at = lq // 2
        for valid in ({"lengths": lengths}, {"key_mask": mask}):
            want = T.cross_attention(q, k, v, **valid)
            assert not want[lengths == 0].any()
            for bad in (math.nan, math.inf, -math.inf):
                bent = q.clone()
                bent[:, at, hq - 1] = bad
                for _ in range(3):
                    got = T.cross_attention(bent, k, v, **valid)
                    assert not got[lengths == 0].any()
                    got[:, at, hq - 1] = want[:, at, hq - 1]
                    assert torch.equal(got, want)


# ------------------------------------------------------------------ streams
@gpu_test
def test_encoder_calls_behind_queued_work(gpu):
    """An answer of the encoder holds its own images' features, also where torch's stream is still busy with
    earlier work when the next call writes the runtime's buffer, and from one current stream to another."""
    from conftest import seeded_input
    from spinnv2_b200.decoder import ImageEncoder

    first, second = (seeded_input((1, 3, 224, 224), seed=i) for i in (1, 2))
    matrix = torch.randn(8192, 8192, generator=gen(1), device="cuda")
    out = torch.empty_like(matrix)

    def busy():
        for _ in range(10):  # some 0.2 s
            torch.mm(matrix, matrix, out=out)

    busy()
    encoder = ImageEncoder("resnet50", 1)
    torch.cuda.synchronize()
    want = []
    for images in (first, second):
        want.append(encoder(images))
        torch.cuda.synchronize()
    assert not torch.equal(*want)
    busy()
    got = [encoder(first), encoder(second)]
    assert got[0].data_ptr() != encoder.features.data_ptr() and got[0].is_contiguous()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    busy()
    a = encoder(first)
    with torch.cuda.stream(torch.cuda.Stream()):
        b = encoder(second)
    torch.cuda.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    encoder.close()
