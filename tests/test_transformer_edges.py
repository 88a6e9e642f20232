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
