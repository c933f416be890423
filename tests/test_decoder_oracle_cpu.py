"""The order of equal logits in the oracle of token_logprobs."""

import math

import pytest
import torch

from . import decoder_reference as ref


@pytest.mark.parametrize("seed", range(5))
def test_equal_logits_go_by_the_lowest_token(seed):
    x = torch.randn(4, 50, generator=torch.Generator().manual_seed(seed))
    x[0, 3] = x[0, 7] = x[0].max() + 1  # at the front
    ranked = x[1].sort(descending=True).indices
    x[1, ranked[6]] = x[1, ranked[5]]  # either side of the cut
    x[2, 10:20] = x[2].max() + 1  # more than there are places
    x[3] = -math.inf
    x[3, 40], x[3, 41] = 0.0, math.nan
    _, _, _, ids = ref.logprobs(x, torch.zeros(4, dtype=torch.int64), 6)
    assert ids[0, :2].tolist() == [3, 7]
    assert ids[1].tolist() == ranked[:5].tolist() + [int(min(ranked[5], ranked[6]))]
    assert ids[2].tolist() == [10, 11, 12, 13, 14, 15]
    assert ids[3].tolist() == [40, 0, 1, 2, 3, 4]
    every = ref.logprobs(x, torch.zeros(4, dtype=torch.int64), 50)[3]
    assert every[3].tolist() == [40] + list(range(40)) + list(range(42, 50)) + [41]  # NaN last
    assert all(sorted(row.tolist()) == list(range(50)) for row in every)
