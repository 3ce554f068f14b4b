"""The part of the vocabulary that score_tokens reads: sizes that it refuses."""

import pytest
import torch
from torch import nn

from neuropress_b200.nn import score_tokens


@pytest.mark.parametrize("size,match", [(0, "positive"), (-1, "positive"), (-20, "positive"), (21, "has 20 logits")])
def test_refused(size, match):
    """-1 would drop the last token, 21 would score targets that have no logit as if they were to be ignored."""
    with pytest.raises(RuntimeError, match=match):
        score_tokens(nn.Linear(8, 20), torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), vocab_size=size)


@pytest.mark.parametrize("size", [1, 20])
def test_taken_up_to_the_kernel(size):
    with pytest.raises(RuntimeError, match="CUDA"):
        score_tokens(nn.Linear(8, 20), torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), vocab_size=size)
