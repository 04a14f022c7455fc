"""Numbers that policy_loss's kernels would not hold in fp32 are refused before any launch."""

import pytest
import torch


@pytest.mark.parametrize("name,bad", [("denominator", 1e39), ("denominator", 1e-39), ("denominator", 5e-324),
                                      ("denominator", 0.0), ("denominator", -1.0), ("denominator", float("inf")),
                                      ("kl_weight", 1e39), ("kl_weight", -1e39), ("target_weight", 1e300),
                                      ("target_weight", float("nan")), ("target_weight", 10 ** 39)])
def test_numbers_out_of_range(name, bad):
    from kingdom_ai import policy_loss
    x = torch.zeros(2, 3)
    with pytest.raises(ValueError, match=name):
        policy_loss(x, target=x, **{name: bad})


@pytest.mark.parametrize("name,good", [("denominator", 3e38), ("denominator", 2.0 ** -126), ("kl_weight", -3e38),
                                       ("target_weight", 0), ("clip", 1e39), ("denominator", 7)])
def test_numbers_in_range(name, good):
    from kingdom_ai import policy_loss
    x = torch.zeros(2, 3)
    with pytest.raises(ValueError, match="requires CUDA"):  # the next check
        policy_loss(x, target=x, **{name: good})
