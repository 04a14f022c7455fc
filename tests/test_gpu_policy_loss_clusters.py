"""policy_loss on rows that a cluster of CTAs shares, with more rows than the
clusters that the device holds at once: each CTA then takes its part of the
next row while it finishes this one. Compared with the formula in 64 bits, at
the tolerances of test_gpu_policy_loss.py."""

import pytest
import torch

from test_gpu_policy_loss import compare, make, run

pytestmark = pytest.mark.gpu


# Four and eight CTAs a row and an odd stride, so that rows start at every
# shift to a 16-byte boundary. At these lengths the number of 16-byte groups of
# a row passes a multiple of the CTAs with its shift, and with it where every
# part begins: the last CTA's part of the next row is up to seven groups longer.
ODD = [(300, 131071, torch.bfloat16), (1000, 83197, torch.bfloat16), (600, 99999, torch.bfloat16),
       (480, 229375, torch.bfloat16), (300, 65535, torch.float32), (600, 50255, torch.float32),
       (400, 99999, torch.float32)]


@pytest.mark.parametrize("n,a,dtype", ODD)
def test_parts_that_grow_from_row_to_row(n, a, dtype):
    compare(*make(n, a, dtype))


@pytest.mark.parametrize("n,a,dtype", [(300, 131071, torch.bfloat16), (300, 65535, torch.float32)])
def test_parts_that_grow_with_mask_and_target(n, a, dtype):
    compare(*make(n, a, dtype, mask=True, clipped=True, target=dtype))


# Two, four and eight CTAs a row with the fewest and with many rows each, the same parts in every row: the
# exchange of what the CTAs found, from the first row on.
@pytest.mark.parametrize("n,a,dtype", [(1, 131072, torch.bfloat16), (40, 65536, torch.bfloat16),
                                       (900, 65536, torch.bfloat16), (500, 131072, torch.bfloat16),
                                       (300, 98304, torch.float32), (3, 20000, torch.float32)])
def test_parts_meet_from_the_first_row_on(n, a, dtype):
    logits, args = make(n, a, dtype)
    first = compare(logits, args)
    for _ in range(5):
        again = run(logits, args)
        assert torch.equal(again[0].loss.detach(), first[0].loss) and torch.equal(again[1], first[1])
