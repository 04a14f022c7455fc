"""linear on tiles that CTAs share along k: every width of a tile that holds
all rows, from one stage of k to more than a CTA's stages, and the same bits
from every call; residuals whose rows are no whole 16 bytes, with aligned or no
steps between them. Compared with the formula in 64 bits, at the tolerances of
test_gpu_linear.py."""

import pytest
import torch

from test_gpu_linear import compare, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [9, 16, 17, 32, 33, 48, 49, 64, 65, 80, 81, 96, 97, 112, 113, 128])
def test_every_width_of_a_thin_tile(m, dtype):
    # Up to 48 rows are thin whatever the weight; up to 128 against wide ones.
    for k, n in ((8, 136), (72, 1024), (1100, 520)) if m <= 48 else ((1024, 8200),):
        compare(make(m, k, n, dtype), "relu")


@pytest.mark.parametrize("m,k,n", [(64, 64, 64), (130, 4096, 70), (200, 520, 300), (12, 8192, 256)])
def test_shared_tiles_repeat_their_bits(m, k, n):
    args = make(m, k, n, torch.bfloat16)
    compare(args, "gelu")
    first = run(*args, "gelu")
    for _ in range(10):
        again = run(*args, "gelu")
        assert all(torch.equal(first[key], again[key]) for key in first)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(2560, 192, 2052), (300, 96, 100), (40, 64, 1001)])
def test_residual_rows_that_end_inside_16_bytes(m, k, n, dtype):
    """A padded matrix, and one row for all: nothing behind a row's end is taken, and its gradient is the row's."""
    x, w, b, r, dy = make(m, k, n, dtype, grad=False)
    wide = torch.full((m, (n + 8) // 8 * 8), float("nan"), dtype=dtype, device="cuda")
    wide[:, :n] = r
    compare((x, w, b, wide[:, :n].requires_grad_(), dy), "gelu")
    row = r[0].clone()
    got, want = (run(x, w, b, t.requires_grad_(), dy, "tanh") for t in (row.expand(m, n), row.expand(m, n).contiguous()))
    assert all(torch.equal(got[key], want[key]) for key in want)
