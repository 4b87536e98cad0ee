"""fp16 paged attention whose probabilities span more than fp16 holds."""

import math

import pytest
import torch

from polylora_b200.paged import paged_attention

pytestmark = pytest.mark.gpu

FH = torch.float16


# A first token of value 0 and score 0, and a tail of value 1 whose probabilities
# fp16 cannot hold next to 1.
@pytest.mark.parametrize("n,D,page,group,power", [
    (131072, 128, 64, 4, -25), (131072, 128, 64, 4, -30), (131072, 64, 12, 1, -26), (8000, 128, 16, 1, -24),
    (8000, 64, 5, 8, -21), (100, 128, 16, 4, -20), (60000, 256, 32, 16, -26), (60000, 128, 16, 20, -27),
])
def test_fp16_probabilities_far_below_the_largest(cuda_status_clean, n, D, page, group, power):
    dev = torch.device("cuda")
    pages = -(-n // page)
    table = torch.ones(1, pages, dtype=torch.int32, device=dev)  # one page for the tail, one for the front
    table[0, 0] = 0
    kc, vc = torch.zeros(2, 1, page, D, dtype=FH, device=dev), torch.ones(2, 1, page, D, dtype=FH, device=dev)
    kc[..., 0] = power * math.log(2)
    kc[0, 0, 0, 0], vc[0, 0, 0] = 0, 0
    q = torch.zeros(1, group, D, dtype=FH, device=dev)
    q[..., 0] = 1
    got = paged_attention(q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device=dev), scale=1.0).double()
    p = math.exp(float(kc[1, 0, 0, 0]))
    want = (n - 1) * p / (1 + (n - 1) * p)
    # the score, 2^-24 of up to 30 thrice, and its exponential; the pair, 2^-22 and half
    # a step of 2^-40; sums of up to n / 16 tiles, split over 8 warps at least; the result
    off = (90 * 2.0**-24 + 2.0**-21 + 2.0**-22 + 2.0**-40 / p + (n / 128 + 64) * 2.0**-22 + 2.0**-11) * want + 2.0**-25
    assert float((got - want).abs().max()) <= off, (float(got.min()), float(got.max()), want)
