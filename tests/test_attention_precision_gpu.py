"""Attention in fp16 where roundings to 16 bits show: results at the type's largest number."""
import math

import pytest
import torch

from encoder_util import starts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("queries,keys,window", [(5, 1000, (-1, -1)), (300, 640, (-1, -1)), (1000, 1000, (255, 0)), (300, 20000, (-1, -1))])
@pytest.mark.parametrize("sign", [1, -1])
def test_results_at_the_largest_number_of_the_type(native_lib, dim, queries, keys, window, sign):
    # All values are the largest, so every result is; most weights (2^-3.99648 of the largest) lie just above the middle of two 16-bit
    # numbers, so that they are all rounded up and the rounded ones add up to a result half a step above.
    q = torch.zeros(queries, 4, dim, dtype=torch.float16, device="cuda")
    q[:, :, :2] = 1.0
    k = torch.zeros(keys, 2, dim, dtype=torch.float16, device="cuda")
    k[:, :, 0], k[:, :, 1] = -4.0, 0.00352
    k[::64] = 0
    v = torch.full_like(k, sign * 65504.0)
    got = native_lib.attention(q, k, v, starts([queries])[1], starts([keys])[1], queries, keys, window=window, scale=math.log(2))
    assert (got == sign * 65504.0).all()
