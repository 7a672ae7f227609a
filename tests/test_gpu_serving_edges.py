"""The serving operators at the edges of what they accept, on the GPU: each test holds a call that once gave
something else than its definition."""
import math

import pytest
import torch

import natten_b200 as nb
from test_gpu_decode import TYPES, _state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("heads", [4, 24])
def test_an_infinite_query_that_attends_nothing(dtype, cache_dtype, heads):
    """Zeros and -inf like any other row without tokens (a drafted place that a short sequence does not
    have, a table without pages); where there are tokens, the row alone is not finite."""
    q, cache, table, n = _state(dtype, cache_dtype, [1, 40, 40], 2, heads, 2, 64, 16)
    table[1] = -1
    for kernel_size in (None, 30):
        good, good_lse = nb.na1d_decode(q, cache, table, n, kernel_size, return_lse=True)
        bad = q.clone()
        bad[0, 0, :, 3] = math.inf
        bad[1, :, :, 5] = -math.inf
        bad[2, 0, 0, 7] = math.inf
        out, lse = nb.na1d_decode(bad, cache, table, n, kernel_size, return_lse=True)
        for rows in ((0, 0), (1, 0), (1, 1)):
            assert not out[rows].any() and torch.isneginf(lse[rows]).all()
        assert torch.isnan(out[2, 0, 0]).all()
        out[2, 0, 0], lse[2, 0, 0] = good[2, 0, 0], good_lse[2, 0, 0]
        assert torch.equal(out, good) and torch.equal(lse, good_lse)
