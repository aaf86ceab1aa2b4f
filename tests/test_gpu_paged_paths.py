"""Paths of the paged operators that depend on the size of a batch, and calls at
the edge of what they take, against plain 64-bit forms; tolerances as derived in
test_gpu_paged.py."""
import numpy as np
import pytest

from pagedref import Batch, append, attention
from test_gpu_paged import (U, check_attention, dtype_of, host, make_cache, ops,  # noqa: F401
                            torch)

pytestmark = pytest.mark.gpu


def device_of(torch, device):  # noqa: F811
    return torch.device("cuda", device)


def test_head_counts_refused(device, torch, ops):  # noqa: F811
    dev = device_of(torch, device)
    b = Batch([(0, [(3, 1)])], 16, np.random.default_rng(1))
    cache = torch.zeros((b.n_pages, 16, 2, 2, 64), device=dev).half()
    # As wide as 3 heads: -1 query heads and 2 + 2 of the cache.
    for heads in (-1, 0):
        with pytest.raises(ops.OmgError, match=f"paged_append: heads {heads}"):
            ops.paged_append(torch.zeros((1, (heads + 4) * 64), device=dev), cache,
                             b.device(ops, torch, dev), heads=heads)
