"""The serving operators at the ends of what their documentation allows, and on tensors that hold what it does not allow, on the GPU."""
import math

import pytest
import torch

from tests import serving_ref as R
from tests.test_gpu_serving import SCALE, fm, pool  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------------------------------------

def evict_and_check(fm, lengths, hkv, keep, recent, fill_weights, seed, width=None):
    """Lists, and what was copied, against the plain restatement.  `width`: pages of a row of the table, where it is wider than the lengths need."""
    cache, table, ls, g = pool(fm, lengths, hkv, seed=seed, spare=len(lengths) * (-(-keep // 128)))
    own = len(lengths) * table.shape[1]
    to = torch.arange(own, cache.shape[0], dtype=torch.int32, device="cuda").view(len(lengths), -1)
    w = fill_weights(torch.rand(cache.shape[0], hkv, 128, generator=g, device="cuda") + 0.01, g)
    if width is not None:
        table = torch.cat([table, torch.full((len(lengths), width - table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    old, old_w = cache.clone(), w.clone()
    new_lengths, kept = fm.flash_msa_cache_evict(cache, w, table, ls, to, keep, recent)
    want = R.evict(old_w, table, lengths, keep, recent)
    for i, length in enumerate(lengths):
        n = min(length, keep)
        assert int(new_lengths[i]) == n
        for h in range(hkv):
            assert kept[i, h].tolist() == want[i, h] + [-1] * (keep - n)
            at, j = torch.tensor(want[i, h], device="cuda"), torch.arange(n, device="cuda")
            for which in "kv":
                assert torch.equal(R.rows_of(cache, to[i], n, h, which), R.rows_of(old, table[i], length, h, which)[at])
            assert torch.equal(w[to[i].long()[j // 128], h, j % 128].view(torch.int32), old_w[table[i].long()[at // 128], h, at % 128].view(torch.int32))
    assert torch.equal(cache[:own], old[:own])


def some_nan(share):
    def fill(w, g):
        w[torch.rand(w.shape, generator=g, device="cuda") < share] = math.nan
        return w
    return fill


# (tables of up to 2K, 8K, 32K and more tokens go to different kernels)
@pytest.mark.parametrize("share", [0.5, 0.9, 1.0])
@pytest.mark.parametrize("lengths,hkv,keep,recent", [([1100, 700], 2, 512, 64), ([4100, 900], 2, 512, 64), ([20000], 2, 4000, 256), ([40000], 1, 4000, 256)])
def test_evict_with_more_nan_than_room(fm, lengths, hkv, keep, recent, share):
    """Weights that are NaN for more tokens than stay (a query row that is not finite leaves them), and finite positive ones: the first of the
    NaN ones stay, and nothing is written behind a list."""
    evict_and_check(fm, lengths, hkv, keep, recent, some_nan(share), seed=41)
