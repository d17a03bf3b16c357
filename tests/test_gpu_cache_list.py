"""A list of caches has each of them once: the moves of tree_accept go through all of its layers at the same time."""
import pytest
import torch

from aici_amd import kernels as K
from aici_amd._lib import HipAttnError

pytestmark = pytest.mark.gpu


def test_a_cache_twice_is_refused(device):
    kcs = [torch.zeros((4, 2, 8, 16, 8), dtype=torch.float16, device=device) for _ in range(3)]
    vcs = [torch.zeros((4, 2, 64, 16), dtype=torch.float16, device=device) for _ in range(3)]
    with pytest.raises(HipAttnError, match="the same cache twice"):
        K.CacheList([kcs[0], kcs[1], kcs[0]], vcs)
    with pytest.raises(HipAttnError, match="the same cache twice"):
        K.CacheList(kcs, [vcs[0], vcs[1], vcs[1]])
    with pytest.raises(HipAttnError, match="the same cache twice"):
        K.CacheList(kcs[:1], [kcs[0].view(4, 2, 64, 16)])
    pool = torch.zeros((4, 3, 2, 8, 16, 8), dtype=torch.float16, device=device)  # layers beside each other in every block are several caches
    assert K.CacheList([pool[:, i] for i in range(3)], vcs).key_ptrs.numel() == 3
    assert K.CacheList([t[:0] for t in kcs], [t[:0] for t in vcs]).key_ptrs.numel() == 3
