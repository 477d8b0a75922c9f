"""Attention of many rows over pages that hold parts of what a wave looks up at once: a table entry outside the cache gives NaN whichever key it is of."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [1, 3, 12])
@pytest.mark.parametrize("key", [0, 3, 7, 21, 63, 100, 130])
def test_a_wrong_page_of_any_key_gives_nan(page, key):
    from quantexperiments_amd.kernels import tree_attention
    g = torch.Generator().manual_seed(page)
    cached, new, pages = 70, 64, -(-134 // page)
    table = torch.randperm(pages, generator=g).int()[None]
    kc, vc = (torch.randn(pages, page, 1, 64, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(new, 2, 64, generator=g).half().cuda()
    lens = torch.tensor([cached], dtype=torch.int32).cuda()
    assert bool(tree_attention(q, kc, vc, table.cuda(), lens).isfinite().all())
    table[0, key // page] = pages
    assert bool(tree_attention(q, kc, vc, table.cuda(), lens)[max(0, key - cached):].isnan().all())
