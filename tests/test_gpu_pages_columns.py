"""New tables beside the old ones in one tensor: memory apart from theirs, row by row."""

import pytest
import torch

from tests.cache8_model import table_for
from tests.test_gpu_pages import assert_same, compacted, device, forked, i32, pool


def test_columns_of_one_tensor_are_told_apart():
    from quantexperiments_amd.kernels.pages import _new
    both = torch.zeros(3, 10, dtype=torch.int32)
    for old, new in ((both[:, :4], both[:, 4:8]), (both[:, 6:], both[:, :4]), (both[:2, :4], both[:, 6:])):
        _new("here", "out_table", new, new.shape, old, torch.zeros(2, dtype=torch.int32))
    for old, new in ((both[:, :4], both[:, 3:7]), (both[:, 2:6], both[:, 2:6]), (both[:, 4:8], both[:, 1:5]), (both[:, :4], both.view(-1)[:24].view(3, 8)[:, 4:])):
        with pytest.raises(ValueError, match="overlaps"):
            _new("here", "out_table", new, new.shape, old)
    flat = torch.zeros(30, dtype=torch.int32)
    with pytest.raises(ValueError, match="overlaps"):
        _new("here", "out_lens", flat[8:11], (3,), flat.view(3, 10)[:, :4])


@pytest.mark.gpu
def test_tables_side_by_side():
    from quantexperiments_amd.kernels import compact_pages, fork_pages
    g = torch.Generator().manual_seed(1)
    lens, parent = [33, 5, 20], [0, 0, 1, 2, 2]
    table, pages, spare = table_for(lens, 16, g, spare=9)
    w = table.shape[1]
    cache, fresh = pool(2, pages, 16, 2, 8, "bf16", g), [-1, *spare[:2].tolist(), -1, int(spare[4])]
    dev, both = device(cache), torch.full((5, 3 * w + 1), 77, dtype=torch.int32, device="cuda")
    both[:3, :w] = table.cuda()
    t, n = fork_pages(*dev, both[:3, :w], i32(lens), i32(parent), i32(fresh), out_table=both[:, w:2 * w])
    want, wt, wn = forked(cache, table, lens, parent, fresh, 16)
    assert torch.equal(t.cpu(), wt) and torch.equal(n.cpu(), wn)
    assert_same(dev, want)
    again, used = compact_pages(*dev, t, n, out_table=both[:, 2 * w:3 * w])
    want, wt2, k = compacted(want, wt, wn.tolist(), 16)
    assert torch.equal(again.cpu(), wt2) and used.tolist() == [k]
    assert_same(dev, want)
    assert torch.equal(both[:3, :w].cpu(), table) and torch.equal(both[:, w:2 * w].cpu(), wt) and bool((both[:, 3 * w:] == 77).all()) and bool((both[3:, :w] == 77).all())
