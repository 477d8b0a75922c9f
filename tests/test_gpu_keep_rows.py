"""keep_drafted with a path that falls back early: its later entries' targets lie behind the table row, where nothing may be looked up."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_table_entry_behind_its_row_is_read():
    from quantexperiments_amd.kernels import keep_drafted
    g = torch.Generator().manual_seed(13)
    table = torch.randperm(3, generator=g).int()[None].cuda()
    kc, vc = (torch.randn(3, 16, 1, 32, generator=g).half().cuda() for _ in range(2))
    was = kc.clone(), vc.clone()
    path = torch.tensor([[0, 1, 1, 1, *range(2, 60)]], dtype=torch.int32).cuda()              # 62 entries behind slot 20 of 48
    keep_drafted(kc, vc, table, torch.tensor([20], dtype=torch.int32).cuda(), path, torch.tensor([62], dtype=torch.int32).cuda())
    assert torch.equal(kc, was[0]) and torch.equal(vc, was[1])          # (rows 0 and 1 stay in place)
