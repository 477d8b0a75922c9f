"""Sequences longer than their table rows, by one token and by as many as 32 bits hold: they get NaN, and the other sequences of the call what they would get without them."""

import pytest
import torch

from tests.test_gpu_attention8 import Setup, attend

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


def check_of(s, part, got, lse):
    """The formula for sequences `part`, neighbours, alone."""
    t = object.__new__(Setup)
    t.__dict__.update(s.__dict__)
    t.lens, t.news, t.sees, t.places = ([x[b] for b in part] for x in (s.lens, s.news, s.sees, s.places))
    t.starts = s.starts[part[0]:part[-1] + 2]
    t.check(got, lse)


@pytest.mark.parametrize("far", [MOST, MOST - 100, MOST - 4096 - 150, 0])
@pytest.mark.parametrize("lens,news,hq,hk,d,tree", [
    ([4000, 3000, 2000, 1000], [200] * 4, 28, 4, 128, False),         # blocks of rows share workgroups by their work
    ([4000, 3000, 2000, 1000], [200] * 4, 10, 2, 256, False),
    ([4000, 3000, 2000, 1000], [48] * 4, 28, 4, 128, True),
    ([90] * 40, [20] * 40, 28, 4, 128, False),                        # as many as there are
    ([500, 300, 20], [1, 1, 1], 7, 1, 128, False),                    # few rows
    ([500, 300, 20], [40, 1, 9], 7, 1, 64, False),
])
def test_a_length_that_32_bits_barely_hold(lens, news, hq, hk, d, tree, far):
    s = Setup(lens, news, hq, hk, d, 16, tree=tree, seed=d + len(lens))
    at = 1
    told = list(lens)
    told[at] = far or s.table.shape[1] * 16 - news[at] + 1           # (0: one token too many)
    got, lse = attend(s, lens=torch.tensor(told, dtype=torch.int32).cuda(), out=torch.full((s.n, hq, d), 7.0).to(s.dt).cuda())
    rows = slice(s.starts[at], s.starts[at + 1])
    assert bool(got[rows].isnan().all()) and bool(lse[rows].isnan().all())
    check_of(s, range(at), got, lse)
    check_of(s, range(at + 1, len(lens)), got, lse)


@pytest.mark.parametrize("new", [1, 40])
def test_over_a_16_bit_cache(new):
    from quantexperiments_amd.kernels import tree_attention
    g = torch.Generator().manual_seed(new)
    kc, vc = (torch.randn(3 * 30, 16, 2, 64, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(3 * new, 8, 64, generator=g).half().cuda()
    table, lse = torch.randperm(90, generator=g).int().view(3, 30).cuda(), torch.empty(3 * new, 8, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()
    want = tree_attention(q, kc, vc, table, i32(400, 300, 200))
    assert bool(want.isfinite().all())
    for far in (MOST, MOST - 10, 480 - new + 1):
        got = tree_attention(q, kc, vc, table, i32(400, far, 200), lse=lse)
        assert bool(got[new:2 * new].isnan().all()) and bool(lse[new:2 * new].isnan().all())
        assert torch.equal(got[:new], want[:new]) and torch.equal(got[2 * new:], want[2 * new:])
