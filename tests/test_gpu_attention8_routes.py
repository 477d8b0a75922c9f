"""Attention over an 8-bit cache at sizes that take each of its ways through the GPU: blocks of 16 and of 32 rows, and tiles of many, whole, cut, and with a last one that is cut less.  Against the
formula in 64 bits, with the tolerance of tests/test_gpu_attention8.py."""

import pytest
import torch

from tests.test_gpu_attention8 import Setup, attend

pytestmark = pytest.mark.gpu


def ragged(seqs, most_cached, most_new):
    g = torch.Generator().manual_seed(seqs + most_new)
    lens = torch.randint(0, most_cached + 1, (seqs,), generator=g).tolist()
    news = torch.randint(0, most_new + 1, (seqs,), generator=g).tolist()
    news[seqs // 2] = most_new
    return lens, news


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("d", [64, 80, 128, 256])
def test_many_short_sequences(d, tree, dtype):
    """Tiles of up to 128 rows, as many as there are sequences and key heads."""
    lens, news = ragged(40, 90, 20)
    s = Setup(lens, news, 8, 4, d, 16, dtype=dtype, tree=tree, seed=d, extra_rows=2)
    s.check(*attend(s))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_tiles_of_long_ones(d):
    """Tiles of 256 rows (128 of heads of 256): cut, the last one filled by half and cut less."""
    s = Setup([5000, 4100], [48, 40], 28, 4, d, 32, blocks=2, tree=True, seed=1)
    s.check(*attend(s))
    s = Setup([1600], [500], 8, 2, d, 16, seed=2)
    s.check(*attend(s))


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("lens,news,hq,hk,tree", [
    ([700, 13, 0, 300, 299], [9, 1, 8, 5, 9], 14, 2, True),          # rows in several blocks, most of the last one empty
    ([0], [260], 7, 1, False),                                       # a prompt
    ([900, 20], [64, 3], 10, 2, True),
    ([250] * 9, [4] * 9, 35, 5, False),
    ([2000] * 24, [6] * 24, 12, 2, False),                           # blocks of 32, uncut
])
def test_blocks_of_few_rows(d, lens, news, hq, hk, tree):
    s = Setup(lens, news, hq, hk, d, 16, tree=tree, seed=len(lens), extra_rows=1)
    s.check(*attend(s))


@pytest.mark.parametrize("seqs,new", [(3, 17), (40, 20)])
def test_a_wrong_page_and_masked_nan(seqs, new):
    s = Setup([70 + b % 9 for b in range(seqs)], [new] * seqs, 8, 4, 128, 16, tree=True, seed=seqs)
    for m in s.sees:
        m[:, 0] = False                                      # (the first new token is seen by none, and holds NaN)
    for b in range(seqs):
        pg, off = s.places[b]
        s.pool.codes[:, pg[s.lens[b]], off[s.lens[b]]] = 0x7F
    table = s.table.clone()
    table[seqs // 2, 2] = s.pool.codes.shape[1] + 5
    got, lse = attend(s, table=table.cuda())
    rows = slice(s.starts[seqs // 2], s.starts[seqs // 2 + 1])
    assert bool(got[rows].isnan().all()) and bool(lse[rows].isnan().all())
    clean = s.pool.codes.clone()
    clean[clean == 0x7F] = 0                                 # (the formula's zero weights need numbers)
    s.pool.codes = clean
    for part in (range(seqs // 2), range(seqs // 2 + 1, seqs)):
        t = object.__new__(Setup)
        t.__dict__.update(s.__dict__)
        t.lens, t.news, t.sees, t.places = ([x[b] for b in part] for x in (s.lens, s.news, s.sees, s.places))
        t.starts = s.starts[part[0]:part[-1] + 2]
        t.check(got, lse)


def test_the_same_under_a_table_of_any_width():
    """How rows are dealt out follows the table's width; results agree to the tolerance, whichever way was taken."""
    s = Setup([300, 40], [30, 7], 14, 2, 128, 16, tree=True, seed=5)
    for width in (0, 100, 4000):
        wide = torch.cat((s.table, torch.full((2, width), -1, dtype=torch.int32)), 1)
        s.check(*attend(s, table=wide.cuda()))


@pytest.mark.parametrize("d,hq,hk,new,tree", [(128, 14, 2, 48, True), (64, 8, 1, 150, False), (256, 10, 2, 40, True)])
def test_sequences_of_all_lengths_in_a_captured_call(d, hq, hk, new, tree):
    """Parts are dealt to sequences by their lengths, which change from replay to replay: long ones beside short and empty ones, all alike, one alone."""
    from quantexperiments_amd.kernels import tree_attention8
    top = 4200
    s = Setup([top] * 9, [new] * 9, hq, hk, d, 16, tree=tree, seed=d)
    dev, lse = s.device(), torch.empty(s.n, hq, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = tree_attention8(**dev, lse=lse)
    for lens in ([top, 3, 0, 3000, 64, 63, 2000, 1, 900], [1000] * 9, [0] * 8 + [top], [top] + [0] * 8, [top - 64 * b for b in range(9)]):
        s.lens = lens
        s.places = [(s.table[b, torch.arange(n + new) // 16].long(), torch.arange(n + new) % 16) for b, n in enumerate(lens)]
        dev["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        s.check(out, lse)


@pytest.mark.parametrize("seqs", [63, 64, 65])
def test_as_many_sequences_as_a_wave_has_lanes(seqs):
    lens = [(b * 37) % 700 if b % 5 else 0 for b in range(seqs)]
    news = [0 if b % 7 == 3 else 40 - b % 3 for b in range(seqs)]
    s = Setup(lens, news, 4, 1, 64, 16, seed=seqs, extra_rows=3)
    wide = torch.cat((s.table, torch.full((seqs, 200), -1, dtype=torch.int32)), 1)          # (many parts)
    s.check(*attend(s, table=wide.cuda()))


@pytest.mark.parametrize("d", [16, 48, 144, 208])
@pytest.mark.parametrize("lens,news,hq,hk,tree", [([500, 3], [1, 1], 71, 1, False), ([700, 0, 64], [2, 3, 1], 300, 1, True), ([90] * 40, [20] * 40, 9, 3, True), ([3300, 2000, 5], [60, 60, 1], 12, 1, True)])
def test_groups_and_widths_that_fill_no_block(lens, news, hq, hk, tree, d):
    s = Setup(lens, news, hq, hk, d, 48, blocks=3, tree=tree, seed=d + hq)
    s.check(*attend(s))
