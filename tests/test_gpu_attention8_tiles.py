"""Tiles of many rows over an 8-bit cache, one by one, cut, and sharing workgroups by their work: layouts, scales, masks, wrong pages and lengths, each at sizes that are planned so.  Against the
formula in 64 bits, with the tolerance of tests/test_gpu_attention8.py."""

import math

import pytest
import torch

from tests.attention8_plan import plan
from tests.test_gpu_attention8 import H, Setup, attend, i32
from tests.test_gpu_attention8_lengths import check_of

pytestmark = pytest.mark.gpu
BAD = 2 ** 31 - 1                                            # a table entry behind the sequences, outside any cache
WAYS = ["whole", "cut", "shared", "many_shared"]


def ragged(seqs, most_cached, most_new):
    return [(b * 37) % most_cached if b % 5 else 0 for b in range(seqs)], [0 if b % 7 == 3 else most_new - b % 4 for b in range(seqs)]


def setup(way, d, page=16, **kw):
    """(sequences, device's table for them), the table as wide as it takes for tiles; way "whole": more sequences than share workgroups, none cut; "cut": one in parts; "shared": a few, by their
    work, 256 rows a tile (128 of wide heads); "many_shared": as many as there are, 128 (64)."""
    lens, news, hq, hk = {"whole": (*ragged(50, 90, 20), 8, 4), "cut": ([2500], [30 if d > 128 else 50], 32, 8), "shared": ([500, 70, 0, 230], [50, 33, 47, 50], 8, 2),
                          "many_shared": (*ragged(40, 90, 20), 8, 4)}[way]
    s = Setup(lens, news, hq, hk, d, page, seed=d + len(lens) + page, extra_rows=2, **kw)
    cus, width = torch.cuda.get_device_properties(0).multi_processor_count, s.table.shape[1] - 1          # (its last column is no sequence's)
    while True:
        p = plan(s.n, len(lens), max(news), hq, hk, d, width * page, cus)
        right = {"whole": p.way == "tiles" and p.slots == 1, "cut": p.way == "tiles" and p.slots > 1, "shared": p.way == "shared", "many_shared": p.way == "shared"}[way]
        if right:
            break
        width += max(1, width // 2)
        assert width * page < 1 << 20, (way, p)              # (no width is planned so any more: choose other sizes)
    return s, widened(s, width)


def widened(s, width):
    return torch.cat((s.table, torch.full((s.table.shape[0], max(0, width - s.table.shape[1])), BAD, dtype=torch.int32)), 1)[:, :width].contiguous().cuda()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [16, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("way", WAYS)
def test_scales_far_apart(way, d, dtype):
    """Neighbouring blocks and heads with scales 2^20 apart, of keys and of values; entries behind the sequences are outside the cache."""
    s, table = setup(way, d, page=32, blocks=2, dtype=dtype)
    s.pool.scales[0] = torch.randint(100, 119, s.pool.scales[0].shape, generator=s.g).to(torch.uint8)
    s.pool.scales[1] = torch.randint(112 if dtype == "f16" else 60, 132, s.pool.scales[1].shape, generator=s.g).to(torch.uint8)
    s.check(*attend(s, table=table))


@pytest.mark.parametrize("permute", [(0, 2, 1, 3), (1, 0, 2, 3)])
@pytest.mark.parametrize("d", [48, 128, 256])
@pytest.mark.parametrize("way", WAYS)
def test_layouts(way, d, permute):
    """Pages with heads before slots and slots before pages, scales with heads before blocks, rows of a wider tensor; what lies beside the output stays."""
    s, table = setup(way, d, page=96, blocks=3)
    scales = [x.permute(2, 0, 1).contiguous().cuda().view(torch.float8_e8m0fnu).permute(1, 2, 0) for x in s.pool.scales]
    wide = torch.randn(s.n, s.hq + 3, d + 16, device="cuda").bfloat16()
    out = torch.full((s.n, s.hq + 2, d + 8), 3.0, device="cuda").bfloat16()
    q, o = wide[:, 2:2 + s.hq, 8:8 + d], out[:, 1:1 + s.hq, :d]
    q.copy_(s.q)
    got, lse = attend(s, permute, table=table, k_scale=scales[0], v_scale=scales[1], q=q, out=o)
    assert got is o
    s.check(got, lse)
    assert bool((out[:, 0] == 3).all()) and bool((out[:, -1] == 3).all()) and bool((out[..., d:] == 3).all()) and bool((out[s.starts[-1]:] == 3).all())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("way", WAYS)
def test_rows_that_see_nothing_and_masked_keys_that_hold_nan(way, d):
    s, table = setup(way, d, tree=True)
    b = max(i for i, n in enumerate(s.news) if n > 12 and s.lens[i])
    for i, n in enumerate(s.news):
        if n > 5:
            s.sees[i][:, 3] = False                          # nobody sees new token 3, whose key and value are NaN
            pg, off = s.places[i]
            s.pool.codes[:, pg[s.lens[i] + 3], off[s.lens[i] + 3]] = 0xFF
            s.sees[i][5] = False                             # and new token 5 sees none but the cached ones
    got, lse = attend(s, table=table)
    codes = s.pool.codes.clone()
    s.pool.codes[s.pool.codes & 127 == 127] = 0              # (the formula's zero weights need numbers)
    s.check(got, lse)
    for i, n in enumerate(s.news):
        if n > 5 and not s.lens[i]:
            row = s.starts[i] + 5
            assert not bool(got[row].any()) and bool((lse[row] == -math.inf).all())
    s.pool.codes = codes
    pg, off = s.places[b]
    s.pool.codes[1, pg[s.lens[b] + 8], off[s.lens[b] + 8], :, 7] = 0x7F          # a value's element is NaN: where it is seen, that element is
    again, _ = attend(s, table=table)
    sees, rows = s.sees[b][:, 8], slice(s.starts[b], s.starts[b + 1])
    new, old = again[rows].cpu(), got[rows].cpu()
    assert bool(new[sees][:, :, 7].isnan().all()) and not bool(new[~sees].isnan().any())
    new[sees, :, 7] = old[sees, :, 7]
    assert torch.equal(new, old)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("d", [80, 128, 256])
@pytest.mark.parametrize("way", WAYS)
def test_wrong_pages_and_sequences_beyond_their_tables(way, d, tree):
    s, table = setup(way, d, tree=tree)
    big = [b for b, (l, n) in enumerate(zip(s.lens, s.news)) if l > 48 and n]
    told, wrong = list(s.lens), []
    table[big[0], 2] = s.pool.codes.shape[1]
    wrong.append(big[0])
    if len(big) > 2:
        table[big[1], 3] = -1
        told[big[2]] = table.shape[1] * 16 - s.news[big[2]] + 1
        wrong += big[1:3]
    got, lse = attend(s, table=table, lens=i32(told))
    for b in wrong:
        rows = slice(s.starts[b], s.starts[b + 1])
        assert bool(got[rows].isnan().all()) and bool(lse[rows].isnan().all()), b
    for b in range(len(s.lens)):
        if b not in wrong:
            check_of(s, range(b, b + 1), got, lse)
    if len(big) < 3:
        told[big[0]] = table.shape[1] * 16
        table[big[0], 2] = s.table[big[0], 2].item()
        got, lse = attend(s, table=table, lens=i32(told))
        assert bool(got[s.starts[big[0]]:s.starts[big[0] + 1]].isnan().all())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("way", WAYS)
def test_large_scores(way, d):
    """Scores of some thousands.  Weights far below a row's largest then end where 32 bits (and bf16) do: what is taken off the exponents is at most the row's maximum, so the largest weight
    and the total are 1 or more, and a weight, a product of a weight and a value, or a sum scaled down to a later maximum is lost below 2^-126.  L keys have L of the first two, and no sum is
    scaled more often than there are keys: off by at most (2 + 1) L 2^-126 max(1, max |v|), and by 2^-126 where the result is.  It shows where the key of the largest weight has a value of zero."""
    s, table = setup(way, d, low=124, high=131)
    got, lse = attend(s, table=table)
    values, group = s.pool.values(), s.hq // s.hk
    for b, (l, n) in enumerate(zip(s.lens, s.news)):
        if not n:
            continue
        rows, (pg, off) = slice(s.starts[b], s.starts[b + 1]), s.places[b]
        k, v = (values[i, pg, off].transpose(0, 1).repeat_interleave(group, 0) for i in range(2))
        q = s.q[rows].double().transpose(0, 1)
        sees = torch.cat((torch.ones(n, l, dtype=torch.bool), s.sees[b]), 1)
        score = torch.where(sees, (q @ k.transpose(1, 2)) * s.scale, -math.inf)
        ds = (d + 4) * H * s.scale * torch.where(sees, q.abs() @ k.abs().transpose(1, 2), 0.0).amax(-1)
        p = torch.softmax(score, -1)
        out, big = p @ v, p @ v.abs()
        lost = 2.0 ** -126 * (3 * (l + n) * max(1.0, float(v.abs().max())) + 1)
        tol = (2.0 ** -8 * 1.01 + 2 * ds[..., None] + (l + n + 64) * H) * big + 2.0 ** -8 * out.abs() + lost
        off_by = (got[rows].cpu().double().transpose(0, 1) - out).abs()
        assert bool((off_by <= tol).all()), (b, float((off_by / tol).max()))
        want = torch.logsumexp(score, -1)
        assert bool(((lse[rows].cpu().double().T - want).abs() <= ds + (l + n + 64) * H + 4 * H * torch.maximum(want.abs(), score.amax(-1).abs()).clamp(min=1)).all()), b


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("way", ["cut", "shared"])
def test_pages_gigabytes_apart(way, d):
    s, table = setup(way, d, page=64)
    dev, n, size = s.device(), s.pool.codes.shape[1], 64 * s.hk * d
    far = torch.zeros(5 * 2 ** 30 // 2048 * 2048, dtype=torch.uint8, device="cuda")
    step = far.numel() // n // 2048 * 2048
    assert step >= 2 * size and (n - 1) * step > 2 ** 32
    caches = [torch.as_strided(far, (n, 64, s.hk, d), (step, s.hk * d, d, 1), at * size) for at in range(2)]
    for c, kind in zip(caches, ("k_cache", "v_cache")):
        c.copy_(dev[kind].view(torch.uint8))
    s.check(*attend(s, table=table, k_cache=caches[0].view(torch.float8_e4m3fn), v_cache=caches[1].view(torch.float8_e4m3fn)))


@pytest.mark.parametrize("blocks", [1, 4, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_page_per_sequence(d, blocks):
    """The contiguous cache, one page each, of one block and of many."""
    s = Setup([900, 0, 300], [70, 3, 50], 8, 2, d, 1024, blocks, seed=blocks)
    width = 1
    while plan(s.n, 3, 70, 8, 2, d, width * 1024, torch.cuda.get_device_properties(0).multi_processor_count).way != "shared":
        width += 1
        assert width < 1000
    s.check(*attend(s, table=widened(s, max(width, s.table.shape[1]))))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("way", WAYS)
def test_the_same_bits_every_time(way, d):
    s, table = setup(way, d, tree=True)
    first, lse = attend(s, table=table)
    for _ in range(3):
        again, other = attend(s, table=table)
        assert torch.equal(again[:s.starts[-1]], first[:s.starts[-1]]) and torch.equal(other, lse)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_a_last_tile_cut_into_fewer_parts(d, tree, dtype):
    """More sequences than share workgroups, each of a whole tile and one filled by half and cut less."""
    seqs, new = 40 if d == 256 else 35, 40 if d == 256 else 75
    lens = [(b * 61) % 700 for b in range(seqs)]
    s = Setup(lens, [new - b % 3 for b in range(seqs)], 4, 1, d, 16, dtype=dtype, tree=tree, seed=d)
    cus, width = torch.cuda.get_device_properties(0).multi_processor_count, s.table.shape[1]
    while True:
        p = plan(s.n, seqs, new, 4, 1, d, width * 16, cus)
        if p.way == "tiles" and p.blocks == 2 and 1 < p.last_splits < p.splits:
            break
        width += 8
        assert width * 16 < 1 << 16, p
    s.check(*attend(s, table=widened(s, width)))
