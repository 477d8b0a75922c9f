"""Attention over a cache held in 8 bits, against its formula in 64 bits on the numbers that the cache holds.

Tolerance of a result, from what the kernels round; it is that of attention over a 16-bit cache, since code * scale goes into the products exactly.  Half a step of 32 bits is
h = 2^-24, of the type u = finfo.eps / 2.  A score is a sum of D exact products, off by at most D h scale sum |q||k|, and a rounding of its scaled value and of the
exponential: ds = (D + 4) h scale max_j sum |q||k|, which is what weights are off by, relative, in numerator and denominator alike (2 ds).  The weights of the second product are rounded
to the type (u), the sums of L terms and their joining in 32 bits add at most (L + 64) h, all relative to A = sum softmax |v|; the result is rounded once: u |out|.
lse: ds, the total's (L + 64) h, and the logarithm's rounding, 4 h max(1, |lse|, |maximum|)."""

import math

import pytest
import torch

from tests.cache8_model import CODES, Pool, table_for
from tests.test_gpu_attention import tree_of, words_of

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
H = 2.0 ** -24
i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()


class Setup:
    """Sequences of `lens` cached and `news` new tokens in a pool whose other slots hold NaN, in blocks of scales of their own."""

    def __init__(self, lens, news, hq, hk, d, page, blocks=1, dtype="bf16", tree=False, seed=0, extra_rows=0, spare=3, low=115, high=121):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.news, self.hq, self.hk, self.d, self.dt, self.tree = lens, news, hq, hk, d, DT[dtype], tree
        self.table, pages, _ = table_for([a + b for a, b in zip(lens, news)], page, g, spare)
        self.pool = Pool(pages, page, blocks, hk, d, g)
        self.pool.codes = torch.randint(0, 120, self.pool.codes.shape, generator=g).to(torch.uint8) | torch.randint(0, 2, self.pool.codes.shape, generator=g).to(torch.uint8) << 7
        self.pool.scales = torch.randint(low, high, self.pool.scales.shape, generator=g).to(torch.uint8)
        self.places = []
        taken = torch.zeros(pages, page, dtype=torch.bool)
        for b, (l, n) in enumerate(zip(lens, news)):
            s = torch.arange(l + n)
            pg = self.table[b, s // page].long()
            self.places.append((pg, s % page))
            taken[pg, s % page] = True
        self.pool.codes[:, ~taken] = 0x7F                    # NaN
        self.starts = [0]
        for n in news:
            self.starts.append(self.starts[-1] + n)
        self.n = self.starts[-1] + extra_rows
        self.q = torch.randn(self.n, hq, d, generator=g).to(self.dt)
        self.sees = [tree_of(n, g) if tree else torch.ones(n, n, dtype=torch.bool).tril() for n in news]
        self.scale = d ** -0.5
        self.g = g

    def mask(self):
        if not self.tree:
            return None
        rows = torch.zeros(self.n, max(1, max(self.news)), dtype=torch.bool)
        for b, s in enumerate(self.sees):
            rows[self.starts[b]:self.starts[b + 1], :s.shape[1]] = s
        return words_of(rows).cuda()

    def device(self, permute=None):
        kc, vc, ks, vs = self.pool.device(permute)
        return dict(q=self.q.cuda(), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, table=self.table.cuda(), lens=i32(self.lens), starts=i32(self.starts),
                    most_new=max(self.news), mask=self.mask(), scale=self.scale)

    def check(self, got, got_lse=None):
        u, group, values = torch.finfo(self.dt).eps / 2, self.hq // self.hk, self.pool.values()
        floor = torch.finfo(self.dt).tiny * torch.finfo(self.dt).eps
        for b, (l, n) in enumerate(zip(self.lens, self.news)):
            if not n:
                continue
            pg, off = self.places[b]
            k, v = (values[i, pg, off].transpose(0, 1).repeat_interleave(group, 0) for i in range(2))          # [hq, l + n, d]
            q = self.q[self.starts[b]:self.starts[b + 1]].double().transpose(0, 1)
            sees = torch.cat((torch.ones(n, l, dtype=torch.bool), self.sees[b]), 1)
            s = (q @ k.transpose(1, 2)) * self.scale
            s = torch.where(sees, s, -math.inf)
            ds = (self.d + 4) * H * self.scale * torch.where(sees, q.abs() @ k.abs().transpose(1, 2), 0.0).amax(-1)
            some = sees.any(-1)
            p = torch.where(some[:, None], torch.softmax(s, -1), 0.0)
            out, big = p @ v, p @ v.abs()
            tol = (u * 1.01 + 2 * ds[..., None] + (l + n + 64) * H) * big + u * out.abs() + floor
            mine = got.cpu().double()[self.starts[b]:self.starts[b + 1]].transpose(0, 1)
            off_by = (mine - out).abs()
            assert bool((off_by <= tol).all()), (b, float((off_by / tol).nan_to_num(posinf=1e30).max()), int((~(off_by <= tol)).sum()))
            if got_lse is not None:
                lse = torch.logsumexp(s, -1)
                top = s.amax(-1).abs().nan_to_num(posinf=0.0)
                ltol = ds + (l + n + 64) * H + 4 * H * torch.maximum(torch.ones_like(top), torch.maximum(lse.abs().nan_to_num(posinf=0.0), top))
                gl = got_lse.cpu().double()[self.starts[b]:self.starts[b + 1]].T
                assert bool(((gl == lse) | ((gl - lse).abs() <= ltol)).all()), (b, float((gl - lse).abs().nan_to_num().max()))


def attend(s, permute=None, **kw):
    from quantexperiments_amd.kernels import tree_attention8
    lse = torch.full((s.n, s.hq), 5.0, device="cuda")
    return tree_attention8(**{**s.device(permute), **kw}, lse=lse), lse


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("d", [16, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("lens,news,hq,hk,page,blocks,tree", [
    ([0], [1], 1, 1, 16, 1, False), ([1], [1], 7, 1, 16, 1, False), ([15, 16, 30, 31, 32, 33], [1, 1, 1, 1, 1, 1], 4, 2, 16, 1, False), ([700], [1], 14, 2, 32, 2, False),
    ([130, 0, 65], [3, 0, 17], 6, 3, 48, 1, True), ([40], [70], 2, 1, 64, 4, True), ([5, 300], [40, 2], 5, 1, 96, 3, False), ([0, 17], [33, 64], 8, 2, 16, 1, False)])
def test_matches_the_formula(lens, news, hq, hk, page, blocks, tree, d, dtype):
    s = Setup(lens, news, hq, hk, d, page, blocks, dtype, tree, seed=d + len(lens), extra_rows=2)
    s.check(*attend(s))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens,news,hq,hk,tree", [([3000], [1], 8, 2, False), ([2000, 900], [48, 30], 14, 2, True), ([1500, 40], [200, 333], 4, 1, False), ([5000, 4000, 1], [2, 1, 2], 10, 2, False)])
def test_longer_ones(lens, news, hq, hk, tree, d, dtype):
    s = Setup(lens, news, hq, hk, d, 64, 2, dtype, tree, seed=d)
    s.check(*attend(s))


def test_one_key_is_its_value():
    """A softmax of one key is 1: every finite code at every scale comes out as the number it stands for, as far as the type has it as a normal number."""
    from quantexperiments_amd.kernels import tree_attention8
    codes = torch.arange(256, dtype=torch.uint8)
    codes[codes & 127 == 127] = 0
    for dtype, scales in ((torch.bfloat16, range(1, 255)), (torch.float16, range(100, 136))):
        e = torch.tensor(list(scales), dtype=torch.uint8)
        n = len(e)
        kc = torch.zeros(n, 16, 1, 256, dtype=torch.uint8, device="cuda")
        vc = kc.clone()
        vc[:, 0, 0] = codes.cuda()
        ks, vs = torch.full((n, 1, 1), 127, dtype=torch.uint8, device="cuda"), e.cuda().view(n, 1, 1)
        out = tree_attention8(torch.randn(n, 1, 256, device="cuda").to(dtype), kc.view(torch.float8_e4m3fn), vc.view(torch.float8_e4m3fn), ks.view(torch.float8_e8m0fnu),
                              vs.contiguous().view(torch.float8_e8m0fnu), torch.arange(n, dtype=torch.int32, device="cuda")[:, None], i32([0] * n))
        want = CODES[codes.long()] * torch.pow(2.0, e.double() - 127)[:, None]
        top, small = torch.finfo(dtype).max, torch.finfo(dtype).tiny if dtype == torch.bfloat16 else 2.0 ** -24
        fits = (want.abs() <= top) & (want == want.to(dtype).double()) & ((want == 0) | (want.abs() >= small))
        assert torch.equal(out[:, 0].cpu().double()[fits], want[fits]), dtype
        assert dtype == torch.float16 or bool(fits[26:246].all())             # (the scales that put_tokens8 makes)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("hq,news", [(4, 1), (4, 40), (8, 40)])
def test_scales_far_apart(dtype, hq, news):
    """Neighbouring blocks and heads with scales 2^20 apart, of keys and of values."""
    s = Setup([500], [news], hq, 2, 64, 32, 2, dtype, seed=5)
    s.pool.scales[0] = torch.randint(100, 119, s.pool.scales[0].shape, generator=s.g).to(torch.uint8)
    s.pool.scales[1] = torch.randint(112 if dtype == "f16" else 60, 132, s.pool.scales[1].shape, generator=s.g).to(torch.uint8)
    s.check(*attend(s))


@pytest.mark.parametrize("permute", [None, (0, 2, 1, 3), (1, 0, 2, 3)])
@pytest.mark.parametrize("news", [[1, 2], [60, 3]])
def test_layouts(permute, news):
    s = Setup([70, 200], news, 6, 3, 96, 32, 2, "bf16", seed=6)
    s.check(*attend(s, permute))
    wide = torch.randn(s.n, 9, 112, device="cuda").bfloat16()
    out = torch.full((s.n, 8, 104), 3.0, device="cuda").bfloat16()
    q, o = wide[:, 2:8, 8:104], out[:, 1:7, :96]
    q.copy_(s.q)
    got, lse = attend(s, permute, q=q, out=o)
    assert got is o
    s.check(got, lse)
    assert bool((out[:, 0] == 3).all()) and bool((out[:, 7] == 3).all()) and bool((out[..., 96:] == 3).all())


@pytest.mark.parametrize("news", [[1, 1, 1], [7, 0, 90]])
def test_rows_behind_the_last_sequence_are_left(news):
    from quantexperiments_amd.kernels import tree_attention8
    s = Setup([40, 3, 100], news, 4, 1, 64, 16, seed=7, extra_rows=5)
    out, lse = torch.full((s.n, 4, 64), 9.0, device="cuda").bfloat16(), torch.full((s.n, 4), 9.0, device="cuda")
    tree_attention8(**s.device(), out=out, lse=lse)
    s.check(out, lse)
    assert bool((out[s.starts[-1]:] == 9).all()) and bool((lse[s.starts[-1]:] == 9).all())


@pytest.mark.parametrize("hq,new", [(2, 9), (8, 60)])
def test_rows_that_see_nothing_and_masked_keys_that_hold_nan(hq, new):
    s = Setup([0, 50], [new, new], hq, 2, 128, 16, tree=True, seed=8)
    for b in range(2):
        s.sees[b][:, 3] = False                              # nobody sees new token 3, whose key and value are NaN
        pg, off = s.places[b]
        s.pool.codes[:, pg[s.lens[b] + 3], off[s.lens[b] + 3]] = 0xFF
    s.sees[0][5] = False
    s.sees[0][3] = False
    got, lse = attend(s)
    values = s.pool.codes.clone()
    s.pool.codes[s.pool.codes & 127 == 127] = 0
    s.check(got, lse)
    assert not bool(got[3].any()) and not bool(got[5].any()) and bool((lse[5] == -math.inf).all())
    s.pool.codes = values
    pg, off = s.places[1]
    s.pool.codes[1, pg[s.lens[1] + 2], off[s.lens[1] + 2], :, 7] = 0x7F          # a value's element is NaN: where it is seen, that element is
    got2, _ = attend(s)
    sees = s.sees[1][:, 2]
    rows = got2[s.starts[1]:].cpu()
    assert bool(rows[sees][:, :, 7].isnan().all()) and not bool(rows[~sees].isnan().any())
    keep = torch.ones(128, dtype=torch.bool)
    keep[7] = False
    assert torch.equal(rows[..., keep], got.cpu()[s.starts[1]:][..., keep])


def test_an_empty_mask_shows_the_cached_tokens_alone():
    s = Setup([33, 0], [4, 3], 4, 2, 64, 16, tree=True, seed=9)
    for m in s.sees:
        m[:] = False
    got, lse = attend(s, mask=torch.empty(s.n, 0, dtype=torch.int64, device="cuda"))
    s.check(got, lse)


@pytest.mark.parametrize("news", [[1, 1, 1, 1], [50, 60, 2, 1]])
def test_pages_outside_the_cache_and_sequences_beyond_their_table(news):
    s = Setup([100, 20, 100, 40], news, 4, 1, 64, 16, seed=10)
    table = s.table.clone()
    table[0, 3] = s.pool.codes.shape[1]
    table[2, 5] = -1
    lens = list(s.lens)
    lens[1] = table.shape[1] * 16
    got, lse = attend(s, table=table.cuda(), lens=i32(lens))
    for b in range(3):
        rows = slice(s.starts[b], s.starts[b + 1])
        assert bool(got[rows].isnan().all()) and bool(lse[rows].isnan().all()), b
    s.lens, s.news = s.lens[3:], s.news[3:]
    s.starts, s.places, s.sees = s.starts[3:], s.places[3:], s.sees[3:]
    s.check(got, lse)
    s2 = Setup([3], [2], 4, 1, 64, 16, seed=11)
    got, _ = attend(s2, lens=i32([-50]), most_new=2)
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("rows", [1, 45])
def test_bad_entries_behind_a_sequence_do_not_matter(rows):
    s = Setup([90], [rows], 4, 2, 128, 16, seed=12)
    wide = torch.cat((s.table, torch.full((1, 40), 2 ** 31 - 1, dtype=torch.int32)), 1)
    s.check(*attend(s, table=wide.cuda()))


def test_large_scores_and_pages_far_apart():
    """Scores of some thousands; a pool whose pages lie gigabytes apart."""
    from quantexperiments_amd.kernels import tree_attention8
    s = Setup([300], [1], 4, 1, 64, 16, seed=13, low=124, high=131)
    s.check(*attend(s))
    for news in ([1], [40]):
        s = Setup([400], news, 4, 1, 64, 16, seed=14)
        dev = s.device()
        n = s.pool.codes.shape[1]
        far = torch.zeros(3 * 2 ** 30 // 1024 * 1024, dtype=torch.uint8, device="cuda")
        step = far.numel() // n // 1024 * 1024
        k = torch.as_strided(far, (n, 16, 1, 64), (step, 64, 64, 1))
        k.copy_(dev["k_cache"].view(torch.uint8))
        v = torch.as_strided(far, (n, 16, 1, 64), (step, 64, 64, 1), 16 * 64)
        v.copy_(dev["v_cache"].view(torch.uint8))
        lse = torch.empty(s.n, 4, device="cuda")
        s.check(tree_attention8(**{**dev, "k_cache": k.view(torch.float8_e4m3fn), "v_cache": v.view(torch.float8_e4m3fn)}, lse=lse), lse)


@pytest.mark.parametrize("d,hk,cached,new", [(128, 4, 4900, 1), (64, 8, 4900, 1), (128, 4, 2400, 40), (128, 4, 4500, 140), (256, 4, 2200, 20)])
def test_many_sequences_of_long_ones(d, hk, cached, new):
    """As many as fill the chip, so that a wave walks through more keys than it looks up at once; against the formula on the GPU, in 64 bits."""
    from quantexperiments_amd.kernels import tree_attention8
    seqs, page = 256 // hk, 64
    g = torch.Generator(device="cuda").manual_seed(d + new)
    lens = [cached + 3 * b for b in range(seqs)]
    need = [-(-(l + new) // page) for l in lens]
    order = torch.randperm(sum(need), generator=g, device="cuda").int()
    table, at = torch.full((seqs, max(need)), -1, dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (sum(need), page, hk, d)
    codes = [torch.randint(0, 120, shape, generator=g, device="cuda", dtype=torch.uint8) | torch.randint(0, 2, shape, generator=g, device="cuda", dtype=torch.uint8) << 7 for _ in range(2)]
    scales = [torch.randint(114, 121, (sum(need), 2, hk), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
    q = torch.randn(seqs * new, hk, d, generator=g, device="cuda").bfloat16()
    out = tree_attention8(q, *(c.view(torch.float8_e4m3fn) for c in codes), *(s.view(torch.float8_e8m0fnu) for s in scales), table, i32(lens))
    known, u = CODES.cuda(), 2.0 ** -8
    for b in range(0, seqs, 5):
        s = torch.arange(lens[b] + new, device="cuda")
        pg, off = table[b, s // page].long(), s % page
        k, v = ((known[c[pg, off].long()] * torch.pow(2.0, f[pg, off // 32].double() - 127)[..., None]).transpose(0, 1).contiguous() for c, f in zip(codes, scales))
        x = q[b * new:(b + 1) * new].double().transpose(0, 1)
        score = torch.matmul(x, k.transpose(1, 2).contiguous()) * d ** -0.5
        sees = s <= lens[b] + torch.arange(new, device="cuda")[:, None]
        p = torch.softmax(torch.where(sees, score, -math.inf), -1)
        want, big = torch.matmul(p, v), torch.matmul(p, v.abs())
        ds = (d + 4) * H * d ** -0.5 * torch.matmul(x.abs(), k.abs().transpose(1, 2).contiguous()).amax(-1)
        tol = (u * 1.01 + 2 * ds[..., None] + (len(s) + 64) * H) * big + u * want.abs()
        off_by = (out[b * new:(b + 1) * new].double().transpose(0, 1) - want).abs()
        assert bool((off_by <= tol).all()), (b, float((off_by / tol).max()))


def test_a_page_per_sequence_and_strided_scales():
    """The contiguous cache: one page each, of one block and of many; scales whose heads come before their blocks."""
    for news in ([1, 1, 1], [70, 3, 1]):
        for blocks in (1, 4, 64):
            s = Setup([900, 0, 300], news, 4, 2, 64, 1024, blocks, seed=blocks)
            s.check(*attend(s))
            wide = [x.permute(2, 0, 1).contiguous().cuda().view(torch.float8_e8m0fnu).permute(1, 2, 0) for x in s.pool.scales]
            s.check(*attend(s, k_scale=wide[0], v_scale=wide[1]))


def test_captured_with_changing_lengths_on_two_streams():
    from quantexperiments_amd.kernels import tree_attention8
    s = Setup([900, 500], [1, 1], 8, 2, 128, 16, seed=15)
    dev = s.device()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = tree_attention8(**dev)
    for lens in ([900, 500], [3, 499], [0, 0], [700, 16]):
        dev["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        eager = tree_attention8(**dev)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        t = Setup([900, 500], [1, 1], 8, 2, 128, 16, seed=15)
        t.lens = lens
        t.places = [(pg[:l + 1], off[:l + 1]) for (pg, off), l in zip(t.places, lens)]
        t.check(eager)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(tree_attention8(**dev))
    torch.cuda.synchronize()
    assert all(torch.equal(g, eager) for g in got)


def test_the_same_bits_every_time():
    from quantexperiments_amd.kernels import tree_attention8
    for lens, news, tree in (([3000, 10], [1, 1], False), ([800, 300], [48, 47], True)):
        s = Setup(lens, news, 14, 2, 128, 32, 2, tree=tree, seed=16)
        dev = s.device()
        first = tree_attention8(**dev)
        for _ in range(3):
            assert torch.equal(tree_attention8(**dev), first)


def test_a_generation_with_drafts_forks_and_compaction():
    """A prompt put and attended in chunks, forked, drafted trees verified and kept, a sequence ended and its pages freed: at the end the cache holds every
    token of each sequence to its rounding, and attention is that over what it holds."""
    from quantexperiments_amd import kernels as K
    g = torch.Generator().manual_seed(17)
    hq, hk, d, page, pages = 8, 2, 64, 16, 40
    kc, vc = (torch.full((1, pages, page, hk, d), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros(1, pages, 1, hk, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
    layer = (kc[0], vc[0], ks[0], vs[0])
    order = torch.randperm(pages, generator=g).int()
    table, lens, free = torch.full((1, 8), -1, dtype=torch.int32), [0], order[4:].tolist()
    table[0, :4] = order[:4]
    table = table.cuda()
    hist = [([], [])]                                        # keys and values of each sequence, as held in 16 bits
    new = lambda n: tuple((torch.randn(n, hk, d, generator=g) * 0.5).bfloat16() for _ in range(2))

    def step(news, mask=None):
        k, v = (torch.cat(x) for x in zip(*news))
        starts, at = [0], 0
        for n in news:
            starts.append(starts[-1] + len(n[0]))
        most = max(len(n[0]) for n in news)
        K.put_tokens8(k.cuda(), v.cuda(), *layer, table, i32(lens), i32(starts), most_new=most)
        q = torch.randn(len(k), hq, d, generator=g).bfloat16().cuda()
        return q, K.tree_attention8(q, *layer, table, i32(lens), i32(starts), most_new=most, mask=mask), starts

    for n in (20, 13):                                       # chunks of the prompt
        x = new(n)
        step([x])
        hist[0][0].append(x[0])
        hist[0][1].append(x[1])
        lens[0] += n
    table, l = K.fork_pages(kc, vc, table, i32(lens), i32([0, 0, 0]), i32([-1, free[0], free[1]]), k_scale=ks, v_scale=vs)
    free = free[2:]
    lens = l.tolist()
    hist = [([*hist[0][0]], [*hist[0][1]]) for _ in range(3)]
    own = [free[:2], free[2:4], free[4:6]]
    t = table.cpu()
    for b in range(3):
        t[b, 3:5] = torch.tensor(own[b], dtype=torch.int32)
    table = t.cuda()
    # trees of 12 drafts: a spine 0, 2, 5, 11 and others; the spine is kept as far as it was accepted
    parents = [-1, 0, 0, 1, 2, 2, 3, 4, 5, 5, 8, 9]
    sees = torch.eye(12, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            sees[i] |= sees[p]
    drafts = [new(12) for _ in range(3)]
    step(drafts, words_of(torch.cat([sees] * 3)).cuda())
    path, counts = i32([[0, 2, 5, 9]] * 3), [4, 1, 3]
    K.keep_drafted8(kc, vc, ks, vs, table, i32(lens), path, i32(counts))
    for b, c in enumerate(counts):
        for j in range(2):
            hist[b][j].append(drafts[b][j][[0, 2, 5, 9][:c]])
        lens[b] += c
    # the second one ends
    keep = [0, 2]
    table, lens, hist = table[keep].contiguous(), [lens[b] for b in keep], [hist[b] for b in keep]
    table, used = K.compact_pages(kc, vc, table, i32(lens), k_scale=ks, v_scale=vs)
    need = {int(table[b, j]) for b in range(2) for j in range(-(-lens[b] // page))}
    assert need == set(range(int(used)))
    last = [new(1) for _ in range(2)]
    t = table.cpu()
    for b in range(2):
        if lens[b] % page == 0:
            t[b, lens[b] // page] = int(used) + b
    table = t.cuda()
    q, got, starts = step(last)
    for b in range(2):
        for j in range(2):
            hist[b][j].append(last[b][j])
        k, v = (torch.cat(x).double() for x in hist[b])
        lay = [c.cpu().view(torch.uint8) for c in layer]
        tb = table.cpu()
        s = torch.arange(lens[b] + 1)
        pg, off = tb[b, s // page].long(), s % page
        kv = [CODES[lay[j][pg, off].long()] * torch.pow(2.0, lay[2 + j][pg, 0].double() - 127)[..., None] for j in range(2)]
        for x, y in ((kv[0], k), (kv[1], v)):
            # one rounding, by 2^-4 of the element or 2^-10 of the block's scale, which is at most 2 / 448 of its largest; another 2^-10 where that grew
            assert bool(((x - y).abs() <= 2.0 ** -4 * y.abs() + 2 * 2.0 ** -10 * 2 / 448 * y.abs().max()).all())
        sc = torch.einsum("hd,shd->hs", q[b].cpu().double(), kv[0].repeat_interleave(4, 1)) * d ** -0.5
        out = torch.einsum("hs,shd->hd", torch.softmax(sc, -1), kv[1].repeat_interleave(4, 1))
        big = torch.einsum("hs,shd->hd", torch.softmax(sc, -1), kv[1].abs().repeat_interleave(4, 1))
        assert bool(((got[b].cpu().double() - out).abs() <= 2.0 ** -8 * (1.02 * big + out.abs())).all())


def test_refusals():
    from quantexperiments_amd.kernels import tree_attention8
    from quantexperiments_amd._lib import SqError
    s = Setup([20, 9], [2, 2], 4, 2, 64, 32, 2, seed=18)
    ok = s.device()
    q, kc, ks = ok["q"], ok["k_cache"], ok["k_scale"]
    bad = [dict(q=q.float()), dict(q=q[0]), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(k_cache=kc.view(torch.uint8)), dict(k_cache=kc[:1]), dict(k_scale=ks.view(torch.uint8)), dict(k_scale=ks[:, :1]),
           dict(k_scale=ks[:1], v_scale=ks[:1]), dict(table=ok["table"].long()), dict(table=ok["table"][:1]), dict(lens=ok["lens"].cpu()), dict(starts=ok["starts"][:2]), dict(starts=None),
           dict(most_new=-1), dict(scale=0.0), dict(scale=float("nan")), dict(mask=torch.zeros(3, 1, dtype=torch.int64, device="cuda")), dict(out=q), dict(out=q.half()), dict(out=q[:1].expand_as(q)),
           dict(lse=torch.empty(4, 4, device="cuda").half()), dict(lse=torch.empty(4, 3, device="cuda"))]
    for b in bad:
        if b == dict(starts=None):
            b = dict(starts=None, most_new=1)
        try:
            tree_attention8(**{**ok, **b})
        except ValueError:
            continue
        raise AssertionError(list(b))
    for b in (dict(q=q[..., 1:49], k_cache=kc[..., :48], v_cache=ok["v_cache"][..., :48]), dict(q=q[..., :24].contiguous(), k_cache=kc[..., :24], v_cache=ok["v_cache"][..., :24])):
        with pytest.raises(SqError):
            tree_attention8(**{**ok, **b})
    with pytest.raises(NotImplementedError):
        tree_attention8(**{**ok, "q": q.clone().requires_grad_()})
