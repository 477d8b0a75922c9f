"""Attention of new tokens over a paged cache, against its formula in 64 bits.

Tolerance of a result, from what the kernel rounds.  Half a step of 32 bits is h = 2^-24, of the type u = finfo.eps / 2.  A score is a sum of D
exact products, off by at most D h scale sum |q||k|, and a rounding of its scaled value and of the exponential: ds = (D + 4) h scale max_j sum |q||k|.  That is
what weights are off by, relative, in numerator and denominator alike (2 ds).  The weights of the second product are rounded to the type (u), the sums
of L terms and their joining in 32 bits add at most (L + 64) h, all relative to A = sum softmax |v|; the result is rounded once: u |out|.
lse: ds, the total's (L + 64) h, and the logarithm's rounding, 4 h max(1, |lse|, |maximum|)."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
H = 2.0 ** -24


def words_of(sees):
    """Truth values [N, n] as 64-bit words [N, ceil(n / 64)]."""
    n, w = sees.shape[1], max(1, -(-sees.shape[1] // 64))
    out = np.zeros((sees.shape[0], w), dtype=np.uint64)
    s = sees.numpy()
    for j in range(n):
        out[:, j // 64] |= s[:, j].astype(np.uint64) << np.uint64(j % 64)
    return torch.from_numpy(out.view(np.int64))


def tree_of(n, g):
    """Ancestors-and-self of a random tree, [n, n]."""
    sees = torch.eye(n, dtype=torch.bool)
    for t in range(1, n):
        p = int(torch.randint(-1, t, (1,), generator=g))
        if p >= 0:
            sees[t] |= sees[p]
    return sees


class Setup:
    """Sequences of `lens` cached and `news` new tokens in a paged cache of slots that otherwise hold NaN."""

    def __init__(self, lens, news, hq, hk, d, page, dtype="bf16", tree=False, seed=0, extra_rows=0, scale=2.0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.g, self.lens, self.news, self.hq, self.hk, self.d, self.page, self.dt = g, lens, news, hq, hk, d, page, DT[dtype]
        need = [-(-(a + b) // page) for a, b in zip(lens, news)]
        order = torch.randperm(sum(need) + spare, generator=g)
        self.table = torch.full((len(lens), max(need) + 1), -7, dtype=torch.int32)
        at = 0
        self.k, self.v = [], []
        self.kc, self.vc = (torch.full((len(order), page, hk, d), float("nan"), dtype=self.dt) for _ in range(2))
        for b, (l, n) in enumerate(zip(lens, news)):
            self.table[b, :need[b]] = order[at:at + need[b]].int()
            at += need[b]
            k, v = (torch.randn(l + n, hk, d, generator=g).to(self.dt) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
        self.put()
        self.starts = [0]
        for n in news:
            self.starts.append(self.starts[-1] + n)
        self.n = self.starts[-1] + extra_rows
        self.q = (torch.randn(self.n, hq, d, generator=g) * scale).to(self.dt)
        self.sees = [tree_of(n, g) if tree else torch.ones(n, n, dtype=torch.bool).tril() for n in news]
        self.tree = tree
        self.scale = d ** -0.5

    def put(self):
        for b, (k, v) in enumerate(zip(self.k, self.v)):
            s = torch.arange(len(k))
            pg = self.table[b, s // self.page].long()
            self.kc[pg, s % self.page], self.vc[pg, s % self.page] = k, v

    def mask(self):
        if not self.tree:
            return None
        most = max(1, max(self.news))
        rows = torch.zeros(self.n, most, dtype=torch.bool)
        for b, s in enumerate(self.sees):
            rows[self.starts[b]:self.starts[b + 1], :s.shape[1]] = s
        return words_of(rows).cuda()

    def device(self):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
        return dict(q=self.q.cuda(), k_cache=self.kc.cuda(), v_cache=self.vc.cuda(), table=self.table.cuda(), lens=i32(self.lens), starts=i32(self.starts),
                    most_new=max(self.news), mask=self.mask(), scale=self.scale)

    def reference(self):
        """(out, tolerance, lse, tolerance), rows of no sequence NaN."""
        hq, hk, d = self.hq, self.hk, self.d
        out, tol = (torch.full((self.n, hq, d), float("nan"), dtype=torch.float64) for _ in range(2))
        lse, ltol = (torch.full((self.n, hq), float("nan"), dtype=torch.float64) for _ in range(2))
        u = torch.finfo(self.dt).eps / 2
        for b, (l, n) in enumerate(zip(self.lens, self.news)):
            k, v = self.k[b].double(), self.v[b].double()
            sees = torch.cat((torch.ones(n, l, dtype=torch.bool), self.sees[b]), 1)
            for h in range(hq):
                q = self.q[self.starts[b]:self.starts[b + 1], h].double()
                kk, vv = k[:, h // (hq // hk)], v[:, h // (hq // hk)]
                for t in range(n):
                    see = sees[t]
                    r = self.starts[b] + t
                    if not see.any():
                        out[r, h], tol[r, h], lse[r, h], ltol[r, h] = 0, 0, -math.inf, 0
                        continue
                    s = kk[see] @ q[t] * self.scale
                    ds = (d + 4) * H * self.scale * float((kk[see].abs() @ q[t].abs()).max())
                    p = torch.softmax(s, 0)
                    big = (p[:, None] * vv[see].abs()).sum(0)
                    out[r, h] = p @ vv[see]
                    tol[r, h] = (u * 1.01 + 2 * ds + (len(s) + 64) * H) * big + u * out[r, h].abs() + torch.finfo(self.dt).tiny * torch.finfo(self.dt).eps
                    lse[r, h] = torch.logsumexp(s, 0)
                    ltol[r, h] = ds + (len(s) + 64) * H + 4 * H * max(1.0, abs(float(lse[r, h])), abs(float(s.max())))
        return out, tol, lse, ltol

    def check(self, got, got_lse=None):
        out, tol, lse, ltol = self.reference()
        rows = self.starts[-1]
        got = got.cpu().double()[:rows]
        off = (got - out[:rows]).abs()
        assert bool((off <= tol[:rows]).all()), (float((off / tol[:rows]).nan_to_num(posinf=1e30).max()), int((~(off <= tol[:rows])).sum()))
        if got_lse is not None:
            gl = got_lse.cpu().double()[:rows]
            same = (gl == lse[:rows]) | ((gl - lse[:rows]).abs() <= ltol[:rows])
            assert bool(same.all()), float((gl - lse[:rows]).abs().nan_to_num().max())


def attend(s, **kw):
    from quantexperiments_amd.kernels import tree_attention
    lse = torch.full((s.n, s.hq), 5.0, device="cuda")
    a = {**s.device(), **kw}
    return tree_attention(**a, lse=lse), lse


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("d", [8, 64, 72, 96, 128, 136, 256])
@pytest.mark.parametrize("lens,news,hq,hk,page,tree", [
    ([0], [1], 1, 1, 16, False), ([1], [1], 7, 1, 16, False), ([30, 31, 32, 33], [1, 1, 1, 1], 4, 2, 16, False), ([200], [1], 14, 2, 1, False),
    ([130, 0, 65], [3, 0, 17], 6, 3, 24, True), ([40], [70], 2, 1, 64, True), ([5, 300], [40, 2], 5, 1, 100, False)])
def test_matches_the_formula(lens, news, hq, hk, page, tree, d, dtype):
    s = Setup(lens, news, hq, hk, d, page, dtype, tree, seed=d + len(lens))
    s.check(*attend(s))


@pytest.mark.parametrize("page", [1, 2, 3, 5, 16, 31, 32, 33, 64, 1000])
def test_pages_of_any_size(page):
    s = Setup([77, 255, 256, 1], [1, 5, 2, 9], 4, 2, 128, page, tree=True, seed=page)
    s.check(*attend(s))


@pytest.mark.parametrize("length", [15, 127, 128, 129, 1023, 2500, 9001])
@pytest.mark.parametrize("hq,hk,new", [(7, 1, 1), (2, 2, 4), (16, 1, 9)])
def test_long_caches_cut_into_parts_and_joined(length, hq, hk, new):
    s = Setup([length], [new], hq, hk, 128, 16, "f16", tree=new > 1, seed=length)
    s.check(*attend(s))
    s = Setup([length, 3], [new, 1], hq, hk, 64, 8, "bf16", tree=new > 1, seed=length + 1)
    s.check(*attend(s))


@pytest.mark.parametrize("lens,news", [([0], [300]), ([100, 7], [150, 129]), ([33], [257])])
@pytest.mark.parametrize("d,hq,hk", [(128, 7, 1), (64, 3, 3), (256, 4, 2)])
def test_chunks_of_a_prompt(lens, news, d, hq, hk):
    s = Setup(lens, news, hq, hk, d, 16, seed=d)
    s.check(*attend(s))


def test_trees_wider_than_words_and_masks_that_leave_a_row_nothing():
    s = Setup([0, 10, 0], [65, 130, 3], 4, 2, 128, 16, tree=True, seed=5)
    s.sees[0][3] = False
    s.sees[0][64] = False
    s.sees[1][7] = False                                     # (still sees the cached ones)
    s.sees[2][:] = False
    out, lse = attend(s)
    s.check(out, lse)
    assert bool((out[3] == 0).all()) and bool((lse[3] == -math.inf).all()) and bool((out[-3:] == 0).all())
    s.sees = [t[:, :64].clone() for t in s.sees]             # a mask of one word: new tokens beyond it are seen by nobody
    s.sees = [torch.cat((t, torch.zeros(len(t), max(0, n - t.shape[1]), dtype=torch.bool)), 1) for t, n in zip(s.sees, s.news)]
    m = s.mask()[:, :1]
    s.check(*attend(s, mask=m))
    s.check(*attend(s, mask=s.mask()))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_what_a_token_does_not_see_does_not_touch_it(value, dtype):
    s = Setup([37, 0], [6, 40], 4, 2, 128, 16, dtype, tree=True, seed=9)
    clean, clean_lse = attend(s)
    s.check(clean, clean_lse)
    # new token 2 of either sequence holds what is not finite; some see it, others do not
    s.sees[0][4, 2], s.sees[0][5, 2] = True, False
    s.sees[1][:, 2] = False
    s.sees[1][30, 2] = True
    clean, clean_lse = attend(s)
    for b, (l, where) in enumerate(((37, "k"), (0, "v"))):
        (s.k if where == "k" else s.v)[b][l + 2, 1, 5] = value
    s.put()
    out, lse = attend(s)
    blind = torch.ones(s.n, dtype=torch.bool)
    for b in range(2):
        blind[s.starts[b]:s.starts[b + 1]] = ~s.sees[b][:, 2]
    assert torch.equal(out[blind.cuda()], clean[blind.cuda()]) and torch.equal(lse[blind.cuda()], clean_lse[blind.cuda()])
    saw = s.starts[1] + 30                                   # a value: its element of the heads that read it, nothing else
    row = out[saw].cpu()
    assert torch.equal(row[:2], clean[saw].cpu()[:2]) and torch.equal(row[2:, :5], clean[saw].cpu()[2:, :5]) and torch.equal(row[2:, 6:], clean[saw].cpu()[2:, 6:])
    bad = row[2:, 5]
    assert bool(bad.isnan().all() if math.isnan(value) else (bad == value).all())
    assert torch.equal(lse[saw], clean_lse[saw])


def test_scores_at_the_ends_of_the_range():
    s = Setup([64], [1], 2, 1, 64, 16, "f16", seed=4)
    s.k[0][:] = 0
    s.k[0][5, 0, 0] = 60000.0
    s.q[0, 0], s.q[0, 1] = 0, 0
    s.q[0, 0, 0], s.q[0, 1, 0] = 60000.0, -60000.0           # one key has everything; it has nothing and the others share alike
    s.put()
    s.scale = 1.0
    out, lse = attend(s)
    assert torch.equal(out[0, 0].cpu(), s.v[0][5, 0]) and abs(float(lse[0, 0]) - 3.6e9) <= 4 * H * 3.6e9      # (four factors and products of 32 bits)
    rest = torch.cat((s.v[0][:5, 0], s.v[0][6:, 0])).double()
    assert float((out[0, 1].cpu().double() - rest.mean(0)).abs().max()) <= 2 ** -11 * float(rest.abs().mean(0).max()) * 2.2
    assert abs(float(lse[0, 1]) - math.log(64)) < 1e-5
    s.k[0][:] = torch.finfo(torch.float16).min               # all scores alike, and far below zero
    s.q[0] = 1.0
    s.put()
    out, lse = attend(s)
    assert float((out[0, 0].cpu().double() - s.v[0][:, 0].double().mean(0)).abs().max()) <= 2 ** -11 * 2.2
    assert float(lse[0, 0]) == pytest.approx(-65504.0 * 64, rel=1e-6)


def test_strides_orders_and_rows_of_no_sequence():
    s = Setup([50, 0, 9], [2, 3, 4], 6, 2, 128, 16, tree=True, seed=6, extra_rows=3)
    a = s.device()
    want, want_lse = attend(s, out=torch.full(s.q.shape, 9.0, dtype=s.dt, device="cuda"))
    s.check(want, want_lse)
    assert bool((want[-3:] == 9).all()) and bool((want_lse[-3:] == 5).all())
    stacked = torch.empty(s.n, 10, 128, dtype=s.dt, device="cuda")
    stacked[:, 1:7] = a["q"]
    out = torch.full((6, s.n, 160), 9.0, dtype=s.dt, device="cuda")
    kt, vt = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (a["k_cache"], a["v_cache"]))
    both = torch.stack((a["k_cache"], a["v_cache"]), 1)      # one pool of pages, keys and values of a page side by side
    wide = torch.full((3, a["table"].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :-5] = a["table"]
    for k, v in ((kt, vt), (both[:, 0], both[:, 1]), (a["k_cache"], vt)):
        o = out.transpose(0, 1)[..., 16:144]
        o.fill_(9.0)
        got, lse = attend(s, q=stacked[:, 1:7], k_cache=k, v_cache=v, out=o, table=wide[:, :-5])
        assert got is o and torch.equal(o, want) and torch.equal(lse, want_lse)
    assert bool((out[..., :16] == 9).all()) and bool((out[..., 144:] == 9).all())
    flipped = a["k_cache"].flip(0).contiguous().flip(0), a["v_cache"]
    got, _ = attend(s, k_cache=flipped[0], out=torch.full(s.q.shape, 9.0, dtype=s.dt, device="cuda"))
    assert torch.equal(got, want)


def test_as_many_new_tokens_each_and_bounds_that_are_too_large():
    s = Setup([100, 20, 3], [2, 2, 2], 4, 2, 64, 16, seed=8)
    want, lse = attend(s)
    s.check(want, lse)
    got, _ = attend(s, starts=None)
    assert torch.equal(got, want)
    got, _ = attend(s, starts=None, most_new=None)
    assert torch.equal(got, want)
    s.check(*attend(s, most_new=None))                       # (as many as there are rows: another cut)
    got, _ = attend(s, most_new=1, out=torch.full(s.q.shape, 9.0, dtype=s.dt, device="cuda"))
    assert bool((got[1::2] == 9).all())                      # new tokens beyond the bound are left


def test_a_contiguous_cache_is_a_page_per_sequence():
    from quantexperiments_amd.kernels import tree_attention
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(3, 200, 2, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn(3, 14, 128, generator=g).to(torch.bfloat16).cuda()
    lens = torch.tensor([199, 0, 100], dtype=torch.int32).cuda()
    out = tree_attention(q, k, v, torch.arange(3, dtype=torch.int32).cuda()[:, None], lens)
    for b in range(3):
        n = int(lens[b]) + 1
        qq, kk, vv = q[b].double().cpu(), *(c[b, :n].double().cpu().repeat_interleave(7, 1) for c in (k, v))
        p = torch.softmax(torch.einsum("hd,lhd->hl", qq, kk) * 128 ** -0.5, -1)
        ref, big = torch.einsum("hl,lhd->hd", p, vv), torch.einsum("hl,lhd->hd", p, vv.abs())
        ds = 132 * H * 128 ** -0.5 * float(torch.einsum("hd,lhd->hl", qq.abs(), kk.abs()).max())
        assert bool(((out[b].double().cpu() - ref).abs() <= (2 ** -9 * 1.01 * 2 + 2 * ds + (n + 64) * H) * big + 2 ** -9 * 2 * ref.abs()).all())


def test_wrong_tables_give_nan_for_their_sequence_alone():
    s = Setup([100, 40, 60], [2, 2, 2], 4, 2, 128, 16, seed=3)
    want, _ = attend(s)
    for bad in (10 ** 6, -1, s.kc.shape[0]):
        t = s.table.clone()
        t[1, 1] = bad
        out, lse = attend(s, table=t.cuda())
        assert bool(out[2:4].isnan().all()) and bool(lse[2:4].isnan().all())
        assert torch.equal(out[:2], want[:2]) and torch.equal(out[4:], want[4:])
    out, _ = attend(s, lens=torch.tensor([100, 10 ** 6, 60], dtype=torch.int32).cuda(), table=s.table.clamp(min=0).cuda())   # more tokens than the table has slots
    assert bool(out[2:4].isnan().all()) and torch.equal(out[:2], want[:2]) and torch.equal(out[4:], want[4:])
    wild = torch.tensor([0, 2, 2 ** 31 - 1, -5], dtype=torch.int32).cuda()      # starts that leave the rows are cut off
    out, _ = attend(s, starts=wild, most_new=2)
    assert torch.equal(out[:2], want[:2])


def test_offsets_beyond_32_bits():
    from quantexperiments_amd.kernels import tree_attention
    pages, page, hk, d = 3, 64, 2, 64
    big = torch.empty(2, (1 << 31) + (1 << 21), dtype=torch.float16, device="cuda")       # pages 2^30 elements apart: offsets of 4 GiB
    k, v = (t.as_strided((pages, page, hk, d), (1 << 30, hk * d, d, 1), t.storage_offset()) for t in big)
    g = torch.Generator().manual_seed(1)
    kh, vh = (torch.randn(pages, page, hk, d, generator=g).half() for _ in range(2))
    k.copy_(kh)
    v.copy_(vh)
    q = torch.randn(1, 4, d, generator=g).half().cuda()
    table, lens = torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda(), torch.tensor([170], dtype=torch.int32).cuda()
    got = tree_attention(q, k, v, table, lens)
    want = tree_attention(q, kh.cuda(), vh.cuda(), table, lens)
    assert torch.equal(got, want)
    far_k, far_v = (t.as_strided((2, 3, hk, d), (1 << 20, 1 << 30, d, 1), t.storage_offset()) for t in big)      # slots that far apart
    far_k.copy_(kh[:2, :3])
    far_v.copy_(vh[:2, :3])
    lens = torch.tensor([4], dtype=torch.int32).cuda()
    table = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    assert torch.equal(tree_attention(q, far_k, far_v, table, lens), tree_attention(q, kh[:2, :3].contiguous().cuda(), vh[:2, :3].contiguous().cuda(), table, lens))


def test_the_same_bits_every_time_and_on_two_streams_at_once():
    from quantexperiments_amd.kernels import tree_attention
    s = Setup([3000], [4], 28, 4, 128, 16, tree=True, seed=1)
    t = Setup([2000, 100], [4, 1], 28, 4, 128, 16, tree=True, seed=2)
    a, b = s.device(), t.device()
    want = tree_attention(**a), tree_attention(**b)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, args in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(tree_attention(**args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(got, want) for o in os)


def test_captured_twice_and_replayed_with_other_lengths():
    from quantexperiments_amd.kernels import tree_attention
    s = Setup([900, 30], [3, 1], 8, 2, 128, 16, tree=True, seed=3)
    a = s.device()
    outs = [torch.zeros_like(a["q"]) for _ in range(2)]
    tree_attention(**a)
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            tree_attention(**a, out=o)
        graphs.append(g)
    side = torch.cuda.Stream()
    for lens in ([900, 30], [5, 0], [899, 29], [0, 0]):
        a["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        a["q"].mul_(-1)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        want = tree_attention(**a)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_a_drafted_step_equals_the_tokens_decoded_one_by_one():
    """q|k|v heads of a draft tree through norm, rotation, cache, attention and the kept path; then the accepted tokens again, one at a time."""
    from quantexperiments_amd.kernels import keep_drafted, qk_norm_rotary, rotary_freqs, tree_attention
    hq, hk, d, page, n, layers = 8, 2, 64, 16, 6, 2
    g = torch.Generator().manual_seed(11)
    dt = torch.float16
    lens0 = [37, 5]
    table = torch.tensor([[0, 3, 1, 6], [2, 7, 4, 5]], dtype=torch.int32).cuda()
    freqs, scale = rotary_freqs(d, 10000.0, {"type": "yarn", "factor": 4.0, "original": 4096})
    qw, kw = ((torch.rand(d, generator=g) + 0.5).to(dt).cuda() for _ in range(2))
    caches = [torch.zeros(layers, 8, page, hk, d, dtype=dt, device="cuda") for _ in range(2)]
    past = torch.randn(layers, 2, max(lens0), hq + 2 * hk, d, generator=g).to(dt).cuda()
    parents = [-1, 0, 0, 1, 2, 4]                            # accepted: 0, 2, 4, 5
    sees = torch.eye(n, dtype=torch.bool)
    depth = []
    for t, p in enumerate(parents):
        depth.append(0 if p < 0 else depth[p] + 1)
        if p >= 0:
            sees[t] |= sees[p]
    mask = words_of(sees).repeat(2, 1).cuda()
    draft = torch.randn(layers, 2, n, hq + 2 * hk, d, generator=g).to(dt).cuda()
    slot = lambda b, s: int(table[b, s // page]) * page + s % page

    def step(layer, y, b_of, pos, at, kc, vc):
        slots = torch.tensor([slot(b, s) for b, s in zip(b_of, at)]).cuda()
        return qk_norm_rotary(y[:, :hq], y[:, hq:hq + hk], torch.tensor(pos).cuda(), freqs, qw, kw, v=y[:, hq + hk:], k_cache=kc[layer], v_cache=vc[layer], slots=slots, scale=scale)[0]

    for layer in range(layers):
        for b, l in enumerate(lens0):
            step(layer, past[layer, b, :l], [b] * l, list(range(l)), list(range(l)), *caches)
    one_by_one = [c.clone() for c in caches]
    lens = torch.tensor(lens0, dtype=torch.int32).cuda()
    outs = []
    for layer in range(layers):
        b_of = [0] * n + [1] * n
        q = step(layer, draft[layer].reshape(2 * n, -1, d), b_of, [lens0[b] + depth[i % n] for i, b in enumerate(b_of)], [lens0[b] + i % n for i, b in enumerate(b_of)], *caches)
        outs.append(tree_attention(q, caches[0][layer], caches[1][layer], table, lens, mask=mask).view(2, n, hq, d))
    path = torch.tensor([[0, 2, 4, 5]] * 2, dtype=torch.int32).cuda()
    counts = torch.tensor([4, 3], dtype=torch.int32).cuda()
    keep_drafted(*caches, table, lens, path, counts)
    lens += counts
    for b in range(2):
        for i, t in enumerate((0, 2, 4, 5)[:int(counts[b])]):
            for layer in range(layers):
                q = step(layer, draft[layer, b, t:t + 1], [b], [lens0[b] + i], [lens0[b] + i], *one_by_one)
                o = tree_attention(q, one_by_one[0][layer], one_by_one[1][layer], table[b:b + 1], torch.tensor([lens0[b] + i], dtype=torch.int32).cuda())
                # the same keys in another order of additions: twice the tolerance of a result, with |v| < 5 and A < 5
                assert float((o[0].double() - outs[layer][b, t].double()).abs().max()) <= 2 * (2 * 2 ** -11 * 5 + 2 * (d + 4) * H * 64 + 128 * H * 5)
        total = lens0[b] + int(counts[b])
        rows = torch.tensor([slot(b, s) for s in range(total)]).cuda()
        for c, o in zip(caches, one_by_one):
            assert torch.equal(c.view(layers, -1, hk, d)[:, rows], o.view(layers, -1, hk, d)[:, rows])


@pytest.mark.parametrize("seqs,hq,hk,new,page", [(70, 2, 1, 1, 16), (130, 3, 1, 2, 5), (3, 7, 1, 20, 16), (9, 4, 2, 1, 64), (2, 2, 2, 40, 16), (66, 1, 1, 33, 16)])
def test_sequences_of_unlike_lengths_cut_into_parts_of_one(seqs, hq, hk, new, page):
    g = torch.Generator().manual_seed(seqs)
    lens = [int(x) for x in torch.randint(0, 60, (seqs,), generator=g)]
    lens[seqs // 2], lens[0], lens[-1] = 3100, 0, 700        # one takes most of the parts, others none of their own
    news = [max(0, new - b % 3) if b != seqs // 2 else new for b in range(seqs)]
    s = Setup(lens, news, hq, hk, 64, page, tree=new > 1, seed=seqs)
    s.check(*attend(s))


def test_queries_that_barely_differ_and_rows_that_see_the_same_agree_in_every_part():
    # rows of one token with equal queries are equal bit for bit, wherever their key head's keys are cut
    s = Setup([4000, 77], [5, 1], 16, 2, 128, 16, seed=12)
    s.q[:, 1:8] = s.q[:, :1]
    s.q[:, 9:] = s.q[:, 8:9]
    out, lse = attend(s)
    assert torch.equal(out[:, 1:8], out[:, :1].expand(-1, 7, -1)) and torch.equal(lse[:, 9:], lse[:, 8:9].expand(-1, 7))
    s.check(out, lse)


@pytest.mark.parametrize("d", [8, 40, 64, 72, 80, 128, 144, 256])
@pytest.mark.parametrize("new,length", [(1, 70), (40, 33)])
def test_a_key_with_an_infinite_score_of_minus_infinity_weighs_nothing(d, new, length):
    # (a key's -inf against an element of q that is above zero, all others finite: the score is -inf and the weight zero, in heads of any width)
    s = Setup([length], [new], 2, 1, d, 16, seed=d)
    s.q = s.q.abs() + 0.0625
    for j in (0, 5, 31, 32, length - 1):
        s.k[0][j, 0, 0 if j % 2 else d - 1] = -math.inf
    s.put()
    got, lse = attend(s)
    keep = torch.tensor([j for j in range(length + new) if j not in (0, 5, 31, 32, length - 1)])
    s.k[0], s.v[0] = s.k[0][keep], s.v[0][keep]
    s.lens, s.sees = [len(keep) - new], s.sees
    s.check(got, lse)


def test_threads_with_streams_of_their_own_get_what_one_gets():
    import threading
    from quantexperiments_amd.kernels import tree_attention
    setups = [Setup([700, 30], [1, 3], 7, 1, 128, 16, seed=3), Setup([900], [40], 6, 2, 64, 16, tree=True, seed=4), Setup([400], [2], 4, 2, 256, 16, seed=5)]
    args = [s.device() for s in setups]
    alone = [tree_attention(**a) for a in args]
    torch.cuda.synchronize()
    got = [[] for _ in args]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i].append(tree_attention(**args[i]))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(args))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs, one in zip(got, alone):
        assert len(outs) == 20 and all(torch.equal(o, one) for o in outs)


FIRST = """
import torch
from quantexperiments_amd.kernels import qk_norm_rotary, tree_attention
g = torch.Generator().manual_seed(0)
q = torch.randn(40, 4, 128, generator=g).half().cuda()
kc, vc = (torch.randn(64, 16, 2, 128, generator=g).half().cuda() for _ in range(2))
i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
table, lens = torch.arange(64, dtype=torch.int32)[None].cuda(), i32([900])
pos, f = torch.arange(40).cuda(), torch.rand(64, dtype=torch.float64, generator=g).cuda()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    turned, _ = qk_norm_rotary(q, q[:, :2], pos, f)
    out = tree_attention(turned, kc, vc, table, lens)
for n in (900, 17):
    lens.fill_(n)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, tree_attention(qk_norm_rotary(q, q[:, :2], pos, f)[0], kc, vc, table, lens))
print("captured first")
"""


def test_a_process_whose_first_calls_are_captured():
    import pathlib
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=pathlib.Path(__file__).parents[1], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("d,hq,new,length", [(64, 4, 1, 600), (64, 4, 20, 600), (128, 7, 40, 700), (256, 4, 20, 500)])
def test_scores_a_rounding_step_apart_where_steps_are_large(d, hq, new, length, dtype):
    """Scores of 2^27 and, behind them, of the next larger number of 32 bits, 16 above: weights of 2^16 beside the first ones', which fp16 cannot hold.

    Scores and their product with scale * log2 e = 1 are exact, so the first ones' weights are 2^-16 of the others', exactly in either type: only the sums' additions and the
    result's rounding are left (and the total's of rounded weights, which are exact)."""
    s = Setup([length], [new], hq, 1, d, 16, dtype, seed=d + new)
    s.q[:] = 0
    s.q[..., 0], s.q[..., 1] = 2.0 ** 14, 4.0
    k = s.k[0]
    k[:] = 0
    k[..., 0] = 2.0 ** 13
    larger = torch.arange(len(k)) % 128 >= 64                # (in whole steps of keys, behind smaller ones in one walk over them)
    k[larger, :, 1] = 4.0
    s.v[0] = (s.v[0].abs() + 1).to(s.dt)
    s.put()
    a, many = s.device(), 300                                # (so many sequences with the same pages that none is cut into parts)
    lse = torch.empty(many * new, hq, device="cuda")
    from quantexperiments_amd.kernels import tree_attention
    out = tree_attention(a["q"].repeat(many, 1, 1), a["k_cache"], a["v_cache"], a["table"].repeat(many, 1), a["lens"].repeat(many), scale=math.log(2.0), lse=lse)
    out, lse = out.view(many, new, hq, d), lse.view(many, new, hq)
    assert torch.equal(out, out[:1].expand_as(out)) and torch.equal(lse, lse[:1].expand_as(lse))
    u = torch.finfo(s.dt).eps / 2
    for t in range(new):
        n = length + t + 1
        w = torch.where(larger[:n], 1.0, 2.0 ** -16).double()
        want = (w[:, None] * s.v[0][:n, 0].double()).sum(0) / w.sum()
        assert bool(((out[0, t].cpu().double() - want).abs() <= (u + (n + 64) * H) * 1.01 * want).all())
        top = (2.0 ** 27 + 16) * math.log(2.0)
        assert bool(((lse[0, t].cpu().double() - top - math.log(float(w.sum()))).abs() <= 4 * H * top).all())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("above", [9, 14, 17, 20])
@pytest.mark.parametrize("d,hq,hk,news,length", [(64, 4, 1, [1], 900), (128, 6, 2, [3, 1], 1000), (256, 4, 1, [2], 700), (64, 4, 1, [20], 900), (128, 7, 1, [40], 700), (256, 2, 1, [70], 500),
                                                 (96, 7, 1, [40, 3], 400)])
def test_weights_far_below_the_largest(d, hq, hk, news, length, above, dtype):
    """Keys in every 64 slots whose scores are `above` higher than the others' mean and whose values are zero, so that the result is what the others' weights leave.

    A weight of fp16 is held times 2^7 beside a reference that is at most the row's largest score: with u relative where that is 2^-14 or more, with half a step of 2^-24 below.
    So it is off by u of itself or by 2^-25 / 2^7 of the largest weight, and a result by up to 2^-32 sum |v| / sum exp(s - max) more than by the others' bound."""
    s = Setup([length] * len(news), news, hq, hk, d, 16, dtype, tree=news[0] > 1, seed=above + d, scale=1.0)
    s.q[..., 0] = 8.0
    for b in range(len(news)):
        s.k[b][..., 0] = 0
        s.k[b][::64] = 0
        s.k[b][::64, :, 0] = above * d ** 0.5 / 8
        s.v[b] = (4000 * (0.5 + torch.rand(s.v[b].shape, generator=s.g))).to(s.dt)
        s.v[b][::64] = 0
    s.put()
    got, got_lse = attend(s)
    out, tol, lse, ltol = s.reference()
    if dtype == "f16":
        for b, (k, v) in enumerate(zip(s.k, s.v)):
            tol[s.starts[b]:s.starts[b + 1]] += 2.0 ** -32 * float(v.double().abs().sum(0).max()) / len(k[:length:64])
    off, off_lse = (got.cpu().double() - out).abs(), (got_lse.cpu().double() - lse).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    assert bool((off_lse <= ltol).all()), float((off_lse / ltol).max())


def test_a_mask_without_words_shows_the_cached_tokens_alone():
    s = Setup([40, 0, 5], [3, 1, 50], 4, 2, 64, 16, tree=True, seed=14)
    s.sees = [torch.zeros_like(t) for t in s.sees]
    zeros, zeros_lse = attend(s, mask=torch.zeros(s.n, 1, dtype=torch.int64, device="cuda"))
    s.check(zeros, zeros_lse)
    out, lse = attend(s, mask=torch.empty(s.n, 0, dtype=torch.int64, device="cuda"))
    assert torch.equal(out, zeros) and torch.equal(lse, zeros_lse)
    strided = torch.zeros(s.n, 4, dtype=torch.int64, device="cuda")[:, 2:2]
    out, lse = attend(s, mask=strided)
    assert torch.equal(out, zeros) and torch.equal(lse, zeros_lse)


def test_a_mask_without_words_through_the_call_path_in_python(monkeypatch):
    from quantexperiments_amd import _lib

    class NotCovered:
        def __getattr__(self, name):
            return lambda *args: 1

    monkeypatch.setattr(_lib, "native", lambda: NotCovered())
    test_a_mask_without_words_shows_the_cached_tokens_alone()


def test_tensors_with_a_tangent_are_refused():
    """Forward mode: a dual tensor asks for no gradient, and what is computed from its values alone would have a derivative of zero."""
    from torch.autograd import forward_ad
    from quantexperiments_amd.kernels import keep_drafted, qk_norm_rotary, rotary, tree_attention
    s = Setup([20], [2], 4, 2, 64, 16, seed=15)
    a = {**s.device(), "mask": None}
    pos, f = torch.arange(2).cuda(), torch.ones(32, dtype=torch.float64).cuda()
    x, k, w = a["q"], a["q"][:, :2], torch.ones(64, dtype=s.dt).cuda()
    cache, slots = dict(v=k, k_cache=a["k_cache"], v_cache=a["v_cache"]), torch.arange(2).cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: rotary(dual(x), pos, f), lambda: rotary(x, pos, dual(f)), lambda: rotary(x, pos, f, dual(torch.empty_like(x))),
                 lambda: qk_norm_rotary(dual(x), k, pos, f), lambda: qk_norm_rotary(x, dual(k), pos, f), lambda: qk_norm_rotary(x, k, pos, dual(f)),
                 lambda: qk_norm_rotary(x, k, pos, f, dual(w), w), lambda: qk_norm_rotary(x, k, pos, f, w, dual(w)), lambda: keep_drafted(dual(a["k_cache"]), a["v_cache"], a["table"], a["lens"], i32([[0]]), i32([1])),
                 lambda: keep_drafted(a["k_cache"], dual(a["v_cache"]), a["table"], a["lens"], i32([[0]]), i32([1]))]
        calls += [lambda n=n: qk_norm_rotary(x, k, pos, f, slots=slots, **{**cache, n: dual(cache[n])}) for n in cache]
        calls += [lambda n=n: tree_attention(**{**a, n: dual(a[n])}) for n in ("q", "k_cache", "v_cache")]
        calls += [lambda: tree_attention(**a, out=dual(torch.empty_like(x)))]
        for grad in (True, False):                           # (tangents are carried under no_grad too)
            for i, call in enumerate(calls):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    call()
                    print("not refused:", i)
        s.check(tree_attention(**a))


def test_scales_at_the_ends_of_the_range():
    from quantexperiments_amd.kernels import tree_attention
    s = Setup([40], [1], 2, 1, 64, 16, seed=16)
    for scale in (2.4e38, 3.4e38, math.inf, 0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="scale"):
            tree_attention(**{**s.device(), "scale": scale})
    s.q[:] = 0                                               # scores of zero, whatever the scale: the mean of all values
    for s.scale in (2.2e38, 1e-30):
        s.check(*attend(s))


@pytest.mark.parametrize("d,hq,hk,new,seqs,length,page,tree,dtype", [
    # eight waves of 32 rows (16 of heads of 256), a workgroup per sequence, key head and block of rows
    (128, 9, 3, 80, 100, 700, 8, True, "f16"), (128, 9, 3, 80, 100, 640, 24, False, "bf16"), (64, 9, 3, 80, 100, 1100, 8, False, "bf16"), (64, 9, 3, 80, 100, 700, 7, True, "f16"),
    (96, 9, 3, 80, 100, 700, 16, True, "bf16"), (256, 6, 3, 64, 100, 420, 16, True, "bf16"), (256, 6, 3, 64, 100, 420, 5, False, "f16"), (128, 6, 2, 90, 100, 640, 1, True, "bf16"),
    # four waves
    (128, 9, 3, 40, 100, 420, 16, True, "bf16"), (256, 6, 3, 32, 100, 420, 16, False, "f16"), (96, 9, 3, 40, 100, 420, 9, False, "f16"), (64, 9, 3, 40, 100, 420, 16, True, "bf16"),
    # several blocks of rows, which see unlike numbers of keys; sequences cut into parts of several rounds each
    (128, 7, 1, 300, 40, 900, 16, False, "bf16"), (128, 28, 4, 48, 8, 2500, 16, True, "f16")])
def test_rings_that_are_filled_again_and_again(d, hq, hk, new, seqs, length, page, tree, dtype):
    """Workgroups that walk through many stages of keys, so that every place in LDS is filled, read and filled again; lengths that differ by some keys, so that the last
    stages do too; tables of more than 64 pages among them, so that a wave fetches entries again.  Checked: some rows of some sequences."""
    g = torch.Generator().manual_seed(d + new + page)
    lens = [length - int(x) for x in torch.randint(0, 40, (seqs,), generator=g)]
    news = [new - b % 3 for b in range(seqs)]
    s = Setup(lens, news, hq, hk, d, page, dtype, tree, seed=d + new)
    got, lse = attend(s)
    again, lse2 = attend(s)
    assert torch.equal(got, again) and torch.equal(lse, lse2) and bool(got.isfinite().all())
    u = torch.finfo(s.dt).eps / 2
    for b in (0, 1, seqs // 2, seqs - 1):
        l, n = lens[b], news[b]
        k, v = s.k[b].double(), s.v[b].double()
        for t in sorted({0, 1, n // 2, n - 2, n - 1}):
            see = torch.cat((torch.ones(l, dtype=torch.bool), s.sees[b][t]))
            r = s.starts[b] + t
            for h in range(hq):
                kk, vv, q = k[see, h // (hq // hk)], v[see, h // (hq // hk)], s.q[r, h].double()
                sc = kk @ q * s.scale
                ds = (d + 4) * H * s.scale * float((kk.abs() @ q.abs()).max())
                p = torch.softmax(sc, 0)
                out, big, top = p @ vv, p @ vv.abs(), torch.logsumexp(sc, 0)
                tol = (u * 1.01 + 2 * ds + (len(sc) + 64) * H) * big + u * out.abs() + torch.finfo(s.dt).tiny * torch.finfo(s.dt).eps
                assert bool(((got[r, h].cpu().double() - out).abs() <= tol).all()), (b, t, h)
                assert abs(float(lse[r, h]) - float(top)) <= ds + (len(sc) + 64) * H + 4 * H * max(1.0, abs(float(top)), abs(float(sc.max()))), (b, t, h)
