"""Sequences forked and pools compacted: tables, lengths and every byte of the pools against their definition."""

import pytest
import torch

from tests.cache8_model import table_for

pytestmark = pytest.mark.gpu
i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
KINDS = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.uint8}


def pool(layers, pages, page, heads, dim, kind, g, blocks=0):
    """[k, v] or [k, v, k_scale, v_scale] on the CPU, bytes for the 8-bit types."""
    dt = KINDS[kind]
    out = [torch.randint(0, 255, (layers, pages, page, heads, dim), generator=g).to(dt) for _ in range(2)]
    return out + [torch.randint(0, 255, (layers, pages, blocks, heads), generator=g, dtype=torch.uint8) for _ in range(2 if blocks else 0)]


def device(cache, one=False):
    out = [t.cuda().clone() for t in cache]
    out = [t.view(torch.float8_e4m3fn) if t.dtype == torch.uint8 and i < 2 else t.view(torch.float8_e8m0fnu) if i > 1 else t for i, t in enumerate(out)]
    return [t[0] for t in out] if one else out


def assert_same(got, want):
    for i, (a, b) in enumerate(zip(got, want)):
        a = a.cpu()
        a = a.view(torch.uint8) if a.element_size() == 1 else a
        b = b[0] if a.dim() < b.dim() else b
        assert torch.equal(a, b), (i, (a != b).nonzero()[:3])


def scales(cache):
    return dict(zip(("k_scale", "v_scale"), cache[2:]))


def forked(cache, table, lens, parent, fresh, page):
    """What fork_pages leaves, and returns: (caches, table, lens)."""
    cache = [t.clone() for t in cache]
    pages, width = cache[0].shape[1], table.shape[1]
    rows, sizes = [], []
    for p, f in zip(parent, fresh):
        if not 0 <= p < len(lens):
            rows.append([-1] * width)
            sizes.append(0)
            continue
        whole, rest = divmod(max(lens[p], 0), page)
        row = table[p].tolist()
        if f >= 0:
            if f < pages and rest and whole < width and 0 <= row[whole] < pages:
                for t in cache:
                    n = -(-rest * t.shape[2] // page)
                    t[:, f, :n] = t[:, row[whole], :n]
            row = (row[:whole] + [f] + [-1] * width)[:width]
        rows.append(row)
        sizes.append(lens[p])
    return cache, torch.tensor(rows, dtype=torch.int32).reshape(len(parent), width), torch.tensor(sizes, dtype=torch.int32)


@pytest.mark.parametrize("kind,heads,dim,blocks", [("bf16", 4, 128, 0), ("bf16", 3, 5, 0), ("f32", 2, 3, 0), ("e4m3", 4, 128, 1), ("e4m3", 3, 5, 2), ("e4m3", 1, 16, 3)])
@pytest.mark.parametrize("layers", [0, 1, 5])
def test_fork_matches_its_definition(kind, heads, dim, blocks, layers):
    from quantexperiments_amd.kernels import fork_pages
    g = torch.Generator().manual_seed(dim + layers)
    page, lens = 12 if not blocks else 48, [0, 1, 12, 13, 47, 48, 49, 100]
    table, pages, spare = table_for(lens, page, g, spare=12)
    cache = pool(max(layers, 1), pages, page, heads, dim, kind, g, blocks)
    parent = [7, 7, 7, 0, 1, 2, 3, 4, 5, 6, 4, 0]
    fresh = spare.tolist()
    fresh[0] = fresh[8] = -1
    dev = device(cache, layers == 0)
    t, n = fork_pages(*dev[:2], table.cuda(), i32(lens), i32(parent), i32(fresh), **scales(dev))
    want, wt, wn = forked(cache, table, lens, parent, fresh, page)
    assert torch.equal(t.cpu(), wt) and torch.equal(n.cpu(), wn)
    assert_same(dev, want)


def test_fork_of_what_is_not_there():
    """Parents outside the batch, pages outside the cache, lengths beyond the table, below zero; into memory given."""
    from quantexperiments_amd.kernels import fork_pages
    g = torch.Generator().manual_seed(3)
    lens = [20, 40, -5, 1000, 7]
    table, pages, spare = table_for([20, 40, 1, 40, 7], 16, g, spare=8)
    table[1, 2] = pages
    cache = pool(2, pages, 16, 2, 8, "bf16", g)
    parent = [-1, 5, 0, 0, 1, 2, 3, 4, 2 ** 31 - 1]
    s = spare.tolist()
    fresh = [s[0], s[1], pages, 2 ** 31 - 1, s[2], s[3], s[4], s[5], -5]
    dev = device(cache)
    big = torch.full((9, 20), 77, dtype=torch.int32, device="cuda")
    out, sizes = big[:, 3:3 + table.shape[1]], torch.empty(9, dtype=torch.int32, device="cuda")
    t, n = fork_pages(*dev[:2], table.cuda(), i32(lens), i32(parent), i32(fresh), out_table=out, out_lens=sizes)
    assert t is out and n is sizes
    want, wt, wn = forked(cache, table, lens, parent, fresh, 16)
    assert torch.equal(t.cpu(), wt) and torch.equal(n.cpu(), wn)
    assert_same(dev, want)
    assert bool((big[:, :3] == 77).all()) and bool((big[:, 3 + table.shape[1]:] == 77).all())


def compacted(cache, table, lens, page):
    cache = [t.clone() for t in cache]
    pages = cache[0].shape[1]
    kept = [min(-(-max(l, 0) // page), table.shape[1]) for l in lens]
    used = sorted({int(table[b, j]) for b, m in enumerate(kept) for j in range(m) if 0 <= int(table[b, j]) < pages})
    n = len(used)
    holes = sorted(set(range(n)) - set(used))
    to = dict(zip([p for p in used if p >= n], holes))
    for p, h in to.items():
        for t in cache:
            t[:, h] = t[:, p]
    new = [[to.get(int(x), int(x)) if j < kept[b] else -1 for j, x in enumerate(row)] for b, row in enumerate(table)]
    return cache, torch.tensor(new, dtype=torch.int32).reshape(table.shape), n


@pytest.mark.parametrize("kind,heads,dim,blocks", [("bf16", 4, 64, 0), ("f32", 1, 3, 0), ("e4m3", 3, 5, 2), ("e4m3", 4, 128, 1)])
@pytest.mark.parametrize("lens,spare", [([1], 0), ([0, 0], 5), ([5, 17, 48, 0, 33], 0), ([5, 17, 48, 0, 33], 9), ([300, 2, 511], 100), ([16] * 40, 7)])
def test_compact_matches_its_definition(lens, spare, kind, heads, dim, blocks):
    from quantexperiments_amd.kernels import compact_pages
    g = torch.Generator().manual_seed(dim + len(lens))
    table, pages, _ = table_for([max(l, 1) for l in lens], 16, g, spare)
    cache = pool(3, pages, 16, heads, dim, kind, g, 1 if blocks else 0)
    dev = device(cache)
    t, used = compact_pages(*dev[:2], table.cuda(), i32(lens), **scales(dev))
    want, wt, n = compacted(cache, table, lens, 16)
    assert torch.equal(t.cpu(), wt) and used.tolist() == [n]
    assert_same(dev, want)
    again, used = compact_pages(*dev[:2], t, i32(lens), **scales(dev))          # nothing is left to do
    assert torch.equal(again.cpu(), wt) and used.tolist() == [n]
    assert_same(dev, want)


def test_compact_shared_bad_and_many_pages():
    from quantexperiments_amd.kernels import compact_pages
    g = torch.Generator().manual_seed(9)
    for pages, seqs, width in ((2 ** 20, 20, 900), (70000, 30, 700), (33, 3, 9), (1, 1, 1), (32, 2, 16), (64, 70, 2)):
        table = torch.randint(-2, pages + 2, (seqs, width), generator=g, dtype=torch.int32)           # (some shared, some outside)
        lens = torch.randint(-3, width * 2 + 4, (seqs,), generator=g).tolist()                         # (some longer than their rows)
        cache = pool(1, pages, 2, 1, 4, "bf16", g)
        dev = device(cache, True)
        t, used = compact_pages(*dev, table.cuda(), i32(lens))
        want, wt, n = compacted(cache, table, lens, 2)
        assert torch.equal(t.cpu(), wt) and used.tolist() == [n]
        assert_same(dev, want)


def test_strided_caches():
    """Heads before slots in a page, layers inside pages, and elements between the heads that are not theirs."""
    from quantexperiments_amd.kernels import compact_pages, fork_pages
    g = torch.Generator().manual_seed(10)
    lens = [33, 5, 20]
    table, pages, spare = table_for(lens, 16, g, spare=6)
    wide = [torch.randint(0, 99, (pages, 2, 3, 16, 24), generator=g).half().cuda() for _ in range(2)]              # [pages, layers, heads, slots, ..]
    view = lambda w: w[..., 4:20].permute(1, 0, 3, 2, 4)
    cache = [view(w).cpu().clone() for w in wide]
    rest = [w.clone() for w in wide]
    parent, fresh = [0, 0, 1, 2], spare[:4].tolist()
    t, n = fork_pages(view(wide[0]), view(wide[1]), table.cuda(), i32(lens), i32(parent), i32(fresh))
    want, wt, wn = forked(cache, table, lens, parent, fresh, 16)
    assert torch.equal(t.cpu(), wt) and torch.equal(n.cpu(), wn)
    assert_same([view(w) for w in wide], want)
    t2, used = compact_pages(view(wide[0]), view(wide[1]), t, n)
    want, wt, k = compacted(want, wt, wn.tolist(), 16)
    assert torch.equal(t2.cpu(), wt) and used.tolist() == [k]
    assert_same([view(w) for w in wide], want)
    for w, r in zip(wide, rest):
        assert torch.equal(w[..., :4], r[..., :4]) and torch.equal(w[..., 20:], r[..., 20:])


def test_captured_and_replayed():
    from quantexperiments_amd.kernels import compact_pages, fork_pages
    g = torch.Generator().manual_seed(11)
    lens = [33, 5, 20]
    table, pages, spare = table_for(lens, 16, g, spare=6)
    cache = pool(2, pages, 16, 2, 32, "bf16", g)
    dev, td, ld, parent, fresh = device(cache), table.cuda(), i32(lens), i32([0, 0, 1]), i32(spare[:3].tolist())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        t, n = fork_pages(*dev, td, ld, parent, fresh)
        t2, used = compact_pages(*dev, t, n)
    for who in ([0, 0, 1], [2, 1, 1], [1, 2, 0]):
        for d, c in zip(dev, cache):
            d.copy_(c)
        parent.copy_(torch.tensor(who, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want, wt, wn = forked(cache, table, lens, who, spare[:3].tolist(), 16)
        assert torch.equal(t.cpu(), wt) and torch.equal(n.cpu(), wn)
        want, wt, k = compacted(want, wt, wn.tolist(), 16)
        assert torch.equal(t2.cpu(), wt) and used.tolist() == [k]
        assert_same(dev, want)


def test_two_streams_at_once():
    """Workspaces are the calls' own."""
    from quantexperiments_amd.kernels import compact_pages
    g = torch.Generator().manual_seed(12)
    sets, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for lens in ([33, 5, 20], [200, 17, 1]):
        table, pages, _ = table_for(lens, 16, g, spare=40)
        cache = pool(2, pages, 16, 2, 32, "bf16", g)
        sets.append((lens, table, cache, device(cache), table.cuda(), i32(lens)))
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, (lens, table, cache, dev, td, ld) in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(compact_pages(*dev, td, ld))
    torch.cuda.synchronize()
    for i, (t, used) in enumerate(got):
        lens, table, cache, dev, _, _ = sets[i % 2]
        want, wt, n = compacted(cache, table, lens, 16)
        assert torch.equal(t.cpu(), wt) and used.tolist() == [n]
        assert_same(dev, want)


def test_empty_batches():
    from quantexperiments_amd.kernels import compact_pages, fork_pages
    g = torch.Generator().manual_seed(13)
    cache = pool(2, 6, 16, 2, 32, "bf16", g)
    dev = device(cache)
    none = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    t, used = compact_pages(*dev, none, i32([]))
    assert t.shape == (0, 4) and used.tolist() == [0]
    t, n = fork_pages(*dev, torch.zeros(2, 4, dtype=torch.int32, device="cuda"), i32([3, 3]), i32([]), i32([]))
    assert t.shape == (0, 4) and n.shape == (0,)
    t, n = fork_pages(*dev, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), i32([0, 3]), i32([1, 0]), i32([2, -1]))
    assert t.shape == (2, 0) and n.tolist() == [3, 0]
    t, used = compact_pages(*dev, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), i32([0, 3]))
    assert t.shape == (2, 0) and used.tolist() == [0]
    empty = [torch.empty(2, 0, 16, 2, 32, device="cuda") for _ in range(2)]
    t, used = compact_pages(*empty, torch.full((1, 2), -1, dtype=torch.int32, device="cuda"), i32([5]))
    assert t.tolist() == [[-1, -1]] and used.tolist() == [0]
    assert_same(dev, cache)


def refused(error, f, base, change):
    try:
        f(**{**base, **change})
    except error:
        return
    raise AssertionError({k: (tuple(t.shape), t.dtype, t.stride()) if isinstance(t, torch.Tensor) else t for k, t in change.items()})


def test_refusals():
    from quantexperiments_amd.kernels import compact_pages, fork_pages
    from quantexperiments_amd._lib import SqError
    k, v = (torch.zeros(6, 16, 2, 32, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(6, 1, 2, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
    table, lens, parent, pages = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), i32([4, 5]), i32([0, 1, 1]), i32([3, 4, 5])
    ok = dict(k_cache=k, v_cache=v, table=table, lens=lens)
    fork = dict(**ok, parent=parent, pages=pages)
    bad = [dict(v_cache=v[:5]), dict(v_cache=v.half()), dict(k_cache=k[0], v_cache=v[0]), dict(v_cache=k), dict(k_cache=k[:1].expand_as(k)), dict(k_cache=k.transpose(2, 3), v_cache=v.transpose(2, 3)),
           dict(k_scale=ks), dict(k_scale=ks[:5], v_scale=vs[:5]), dict(k_scale=ks, v_scale=ks), dict(table=table.long()), dict(table=table[0]), dict(lens=lens[:1]), dict(lens=lens.cpu()),
           dict(k_scale=ks.expand(6, 5, 2), v_scale=vs.expand(6, 5, 2))]
    for b in bad:
        for f, base in ((fork_pages, fork), (compact_pages, ok)):
            refused(ValueError, f, base, b)
    for b in (dict(parent=parent.long()), dict(pages=pages[:2]), dict(out_table=table), dict(out_lens=lens), dict(out_lens=torch.empty(3, device="cuda")), dict(out_lens=parent)):
        refused(ValueError, fork_pages, fork, b)
    with pytest.raises(ValueError, match="overlaps"):
        compact_pages(**ok, out_table=table)
    with pytest.raises(NotImplementedError):
        compact_pages(**{**ok, "k_cache": k.clone().requires_grad_()})
    with pytest.raises(SqError):                             # more pages than it keeps bits for
        few = torch.zeros(2 ** 20 + 1, 1, 1, 1, device="cuda", dtype=torch.float16)
        compact_pages(few, few.clone(), table, lens)
