"""New tokens put into an 8-bit cache, and drafts kept in it, against their definition in 64 bits: every code and scale of the whole pool has to be the same, so
nothing here has a tolerance (a code is one rounding of an exact product, ties to even)."""

import pytest
import torch

from tests.cache8_model import MOST, Pool, table_for

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()


def starts_of(news):
    s = [0]
    for n in news:
        s.append(s[-1] + n)
    return s


def tokens(n, heads, dim, dtype, g, spread=3.0):
    """k, v as columns of a stacked product, some tokens and heads much larger than others."""
    y = torch.randn(n, 3 * heads, dim, generator=g) * torch.exp(torch.randn(n, 3 * heads, 1, generator=g) * spread)
    y = y.clamp(-6e4, 6e4).to(DT[dtype])
    return y[:, heads:2 * heads], y[:, 2 * heads:]


def put(pool, k, v, table, lens, news, starts=None, permute=None, **kw):
    from quantexperiments_amd.kernels import put_tokens8
    dev = pool.device(permute)
    y = k._base.cuda() if k._base is not None else None
    h = k.shape[1]
    kd, vd = (y[:, h:2 * h], y[:, 2 * h:]) if y is not None else (k.cuda(), v.cuda())
    put_tokens8(kd, vd, *dev, table.cuda(), i32(lens), i32(starts or starts_of(news)), **kw)
    return dev


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dim", [16, 80, 128, 256])
@pytest.mark.parametrize("lens,news,heads,page,blocks", [
    ([0], [1], 1, 16, 1), ([5], [1], 4, 16, 1), ([15, 16, 17, 0], [1, 1, 1, 3], 3, 16, 1), ([7, 0, 40], [9, 33, 0], 2, 32, 2), ([3], [130], 2, 48, 1), ([20, 50], [77, 2], 1, 96, 3),
    ([100], [200], 1, 128, 1)])
def test_put_matches_the_definition(lens, news, heads, page, blocks, dim, dtype):
    g = torch.Generator().manual_seed(dim + page)
    table, pages, _ = table_for([a + b for a, b in zip(lens, news)], page, g)
    pool = Pool(pages, page, blocks, heads, dim, g)
    k, v = tokens(sum(news) + 2, heads, dim, dtype, g)                    # (two rows behind the last sequence)
    got = put(pool, k, v, table, lens, news, most_new=max(news))
    pool.put(k, v, table, lens, starts_of(news))
    pool.assert_same(*got)


def test_put_in_parts_is_put_at_once_where_no_scale_grows():
    from quantexperiments_amd.kernels import put_tokens8
    g = torch.Generator().manual_seed(2)
    table, pages, _ = table_for([100], 32, g)
    pool = Pool(pages, 32, 2, 2, 64, g)
    k, v = tokens(100, 2, 64, "bf16", g, spread=0.0)
    k[::16, :, 0], v[::16, :, 0] = 300.0, -300.0             # the largest element of every block comes first
    whole, parts = pool.device(), pool.device()
    kd, vd = k.cuda(), v.cuda()
    put_tokens8(kd, vd, *whole, table.cuda(), i32([0]))
    for at, n in ((0, 1), (1, 16), (17, 15), (32, 50), (82, 18)):
        put_tokens8(kd[at:at + n], vd[at:at + n], *parts, table.cuda(), i32([at]))
    for a, b in zip(whole, parts):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", list(DT))
def test_put_scales_a_block_that_grows(dtype):
    """Token by token with magnitudes up and down over forty powers of two; codes that fall below 2^-6 of the scale are rounded again."""
    from quantexperiments_amd.kernels import put_tokens8
    g = torch.Generator().manual_seed(3)
    table, pages, _ = table_for([16], 16, g)
    pool = Pool(pages, 16, 1, 2, 32, g)
    dev = pool.device()
    top = 15 if dtype == "f16" else 60
    for t in range(16):
        size = 2.0 ** float(torch.randint(-top, top, (1,), generator=g))
        k, v = ((torch.randn(1, 2, 32, generator=g) * size).to(DT[dtype]) for _ in range(2))
        put_tokens8(k.cuda(), v.cuda(), *dev, table.cuda(), i32([t]))
        pool.put(k, v, table, [t], [0, 1])
        pool.assert_same(*dev)


@pytest.mark.parametrize("dtype", list(DT))
def test_put_of_edge_values(dtype):
    dt, top = DT[dtype], MOST[DT[dtype]]
    g = torch.Generator().manual_seed(4)
    inf, nan = float("inf"), float("nan")
    tiny = torch.finfo(dt).tiny
    rows = [[0.0] * 16, [-0.0] * 16, [inf, 1.0, -2.0] + [0.5] * 13, [nan, -inf, inf] + [0.0] * 13, [nan] * 16, [448.0, 449.0, 464.0, -432.0] + [1.0] * 12,
            [1.75, -1.75, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9] + [2.0 ** -17, 3 * 2.0 ** -17, 2.0 ** -18] + [0.0] * 8, [torch.finfo(dt).max, -torch.finfo(dt).max, top] + [1.0] * 13,
            [tiny, tiny / 2, -tiny] + [0.0] * 13, [1.0625, 1.1875, -1.0625, -1.3125] + [448 * 2.0 ** -8] * 12]
    for spread in (False, True):                             # each row a block of its own, and all of them in one
        n = len(rows)
        lens, news = ([0] * n, [1] * n) if spread else ([3], [n])
        table, pages, _ = table_for([a + b for a, b in zip(lens, news)], 16, g)
        pool = Pool(pages, 16, 1, 1, 16, g)
        k = torch.tensor(rows, dtype=torch.float64).to(dt)[:, None].clone()
        v = k.flip(0).contiguous()
        got = put(pool, k, v, table, lens, news)
        pool.put(k, v, table, lens, starts_of(news))
        pool.assert_same(*got)
        held = [c.cpu().float() for c in got[:2]]
        assert all(bool((h.abs().nan_to_num(0) <= 448).all()) for h in held)


@pytest.mark.parametrize("permute", [None, (0, 2, 1, 3), (1, 0, 2, 3)])
def test_put_layouts(permute):
    """Heads before slots within a page, pages inside slots; strided sides; tokens in no particular place."""
    from quantexperiments_amd.kernels import put_tokens8
    g = torch.Generator().manual_seed(5)
    lens, news = [9, 30], [40, 3]
    table, pages, _ = table_for([a + b for a, b in zip(lens, news)], 32, g)
    pool = Pool(pages, 32, 2, 3, 48, g)
    x = torch.randn(50, 7, 64, generator=g).bfloat16()
    k, v = x[::1, 1:4, 8:56], x[:, 4:7, 16:64]
    dev = pool.device(permute)
    xd = x.cuda()
    wide = torch.empty(2, 40, dtype=torch.int32).cuda()[:, 5:5 + table.shape[1]]
    wide.copy_(table)
    put_tokens8(xd[:, 1:4, 8:56], xd[:, 4:7, 16:64], *dev, wide, i32(lens), i32([4, 44, 47]), most_new=40)
    pool.put(k, v, table, lens, [4, 44, 47])
    pool.assert_same(*dev)


@pytest.mark.parametrize("dim,n,odd", [(128, 700, False), (128, 700, True), (16, 2100, True), (256, 60, True)])
def test_put_of_large_blocks(dim, n, odd):
    """More elements in a block than a workgroup holds, and more than a wave does; some that are not finite or beyond what is held."""
    g = torch.Generator().manual_seed(dim)
    page = {16: 2048, 128: 1024, 256: 64}[dim]
    lens, news = [page // 4, 0], [n, 3]
    table, pages, _ = table_for([a + b for a, b in zip(lens, news)], page, g)
    pool = Pool(pages, page, 1, 2, dim, g)
    k, v = tokens(sum(news), 2, dim, "bf16", g)
    k, v = k.clone(), v.clone()
    if odd:
        k[n // 2, 0, 3], k[1, 1, 5], v[n - 1, 0, 0] = float("inf"), float("nan"), 3.3e38
    got = put(pool, k, v, table, lens, news)
    pool.put(k, v, table, lens, starts_of(news))
    pool.assert_same(*got)


def test_put_into_strided_scales():
    """Scales whose heads are apart, blocks inside heads; the bytes between them stay."""
    from quantexperiments_amd.kernels import put_tokens8
    g = torch.Generator().manual_seed(15)
    lens, news = [9, 30], [40, 3]
    table, pages, _ = table_for([a + b for a, b in zip(lens, news)], 32, g)
    pool = Pool(pages, 32, 2, 3, 32, g)
    kc, vc, _, _ = pool.device()
    wide = [torch.full((3, pages, 5), 9, dtype=torch.uint8, device="cuda") for _ in range(2)]              # [heads, pages, blocks ..]
    scales = [w.view(torch.float8_e8m0fnu)[..., 1:3].permute(1, 2, 0) for w in wide]
    for i, w in enumerate(wide):
        w[..., 1:3] = pool.scales[i].permute(2, 0, 1).cuda()
    k, v = tokens(43, 3, 32, "f16", g)
    put_tokens8(k.cuda(), v.cuda(), kc, vc, *scales, table.cuda(), i32(lens), i32(starts_of(news)))
    pool.put(k, v, table, lens, starts_of(news))
    pool.assert_same(kc, vc, *scales)
    assert all(bool((w[..., 0] == 9).all()) and bool((w[..., 3:] == 9).all()) for w in wide)


def test_put_leaves_what_has_no_place():
    g = torch.Generator().manual_seed(6)
    lens, news = [10, 20, 5, -3], [20, 30, 0, 4]
    table, pages, _ = table_for([30, 50, 5, 4], 16, g)
    table[0, 1] = pages                                      # outside the cache
    table[1, 2] = -1
    table = table[:, :3]                                     # (sequence 1 is longer than its row)
    pool = Pool(pages, 16, 1, 2, 32, g)
    k, v = tokens(60, 2, 32, "bf16", g)
    got = put(pool, k, v, table, lens, news, starts=[0, 20, 50, 50, 54], most_new=25)
    pool.put(k, v, table, lens, [0, 20, 50, 50, 54], 25)
    pool.assert_same(*got)


def test_put_of_no_tokens_and_bounds_that_lie():
    from quantexperiments_amd.kernels import put_tokens8
    g = torch.Generator().manual_seed(7)
    table, pages, _ = table_for([20], 16, g)
    pool = Pool(pages, 16, 1, 2, 32, g)
    dev = pool.device()
    put_tokens8(torch.empty(0, 2, 32, dtype=torch.bfloat16).cuda(), torch.empty(0, 2, 32, dtype=torch.bfloat16).cuda(), *dev, table.cuda(), i32([0]), i32([0, 0]))
    k, v = tokens(4, 2, 32, "bf16", g)
    put_tokens8(k.cuda(), v.cuda(), *dev, table.cuda(), i32([0]), i32([0, 4]), most_new=0)
    pool.assert_same(*dev)
    put_tokens8(k.cuda(), v.cuda(), *dev, table.cuda(), i32([3]), i32([2, 1000]))          # (cut off at the last row)
    pool.put(k, v, table, [3], [2, 4])
    pool.assert_same(*dev)


def test_put_captured_and_on_another_stream():
    from quantexperiments_amd.kernels import put_tokens8
    g = torch.Generator().manual_seed(8)
    table, pages, _ = table_for([60, 60], 16, g)
    pool = Pool(pages, 16, 1, 2, 64, g)
    dev, lens, td = pool.device(), i32([0, 0]), table.cuda()
    k, v = (torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        put_tokens8(k, v, *dev, td, lens)
    for step in range(20):
        x = torch.randn(2, 2, 2, 64, generator=g).half() * (1 + step % 7)
        k.copy_(x[0])
        v.copy_(x[1])
        lens.fill_(step)
        lens[1] += 30
        graph.replay()
        pool.put(x[0], x[1], table, [step, step + 30], [0, 1, 2])
        torch.cuda.synchronize()
        pool.assert_same(*dev)
    with torch.cuda.stream(side):
        put_tokens8(k, v, *dev, td, lens)
    side.synchronize()
    pool.put(x[0], x[1], table, [19, 49], [0, 1, 2])
    pool.assert_same(*dev)


@pytest.mark.parametrize("dim", [16, 80, 96, 128, 256])
@pytest.mark.parametrize("lens,most,page,blocks,heads", [([0], 1, 16, 1, 1), ([3, 16, 31], 9, 16, 1, 4), ([13, 5], 40, 32, 2, 2), ([100, 0], 30, 128, 1, 3), ([61], 150, 96, 2, 1),
                                                         ([7], 100, 128, 1, 2)])
def test_keep_matches_the_definition(lens, most, page, blocks, heads, dim):
    from quantexperiments_amd.kernels import keep_drafted8
    g = torch.Generator().manual_seed(dim + most)
    drafted = most + 12
    table, pages, _ = table_for([l + drafted for l in lens], page, g)
    pool = Pool(pages, page, blocks, heads, dim, g)
    path = torch.stack([torch.randperm(drafted, generator=g)[:most].sort().values for _ in lens]).int()
    counts = [most - (b * most) // 4 for b in range(len(lens))]
    dev = pool.device()
    keep_drafted8(*dev, table.cuda(), i32(lens), path.cuda(), i32(counts))
    pool.keep(table, lens, path, counts)
    pool.assert_same(*dev)


def test_keep_all_layers_at_once_and_strided():
    from quantexperiments_amd.kernels import keep_drafted8
    g = torch.Generator().manual_seed(11)
    lens, page = [5, 40, 0], 16
    table, pages, _ = table_for([l + 20 for l in lens], page, g)
    pools = [Pool(pages, page, 1, 2, 32, g) for _ in range(3)]
    path = torch.tensor([[0, 2, 3, 11], [4, 5, 6, 19], [1, 2, 3, 4]], dtype=torch.int32)
    counts = [4, 3, 2]
    wide = [torch.zeros(3, *pools[0].codes.shape[1:-1], 64, dtype=torch.uint8, device="cuda") for _ in range(2)]
    dev = [w.view(torch.float8_e4m3fn)[..., 16:48] for w in wide]
    scales = [torch.stack([p.scales[i] for p in pools], 1).cuda().view(torch.float8_e8m0fnu).transpose(0, 1) for i in range(2)]          # layers inside pages
    for i, w in enumerate(wide):
        w[..., 16:48] = torch.stack([p.codes[i] for p in pools]).cuda()
    keep_drafted8(*dev, *scales, table.cuda(), i32(lens), path.cuda(), i32(counts))
    for l, p in enumerate(pools):
        p.keep(table, lens, path, counts)
        p.assert_same(dev[0][l], dev[1][l], scales[0][l], scales[1][l])
    assert not any(bool(w[..., :16].any()) or bool(w[..., 48:].any()) for w in wide)


def test_keep_ignores_what_is_no_path():
    from quantexperiments_amd.kernels import keep_drafted8
    g = torch.Generator().manual_seed(12)
    lens = [4, 4, 4, 4, 4, 30, 4, -9]
    table, pages, _ = table_for([40] * len(lens), 16, g)
    table = table[:, :3].clone()
    table[3, 1] = -1
    table[5, 2] = pages + 5
    pool = Pool(pages, 16, 1, 2, 32, g)
    path = torch.tensor([[1, 3, 2, 9], [-1, 2, 3, 4], [2, 2, 5, 6], [1, 2, 12, 14], [0, 43, 44, 45], [0, 1, 3, 9], [2 ** 31 - 1, 1, 2, 3], [1, 3, 5, 8]], dtype=torch.int32)
    counts = [4, 4, 4, 4, 9, 4, 4, 3]
    dev = pool.device()
    keep_drafted8(*dev, table.cuda(), i32(lens), path.cuda(), i32(counts))
    pool.keep(table, lens, path, counts)
    pool.assert_same(*dev)
    for bad in ([0] * 8, [-2 ** 31] * 8):
        keep_drafted8(*dev, table.cuda(), i32(lens), path.cuda(), i32(bad))
    pool.assert_same(*dev)


def test_keep_reads_no_table_behind_its_row():
    """A path that falls back early, so that later entries would go behind the last page of the table: nothing of it is looked up."""
    from quantexperiments_amd.kernels import keep_drafted8
    g = torch.Generator().manual_seed(13)
    table, pages, _ = table_for([48], 16, g)
    table = table[:, :3].contiguous()
    pool = Pool(pages, 16, 1, 1, 32, g)
    path = torch.tensor([[0, 1, 1, 1, *range(2, 60)]], dtype=torch.int32)
    dev = pool.device()
    keep_drafted8(*dev, table.cuda(), i32([20]), path.cuda(), i32([62]))
    pool.keep(table, [20], path, [62])
    pool.assert_same(*dev)


def refused(error, f, base, change):
    try:
        f(**{**base, **change})
    except error:
        return
    raise AssertionError({k: (tuple(t.shape), t.dtype, t.stride()) if isinstance(t, torch.Tensor) else t for k, t in change.items()})


def test_refusals():
    from quantexperiments_amd.kernels import keep_drafted8, put_tokens8
    g = torch.Generator().manual_seed(14)
    table, pages, _ = table_for([20], 32, g)
    pool = Pool(pages, 32, 2, 2, 32, g)
    kc, vc, ks, vs = pool.device()
    k, v = (torch.randn(3, 2, 32, generator=g).half().cuda() for _ in range(2))
    td, lens = table.cuda(), i32([4])
    ok = dict(k=k, v=v, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, table=td, lens=lens)
    raw = kc.view(torch.uint8)
    bad = [dict(k=k.float(), v=v.float()), dict(v=v.bfloat16()), dict(v=v[:2]), dict(k=k[0]), dict(k_cache=raw, v_cache=vc.view(torch.uint8)), dict(k_cache=kc[..., :16]),
           dict(k_cache=kc[:, :, :1], v_cache=vc[:, :, :1]), dict(k_scale=ks.view(torch.uint8)), dict(k_scale=ks[:, :1]), dict(k_scale=ks[..., :1], v_scale=vs[..., :1]), dict(v_cache=kc),
           dict(v_scale=ks), dict(k_scale=ks[:1].expand_as(ks)), dict(k_cache=kc[:1].expand_as(kc)), dict(table=td.long()), dict(table=td[0]), dict(lens=lens.long()), dict(starts=i32([0])),
           dict(starts=i32([0, 3]), most_new=-1), dict(most_new=2), dict(lens=lens.cpu()), dict(k_cache=kc[..., ::2][..., :16], v_cache=vc[..., ::2][..., :16], k=k[..., :16], v=v[..., :16])]
    for b in bad:
        refused(ValueError, put_tokens8, ok, b)
    from quantexperiments_amd._lib import SqError
    for b in (dict(k=k[..., :24].contiguous(), v=v[..., :24].contiguous(), k_cache=kc[..., :24], v_cache=vc[..., :24]),                     # no multiple of 16
              dict(k_cache=kc.transpose(0, 1)[:8].transpose(0, 1), v_cache=vc.transpose(0, 1)[:8].transpose(0, 1), k_scale=ks[:, :1], v_scale=vs[:, :1]),      # blocks of 8
              dict(k=torch.randn(3, 2, 33, device="cuda").half()[..., 1:])):                                                                # not aligned
        refused(SqError, put_tokens8, ok, b)
    with pytest.raises(NotImplementedError):
        put_tokens8(**{**ok, "k": k.clone().requires_grad_()})
    with torch.no_grad():
        put_tokens8(**{**ok, "k": k.clone().requires_grad_()})
    path, counts = i32([[0, 2]]), i32([2])
    keep = dict(k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, table=td, lens=lens, path=path, counts=counts)
    for b in (dict(path=path.long()), dict(path=path[0]), dict(counts=counts.long()), dict(counts=i32([1, 2])), dict(k_scale=ks[0]), dict(v_cache=kc), dict(k_cache=raw), dict(lens=lens.cpu()),
              dict(k_cache=kc[None], v_cache=vc[None])):
        refused(ValueError, keep_drafted8, keep, b)
    x = torch.zeros(3, 2, 32, dtype=torch.float16, device="cuda")
    whole = x.view(torch.uint8).view(-1).view(torch.float8_e4m3fn)[:192].view(1, 3, 2, 32)
    with pytest.raises(ValueError, match="overlaps"):
        put_tokens8(x, x.clone(), whole, whole.clone(), torch.zeros(1, 1, 2, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu),
                    torch.zeros(1, 1, 2, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu), td, lens)
