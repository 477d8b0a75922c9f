"""8-bit caches whose pages, layers and scales lie further apart than 32 bits count bytes: tokens put, drafts kept, sequences forked and a pool compacted in them."""

import pytest
import torch

from tests.cache8_model import Pool, table_for

pytestmark = pytest.mark.gpu
i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()


def test_pages_gigabytes_apart():
    from quantexperiments_amd.kernels import compact_pages, fork_pages, keep_drafted8, put_tokens8
    g = torch.Generator().manual_seed(31)
    lens, news = [70, 9, 31], [5, 6, 20]
    table, pages, spare = table_for([a + b for a, b in zip(lens, news)], 32, g, spare=4)
    pool = Pool(pages, 32, 2, 2, 64, g)
    bytes_ = 32 * 2 * 64
    step = (6 * 2 ** 30 // (pages - 1)) // 4096 * 4096               # the last page 6 GiB behind the first one
    memory = torch.zeros(step * (pages - 1) + 2 * bytes_ + 8, dtype=torch.uint8, device="cuda")
    codes = [torch.as_strided(memory, (pages, 32, 2, 64), (step, 128, 64, 1), i * bytes_) for i in range(2)]
    scales = [torch.as_strided(memory, (pages, 2, 2), (step, 2, 1), 2 * bytes_ + 4 * i) for i in range(2)]
    for i in range(2):
        codes[i].copy_(pool.codes[i])
        scales[i].copy_(pool.scales[i])
    cache = [t.view(torch.float8_e4m3fn) for t in codes] + [t.view(torch.float8_e8m0fnu) for t in scales]

    y = (torch.randn(sum(news), 4, 64, generator=g) * 4).bfloat16()
    starts, tl, ll = [0, 5, 11, 31], table.cuda(), i32(lens)
    put_tokens8(y[:, :2].cuda(), y[:, 2:].cuda(), *cache, tl, ll, i32(starts), most_new=20)
    pool.put(y[:, :2], y[:, 2:], table, lens, starts)
    pool.assert_same(*cache)

    path, counts = torch.tensor([[1, 2, 4], [0, 3, 5], [7, 8, 19]], dtype=torch.int32), [2, 3, 3]
    keep_drafted8(*cache, tl, ll, path.cuda(), i32(counts))
    pool.keep(table, lens, path, counts)
    pool.assert_same(*cache)

    lens = [a + b for a, b in zip(lens, counts)]
    both = dict(k_scale=cache[2], v_scale=cache[3])
    parent, fresh = [0, 0, 2, 1], [-1] + spare[:3].tolist()
    t, n = fork_pages(*cache[:2], tl, i32(lens), i32(parent), i32(fresh), **both)
    for p, f in zip(parent, fresh):
        whole, rest = divmod(lens[p], 32)
        if f >= 0 and rest:
            at, blocks = int(table[p, whole]), -(-rest // 16)
            pool.codes[:, f, :rest] = pool.codes[:, at, :rest]
            pool.scales[:, f, :blocks] = pool.scales[:, at, :blocks]
    pool.assert_same(*cache)
    assert n.tolist() == [lens[p] for p in parent]

    rows = t.cpu()
    held = [rows[i, :-(-lens[p] // 32)].tolist() for i, p in enumerate(parent)]
    t2, used = compact_pages(*cache[:2], t, n, **both)
    inuse = sorted({x for r in held for x in r})
    movers = [x for x in inuse if x >= len(inuse)]
    place = dict(zip(movers, [x for x in range(len(inuse)) if x not in inuse]))
    assert movers                                                    # (the seed's tables leave something to move)
    for a, b in place.items():
        pool.codes[:, b], pool.scales[:, b] = pool.codes[:, a], pool.scales[:, a]
    assert used.tolist() == [len(inuse)]
    for i, r in enumerate(held):
        assert t2[i].tolist() == [place.get(x, x) for x in r] + [-1] * (t2.shape[1] - len(r))
    pool.assert_same(*cache)
