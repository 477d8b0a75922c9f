"""A paged cache of keys and values held in 8 bits, and the pages of a cache, as a list of cases that can be timed.

A case is a dict of plain values; `prepare` makes what the program has in hand, `run` is one pass through an operator: with `own`
through quantexperiments_amd.kernels, without it in plain torch.  Operators:

  put_tokens8      keys and values of new tokens put into the cache: e4m3 codes, a power of two for each block of tokens and head
  tree_attention8  attention of new tokens (one: a decode step; a chain: a prompt's chunk; a tree: drafts) over it
  keep_drafted8    the accepted path of a draft moved behind the cached tokens, in the caches of all layers
  fork_pages       a batch whose rows continue sequences of another one: whole pages shared, last pages copied (beams, samples of a prompt)
  compact_pages    pages that no sequence uses any more freed: those in use moved to the front of the pool

Head counts and widths are those of the layers of bench.py and the tests, or generic.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"bf16": 2, "f16": 2, "e4m3": 1}
_MOST = {"bf16": 1.875 * 2.0 ** 127, "f16": 1.875 * 2.0 ** 15}          # largest number of four bits of mantissa


# ------------------------------------------------------------------ the cases

def _put(name, seqs, new, cached, hkv, dim, **kw):
    return {"name": name, "op": "put_tokens8", "seqs": seqs, "new": new, "cached": cached, "hkv": hkv, "dim": dim, "dtype": "bf16", "page": 16,
            "blocks": 1, "ragged": False, **kw}


def _attn(name, seqs, new, cached, hq, hkv, dim, **kw):
    return {"name": name, "op": "tree_attention8", "seqs": seqs, "new": new, "cached": cached, "hq": hq, "hkv": hkv, "dim": dim,
            "dtype": "bf16", "page": 16, "blocks": 1, "tree": False, "ragged": False, "lse": False, **kw}


def _keep(name, seqs, drafted, kept, layers, hkv, dim, **kw):
    return {"name": name, "op": "keep_drafted8", "seqs": seqs, "drafted": drafted, "kept": kept, "layers": layers, "hkv": hkv, "dim": dim,
            "page": 16, "blocks": 1, **kw}


def _fork(name, olds, rows, cached, layers, hkv, dim, **kw):
    return {"name": name, "op": "fork_pages", "olds": olds, "rows": rows, "cached": cached, "layers": layers, "hkv": hkv, "dim": dim,
            "cache": "bf16", "page": 16, "blocks": 1, "width": 64, **kw}


def _compact(name, seqs, cached, pages, layers, hkv, dim, **kw):
    return {"name": name, "op": "compact_pages", "seqs": seqs, "cached": cached, "pages": pages, "layers": layers, "hkv": hkv, "dim": dim,
            "cache": "bf16", "page": 16, "blocks": 1, **kw}


def listed():
    return [
        # a decode batch's keys and values of one layer, each into a block that holds tokens already: latency
        _put("put_64seqs_1token", 64, 1, 500, 4, 128, ragged=True),
        # a long prompt's chunk behind a part that ends inside a block, two blocks a page
        _put("put_8000tokens", 1, 8000, 1003, 8, 128, page=64, blocks=2),
        # batch-1 decode, short context: latency
        _attn("attention8_1seq_500", 1, 1, 500, 28, 4, 128),
        # a decode batch of ragged contexts
        _attn("attention8_32seqs_ragged", 32, 1, 8192, 40, 8, 128, page=64, ragged=True),
        # drafted trees of 48 tokens verified for 8 sequences
        _attn("attention8_8trees_of_48", 8, 48, 4096, 28, 4, 128, tree=True, ragged=True, dtype="f16", lse=True),
        # a prompt's chunk behind a cached part
        _attn("attention8_chunk_1900", 1, 1900, 2100, 28, 4, 128, page=32, blocks=2),
        # the accepted path of one tree, all layers of a 7B-shaped model
        _keep("keep8_1seq", 1, 48, 5, 28, 4, 128),
        # a batch of sequences
        _keep("keep8_64seqs", 64, 32, 8, 28, 4, 128),
        # one prompt sampled four times: three last pages copied, all layers
        _fork("fork_4samples", 1, 4, 1003, 28, 4, 128),
        # a beam step of 16 sequences of 4 beams over 8-bit pages of 64 slots
        _fork("fork_64beams", 64, 64, 500, 28, 4, 128, cache="e4m3", page=64, width=32),
        # one of a few short sequences ended in a small pool: latency
        _compact("compact_4seqs", 4, 100, 40, 4, 4, 128, cache="e4m3"),
        # a pool half of whose pages lie free
        _compact("compact_512pages", 24, 500, 1024, 28, 4, 128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("put_tokens8", "tree_attention8", "tree_attention8", "tree_attention8", "keep_drafted8", "fork_pages", "compact_pages"))
    hq, hkv, dim = rng.choice(((28, 4, 128), (40, 8, 128), (20, 4, 256), (14, 2, 64), (8, 8, 64), (6, 2, 96), (rng.randint(1, 16), 1, 80)))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    page, blocks = rng.choice(((16, 1), (16, 1), (32, 1), (32, 2), (64, 1), (64, 4), (48, 1), (96, 3)))
    held = dict(page=page, blocks=blocks)
    if op == "put_tokens8":
        seqs = _log(rng, 1, 64)
        c = _put("", seqs, rng.choice((1, rng.randint(2, 64), _log(rng, 65, 8000))) if seqs < 4 else rng.choice((1, 1, rng.randint(2, 64))),
                 _log(rng, 1, 1000), hkv, dim, dtype=dtype, ragged=rng.random() < 0.6, **held)
    elif op == "tree_attention8":
        kind = rng.choice(("single", "single", "tree", "tree", "chain"))
        if kind == "single":
            seqs, new = _log(rng, 1, 64), 1
            cached = _log(rng, 1, max(1, 131072 // seqs))
        elif kind == "tree":
            seqs, new = _log(rng, 1, 16), rng.randint(2, 100)
            cached = _log(rng, 1, max(1, 32768 // seqs))
        else:
            seqs, new = rng.randint(1, 3), _log(rng, 65, 600)
            cached = _log(rng, 1, 2000)
        hq, hkv, dim = (hq, hkv, dim) if hkv * dim <= 512 else (28, 4, 128)
        c = _attn("", seqs, new, cached, hq, hkv, dim, dtype=dtype, tree=kind == "tree", ragged=rng.random() < 0.6, lse=rng.random() < 0.3, **held)
    elif op == "keep_drafted8":
        drafted = _log(rng, 2, 64)
        c = _keep("", _log(rng, 1, 48), drafted, rng.randint(1, min(12, drafted)), rng.randint(1, 28), min(hkv, 4), min(dim, 128), **held)
    elif op == "fork_pages":
        olds = _log(rng, 1, 32)
        c = _fork("", olds, _log(rng, 1, 64), _log(rng, 1, 500), rng.randint(1, 28), min(hkv, 4), min(dim, 128), cache=rng.choice(("bf16", "e4m3", "f16")),
                  width=rng.randint(33, 80), **held)
    else:
        pages = _log(rng, 8, 8192 // page)
        seqs = _log(rng, 1, min(32, pages))
        c = _compact("", seqs, _log(rng, 1, max(1, pages // seqs * page)), pages, rng.randint(1, 28), min(hkv, 4), min(dim, 128),
                     cache=rng.choice(("bf16", "e4m3", "f16")), **held)
    del c["name"]
    return c


# ------------------------------------------------------------------ what a program has in hand before the call

def _spread(case):
    """Cached tokens of each sequence: all alike, or from a quarter of the most to all of it."""
    n, most = case["seqs"], case["cached"]
    return [max(1, most - (b * 3 * most) // (4 * n)) if case["ragged"] else most for b in range(n)]


def _news(case):
    return [max(1, case["new"] - (b % 3 if case["ragged"] else 0)) for b in range(case["seqs"])]


def _table(slots, page, cpu, spare=0, width=0):
    """A page table [sequences, pages] for that many slots each, its pages scattered over the pool, the pool's size and the pages left over."""
    need = [-(-s // page) for s in slots]
    total = sum(need) + spare
    order = torch.randperm(total, generator=cpu).to(torch.int32)
    table = torch.full((len(slots), max(max(need), width)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total, order[at:]


def _scale_of(exponents):
    return (exponents + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _times(x, e):
    """x * 2 ** e, whole e, exact but for the result's rounding (below 2 ** -126: as 2 ** -126)."""
    return x * (e.clamp(-126, 127) + 127).to(torch.int32).bitwise_left_shift(23).view(torch.float32)


def _held(x, blocks):
    """x [pages, slots, heads, dim] as codes and scales: the exponents by which no block is beyond the codes' range."""
    pages, page, heads, dim = x.shape
    x = x.view(pages, blocks, page // blocks, heads, dim)
    m, e = torch.frexp(x.abs().amax((2, 4)) / 448)
    e = torch.where(m > 0.5, e, e - 1)
    codes = _times(x, -e[:, :, None, :, None]).to(torch.float8_e4m3fn)
    return codes.view(pages, page, heads, dim), _scale_of(e)


def _codes(gen, *shape):
    """Codes of every finite value."""
    b = torch.randint(0, 254, shape, dtype=torch.uint8, device="cuda", generator=gen)
    return (b + (b >= 127)).to(torch.uint8).view(torch.float8_e4m3fn)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    op, page, blocks, hkv, dim = (case[k] for k in ("op", "page", "blocks", "hkv", "dim"))
    randn = lambda *shape: torch.randn(*shape, device=dev, generator=gen)
    spread = lambda pages: torch.exp(randn(pages, 1, hkv, 1) * 0.7)          # of a page and head: some hold larger values
    exponents = lambda *shape: _scale_of(torch.randint(-9, -5, shape, device=dev, generator=gen))
    s = {"case": case}
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    if op in ("put_tokens8", "tree_attention8"):
        dt = _DT[case["dtype"]]
        lens, news = _spread(case), _news(case)
        table, pages, _ = _table([a + b for a, b in zip(lens, news)], page, cpu)
        s["table"], s["lens"], s["starts"] = table.to(dev), i32(lens), i32([0] + list(np.cumsum(news)))
        s["most_new"], s["most_cached"] = max(news), max(lens)
        for n in "kv":
            s[n + "c"], s[n + "s"] = _held(randn(pages, page, hkv, dim) * spread(pages), blocks)
        if op == "put_tokens8":
            y = (randn(sum(news), 3 * hkv, dim) * torch.exp(randn(sum(news), 3 * hkv, 1) * 0.7)).to(dt)          # q|k|v as the stacked product writes them
            s["k"], s["v"] = y[:, hkv:2 * hkv], y[:, 2 * hkv:]
        else:
            s["q"] = (randn(sum(news), case["hq"], dim) * 2).to(dt)
            s["mask"] = _tree_words(news, cpu).to(dev) if case["tree"] else None
        return s
    layers = case["layers"]
    if op == "keep_drafted8":
        b = case["seqs"]
        lens = [1 + (37 * i) % 61 for i in range(b)]
        table, pages, _ = _table([n + case["drafted"] for n in lens], page, cpu)
        s["table"], s["lens"] = table.to(dev), i32(lens)
        s["path"] = torch.stack([torch.randperm(case["drafted"], generator=cpu)[:case["kept"]].sort().values for _ in range(b)]).to(torch.int32).to(dev)
        s["counts"] = torch.full((b,), case["kept"], dtype=torch.int32, device=dev)
        kind = "e4m3"
    elif op == "fork_pages":
        lens = [max(1, case["cached"] - 29 * i % max(1, case["cached"] // 2)) for i in range(case["olds"])]
        table, pages, spare = _table(lens, page, cpu, case["rows"], case["width"])
        parent = [int(x) for x in torch.randint(0, case["olds"], (case["rows"],), generator=cpu).sort().values]
        fresh = spare[:case["rows"]].tolist()
        first = [i == 0 or p != parent[i - 1] for i, p in enumerate(parent)]          # (the first row of a sequence goes on in its own last page)
        s["table"], s["lens"], s["parent"], s["pages"] = table.to(dev), i32(lens), i32(parent), i32([-1 if f else p for f, p in zip(first, fresh)])
        kind = case["cache"]
    else:
        lens = [max(1, case["cached"] - 31 * i % max(1, case["cached"] // 2)) for i in range(case["seqs"])]
        need = sum(-(-n // page) for n in lens)
        table, pages, _ = _table(lens, page, cpu, max(0, case["pages"] - need))
        s["table"], s["lens"] = table.to(dev), i32(lens)
        kind = case["cache"]
    shape = (layers, pages, page, hkv, dim)
    for n in "kv":
        s[n + "c"] = _codes(gen, *shape) if kind == "e4m3" else torch.randn(shape, dtype=_DT[kind], device=dev, generator=gen)
        s[n + "s"] = exponents(layers, pages, blocks, hkv) if kind == "e4m3" else None
    return s


def _tree_words(news, cpu):
    """Which drafted tokens each drafted token sees (itself and its ancestors) as 64-bit words [tokens, words]."""
    words = max(-(-n // 64) for n in news)
    rows = []
    for n in news:
        pick = torch.rand(n, generator=cpu).tolist()
        seen = []
        for t in range(n):
            parent = t - 1 - int(pick[t] ** 2 * min(t, 6))           # mostly the tokens drafted last; -1: the root
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << t)
        rows += [[(s >> 64 * w) & (1 << 64) - 1 for w in range(words)] for s in seen]
    return torch.from_numpy(np.array(rows, dtype=np.uint64).view(np.int64).reshape(len(rows), words))


# ------------------------------------------------------------------ one pass

def _exponents(scale):
    return scale.view(torch.uint8).to(torch.int32) - 127


def _values(codes, scale):
    """[.., slots, heads, dim] codes and [.., blocks, heads] scales as 32-bit values."""
    n = codes.shape[-3] // scale.shape[-2]
    return _times(codes.float(), _exponents(scale).repeat_interleave(n, -2)[..., None])


def _smallest(a):
    """The smallest exponents, from -100 on, by which a is not beyond the codes' range."""
    m, e = torch.frexp(a / 448)
    return torch.where(a > 0, torch.where(m > 0.5, e, e - 1), -100).clamp(min=-100)


def _places(s, at):
    """Pages and slots in them of slots `at` [sequences, n] (those behind a sequence's pages: some)."""
    page = s["case"]["page"]
    return s["table"].long().gather(1, (at // page).clamp(max=s["table"].shape[1] - 1)).clamp(min=0), at % page


def _plain_put(s, case):
    page, blocks, dev = case["page"], case["blocks"], s["kc"].device
    size, lens = page // blocks, s["lens"].long()
    news = (s["starts"][1:] - s["starts"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(lens), device=dev), news, output_size=s["k"].shape[0])
    slot = lens[seq] + torch.arange(len(seq), device=dev) - s["starts"].long()[seq]
    pg, off = s["table"].long()[seq, slot // page], slot % page
    block = pg * blocks + off // size
    first = lens // size * size                                                   # of the block that the new tokens start in
    old = first[:, None] + torch.arange(size, device=dev)
    old_pg, old_off = _places(s, old)
    held = old < lens[:, None]
    begun = torch.zeros(s["ks"].shape[0] * blocks + 1, dtype=torch.bool, device=dev)
    begun[torch.where(lens > first, old_pg[:, 0] * blocks + old_off[:, 0] // size, -1)] = True
    for new, codes, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = new.float().clamp(-_MOST[case["dtype"]], _MOST[case["dtype"]])
        x = torch.where(new.isfinite(), x, math.nan)
        top = torch.zeros(scale.shape[0] * blocks, scale.shape[2], device=dev)
        top.scatter_reduce_(0, block[:, None].expand(-1, x.shape[1]), x.nan_to_num(0.0).abs().amax(-1), "amax")
        e0 = _exponents(scale).reshape(top.shape)
        e = torch.maximum(_smallest(top), torch.where(begun[:-1, None], e0, -100))
        touched = torch.zeros(len(top), dtype=torch.bool, device=dev)
        touched[block] = True
        e = torch.where(touched[:, None], e, e0)
        raw, flat = codes.view(torch.uint8), scale.view(torch.uint8)
        was = _times(codes[old_pg, old_off].float(), (e0 - e)[(old_pg * blocks + old_off // size)][..., None]).to(codes.dtype).view(torch.uint8)
        raw[old_pg[held], old_off[held]] = was[held]
        raw[pg, off] = _times(x, -e[block][..., None]).to(codes.dtype).view(torch.uint8)
        flat.copy_((e + 127).to(torch.uint8).view(scale.shape))
    return s["kc"], s["vc"], s["ks"], s["vs"]


def _plain_attention(s, case):
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    size = page // case["blocks"]
    group, new, dev = hq // hkv, s["most_new"], s["q"].device
    lens, starts = s["lens"].long(), s["starts"].long()
    news = starts[1:] - starts[:-1]
    at = torch.arange(s["most_cached"] + new, device=dev)
    pg, off = _places(s, at.expand(len(lens), -1))

    def gathered(codes, scale):
        e = _exponents(scale)[pg, off // size]
        return _times(codes[pg, off].float(), e[..., None]).transpose(1, 2).contiguous()                       # [b, hkv, slots, dim]
    k, v = gathered(s["kc"], s["ks"]), gathered(s["vc"], s["vs"])
    tok = starts[:-1, None] + torch.arange(new, device=dev)                                                         # [b, new]
    there = torch.arange(new, device=dev) < news[:, None]
    tok = torch.where(there, tok, 0)
    q = s["q"].float()[tok].reshape(len(lens), new, hkv, group, dim).transpose(1, 2).reshape(len(lens), hkv, new * group, dim)
    j = at - lens[:, None]                                                                                          # [b, slots]: drafted token of a slot
    if s["mask"] is None:
        sees = j[:, None, :] <= torch.arange(new, device=dev)[:, None]
    else:
        word = s["mask"][tok].gather(2, (j.clamp(min=0) >> 6).clamp(max=s["mask"].shape[1] - 1)[:, None, :].expand(-1, new, -1))
        sees = (j[:, None, :] < 0) | ((word >> (j.clamp(min=0) & 63)[:, None, :]) & 1).bool()
    sees = (sees & (j < news[:, None])[:, None, :]).repeat_interleave(group, 1)[:, None]                            # [b, 1, rows, slots]
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * dim ** -0.5
    score = torch.where(sees, score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / total.clamp(min=1e-38)
    back = lambda t: t.reshape(len(lens), hkv, new, group, -1).transpose(1, 2).reshape(len(lens), new, hq, -1)[there]
    out = back(out).to(s["q"].dtype)
    return (out, back(top + torch.log(total))[..., 0]) if case["lse"] else out


def _plain_keep(s, case):
    blocks, size, dev = case["blocks"], case["page"] // case["blocks"], s["kc"].device
    lens, m = s["lens"].long(), s["path"].shape[1]
    i = torch.arange(m, device=dev)
    src, dst = lens[:, None] + s["path"].long(), lens[:, None] + i
    keeps = i < s["counts"].long()[:, None]
    (sp, so), (dp, do) = _places(s, src), _places(s, dst)
    first = lens // size * size
    old = first[:, None] + torch.arange(size, device=dev)
    op_, oo = _places(s, old)
    held = (old < lens[:, None]) & keeps[:, :1]
    target = dp * blocks + do // size
    begun = torch.where((lens > first) & keeps[:, 0], op_[:, 0] * blocks + oo[:, 0] // size, -1)
    for codes, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        layers, pages, _, heads = scale.shape
        e0 = _exponents(scale).reshape(layers, pages * blocks, heads)
        es = e0[:, sp * blocks + so // size]                                       # [layers, b, m, heads]
        e = torch.full((layers, pages * blocks + 1, heads), -127, dtype=torch.int32, device=dev)
        e[:, begun] = torch.cat((e0, e[:, -1:]), 1)[:, begun]
        put = torch.where(keeps, target, pages * blocks).reshape(-1)
        e.scatter_reduce_(1, put[None, :, None].expand(layers, -1, heads), es.flatten(1, 2), "amax")
        touched = torch.zeros(pages * blocks + 1, dtype=torch.bool, device=dev)
        touched[put] = True
        e = torch.where(touched[:-1, None], e[:, :-1], e0)
        raw = codes.view(torch.uint8)
        rows = _times(codes[:, sp, so].float(), (es - e[:, target])[..., None]).to(codes.dtype).view(torch.uint8)
        ob = op_ * blocks + oo // size
        was = _times(codes[:, op_, oo].float(), (e0 - e)[:, ob][..., None]).to(codes.dtype).view(torch.uint8)
        raw[:, op_[held], oo[held]] = was[:, held]
        raw[:, dp[keeps], do[keeps]] = rows[:, keeps]
        scale.view(torch.uint8).copy_((e + 127).to(torch.uint8).view(scale.shape))
    return s["kc"], s["vc"], s["ks"], s["vs"]


def _bits(t):
    return t if t is None or t.element_size() > 1 else t.view(torch.uint8)


def _plain_fork(s, case):
    page, dev = case["page"], s["kc"].device
    parent, fresh = s["parent"].long(), s["pages"].long()
    table, lens = s["table"][parent], s["lens"][parent]
    whole, rest = (lens // page).long(), (lens % page).long()
    rows = torch.arange(len(parent), device=dev)
    copy = (fresh >= 0) & (rest > 0)
    at = whole.clamp(max=table.shape[1] - 1)
    src = table[rows, at].long()
    slots = torch.arange(page, device=dev)
    which, slot = (copy[:, None] & (slots < rest[:, None])).nonzero(as_tuple=True)
    for c in (s["kc"], s["vc"]):
        _bits(c)[:, fresh[which], slot] = _bits(c)[:, src[which], slot]
    if s["ks"] is not None:
        size = page // case["blocks"]
        which, block = (copy[:, None] & (torch.arange(case["blocks"], device=dev) * size < rest[:, None])).nonzero(as_tuple=True)
        for c in (s["ks"], s["vs"]):
            _bits(c)[:, fresh[which], block] = _bits(c)[:, src[which], block]
    j = torch.arange(table.shape[1], device=dev)
    forked = torch.where(j < whole[:, None], table, torch.where(j == whole[:, None], s["pages"][:, None], -1))
    return torch.where(fresh[:, None] >= 0, forked, table), lens


def _plain_compact(s, case):
    page, dev = case["page"], s["kc"].device
    pages = s["kc"].shape[1]
    live = torch.arange(s["table"].shape[1], device=dev) < ((s["lens"] + page - 1) // page)[:, None]
    used = torch.zeros(pages, dtype=torch.bool, device=dev)
    used[s["table"][live].long()] = True
    n = used.sum()
    ids = torch.arange(pages, device=dev)
    holes, movers = ids[(ids < n) & ~used], ids[(ids >= n) & used]
    to = ids.clone()
    to[movers] = holes
    for c in (s["kc"], s["vc"], s["ks"], s["vs"]):
        if c is not None:
            _bits(c)[:, holes] = _bits(c)[:, movers]
    return torch.where(live, to[s["table"].clamp(min=0).long()].int(), -1), n.int()[None]


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        from quantexperiments_amd import kernels as K
        cache = (s["kc"], s["vc"], s["ks"], s["vs"])
        if op == "put_tokens8":
            K.put_tokens8(s["k"], s["v"], *cache, s["table"], s["lens"], s["starts"], most_new=s["most_new"])
            return cache
        if op == "tree_attention8":
            lse = torch.empty(s["q"].shape[:2], device=s["q"].device) if case["lse"] else None
            out = K.tree_attention8(s["q"], *cache, s["table"], s["lens"], s["starts"], most_new=s["most_new"], mask=s["mask"], lse=lse)
            return out if lse is None else (out, lse)
        if op == "keep_drafted8":
            K.keep_drafted8(*cache, s["table"], s["lens"], s["path"], s["counts"])
            return cache
        if op == "fork_pages":
            return (*K.fork_pages(s["kc"], s["vc"], s["table"], s["lens"], s["parent"], s["pages"], k_scale=s["ks"], v_scale=s["vs"]), *cache)
        return (*K.compact_pages(s["kc"], s["vc"], s["table"], s["lens"], k_scale=s["ks"], v_scale=s["vs"]), *cache)
    if op == "put_tokens8":
        return _plain_put(s, case)
    if op == "tree_attention8":
        return _plain_attention(s, case)
    if op == "keep_drafted8":
        return _plain_keep(s, case)
    return (*(_plain_fork if op == "fork_pages" else _plain_compact)(s, case), s["kc"], s["vc"], s["ks"], s["vs"])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op, row = case["op"], case["hkv"] * case["dim"]
    if op in ("put_tokens8", "tree_attention8"):
        lens, news = _spread(case), _news(case)
    if op == "put_tokens8":
        size = case["page"] // case["blocks"]
        blocks = sum((l + n - 1) // size - l // size + 1 for l, n in zip(lens, news))
        return {"bytes": 2 * sum(news) * row * 3 + 2 * blocks * case["hkv"] * 2, "flops": 4 * sum(news) * row}
    if op == "tree_attention8":
        rows = sum(news) * case["hq"]
        seen = sum(n * l + (n * (n + 1) // 2) for l, n in zip(lens, news)) * case["hq"]
        held = sum(l + n for l, n in zip(lens, news))
        return {"bytes": 2 * held * row + 4 * rows * case["dim"], "flops": 4 * seen * case["dim"]}
    if op == "keep_drafted8":
        return {"bytes": 4 * case["seqs"] * case["kept"] * case["layers"] * row, "flops": 0}
    row *= _SIZE[case["cache"]] * case["layers"]
    if op == "fork_pages":
        # (about half a page a row)
        return {"bytes": 4 * case["rows"] * (case["page"] // 2) * row + 8 * case["rows"] * case["width"], "flops": 0}
    need = sum(-(-max(1, case["cached"] - 31 * i % max(1, case["cached"] // 2)) // case["page"]) for i in range(case["seqs"]))
    pages = max(need, case["pages"])
    # (the pages in use lie anywhere: as many of them as of all lie behind the number in use)
    return {"bytes": round(4 * need * (pages - need) / pages) * case["page"] * row + 12 * need, "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits

_CODES = [(-1) ** (b >> 7) * ((b & 7) / 8 * 2.0 ** -6 if (b >> 3) & 15 == 0 else math.nan if b & 127 == 127 else (1 + (b & 7) / 8) * 2.0 ** (((b >> 3) & 15) - 7))
          for b in range(256)]


def _two_to(n):
    return ((n + 1023) << 52).view(torch.float64)


def _read(codes, scale):
    """The numbers that codes [.., slots, heads, dim] stand for and their scales [.., blocks, heads], in 64 bits."""
    size = codes.shape[-3] // scale.shape[-2]
    x = torch.tensor(_CODES, dtype=torch.float64, device=codes.device)[codes.view(torch.uint8).long()]
    f = _two_to(scale.view(torch.uint8).long() - 127)
    return x, f, x * torch.repeat_interleave(f, size, -2).unsqueeze(-1)


def _nearest(x):
    """x (64 bits) rounded to the nearest code, ties to the even one."""
    step = _two_to(torch.frexp(x.nan_to_num(0.0).abs().clamp(min=2.0 ** -6)).exponent.long() - 4)
    return torch.round(x / step) * step


def _fits(a):
    """2 ** e for the smallest whole e, from -100 on, with a <= 448 * 2 ** e."""
    f = torch.full_like(a, 2.0 ** -100)
    for _ in range(230):
        f = torch.where(a > 448 * f, 2 * f, f)
    return f


def _exact_put(s, case):
    page, size = case["page"], case["page"] // case["blocks"]
    out = []
    for new, codes, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        code, f, value = _read(codes, scale)
        top = _MOST[case["dtype"]]
        row = 0
        for b, (l, n) in enumerate(zip(_spread(case), _news(case))):
            x = new[row:row + n].double()
            x = torch.where(x.abs() < math.inf, x.clamp(-top, top), math.nan)
            row += n
            at = l
            while at < l + n:
                first = at // size * size
                end = min(first + size, l + n)
                pg, o = int(s["table"][b, first // page]), first % page
                y = x[at - l:end - l]
                g = _fits(y.nan_to_num(0.0).abs().amax((0, 2)))
                if at > first:
                    g = torch.maximum(g, f[pg, o // size])
                    code[pg, o:o + at - first] = _nearest(value[pg, o:o + at - first] / g[:, None])
                code[pg, o + at - first:o + end - first] = _nearest(y / g[:, None])
                f[pg, o // size] = g
                at = end
        out.append((code, f))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attention(s, case):
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    size = page // case["blocks"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device=s["q"].device)
    known = torch.tensor(_CODES, dtype=torch.float64, device=out.device)
    first = 0
    for b, (l, n) in enumerate(zip(_spread(case), _news(case))):
        at = torch.arange(l + n, device=out.device)
        pages, off = s["table"][b].long()[at // page], at % page
        j = torch.arange(n, device=out.device)
        if s["mask"] is None:
            sees = j[:, None] >= j
        else:
            sees = (s["mask"][first:first + n][:, j // 64] >> (j % 64)) % 2 == 1
        bias = torch.zeros(n, l + n, dtype=torch.float64, device=out.device)
        bias[:, l:].masked_fill_(~sees, -math.inf)
        for h in range(hkv):
            k, v = (known[c.view(torch.uint8)[pages, off, h].long()] * _two_to(f.view(torch.uint8)[pages, off // size, h].long() - 127)[:, None]
                    for c, f in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
            for g in range(h * hq // hkv, (h + 1) * hq // hkv):
                score = s["q"][first:first + n, g].double() @ k.T / math.sqrt(dim) + bias
                lse[first:first + n, g] = torch.logsumexp(score, -1)
                out[first:first + n, g] = torch.softmax(score, -1) @ v
        first += n
    return (out, lse) if case["lse"] else out


def _exact_keep(s, case):
    page, size = case["page"], case["page"] // case["blocks"]
    table, path, lens = s["table"].tolist(), s["path"].tolist(), s["lens"].tolist()
    out = []
    for codes, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        code, f, value = _read(codes, scale)
        old_code, old_f = code.clone(), f.clone()
        for b, l in enumerate(lens):
            spot = lambda slot: (table[b][slot // page], slot % page)
            for first in range(l // size * size, l + len(path[b]), size):
                mine = [i for i in range(len(path[b])) if first <= l + i < first + size]
                if not mine:
                    continue
                froms = [spot(l + path[b][i]) for i in mine]
                g = torch.stack([old_f[:, p, o // size] for p, o in froms]).amax(0)
                pg, o = spot(first)
                if first < l:
                    g = torch.maximum(g, old_f[:, pg, o // size])
                    code[:, pg, o:o + l - first] = _nearest(value[:, pg, o:o + l - first] / g[:, None, :, None])
                for i, (p, at) in zip(mine, froms):
                    tp, to = spot(l + i)
                    code[:, tp, to] = _nearest(value[:, p, at] / g[..., None])
                f[:, pg, o // size] = g
        out.append((code, f))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_pages(s, case):
    page = case["page"]
    table, lens = s["table"].tolist(), s["lens"].tolist()
    cache = [s["kc"].clone(), s["vc"].clone(), None if s["ks"] is None else s["ks"].clone(), None if s["vs"] is None else s["vs"].clone()]
    raw = [_bits(c) for c in cache]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=s["table"].device)
    if case["op"] == "fork_pages":
        rows, sizes = [], []
        for p, f in zip(s["parent"].tolist(), s["pages"].tolist()):
            whole, rest = divmod(lens[p], page)
            row = list(table[p])
            if f >= 0:
                for i, c in enumerate(raw):
                    n = rest if i < 2 else -(-rest * case["blocks"] // page)
                    if c is not None and rest:
                        c[:, f, :n] = c[:, row[whole], :n]
                row = (row[:whole] + [f] + [-1] * len(row))[:len(row)]
            rows.append(row)
            sizes.append(lens[p])
        return (i32(rows), i32(sizes), *cache)
    in_use = sorted({table[b][j] for b in range(len(lens)) for j in range(-(-lens[b] // page))})
    n = len(in_use)
    to = dict(zip(in_use, in_use))
    holes = [p for p in range(n) if p not in to]
    for p, h in zip([p for p in in_use if p >= n], holes):
        to[p] = h
        for c in raw:
            if c is not None:
                c[:, h] = c[:, p]
    new = [[to[p] if j * page < lens[b] else -1 for j, p in enumerate(row)] for b, row in enumerate(table)]
    return (i32(new), i32([n]), *cache)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "put_tokens8":
        return _exact_put(s, case)
    if case["op"] == "tree_attention8":
        return _exact_attention(s, case)
    return _exact_keep(s, case) if case["op"] == "keep_drafted8" else _exact_pages(s, case)
