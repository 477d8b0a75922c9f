"""What a decoder layer does between its q|k|v product and its o product, as a list of cases that can be timed.

A case is a dict of plain values; `prepare` makes what the program has in hand, `run` is one pass through an operator: with `own`
through quantexperiments_amd.kernels, without it in plain torch.  Operators:

  rotary          rotation of the heads of queries and keys by their tokens' positions
  qk_norm_rotary  RMS norm of each query and key head and the rotation in one pass, keys and values put in their cache slots
  tree_attention  attention of drafted tokens (one: a decode step; a chain: a prompt's chunk; a tree: drafts) over a paged cache
  keep_drafted    the accepted path of a draft moved behind the cached tokens, in the caches of all layers

Head counts and widths are those of the layers of bench.py and the tests, or generic.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------ the cases

def _rotary(name, tokens, hq, hkv, dim, **kw):
    return {"name": name, "op": "rotary", "tokens": tokens, "hq": hq, "hkv": hkv, "dim": dim, "rot": dim, "dtype": "bf16",
            "interleaved": False, "scaling": "none", "far": 4096, **kw}


def _norm(name, tokens, hq, hkv, dim, **kw):
    return {"name": name, "op": "qk_norm_rotary", "tokens": tokens, "hq": hq, "hkv": hkv, "dim": dim, "rot": dim, "dtype": "bf16",
            "interleaved": False, "scaling": "none", "far": 4096, "norm": True, "offset": 0.0, "page": 16, **kw}


def _attn(name, seqs, new, cached, hq, hkv, dim, **kw):
    return {"name": name, "op": "tree_attention", "seqs": seqs, "new": new, "cached": cached, "hq": hq, "hkv": hkv, "dim": dim,
            "dtype": "bf16", "page": 16, "tree": False, "ragged": False, "lse": False, **kw}


def _keep(name, seqs, drafted, kept, layers, hkv, dim, **kw):
    return {"name": name, "op": "keep_drafted", "seqs": seqs, "drafted": drafted, "kept": kept, "layers": layers, "hkv": hkv, "dim": dim,
            "dtype": "bf16", "page": 16, **kw}


def listed():
    return [
        # one decoded token of a 7B-shaped layer without head norms: latency
        _rotary("rotary_1token", 1, 28, 4, 128),
        # a prompt's chunk far into a long context, frequencies stretched for it
        _rotary("rotary_2048tokens_far", 2048, 28, 4, 128, scaling="yarn", far=131072),
        # a decode batch of a 27B-class layer
        _norm("norm_rotary_8tokens", 8, 40, 8, 128),
        # a ragged chunk, a quarter of wide heads rotated in pairs, norm weights stored as w - 1
        _norm("norm_rotary_333tokens_part", 333, 20, 4, 256, rot=64, interleaved=True, offset=1.0, page=64, dtype="f16"),
        # a chunk of a chunked prefill
        _norm("norm_rotary_2048tokens", 2048, 28, 4, 128),
        # batch-1 decode, short context: latency
        _attn("attention_1seq_500", 1, 1, 500, 28, 4, 128),
        # batch-1 decode, long context: one sequence over the whole chip; partial results joined
        _attn("attention_1seq_131072", 1, 1, 131072, 28, 4, 128, page=64, lse=True),
        # a decode batch of ragged contexts
        _attn("attention_32seqs_ragged", 32, 1, 8192, 40, 8, 128, ragged=True),
        # drafted trees of 48 tokens verified for 8 sequences
        _attn("attention_8trees_of_48", 8, 48, 4096, 28, 4, 128, tree=True, ragged=True, dtype="f16"),
        # a prompt's chunk behind a cached part
        _attn("attention_chunk_1900", 1, 1900, 2100, 28, 4, 128),
        # the accepted path of one tree, all layers of a 7B-shaped model
        _keep("keep_1seq", 1, 48, 5, 28, 4, 128),
        # a batch of sequences
        _keep("keep_64seqs", 64, 32, 8, 28, 4, 128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _heads(rng):
    return rng.choice(((28, 4, 128), (40, 8, 128), (20, 4, 256), (14, 2, 64), (8, 8, 128), (6, 2, 96), (rng.randint(1, 16), 1, 80)))


def draw(rng):
    op = rng.choice(("rotary", "qk_norm_rotary", "tree_attention", "tree_attention", "tree_attention", "keep_drafted"))
    hq, hkv, dim = _heads(rng)
    dtype = rng.choice(("bf16", "bf16", "f16"))
    page = rng.choice((16, 16, 64, 24, 1))
    if op == "keep_drafted":
        drafted = _log(rng, 2, 64)
        c = _keep("", _log(rng, 1, 32), drafted, rng.randint(1, min(8, drafted)), rng.randint(1, 28), min(hkv, 4), min(dim, 128), dtype=dtype, page=page)
    elif op == "tree_attention":
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
        c = _attn("", seqs, new, cached, hq, hkv, dim, dtype=dtype, page=page, tree=kind == "tree", ragged=rng.random() < 0.6,
                  lse=rng.random() < 0.3)
    else:
        rot = rng.choice((dim, dim, dim // 2, dim // 4 // 2 * 2))
        kw = dict(rot=rot, interleaved=rng.random() < 0.4, scaling=rng.choice(("none", "linear", "yarn", "bands")), far=_log(rng, 64, 1000000))
        tokens = _log(rng, 1, 2048)
        if op == "rotary":
            c = _rotary("", tokens, hq, hkv, dim, dtype=rng.choice(("bf16", "f16", "f32")), **kw)
        else:
            c = _norm("", tokens, hq, hkv, dim, dtype=dtype, page=page, norm=rng.random() < 0.7, offset=rng.choice((0.0, 1.0)), **kw)
    del c["name"]
    return c


# ------------------------------------------------------------------ what a program has in hand before the call

def _freqs(rot, scaling):
    """(radians per position of each pair in 64 bits, amplitude) for a context stretched four times, and its amplitude."""
    base, factor, trained = 10000.0, 4.0, 32768
    i = np.arange(rot // 2, dtype=np.float64)
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        turn = lambda n: rot * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rot - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        return f / factor * ramp + f * (1.0 - ramp), 0.1 * math.log(factor) + 1.0
    if scaling == "bands":
        smooth = np.clip((trained * f / (2 * math.pi) - 1.0) / 3.0, 0.0, 1.0)
        return (1.0 - smooth) * f / factor + smooth * f, 1.0
    return f, 1.0


def _spread(case, most):
    """Cached tokens (or other sizes up to `most`) of each sequence: all alike, or from a quarter of it to all of it."""
    n = case["seqs"]
    return [max(1, most - (b * 3 * most) // (4 * n)) if case.get("ragged") else most for b in range(n)]


def _news(case):
    return [max(1, case["new"] - (b % 3 if case["ragged"] else 0)) for b in range(case["seqs"])]


def _table(slots, page, cpu):
    """A page table [sequences, pages] for that many slots each, its pages scattered over the pool, and the pool's size."""
    need = [-(-s // page) for s in slots]
    total = sum(need)
    order = torch.randperm(total, generator=cpu).to(torch.int32)
    table = torch.zeros(len(slots), max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


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


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    dt, op = _DT[case["dtype"]], case["op"]
    randn = lambda *shape: torch.randn(*shape, device=dev, generator=gen)
    s = {"case": case}
    if op in ("rotary", "qk_norm_rotary"):
        n, hq, hkv, dim = case["tokens"], case["hq"], case["hkv"], case["dim"]
        f, s["scale"] = _freqs(case["rot"], case["scaling"])
        s["freqs"] = torch.from_numpy(f).to(dev)
        first = int(torch.randint(0, max(1, case["far"] - n + 1), (1,), generator=cpu))
        s["positions"] = torch.arange(first, first + n, device=dev)
        y = (randn(n, hq + 2 * hkv, dim) * 2).to(dt)                 # q|k|v as the stacked product writes them
        s["q"], s["k"], s["v"], s["qk"] = y[:, :hq], y[:, hq:hq + hkv], y[:, hq + hkv:], y[:, :hq + hkv]
        if op == "qk_norm_rotary":
            s["q_w"], s["k_w"] = ((torch.rand(dim, device=dev, generator=gen) + 0.5 - case["offset"]).to(dt) if case["norm"] else None for _ in range(2))
            table, pages = _table([n], case["page"], cpu)
            at = torch.arange(n)
            s["slots"] = (table[0, at // case["page"]].long() * case["page"] + at % case["page"]).to(dev)
            s["kc"], s["vc"] = (torch.zeros(pages, case["page"], hkv, dim, dtype=dt, device=dev) for _ in range(2))
    elif op == "tree_attention":
        hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
        lens, news = _spread(case, case["cached"]), _news(case)
        table, pages = _table([a + b for a, b in zip(lens, news)], page, cpu)
        s["table"], s["lens"] = table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
        s["starts"] = torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32, device=dev)
        s["most_new"], s["most_cached"] = max(news), max(lens)
        s["q"] = (randn(sum(news), hq, dim) * 2).to(dt)
        s["kc"], s["vc"] = (randn(pages, page, hkv, dim).to(dt) for _ in range(2))
        s["mask"] = _tree_words(news, cpu).to(dev) if case["tree"] else None
    else:
        b, layers, page = case["seqs"], case["layers"], case["page"]
        lens = [1 + (37 * i) % 61 for i in range(b)]
        table, pages = _table([n + case["drafted"] for n in lens], page, cpu)
        s["table"], s["lens"] = table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
        s["path"] = torch.stack([torch.randperm(case["drafted"], generator=cpu)[:case["kept"]].sort().values for _ in range(b)]).to(torch.int32).to(dev)
        s["counts"] = torch.full((b,), case["kept"], dtype=torch.int32, device=dev)
        s["kc"], s["vc"] = (randn(layers, pages, page, case["hkv"], case["dim"]).to(dt) for _ in range(2))
    return s


# ------------------------------------------------------------------ one pass

def _turned(x, s, case):
    """x [tokens, heads, dim] (32 bits) rotated by its tokens' positions."""
    angle = s["positions"].double()[:, None] * s["freqs"]
    cos, sin = ((t * s["scale"]).float()[:, None] for t in (angle.cos(), angle.sin()))
    r = case["rot"]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((y, x[..., r:]), dim=-1)


def _normed(x, w, offset):
    x = x.float()
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (w.float() + offset)


def _slots_of(s, at):
    """Pool rows of slots `at` [sequences, n] (those behind a sequence's pages: some row)."""
    page = s["case"]["page"]
    pages = s["table"].long().gather(1, (at // page).clamp(max=s["table"].shape[1] - 1))
    return pages * page + at % page


def _plain_attention(s, case):
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    group, new, dev = hq // hkv, s["most_new"], s["q"].device
    lens, starts = s["lens"].long(), s["starts"].long()
    news = starts[1:] - starts[:-1]
    at = torch.arange(s["most_cached"] + new, device=dev)
    rows = _slots_of(s, at.expand(len(lens), -1))
    k, v = (c.reshape(-1, hkv, dim)[rows].float().transpose(1, 2).contiguous() for c in (s["kc"], s["vc"]))          # [b, hkv, slots, dim]
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


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        from quantexperiments_amd import kernels as K
        if op == "rotary":
            return K.rotary(s["qk"], s["positions"], s["freqs"], interleaved=case["interleaved"], scale=s["scale"])
        if op == "qk_norm_rotary":
            q, _ = K.qk_norm_rotary(s["q"], s["k"], s["positions"], s["freqs"], s["q_w"], s["k_w"], 1e-6, v=s["v"], k_cache=s["kc"], v_cache=s["vc"],
                                    slots=s["slots"], interleaved=case["interleaved"], scale=s["scale"], weight_offset=case["offset"])
            return q, s["kc"], s["vc"]
        if op == "tree_attention":
            lse = torch.empty(s["q"].shape[:2], device=s["q"].device) if case["lse"] else None
            out = K.tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["starts"], most_new=s["most_new"], mask=s["mask"], lse=lse)
            return out if lse is None else (out, lse)
        K.keep_drafted(s["kc"], s["vc"], s["table"], s["lens"], s["path"], s["counts"])
        return s["kc"], s["vc"]
    if op == "rotary":
        return _turned(s["qk"].float(), s, case).to(s["qk"].dtype)
    if op == "qk_norm_rotary":
        q = _turned(_normed(s["q"], s["q_w"], case["offset"]), s, case).to(s["q"].dtype)
        flat = lambda c: c.view(-1, *c.shape[2:])
        flat(s["kc"])[s["slots"]] = _turned(_normed(s["k"], s["k_w"], case["offset"]), s, case).to(s["k"].dtype)
        flat(s["vc"])[s["slots"]] = s["v"]
        return q, s["kc"], s["vc"]
    if op == "tree_attention":
        return _plain_attention(s, case)
    m = s["path"].shape[1]
    i = torch.arange(m, device=s["path"].device)
    src = _slots_of(s, s["lens"].long()[:, None] + s["path"].long())
    dst = _slots_of(s, s["lens"].long()[:, None] + i)
    dst = torch.where(i < s["counts"].long()[:, None], dst, src)
    for c in (s["kc"], s["vc"]):
        flat = c.view(c.shape[0], -1, *c.shape[3:])
        flat[:, dst.reshape(-1)] = flat[:, src.reshape(-1)]
    return s["kc"], s["vc"]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op, size = case["op"], _SIZE[case["dtype"]]
    if op in ("rotary", "qk_norm_rotary"):
        turned = case["tokens"] * (case["hq"] + case["hkv"]) * case["dim"]
        moved = turned + (case["tokens"] * case["hkv"] * case["dim"] if op == "qk_norm_rotary" else 0)
        return {"bytes": 2 * moved * size + case["tokens"] * 8, "flops": 3 * turned + (4 * turned if case.get("norm") else 0)}
    if op == "tree_attention":
        lens, news = _spread(case, case["cached"]), _news(case)
        rows = sum(news) * case["hq"]
        seen = sum(n * l + (n * (n + 1) // 2) for l, n in zip(lens, news)) * case["hq"]
        cache = sum(l + n for l, n in zip(lens, news)) * case["hkv"]
        return {"bytes": 2 * (cache + rows) * case["dim"] * size, "flops": 4 * seen * case["dim"]}
    return {"bytes": 4 * case["seqs"] * case["kept"] * case["layers"] * case["hkv"] * case["dim"] * size, "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_turn(x, positions, freqs, scale, rot, interleaved):
    z = torch.polar(torch.full_like(freqs, scale).expand(len(positions), -1), torch.outer(positions.double(), freqs))[:, None]
    y = x.clone()
    i = torch.arange(rot // 2, device=x.device)
    ai, bi = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    t = torch.complex(x[..., ai], x[..., bi]) * z
    y[..., ai], y[..., bi] = t.real, t.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    turn = lambda x: _exact_turn(x, s["positions"], s["freqs"], s["scale"], case["rot"], case["interleaved"])
    if op == "rotary":
        return turn(s["qk"].double())
    if op == "qk_norm_rotary":
        def one(x, w):
            x = x.double()
            return turn(x if w is None else x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (w.double() + case["offset"]))
        kc, vc = s["kc"].double(), s["vc"].double()
        page = case["page"]
        kc[s["slots"] // page, s["slots"] % page] = one(s["k"], s["k_w"])
        vc[s["slots"] // page, s["slots"] % page] = s["v"].double()
        return one(s["q"], s["q_w"]), kc, vc
    if op == "keep_drafted":
        kc, vc = s["kc"].double(), s["vc"].double()
        page, table, path, lens = case["page"], s["table"].tolist(), s["path"].tolist(), s["lens"].tolist()
        for b, l in enumerate(lens):
            for i, p in enumerate(path[b]):
                (sp, so), (dp, do) = divmod(l + p, page), divmod(l + i, page)
                for c in (kc, vc):
                    c[:, table[b][dp], do] = c[:, table[b][sp], so]
        return kc, vc
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device=s["q"].device)
    first = 0
    for b, (l, n) in enumerate(zip(_spread(case, case["cached"]), _news(case))):
        at = torch.arange(l + n, device=out.device)
        pages = s["table"][b].long()[at // page]
        j = torch.arange(n, device=out.device)
        if s["mask"] is None:
            sees = j[:, None] >= j
        else:
            sees = (s["mask"][first:first + n][:, j // 64] >> (j % 64)) % 2 == 1
        bias = torch.zeros(n, l + n, dtype=torch.float64, device=out.device)
        bias[:, l:].masked_fill_(~sees, -math.inf)
        for h in range(hkv):
            k, v = (c[pages, at % page, h].double() for c in (s["kc"], s["vc"]))
            for g in range(h * hq // hkv, (h + 1) * hq // hkv):
                score = s["q"][first:first + n, g].double() @ k.T / math.sqrt(dim) + bias
                lse[first:first + n, g] = torch.logsumexp(score, -1)
                out[first:first + n, g] = torch.softmax(score, -1) @ v
        first += n
    return (out, lse) if case["lse"] else out
