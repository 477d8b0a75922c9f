"""8-bit caches in 64 bits, by their definition: codes, scales, and what the calls on them leave.  CPU tensors, written without the package."""

import math

import torch

CODES = torch.tensor([(-1.0) ** (b >> 7) * ((b & 7) / 8 * 2.0 ** -6 if not b >> 3 & 15 else math.nan if b & 127 == 127 else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3 & 15) - 7))
                      for b in range(256)], dtype=torch.float64)
POSITIVE = CODES[:127]                                       # ascending
MOST = {torch.bfloat16: 1.875 * 2.0 ** 127, torch.float16: 1.875 * 2.0 ** 15}


def code_values(codes):
    return CODES[codes.view(torch.uint8).long()]


def nearest(x):
    """Codes (bytes) nearest to x (64 bits, at most 448 in magnitude), ties to the even code; NaN: 127."""
    a = x.nan_to_num(0.0).abs()
    hi = torch.searchsorted(POSITIVE, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = POSITIVE[hi] - a, a - POSITIVE[lo]
    b = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.where(x.isnan(), 127, b + 128 * (torch.signbit(x)).long()).to(torch.uint8)


def same_codes(a, b):
    """Equal bytes, any NaN like any other."""
    a, b = (t.contiguous().view(torch.uint8) for t in (a, b))
    return torch.equal(torch.where(a & 127 == 127, 127, a.int()), torch.where(b & 127 == 127, 127, b.int()))


def smallest(a):
    """The smallest exponent from -100 on with a <= 448 * 2 ** e."""
    e = -100
    while a > 448 * 2.0 ** e:
        e += 1
    return e


def rescaled(codes, down):
    return nearest(code_values(codes) * 2.0 ** -down)


class Pool:
    """One layer's cache on the CPU: bytes of codes [2, pages, page, heads, dim] and of scales [2, pages, blocks, heads] of keys and values."""

    def __init__(self, pages, page, blocks, heads, dim, g):
        b = torch.randint(0, 254, (2, pages, page, heads, dim), generator=g)
        self.codes = (b + (b >= 127)).to(torch.uint8)
        self.scales = torch.randint(115, 125, (2, pages, blocks, heads), generator=g).to(torch.uint8)
        self.page, self.size = page, page // blocks

    def copy(self):
        p = object.__new__(Pool)
        p.codes, p.scales, p.page, p.size = self.codes.clone(), self.scales.clone(), self.page, self.size
        return p

    def device(self, permute=None):
        """(k_cache, v_cache, k_scale, v_scale) on the GPU; permute: the order of a page's dimensions in memory."""
        out = []
        for t, kind in ((self.codes, torch.float8_e4m3fn), (self.scales, torch.float8_e8m0fnu)):
            for i in range(2):
                x = t[i]
                if permute and x.dim() == 4:
                    x = x.permute(permute).contiguous().permute([permute.index(j) for j in range(4)]).cuda()
                out.append((x if x.is_cuda else x.cuda().clone()).view(kind))
        return tuple(out)

    def values(self):
        """[2, pages, page, heads, dim] in 64 bits."""
        return CODES[self.codes.long()] * torch.pow(2.0, self.scales.double() - 127).repeat_interleave(self.size, 2)[..., None]

    def assert_same(self, kc, vc, ks, vs):
        for i, (c, s) in enumerate(((kc, ks), (vc, vs))):
            assert torch.equal(s.cpu().view(torch.uint8), self.scales[i]), ("scales of " + "kv"[i], (s.cpu().view(torch.uint8) != self.scales[i]).nonzero()[:4])
            assert same_codes(c.cpu(), self.codes[i]), ("codes of " + "kv"[i], (c.cpu().view(torch.uint8) != self.codes[i]).nonzero()[:4])

    def spot(self, table, b, slot):
        """(page, slot in page) or None."""
        j = slot // self.page
        if j >= table.shape[1] or not 0 <= int(table[b, j]) < self.codes.shape[1]:
            return None
        return int(table[b, j]), slot % self.page

    def put(self, k, v, table, lens, starts, most_new=None):
        for i, x in enumerate((k, v)):
            top = MOST[x.dtype]
            d = x.double()
            d = torch.where(d.abs() < math.inf, d.clamp(-top, top), math.nan)
            for b, l in enumerate(lens):
                rows = d[starts[b]:starts[b + 1]][:most_new]
                at = max(l, 0)
                end = at + len(rows)
                while at < end:
                    stop = min(at // self.size * self.size + self.size, end)
                    spot = self.spot(table, b, at)
                    if spot:
                        p, o = spot
                        new = rows[at - max(l, 0):stop - max(l, 0)]
                        for h in range(d.shape[1]):
                            e = smallest(float(new[:, h].nan_to_num(0.0).abs().max()))
                            held = o % self.size
                            was = int(self.scales[i, p, o // self.size, h]) - 127
                            if held and e > was:
                                old = self.codes[i, p, o - held:o, h]
                                self.codes[i, p, o - held:o, h] = rescaled(old, e - was)
                            e = max(e, was) if held else e
                            self.codes[i, p, o:o + len(new), h] = nearest(new[:, h] * 2.0 ** -e)
                            self.scales[i, p, o // self.size, h] = e + 127
                    at = stop

    def keep(self, table, lens, path, counts):
        old = self.copy()
        for b, l in enumerate(lens):
            l = max(l, 0)
            moves = []
            for i in range(min(int(counts[b]), path.shape[1])):
                x = int(path[b, i])
                src, dst = (self.spot(table, b, l + x) if x >= 0 else None), self.spot(table, b, l + i)
                if x < 0 or (i and x <= int(path[b, i - 1])) or src is None or dst is None:
                    break
                moves.append((src, dst))
            blocks = {}
            for i, (src, dst) in enumerate(moves):
                blocks.setdefault((l + i) // self.size, []).append((src, dst))
            for first, mine in blocks.items():
                p, o = mine[0][1]
                held = o % self.size if first * self.size < l else 0
                for i in range(2):
                    for h in range(self.codes.shape[3]):
                        e = max(int(old.scales[i, sp, so // self.size, h]) for (sp, so), _ in mine)
                        if held:
                            was = int(old.scales[i, p, o // self.size, h])
                            e = max(e, was)
                            if e > was:
                                self.codes[i, p, o - held:o, h] = rescaled(old.codes[i, p, o - held:o, h], e - was)
                        for (sp, so), (dp, do) in mine:
                            down = e - int(old.scales[i, sp, so // self.size, h])
                            row = old.codes[i, sp, so, h]
                            self.codes[i, dp, do, h] = rescaled(row, down) if down else row
                        self.scales[i, p, o // self.size, h] = e


def table_for(slots, page, g, spare=3, width=0):
    """A table of scattered pages for that many slots each, entries behind them outside the cache, and the number of pages."""
    need = [-(-s // page) for s in slots]
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    table = torch.full((len(slots), max(max(need, default=0) + 1, width)), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, len(order), order[at:]
