"""What a decoder layer does between its q|k|v product and its o product: the heads normalised and rotated by their tokens'
positions, keys and values put in a paged cache, attention of new tokens (one, a chunk, or a tree of drafts) over it, and the accepted
path of a draft moved behind the cached tokens.

A paged cache is a pair of tensors [pages, slots per page, key heads, D] (any strides, neighbouring elements; a contiguous cache
[sequences, slots, heads, D] is one with a page per sequence) and a table int32 [sequences, pages of a sequence]: slot s of
sequence b is slot s % page of page table[b, s // page].

Everything launches on torch's current stream, allocates from torch and reads no device value on the host, so calls can be captured into HIP graphs;
what lengths, tables and masks hold may change between replays.  The kernels index with them and cut off what lies outside the
buffers, as include/sqhip.h says call by call.  Inference only: tensors that require a gradient are refused where one would be recorded, and
tensors with a tangent (forward mode).
The reference's engine has these steps as rope_cache, attn_rope and attn (reference shapequant/kernels/decode_e2e.py:142-225) and
attn_prep (shapequant/kernels/qwen35_kernels.py:50-190), for single tokens and a contiguous cache."""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._lib import SqAttention, SqCache, SqHeads, SqRotation


def rotary_freqs(rot: int, base: float = 10000.0, scaling: dict | None = None, device="cuda") -> tuple:
    """(freqs, scale) for `rotary`: radians per position of each of the rot / 2 pairs, float64 on `device`, and the factor on rotated
    values.  scaling: None, or how a context longer than the trained one is reached, {"type": ..., "factor": f, ...}:
      linear  all frequencies divided by f
      ntk     the base raised so that the slowest pair turns f times slower and the fastest as before
      yarn    pairs that turn more than beta_fast (32) times in `original` positions as they are, fewer than beta_slow (1) divided by
              f, a ramp over the pairs in between; scale 0.1 ln f + 1 unless "scale" gives one
      bands   wavelengths below original / high (4) as they are, above original / low (1) divided by f, blended in between"""
    if rot < 0 or rot % 2:
        raise ValueError(f"rotary_freqs: {rot} elements are not pairs")
    kind = None if scaling is None else scaling.get("type")
    f = 1.0 if scaling is None else float(scaling["factor"])
    if not (f > 0 and math.isfinite(f) and base > 0):
        raise ValueError(f"rotary_freqs: base {base}, factor {f}")
    if kind == "ntk":
        if rot < 4:
            raise ValueError("rotary_freqs: ntk needs two pairs")
        base = base * f ** (rot / (rot - 2))
    i = torch.arange(rot // 2, dtype=torch.float64)
    w = base ** (-2.0 * i / max(rot, 1))
    scale = 1.0
    if kind == "linear":
        w = w / f
    elif kind == "yarn":
        n = float(scaling["original"])
        pair = lambda turns: rot * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))     # the pair that turns so often in n positions
        lo = max(math.floor(pair(scaling.get("beta_fast", 32.0))), 0)
        hi = min(math.ceil(pair(scaling.get("beta_slow", 1.0))), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        w = w / f * ramp + w * (1 - ramp)
        scale = float(scaling.get("scale", 0.1 * math.log(f) + 1 if f > 1 else 1.0))
    elif kind == "bands":
        n, lo, hi = float(scaling["original"]), float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        keep = ((n * w / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
        w = keep * w + (1 - keep) * w / f
    elif kind not in (None, "ntk"):
        raise ValueError(f"rotary_freqs: scaling type {kind!r}")
    return w.to(device), scale


# ------------------------------------------------------------------ arguments

def _no_grad(who: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{who} has no autograd formula: call it under torch.no_grad()")
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{who} has no formula for tangents (forward mode): pass the primal tensors")


def _on_gpu(who: str, dev, **tensors) -> None:
    if dev.type != "cuda":
        raise ValueError(f"{who}: tensors must be on the GPU (there is no CPU path)")
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{who}: {name} is on {t.device}, not on {dev}")


def _fits(who: str, *sizes: int) -> None:
    if max(sizes) > 2 ** 31 - 1:
        raise ValueError(f"{who}: sizes beyond 32 bits: {sizes}")


def _heads3(who: str, name: str, t: torch.Tensor, shape=None) -> None:
    if t.dim() != 3 or t.dtype not in _lib.DTYPES or (t.shape[2] > 1 and t.stride(2) != 1) or (shape is not None and tuple(t.shape) != tuple(shape)):
        want = "[tokens, heads, D]" if shape is None else str(tuple(shape))
        raise ValueError(f"{who}: {name} must be {want}, fp16 / bf16 / fp32, with neighbouring elements: got {tuple(t.shape)} {t.dtype}, strides {t.stride()}")
    _fits(who, *t.shape)


def _vector(who: str, name: str, t: torch.Tensor, n: int, *dtypes) -> None:
    if t.dim() != 1 or t.shape[0] != n or t.dtype not in dtypes or not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be a contiguous {' / '.join(str(d) for d in dtypes)} vector of {n}: got {tuple(t.shape)} {t.dtype}")


def _rows2(who: str, name: str, t: torch.Tensor, n: int, dtype) -> None:
    if t.dim() != 2 or t.shape[0] != n or t.dtype != dtype or (t.shape[1] > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{who}: {name} must be {dtype} with {n} rows and unit column stride: got {tuple(t.shape)} {t.dtype}, strides {t.stride()}")
    _fits(who, *t.shape)


def _extent(t: torch.Tensor) -> tuple:
    lo = hi = t.data_ptr()
    for n, s in zip(t.shape, t.stride()):
        if s > 0:
            hi += (n - 1) * s * t.element_size()
        else:
            lo += (n - 1) * s * t.element_size()
    return lo, hi + t.element_size()


def _clash(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [tokens, heads, D] views may share an element.  Columns of one stacked product lie inside each other's extents; they
    are told apart by their places in its rows."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (alo, ahi), (blo, bhi) = _extent(a), _extent(b)
    if ahi <= blo or bhi <= alo:
        return False
    row = a.stride(0)
    width = lambda t: (t.shape[1] - 1) * t.stride(1) + t.shape[2]
    if a.element_size() != b.element_size() or row != b.stride(0) or row <= 0 or a.stride(1) < 0 or b.stride(1) < 0 or (blo - alo) % a.element_size():
        return True
    at = (blo - alo) // a.element_size() % row
    return not (at >= width(a) and at + width(b) <= row)


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and all(x == y or n <= 1 for n, x, y in zip(a.shape, a.stride(), b.stride()))


def _apart(who: str, name: str, out: torch.Tensor, own, *others) -> None:
    if own is not None and not _same(out, own) and _clash(out, own):
        raise ValueError(f"{who}: {name} overlaps its input without being it")
    for t in others:
        if t is not None and _clash(out, t):
            raise ValueError(f"{who}: {name} overlaps another operand")


def _rotation(who: str, positions, freqs, n: int, dim: int, interleaved, scale, inverse, dev) -> SqRotation:
    _vector(who, "positions", positions, n, torch.int64, torch.int32)
    _vector(who, "freqs", freqs, freqs.numel(), torch.float64)
    if 2 * freqs.numel() > dim:
        raise ValueError(f"{who}: {freqs.numel()} pairs in heads of {dim}")
    _on_gpu(who, dev, positions=positions, freqs=freqs)
    return SqRotation(freqs.data_ptr(), positions.data_ptr(), freqs.numel(), positions.dtype == torch.int64, bool(interleaved), bool(inverse), float(scale))


def _part(x: torch.Tensor, out, w=None) -> SqHeads:
    o = x if out is None else out
    return SqHeads(x.data_ptr(), None if out is None else out.data_ptr(), None if w is None else w.data_ptr(), x.stride(0), x.stride(1), o.stride(0), o.stride(1),
                   x.shape[1])


def _cache(who: str, k: torch.Tensor, v: torch.Tensor, written: bool = False) -> SqCache:
    """sq_cache of the last four dimensions of a pair of caches."""
    if k.dim() not in (4, 5) or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _lib.DTYPES or v.device != k.device:
        raise ValueError(f"{who}: caches must be two tensors [pages, slots, heads, D] of one type: got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    for t in (k, v):
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{who}: the elements of a head must be neighbours in the caches (strides {t.stride()})")
        if written and any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"{who}: a cache that is written must not be expanded (strides {t.stride()})")
    _fits(who, *k.shape)
    if k.shape[-3] < 1:
        raise ValueError(f"{who}: pages without slots")
    if written and k.numel() and _extent(k)[0] < _extent(v)[1] and _extent(v)[0] < _extent(k)[1] and _same(k, v):
        raise ValueError(f"{who}: keys and values are one tensor")
    return SqCache(k.data_ptr(), v.data_ptr(), *k.stride()[-4:-1], *v.stride()[-4:-1], k.shape[-4], k.shape[-3], k.shape[-2], k.shape[-1], _lib.DTYPES[k.dtype])


# ------------------------------------------------------------------ operators

def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, out: torch.Tensor | None = None, *, interleaved: bool = False, scale: float = 1.0,
           inverse: bool = False) -> torch.Tensor:
    """The heads x [N, H, D] (fp16 / bf16 / fp32, any strides) rotated by their tokens' positions (int64 / int32 [N]): of the first 2 P elements of
    a head, P = len(freqs), pair i turns by positions * freqs[i] radians (float64 [P], `rotary_freqs`) and is multiplied by `scale`; the pair is
    elements i and P + i, or 2i and 2i + 1 if interleaved; the other elements keep their values (sq_rotary).  out: x itself, or memory
    apart from it (default: new).  inverse turns back: the adjoint, for gradients, and the way to move rotated keys to other positions."""
    done = _lib.native().rotary(x, positions, freqs, out, interleaved, scale, inverse)
    if type(done) is not int:
        return done
    if done < 0:
        _lib.check(done)
    who = "rotary"
    _heads3(who, "x", x)
    _no_grad(who, x, freqs, out)
    n, _, d = x.shape
    dev = x.device
    _on_gpu(who, dev, out=out)
    rot = _rotation(who, positions, freqs, n, d, interleaved, scale, inverse, dev)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    else:
        _heads3(who, "out", out, x.shape)
        if out.dtype != x.dtype:
            raise ValueError(f"{who}: out is {out.dtype}, x {x.dtype}")
        _apart(who, "out", out, x)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().sq_rotary(ctypes.byref(_part(x, out)), n, d, _lib.DTYPES[x.dtype], ctypes.byref(rot), _lib.stream_ptr(dev)))
    return out


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, q_w: torch.Tensor | None = None,
                   k_w: torch.Tensor | None = None, eps: float = 1e-6, *, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                   v: torch.Tensor | None = None, k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None,
                   slots: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0, weight_offset: float = 0.0) -> tuple:
    """RMS norm of each head of q [N, Hq, D] and k [N, Hk, D] (weights q_w, k_w [D] + weight_offset; None: no norm) and the rotation of `rotary`
    in one pass, in 32 bits, rounded once (sq_qk_norm_rotary).  q_out: q itself or memory apart (default: new).  With caches, keys and v
    [N, Hk, D] go to slots (int64 / int32 [N]: page * slots per page + slot in page, distinct; tokens with a slot outside the cache, as -1, are not
    written); k_out is then optional, without caches it is new by default.  Returns (q_out, k_out or None)."""
    done = _lib.native().qk_norm_rotary(q, k, positions, freqs, q_w, k_w, eps, q_out, k_out, v, k_cache, v_cache, slots, interleaved, scale, weight_offset)
    if type(done) is not int:
        return done
    if done < 0:
        _lib.check(done)
    who = "qk_norm_rotary"
    _heads3(who, "q", q)
    n, hq, d = q.shape
    _heads3(who, "k", k, (n, k.shape[1], d) if k.dim() == 3 else (n, -1, d))
    _no_grad(who, q, k, v, q_w, k_w, freqs, q_out, k_out, k_cache, v_cache)
    dev = q.device
    _on_gpu(who, dev, k=k, v=v, q_w=q_w, k_w=k_w, q_out=q_out, k_out=k_out, k_cache=k_cache, v_cache=v_cache, slots=slots)
    if k.dtype != q.dtype:
        raise ValueError(f"{who}: k is {k.dtype}, q {q.dtype}")
    wd = None
    for name, w in (("q_w", q_w), ("k_w", k_w)):
        if w is not None:
            _vector(who, name, w, d, *_lib.DTYPES)
            if wd is not None and w.dtype != wd:
                raise ValueError(f"{who}: q_w and k_w differ in type")
            wd = w.dtype
    rot = _rotation(who, positions, freqs, n, d, interleaved, scale, False, dev)
    cached = k_cache is not None
    if any((t is not None) != cached for t in (v_cache, v, slots)):
        raise ValueError(f"{who}: k_cache, v_cache, v and slots come together")
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if k_out is None and not cached:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=dev)
    for name, t, own, others in (("q_out", q_out, q, (k, v, k_out)), ("k_out", k_out, k, (q, v))):
        if t is not None:
            _heads3(who, name, t, own.shape)
            if t.dtype != q.dtype:
                raise ValueError(f"{who}: {name} is {t.dtype}, q {q.dtype}")
            _apart(who, name, t, own, *others)
    cache = None
    if cached:
        _heads3(who, "v", v, k.shape)
        _vector(who, "slots", slots, n, torch.int64, torch.int32)
        if v.dtype != q.dtype or k_cache.dtype != q.dtype or k_cache.dim() != 4 or tuple(k_cache.shape[2:]) != tuple(k.shape[1:]):
            raise ValueError(f"{who}: caches {tuple(k_cache.shape)} {k_cache.dtype} and v {v.dtype} for keys {tuple(k.shape)} {k.dtype}")
        cache = _cache(who, k_cache, v_cache, written=True)
        for c in (k_cache, v_cache):
            for t in (q, k, v, q_out, k_out):
                if t is not None and c.numel() and t.numel() and _extent(c)[0] < _extent(t)[1] and _extent(t)[0] < _extent(c)[1]:
                    raise ValueError(f"{who}: a cache overlaps another operand")
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().sq_qk_norm_rotary(
            ctypes.byref(_part(q, q_out, q_w)), ctypes.byref(_part(k, k_out, k_w)), ctypes.byref(_part(v, None)) if cached else None, n, d, _lib.DTYPES[q.dtype],
            ctypes.byref(rot), _lib.DTYPES[wd or q.dtype], float(eps), float(weight_offset), ctypes.byref(cache) if cached else None,
            slots.data_ptr() if cached else None, cached and slots.dtype == torch.int64, _lib.stream_ptr(dev)))
    return q_out, k_out


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor | None = None, *,
                   most_new: int | None = None, mask: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                   lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens q [N, Hq, D] (fp16 / bf16) over a paged cache that holds lens[b] (int32 [B]) cached tokens of each sequence and, in the
    slots behind them, its new tokens' keys and values (sq_tree_attention).  The new tokens of sequence b are rows starts[b] .. starts[b + 1] - 1
    (int32 [B + 1]; None: N / B each) of q, at most `most_new` of them (default: N; a bound near the truth makes the launch smaller, as a table that
    is not much wider than the longest sequence does: table[:, :pages] may be passed).  A token sees all cached
    tokens, and of the new ones those in its row of mask (int64 [N, words], bit j % 64 of word j / 64: new token j of its sequence; a drafted tree's
    ancestors and the token itself), or, without a mask, those up to itself (single tokens, chunks of a prompt).  Query head h reads
    key head h / (Hq / Hk).  scale: default D ** -0.5.  out [N, Hq, D]: rows that belong to no sequence are left as they are (default: new, they
    hold anything); lse: fp32 [N, Hq] contiguous, log of the sum of exponentials.  A token that sees nothing: zeros, -inf.  D: a multiple
    of 8 up to 256, heads 16-byte aligned."""
    done = _lib.native().tree_attention(q, k_cache, v_cache, table, lens, starts, most_new, mask, scale, out, lse)
    if type(done) is not int:
        return done
    if done < 0:
        _lib.check(done)
    who = "tree_attention"
    _heads3(who, "q", q)
    _no_grad(who, q, k_cache, v_cache, out, lse)
    n, hq, d = q.shape
    dev = q.device
    _on_gpu(who, dev, k_cache=k_cache, v_cache=v_cache, table=table, lens=lens, starts=starts, mask=mask, out=out, lse=lse)
    cache = _cache(who, k_cache, v_cache)
    if q.dtype == torch.float32 or k_cache.dim() != 4 or k_cache.dtype != q.dtype or k_cache.shape[3] != d or k_cache.shape[2] < 1 or hq < 1 or hq % k_cache.shape[2]:
        raise ValueError(f"{who}: q {tuple(q.shape)} {q.dtype} and caches {tuple(k_cache.shape)} {k_cache.dtype} (fp16 or bf16)")
    b = lens.shape[0] if lens.dim() == 1 else -1
    _vector(who, "lens", lens, b, torch.int32)
    _rows2(who, "table", table, b, torch.int32)
    if starts is not None:
        _vector(who, "starts", starts, b + 1, torch.int32)
    elif b == 0 or n % b:
        raise ValueError(f"{who}: {n} tokens are not as many for each of {b} sequences: pass starts")
    if most_new is None:
        most_new = n if starts is not None else n // b
    elif starts is not None:
        most_new = min(most_new, n)                          # (no sequence has more)
    if most_new < 0 or (starts is None and most_new * b != n):
        raise ValueError(f"{who}: most_new {most_new} for {n} tokens of {b} sequences")
    if mask is not None:
        _rows2(who, "mask", mask, n, torch.int64)
    if scale is None:
        scale = d ** -0.5
    if not 0 < scale < 2.3e38:                                # (times log2 e a number)
        raise ValueError(f"{who}: scale {scale}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        _heads3(who, "out", out, q.shape)
        if out.dtype != q.dtype:
            raise ValueError(f"{who}: out is {out.dtype}, q {q.dtype}")
        if _clash(out, q):
            raise ValueError(f"{who}: out overlaps q")
        for c in (k_cache, v_cache):
            if c.numel() and out.numel() and _extent(c)[0] < _extent(out)[1] and _extent(out)[0] < _extent(c)[1]:
                raise ValueError(f"{who}: out overlaps a cache")
        if any(s == 0 and m > 1 for m, s in zip(out.shape, out.stride())):
            raise ValueError(f"{who}: out must not be expanded")
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (n, hq) or not lse.is_contiguous()):
        raise ValueError(f"{who}: lse must be contiguous fp32 [{n}, {hq}]")
    # (a mask without words has no address of its own, and none would mean no mask: any other does, nothing is read there)
    a = SqAttention(q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), table.data_ptr(), lens.data_ptr(),
                    None if starts is None else starts.data_ptr(), None if mask is None else mask.data_ptr() or lens.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                    table.stride(0) if b > 1 else table.shape[1], 0 if mask is None else mask.stride(0) if n > 1 else mask.shape[1], n, b, most_new, hq, table.shape[1],
                    0 if mask is None else mask.shape[1], scale)
    L = _lib.lib()
    with torch.cuda.device(dev):
        need = L.sq_tree_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(cache))
        # (a buffer of the call's own: streams and captured graphs run side by side)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(L.sq_tree_attention(ctypes.byref(a), ctypes.byref(cache), None if ws is None else ws.data_ptr(), need, _lib.stream_ptr(dev)))
    return out


def keep_drafted(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, path: torch.Tensor, counts: torch.Tensor) -> None:
    """The accepted path of a drafted tree moved behind the cached tokens, in place, in caches [pages, slots, heads, D] of one layer or [layers, pages, slots,
    heads, D] of all: new token path[b, i] (int32 [B, m], ascending) of sequence b, i < counts[b] (int32 [B]), moves from slot lens[b] + path[b, i] to
    slot lens[b] + i (sq_keep_drafted).  Entries from the first one on that does not ascend or has no slot are ignored; lens is left as it is.  Sequences
    must not share the pages that are written."""
    done = _lib.native().keep_drafted(k_cache, v_cache, table, lens, path, counts)
    if done <= 0:
        if done:
            _lib.check(done)
        return
    who = "keep_drafted"
    _no_grad(who, k_cache, v_cache)
    dev = k_cache.device
    _on_gpu(who, dev, v_cache=v_cache, table=table, lens=lens, path=path, counts=counts)
    cache = _cache(who, k_cache, v_cache, written=True)
    b = lens.shape[0] if lens.dim() == 1 else -1
    _vector(who, "lens", lens, b, torch.int32)
    _vector(who, "counts", counts, b, torch.int32)
    _rows2(who, "table", table, b, torch.int32)
    _rows2(who, "path", path, b, torch.int32)
    stacked = k_cache.dim() == 5
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().sq_keep_drafted(
            ctypes.byref(cache), k_cache.shape[0] if stacked else 1, k_cache.stride(0) if stacked else 0, v_cache.stride(0) if stacked else 0, table.data_ptr(),
            table.stride(0) if b > 1 else table.shape[1], table.shape[1], lens.data_ptr(), path.data_ptr(), path.stride(0) if b > 1 else path.shape[1], path.shape[1],
            counts.data_ptr(), b, _lib.stream_ptr(dev)))
