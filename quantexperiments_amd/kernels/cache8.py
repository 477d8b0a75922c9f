"""A paged cache of keys and values held in 8 bits: new tokens put into it, attention over it, and the accepted path of a draft moved in it.

The cache is four tensors of a layer (or, with one more dimension in front, of all layers):
  k_cache, v_cache  torch.float8_e4m3fn    [pages, slots per page, key heads, D]: codes
  k_scale, v_scale  torch.float8_e8m0fnu   [pages, blocks per page, key heads]: a power of two for each block of tokens and head
and an element is code * scale.  A page has a multiple of 16 slots in each of its blocks; D is a multiple of 16 up to 256.  The scale of a block fits
its largest element, and grows with it.  Attention reads exactly what is held, in half the bytes of a 16-bit cache.  What is held is off by up to 2^-4 of an element of 2^-6 of its
block's scale or more (an element alone in setting its scale is 224 to 448 times that), and of a smaller one by up to 2^-10 of the scale, which may be all of it.  Whenever the scale grows,
elements that then lie below 2^-6 of it are rounded again, by up to 2^-10 of it once more.  Scales do not fall: a drafted token with a large element raises the scale of the
block it lies in, and whether it is kept or not, the small elements of cached tokens there lose those bits for good, and the block's later tokens are held at that scale.
Tables, lengths and the new tokens' rows are those of `tree_attention`; everything launches on torch's current stream, reads no device value on the host and can be
captured.  Nothing of the reference is like it: its engine keeps its cache in 16 bits (reference shapequant/kernels/decode_e2e.py:142-225)."""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .._lib import SqAttention, SqCache8
from .attention import _clash, _extent, _fits, _heads3, _no_grad, _on_gpu, _part, _rows2, _vector

DTYPES = (torch.float16, torch.bfloat16)


def _near(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the bytes between the first and the last of both meet."""
    return a.numel() > 0 and b.numel() > 0 and _extent(a)[0] < _extent(b)[1] and _extent(b)[0] < _extent(a)[1]


def _cache8(who: str, k: torch.Tensor, v: torch.Tensor, ks: torch.Tensor, vs: torch.Tensor, dims=(4,), written: bool = False) -> SqCache8:
    """sq_cache8 of the last dimensions of the four tensors."""
    if k.dim() not in dims or k.shape != v.shape or k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
        raise ValueError(f"{who}: caches must be two float8_e4m3fn tensors [pages, slots, heads, D]: got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    if ks.dim() != k.dim() - 1 or ks.shape != vs.shape or ks.dtype != torch.float8_e8m0fnu or vs.dtype != torch.float8_e8m0fnu or \
            ks.shape[:-2] != k.shape[:-3] or ks.shape[-1] != k.shape[-2]:
        raise ValueError(f"{who}: scales must be two float8_e8m0fnu tensors [pages, blocks, heads] of the caches {tuple(k.shape)}: got {tuple(ks.shape)} {ks.dtype} and "
                         f"{tuple(vs.shape)} {vs.dtype}")
    page, blocks = k.shape[-3], ks.shape[-2]
    if page < 1 or blocks < 1 or page % blocks:
        raise ValueError(f"{who}: {blocks} blocks in a page of {page} slots")
    _fits(who, *k.shape)
    for t in (k, v):
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{who}: the elements of a head must be neighbours in the caches (strides {t.stride()})")
    if written:
        every = (k, v, ks, vs)
        if any(s == 0 and n > 1 for t in every for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"{who}: a cache that is written must not be expanded")
        if any(a.numel() and a.data_ptr() == b.data_ptr() for i, a in enumerate(every) for b in every[:i]):
            raise ValueError(f"{who}: two of the caches and scales are one tensor")
    return SqCache8(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *k.stride()[-4:-1], *v.stride()[-4:-1], *ks.stride()[-3:], *vs.stride()[-3:],
                    k.shape[-4], page, blocks, k.shape[-2], k.shape[-1])


def _sequences(who: str, n: int, table, lens, starts, most_new) -> tuple:
    """(sequences, most new tokens of one) of n tokens."""
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
    return b, most_new


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def put_tokens8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, table: torch.Tensor,
                lens: torch.Tensor, starts: torch.Tensor | None = None, *, most_new: int | None = None) -> None:
    """Keys and values k, v [N, Hk, D] (fp16 / bf16, 16-byte aligned heads, any strides) of new tokens put into an 8-bit cache, in place: token t of sequence b, row
    starts[b] + t (int32 [B + 1]; None: N / B each), goes to slot lens[b] + t (sq_put_tokens8); lens (int32 [B]) is left as it is.  most_new: at most so many of a sequence (default:
    N; a bound near the truth makes the launch smaller).  A block's scale is the smallest power of two by which its largest new element is not beyond 448, and not less than the one it has where it
    holds tokens before lens[b], which are scaled to it when it grows.  Elements that are not finite become NaN; larger magnitudes than 61,440 in fp16 (1.875 * 2^127 in bf16) are held as that, so that what is
read is finite in the tokens' type.  Sequences must not share pages that are written."""
    done = _lib.native().put_tokens8(k, v, k_cache, v_cache, k_scale, v_scale, table, lens, starts, most_new)
    if done <= 0:
        if done:
            _lib.check(done)
        return
    who = "put_tokens8"
    _heads3(who, "k", k)
    n, h, d = k.shape
    _heads3(who, "v", v, (n, h, d))
    _no_grad(who, k, v, k_cache, v_cache, k_scale, v_scale)
    dev = k.device
    _on_gpu(who, dev, v=v, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, table=table, lens=lens, starts=starts)
    if k.dtype not in DTYPES or v.dtype != k.dtype:
        raise ValueError(f"{who}: k is {k.dtype}, v {v.dtype} (fp16 or bf16)")
    cache = _cache8(who, k_cache, v_cache, k_scale, v_scale, written=True)
    if tuple(k_cache.shape[2:]) != (h, d):
        raise ValueError(f"{who}: caches {tuple(k_cache.shape)} for keys {tuple(k.shape)}")
    b, most_new = _sequences(who, n, table, lens, starts, most_new)
    for c in (k_cache, v_cache, k_scale, v_scale):
        if _near(c, k) or _near(c, v):
            raise ValueError(f"{who}: a cache overlaps another operand")
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().sq_put_tokens8(ctypes.byref(_part(k, None)), ctypes.byref(_part(v, None)), n, _lib.DTYPES[k.dtype], ctypes.byref(cache), table.data_ptr(),
                                             _ld(table), table.shape[1], lens.data_ptr(), None if starts is None else starts.data_ptr(), b, most_new, _lib.stream_ptr(dev)))


def tree_attention8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                    starts: torch.Tensor | None = None, *, most_new: int | None = None, mask: torch.Tensor | None = None, scale: float | None = None,
                    out: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
    """`tree_attention` over an 8-bit cache: attention of new tokens q [N, Hq, D] (fp16 / bf16) over lens[b] cached tokens of each sequence and, in the slots behind them, its new
    tokens' keys and values, as put_tokens8 puts them there (sq_tree_attention8).  Rows, starts, most_new, mask, scale, out, lse and what a token sees are as there.  Keys and
    values are what the cache holds, code * scale, exactly in bf16; in fp16 as far as fp16 has them, which is all that put_tokens8 made of fp16 tokens.  Lengths are on the device, so work is dealt out
for sequences that fill their table rows: short ones under a wide table take several times as long, and table[:, :n], n pages at least of the longest one, costs nothing."""
    done = _lib.native().tree_attention8(q, k_cache, v_cache, k_scale, v_scale, table, lens, starts, most_new, mask, scale, out, lse)
    if type(done) is not int:
        return done
    if done < 0:
        _lib.check(done)
    who = "tree_attention8"
    _heads3(who, "q", q)
    _no_grad(who, q, k_cache, v_cache, k_scale, v_scale, out, lse)
    n, hq, d = q.shape
    dev = q.device
    _on_gpu(who, dev, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, table=table, lens=lens, starts=starts, mask=mask, out=out, lse=lse)
    cache = _cache8(who, k_cache, v_cache, k_scale, v_scale)
    if q.dtype not in DTYPES or k_cache.shape[3] != d or k_cache.shape[2] < 1 or hq < 1 or hq % k_cache.shape[2]:
        raise ValueError(f"{who}: q {tuple(q.shape)} {q.dtype} (fp16 or bf16) and caches {tuple(k_cache.shape)}")
    b, most_new = _sequences(who, n, table, lens, starts, most_new)
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
        if any(_near(c, out) for c in (k_cache, v_cache, k_scale, v_scale)):
            raise ValueError(f"{who}: out overlaps a cache")
        if any(s == 0 and m > 1 for m, s in zip(out.shape, out.stride())):
            raise ValueError(f"{who}: out must not be expanded")
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (n, hq) or not lse.is_contiguous()):
        raise ValueError(f"{who}: lse must be contiguous fp32 [{n}, {hq}]")
    # (a mask without words has no address of its own, and none would mean no mask: any other does, nothing is read there)
    a = SqAttention(q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), table.data_ptr(), lens.data_ptr(),
                    None if starts is None else starts.data_ptr(), None if mask is None else mask.data_ptr() or lens.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                    _ld(table), 0 if mask is None else _ld(mask), n, b, most_new, hq, table.shape[1], 0 if mask is None else mask.shape[1], scale)
    L, dt = _lib.lib(), _lib.DTYPES[q.dtype]
    with torch.cuda.device(dev):
        need = L.sq_tree_attention8_workspace_bytes(ctypes.byref(a), ctypes.byref(cache), dt)
        # (a buffer of the call's own: streams and captured graphs run side by side)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(L.sq_tree_attention8(ctypes.byref(a), ctypes.byref(cache), dt, None if ws is None else ws.data_ptr(), need, _lib.stream_ptr(dev)))
    return out


def keep_drafted8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, path: torch.Tensor,
                  counts: torch.Tensor) -> None:
    """`keep_drafted` in 8-bit caches [pages, slots, heads, D] of one layer or [layers, pages, slots, heads, D] of all: new token path[b, i] (int32 [B, m], ascending) of sequence
    b, i < counts[b] (int32 [B]), moves from slot lens[b] + path[b, i] to slot lens[b] + i (sq_keep_drafted8).  A block that tokens move to takes the largest scale of theirs and, where it
    holds cached tokens, its own (which drafts that are not kept may have raised).  Entries from the first one on that does not ascend or has no slot are ignored; lens is left as it is.  Sequences must not
    share the pages that are written."""
    done = _lib.native().keep_drafted8(k_cache, v_cache, k_scale, v_scale, table, lens, path, counts)
    if done <= 0:
        if done:
            _lib.check(done)
        return
    who = "keep_drafted8"
    _no_grad(who, k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _on_gpu(who, dev, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, table=table, lens=lens, path=path, counts=counts)
    cache = _cache8(who, k_cache, v_cache, k_scale, v_scale, (4, 5), written=True)
    b = lens.shape[0] if lens.dim() == 1 else -1
    _vector(who, "lens", lens, b, torch.int32)
    _vector(who, "counts", counts, b, torch.int32)
    _rows2(who, "table", table, b, torch.int32)
    _rows2(who, "path", path, b, torch.int32)
    layers = k_cache.shape[0] if k_cache.dim() == 5 else 1
    step = [t.stride(0) if k_cache.dim() == 5 else 0 for t in (k_cache, v_cache, k_scale, v_scale)]
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().sq_keep_drafted8(ctypes.byref(cache), layers, *step, table.data_ptr(), _ld(table), table.shape[1], lens.data_ptr(), path.data_ptr(), _ld(path),
                                               path.shape[1], counts.data_ptr(), b, _lib.stream_ptr(dev)))
