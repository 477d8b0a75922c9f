"""The life of a paged cache's pages, in caches of any type (16-bit ones of `tree_attention`, 8-bit ones of `tree_attention8` with their scales), of one layer or of all.

Which pages a sequence has is in its row of the table and its length alone, both on the device: there is no list of free pages and no count of users to keep in step.
`fork_pages` makes the tables of a batch whose sequences go on where others are (several samples of a prompt, the beams of a step): whole pages are
shared, and of the last one the slots in use are copied to a page of the new sequence's own.  `compact_pages` frees what no sequence uses: pages in use move
to the front of the pool, and the first so many are the ones in use.  A sequence is ended by leaving its row out, or by a length of zero.
Both launch on torch's current stream, read no device value on the host and can be captured.  The reference keeps one contiguous cache per sequence and
has nothing like them (reference shapequant/kernels/decode_e2e.py:142-225)."""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .._lib import SqPlane
from .attention import _clash, _fits, _no_grad, _on_gpu, _rows2, _vector
from .cache8 import _ld, _near


def _planes(who: str, k, v, ks, vs) -> tuple:
    """(array of sq_plane, layers, pages, slots of a page) of a pair of caches and, in pairs too, their scales."""
    if k.dim() not in (4, 5) or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"{who}: caches must be two tensors [pages, slots, heads, D] or [layers, pages, slots, heads, D] of one type: got {tuple(k.shape)} {k.dtype} and "
                         f"{tuple(v.shape)} {v.dtype}")
    if (ks is None) != (vs is None):
        raise ValueError(f"{who}: k_scale and v_scale come together")
    every = [k, v]
    if ks is not None:
        if ks.dim() != k.dim() - 1 or ks.shape != vs.shape or ks.dtype != vs.dtype or ks.shape[:-2] != k.shape[:-3]:
            raise ValueError(f"{who}: scales must be two tensors [pages, blocks, heads], with the caches' layers: got {tuple(ks.shape)} {ks.dtype} and {tuple(vs.shape)} {vs.dtype}")
        every += [ks, vs]
    layers, pages, page = (k.shape[0] if k.dim() == 5 else 1), k.shape[-4], k.shape[-3]
    _fits(who, *k.shape)
    if page < 1:
        raise ValueError(f"{who}: pages without slots")
    out = (SqPlane * len(every))()
    for i, t in enumerate(every):
        size, code = t.element_size(), i < 2
        rows, heads = (t.shape[-3], t.shape[-2]) if code else (t.shape[-2], t.shape[-1])
        if rows < 1 or page % rows:
            raise ValueError(f"{who}: {rows} blocks in a page of {page} slots")
        if code and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{who}: the elements of a head must be neighbours in the caches (strides {t.stride()})")
        if any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"{who}: a cache that is written must not be expanded (strides {t.stride()})")
        if any(t.numel() and t.data_ptr() == o.data_ptr() for o in every[:i]):
            raise ValueError(f"{who}: two of the caches and scales are one tensor")
        at = t.dim() - (4 if code else 3)
        bytes_ = [t.stride(at + j) * size for j in range(3)]
        out[i] = SqPlane(t.data_ptr(), t.stride(0) * size if at else 0, *bytes_, rows, heads, (t.shape[-1] if code else 1) * size)
    return out, layers, pages, page


def _batch(who: str, table, lens) -> int:
    b = lens.shape[0] if lens.dim() == 1 else -1
    _vector(who, "lens", lens, b, torch.int32)
    _rows2(who, "table", table, b, torch.int32)
    return b


def _new(who: str, name: str, t, shape, *olds) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or (t.dim() == 1 and not t.is_contiguous()):
        raise ValueError(f"{who}: {name} must be int32 {tuple(shape)}: got {tuple(t.shape)} {t.dtype}")
    if t.dim() == 2:
        _rows2(who, name, t, shape[0], torch.int32)
    # (columns of one tensor's rows are told apart)
    if any(_clash(t[:, None], o[:, None]) if t.dim() == o.dim() == 2 else _near(t, o) for o in olds):
        raise ValueError(f"{who}: {name} overlaps another operand")


def fork_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, parent: torch.Tensor, pages: torch.Tensor, *,
               k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, out_table: torch.Tensor | None = None,
               out_lens: torch.Tensor | None = None) -> tuple:
    """(table, lens) of a batch of R sequences whose i-th goes on where sequence parent[i] (int32 [R]) of the batch table (int32 [B, W]), lens (int32 [B]) is (sq_fork_pages).  Where pages[i]
    (int32 [R]) is a free page, the row is the parent's whole pages and, in place of the page that slot lens[parent[i]] is in, pages[i], to which that page's slots in use are
    copied in the caches (and scales) of all layers; the rest of the row is -1.  Where it is negative, the row is the parent's: it goes on in the same
    pages, which one sequence may.  The pages given are distinct and no sequence's.  out_table [R, W], out_lens [R]: memory apart from the old ones (default: new)."""
    done = _lib.native().fork_pages(k_cache, v_cache, table, lens, parent, pages, k_scale, v_scale, out_table, out_lens)
    if type(done) is not int:
        return done
    if done < 0:
        _lib.check(done)
    who = "fork_pages"
    _no_grad(who, k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _on_gpu(who, dev, v_cache=v_cache, table=table, lens=lens, parent=parent, pages=pages, k_scale=k_scale, v_scale=v_scale, out_table=out_table, out_lens=out_lens)
    planes, layers, n, page = _planes(who, k_cache, v_cache, k_scale, v_scale)
    b = _batch(who, table, lens)
    r = parent.shape[0] if parent.dim() == 1 else -1
    _vector(who, "parent", parent, r, torch.int32)
    _vector(who, "pages", pages, r, torch.int32)
    w = table.shape[1]
    if out_table is None:
        out_table = torch.empty(r, w, dtype=torch.int32, device=dev)
    if out_lens is None:
        out_lens = torch.empty(r, dtype=torch.int32, device=dev)
    _new(who, "out_table", out_table, (r, w), table, lens, parent, pages, out_lens)
    _new(who, "out_lens", out_lens, (r,), table, lens, parent, pages)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().sq_fork_pages(planes, len(planes), layers, n, page, table.data_ptr(), _ld(table), w, lens.data_ptr(), b, parent.data_ptr(), pages.data_ptr(), r,
                                            out_table.data_ptr(), _ld(out_table), out_lens.data_ptr(), _lib.stream_ptr(dev)))
    return out_table, out_lens


def compact_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                  v_scale: torch.Tensor | None = None, out_table: torch.Tensor | None = None) -> tuple:
    """(table, used): the pages that hold none of the first lens[b] slots (int32 [B]; lengths, or more where pages ahead of them are kept) of any sequence of table (int32 [B, W]) are
    freed, and the others moved to the front of the pool in the caches (and scales) of all layers (sq_compact_pages).  With used[0] (int32 [1]) pages in use, the ones behind page
    used[0] move to the lowest free ones, in order, and pages used[0] .. are free.  The new table has -1 behind a sequence's pages; sequences may share pages.  out_table [B, W]: memory apart
    from the old one (default: new).  The pages that moved hold what they held until they are used again.  Up to 2^20 pages."""
    done = _lib.native().compact_pages(k_cache, v_cache, table, lens, k_scale, v_scale, out_table)
    if type(done) is not int:
        return done
    if done < 0:
        _lib.check(done)
    who = "compact_pages"
    _no_grad(who, k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _on_gpu(who, dev, v_cache=v_cache, table=table, lens=lens, k_scale=k_scale, v_scale=v_scale, out_table=out_table)
    planes, layers, n, page = _planes(who, k_cache, v_cache, k_scale, v_scale)
    b, w = _batch(who, table, lens), table.shape[1]
    if out_table is None:
        out_table = torch.empty(b, w, dtype=torch.int32, device=dev)
    _new(who, "out_table", out_table, (b, w), table, lens)
    used = torch.empty(1, dtype=torch.int32, device=dev)
    L = _lib.lib()
    with torch.cuda.device(dev):
        need = L.sq_compact_pages_workspace_bytes(n)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)          # (of the call's own: streams and captured graphs run side by side)
        _lib.check(L.sq_compact_pages(planes, len(planes), layers, n, page, table.data_ptr(), _ld(table), w, lens.data_ptr(), b, out_table.data_ptr(), _ld(out_table),
                                      used.data_ptr(), ws.data_ptr(), need, _lib.stream_ptr(dev)))
    return out_table, used
