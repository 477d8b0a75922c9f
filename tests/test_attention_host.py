"""What the heads and attention calls refuse, and the frequencies of their rotation.  CPU only: no kernel is launched here."""

import ctypes
import math

import pytest
import torch

from quantexperiments_amd import _lib
from quantexperiments_amd.kernels import keep_drafted, qk_norm_rotary, rotary, rotary_freqs, tree_attention

P = 0x10000                                                  # an address that is never read


def heads(**kw):
    return _lib.SqHeads(**{**dict(in_=P, out=2 * P, in_token=256, in_head=64, out_token=256, out_head=64, heads=4), **kw})


def rotation(**kw):
    return _lib.SqRotation(**{**dict(freqs=P, positions=P, pairs=32, positions_64=1, scale=1.0), **kw})


def cache(**kw):
    return _lib.SqCache(**{**dict(k=P, v=2 * P, k_page=4096, k_slot=256, k_head=64, v_page=4096, v_slot=256, v_head=64, pages=8, page=16, heads=4, dim=64,
                                  dtype=_lib.SQ_F16), **kw})


def attention(**kw):
    return _lib.SqAttention(**{**dict(q=P, out=2 * P, table=P, lens=P, q_token=512, q_head=64, out_token=512, out_head=64, ld_table=8, tokens=2, seqs=2, most_new=1, q_heads=8,
                                      max_pages=8, scale=0.125), **kw})


def test_structs_match_the_header():
    assert ctypes.sizeof(_lib.SqHeads) == 3 * 8 + 4 * 8 + 8 and _lib.SqHeads.heads.offset == 56
    assert ctypes.sizeof(_lib.SqRotation) == 2 * 8 + 4 * 4 + 8 and _lib.SqRotation.scale.offset == 32
    assert ctypes.sizeof(_lib.SqCache) == 2 * 8 + 6 * 8 + 5 * 4 + 4 and _lib.SqCache.dtype.offset == 80
    assert ctypes.sizeof(_lib.SqAttention) == 7 * 8 + 6 * 8 + 7 * 4 + 4 and _lib.SqAttention.scale.offset == 128 and _lib.SqAttention.tokens.offset == 104


def test_rotary_refuses():
    L = _lib.lib()
    call = lambda h=None, r=None, n=3, d=64, t=_lib.SQ_F16: L.sq_rotary(h or heads(), n, d, t, r or rotation(), None)
    for bad in (dict(t=3), dict(t=-1), dict(n=-1), dict(n=(1 << 30) + 1), dict(d=0), dict(d=65537), dict(h=heads(heads=-1)), dict(h=heads(in_=None)), dict(h=heads(out=None)),
                dict(r=rotation(pairs=-1)), dict(r=rotation(pairs=33)), dict(r=rotation(freqs=None)), dict(r=rotation(positions=None)),
                dict(h=heads(out_token=255)), dict(h=heads(out_head=63)), dict(h=heads(out_head=0)), dict(h=heads(out_token=0)), dict(h=heads(out=P, out_token=512))):
        assert call(**bad) == _lib.SQ_EINVAL, bad
    assert L.sq_rotary(None, 1, 64, _lib.SQ_F16, rotation(), None) == _lib.SQ_EINVAL
    assert call(n=0) == _lib.SQ_OK and call(h=heads(heads=0)) == _lib.SQ_OK


def test_qk_norm_rotary_refuses():
    L = _lib.lib()

    def call(q=None, k=None, v=None, c=None, slots=P, n=2, d=64, t=_lib.SQ_F16, wt=_lib.SQ_F16, r=None):
        return L.sq_qk_norm_rotary(q or heads(), k or heads(in_=3 * P, out=4 * P), v, n, d, t, r or rotation(), wt, 1e-6, 0.0, c, slots, 1, None)

    for bad in (dict(t=7), dict(wt=7), dict(n=-1), dict(q=heads(out=None)), dict(k=heads(out=None)), dict(v=heads()), dict(c=cache()), dict(v=heads(), c=cache(), slots=None),
                dict(v=heads(heads=3), c=cache()), dict(v=heads(), c=cache(heads=5)), dict(v=heads(), c=cache(dim=32)), dict(v=heads(), c=cache(dtype=_lib.SQ_BF16)),
                dict(v=heads(), c=cache(page=0)), dict(v=heads(), c=cache(pages=-1)), dict(v=heads(), c=cache(pages=1 << 20, page=1 << 12)), dict(v=heads(), c=cache(k=None)),
                dict(v=heads(in_=None), c=cache()), dict(r=rotation(pairs=40))):
        assert call(**bad) == _lib.SQ_EINVAL, bad
    assert call(n=0) == _lib.SQ_OK


def test_tree_attention_refuses():
    L = _lib.lib()
    call = lambda a=None, c=None, ws=None, n=0: L.sq_tree_attention(a or attention(), c or cache(), ws, n, None)
    E, U, W = _lib.SQ_EINVAL, _lib.SQ_EUNSUPPORTED, _lib.SQ_EWORKSPACE
    nan = float("nan")
    for want, bad in ((E, dict(c=cache(dtype=_lib.SQ_F32))), (E, dict(c=cache(dtype=9))), (U, dict(c=cache(dim=0))), (U, dict(c=cache(dim=12))), (U, dict(c=cache(dim=264))),
                      (E, dict(c=cache(heads=3))), (E, dict(c=cache(heads=0))), (E, dict(a=attention(q_heads=0))), (E, dict(a=attention(tokens=-1))),
                      (E, dict(a=attention(scale=0.0))), (E, dict(a=attention(scale=-1.0))), (E, dict(a=attention(scale=nan))), (E, dict(a=attention(scale=math.inf))),
                      (E, dict(a=attention(tokens=3))), (E, dict(a=attention(most_new=2))), (E, dict(a=attention(ld_table=7))), (E, dict(a=attention(max_pages=0))),
                      (E, dict(c=cache(pages=0))), (E, dict(c=cache(page=0))), (E, dict(a=attention(q=None))), (E, dict(a=attention(out=None))), (E, dict(a=attention(table=None))),
                      (E, dict(a=attention(lens=None))), (E, dict(c=cache(k=None))), (E, dict(c=cache(v=None))), (U, dict(a=attention(q_head=65))), (U, dict(a=attention(out_token=4))),
                      (U, dict(a=attention(q=P + 8))), (U, dict(c=cache(k=P + 2))), (U, dict(c=cache(v_slot=260))), (E, dict(a=attention(mask_words=-1))),
                      (U, dict(a=attention(tokens=2, seqs=1 << 23, most_new=1, starts=P)))):
        assert call(**bad) == want, (bad, L.sq_last_error())
    assert L.sq_tree_attention(None, cache(), None, 0, None) == E
    assert call(a=attention(tokens=0, seqs=0)) == _lib.SQ_OK and call(a=attention(most_new=0, starts=P)) == _lib.SQ_OK
    # one long sequence is cut into parts, whose sums need room
    long, big = attention(seqs=1, most_new=2, max_pages=1000, ld_table=1000), cache(pages=1000)
    need = L.sq_tree_attention_workspace_bytes(long, big)
    assert need > 0 and need % (64 * 4 + 8) == 0
    assert call(a=long, c=big) == W and call(a=long, c=big, ws=P, n=need - 1) == W and call(a=long, c=big, ws=P + 128, n=need) == W
    assert L.sq_tree_attention_workspace_bytes(attention(), cache()) == 0 and L.sq_tree_attention_workspace_bytes(attention(scale=-1.0), cache()) == 0


def test_keep_drafted_refuses():
    L = _lib.lib()

    def call(c=None, layers=2, table=P, ld=8, pages=8, lens=P, path=P, ldp=4, most=4, counts=P, seqs=2):
        return L.sq_keep_drafted(c or cache(), layers, 1 << 20, 1 << 20, table, ld, pages, lens, path, ldp, most, counts, seqs, None)

    for bad in (dict(c=cache(dtype=4)), dict(c=cache(page=0)), dict(c=cache(pages=-1)), dict(c=cache(heads=-1)), dict(c=cache(dim=0)), dict(c=cache(k=None)), dict(layers=-1),
                dict(seqs=-1), dict(seqs=65536), dict(most=-1), dict(ld=7), dict(ldp=3), dict(pages=-1), dict(table=None), dict(lens=None), dict(path=None), dict(counts=None)):
        assert call(**bad) == _lib.SQ_EINVAL, bad
    assert call(layers=0) == call(seqs=0) == call(most=0, ldp=0) == call(c=cache(pages=0)) == _lib.SQ_OK


def test_python_calls_have_no_cpu_path():
    x, pos, f = torch.zeros(2, 4, 64, dtype=torch.float16), torch.arange(2), torch.ones(32, dtype=torch.float64)
    c, i32 = torch.zeros(3, 16, 2, 64, dtype=torch.float16), lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(ValueError, match="on the GPU"):
        rotary(x, pos, f)
    with pytest.raises(ValueError, match="on the GPU"):
        qk_norm_rotary(x, x[:, :2], pos, f)
    with pytest.raises(ValueError, match="on the GPU"):
        tree_attention(x, c, c, i32(2, 1), i32(2))
    with pytest.raises(ValueError, match="on the GPU"):
        keep_drafted(c, c.clone(), i32(2, 1), i32(2), i32(2, 2), i32(2))
    with pytest.raises(ValueError):
        rotary(x[0], pos, f)
    with pytest.raises(NotImplementedError):
        rotary(x.float().requires_grad_(), pos, f)


def test_frequencies():
    f, s = rotary_freqs(8, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15) and s == 1.0
    f4, s = rotary_freqs(8, 10000.0, {"type": "linear", "factor": 4}, device="cpu")
    assert torch.equal(f4, f / 4) and s == 1.0
    # ntk: the fastest pair as it was, the slowest four times slower
    f4, _ = rotary_freqs(8, 10000.0, {"type": "ntk", "factor": 4}, device="cpu")
    assert f4[0] == 1 and float(f4[-1] * 4 / f[-1]) == pytest.approx(1.0, rel=1e-12) and bool((f4 <= f).all())
    # yarn: pairs that turn more than 32 times in the trained context as they were, less than once divided, in between in between; amplitude 0.1 ln f + 1
    base, rot, n = 10000.0, 128, 4096
    f = rotary_freqs(rot, base, device="cpu")[0]
    g, s = rotary_freqs(rot, base, {"type": "yarn", "factor": 8.0, "original": n}, device="cpu")
    turns = n * f / (2 * math.pi)
    assert torch.equal(g[turns > 34], f[turns > 34]) and torch.allclose(g[turns < 0.95], f[turns < 0.95] / 8, rtol=1e-15)
    assert bool((g <= f).all()) and bool((g >= f / 8).all()) and bool((g[1:] < g[:-1]).all()) and s == pytest.approx(0.1 * math.log(8) + 1)
    assert rotary_freqs(rot, base, {"type": "yarn", "factor": 8.0, "original": n, "scale": 1.0}, device="cpu")[1] == 1.0
    # bands: wavelengths below n / 4 as they were, above n divided, and the blend's own formula in between
    g, s = rotary_freqs(rot, base, {"type": "bands", "factor": 8.0, "original": n}, device="cpu")
    assert s == 1.0
    for a, b in zip(f.tolist(), g.tolist()):
        wave = 2 * math.pi / a
        k = min(1.0, max(0.0, (n / wave - 1) / 3))
        assert b == pytest.approx((1 - k) * a / 8 + k * a, rel=1e-14)
    for bad in (dict(rot=7), dict(rot=-2), dict(rot=8, base=0.0), dict(rot=8, scaling={"type": "linear", "factor": 0}), dict(rot=8, scaling={"type": "x", "factor": 2}),
                dict(rot=2, scaling={"type": "ntk", "factor": 2})):
        with pytest.raises(ValueError):
            rotary_freqs(device="cpu", **bad)
    assert rotary_freqs(0, device="cpu")[0].numel() == 0


def test_sizes_whose_products_pass_64_bits_are_refused():
    L = _lib.lib()
    U, E = _lib.SQ_EUNSUPPORTED, _lib.SQ_EINVAL
    for seqs, new, hq in ((1, 1 << 30, 1 << 10), ((1 << 31) - 1, (1 << 31) - 1, 1 << 16), (1 << 16, 1 << 15, 1)):
        a, c = attention(tokens=2, seqs=seqs, most_new=new, q_heads=hq, starts=P), cache(heads=1)
        assert L.sq_tree_attention(a, c, None, 0, None) == U and L.sq_tree_attention_workspace_bytes(a, c) == 0
    keep = lambda layers, **kw: L.sq_keep_drafted(cache(**kw), layers, 0, 0, P, 8, 8, P, P, 4, 4, P, 1, None)
    for layers, kw in (((1 << 31) - 1, dict(heads=(1 << 31) - 1, dim=1 << 16)), ((1 << 20) + 1, {}), (1, dict(heads=(1 << 20) + 1)), (1, dict(dim=65537))):
        assert keep(layers, **kw) == E
    assert keep(1 << 20, heads=1 << 20, dim=1 << 16) == U


def test_outputs_of_attention_whose_rows_overlap_are_refused():
    L = _lib.lib()
    for kw in (dict(out_token=256), dict(out_head=56), dict(out_token=0), dict(out_token=64, out_head=64)):
        assert L.sq_tree_attention(attention(**kw), cache(), None, 0, None) == _lib.SQ_EINVAL, kw


def test_python_calls_refuse_tangents():
    from torch.autograd import forward_ad
    x, pos, f = torch.zeros(2, 4, 64, dtype=torch.float16), torch.arange(2), torch.ones(32, dtype=torch.float64)
    c, i32 = torch.zeros(3, 16, 2, 64, dtype=torch.float16), lambda *s: torch.zeros(*s, dtype=torch.int32)
    with forward_ad.dual_level():
        d, dc = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, c))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: rotary(d, pos, f), lambda: qk_norm_rotary(x, d[:, :2], pos, f), lambda: tree_attention(d, c, c, i32(2, 1), i32(2)),
                             lambda: keep_drafted(c, dc, i32(2, 1), i32(2), i32(2, 2), i32(2))):
                    with pytest.raises(NotImplementedError, match="tangents"):
                        call()


def test_scales_whose_product_with_log2_e_is_no_number_are_refused():
    L = _lib.lib()
    for scale in (2.4e38, 2.9e38, 3.4e38):
        assert L.sq_tree_attention(attention(scale=scale), cache(), None, 0, None) == _lib.SQ_EINVAL, scale
        assert L.sq_tree_attention(attention(scale=scale, tokens=0, seqs=0), cache(), None, 0, None) == _lib.SQ_EINVAL, scale
    assert L.sq_tree_attention(attention(scale=2.2e38, tokens=0, seqs=0), cache(), None, 0, None) == _lib.SQ_OK
