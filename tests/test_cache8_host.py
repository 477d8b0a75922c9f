"""What the calls on 8-bit caches and on pages refuse.  CPU only: no kernel is launched here."""

import ctypes

from quantexperiments_amd import _lib

P = 0x10000                                                  # an address that is never read
E, U, W, OK = _lib.SQ_EINVAL, _lib.SQ_EUNSUPPORTED, _lib.SQ_EWORKSPACE, _lib.SQ_OK


def heads(**kw):
    return _lib.SqHeads(**{**dict(in_=P, in_token=256, in_head=64, heads=4), **kw})


def cache(**kw):
    return _lib.SqCache8(**{**dict(k=P, v=2 * P, k_scale=3 * P, v_scale=4 * P, k_page=8192, k_slot=256, k_head=64, v_page=8192, v_slot=256, v_head=64, ks_page=8, ks_block=4, ks_head=1,
                                   vs_page=8, vs_block=4, vs_head=1, pages=8, page=32, blocks=2, heads=4, dim=64), **kw})


def plane(**kw):
    return _lib.SqPlane(**{**dict(at=P, layer=65536, page=8192, row=256, head=64, rows=32, heads=4, bytes=64), **kw})


CACHES = [(U, dict(dim=0)), (U, dict(dim=24)), (U, dict(dim=272)), (E, dict(heads=-1)), (E, dict(pages=-1)), (E, dict(page=0)), (E, dict(blocks=0)), (E, dict(blocks=3)),
          (U, dict(blocks=4)), (U, dict(page=24, blocks=1)), (E, dict(pages=1 << 27)), (U, dict(k_slot=8)), (U, dict(v_head=72)), (U, dict(k=P + 8)), (U, dict(k_slot=-256)), (U, dict(v_slot=1 << 27)),
          (E, dict(k=None)), (E, dict(v_scale=None))]


def test_structs_match_the_header():
    assert ctypes.sizeof(_lib.SqCache8) == 4 * 8 + 12 * 8 + 5 * 4 + 4 and _lib.SqCache8.dim.offset == 144 and _lib.SqCache8.ks_page.offset == 80
    assert ctypes.sizeof(_lib.SqPlane) == 5 * 8 + 3 * 4 + 4 and _lib.SqPlane.bytes.offset == 48


def test_put_tokens8_refuses():
    L = _lib.lib()

    def call(k=None, v=None, n=2, t=_lib.SQ_F16, c=None, table=P, ld=8, pages=8, lens=P, starts=None, seqs=2, most=1):
        return L.sq_put_tokens8(k or heads(), v or heads(in_=5 * P), n, t, c or cache(), table, ld, pages, lens, starts, seqs, most, None)

    for want, bad in [(w, dict(c=cache(**b))) for w, b in CACHES] + [
            (E, dict(t=_lib.SQ_F32)), (E, dict(t=5)), (E, dict(k=heads(heads=3))), (E, dict(v=heads(heads=5))), (E, dict(n=-1)), (E, dict(seqs=-1)), (E, dict(most=-1)), (E, dict(n=3)), (E, dict(most=2)),
            (E, dict(ld=7)), (E, dict(pages=-1)), (E, dict(pages=0)), (E, dict(c=cache(pages=0))), (E, dict(k=heads(in_=None))), (E, dict(v=heads(in_=None))), (E, dict(table=None)), (E, dict(lens=None)),
            (U, dict(k=heads(in_token=260))), (U, dict(v=heads(in_head=4))), (U, dict(v=heads(in_=P + 2))), (U, dict(n=1 << 30, starts=P, seqs=1 << 16, most=1 << 16))]:
        assert call(**bad) == want, (bad, L.sq_last_error())
    assert L.sq_put_tokens8(None, heads(), 2, _lib.SQ_F16, cache(), P, 8, 8, P, None, 2, 1, None) == E
    assert call(n=0, seqs=0) == OK and call(most=0, starts=P) == OK and call(c=cache(heads=0), k=heads(heads=0), v=heads(heads=0)) == OK


def test_keep_drafted8_refuses():
    L = _lib.lib()

    def call(c=None, layers=2, step=65536, s_step=64, table=P, ld=8, pages=8, lens=P, path=P, ld_path=4, most=4, counts=P, seqs=2):
        return L.sq_keep_drafted8(c or cache(), layers, step, step, s_step, s_step, table, ld, pages, lens, path, ld_path, most, counts, seqs, None)

    for want, bad in [(w, dict(c=cache(**b))) for w, b in CACHES] + [
            (E, dict(layers=-1)), (E, dict(seqs=-1)), (E, dict(seqs=65536)), (E, dict(most=-1)), (E, dict(ld_path=3)), (E, dict(ld=7)), (E, dict(pages=-1)), (E, dict(table=None)), (E, dict(lens=None)),
            (E, dict(path=None)), (E, dict(counts=None)), (U, dict(step=8))]:
        assert call(**bad) == want, (bad, L.sq_last_error())
    assert L.sq_keep_drafted8(None, 1, 0, 0, 0, 0, P, 8, 8, P, P, 4, 4, P, 2, None) == E
    assert all(call(**{k: 0}) == OK for k in ("layers", "seqs", "most", "pages")) and call(c=cache(pages=0)) == OK


def test_fork_and_compact_refuse():
    L = _lib.lib()
    planes = lambda *p: (_lib.SqPlane * len(p))(*p)

    def fork(p=None, n=1, layers=2, pages=8, page=32, table=P, ld=8, width=8, lens=2 * P, seqs=2, parent=P, fresh=P, rows=3, out=3 * P, ld_out=8, out_lens=4 * P):
        return L.sq_fork_pages(p or planes(plane()), n, layers, pages, page, table, ld, width, lens, seqs, parent, fresh, rows, out, ld_out, out_lens, None)

    def compact(p=None, n=1, layers=2, pages=8, page=32, table=P, ld=8, width=8, lens=2 * P, seqs=2, out=3 * P, ld_out=8, used=P, ws=16 * P, n_ws=1 << 30):
        return L.sq_compact_pages(p or planes(plane()), n, layers, pages, page, table, ld, width, lens, seqs, out, ld_out, used, ws, n_ws, None)

    both = [(E, dict(n=-1)), (E, dict(n=5)), (E, dict(layers=-1)), (E, dict(pages=-1)), (E, dict(page=0)), (E, dict(pages=1 << 27)), (E, dict(p=planes(plane(rows=0)))), (E, dict(p=planes(plane(rows=33)))),
            (E, dict(p=planes(plane(rows=5)))), (E, dict(p=planes(plane(heads=-1)))), (E, dict(p=planes(plane(bytes=-1)))), (E, dict(p=planes(plane(at=None)))), (E, dict(ld=7)), (E, dict(ld_out=7)), (E, dict(seqs=-1)),
            (E, dict(width=-1)), (E, dict(lens=None)), (E, dict(table=None)), (E, dict(out=None)), (E, dict(out=P)), (U, dict(layers=1 << 20, p=planes(plane(heads=1 << 10))))]
    for want, bad in both + [(E, dict(rows=-1)), (E, dict(rows=65536)), (E, dict(parent=None)), (E, dict(fresh=None)), (E, dict(out_lens=None)), (E, dict(out_lens=2 * P)), (E, dict(seqs=0))]:
        assert fork(**bad) == want, (bad, L.sq_last_error())
    for want, bad in both + [(E, dict(used=None)), (U, dict(pages=(1 << 20) + 1)), (W, dict(ws=None)), (W, dict(ws=P + 4)), (W, dict(n_ws=L.sq_compact_pages_workspace_bytes(8) - 1))]:
        assert compact(**bad) == want, (bad, L.sq_last_error())
    assert fork(rows=0) == OK
    assert L.sq_compact_pages_workspace_bytes(8) >= 8 and L.sq_compact_pages_workspace_bytes(-1) == 0
