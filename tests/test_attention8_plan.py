"""The second writing of how attention over an 8-bit cache is cut, which tests choose their sizes by, against the workspace that a call asks for (on the host, for 256 compute units where there is no GPU)."""

import ctypes
import math
import random

from quantexperiments_amd import _lib
from tests.attention8_plan import plan

P = 0x10000                                                  # an address that is never read


def workspace(tokens, seqs, most_new, hq, hk, d, slots, page=16):
    c = _lib.SqCache8(k=P, v=P, k_scale=P, v_scale=P, k_page=page * hk * 256, k_slot=hk * 256, k_head=256, v_page=page * hk * 256, v_slot=hk * 256, v_head=256, ks_page=hk, ks_block=hk, ks_head=1,
                      vs_page=hk, vs_block=hk, vs_head=1, pages=8, page=page, blocks=1, heads=hk, dim=d)
    a = _lib.SqAttention(q=P, out=2 * P, table=P, lens=P, starts=P, q_token=hq * 256, q_head=256, out_token=hq * 256, out_head=256, ld_table=slots // page, tokens=tokens, seqs=seqs,
                         most_new=most_new, q_heads=hq, max_pages=slots // page, scale=1.0)
    return _lib.lib().sq_tree_attention8_workspace_bytes(ctypes.byref(a), ctypes.byref(c), _lib.SQ_BF16)


def test_workspaces_are_those_of_the_plan():
    rng = random.Random(3)
    log = lambda lo, hi: round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
    ways = {}
    for _ in range(30000):
        hk, seqs, new, d = rng.choice((1, 2, 3, 4, 5, 8, 16)), log(1, 100), log(1, 2000), rng.choice((16, 64, 80, 128, 144, 256))
        hq, slots = hk * rng.randint(1, 10), log(1, 20000) * 16
        p = plan(seqs * new, seqs, new, hq, hk, d, slots)
        assert workspace(seqs * new, seqs, new, hq, hk, d, slots) == p.workspace, (seqs, new, hq, hk, d, slots, p)
        ways.setdefault(p.way, set()).add((p.rows, p.slots > 1, p.last_splits < p.splits))
    assert ways["few"] == {(r, s, False) for r in (16, 32) for s in (False, True)}
    assert {r for r, _, _ in ways["shared"]} == {r for r, _, _ in ways["tiles"]} == {64, 128, 256}
    assert any(less for _, _, less in ways["tiles"])
