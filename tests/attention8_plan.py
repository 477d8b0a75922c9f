"""How attention over an 8-bit cache is cut into workgroups, written down a second time: for tests that are to take a certain way through the GPU, and say so where they no longer do."""

from dataclasses import dataclass

STEP, SPLITS_MAX, WAVES = 32, 128, 4


@dataclass
class Plan:
    """way: "few" (blocks of rows whose waves split the keys), "tiles" (of many rows) or "shared" (tiles, the workgroups of a key head shared by work)."""
    way: str
    rows: int                    # of a block
    blocks: int
    splits: int
    last_splits: int
    slots: int                   # the most parts of a row's keys
    workspace: int


def plan(tokens, seqs, most_new, hq, hk, d, slots, cus=256):
    """slots: of a table row, in whole pages."""
    dp = 64 if d <= 64 else 128 if d <= 128 else 256
    rows, steps = most_new * (hq // hk), -(-slots // STEP)
    units = seqs * hk * -(-rows // 16)
    load = units * steps
    few = rows <= (16 if dp == 256 else 32)
    if not few:
        tiles = seqs * hk * (1 if rows <= 128 else -(-rows // 256))
        if dp == 256:
            few = (units <= cus and load <= 48 * cus) or (rows <= 32 and steps >= 32)
        else:
            few = (rows <= 128 and steps >= 8) or (tiles * (4 if steps < 4 else 2) <= cus and (load <= 96 * cus or (steps <= 96 and load <= 256 * cus)))
    if few:
        nw, mt = 0, 1 if rows <= 16 or dp == 256 or (units <= 2 * cus and load <= 32 * cus) else 2
        per, most = mt * 16, steps // WAVES
        if most <= (4 if dp < 256 else 2):
            most = 1
    else:
        mt = 1 if dp == 256 else 2
        nw = 4 if rows <= 64 * mt else 8
        per = mt * 16 * nw
        most = steps // 4 if steps // 4 > 8 else min(steps // 2, 8)
    blocks = -(-rows // per)
    base = seqs * hk * blocks
    want = cus // base
    if not nw:
        if dp == 64:
            want = 2 * cus // base
        want = max(want, steps // (20 * WAVES))
    splits = last = min(max(min(want, most), 1), SPLITS_MAX)
    if nw == 8 and blocks > 1 and -(-(rows - (blocks - 1) * per) // (mt * 16)) <= 4:
        room = cus // (seqs * hk)
        for s in range(min(room, most), 1, -1):
            less = (s * 60 + 99) // 100
            if (blocks - 1) * s + less <= room:
                if s <= SPLITS_MAX:
                    splits, last = s, less
                break
    items, room, shared, parts = seqs * blocks, cus // hk, False, splits
    if nw and 1 < items <= 64 and (8 * items <= 7 * room if seqs == 1 else 3 * items <= 2 * room) and steps < 1 << 17:
        shared, parts = True, 2 * room // items
        parts = 8 if 8 < parts <= 16 else min(parts, SPLITS_MAX)
    need = 0 if parts == 1 else tokens * hq * parts * (dp * 4 + 8) + (blocks * seqs * 4 if shared else 0)
    return Plan("shared" if shared else "tiles" if nw else "few", per, blocks, splits, last, parts, need)
