"""CPU restatement of how an attention call is cut into tickets and of how many partial results it leaves, against the slots
that its scratch has (test infrastructure).  Lengths and rows are numpy arrays, one entry per sequence."""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

WORKERS, BLOCK, UNIT_ROWS, UNIT_ROWS_MOST, UNIT_WAVES = 8, 16, 16, 32, 2
TILE, ITEM_ROWS, MIN_RUN, MIN_TILES, SHARE_ROWS, MERGE_ROWS_MOST = 128, 256, 4, 4, 64, 32
TILE_US, BLOCK_US = np.float32(2.6), np.float32(0.0015)


def up(a, b):
    return -(-a // b)


@dataclass
class Cut:
    tiles: int              # items, units, merges: their sum is a task's tiles
    units: int
    merges: int
    parts: int              # partial results of 16 rows each
    prefix: bool            # the prefix is read once for all
    halved: bool            # items of up to 128 rows leave two results


def part_slots(sms, heads, rows, n, q_heads):
    group, most = q_heads // heads, min(n, rows)
    base = 2 * UNIT_WAVES * sms * WORKERS + 128 * sms
    own = heads * most * (1 if rows <= n and group <= UNIT_ROWS else 8)
    pre_rows = min(rows * group, most * SHARE_ROWS)
    pre = 16 * (heads * up(pre_rows, ITEM_ROWS) + 4 * sms)
    return base + min(own + pre, 1 << 16)


def scratch_bytes(sms, heads, dim, rows, n, q_heads, most_seqs=1024, control=16640):
    slots = part_slots(sms, heads, rows, n, q_heads)
    return up(control, 256) * 256 + up((most_seqs + 1) * heads * 4, 256) * 256 + up(slots * UNIT_ROWS * 8, 256) * 256 + slots * UNIT_ROWS * dim * 4


def _round(sms, heads, dim, group, t, lens, shared, share, halved):
    halves = lambda r: np.where(np.asarray(r) <= (TILE if halved else 0), 2, 1)
    rows, real = t * group, t > 0
    own = np.where(real, lens - np.where(share, shared, 0), 0)
    by_tiles = real & (rows > UNIT_ROWS_MOST)
    by_units = real & ~by_tiles
    groups = up(rows, UNIT_ROWS)
    blocks = int((up(own, BLOCK) * groups)[by_units].sum()) * heads
    pre_rows = int(rows[share].sum())
    tiles = (int((up(own, TILE) * up(rows, ITEM_ROWS))[by_tiles].sum()) + up(shared, TILE) * up(pre_rows, ITEM_ROWS)) * heads
    waves = sms * WORKERS * UNIT_WAVES
    target = max(waves - min(waves, int(groups[by_units].sum()) * heads // 2), waves // 4)
    run = max(MIN_RUN, up(blocks, target))
    tile_us = TILE_US * np.float32(tiles) * (np.float32(dim) / np.float32(128))
    block_us = BLOCK_US * np.float32(dim) * np.float32(blocks)
    part = np.float32(0) if tiles == 0 else np.float32(1) if blocks == 0 else tile_us / (tile_us + block_us)
    items = max(int(np.float32(sms) * part), 1)
    tile_run = max(MIN_TILES, up(tiles, items))
    tile_runs = lambda positions: np.maximum(1, (up(np.asarray(positions), TILE) + tile_run // 2) // tile_run)
    runs = np.where(by_tiles, tile_runs(own) * halves(rows), np.maximum(1, up(up(own, BLOCK), run)))
    leaves = real & ((runs > 1) | share)
    parts = int((groups * runs)[leaves].sum()) * heads
    items_all = int((up(rows, ITEM_ROWS) * (runs // halves(rows)))[by_tiles].sum()) * heads
    if shared > 0:
        parts += up(pre_rows, UNIT_ROWS) * heads * int(tile_runs(shared)) * int(halves(pre_rows))
        items_all += up(pre_rows, ITEM_ROWS) * heads * int(tile_runs(shared))
    return items_all, int((groups * runs)[by_units].sum()) * heads, parts


def cut(sms, heads, dim, q_heads, page, t, lens, shared=0, rows=None, fallback=True):
    """t: rows of q of each sequence, lens: positions held (-1: padding).  `fallback`: whether what does not fit is cut again."""
    t, lens = np.asarray(t, dtype=np.int64), np.asarray(lens, dtype=np.int64)
    group, rows = q_heads // heads, int(t.sum()) if rows is None else rows
    slots = part_slots(sms, heads, rows, len(t), q_heads)
    t = np.where(lens < 0, 0, t)
    shared = shared // page * page
    share = (shared > 0) & (t > 0) & (t * group <= SHARE_ROWS) & (lens - t >= shared)
    if int(share.sum()) < 2:
        shared, share = 0, np.zeros_like(share)
    halved = True
    while True:
        tiles, units, parts = _round(sms, heads, dim, group, t, lens, shared, share, halved)
        if parts <= slots or (shared == 0 and not (halved and fallback)):
            break
        halved = halved and shared > 0
        shared, share = 0, np.zeros_like(share)
    out_rows, per = rows * q_heads, 1
    while per < MERGE_ROWS_MOST and per * sms * WORKERS < out_rows:
        per *= 2
    merges = up(out_rows, per) if parts > 0 else 0
    return Cut(tiles, units, max(merges, 1 if tiles + units == 0 else 0), parts, shared > 0, halved)
