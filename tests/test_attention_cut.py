"""The partial results of an attention call fit the scratch that the library asks for: the cut restated on the CPU
(oracle/attention_cut.py) over the whole range of calls, and its constants against the kernels' source."""
import random
import re
from pathlib import Path

import numpy as np
import pytest

from oracle import attention_cut as ac

KERNELS = Path(__file__).resolve().parents[1] / "xsched_b200" / "csrc" / "kernels"
MAX_SEQS = 1024


def _fits(sms, heads, dim, q_heads, page, t, lens, shared=0, **kw):
    x = ac.cut(sms, heads, dim, q_heads, page, t, lens, shared, **kw)
    return x, x.parts <= ac.part_slots(sms, heads, int(np.sum(t)), len(t), q_heads)


def test_constants_are_the_kernels():
    source = (KERNELS / "attention_plan.cuh").read_text()
    for name, value in (("kWorkers", ac.WORKERS), ("kBlock", ac.BLOCK), ("kUnitRows", ac.UNIT_ROWS), ("kUnitRowsMost", ac.UNIT_ROWS_MOST),
                        ("kUnitWaves", ac.UNIT_WAVES), ("kTile", ac.TILE), ("kMinRun", ac.MIN_RUN), ("kMinTiles", ac.MIN_TILES), ("kShareRows", ac.SHARE_ROWS),
                        ("kMergeRowsMost", ac.MERGE_ROWS_MOST)):
        assert int(re.search(rf"constexpr int {name} = (\d+);", source).group(1)) == value, name
    assert re.search(r"constexpr float kTileUs = 2\.6f;", source) and "kItemRows = 2 * kTile" in source and "0.0015f" in source


# sequences, queries each, query and key heads, positions: all leave 16 results a key head and sequence with two groups at work
MANY = [(1024, 32, 32, 8, 40), (256, 128, 32, 32, 200), (200, 128, 32, 32, 500), (512, 16, 128, 16, 100), (175, 128, 32, 32, 130), (698, 32, 32, 8, 64)]


@pytest.mark.parametrize("n, t, q_heads, heads, length", MANY)
def test_many_sequences_of_33_to_128_rows_fit(n, t, q_heads, heads, length):
    args = (148, heads, 128, q_heads, 64, [t] * n, [length] * n)
    assert not _fits(*args, fallback=False)[1], "such a call is what the second cut is for"
    x, fits = _fits(*args)
    assert fits and not x.halved


@pytest.mark.parametrize("sms", [1, 20, 132, 148, 160])
def test_results_fit_the_scratch_over_the_range(sms):
    rng = random.Random(sms)
    log = lambda lo, hi: min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))
    again = without = 0
    for _ in range(1500):
        heads, dim, page = log(1, 128), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16, 17, 32, 33, 64, 65, 128])
        n, kind = log(1, MAX_SEQS), rng.choice(["rows", "rows", "alike", "mixed", "single"])
        if kind == "rows":                      # at the borders between the kinds of tickets
            t = [max(1, rng.choice([15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129, 255, 256, 257]) // group)] * n
        elif kind == "alike":
            t = [log(1, 300)] * n
        elif kind == "single":
            t = [1] * n
        else:
            t = [rng.choice([0, 1, 1, 2, log(1, 600)]) for _ in range(n)]
        if sum(t) == 0:
            t[0] = 1
        longest = log(1, 200000)
        lens = [rng.choice([-1, 0, 1] + 9 * [rng.randint(1, longest)]) if kind == "mixed" else longest for _ in range(n)]
        shared = rng.choice([0, 0, log(16, 100000)])
        x, fits = _fits(sms, heads, dim, heads * group, page, t, lens, shared)
        assert fits, (heads, dim, page, group, t, lens, shared, x)
        again += not x.halved
        without += not x.prefix and ac.cut(sms, heads, dim, heads * group, page, t, lens, shared, fallback=False).parts > ac.part_slots(sms, heads, sum(t), n, heads * group)
    assert again > 5 and without > 5, "the range has calls that do not fit with two groups at work"


def test_what_is_left_without_halves_is_bounded_by_the_device():
    """64 results an SM, whatever the call: runs of more than one tile or block are what leaves results then."""
    rng = random.Random(7)
    for _ in range(1500):
        sms, heads, group, n = rng.choice([1, 20, 148]), rng.choice([1, 3, 8, 32]), rng.choice([1, 4, 16, 40]), rng.randint(1, MAX_SEQS)
        t = np.array([rng.choice([1, 1, rng.randint(1, 400)]) for _ in range(n)])
        lens = np.array([rng.choice([0, rng.randint(1, 500), rng.randint(1, 300000)]) for _ in range(n)])
        parts = ac._round(sms, heads, 128, group, t, lens, 0, np.zeros(n, dtype=bool), False)[2]
        assert parts <= 64 * sms
