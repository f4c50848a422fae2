"""Attention over the paged cache at the borders of its cut: how many results a call leaves, where they go, and what the
tiles do that ordinary scores hardly reach.  Tolerances are those of test_kv_gpu.py."""
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from oracle import attention_cut as ac                                       # noqa: E402
from test_kv_gpu import TYPES, _attend, _check, _filled, _gen, _ints, _normal, _share, _stream, kv, pk      # noqa: E402,F401


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).tolist()


def _check_some(pk, kv, c, q, out, counts, lens, some, scale=None):
    """The rows of a few of the sequences against the definition."""
    starts = _starts(counts)
    rows = [starts[i] + j for i in some for j in range(counts[i])]
    small = pk.KvCache(c.k, c.v, c.page_table[some].contiguous(), _ints([lens[i] for i in some]), c.refs)
    _check(kv, small, q[rows], out[rows], list(range(len(some))), _starts([counts[i] for i in some]), scale=scale)
    small.destroy()


@pytest.mark.parametrize("n, t, q_heads, heads, length", [(200, 128, 32, 32, 500), (512, 16, 128, 16, 100), (1024, 32, 32, 8, 40)])
def test_many_short_prompts_stay_inside_their_scratch(pk, kv, n, t, q_heads, heads, length):
    """33 to 128 rows a sequence, more of them than two results a row group have room for; a guard behind the scratch stays as it was."""
    c = _filled(pk, [length] * n, 64, heads, 64, torch.float16)
    q = _normal(_gen(40), torch.float16, n * t, q_heads, 64)
    bytes_ = c.attention_scratch_bytes(n * t, n, q_heads)
    guard = (1 << 16) * ac.UNIT_ROWS * 64 * 4
    buffer = torch.zeros(bytes_ + guard, dtype=torch.uint8, device="cuda")
    buffer[bytes_:] = 0x5A
    out = _attend(pk, c, q, None, _ints(_starts([t] * n)), n, scratch=buffer[:bytes_])
    assert bool((buffer[bytes_:] == 0x5A).all())
    assert bool(torch.isfinite(out).all()) and not bool((out == 7).all(-1).any())
    _check_some(pk, kv, c, q, out, [t] * n, [length] * n, [0, n // 2, n - 1])
    c.destroy()


def test_tickets_and_scratch_are_those_of_the_cpu_cut(pk, kv):
    """What the kernel counts as a task's tiles, and the scratch that the library asks for, over random calls."""
    rng = random.Random(3)
    for i in range(24):
        heads, group, dim, page = rng.choice([1, 2, 8]), rng.choice([1, 4, 8]), rng.choice([64, 128]), rng.choice([16, 64])
        n = rng.choice([1, 3, 40, 200])
        counts = [1] * n if i % 3 == 0 else [rng.choice([1, 1, 3, rng.randint(1, 40)]) for _ in range(n)]
        shared = rng.choice([0, 192, 1024])
        lens = [rng.choice([-1, 0, shared + rng.randint(40, 900), shared + rng.randint(40, 900)]) for _ in range(n)]
        c = _filled(pk, [max(x, 0) for x in lens], page, heads, dim, torch.bfloat16)
        first = next((k for k in range(n) if lens[k] >= shared), 0)
        for k in range(n):
            if shared and lens[k] >= shared:
                c.page_table[k, :shared // page] = c.page_table[first, :shared // page]
        rows, q_heads = sum(counts), heads * group
        assert c.attention_scratch_bytes(rows, n, q_heads) == ac.scratch_bytes(_sms(), heads, dim, rows, n, q_heads)
        q = _normal(_gen(i), torch.bfloat16, rows, q_heads, dim)
        out = torch.zeros_like(q)
        scratch = torch.zeros(c.attention_scratch_bytes(rows, n, q_heads), dtype=torch.uint8, device="cuda")
        seqs = _ints([-1 if x < 0 else k for k, x in enumerate(lens)])
        t = pk.Task.attention(c, out, q, seqs, scratch=scratch, starts=_ints(_starts(counts)), shared_len=_ints([shared]) if shared else None)
        t.launch(_stream())
        info = t.wait()
        x = ac.cut(_sms(), heads, dim, q_heads, page, counts, lens, shared, rows=rows)
        assert info.status == pk.STATUS_COMPLETED and info.tiles_total == info.tiles_done == x.tiles + x.units + x.merges
        torch.cuda.synchronize()
        t.destroy()
        c.destroy()


def test_a_prefix_that_just_does_not_fit_is_dropped_by_every_thread_alike(pk, kv):
    """Results fit with the prefix's runs counted as one and do not with the real number: a thread that looked at the next round's
    prefix would go on with another cut than the rest."""
    m, s, heads, prefix = 696, 10, 8, 65536
    counts, lens = [1] * s + [128] * m, [prefix + 40 + i for i in range(s)] + [128] * m
    slots = ac.part_slots(_sms(), heads, sum(counts), s + m, heads)
    share = np.arange(s + m) < s
    _, _, parts = ac._round(_sms(), heads, 64, 1, np.array(counts), np.array(lens), prefix, share, True)
    runs_as_one = 16 * heads * m + heads * s + 2 * heads
    assert _sms() != 148 or runs_as_one <= slots < parts
    c = _filled(pk, [lens[i] if i < s else 128 for i in range(s + m)], 128, heads, 64, torch.bfloat16)
    _share(c, lens[:s], prefix)
    q = _normal(_gen(41), torch.bfloat16, sum(counts), heads, 64)
    starts = _ints(_starts(counts))
    scratch = torch.zeros(c.attention_scratch_bytes(sum(counts), s + m, heads), dtype=torch.uint8, device="cuda")
    out = _attend(pk, c, q, None, starts, s + m, shared=prefix, scratch=scratch)
    _check_some(pk, kv, c, q, out, counts, lens, [0, s - 1, s, s + m - 1])
    for _ in range(20):
        assert torch.equal(_attend(pk, c, q, None, starts, s + m, shared=prefix, scratch=scratch), out)
    t = pk.Task.attention(c, torch.zeros_like(q), q, None, scratch=scratch, starts=starts, shared_len=_ints([prefix]))
    t.launch(_stream())
    info = t.wait()
    x = ac.cut(_sms(), heads, 64, heads, 128, counts, lens, prefix)
    assert info.status == pk.STATUS_COMPLETED and info.tiles_total == x.tiles + x.units + x.merges
    assert torch.equal(out, _attend(pk, c, q, None, starts, s + m, shared=prefix))
    t.destroy()
    c.destroy()


def test_a_task_created_while_its_scratch_is_still_written_on_another_stream(pk, kv):
    """The scratch's last writer is queued on the stream that the task will run on, behind the creation's own clearing."""
    lens = [9000, 4000, 300, 12000]
    c = _filled(pk, lens, 64, 4, 128, torch.bfloat16)
    q = _normal(_gen(42), torch.bfloat16, 4, 16, 128)
    want = _attend(pk, c, q, None, None, 4)
    s = torch.cuda.Stream()
    scratch, out = torch.empty(c.attention_scratch_bytes(4, 4, 16), dtype=torch.uint8, device="cuda"), torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(100_000_000)
        scratch.fill_(0x7F)
    t = pk.Task.attention(c, out, q, None, scratch=scratch)
    for _ in range(2):
        t.launch(s.cuda_stream)
        assert t.wait().status == pk.STATUS_COMPLETED
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        out.zero_()
        torch.cuda.synchronize()
    t.destroy()
    # The first launch captured: nothing is cleared in the graph, and its replays and a direct launch all work.
    t = pk.Task.attention(c, out, q, None, scratch=scratch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.launch(_stream())
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    out.zero_()
    t.launch(_stream())
    assert t.wait().status == pk.STATUS_COMPLETED
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del graph
    t.destroy()
    c.destroy()


def _levels(c, i, n, levels):
    """Keys of sequence i: position p points along one direction, 64 positions at a time as far as `levels` says, plus noise."""
    page, dim = c.k.shape[3], c.dim
    pos = torch.arange(n, device="cuda")
    at = torch.tensor([levels[p % len(levels)] for p in range(-(-n // 64))], device="cuda").repeat_interleave(64)[:n]
    where = c.page_table[i].long()[pos // page]
    k = 0.05 * c.k[0][where, :, pos % page].float()
    k[..., 0] += at[:, None]
    c.k[0][where, :, pos % page] = k.to(c.dtype)


# How far the maximum lies, in units of a score, from 64 positions to the next: up by little and by much, down, and up again from far below.
RISING, FALLING, ZIGZAG = [0.0, 3.0, 9.0, 14.0, 14.5, 22.0, 40.0, 41.0], [30.0, 12.0, 3.0, 0.0], [5.0, 30.0, -20.0, 31.0, 60.0, -60.0, 58.0, 59.0, 75.0]


@pytest.mark.parametrize("dtype, Hq, H, D, page", [("bf16", 8, 2, 128, 64), ("fp16", 6, 2, 64, 16), ("fp16", 3, 1, 128, 128)])
@pytest.mark.parametrize("levels", [RISING, FALLING, ZIGZAG])
@pytest.mark.parametrize("scale", [1.0, -1.0])
@pytest.mark.parametrize("shared, counts, lens", [(0, [20, 300, 9], [700, 900, 64]), (640, [1, 2, 5, 2], [700, 641, 1500, 650])])
def test_tiles_follow_a_maximum_that_moves(pk, kv, dtype, Hq, H, D, page, levels, scale, shared, counts, lens):
    """Results are scaled down wherever a row's maximum grows by more than 2^8; a negative scale turns the queries over."""
    c = _filled(pk, lens, page, H, D, TYPES[dtype])
    if shared:
        _share(c, lens, shared)
    for i, n in enumerate(lens):
        if not shared or i == 0:
            _levels(c, i, n, levels)
    starts = _starts(counts)
    q = 0.3 * _normal(_gen(43), torch.float32, starts[-1], Hq, D)
    q[..., 0] = scale
    q = q.to(TYPES[dtype])
    out = _attend(pk, c, q, None, _ints(starts), len(lens), shared=shared or None, scale=scale)
    _check(kv, c, q, out, list(range(len(lens))), starts, scale=scale)
    c.destroy()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shared", [None, 256])
@pytest.mark.parametrize("scale", [0.0, 0.5, -0.125])
def test_tiles_with_scores_of_hundreds_equal_scores_and_odd_scales(pk, kv, dtype, shared, scale):
    lens, counts = [700, 300, 333], [1, 2, 3] if shared else [140, 9, 40]
    c = _filled(pk, lens, 32, 1, 64, TYPES[dtype])
    if shared:
        _share(c, lens, shared)
    starts = _starts(counts)
    q = _normal(_gen(44), TYPES[dtype], starts[-1], 12, 64, scale=30.0)
    _check(kv, c, q, _attend(pk, c, q, None, _ints(starts), 3, shared=shared, scale=scale), [0, 1, 2], starts, scale=scale)
    q.zero_()
    _check(kv, c, q, _attend(pk, c, q, None, _ints(starts), 3, shared=shared, scale=scale), [0, 1, 2], starts, scale=scale)
    c.destroy()


def test_calls_and_grids_of_any_size_write_the_same_bytes(pk, kv):
    """Single tokens, drafts, a prompt and a shared prefix in one call: repeated, and as a task on 1, 7 and all SMs."""
    lens, counts = [5000, 4200, 4800, 4100, 6000, 4097], [1, 1, 4, 2, 150, 1]
    c = _filled(pk, lens, 64, 2, 128, torch.bfloat16)
    _share(c, lens, 4096)
    starts = _ints(_starts(counts))
    q = _normal(_gen(45), torch.bfloat16, sum(counts), 8, 128, scale=2.0)
    scratch = torch.zeros(c.attention_scratch_bytes(sum(counts), 6, 8), dtype=torch.uint8, device="cuda")
    want = _attend(pk, c, q, None, starts, 6, shared=4096, scratch=scratch)
    for _ in range(20):
        assert torch.equal(_attend(pk, c, q, None, starts, 6, shared=4096, scratch=scratch), want)
    out = torch.zeros_like(q)
    t = pk.Task.attention(c, out, q, None, scratch=torch.zeros_like(scratch), starts=starts, shared_len=_ints([4096]))
    for sms in (1, 7, 0):
        out.zero_()
        t.launch(_stream(), sm_limit=sms)
        assert t.wait(10_000_000).status == pk.STATUS_COMPLETED
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    t.destroy()
    c.destroy()


@pytest.mark.parametrize("dtype, group, heads, dim, page", [("bf16", 33, 1, 64, 16), ("fp16", 64, 2, 128, 64), ("bf16", 100, 1, 128, 128), ("fp16", 129, 1, 64, 32),
                                                            ("bf16", 300, 1, 64, 64)])
@pytest.mark.parametrize("shared", [None, 256])
def test_many_query_heads_on_one_key_head(pk, kv, dtype, group, heads, dim, page, shared):
    """A single token has more rows than a unit takes: tiles, direct and merged, with up to 128 rows and with more."""
    lens = [300, 257, 1200, 400]
    c = _filled(pk, lens, page, heads, dim, TYPES[dtype])
    _share(c, lens, 256)
    q = _normal(_gen(46), TYPES[dtype], 4, heads * group, dim, scale=2.0)
    _check(kv, c, q, _attend(pk, c, q, None, None, 4, shared=shared), list(range(4)), list(range(5)))
    c.destroy()
