"""The paged key/value cache's operators (libxpk.so) against the 64-bit restatement in oracle/kv.py.

Integers and moved pages have to be equal.  Tolerances of computed values: `half` = eps / 2 of the 16-bit type is the
most a rounding is off, relative to the value.
  append     fp32 chain: a sum of 128 squares, rsqrt, two products, a turn: under 2^-17 of |a| + |b| (72 roundings of 2^-24
             and 2 ulp of rsqrtf), the angle 2^-21 of it, then one rounding.
  attention  weights are rounded once (half) and each is off by its score's error, 2 D 2^-24 times the largest sum of
             |q||k| scale; sums of n terms in fp32 add (n + 64) 2^-24; all relative to the weighted mean of |v|; one rounding
             of the result.  fp16 weights under 2^-14 are off by 2^-25 at most: n 2^-25 max|v|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def pk():
    from xsched_b200 import pk as _pk
    return _pk


@pytest.fixture(scope="module")
def kv():
    from oracle import kv as _kv
    return _kv


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


# ---------------------------------------------------------------------------------------------------------- pages
def _cache(pk, kv, layers=2, pages=40, heads=2, page=16, dim=64, seqs=12, width=6, dtype=torch.bfloat16, seed=0):
    g = _gen(seed)
    k, v = _normal(g, dtype, layers, pages, heads, page, dim), _normal(g, dtype, layers, pages, heads, page, dim)
    table, lens, refs = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda"), _ints([0] * seqs), _ints([0] * pages)
    return pk.KvCache(k, v, table, lens, refs), kv.Pages(table.cpu().numpy(), lens.cpu().numpy(), refs.cpu().numpy(),
                                                        [k.view(torch.int16).cpu().numpy(), v.view(torch.int16).cpu().numpy()], page)


def _same(c, o, pools=True):
    assert (c.page_table.cpu().numpy() == o.table).all() and (c.lens.cpu().numpy() == o.lens).all() and (c.refs.cpu().numpy() == o.refs).all()
    if pools:
        assert (c.k.view(torch.int16).cpu().numpy() == o.pools[0]).all() and (c.v.view(torch.int16).cpu().numpy() == o.pools[1]).all()


@pytest.mark.parametrize("seed, page, heads, dim, pages", [(1, 16, 1, 64, 30), (2, 16, 3, 128, 41), (3, 32, 2, 64, 24), (4, 64, 2, 128, 17), (5, 128, 1, 64, 9),
                                                           (6, 16, 2, 64, 5000)])
def test_random_programs_of_page_operations(pk, kv, seed, page, heads, dim, pages):
    rng = np.random.default_rng(seed)
    layers = 1 if pages > 1000 else 3
    c, o = _cache(pk, kv, layers=layers, pages=pages, heads=heads, page=page, dim=dim, seqs=12, width=6, seed=seed)
    failed = copied = moved = 0
    for step in range(60):
        op = rng.choice(["extend", "extend", "extend", "fork", "free", "compact", "copy"])
        n = int(rng.integers(1, 9))
        a = rng.integers(-1, 13, n)
        if op == "extend":
            t = rng.integers(0, 3 * page, n) - rng.integers(0, 3)
            c.extend(_ints(a.tolist()), _ints(t.tolist()), _stream())
            want = o.extend(a.tolist(), t.tolist())
            r = c.result(_stream())
            assert (r.copied, r.missing, r.refused) == want
            failed += want[1] + want[2] > 0
            copied += want[0]
        elif op == "fork":
            b = rng.integers(-2, 14, n)
            c.fork(_ints(a.tolist()), _ints(b.tolist()), _stream())
            o.fork(a.tolist(), b.tolist())
        elif op == "free":
            a = a[:2]
            c.free(_ints(a.tolist()), _stream())
            o.free(a.tolist())
        elif op == "compact":
            c.compact(_stream())
            want = o.compact()
            r = c.result(_stream())
            assert (r.copied, r.live) == want
            moved += want[0]
        else:
            ids = rng.permutation(pages + 2)[:2 * n] - 1            # -1 and `pages` are passed over
            src, dst = ids[0::2], ids[1::2]
            m = min(len(src), len(dst))
            c.copy(_ints(src[:m].tolist()), _ints(dst[:m].tolist()), _stream())
            o.copy(src[:m].tolist(), dst[:m].tolist())
        _same(c, o, pools=pages < 1000 or step % 20 == 19)
    assert copied + failed + moved > 0
    c.destroy()


def test_long_lists_and_equal_entries(pk, kv):
    c, o = _cache(pk, kv, layers=1, pages=4096, heads=1, page=16, seqs=1500, width=3)
    every = list(range(1500))
    for seqs, grow in ((every, [1] * 1500), (every[::-1] + every[:500], [17] * 2000), (every, [30] * 1500)):
        c.extend(_ints(seqs), _ints(grow), _stream())
        want = o.extend(seqs, grow)
        r = c.result(_stream())
        assert (r.copied, r.missing, r.refused) == want
        _same(c, o)
    kids = every[1:900]
    c.free(_ints(kids + kids), _stream())
    o.free(kids + kids)
    c.fork(_ints([0] * 899 + [950] * 899), _ints(kids + kids), _stream())
    o.fork([0] * 899 + [950] * 899, kids + kids)
    _same(c, o)
    c.extend(_ints(kids + [0]), _ints([1] * 900), _stream())
    assert c.result(_stream()).copied == o.extend(kids + [0], [1] * 900)[0] == 899
    _same(c, o)
    c.destroy()


def test_page_ids_out_of_range_are_left_alone(pk, kv):
    c, o = _cache(pk, kv, layers=1, pages=8, seqs=4, width=4)
    for x in (c, o):
        t, n, r = (x.page_table, x.lens, x.refs) if x is c else (x.table, x.lens, x.refs)
        t[0, 0], t[0, 1], t[0, 2], n[0] = 99, -7, 3, 40
        r[3] = 1
        n[2] = -5                                                    # counts as empty
        n[3] = 1 << 30                                               # longer than its row: the row's width counts
        t[3, 0], t[3, 3] = 5, 2 ** 31 - 1
        r[5] = 1
    for _ in range(2):
        c.fork(_ints([0, 3]), _ints([1, 2]), _stream())
        o.fork([0, 3], [1, 2])
        _same(c, o)
        c.extend(_ints([1, 0]), _ints([3, 9]), _stream())
        o.extend([1, 0], [3, 9])
        _same(c, o)
        c.compact(_stream())
        o.compact()
        _same(c, o)
        c.free(_ints([0, 1, 2, 3]), _stream())
        o.free([0, 1, 2, 3])
        _same(c, o)
    c.destroy()


def test_copy_task_stops_and_resumes_with_the_same_bytes(pk, kv):
    n = 300
    c, o = _cache(pk, kv, layers=6, pages=700, heads=4, page=64, dim=128, seqs=2, width=2)
    ids = np.random.default_rng(0).permutation(700)
    src, dst = ids[:n].tolist(), ids[n:2 * n].tolist()
    for flags in (pk.FLAG_NONE, pk.FLAG_NON_PREEMPTIBLE):
        t = pk.Task.kv_copy(c, _ints(src), _ints(dst), flags=flags)
        cuts = 0
        for _ in range(4 if flags == pk.FLAG_NONE else 0):
            t.launch(_stream(), sm_limit=1)
            t.set_flag(1)
            info = t.wait()
            torch.cuda.synchronize()
            t.set_flag(0)
            torch.cuda.synchronize()
            cuts += info.status == pk.STATUS_PREEMPTED
            if info.status == pk.STATUS_COMPLETED:
                break
        while True:
            t.launch(_stream())
            if t.wait().status == pk.STATUS_COMPLETED:
                break
        assert cuts > 0 or flags != pk.FLAG_NONE
        info = t.query()
        assert info.tiles_done == info.tiles_total == -(-n * 6 * 2 * 4 * 64 * 128 * 2 // 65536)
        o.copy(src, dst)
        _same(c, o)
        t.destroy()
        src, dst = dst, ids[2 * n:].tolist() + src[:2 * n + n - 700]
    c.destroy()


# --------------------------------------------------------------------------------------------------------- append
def _filled(pk, lens, page, heads, dim, dtype, layers=1, seed=0, extra=0):
    """A cache whose sequences have the given lengths, on pages in random order; pools random."""
    g = _gen(seed)
    each = [-(-max(n, 0) // page) for n in lens]
    pages = max(1, sum(each)) + 3
    ids = torch.randperm(pages, device="cuda", generator=g).int()
    table = torch.full((len(lens) + extra, max([1] + each) + 1), -1, dtype=torch.int32, device="cuda")
    refs, at = torch.zeros(pages, dtype=torch.int32, device="cuda"), 0
    for i, e in enumerate(each):
        table[i, :e] = ids[at:at + e]
        at += e
    refs[ids[:at].long()] = 1
    k, v = _normal(g, dtype, layers, pages, heads, page, dim), _normal(g, dtype, layers, pages, heads, page, dim)
    return pk.KvCache(k, v, table, _ints(list(lens) + [0] * extra), refs)


APPEND = [
    # dtype, q_heads, kv_heads, dim, page, rotary, interleaved, norm, counts, lens
    ("bf16", 32, 8, 128, 64, 128, False, True, [1], [1]),
    ("bf16", 4, 2, 128, 16, 64, False, True, [1, 1, 1], [17, 16, 900001]),
    ("fp16", 3, 1, 64, 32, 64, True, True, [5, 0, 33, 1], [5, 7, 64, 100]),
    ("fp16", 7, 7, 64, 128, 16, False, False, [40, 300], [129, 300]),
    ("bf16", 8, 1, 128, 16, 0, False, True, [3, 2], [3, 200]),
    ("bf16", 64, 8, 128, 32, 112, False, True, [2, 1], [70, 31]),       # more than three words a thread
    ("fp16", 1, 1, 64, 16, 32, True, False, [16, 17, 15], [16, 17, 31]),
    ("bf16", 2, 2, 64, 16, 0, False, False, [4, 4], [4, 40]),
    ("bf16", 2, 2, 64, 16, 64, True, True, [9, 9], [4, 40]),            # rows before position 0
]


@pytest.mark.parametrize("dtype, Hq, H, D, page, rotary, inter, norm, counts, lens", APPEND)
def test_append(pk, kv, dtype, Hq, H, D, page, rotary, inter, norm, counts, lens):
    dt = TYPES[dtype]
    g = _gen(3)
    layers, layer = 3, 1
    c = _filled(pk, lens, page, H, D, dt, layers=layers)
    behind = 2
    starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
    rows = starts[-1] + behind
    wide = _normal(g, dt, rows, (Hq + 2 * H) * D + 24, scale=2.0)
    qkv = wide[:, 8:-16]                                                  # rows apart, still 16-byte aligned
    qbig = torch.full((rows, Hq + 1, D), 7.0, dtype=dt, device="cuda")
    q = qbig[:, :Hq]
    wq, wk = (1 + 0.3 * _normal(g, dt, D).float()).to(dt), (1 + 0.3 * _normal(g, dt, D).float()).to(dt)
    inv = 500000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / max(rotary, 1)) if rotary else None
    k0, v0 = c.k.clone(), c.v.clone()
    c.append(q, qkv, None, _stream(), starts=_ints(starts), q_weight=wq if norm else None, k_weight=wk if norm else None, eps=1e-5, inv_freq=inv,
             interleaved=inter, layer=layer)
    torch.cuda.synchronize()
    pos = torch.cat([torch.arange(n - t, n, device="cuda") for n, t in zip(lens, counts)])
    eq, ek, ev, bq, bk = kv.append(qkv[:starts[-1]].contiguous(), Hq, H, pos, wq if norm else None, wk if norm else None, float(np.float32(1e-5)), inv, inter)
    half = torch.finfo(dt).eps / 2
    real = pos >= 0

    def near(got, want, both):
        assert bool(((got.double() - want).abs() <= half * want.abs() + (1 + half) * (2.0 ** -17 + 2.0 ** -21) * both + 2.0 ** -25).all())

    near(q[:starts[-1]][real], eq[real], bq[real])
    assert bool((q[:starts[-1]][~real] == 7).all()) and bool((q[starts[-1]:] == 7).all()) and bool((qbig[:, Hq:] == 7).all())
    seq = torch.cat([torch.full((t,), i, device="cuda") for i, t in enumerate(counts)]).long()
    where = c.page_table.long()[seq, (pos // page).clamp(min=0)]
    slot = pos % page
    near(c.k[layer][where[real], :, slot[real]], ek[real], bk[real])
    assert torch.equal(c.v[layer][where[real], :, slot[real]].double(), ev[real])
    touched = torch.zeros(c.k.shape[:4], dtype=torch.bool, device="cuda")
    touched[layer, where[real], :, slot[real]] = True
    assert torch.equal(c.k[~touched], k0[~touched]) and torch.equal(c.v[~touched], v0[~touched])
    c.destroy()


def test_append_passes_padding_and_missing_pages_over(pk, kv):
    c = _filled(pk, [20, 33, 5], 16, 2, 64, torch.bfloat16, extra=1)
    c.page_table[0, 1], c.page_table[1, 2] = -1, 10 ** 6
    k0, v0 = c.k.clone(), c.v.clone()
    q = torch.full((6, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    qkv = _normal(_gen(1), torch.bfloat16, 6, 8 * 64)
    c.append(q, qkv, _ints([0, -1, 1, 4, 3, 2]), _stream())              # 3 is empty: position -1
    torch.cuda.synchronize()
    touched = [bool((q[i] != 7).any()) for i in range(6)]
    assert touched == [True, False, True, False, False, True]
    page = int(c.page_table[2, 0])
    assert torch.equal(c.k[0, page, :, 4], qkv[5].view(8, 64)[4:6]) and torch.equal(c.v[0, page, :, 4], qkv[5].view(8, 64)[6:])
    k0[0, page, :, 4], v0[0, page, :, 4] = c.k[0, page, :, 4], c.v[0, page, :, 4]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)
    c.destroy()


def test_append_far_positions_keep_their_angle(pk, kv):
    """At position 2^30 an fp32 angle would be off by whole turns."""
    page, dt = 128, torch.float16
    n = 1 << 30
    g = _gen(0)
    k = _normal(g, dt, 1, 2, 1, page, 64)
    table = torch.full((1, n // page), -1, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    c = pk.KvCache(k, k.clone(), table, _ints([n]), _ints([0, 1]))
    inv = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64, device="cuda") / 64)
    q, qkv = torch.empty(1, 1, 64, dtype=dt, device="cuda"), _normal(g, dt, 1, 3 * 64)
    c.append(q, qkv, None, _stream(), inv_freq=inv)
    eq, _, _, bq, _ = kv.append(qkv, 1, 1, torch.tensor([n - 1], device="cuda"), None, None, 0.0, inv, False)
    # the fp64 product is off by 2^-53 of 2^30: 2^-23
    assert bool(((q.double() - eq).abs() <= 2.0 ** -11 * eq.abs() + (2.0 ** -17 + 2.0 ** -21) * bq).all())
    c.destroy()


# ------------------------------------------------------------------------------------------------------ attention
def _attend(pk, c, q, seqs, starts, n, shared=None, scale=None, scratch=None, out=None, layer=0):
    rows, heads = q.shape[:2]
    if scratch is None:
        scratch = torch.zeros(c.attention_scratch_bytes(rows, n, heads), dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full((rows, heads, c.dim), 7.0, dtype=q.dtype, device="cuda")
    c.attention(out, q, seqs, _stream(), scratch=scratch, starts=starts, shared_len=None if shared is None else _ints([shared]), scale=scale, layer=layer)
    torch.cuda.synchronize()
    return out


def _check(kv, c, q, out, seqs, starts, scale=None, layer=0):
    scale = float(np.float32(c.dim ** -0.5 if scale is None else scale))
    table, lens = c.page_table.cpu().numpy(), c.lens.cpu().numpy()
    lens = np.minimum(lens, table.shape[1] * c.k.shape[3])
    want, size, big = kv.attention(q, c.k[layer], c.v[layer], table, lens, seqs, starts, scale)
    half = torch.finfo(q.dtype).eps / 2
    longest = int(lens.max())
    vmax = float(c.v[layer][torch.isfinite(c.v[layer])].abs().max())
    inner = half + 2 * c.dim * 2.0 ** -24 * big + (longest + 64) * 2.0 ** -24
    bound = half * want.abs() + (1 + half) * inner * size + (longest * 2.0 ** -25 * vmax + 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -126)
    mine = ~want[:, 0, 0].isnan()
    assert bool((out[~mine] == 7).all()), "rows of no sequence were written"
    off = ((out.double() - want).abs() / bound)[mine]
    worst = float(off.max()) if off.numel() else 0.0                          # NaN stays NaN and fails
    assert worst <= 1.0


SHAPES = [("bf16", 32, 8, 128, 64), ("fp16", 7, 1, 64, 16), ("bf16", 6, 2, 64, 128), ("fp16", 8, 8, 128, 32), ("bf16", 20, 1, 128, 16), ("fp16", 64, 2, 64, 16)]


@pytest.mark.parametrize("dtype, Hq, H, D, page", SHAPES)
@pytest.mark.parametrize("lens", [[1], [0], [15, 16, 17], [64, 65, 63, 128, 129, 127, 1, 0, 500], [3000, 1, 777]])
def test_single_tokens(pk, kv, dtype, Hq, H, D, page, lens):
    c = _filled(pk, lens, page, H, D, TYPES[dtype], layers=2)
    q = _normal(_gen(5), TYPES[dtype], len(lens), Hq, D, scale=2.0)
    out = _attend(pk, c, q, None, None, len(lens), layer=1)
    _check(kv, c, q, out, list(range(len(lens))), list(range(len(lens) + 1)), layer=1)
    c.destroy()


@pytest.mark.parametrize("dtype, Hq, H, D, page", SHAPES)
@pytest.mark.parametrize("counts, lens", [([4, 0, 9, 1], [4, 5, 33, 1]), ([30, 2], [21, 2]), ([130, 5, 260], [130, 400, 1000]), ([17], [17])])
def test_several_tokens_of_a_sequence(pk, kv, dtype, Hq, H, D, page, counts, lens):
    c = _filled(pk, lens, page, H, D, TYPES[dtype])
    starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
    q = _normal(_gen(6), TYPES[dtype], starts[-1] + 3, Hq, D, scale=1.5)      # three rows behind the last sequence
    out = _attend(pk, c, q, None, _ints(starts), len(lens))
    _check(kv, c, q, out, list(range(len(lens))), starts)
    c.destroy()


def _share(c, lens, shared):
    """All sequences get the first one's pages for their first `shared` positions (those that are longer)."""
    page = c.k.shape[3]
    for i, n in enumerate(lens):
        if n >= shared:
            c.page_table[i, :shared // page] = c.page_table[0, :shared // page]


@pytest.mark.parametrize("dtype, Hq, H, D, page", SHAPES)
@pytest.mark.parametrize("shared, counts, lens", [
    (256, [1] * 5, [257, 300, 256 + 16, 1000, 257]),
    (128, [1] * 70, [129 + 3 * i for i in range(70)]),
    (384, [1, 3, 0, 1, 8, 40, 2], [385, 400, 390, 200, 900, 500, 384]),     # one shorter, one with no row, one that just ends there
    (1280, [2, 90, 1], [1300, 1400, 1281]),
    (4096, [1] * 3, [4097, 4100, 5000]),
])
def test_shared_prefix(pk, kv, dtype, Hq, H, D, page, shared, counts, lens):
    c = _filled(pk, lens, page, H, D, TYPES[dtype])
    _share(c, lens, shared)
    starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
    q = _normal(_gen(7), TYPES[dtype], starts[-1], Hq, D, scale=2.0)
    # a length inside a page is honoured up to the page's start
    for said in (shared, shared + page // 2 if min(n for n in lens if n >= shared) > shared + page else shared):
        out = _attend(pk, c, q, None, _ints(starts), len(lens), shared=said)
        _check(kv, c, q, out, list(range(len(lens))), starts)
    c.destroy()


def test_padding_repeated_sequences_and_scratch_that_is_used_again(pk, kv):
    lens = [200, 40, 0, 333]
    c = _filled(pk, lens, 16, 2, 64, torch.bfloat16, extra=2)
    _share(c, lens, 64)                                                   # what shared_len promises
    scratch = torch.zeros(c.attention_scratch_bytes(40, 9, 8), dtype=torch.uint8, device="cuda")
    for seqs, counts in (([3, -1, 0, 3, 9, 2], [1, 2, 3, 4, 1, 2]), ([1], [40]), ([0, 0, 0, 0, 1, 1, 3, 3, 5], [1] * 9), ([-1, -1], [2, 2])):
        starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
        q = _normal(_gen(8), torch.bfloat16, starts[-1], 8, 64)
        out = _attend(pk, c, q, _ints(seqs), _ints(starts), len(seqs), scratch=scratch, shared=64)
        _check(kv, c, q, out, seqs, starts)
    c.destroy()


def test_scratch_serves_calls_of_other_sizes_in_turn(pk, kv):
    """What one call leaves in its partial results must not be where a later, larger call counts."""
    lens = [700 + 13 * i for i in range(40)]
    c = _filled(pk, lens, 16, 4, 64, torch.bfloat16)
    scratch = torch.zeros(c.attention_scratch_bytes(40 * 9, 40, 16), dtype=torch.uint8, device="cuda")
    for seqs, count in (([39], 1), (list(range(40)), 1), ([0, 1], 9), (list(range(40)), 9), ([5, 6, 7], 1), (list(range(40)), 1)):
        starts = [count * i for i in range(len(seqs) + 1)]
        q = _normal(_gen(31), torch.bfloat16, starts[-1], 16, 64)
        out = _attend(pk, c, q, _ints(seqs), None if count == 1 else _ints(starts), len(seqs), scratch=scratch)
        _check(kv, c, q, out, seqs, starts)
    c.destroy()


@pytest.mark.parametrize("shared", [None, 64])
def test_as_many_sequences_as_a_call_takes(pk, kv, shared):
    lens = [65 + (i * 37) % 200 for i in range(pk.ATTENTION_MAX_SEQS)]
    c = _filled(pk, lens, 64, 1, 64, torch.float16)
    _share(c, lens, 64)
    q = _normal(_gen(32), torch.float16, len(lens), 2, 64)
    out = _attend(pk, c, q, None, None, len(lens), shared=shared)
    _check(kv, c, q, out, list(range(len(lens))), list(range(len(lens) + 1)))
    c.destroy()


def test_a_prefix_whose_results_do_not_fit_the_scratch_is_read_by_each_sequence(pk, kv):
    """720 x 64 key heads x 2 row groups leave more results than the scratch takes: the call goes without the prefix."""
    n, H, G, D, t = 720, 64, 8, 64, 3
    lens = [66 + i % 5 for i in range(n)]
    c = _filled(pk, lens, 64, H, D, torch.bfloat16)
    _share(c, lens, 64)
    starts = [t * i for i in range(n + 1)]
    q = _normal(_gen(34), torch.bfloat16, starts[-1], H * G, D)
    out = _attend(pk, c, q, None, _ints(starts), n, shared=64)
    some = [0, 1, 17, 359, 700, 719]
    rows = [starts[i] + j for i in some for j in range(t)]
    table = c.page_table[some].contiguous()
    small = pk.KvCache(c.k, c.v, table, _ints([lens[i] for i in some]), c.refs)
    _check(kv, small, q[rows], out[rows], list(range(len(some))), [t * i for i in range(len(some) + 1)])
    assert bool(torch.isfinite(out).all()) and not bool((out == 7).any())
    c.destroy()
    small.destroy()


def test_missing_pages_are_left_out(pk, kv):
    lens = [300, 64, 20]
    c = _filled(pk, lens, 16, 2, 128, torch.float16)
    c.page_table[0, 3], c.page_table[0, 18], c.page_table[1, :4], c.page_table[2, 0] = -1, 10 ** 7, -5, -1
    q = _normal(_gen(9), torch.float16, 3, 4, 128)
    _check(kv, c, q, _attend(pk, c, q, None, None, 3), [0, 1, 2], [0, 1, 2, 3])
    q = _normal(_gen(9), torch.float16, 84, 4, 128)
    starts = [0, 40, 64, 84]
    _check(kv, c, q, _attend(pk, c, q, None, _ints(starts), 3), [0, 1, 2], starts)
    c.destroy()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("count", [1, 5, 200])
@pytest.mark.parametrize("Hq", [2, 8])
def test_what_a_row_does_not_see_may_hold_anything(pk, kv, dtype, count, Hq):
    lens = [205, 230]
    c = _filled(pk, lens, 64, 2, 64, TYPES[dtype])
    q = _normal(_gen(10), TYPES[dtype], 2 * count, Hq, 64)
    starts = [0, count, 2 * count]
    clean = _attend(pk, c, q, None, _ints(starts), 2)
    for i, n in enumerate(lens):                                          # behind the end of the last page
        last = int(c.page_table[i, n // 64])
        c.k[0, last, :, n % 64:], c.v[0, last, :, n % 64:] = float("nan"), float("inf")
    assert torch.equal(_attend(pk, c, q, None, _ints(starts), 2), clean)
    if count > 1:                                                         # later tokens: earlier rows do not notice
        for i, n in enumerate(lens):
            last = int(c.page_table[i, (n - 2) // 64])
            c.k[0, last, :, (n - 2) % 64], c.v[0, last, :, (n - 2) % 64, 3] = float("nan"), float("-inf")
        got = _attend(pk, c, q, None, _ints(starts), 2)
        for a, b in zip(starts, starts[1:]):
            unseen = [r for r in range(a, b - 2)]
            bound = 2 * torch.finfo(TYPES[dtype]).eps * clean[unseen].float().abs() + 2.0 ** -6
            assert bool(((got[unseen].float() - clean[unseen].float()).abs() <= bound).all()), "finite rows changed"
            assert bool(got[b - 2:b].isnan().any(-1).all())
    c.destroy()


def test_scores_that_overflow_a_sixteen_bit_type_and_equal_scores(pk, kv):
    c = _filled(pk, [700, 33], 32, 1, 64, torch.bfloat16)
    q = _normal(_gen(11), torch.bfloat16, 2, 3, 64, scale=300.0)             # scores of thousands
    _check(kv, c, q, _attend(pk, c, q, None, None, 2, scale=0.5), [0, 1], [0, 1, 2], scale=0.5)
    q.zero_()
    _check(kv, c, q, _attend(pk, c, q, None, None, 2), [0, 1], [0, 1, 2])
    q = _normal(_gen(11), torch.bfloat16, 2, 3, 64)
    _check(kv, c, q, _attend(pk, c, q, None, None, 2, scale=-0.125), [0, 1], [0, 1, 2], scale=-0.125)
    _check(kv, c, q, _attend(pk, c, q, None, None, 2, scale=0.0), [0, 1], [0, 1, 2], scale=0.0)
    c.destroy()


def test_strided_rows(pk, kv):
    c = _filled(pk, [90, 300, 17], 16, 2, 64, torch.float16)
    wide = _normal(_gen(12), torch.float16, 3, 6 + 4, 64)
    q = wide[:, 2:8]
    big = torch.full((3, 9, 64), 7.0, dtype=torch.float16, device="cuda")
    out = _attend(pk, c, q, None, None, 3, out=big[:, 1:7])
    _check(kv, c, q, out, [0, 1, 2], [0, 1, 2, 3])
    assert bool((big[:, 0] == 7).all()) and bool((big[:, 7:] == 7).all())
    c.destroy()


def test_pools_behind_four_gigabytes(pk, kv):
    """Pages whose byte offsets pass 32 bits: 2 x 4.8 GB, the sequence on the last ones."""
    pages, heads, page, dim = 18400, 8, 128, 128
    k = torch.empty(1, pages, heads, page, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    last = list(range(pages - 6, pages))
    k[:, last], v[:, last] = _normal(_gen(13), torch.bfloat16, 1, 6, heads, page, dim), _normal(_gen(14), torch.bfloat16, 1, 6, heads, page, dim)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[last[:4]] = 1
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    table[0] = _ints(last[:4])
    c = pk.KvCache(k, v, table, _ints([450, 0]), refs)
    q, inv = torch.empty(1, 32, dim, dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.float64, device="cuda")
    qkv = _normal(_gen(15), torch.bfloat16, 1, 48 * dim)
    c.append(q, qkv, _ints([0]), _stream(), inv_freq=inv)
    assert torch.equal(v[0, last[3], :, 449 - 384].reshape(-1), qkv[0, 40 * dim:])
    out = _attend(pk, c, q, _ints([0]), None, 1)
    small = pk.KvCache(k[:, last].contiguous(), v[:, last].contiguous(), _ints([[0, 1, 2, 3], [-1] * 4]), _ints([450, 0]), _ints([1, 1, 1, 1, 0, 0]))
    assert torch.equal(out, _attend(pk, small, q, _ints([0]), None, 1))
    _check(kv, small, q, out, [0], [0, 1])
    c.copy(_ints([last[0]]), _ints([last[5]]), _stream())
    assert torch.equal(k[0, last[5]], k[0, last[0]]) and torch.equal(v[0, last[5]], v[0, last[0]])
    c.compact(_stream())
    assert c.page_table[0].tolist() == [0, 1, 2, 3] and torch.equal(k[0, :4], small.k[0, :4])
    c.destroy()
    small.destroy()


# ----------------------------------------------------------------------------------------- tasks, streams, graphs
def test_attention_task_stops_and_resumes_with_the_same_bytes(pk, kv):
    lens = [9000, 4000, 300, 12000]
    c = _filled(pk, lens, 64, 4, 128, torch.bfloat16)
    _share(c, lens, 256)
    counts = [1, 30, 4, 1]
    starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
    q = _normal(_gen(16), torch.bfloat16, starts[-1], 16, 128)
    for shared in (None, 256):
        want = _attend(pk, c, q, None, _ints(starts), 4, shared=shared)
        _check(kv, c, q, want, [0, 1, 2, 3], starts)
        out = torch.zeros_like(q)
        scratch = torch.empty(c.attention_scratch_bytes(starts[-1], 4, 16), dtype=torch.uint8, device="cuda").fill_(0xA5)
        word = None if shared is None else _ints([shared])
        t = pk.Task.attention(c, out, q, None, scratch=scratch, starts=_ints(starts), shared_len=word)
        assert t.query().status == pk.STATUS_IDLE
        for _ in range(2):
            out.zero_()
            cuts = 0
            for _ in range(5):
                t.launch(_stream(), sm_limit=1)
                t.set_flag(1)
                info = t.wait()
                torch.cuda.synchronize()
                t.set_flag(0)
                torch.cuda.synchronize()
                assert info.status in (pk.STATUS_PREEMPTED, pk.STATUS_COMPLETED)
                if info.status == pk.STATUS_COMPLETED:
                    break
                cuts += 1
            while t.query().status != pk.STATUS_COMPLETED:
                t.launch(_stream())
                t.wait()
            assert cuts > 0
            info = t.query()
            assert info.tiles_done == info.tiles_total > 0
            assert torch.equal(out, want)
        # stopped halfway, rewound, and run from the start
        t.launch(_stream(), sm_limit=1)
        t.set_flag(1)
        t.wait()
        torch.cuda.synchronize()
        t.set_flag(0)
        t.reset(_stream())
        out.zero_()
        t.launch(_stream())
        assert t.wait().status == pk.STATUS_COMPLETED and torch.equal(out, want)
        # a launch that finds the flag up does nothing
        t.set_flag(1)
        torch.cuda.synchronize()
        out.zero_()
        t.launch(_stream())
        assert t.wait().status == pk.STATUS_PREEMPTED and not bool(out.any())
        t.set_flag(0)
        torch.cuda.synchronize()
        t.launch(_stream())
        assert t.wait().status == pk.STATUS_COMPLETED and torch.equal(out, want)
        t.destroy()
    c.destroy()


@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [1, 30, 4, 1]])
def test_a_flag_that_goes_up_and_down_while_the_kernel_runs(pk, kv, counts):
    """A warp that saw the flag up has left tickets behind: it must not go on to a merge that waits for them once the flag is down."""
    lens = [9000, 4000, 300, 12000]
    c = _filled(pk, lens, 64, 4, 128, torch.bfloat16)
    starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
    q = _normal(_gen(33), torch.bfloat16, starts[-1], 16, 128)
    want = _attend(pk, c, q, None, _ints(starts), 4)
    out = torch.zeros_like(q)
    scratch = torch.zeros(c.attention_scratch_bytes(starts[-1], 4, 16), dtype=torch.uint8, device="cuda")
    t = pk.Task.attention(c, out, q, None, scratch=scratch, starts=_ints(starts))
    for _ in range(30):
        out.zero_()
        while True:
            t.launch(_stream())
            t.set_flag(1)
            t.set_flag(0)
            info = t.wait()
            torch.cuda.synchronize()
            assert info.status in (pk.STATUS_PREEMPTED, pk.STATUS_COMPLETED) and info.error == 0
            if info.status == pk.STATUS_COMPLETED:
                break
        assert torch.equal(out, want)
    t.destroy()
    c.destroy()


def test_two_streams_with_scratch_of_their_own(pk, kv):
    lens = [3000, 2500, 100]
    c = _filled(pk, lens, 16, 2, 64, torch.bfloat16)
    q = _normal(_gen(17), torch.bfloat16, 3, 8, 64)
    want = _attend(pk, c, q, None, None, 3)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.zeros_like(q) for _ in streams]
    scratch = [torch.zeros(c.attention_scratch_bytes(3, 3, 8), dtype=torch.uint8, device="cuda") for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o, w in zip(streams, outs, scratch):
            c.attention(o, q, None, s.cuda_stream, scratch=w)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    c.destroy()


def test_a_decode_step_in_a_graph_follows_the_lengths(pk, kv):
    """extend, append and attention captured once, replayed while the sequences grow over page borders; against a run without a graph."""
    Hq, H, D, page, layers, n = 8, 2, 64, 16, 2, 3
    lens = [30, 47, 1]
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    wq = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    seqs, one = _ints([0, 1, 2]), _ints([1, 1, 1])
    runs = []
    for graphed in (False, True):
        c = _filled(pk, lens, page, H, D, torch.bfloat16, layers=layers, seed=2)
        pad = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
        pad[:, :c.page_table.shape[1]] = c.page_table
        grown = pk.KvCache(torch.cat([c.k, torch.zeros(layers, 20, H, page, D, dtype=c.k.dtype, device="cuda")], 1),
                           torch.cat([c.v, torch.zeros(layers, 20, H, page, D, dtype=c.k.dtype, device="cuda")], 1), pad, c.lens, torch.cat([c.refs, _ints([0] * 20)]))
        qkv = torch.zeros(layers, n, (Hq + 2 * H) * D, dtype=torch.bfloat16, device="cuda")
        q = torch.zeros(n, Hq, D, dtype=torch.bfloat16, device="cuda")
        out = torch.zeros(layers, n, Hq, D, dtype=torch.bfloat16, device="cuda")
        scratch = torch.zeros(grown.attention_scratch_bytes(n, n, Hq), dtype=torch.uint8, device="cuda")

        def step():
            s = _stream()
            grown.extend(seqs, one, s)
            for layer in range(layers):
                grown.append(q, qkv[layer], seqs, s, q_weight=wq, k_weight=wq, inv_freq=inv, layer=layer)
                grown.attention(out[layer], q, seqs, s, scratch=scratch, layer=layer)

        graph = None
        if graphed:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        g, got = _gen(21), []
        for _ in range(25):
            qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=g))
            graph.replay() if graphed else step()
            got.append(out.clone())
        torch.cuda.synchronize()
        assert grown.lens.tolist() == [55, 72, 26]
        _check(kv, grown, q, out[1], [0, 1, 2], [0, 1, 2, 3], layer=1)
        runs.append((got, grown.page_table.clone(), grown.k.clone(), grown.v.clone()))
        del graph
        c.destroy()
        grown.destroy()
    assert all(torch.equal(a, b) for a, b in zip(runs[0][0], runs[1][0]))
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1:], runs[1][1:]))


# -------------------------------------------------------------------------------------------------------- refusals
def test_refusals(pk, kv):
    import ctypes as C
    c = _filled(pk, [20, 30], 16, 2, 64, torch.bfloat16)
    q, out = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    scratch = torch.zeros(c.attention_scratch_bytes(2, 2, 4), dtype=torch.uint8, device="cuda")
    s = _stream()
    base = c._attention_args(out, q, None, None, None, scratch, 0, None)
    for field, value, code in (("q", 0, 1), ("out", 0, 1), ("scratch", 0, 1), ("n", 0, 1), ("rows", 0, 1), ("layer", 1, 1), ("q_heads", 3, 4), ("n", 1025, 7),
                               ("rows", 1 << 30, 7), ("scratch_bytes", base.scratch_bytes - 1, 1), ("q", base.q + 8, 2), ("scratch", base.scratch + 128, 2),
                               ("q_stride", 8, 1), ("q_stride", 260, 2), ("out_stride", 257, 2), ("scale", float("nan"), 1)):
        a = pk.AttentionArgs.from_buffer_copy(base)
        setattr(a, field, value)
        assert pk.lib.xpkAttention(c.handle, C.byref(a), s) == code, field
        h = C.c_void_p(5)
        assert pk.lib.xpkTaskCreateAttention(C.byref(h), c.handle, C.byref(a), 0, None) == code and h.value == 5
    qkv = torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device="cuda")
    inv = torch.ones(32, dtype=torch.float64, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    base = pk.KvAppendArgs(q.data_ptr(), qkv.data_ptr(), 0, 0, None, None, w.data_ptr(), w.data_ptr(), inv.data_ptr(), 1e-6, 2, 2, 4, 0, 64, 0)
    for field, value, code in (("q", 0, 1), ("qkv", 0, 1), ("n", 0, 1), ("rows", 0, 1), ("layer", 1, 1), ("q_heads", 0, 1), ("inv_freq", 0, 1), ("rotary", 24, 4),
                               ("rotary", 80, 4), ("k_weight", 0, 4), ("eps", -1.0, 1), ("qkv", base.qkv + 2, 2), ("qkv_stride", 504, 1), ("q_stride", 260, 2),
                               ("inv_freq", base.inv_freq + 4, 2)):
        a = pk.KvAppendArgs.from_buffer_copy(base)
        setattr(a, field, value)
        assert pk.lib.xpkKvAppend(c.handle, C.byref(a), s) == code, field
    ids = torch.zeros(4000, dtype=torch.int32, device="cuda")
    for call in (pk.lib.xpkKvFork, pk.lib.xpkKvExtend):
        assert call(c.handle, ids.data_ptr(), ids.data_ptr(), 0, s) == 1 and call(c.handle, None, ids.data_ptr(), 1, s) == 1
        assert call(c.handle, ids.data_ptr(), ids.data_ptr(), 2049, s) == 7 and call(c.handle, ids.data_ptr() + 2, ids.data_ptr(), 1, s) == 2
    assert pk.lib.xpkKvFree(c.handle, None, 1, s) == 1 and pk.lib.xpkKvCopy(c.handle, ids.data_ptr(), None, 1, s) == 1
    with pytest.raises(ValueError):
        c.attention(out, q.half(), None, s, scratch=scratch)
    with pytest.raises(ValueError):
        c.attention(out, q, ids[:1].long(), s, scratch=scratch)
    with pytest.raises(ValueError):
        c.attention(out, q, ids[:1], s, scratch=scratch)
    with pytest.raises(ValueError):
        c.attention(out, q, ids[:2], s, scratch=scratch, starts=ids[:2])
    with pytest.raises(ValueError):
        c.append(q, qkv[:1], None, s)
    with pytest.raises(ValueError):
        c.extend(ids[:2], ids[:3], s)
    with pytest.raises(pk.XpkError):
        c.attention(out, q, None, s, scratch=scratch[:512])
    torch.cuda.synchronize()
    assert not bool(out.any()) and not bool(scratch.any())
    c.destroy()


# ------------------------------------------------------------------------------------------------- in the decode workload
def test_paged_decode_step_equals_attention_over_each_request_by_itself(pk, kv):
    """PagedCache of the decode workload: forks of one prompt that grow at different times, one of them ends and another takes its
    place; each step's attention against the definition, and nothing is left of the pages at the end."""
    from xsched_b200 import llama_decode as ld
    g = _gen(30)
    c = ld.PagedCache(g, 2, 100, 4, 40, torch.device("cuda"))
    live, table = [], lambda: c.cache.page_table.cpu().numpy()
    for step in range(30):
        if step in (0, 3, 20):
            new = {0: [1, 2], 3: [3], 20: [2, 4]}[step]
            c.start(_ints(new))
            live += new
        if step == 15:
            c.stop(_ints([2]))
            live.remove(2)
            c.compact()
        seqs = _ints(live)
        c.extend(seqs)
        for layer in range(2):
            qkv = _normal(g, torch.bfloat16, len(live), (ld.NQ + 2 * ld.NKV) * ld.HD)
            out = c.step(layer, qkv, seqs)
            if step % 7 == 1:
                lens = c.cache.lens.cpu().numpy()
                want, size, big = kv.attention(c.q[:len(live)], c.k[layer], c.v[layer], table(), lens, live, list(range(len(live) + 1)), float(np.float32(ld.HD ** -0.5)))
                bound = 2.0 ** -8 * want.abs() + 1.004 * (2.0 ** -8 + 2 * ld.HD * 2.0 ** -24 * big + 300 * 2.0 ** -24) * size + 2.0 ** -126
                assert float(((out.double() - want).abs() / bound).max()) <= 1.0
    assert c.cache.lens.tolist() == [100, 130, 110, 127, 110]
    c.stop(_ints([1, 2, 3, 4]))
    assert c.cache.refs.sum().item() == 2 and c.cache.lens.tolist() == [100, 0, 0, 0, 0]
    c.cache.destroy()


def test_decode_workload_runs_paged():
    import json
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-m", "xsched_b200.llama_decode", "--requests", "6", "--tokens", "5", "--rate", "200", "--layers", "2", "--kv", "300",
                        "--batched", "--max-batch", "4", "--paged"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    line = json.loads(r.stdout.strip().splitlines()[-1])
    assert line["mode"] == "batched, paged" and line["requests"] == 6 and line["tokens"] == 30
