"""The CPU restatement of the key/value cache's operators against small worked examples, and the refusals of
xpkKvCacheCreate and the Python face that need no GPU."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import kv


def _pages(table, lens, refs, page=4):
    pool = np.arange(2 * len(refs) * 2, dtype=np.int64).reshape(2, len(refs), 2)
    return kv.Pages(np.array(table), np.array(lens), np.array(refs), [pool], page)


def test_fork_then_extend_copies_the_shared_last_page_except_for_its_last_holder():
    p = _pages([[3, 1, -1], [-1] * 3, [-1] * 3], [6, 0, 0], [0, 1, 0, 1, 0, 0])
    p.fork([0, 0, 0, 9], [1, 2, 1, 2])
    assert p.table.tolist() == [[3, 1, -1]] * 3 and p.lens.tolist() == [6, 6, 6] and p.refs.tolist() == [0, 3, 0, 3, 0, 0]
    before = p.pools[0][:, 1].copy()
    assert p.extend([1, 2, 1, -1, 0], [1, 3, 5, 1, 1]) == (2, 0, 0)
    # sequence 1: page 0 copied from 1; sequence 2: page 2 copied and page 4 new; sequence 0 keeps page 1
    assert p.table.tolist() == [[3, 1, -1], [3, 0, -1], [3, 2, 4]]
    assert p.lens.tolist() == [7, 7, 9] and p.refs.tolist() == [1, 1, 1, 3, 1, 0]
    assert (p.pools[0][:, 0] == before).all() and (p.pools[0][:, 2] == before).all()


def test_extend_changes_nothing_when_pages_are_missing_or_the_table_is_too_narrow():
    p = _pages([[0, -1], [-1, -1]], [4, 0], [1, 0])
    state = [x.copy() for x in (p.table, p.lens, p.refs)]
    assert p.extend([0, 1], [1, 1]) == (0, 1, 0)
    assert p.extend([0], [5]) == (0, 0, 1)
    assert all((a == b).all() for a, b in zip(state, (p.table, p.lens, p.refs)))


def test_free_and_compact():
    p = _pages([[5, 2], [4, 2], [1, -1]], [8, 8, 3], [0, 1, 2, 0, 1, 1])
    p.free([2, 2, -1, 7])
    assert p.refs.tolist() == [0, 0, 2, 0, 1, 1] and p.lens.tolist() == [8, 8, 0] and p.table[2].tolist() == [-1, -1]
    five = p.pools[0][:, 5].copy()
    assert p.compact() == (2, 3)
    assert p.table.tolist() == [[1, 2], [0, 2], [-1, -1]] and p.refs.tolist() == [1, 1, 2, 0, 0, 0]
    assert (p.pools[0][:, 1] == five).all()


def test_attention_of_one_position_is_its_value_and_an_empty_row_is_zero():
    k, v = torch.randn(2, 1, 4, 8), torch.randn(2, 1, 4, 8)
    table = np.array([[1, -1], [0, -1]])
    out, _, _ = kv.attention(torch.randn(4, 2, 8), k, v, table, np.array([1, 0]), [0, 1, -1], [0, 2, 3, 4], 0.3)
    assert out[0].abs().max() == 0 and out[2].abs().max() == 0          # before position 0; an empty sequence
    assert torch.allclose(out[1], v[1, 0, 0].double().expand(2, 8))
    assert out[3].isnan().all()                                           # padding


def test_append_keeps_lengths_of_turned_pairs():
    x = torch.randn(3, 4 * 8, dtype=torch.float64)
    inv = 10000.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
    for inter in (False, True):
        q, k, v, _, _ = kv.append(x, 2, 1, torch.tensor([0, 5, 700000]), None, None, 0.0, inv, inter)
        y = x.view(3, 4, 8)
        assert torch.allclose(q[0], y[0, :2]) and torch.equal(v, y[:, 3:])
        assert torch.allclose(q.square().sum(-1), y[:, :2].square().sum(-1))
    q, _, _, _, _ = kv.append(x, 2, 1, torch.tensor([1, 1, 1]), torch.ones(8), torch.ones(8), 0.0, None, False)
    assert torch.allclose(q.square().mean(-1), torch.ones(3, 2, dtype=torch.float64))


@pytest.fixture(scope="module")
def pk():
    from xsched_b200 import pk as _pk
    return _pk


def _desc(pk, **change):
    d = dict(k=0x10000, v=0x20000, page_table=0x30000, lens=0x40000, refs=0x50000, dtype=pk.DTYPE_BF16, layers=2, pages=8, kv_heads=2, page_size=16,
             head_dim=64, seqs=3, table_width=4)
    d.update(change)
    return pk.KvCacheDesc(**d)


@pytest.mark.parametrize("change, code", [
    (dict(k=0), 1), (dict(lens=0), 1), (dict(pages=0), 1), (dict(layers=0), 1), (dict(seqs=0), 1), (dict(table_width=0), 1), (dict(kv_heads=0), 1),
    (dict(dtype=0), 4), (dict(dtype=3), 4), (dict(page_size=8), 4), (dict(page_size=48), 4), (dict(head_dim=96), 4), (dict(head_dim=256), 4),
    (dict(k=0x10008), 2), (dict(v=0x20002), 2), (dict(refs=0x50002), 2),
    (dict(layers=1 << 16, pages=1 << 16), 7), (dict(pages=0xFFFFFFFF), 7),
    (dict(table_width=(1 << 26) + 1), 7), (dict(kv_heads=65537), 7),
])
def test_cache_descriptions_that_are_refused(pk, change, code):
    h = ctypes.c_void_p(77)
    assert pk.lib.xpkKvCacheCreate(ctypes.byref(h), ctypes.byref(_desc(pk, **change))) == code
    assert h.value == 77


def test_null_handles_are_refused(pk):
    lib, one = pk.lib, ctypes.c_void_p(0x1000)
    assert lib.xpkKvCacheCreate(None, ctypes.byref(_desc(pk))) == 1
    assert lib.xpkKvCacheDestroy(None) == 1 and lib.xpkKvFree(None, one, 1, None) == 1 and lib.xpkKvFork(None, one, one, 1, None) == 1
    assert lib.xpkKvExtend(None, one, one, 1, None) == 1 and lib.xpkKvCompact(None, None) == 1 and lib.xpkKvCopy(None, one, one, 1, None) == 1
    assert lib.xpkAttention(None, ctypes.byref(pk.AttentionArgs()), None) == 1 and lib.xpkKvAppend(None, ctypes.byref(pk.KvAppendArgs()), None) == 1
    assert lib.xpkAttentionScratchBytes(None, 1, 1, 1) == 0


def test_python_face_refuses_what_is_not_on_a_gpu_or_of_another_shape(pk):
    k = torch.zeros(1, 4, 2, 16, 64, dtype=torch.bfloat16)
    t, n, r = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for bad in ((k, k, t, n, r), (k.float(), k.float(), t, n, r), (k, k.half(), t, n, r), (k[0], k[0], t, n, r), (k, k, t, n, r.long()),
                (k, k, t, r, r), (k, k, t, n, n)):
        with pytest.raises(ValueError):
            pk.KvCache(*bad)
    x = torch.zeros(4, 6, 8)
    assert pk._rows("x", x, 48) == (4, 0) and pk._rows("x", x[:, :3], 24) == (4, 48) and pk._rows("x", x[::2], 48) == (2, 96)
    with pytest.raises(ValueError):
        pk._rows("x", x[:, :, ::2], 24)
    with pytest.raises(ValueError):
        pk._rows("x", x, 47)


def test_kv_constants_of_header_and_python_face_agree(pk):
    import re
    from pathlib import Path
    text = (Path(pk.__file__).parent.parent / "include" / "xsched_b200" / "pk.h").read_text()
    enums = {m.group(1): int(m.group(2), 0) for m in re.finditer(r"\b(XPK_[A-Z0-9_]+)\s*=\s*(\d+)", text)}
    assert (enums["XPK_KIND_ATTENTION"], enums["XPK_KIND_KV_COPY"]) == (pk.KIND_ATTENTION, pk.KIND_KV_COPY)
    assert (enums["XPK_DTYPE_BF16"], enums["XPK_DTYPE_F16"]) == (pk.DTYPE_BF16, pk.DTYPE_F16)
    defines = {m.group(1): int(m.group(2)) for m in re.finditer(r"#define (XPK_\w+) (\d+)\s", text)}
    assert defines["XPK_KV_MAX_LIST"] == pk.KV_MAX_LIST and defines["XPK_ATTENTION_MAX_SEQS"] == pk.ATTENTION_MAX_SEQS
