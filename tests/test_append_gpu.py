"""Append with rows enough for the form that takes four rows a CTA (test_kv_gpu.py has the form with one), and the two against each
other."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_kv_gpu import TYPES, _filled, _gen, _ints, _normal, _stream, kv, pk      # noqa: E402,F401
from test_kv_gpu import test_append as _appended                                    # noqa: E402

FOUR = 8                    # rows a multiprocessor from which a CTA takes four


@pytest.mark.parametrize("dtype, Hq, H, D, page, rotary, inter, norm", [
    ("bf16", 4, 2, 128, 64, 128, False, True), ("fp16", 3, 1, 64, 16, 64, True, True), ("fp16", 7, 7, 64, 128, 16, False, False),
    ("bf16", 64, 8, 128, 32, 112, False, True), ("bf16", 2, 2, 64, 16, 0, False, True), ("fp16", 1, 1, 128, 32, 32, True, False)])
@pytest.mark.parametrize("counts, lens", [([700, 1, 0, 601, 2], [700, 50, 3, 9001, 1]), ([1] * 1283, [1 + 7 * i % 300 for i in range(1283)]),
                                          ([1300], [1297])])          # three rows before position 0
def test_append_of_many_rows(pk, kv, dtype, Hq, H, D, page, rotary, inter, norm, counts, lens):
    assert sum(counts) >= FOUR * torch.cuda.get_device_properties(0).multi_processor_count
    _appended(pk, kv, dtype, Hq, H, D, page, rotary, inter, norm, counts, lens)


@pytest.mark.parametrize("dtype, D, inter", [("bf16", 128, False), ("fp16", 64, True)])
def test_rows_get_the_same_bytes_in_a_large_call_and_in_small_ones(pk, kv, dtype, D, inter):
    """With padding and missing pages, which are passed over in both."""
    n, Hq, H, page = 1501, 6, 2, 16
    lens = [(i * 37) % 400 for i in range(n)]
    dt = TYPES[dtype]
    c = _filled(pk, lens, page, H, D, dt)
    c.page_table[5::11, 0] = -1
    seqs = torch.arange(n, dtype=torch.int32, device="cuda")
    seqs[3::29] = -1
    qkv = _normal(_gen(50), dt, n, (Hq + 2 * H) * D)
    w = (1 + 0.3 * _normal(_gen(51), dt, D).float()).to(dt)
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    k0, v0 = c.k.clone(), c.v.clone()
    got = []
    for step in (n, 400):
        c.k.copy_(k0), c.v.copy_(v0)
        q = torch.full((n, Hq, D), 7.0, dtype=dt, device="cuda")
        for a in range(0, n, step):
            b = min(a + step, n)
            c.append(q[a:b], qkv[a:b], seqs[a:b].contiguous(), _stream(), q_weight=w, k_weight=w, inv_freq=inv, interleaved=inter)
        torch.cuda.synchronize()
        got.append((q, c.k.clone(), c.v.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    untouched = (seqs < 0) | (_ints(lens) == 0)
    assert bool((got[0][0][untouched] == 7).all()) and not bool((got[0][0][~untouched] == 7).all(-1).any())
    c.destroy()
