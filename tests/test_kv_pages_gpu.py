"""Pages of the key/value cache at sizes where sums and offsets could pass 32 bits, and under streams of their own."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_kv_gpu import _ints, _stream, kv, pk      # noqa: E402,F401


def test_extend_by_more_pages_than_a_32_bit_sum_holds_changes_nothing(pk, kv):
    """512 sequences want 2^22 pages each: 2^31 in all, of which there are 40."""
    n, width, page, pages = 512, 1 << 22, 16, 40
    k = torch.zeros(1, pages, 1, page, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.empty(n, width, dtype=torch.int32, device="cuda")          # 8.6 GB, which nobody reads: all sequences are empty
    c = pk.KvCache(k, torch.zeros_like(k), table, _ints([0] * n), _ints([0] * pages))
    for each in (width, width // 2 + 1, width - 1):
        c.extend(_ints(list(range(n))), _ints([each * page] * n), _stream())
        r = c.result(_stream())
        assert (r.copied, r.missing, r.refused) == (0, 1, 0)                 # as many as are counted: one more than there are
        assert not bool(c.lens.any()) and not bool(c.refs.any())
    c.extend(_ints([3, 7]), _ints([20 * page, 20 * page]), _stream())        # and what fits is given
    assert c.result(_stream()).missing == 0 and c.lens[7].item() == 20 * page and bool((c.refs == 1).all())
    c.destroy()


def test_a_cache_is_ready_for_streams_that_do_not_wait_for_the_default_one(pk, kv):
    """The handle's workspace is cleared when the constructor returns, whatever the default stream is still doing."""
    k = torch.zeros(1, 8, 1, 16, 64, dtype=torch.bfloat16, device="cuda")
    v, refs, lens = torch.zeros_like(k), _ints([1] + [0] * 7), _ints([5, 0, 0])
    table = _ints([[0, -1], [-1, -1], [-1, -1]])
    parents, children = _ints([0, 0]), _ints([1, 2])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        torch.cuda._sleep(1_000_000_000)
        c = pk.KvCache(k, v, table, lens, refs)
        c.fork(parents, children, s.cuda_stream)
        s.synchronize()
        with torch.cuda.stream(s):
            assert lens.tolist() == [5, 5, 5] and refs[0].item() == 3
        c.free(children, s.cuda_stream)
        s.synchronize()
        torch.cuda.synchronize()
        c.destroy()


def test_calls_refuse_tensors_that_require_a_gradient(pk, kv):
    from test_kv_gpu import _filled
    c = _filled(pk, [20, 30], 16, 2, 64, torch.bfloat16)
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    out, qkv, inv = torch.zeros_like(q), torch.ones(2, 8 * 64, dtype=torch.bfloat16, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    scratch = torch.zeros(c.attention_scratch_bytes(2, 2, 4), dtype=torch.uint8, device="cuda")
    grad = lambda x: x.clone().requires_grad_()
    calls = [lambda: c.attention(out, grad(q), None, _stream(), scratch=scratch), lambda: c.attention(grad(out), q, None, _stream(), scratch=scratch),
             lambda: pk.Task.attention(c, out, grad(q), None, scratch=scratch), lambda: c.append(grad(q), qkv, None, _stream()),
             lambda: c.append(q, grad(qkv), None, _stream()), lambda: c.append(q, qkv, None, _stream(), inv_freq=grad(inv)),
             lambda: c.append(q, qkv, None, _stream(), q_weight=grad(w), k_weight=w), lambda: pk.KvCache(grad(c.k), c.v, c.page_table, c.lens, c.refs)]
    for call in calls:
        with pytest.raises(ValueError, match="no_grad"):
            call()
    with torch.no_grad():
        c.append(q, grad(qkv), None, _stream(), inv_freq=inv, q_weight=grad(w), k_weight=w)
        c.attention(out, grad(q), None, _stream(), scratch=scratch)
    torch.cuda.synchronize()
    assert bool(out.any())
    c.destroy()
