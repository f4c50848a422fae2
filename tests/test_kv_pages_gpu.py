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


def test_the_decode_cache_notices_that_its_pages_are_used_up(pk, kv):
    """The decode workload's cache, with room for 28 tokens a request: the step that finds no room any more says so."""
    from xsched_b200 import llama_decode as ld
    prompt, tokens = 100, 28                                                 # to the end of a page: no slack
    c = ld.PagedCache(torch.Generator(device="cuda").manual_seed(0), 1, prompt, 2, tokens, torch.device("cuda"))
    seqs = _ints([1, 2])
    c.start(seqs)
    for _ in range(tokens):
        c.extend(seqs)
        c.check()
    c.extend(seqs)
    with pytest.raises(RuntimeError, match="too small"):
        c.check()
    assert c.cache.lens.tolist() == [prompt, prompt + tokens, prompt + tokens]
    c.stop(_ints([1]))
    c.extend(_ints([2]))
    with pytest.raises(RuntimeError, match="too long"):
        c.check()
    c.cache.destroy()


def test_the_decode_workload_looks_at_every_step(pk, kv, monkeypatch):
    """Its loop stops with an error when a step's extend has found no room."""
    import sys

    from xsched_b200 import llama_decode as ld
    monkeypatch.setattr(sys, "argv", ["llama_decode", "--requests", "3", "--tokens", "80", "--rate", "500", "--layers", "1", "--kv", "64", "--batched",
                                      "--max-batch", "2", "--paged"])
    make = ld.PagedCache.__init__
    monkeypatch.setattr(ld.PagedCache, "__init__", lambda self, g, layers, prompt, slots, tokens, dev: make(self, g, layers, prompt, slots, 1, dev))
    with pytest.raises(RuntimeError, match="too small"):
        ld.main()
