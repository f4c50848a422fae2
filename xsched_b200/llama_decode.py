"""High-priority workload generator: batch-1 decode on a random-init Llama-3-8B-shaped model in bf16
(32 layers, hidden 4096, 32 query / 8 KV heads of 128, FFN 14336, KV length 4096, vocabulary 128256 assumed),
requests of N tokens arriving as a Poisson process.  Pure PyTorch (library kernels): this is a WORKLOAD for the
scheduler, not part of the preemption path — it is meant to be run unchanged under the libcuda interposer,

    LD_LIBRARY_PATH=<dir with libcuda.so.1 -> libshimcuda.so>  XSCHED_AUTO_XQUEUE=ON XSCHED_SCHEDULER=GLB \
    XSCHED_AUTO_XQUEUE_PRIORITY=1  python -m xsched_b200.llama_decode --requests 20 --rate 2

so that its stream becomes a high-priority XQueue.  Weights are synthetic (seeded normal, std 0.02); no
checkpoint or dataset is involved.  Prints one JSON line with per-token and per-request latency percentiles.
Each decode step reads every weight once (~15.0 GB) plus the KV cache (~0.54 GB): HBM-bound, ~2.4 ms at the
measured 6.5 TB/s.

With --batched the requests in flight are decoded together (continuous batching: one step streams the weights once
for all of them, every request is still a batch-1 client with its own KV cache of 4096 positions and its own 128
tokens).  That is what makes the configured 10 requests/s servable at all: one request at a time needs ~0.7 s of
decode per request, seven times more than one GPU has at that rate.  A token's latency is then the duration of the
step that produced it, counted once per request that was in the step.

With --paged (and --batched) the caches are one paged cache (xsched_b200.pk.KvCache) and its operators take the place of
the cache writes, the attention and the slot moves above: every request is a fork of one prompt of --kv positions, whose
pages all share; each token extends it by a position (the first one copies the shared last page), is rotated by its position
and written by `append`, and attends through `attention`, which reads the shared positions once for the whole batch.  A
request that is done frees its pages; the pool is compacted while nothing is in flight.
"""
from __future__ import annotations

import argparse
import json
import random
import time

import torch

H, NQ, NKV, HD, FFN, LAYERS, VOCAB = 4096, 32, 8, 128, 14336, 32, 128256


def pct(v, p):
    v = sorted(v)
    return v[min(len(v) - 1, int(p * (len(v) - 1) + 0.5))] if v else float("nan")


PAGE = 64


class Layer:
    def __init__(self, g, kv_len, dev, slots=1):
        def w(o, i):
            return (torch.randn(o, i, device=dev, generator=g, dtype=torch.float32) * 0.02).to(torch.bfloat16)
        self.wqkv = w((NQ + 2 * NKV) * HD, H)
        self.wo = w(H, NQ * HD)
        self.w_gate_up = w(2 * FFN, H)
        self.w_down = w(H, FFN)
        self.n1 = torch.ones(H, device=dev, dtype=torch.bfloat16)
        self.n2 = torch.ones(H, device=dev, dtype=torch.bfloat16)
        if slots == 0:                                    # the cache is elsewhere (--paged)
            return
        self.k = (torch.randn(1, NKV, kv_len, HD, device=dev, generator=g) * 0.5).to(torch.bfloat16).expand(slots, -1, -1, -1).contiguous()
        self.v = (torch.randn(1, NKV, kv_len, HD, device=dev, generator=g) * 0.5).to(torch.bfloat16).expand(slots, -1, -1, -1).contiguous()

    def __call__(self, x, pos):
        h = torch.nn.functional.rms_norm(x, (H,), self.n1, 1e-5)
        qkv = h @ self.wqkv.T
        q, k, v = qkv.split([NQ * HD, NKV * HD, NKV * HD], dim=-1)
        # the new token's K/V overwrite one cache slot (fixed KV length: a sliding window of 4096)
        self.k[0, :, pos] = k.view(NKV, HD)
        self.v[0, :, pos] = v.view(NKV, HD)
        att = torch.nn.functional.scaled_dot_product_attention(q.view(1, NQ, 1, HD), self.k, self.v, enable_gqa=True)
        x = x + att.reshape(1, NQ * HD) @ self.wo.T
        h = torch.nn.functional.rms_norm(x, (H,), self.n2, 1e-5)
        gu = h @ self.w_gate_up.T
        g_, u_ = gu.split([FFN, FFN], dim=-1)
        return x + (torch.nn.functional.silu(g_) * u_) @ self.w_down.T

    def batched(self, x, rows, pos):
        """n requests at once: x [n, H], rows = arange(n) (their cache slots), pos [n] = each one's write position."""
        n = x.shape[0]
        h = torch.nn.functional.rms_norm(x, (H,), self.n1, 1e-5)
        qkv = h @ self.wqkv.T
        q, k, v = qkv.split([NQ * HD, NKV * HD, NKV * HD], dim=-1)
        self.k[rows, :, pos] = k.view(n, NKV, HD)
        self.v[rows, :, pos] = v.view(n, NKV, HD)
        att = torch.nn.functional.scaled_dot_product_attention(q.view(n, NQ, 1, HD), self.k[:n], self.v[:n], enable_gqa=True)
        x = x + att.reshape(n, NQ * HD) @ self.wo.T
        h = torch.nn.functional.rms_norm(x, (H,), self.n2, 1e-5)
        gu = h @ self.w_gate_up.T
        g_, u_ = gu.split([FFN, FFN], dim=-1)
        return x + (torch.nn.functional.silu(g_) * u_) @ self.w_down.T

    def paged(self, x, index, kv, seqs):
        """The same for n requests in a paged cache: x [n, H], seqs [n] = their slots, already extended by this token."""
        n = x.shape[0]
        h = torch.nn.functional.rms_norm(x, (H,), self.n1, 1e-5)
        att = kv.step(index, h @ self.wqkv.T, seqs)
        x = x + att.view(n, NQ * HD) @ self.wo.T
        h = torch.nn.functional.rms_norm(x, (H,), self.n2, 1e-5)
        gu = h @ self.w_gate_up.T
        g_, u_ = gu.split([FFN, FFN], dim=-1)
        return x + (torch.nn.functional.silu(g_) * u_) @ self.w_down.T

    def move_slot(self, src, dst):
        """The request in cache slot `src` continues in slot `dst` (slots in use stay contiguous)."""
        self.k[dst].copy_(self.k[src])
        self.v[dst].copy_(self.v[src])


class PagedCache:
    """One paged cache for all layers: sequence 0 holds the prompt, sequences 1.. are the requests, forks of it."""

    def __init__(self, g, layers, prompt, slots, tokens, dev):
        from xsched_b200 import pk
        own = -(-(prompt + tokens) // PAGE) - prompt // PAGE      # pages that a request may need of its own
        pages, width = -(-prompt // PAGE) + slots * own, -(-(prompt + tokens) // PAGE)
        self.k = torch.empty(layers, pages, NKV, PAGE, HD, device=dev, dtype=torch.bfloat16)
        self.v = torch.empty_like(self.k)
        for pool in (self.k, self.v):
            for layer in pool:
                layer.copy_(torch.randn(layer.shape, device=dev, generator=g) * 0.5)
        table = torch.full((1 + slots, width), -1, dtype=torch.int32, device=dev)
        lens, refs = torch.zeros(1 + slots, dtype=torch.int32, device=dev), torch.zeros(pages, dtype=torch.int32, device=dev)
        self.cache = pk.KvCache(self.k, self.v, table, lens, refs)
        self.prompt = torch.zeros(1, dtype=torch.int32, device=dev)
        self.one = torch.ones(slots, dtype=torch.int32, device=dev)
        self.shared = torch.full((1,), prompt, dtype=torch.int32, device=dev)
        self.inv_freq = 500000.0 ** (-torch.arange(0, HD, 2, device=dev, dtype=torch.float64) / HD)
        self.q, self.out = (torch.empty(slots, NQ, HD, device=dev, dtype=torch.bfloat16) for _ in range(2))
        self.scratch = torch.zeros(self.cache.attention_scratch_bytes(slots, slots, NQ), dtype=torch.uint8, device=dev)
        self.cache.extend(self.prompt, self.shared, self._stream())
        self.check()

    @staticmethod
    def _stream():
        return torch.cuda.current_stream().cuda_stream

    def check(self):
        """Whether the last extend had room: it changes nothing without, and the step's tokens fell on those of the step before."""
        report = self.cache.result(self._stream())
        if report.missing or report.refused:
            raise RuntimeError(f"the page pool is too small: {report.missing} pages missing, {report.refused} sequences too long")

    def start(self, seqs):
        self.cache.fork(self.prompt.expand(seqs.numel()).contiguous(), seqs, self._stream())

    def stop(self, seqs):
        self.cache.free(seqs, self._stream())

    def extend(self, seqs):
        self.cache.extend(seqs, self.one[:seqs.numel()], self._stream())

    def compact(self):
        self.cache.compact(self._stream())

    def step(self, layer, qkv, seqs):
        n, s = seqs.numel(), self._stream()
        self.cache.append(self.q[:n], qkv, seqs, s, inv_freq=self.inv_freq, layer=layer)
        self.cache.attention(self.out[:n], self.q[:n], seqs, s, scratch=self.scratch, shared_len=self.shared, layer=layer)
        return self.out[:n]


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=20)
    ap.add_argument("--tokens", type=int, default=128)
    ap.add_argument("--rate", type=float, default=10.0, help="mean request arrivals per second (Poisson)")
    ap.add_argument("--kv", type=int, default=4096)
    ap.add_argument("--layers", type=int, default=LAYERS)
    ap.add_argument("--seed", type=int, default=7)
    ap.add_argument("--device", type=int, default=0)
    ap.add_argument("--deadline-ms", type=float, default=0.0, help="count decode steps that took longer than this (0 = off)")
    ap.add_argument("--samples", default="", help="write every per-token latency (ms, one per line) to this file")
    ap.add_argument("--batched", action="store_true", help="decode the requests in flight together (continuous batching)")
    ap.add_argument("--max-batch", type=int, default=16)
    ap.add_argument("--paged", action="store_true", help="with --batched: one paged cache, requests are forks of one prompt of --kv positions")
    a = ap.parse_args()
    if a.paged and not a.batched:
        ap.error("--paged goes with --batched")
    torch.cuda.set_device(a.device)
    dev = torch.device("cuda", a.device)
    g = torch.Generator(device=dev).manual_seed(a.seed)
    layers = [Layer(g, a.kv, dev, 0 if a.paged else a.max_batch if a.batched else 1) for _ in range(a.layers)]
    lm_head = (torch.randn(VOCAB, H, device=dev, generator=g) * 0.02).to(torch.bfloat16)
    norm = torch.ones(H, device=dev, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()          # created after the interposer is in place: gets its own XQueue
    rng = random.Random(a.seed)

    def step(x, pos):
        for l in layers:
            x = l(x, pos)
        logits = torch.nn.functional.rms_norm(x, (H,), norm, 1e-5) @ lm_head.T
        return x, int(logits.argmax())          # the .item() is the device->host read of the step's result

    tok_ms, req_ms = [], []
    batch_sizes = []
    if a.batched:
        with torch.cuda.stream(stream), torch.no_grad():
            xb = torch.randn(a.max_batch, H, device=dev, generator=g).to(torch.bfloat16)
            rows_all = torch.arange(a.max_batch, device=dev)

            kv = PagedCache(g, a.layers, a.kv, a.max_batch, a.tokens + 2 * a.max_batch, dev) if a.paged else None

            def logits_of(x):
                logits = torch.nn.functional.rms_norm(x, (H,), norm, 1e-5) @ lm_head.T
                return logits.argmax(dim=-1).tolist()      # the device->host read of the step's result

            def bstep(n, pos_list):
                x = xb[:n]
                if kv is not None:
                    seqs = torch.tensor(pos_list, dtype=torch.int32, device=dev)
                    kv.extend(seqs)
                    for i, l in enumerate(layers):
                        x = l.paged(x, i, kv, seqs)
                else:
                    pos = torch.tensor(pos_list, device=dev)
                    for l in layers:
                        x = l.batched(x, rows_all[:n], pos)
                xb[:n] = x
                tokens = logits_of(x)
                if kv is not None:
                    kv.check()                            # the stream has just been waited for
                return tokens

            for n in list(range(1, a.max_batch + 1)) * 2:                      # warm-up: every batch size once picks its kernels
                if kv is None:
                    bstep(n, [n] * n)
                    continue
                seqs = list(range(1, n + 1))
                kv.start(torch.tensor(seqs, dtype=torch.int32, device=dev))
                bstep(n, seqs)
                kv.stop(torch.tensor(seqs, dtype=torch.int32, device=dev))
            print("READY", flush=True)
            t0 = time.perf_counter()
            arrivals, t = [], t0
            for _ in range(a.requests):
                t += rng.expovariate(a.rate)
                arrivals.append(t)
            active = []                               # [arrival time, tokens done, write position, or the sequence if paged]; index = cache slot
            free_seqs = list(range(a.max_batch, 0, -1))
            nxt = 0
            while nxt < len(arrivals) or active:
                now = time.perf_counter()
                while nxt < len(arrivals) and arrivals[nxt] <= now and len(active) < a.max_batch:
                    if kv is not None:
                        seq = free_seqs.pop()
                        kv.start(torch.tensor([seq], dtype=torch.int32, device=dev))
                    active.append([arrivals[nxt], 0, (nxt * 37) % a.kv if kv is None else seq])
                    nxt += 1
                if not active:
                    if kv is not None:
                        kv.compact()                  # nobody waits for a page now
                    time.sleep(max(0.0, arrivals[nxt] - time.perf_counter()))
                    continue
                n = len(active)
                ts = time.perf_counter()
                bstep(n, [r[2] for r in active])
                dt = (time.perf_counter() - ts) * 1e3
                tok_ms.extend([dt] * n)
                batch_sizes.append(n)
                end = time.perf_counter()
                slot = 0
                while slot < len(active):
                    r = active[slot]
                    r[1] += 1
                    if kv is None:
                        r[2] = (r[2] + 1) % a.kv
                    if r[1] < a.tokens:
                        slot += 1
                        continue
                    req_ms.append((end - r[0]) * 1e3)
                    last = len(active) - 1
                    if kv is not None:
                        kv.stop(torch.tensor([r[2]], dtype=torch.int32, device=dev))
                        free_seqs.append(r[2])
                    if slot != last:                  # the last slot's request moves into the freed one
                        for l in layers if kv is None else ():
                            l.move_slot(last, slot)
                        xb[slot].copy_(xb[last])
                        active[slot] = active[last]
                    active.pop()
    if not a.batched:
        with torch.cuda.stream(stream), torch.no_grad():
            x = torch.randn(1, H, device=dev, generator=g).to(torch.bfloat16)
            for i in range(3):
                x, _ = step(x, i)                    # warm-up (cuBLAS heuristics, allocator)
            print("READY", flush=True)
            t_next = time.perf_counter()
            for r in range(a.requests):
                t_next += rng.expovariate(a.rate)
                now = time.perf_counter()
                if now < t_next:
                    time.sleep(t_next - now)
                t_arr = t_next                        # latency is counted from the arrival, queueing included
                for t in range(a.tokens):
                    t0 = time.perf_counter()
                    x, _ = step(x, (r * a.tokens + t) % a.kv)
                    tok_ms.append((time.perf_counter() - t0) * 1e3)
                req_ms.append((time.perf_counter() - t_arr) * 1e3)
    print("DONE", flush=True)
    if a.samples:
        with open(a.samples, "w") as f:
            f.write("\n".join(f"{v:.4f}" for v in tok_ms))
    missed = sum(1 for v in tok_ms if a.deadline_ms > 0 and v > a.deadline_ms)
    weights_gb = sum(p.numel() for l in layers for p in (l.wqkv, l.wo, l.w_gate_up, l.w_down)) * 2 / 1e9 + lm_head.numel() * 2 / 1e9
    print(json.dumps({"role": "llama-decode", "requests": len(req_ms), "tokens": len(tok_ms), "token_p50_ms": round(pct(tok_ms, 0.5), 3),
                      "token_p99_ms": round(pct(tok_ms, 0.99), 3), "token_mean_ms": round(sum(tok_ms) / max(1, len(tok_ms)), 3),
                      "request_p50_ms": round(pct(req_ms, 0.5), 2), "request_p99_ms": round(pct(req_ms, 0.99), 2),
                      "weights_gb": round(weights_gb, 2), "kv_gb": round(a.layers * 2 * NKV * a.kv * HD * 2 / 1e9, 3), "rate": a.rate,
                      "mode": "batched, paged" if a.paged else "batched" if a.batched else "one request at a time", "decode_steps": len(batch_sizes) if a.batched else len(tok_ms),
                      "mean_batch": round(sum(batch_sizes) / max(1, len(batch_sizes)), 2) if a.batched else 1.0,
                      "deadline_ms": a.deadline_ms, "deadline_missed": missed, "deadline_miss_rate": round(missed / max(1, len(tok_ms)), 5)}))


if __name__ == "__main__":
    main()
