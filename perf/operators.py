"""The paged key/value cache of a decode loop and the operators around it, as cases to be measured.

Three operators, all on one cache (`pk.KvCache`): pools k, v [layers, pages, kv_heads, page_size, head_dim], a table
page_table [seqs, width] of int32 page ids (-1: none), lens [seqs] (positions held) and refs [pages] (how many table
entries name a page; 0 = free).

append     norms of queries and keys for each head and the rotation by position, in one pass over a projection's output
           [tokens, (q_heads + 2 kv_heads) head_dim]; queries go to a tensor, keys and values to their places in the cache.
attention  attention of every query to its own sequence's positions up to its own; the first `shared` positions are the
           same pages in all sequences and are read once for all of them.
pages      copying, forking (with copy on write when a child grows), compacting and freeing pages.

The last rows of a sequence are its queries: query j of t belongs to position lens - t + j.  `own` chooses between the
plain forms (elementary torch operations in 32 bits, angles in 64) and the calls of the framework."""
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one request alone, shortly after its start: latency is all that counts
        dict(name="attend one", op="attention", dtype="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, n=1, shared=0, own_lo=301, own_hi=301, q_lo=1, q_hi=1, lens=1),
        # the batched decode of the Llama-3-8B-shaped workload: 16 requests on one 4096-long prefix, up to 128 tokens each of their own
        dict(name="attend 16 on 4096", op="attention", dtype="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, n=16, shared=4096, own_lo=1, own_hi=128, q_lo=1, q_hi=1, lens=2),
        # many requests on one long document, each with an answer of its own
        dict(name="attend 256 on 16384", op="attention", dtype="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, n=256, shared=16384, own_lo=1, own_hi=1024, q_lo=1, q_hi=1, lens=3),
        # long requests with nothing in common: the cache is all that is read
        dict(name="attend 32 apart", op="attention", dtype="fp16", q_heads=28, kv_heads=4, head_dim=128, page=16, n=32, shared=0, own_lo=3000, own_hi=12000, q_lo=1, q_hi=1, lens=4),
        # drafts of several tokens checked at once, small heads, a prefix that ends inside a tile
        dict(name="attend drafts", op="attention", dtype="fp16", q_heads=24, kv_heads=8, head_dim=64, page=32, n=40, shared=2016, own_lo=9, own_hi=700, q_lo=1, q_hi=8, lens=5),
        # prompts that come in behind a common system prompt
        dict(name="attend prompts", op="attention", dtype="bf16", q_heads=32, kv_heads=8, head_dim=128, page=128, n=9, shared=2048, own_lo=400, own_hi=1500, q_lo=300, q_hi=1500, lens=6),
        # one token of one request
        dict(name="append one", op="append", dtype="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, n=1, q_lo=1, q_hi=1, len_hi=5000, rotary=128, pairs="halves", norm=True, lens=7),
        # a decode step of a full batch, only part of each head rotated
        dict(name="append 200", op="append", dtype="fp16", q_heads=24, kv_heads=8, head_dim=64, page=16, n=200, q_lo=1, q_hi=1, len_hi=30000, rotary=32, pairs="neighbours", norm=True, lens=8),
        # prompts, at far positions
        dict(name="append prompts", op="append", dtype="bf16", q_heads=32, kv_heads=8, head_dim=128, page=64, n=5, q_lo=700, q_hi=4000, len_hi=900000, rotary=128, pairs="halves", norm=True, lens=9),
        # several samples from each of a few prompts: fork, then every child's first token copies the shared last page
        dict(name="fork 48", op="fork", dtype="bf16", layers=32, kv_heads=8, head_dim=128, page=16, pages=420, parents=3, n=48, len_lo=500, len_hi=2100, grow=1, lens=10),
        # a pool full of holes after many requests have gone
        dict(name="compact", op="compact", dtype="bf16", layers=8, kv_heads=8, head_dim=128, page=64, pages=1024, n=40, keep=0.45, lens=11),
        # a few pages set aside
        dict(name="copy 37 pages", op="copy", dtype="fp16", layers=4, kv_heads=4, head_dim=128, page=32, pages=700, n=37, lens=12),
    ]


def _log(rng, lo, hi):
    """A whole number, spread over the logarithm of lo..hi."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    """A case of the same ranges that costs no more than the largest listed one."""
    most = [work(c) for c in listed()]
    while True:
        c = _draw(rng)
        w = work(c)
        if all(w[k] <= max(m[k] for m in most) for k in w):
            return c


def _draw(rng):
    lens = rng.randrange(1 << 20)
    op = rng.choice(["attention", "attention", "attention", "append", "append", "fork", "compact", "copy"])
    dtype, head_dim, page = rng.choice(["bf16", "fp16"]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    if op == "attention":
        kind = rng.choice(["decode", "decode", "drafts", "prompts"])
        n = _log(rng, 1, {"decode": 200, "drafts": 48, "prompts": 8}[kind])
        shared = rng.choice([0, _log(rng, 16, 12000 if kind == "decode" else 3000)]) // page * page
        q_lo, q_hi = {"decode": (1, 1), "drafts": (1, 8), "prompts": (20, _log(rng, 40, 1200))}[kind]
        own_lo = q_lo + rng.randrange(100)
        own_hi = own_lo + _log(rng, 1, 1000 if n > 32 else 5000 if kind == "decode" else 1200)
        return dict(op=op, dtype=dtype, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, n=n, shared=shared,
                    own_lo=own_lo, own_hi=own_hi, q_lo=q_lo, q_hi=q_hi, lens=lens)
    if op == "append":
        prompts = rng.random() < 0.4
        n = _log(rng, 1, 5 if prompts else 200)
        q_hi = _log(rng, 10, 2500) if prompts else 1
        return dict(op=op, dtype=dtype, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, n=n, q_lo=max(1, q_hi // 3), q_hi=q_hi,
                    len_hi=_log(rng, 4000, 900000), rotary=rng.choice([head_dim, head_dim // 2, 16]), pairs=rng.choice(["halves", "neighbours"]),
                    norm=rng.random() < 0.7, lens=lens)
    layers = rng.choice([1, 2, 5, 8])
    if op == "fork":
        n = _log(rng, 1, 60)
        return dict(op=op, dtype=dtype, layers=layers, kv_heads=kv_heads, head_dim=head_dim, page=page, pages=600, parents=rng.randint(1, 4), n=n,
                    len_lo=1, len_hi=rng.randint(2, 40 * page), grow=rng.randint(1, 2 * page), lens=lens)
    if op == "compact":
        return dict(op=op, dtype=dtype, layers=layers, kv_heads=kv_heads, head_dim=head_dim, page=page, pages=_log(rng, 20, 900), n=_log(rng, 1, 40),
                    keep=round(0.05 + 0.9 * rng.random(), 2), lens=lens)
    return dict(op=op, dtype=dtype, layers=layers, kv_heads=kv_heads, head_dim=head_dim, page=page, pages=_log(rng, 20, 900), n=_log(rng, 1, 200), lens=lens)


# ------------------------------------------------------------------------------------------------ sizes from a case alone
def _sizes(c):
    """(length of each sequence, queries of each sequence) of an attention or append case; the same for every seed."""
    r = random.Random(c["lens"])
    qs = [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["n"])]
    if c["op"] == "attention":
        return [c["shared"] + max(q, r.randint(c["own_lo"], c["own_hi"])) for q in qs], qs
    return [r.randint(q, max(q, c["len_hi"])) for q in qs], qs


def _parents(c):
    r = random.Random(c["lens"])
    return [r.randint(c["len_lo"], c["len_hi"]) for _ in range(c["parents"])]


def _kept(c):
    """Lengths in pages of the sequences that are left in a pool of which about `keep` is in use."""
    r = random.Random(c["lens"])
    left, out = max(1, int(c["pages"] * c["keep"])), []
    for i in range(c["n"]):
        out.append(min(left, r.randint(0, max(1, 2 * int(c["pages"] * c["keep"]) // c["n"]))))
        left -= out[-1]
    return out


def work(case):
    c = case
    size, D = 2, c["head_dim"]
    token = 2 * c["kv_heads"] * D * size
    if c["op"] == "attention":
        lens, qs = _sizes(c)
        seen = sum(q * (n - q) + q * (q + 1) // 2 for n, q in zip(lens, qs))
        read = c["shared"] + sum(n - c["shared"] for n in lens)
        return {"bytes": read * token + 2 * sum(qs) * c["q_heads"] * D * size, "flops": 4 * D * c["q_heads"] * seen}
    if c["op"] == "append":
        t = sum(_sizes(c)[1])
        return {"bytes": 2 * t * (c["q_heads"] + 2 * c["kv_heads"]) * D * size, "flops": 10 * t * (c["q_heads"] + c["kv_heads"]) * D}
    page = c["layers"] * c["page"] * token
    if c["op"] == "fork":
        held = _parents(c)
        moved = sum(1 for i in range(c["n"]) if held[i % c["parents"]] % c["page"])
        table = sum(-(-held[i % c["parents"]] // c["page"]) for i in range(c["n"]))
        return {"bytes": 2 * moved * page + 8 * table + 4 * c["pages"], "flops": 0}
    if c["op"] == "compact":
        live = sum(_kept(c))
        return {"bytes": 2 * max(1, int(live * (1 - live / c["pages"]))) * page + 8 * live + 4 * c["pages"], "flops": 0}
    return {"bytes": 2 * min(c["n"], c["pages"] // 2) * page, "flops": 0}


# ----------------------------------------------------------------------------------------------------------- inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(counts):
    out = [0]
    for v in counts:
        out.append(out[-1] + v)
    return _ints(out)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    dt = TYPES[c["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dt)

    def shuffled(n):
        return torch.randperm(n, device=DEV, generator=g).to(torch.int32)

    D, page, H = c["head_dim"], c["page"], c["kv_heads"]
    if c["op"] == "attention":
        lens, qs = _sizes(c)
        head = c["shared"] // page
        each = [-(-n // page) - head for n in lens]
        pages = head + sum(each)
        ids = shuffled(pages)
        table = torch.full((c["n"], head + max(each)), -1, dtype=torch.int32, device=DEV)
        table[:, :head] = ids[:head]
        at = head
        for i, e in enumerate(each):
            table[i, head:head + e] = ids[at:at + e]
            at += e
        refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        used = table[table >= 0].long()
        refs.index_add_(0, used, torch.ones_like(used, dtype=torch.int32))
        k, v = normal(1, pages, H, page, D), normal(1, pages, H, page, D)
        s.update(k=k, v=v, table=table, lens=_ints(lens), refs=refs, seqs=_ints(list(range(c["n"]))), starts=_starts(qs), rows=sum(qs), q_max=max(qs),
                 own_max=max(lens) - c["shared"], decode=max(qs) == 1, shared=_ints([c["shared"]]), q=normal(sum(qs), c["q_heads"], D, scale=1.8))
        if own:
            from xsched_b200 import pk
            s["cache"] = pk.KvCache(k, v, table, s["lens"], refs)
            s["scratch"] = torch.zeros(s["cache"].attention_scratch_bytes(s["rows"], c["n"], c["q_heads"]), dtype=torch.uint8, device=DEV)
            s["out"] = torch.empty_like(s["q"])
    elif c["op"] == "append":
        lens, qs = _sizes(c)
        first = [(n - q) // page for n, q in zip(lens, qs)]
        last = [(n - 1) // page for n in lens]
        pages = sum(b - a + 1 for a, b in zip(first, last))
        ids = shuffled(pages)
        table = torch.full((c["n"], max(last) + 1), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, (a, b) in enumerate(zip(first, last)):
            table[i, a:b + 1] = ids[at:at + b - a + 1]
            at += b - a + 1
        refs = torch.ones(pages, dtype=torch.int32, device=DEV)
        rot = torch.arange(0, c["rotary"], 2, device=DEV, dtype=torch.float64)
        s.update(k=normal(1, pages, H, page, D), v=normal(1, pages, H, page, D), table=table, lens=_ints(lens), refs=refs, seqs=_ints(list(range(c["n"]))),
                 starts=_starts(qs), rows=sum(qs), decode=max(qs) == 1, qkv=normal(sum(qs), (c["q_heads"] + 2 * H) * D, scale=2.0), inv_freq=500000.0 ** (-rot / c["rotary"]),
                 wq=(1 + 0.2 * normal(D).float()).to(dt) if c["norm"] else None, wk=(1 + 0.2 * normal(D).float()).to(dt) if c["norm"] else None)
        s["q"] = torch.zeros(sum(qs), c["q_heads"], D, dtype=dt, device=DEV)
    else:
        P, L = c["pages"], c["layers"]
        s.update(k=normal(L, P, H, page, D), v=normal(L, P, H, page, D))
        refs, ids = torch.zeros(P, dtype=torch.int32, device=DEV), shuffled(P)
        if c["op"] == "fork":
            held = _parents(c)
            table = torch.full((c["parents"] + c["n"], -(-(c["len_hi"] + c["grow"]) // page)), -1, dtype=torch.int32, device=DEV)
            at = 0
            for i, h in enumerate(held):
                e = -(-h // page)
                table[i, :e] = ids[at:at + e]
                at += e
            lens = _ints(held + [0] * c["n"])
            refs[ids[:at].long()] = 1
            s.update(parents=_ints([i % c["parents"] for i in range(c["n"])]), children=_ints(list(range(c["parents"], c["parents"] + c["n"]))), grow=_ints([c["grow"]] * c["n"]))
        elif c["op"] == "compact":
            held = _kept(c)
            table = torch.full((c["n"], max(1, max(held))), -1, dtype=torch.int32, device=DEV)
            at = 0
            for i, e in enumerate(held):
                table[i, :e] = ids[at:at + e]
                at += e
            lens = _ints([e * page for e in held])
            refs[ids[:at].long()] = 1
            s.update(table0=table.clone(), refs0=refs.clone())
        else:
            n = min(c["n"], P // 2)
            table, lens = torch.full((1, 1), -1, dtype=torch.int32, device=DEV), _ints([0])
            s.update(src=ids[:n].contiguous(), dst=ids[n:2 * n].contiguous())
        s.update(table=table, lens=lens, refs=refs)
    if own and c["op"] != "attention":
        from xsched_b200 import pk
        s["cache"] = pk.KvCache(s["k"], s["v"], s["table"], s["lens"], s["refs"])
    return s


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    return {"attention": _attention, "append": _append, "fork": _fork, "compact": _compact, "copy": _copy}[c["op"]](s, c)


def _run_own(s, c):
    stream, cache = torch.cuda.current_stream().cuda_stream, s["cache"]
    if c["op"] == "attention":
        cache.attention(s["out"], s["q"], s["seqs"], stream, starts=None if s["decode"] else s["starts"], shared_len=s["shared"] if c["shared"] else None, scratch=s["scratch"])
        return s["out"]
    if c["op"] == "append":
        cache.append(s["q"], s["qkv"], s["seqs"], stream, starts=None if s["decode"] else s["starts"], q_weight=s["wq"], k_weight=s["wk"], eps=1e-6,
                     inv_freq=s["inv_freq"], interleaved=c["pairs"] == "neighbours")
        return s["q"], s["k"], s["v"]
    if c["op"] == "fork":  # the last round's children go, new ones come and take their first tokens' room
        cache.free(s["children"], stream)
        cache.fork(s["parents"], s["children"], stream)
        cache.extend(s["children"], s["grow"], stream)
        return s["table"], s["lens"], s["refs"], s["k"], s["v"]
    if c["op"] == "compact":  # the table of before is put back first: every pass finds the same holes
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
        cache.compact(stream)
        return s["table"], s["refs"], s["k"], s["v"]
    cache.copy(s["src"], s["dst"], stream)
    return s["k"], s["v"]


# ------------------------------------------------------------------------------------------------- the plain forms
def _take(pool, table):
    """[sequences, positions, kv_heads, head_dim] in 32 bits of the pages that `table` [sequences, pages] names; page -1 reads as zeros."""
    got = pool[0][table.clamp(min=0).long()].float() * (table >= 0)[:, :, None, None, None]
    n, e, H, page, D = got.shape
    return got.permute(0, 1, 3, 2, 4).reshape(n, e * page, H, D)


def _attention(s, c):
    n, H, D, page, shared = c["n"], c["kv_heads"], c["head_dim"], c["page"], c["shared"]
    G, T = c["q_heads"] // H, s["q_max"]
    lens, starts, dev = s["lens"].long(), s["starts"].long(), s["q"].device
    count = starts[1:] - starts[:-1]
    place = torch.arange(T, device=dev)
    real = place[None] < count[:, None]                                       # [n, T]: the rows that a sequence has
    row = (starts[:-1, None] + place[None]).clamp(max=s["rows"] - 1)
    q = s["q"].float()[row].view(n, T, H, G, D) * D ** -0.5
    sees = (lens - count)[:, None] + place[None] + 1                          # positions before and at the query's own
    head = shared // page
    own_k, own_v = _take(s["k"], s["table"][:, head:]), _take(s["v"], s["table"][:, head:])
    at = shared + torch.arange(own_k.shape[1], device=dev)
    q2 = q.permute(0, 2, 1, 3, 4).reshape(n, H, T * G, D)
    scores = torch.matmul(q2, own_k.permute(0, 2, 3, 1))                      # [n, H, T G, own]
    hidden = (at[None, None] >= sees[:, :, None]).repeat_interleave(G, dim=1)  # [n, T G, own]
    scores.masked_fill_(hidden[:, None], float("-inf"))
    most = scores.amax(dim=-1, keepdim=True)
    if shared:
        pre_k, pre_v = _take(s["k"], s["table"][:1, :head])[0], _take(s["v"], s["table"][:1, :head])[0]
        q3 = q.permute(2, 0, 1, 3, 4).reshape(H, n * T * G, D)
        first = torch.matmul(q3, pre_k.permute(1, 2, 0)).view(H, n, T * G, shared)
        most = torch.maximum(most, first.amax(dim=-1, keepdim=True).transpose(0, 1))
    scores = torch.exp(scores - most)
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores, own_v.permute(0, 2, 1, 3))
    if shared:
        first = torch.exp(first - most.transpose(0, 1))
        total = total + first.sum(dim=-1, keepdim=True).transpose(0, 1)
        out = out + torch.matmul(first.view(H, n * T * G, shared), pre_v.permute(1, 0, 2)).view(H, n, T * G, D).transpose(0, 1)
    out = (out / total).view(n, H, T, G, D).permute(0, 2, 1, 3, 4).reshape(n, T, H * G, D)
    return out[real].to(s["q"].dtype)


def _append(s, c):
    H, D, page, rot, Hq = c["kv_heads"], c["head_dim"], c["page"], c["rotary"], c["q_heads"]
    rows = s["rows"]
    starts, dev = s["starts"].long(), s["q"].device
    token = torch.arange(rows, device=dev)
    seq = torch.searchsorted(starts, token, right=True) - 1
    pos = s["lens"].long()[seq] - starts[seq + 1] + token
    x = s["qkv"].view(rows, Hq + 2 * H, D).float()

    def normed(y, w):
        return y if w is None else y * torch.rsqrt((y * y).mean(dim=-1, keepdim=True) + 1e-6) * w.float()

    angle = pos.double()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(y):
        r, rest = y[..., :rot], y[..., rot:]
        if c["pairs"] == "halves":
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        return torch.cat((r, rest), dim=-1).to(s["q"].dtype)

    s["q"].copy_(turned(normed(x[:, :Hq], s["wq"])))
    where = s["table"].long()[seq, pos // page]
    s["k"][0][where, :, pos % page] = turned(normed(x[:, Hq:Hq + H], s["wk"]))
    s["v"][0][where, :, pos % page] = s["qkv"].view(rows, Hq + 2 * H, D)[:, Hq + H:]
    return s["q"], s["k"], s["v"]


def _counted(refs, ids, by):
    """refs with `by` added for every page that `ids` names (-1: none)."""
    held = ids.flatten().long()
    refs.index_add_(0, held.clamp(min=0), torch.where(held >= 0, by, 0).to(refs.dtype))


def _fork(s, c):
    table, lens, refs, page = s["table"], s["lens"], s["refs"], c["page"]
    children, parents = s["children"].long(), s["parents"].long()
    _counted(refs, table[children], -1)                                      # free
    table[children] = -1
    lens[children] = 0
    table[children] = table[parents]                                         # fork
    lens[children] = lens[parents]
    _counted(refs, table[children], 1)
    n, grow = lens[children].long(), s["grow"].long()                         # extend
    had, has = (n + page - 1) // page, (n + grow + page - 1) // page
    inside = (n % page != 0) & (grow > 0)
    tail = torch.where(inside, table[children, (had - 1).clamp(min=0)].long(), -1)
    before = ((tail[:, None] == tail[None]) & inside[:, None]).tril(-1).sum(dim=1)
    split = inside & (refs[tail.clamp(min=0)] - before > 1)                   # someone else still holds the last page
    need = has - had + split
    free = torch.nonzero(refs == 0).flatten()                                # lowest first
    at = torch.cumsum(need, 0) - need
    old, new = tail[split], free[at[split]]
    table[children[split], had[split] - 1] = new.int()
    refs.index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    col = torch.arange(table.shape[1], device=table.device)[None]
    fresh = (col >= had[:, None]) & (col < has[:, None])
    which = (at + split)[:, None] + col - had[:, None]
    table[children] = torch.where(fresh, free[which.clamp(0, len(free) - 1)].int(), table[children])
    refs[free[:int(need.sum())]] = 1
    lens[children] = (n + grow).int()
    s["k"][:, new] = s["k"][:, old]
    s["v"][:, new] = s["v"][:, old]
    return table, lens, refs, s["k"], s["v"]


def _compact(s, c):
    table, refs = s["table"], s["refs"]
    table.copy_(s["table0"])
    refs.copy_(s["refs0"])
    live = refs > 0
    count = live.sum()
    low = torch.arange(len(refs), device=refs.device) < count
    old, new = torch.nonzero(live & ~low).flatten(), torch.nonzero(~live & low).flatten()
    to = torch.arange(len(refs), device=refs.device)
    to[old] = new
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table))
    refs[new] = refs[old]
    refs[old] = 0
    s["k"][:, new] = s["k"][:, old]
    s["v"][:, new] = s["v"][:, old]
    return table, refs, s["k"], s["v"]


def _copy(s, c):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return s["k"], s["v"]


# ---------------------------------------------------------------------------------------------- from the definition
def exact(case, seed):
    c = case
    if c["op"] not in ("attention", "append"):
        return None  # pages are moved, not computed
    s = prepare(case, seed)
    lens, qs = _sizes(c)
    H, D, page, Hq = c["kv_heads"], c["head_dim"], c["page"], c["q_heads"]
    G, at = Hq // H, 0
    if c["op"] == "attention":
        out = torch.empty(sum(qs), Hq, D, dtype=torch.float64, device=DEV)
        for i, (n, t) in enumerate(zip(lens, qs)):
            ids = s["table"][i, :-(-n // page)].long()
            k = s["k"][0, ids].transpose(0, 1).reshape(H, -1, D)[:, :n].double()
            v = s["v"][0, ids].transpose(0, 1).reshape(H, -1, D)[:, :n].double()
            for h in range(H):
                q = s["q"][at:at + t, h * G:(h + 1) * G].double()
                x = torch.einsum("tgd,nd->tgn", q, k[h]) / D ** 0.5
                x[:, :, n - t:] += torch.full((t, t), float("-inf"), dtype=torch.float64, device=DEV).triu(1)[:, None]
                out[at:at + t, h * G:(h + 1) * G] = torch.softmax(x, dim=-1) @ v[h]
            at += t
        return out
    q_out, k_out, v_out = s["q"].double(), s["k"].double(), s["v"].double()
    rot = c["rotary"]
    for i, (n, t) in enumerate(zip(lens, qs)):
        x = s["qkv"][at:at + t].double().view(t, Hq + 2 * H, D)
        pos = torch.arange(n - t, n, device=DEV)
        turn = torch.polar(torch.ones(t, rot // 2, dtype=torch.float64, device=DEV), pos.double()[:, None] * s["inv_freq"])[:, None]
        parts = []
        for y, w in ((x[:, :Hq], s["wq"]), (x[:, Hq:Hq + H], s["wk"])):
            if w is not None:
                y = y / (y.square().sum(dim=-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
            if c["pairs"] == "halves":
                z = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * turn
                parts.append(torch.cat((z.real, z.imag, y[..., rot:]), dim=-1))
            else:
                z = torch.view_as_complex(y[..., :rot].reshape(t, -1, rot // 2, 2).contiguous()) * turn
                parts.append(torch.cat((torch.view_as_real(z).reshape(t, -1, rot), y[..., rot:]), dim=-1))
        q_out[at:at + t] = parts[0]
        where = s["table"][i].long()[pos // page]
        k_out[0][where, :, pos % page] = parts[1]
        v_out[0][where, :, pos % page] = x[:, Hq + H:]
        at += t
    return q_out, k_out, v_out
