// Tiles of an attention call (see attention.cu): up to 256 rows against 128 positions at a time on the tensor pipe.
//
// Two groups of four warps take 128 rows each (thread = row), or, where an item has at most 128 rows, the same rows and one
// half of the positions each.  Per step of 64 positions and group:
//
//   S = Q K^T     tcgen05.mma M128 N64, Q and K from shared memory (K-major), S fp32 in tensor memory, two buffers
//   P = exp2(..)  the group's threads read their rows of S, keep maximum and sum, and write P (16 bit) over S
//   O += P V      tcgen05.mma with P from tensor memory and V from shared memory (dimension-major: V lies as it is stored)
//
// One warp issues the MMAs of both groups in turn, always by the same lane; S of step s + 2 follows P V of step s, so a group always
// finds its next scores there while the pipe works for the other.  MMAs of one thread execute in the order of issue: that is what lets
// S of step s + 2 overwrite P of step s.  Another warp claims the items and fills a ring of eight stages (a step of K or of V,
// 16 KB each at 128) by TMA, page by page, and runs ahead of the rest into the next item.
//
// P is rounded to the cache's 16-bit type, since that is what the tensor pipe multiplies V's type with; its sum, S and O are fp32.
// A weight is off by half a step (2^-8 in bf16, 2^-11 in fp16), which takes the error of a result over a long prefix from 0.0017 to
// 0.0023 relative (bf16) and from 0.00021 to 0.00027 (fp16), most of it the result's own rounding.
//
// O is not rescaled whenever the maximum grows: p is taken relative to a reference that follows the maximum only when it
// falls 2^8 behind, so p stays below 2^8 (fp16 holds 2^15) and almost every step leaves O alone.
//
// Both the tensor pipe (4 * 128 * 128 * head_dim flop per group and tile: 0.55 us at 128) and the exponentials (16 a clock and SM:
// 0.55 us) would allow a tile of 256 rows in 1.1 us; it takes 3.0 us, at head_dim 64 as well (prompts of 1024 on 8192, ends and starts of
// items included), since a step is a chain from scores to weights to the next scores.  K and V of a tile are fetched once for 256 rows.
#pragma once
#include "attention_units.cuh"

#include <type_traits>

namespace xpk {

constexpr float kLag = 8.f;                                  // log2 units that the reference may fall behind the maximum

// ---- instructions ------------------------------------------------------------------------------------------------
// The issuing warp runs as one (its addresses and descriptors stay in uniform registers); `lead` is 1 in the one lane that issues.
__device__ __forceinline__ uint32_t elect_lead() {
    uint32_t lead;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(lead));
    return lead;
}
__device__ __forceinline__ void attn_commit(void *bar, uint32_t lead) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" :: "r"(smem_u32(bar)), "r"(lead) : "memory");
}
__device__ __forceinline__ void attn_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void attn_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                    "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                    "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                    "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                    "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr) : "memory");
}
// Waits for loads from tensor memory.  The registers pass through an empty statement behind the wait: arithmetic on them has
// no other reason to stay behind it.
template <int N>
__device__ __forceinline__ void tc_pin(uint32_t (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
template <int N>
__device__ __forceinline__ void tc_landed(uint32_t (&r)[N]) {
    tc_wait_ld();
    tc_pin(r);
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max_three(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t x;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
    return x;
}
__device__ __forceinline__ float2 of_two(uint64_t x) {
    float2 y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
    return y;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul_two(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// V as B operand with the dimension contiguous: atoms of 64 dimensions x 8 positions (1024 B, 128-byte swizzle), the next
// eight positions behind it, the next 64 dimensions a whole step of 64 positions further.
__device__ __forceinline__ uint64_t make_v_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)((kStep * 128u) >> 4) << 16;              // leading byte offset: between blocks of 64 dimensions
    d |= (uint64_t)(1024u >> 4) << 32;                       // stride byte offset: between groups of eight positions
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
template <class T> __host__ __device__ constexpr uint32_t mma_type() { return sizeof(T) == 2 ? 1u : 0u; }
template <> __host__ __device__ constexpr uint32_t mma_type<__half>() { return 0u; }
// D fp32, M = 128 rows; N = 64 positions, both K-major; N = kDim, B with N contiguous.
template <class T> __host__ __device__ constexpr uint32_t idesc_s() {
    return (1u << 4) | (mma_type<T>() << 7) | (mma_type<T>() << 10) | ((uint32_t)(kStep >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
template <class T, int kDim> __host__ __device__ constexpr uint32_t idesc_o() {
    return (1u << 4) | (mma_type<T>() << 7) | (mma_type<T>() << 10) | (1u << 16) | ((uint32_t)(kDim >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
constexpr uint32_t kAttnTmemCols = 512;                      // two S of both groups (64 columns each), O of both (head_dim each)

// ---- an item -----------------------------------------------------------------------------------------------------
struct TileItem {
    int entry;                  // -1: the prefix
    int head, r0, rows;         // first row (of the sequence, or of all sharing ones), rows (up to 256)
    int from, end;              // positions [from, end) are the item's
    int seq;                    // whose table names the pages
    bool both;                  // both groups take every tile
    int pos0, pos1;             // where the two groups begin
    int steps0, steps1;         // and how many steps of 64 positions they take
    int groups, half;           // groups of 16 rows; results per row of one run (2: one from each group of workers)
    int slot0, step;            // partial results: slot0 + group of 16 rows * step (+ half); slot0 < 0: the output itself
};

__device__ __forceinline__ TileItem tile_ticket(const AttnArgs &a, const CacheView &c, const AttnShared *sh, int ticket) {
    TileItem x;
    long long all;
    int own, local;
    if (ticket < sh->pre_tiles) {
        x.entry = -1;
        x.seq = sh->shared_seq;
        x.from = 0;
        own = sh->shared;
        all = sh->pre_rows;
        local = ticket;
    } else {
        int lo = 0, hi = (int)a.n - 1;                       // the last sequence with at most this many items before it
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (sh->tile0[mid] <= ticket) lo = mid; else hi = mid - 1;
        }
        x.entry = lo;
        x.seq = sh->plan[lo].seq;
        x.from = own_from(sh, lo);
        own = sh->plan[lo].len - x.from;
        all = rows_of(sh->plan[lo], a.group);
        local = ticket - sh->tile0[lo];
    }
    const int runs = tile_runs(sh, own), tiles = row_tiles(all), run = local % runs;
    x.half = halves(sh, all);
    // Late rows see most: they come first.
    const int rt = tiles - 1 - (local / runs) % tiles;
    x.head = local / (runs * tiles);
    x.r0 = rt * kItemRows;
    x.rows = (int)min(all - x.r0, (long long)kItemRows);
    x.groups = row_groups(x.rows);
    x.end = x.from + own;
    int most = own;
    if (x.entry >= 0) {
        const SeqPlan &p = sh->plan[x.entry];
        most = min(max(p.len - p.t + (x.r0 + x.rows - 1) / (int)a.group + 1 - x.from, 0), own);
    }
    const int each = (tiles_of(own) + runs - 1) / runs, first = run * each, last = min(first + each, tiles_of(most)), count = max(last - first, 0);
    x.both = x.half == 1 && x.rows > kTile;
    const int head_tiles = x.half == 2 ? (count + 1) / 2 : count;              // of the first group where each takes a half
    x.pos0 = x.from + first * kTile;
    x.pos1 = x.half == 2 ? x.pos0 + head_tiles * kTile : x.pos0;
    const int left = x.from + min(most, last * kTile);                          // nothing behind it is seen
    x.steps0 = max(0, min(2 * head_tiles, (left - x.pos0 + kStep - 1) / kStep));
    x.steps1 = x.both ? x.steps0 : x.half == 2 ? max(0, (left - x.pos1 + kStep - 1) / kStep) : 0;
    const int base = x.entry < 0 ? sh->pre_part0 : sh->part0[x.entry];
    x.step = runs * x.half;
    x.slot0 = base < 0 ? -1 : base + (x.head * row_groups(all) + x.r0 / kUnitRows) * x.step + run * x.half;
    return x;
}

// The order in which steps of K and V are loaded and used: both groups' (or the common) first two K, then V of a step and K of
// the step after next.  f(step, is_v, group).
template <class F>
__device__ __forceinline__ bool in_order(const TileItem &x, F f) {
    const int n0 = x.steps0, n1 = x.both ? 0 : x.steps1;
    for (int s = 0; s < min(2, n0); ++s)
        if (!f(s, false, 0)) return false;
    for (int s = 0; s < min(2, n1); ++s)
        if (!f(s, false, 1)) return false;
    for (int s = 0; s < max(n0, n1); ++s) {
        if (s < n0 && !f(s, true, 0)) return false;
        if (s + 2 < n0 && !f(s + 2, false, 0)) return false;
        if (s < n1 && !f(s, true, 1)) return false;
        if (s + 2 < n1 && !f(s + 2, false, 1)) return false;
    }
    return true;
}
__device__ __forceinline__ uint32_t stages_of(const TileItem &x) { return 2u * (uint32_t)(x.steps0 + (x.both ? 0 : x.steps1)); }
// Where V of a group's step lies in that order.
__device__ __forceinline__ uint32_t v_stage(const TileItem &x, int w, int s) {
    const int n0 = x.steps0, n1 = x.both ? 0 : x.steps1, before0 = w == 0 || x.both ? s : s + 1, before1 = s;
    return (uint32_t)(min(2, n0) + min(2, n1) + min(before0, n0) + min(before0, max(n0 - 2, 0)) + min(before1, n1) + min(before1, max(n1 - 2, 0)));
}

// ---- loader (one warp) -------------------------------------------------------------------------------------------
// The ids of 32 pages of an order of steps, one per lane (-1: not there); `base`: the first one, counted from the order's first page.
struct PageWindow {
    int base, id;
    uint32_t there;             // bit l: lane l's page is there
};

// A stage costs the loading warp about forty instructions: a thread by itself, looking pages up one by one, was what bounded a step
// (0.5 us a stage).  Lanes hold page ids ahead and each issues one box.
template <int kDim>
__device__ __forceinline__ bool load_steps(const CacheView &c, const AttnArgs &a, const CUtensorMap *map_k, const CUtensorMap *map_v, AttnShared *sh,
                                           Ctl *ctl, unsigned char *ring, uint32_t &stage, uint32_t &keys0, uint32_t &keys1, const TileItem &x) {
    constexpr int kHalves = kDim / 64;
    const int lane = threadIdx.x & 31, shift = (int)c.page_shift;
    const int32_t *row = c.table + (size_t)x.seq * c.width;
    const int boxes = max(1, kStep >> shift);                 // pages of a step; a page of 128 holds two steps
    const int mine = lane / kHalves, half = lane % kHalves;   // page and half of this lane's box
    auto window = [&](int first, int pos0) {
        PageWindow p;
        p.base = first;
        const long long at = (long long)((pos0 >> shift) + first + lane) << shift;
        p.id = at < x.end ? row[at >> shift] : -1;
        if (p.id < 0 || (uint32_t)p.id >= c.pages) p.id = -1;
        p.there = __ballot_sync(0xffffffffu, p.id >= 0);
        return p;
    };
    PageWindow win[2] = {window(0, x.pos0), {0, -1, 0u}};
    if (!x.both && x.steps1 > 0) win[1] = window(0, x.pos1);
    return in_order(x, [&](int step, bool is_v, int w) {
        const int pos0 = w == 0 ? x.pos0 : x.pos1, pos = pos0 + step * kStep;
        PageWindow &p = win[w];
        const int first = (pos >> shift) - (pos0 >> shift);
        // Keys run ahead of values by two steps: the window moves with them and keeps what the values still need.
        if (first + boxes > p.base + 32) p = window(((pos0 + max(step - 2, 0) * kStep) >> shift) - (pos0 >> shift), pos0);
        const uint32_t s = stage % kRing;
        if (!__all_sync(0xffffffffu, wait_bar(&sh->ring_empty[s], ((stage / kRing) & 1u) ^ 1u, sh, ctl, kErrAttnTile))) return false;
        const int id = __shfl_sync(0xffffffffu, p.id, first - p.base + min(mine, boxes - 1));
        if (lane == 0) {
            // The workers read the word of a step's keys once they have its scores; they are less than a ring behind.
            if (!is_v) sh->pages[w][(w == 0 ? keys0 : keys1) % kPageWords] = p.there >> (first - p.base) & ((1u << boxes) - 1u);
            mbar_arrive_expect_tx(&sh->ring_full[s], step_bytes<kDim>());
        }
        if (!is_v) { if (w == 0) ++keys0; else ++keys1; }
        __syncwarp();
        if (lane < boxes * kHalves)                            // a page that is not there: outside the pool, zeros
            tma_load_3d(ring + (size_t)s * step_bytes<kDim>() + half * (kStep * 128) + ((size_t)mine << shift) * 128, is_v ? map_v : map_k,
                        &sh->ring_full[s], half * 64, x.head * (int)c.page + (pos & (int)(c.page - 1)), id < 0 ? -1 : (int)(a.layer * c.pages) + id);
        ++stage;
        return true;
    });
}

// ---- issuer (one warp) -------------------------------------------------------------------------------------------
struct IssueState {
    uint32_t stage;             // ring stages consumed, in the order of loading
    uint32_t q, p;              // parities to wait for: queries (bit: group), weights (bit: 2 * group + buffer)
};

// A step is 2 * (8 + 4) MMAs, six commits and four waits at head_dim 128, and has to be issued in about 1300 clocks.  Groups and buffers
// are unrolled, so descriptors are constants plus the stage's offset and parities are bits of one register.
template <class T, int kDim>
__device__ __forceinline__ bool issue_steps(AttnShared *sh, Ctl *ctl, unsigned char *smem_q, unsigned char *ring, IssueState &st, int n0, int n1,
                                            bool both, uint32_t lead) {
    const uint32_t tmem = __shfl_sync(0xffffffffu, *(volatile uint32_t *)&sh->tmem, 0);
    const uint64_t qd = make_kmajor_sw128_desc(smem_u32(smem_q)), kd = make_kmajor_sw128_desc(smem_u32(ring)), vd = make_v_desc(smem_u32(ring));
    auto full = [&](uint32_t stage) {
        const bool ok = __all_sync(0xffffffffu, wait_bar(&sh->ring_full[stage % kRing], (stage / kRing) & 1u, sh, ctl, kErrAttnTile));
        tc_fence_after();
        return ok;
    };
    auto scores = [&](int w, int b, uint32_t stage) {         // S_w = Q_w K^T, into buffer b
        const uint64_t q = qd + (uint64_t)(w * (query_bytes<kDim>() >> 4)), k = kd + (uint64_t)((stage % kRing) * (step_bytes<kDim>() >> 4));
        const uint32_t d = tmem + w * kTile + b * kStep;
#pragma unroll
        for (int i = 0; i < kDim / 16; ++i)
            attn_mma_ss(d, q + (uint64_t)((i / 4) * (kTile * 128 >> 4) + (i % 4) * 2), k + (uint64_t)((i / 4) * (kStep * 128 >> 4) + (i % 4) * 2),
                        idesc_s<T>(), i > 0, lead);
        attn_commit(&sh->s_full[w][b], lead);
    };
    // O_w (+)= P_w V.  pv_done counts products: the group looks at it only for the newest or the one before, since a parity tells
    // no more apart; the item's last one has a barrier of its own.
    auto product = [&](int w, int b, uint32_t stage, bool first, bool last) {
        const uint64_t v = vd + (uint64_t)((stage % kRing) * (step_bytes<kDim>() >> 4));
        const uint32_t d = tmem + 2 * kTile + w * kDim, p = tmem + w * kTile + b * kStep;
#pragma unroll
        for (int i = 0; i < kStep / 16; ++i) attn_mma_ts(d, p + i * 8, v + (uint64_t)(i * (2048 >> 4)), idesc_o<T, kDim>(), !first || i > 0, lead);
        attn_commit(&sh->pv_done[w], lead);
        if (last) attn_commit(&sh->o_full[w], lead);
    };
    auto release = [&](uint32_t stage) { attn_commit(&sh->ring_empty[stage % kRing], lead); };
    auto queries = [&](int w) {
        const bool ok = __all_sync(0xffffffffu, wait_bar(&sh->q_full[w], st.q >> w & 1u, sh, ctl, kErrAttnTile));
        st.q ^= 1u << w;
        return ok;
    };
    auto weights = [&](int w, int b) {
        const bool ok = __all_sync(0xffffffffu, wait_bar(&sh->p_full[w][b], st.p >> (2 * w + b) & 1u, sh, ctl, kErrAttnTile));
        st.p ^= 1u << (2 * w + b);
        tc_fence_after();
        return ok;
    };
    uint32_t next = st.stage;                                  // the order of in_order()
    if (both) {
        const int n = n0;
        if (n > 0 && !queries(0)) return false;
        const uint32_t first = next;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if (b >= n) break;
            if (!full(next)) return false;
            scores(0, b, next++);
        }
        if (n > 0 && !queries(1)) return false;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if (b >= n) break;
            scores(1, b, first + b);
            release(first + b);
        }
        for (int s0 = 0; s0 < n; s0 += 2) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int s = s0 + b;
                if (s >= n) break;
                const bool more = s + 2 < n;
                const uint32_t v = next++, k = next;
                if (more) ++next;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (!weights(w, b) || (w == 0 && !full(v))) return false;
                    product(w, b, v, s == 0, s + 1 == n);
                    if (w == 1) release(v);
                    if (!more) continue;
                    if (w == 0 && !full(k)) return false;
                    scores(w, b, k);
                    if (w == 1) release(k);
                }
            }
        }
    } else {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int n = w == 0 ? n0 : n1;
            if (n > 0 && !queries(w)) return false;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (b >= n) break;
                if (!full(next)) return false;
                scores(w, b, next);
                release(next++);
            }
        }
        for (int s0 = 0; s0 < max(n0, n1); s0 += 2) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const int s = s0 + b, n = w == 0 ? n0 : n1;
                    if (s >= n) continue;
                    if (!weights(w, b) || !full(next)) return false;
                    product(w, b, next, s == 0, s + 1 == n);
                    release(next++);
                    if (s + 2 >= n) continue;
                    if (!full(next)) return false;
                    scores(w, b, next);
                    release(next++);
                }
        }
    }
    st.stage = next;
    return true;
}

// ---- workers (two groups of 128 threads) -------------------------------------------------------------------------
// Row `i` of an item: where its query and its output are, the positions it sees, and its row among its kind.
struct RowOf {
    long long token;            // row of q
    int sub;                    // query head within the key head's group
    int limit;                  // positions below it are seen
};
__device__ __forceinline__ RowOf row_of(const AttnArgs &a, const AttnShared *sh, const TileItem &x, int i) {
    RowOf r;
    int e = x.entry, in = x.r0 + i;
    if (e < 0) {
        int lo = 0, hi = (int)a.n - 1;                       // the last sequence with at most `in` sharing rows before it
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (sh->pre0[mid] <= in) lo = mid; else hi = mid - 1;
        }
        e = lo;
        in -= sh->pre0[lo];
    }
    const SeqPlan &p = sh->plan[e];
    r.token = (long long)p.row0 + in / (int)a.group;
    r.sub = in % (int)a.group;
    r.limit = x.entry < 0 ? x.end : p.len - p.t + in / (int)a.group + 1;
    return r;
}

// Queries of a group's 128 rows into shared memory (rows beyond the item's: zeros), K-major, 128-byte swizzle; their signs
// flipped where the scale is negative, so that the largest score is the largest product.
template <class T, int kDim>
__device__ __forceinline__ void stage_queries(const AttnArgs &a, unsigned char *dst, const TileItem &x, const RowOf &mine, bool real, int group_warp) {
    constexpr int kLanes = kDim / 8, kAtOnce = 32 / kLanes;
    const int lane = threadIdx.x & 31;
    const T *src = static_cast<const T *>(a.q) + (size_t)mine.token * a.q_stride + (size_t)(x.head * (int)a.group + mine.sub) * kDim;
    const unsigned long long at = (unsigned long long)src;      // a row that is not real: some row's queries, thrown away
    const uint32_t reals = __ballot_sync(0xffffffffu, real), flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    // All loads first, without conditions: one after another they would cost a round trip each.
    uint4 v[32 / kAtOnce];
#pragma unroll
    for (int i = 0; i < 32 / kAtOnce; ++i)
        v[i] = __ldg(reinterpret_cast<const uint4 *>(__shfl_sync(0xffffffffu, at, i * kAtOnce + lane / kLanes)) + lane % kLanes);
#pragma unroll
    for (int i = 0; i < 32 / kAtOnce; ++i) {
        const int r = i * kAtOnce + lane / kLanes;
        const bool keep = reals >> r & 1u;
        v[i] = keep ? make_uint4(v[i].x ^ flip, v[i].y ^ flip, v[i].z ^ flip, v[i].w ^ flip) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4 *>(dst + swz((uint32_t)(group_warp * 32 + r), (uint32_t)(lane % kLanes), kTile)) = v[i];
    }
}

struct WorkState {
    uint32_t stage;             // ring stages of the items so far
    uint32_t s, o;              // parities to wait for: scores (bit: buffer), results
    uint32_t pv, keys0, keys1;  // products of the group, and steps of both orders of keys, in the items so far
    uint32_t bar;               // meetings of the group
};

// The four warps of a group meet; bounded like every wait, since a warp that gave up does not come.
__device__ __forceinline__ bool group_meet(AttnShared *sh, Ctl *ctl, WorkState &st, int w) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sh->group_bar[w]);
    return __all_sync(0xffffffffu, wait_bar(&sh->group_bar[w], st.bar++ & 1u, sh, ctl, kErrAttnTile));
}

// A group's rows of an item by units, which add values that are not finite with selects.  Their rings lie where the group's queries
// were (a stage each), which nobody reads any more.  Not inlined: it never runs on sane data and would cost the loop registers.
template <class T, int kDim>
__device__ __noinline__ void redo_rows(const CacheView &c, const AttnArgs &a, const CUtensorMap *map_k, const CUtensorMap *map_v, AttnShared *sh, Ctl *ctl,
                                       unsigned char *place, Ring &units, const TileItem &x, int w, int warp, int pos0, int steps) {
    units.move(place + warp * unit_stage_bytes<kDim>(), 1);
    const int begin = x.both ? w * (kTile / kUnitRows) : 0, end = x.both ? min(x.groups, begin + kTile / kUnitRows) : x.groups;
    for (int i = begin + warp; i < end; i += 4) {
        Unit u;
        u.entry = x.entry;
        u.head = x.head;
        u.r0 = x.r0 + i * kUnitRows;
        u.rows = min(kUnitRows, x.rows - i * kUnitRows);
        u.from = x.from;
        u.first = (pos0 - x.from) / kBlock;
        u.last = min(u.first + steps * (kStep / kBlock), (x.end - x.from + kBlock - 1) / kBlock);
        u.slot = x.slot0 < 0 ? -1 : x.slot0 + i * x.step + (x.half == 2 ? w : 0);
        run_unit<T, kDim, 2>(c, a, map_k, map_v, sh, ctl, units, u);
    }
}

template <class T, int kDim>
__device__ __forceinline__ void work_tiles(const CacheView &c, const AttnArgs &a, const CUtensorMap *map_k, const CUtensorMap *map_v, AttnShared *sh,
                                           Ctl *ctl, unsigned char *smem_q, unsigned char *ring, WorkState &st, Ring &units, const TileItem &x) {
    const int w = threadIdx.x >> 7, in_group = threadIdx.x & 127, warp = in_group >> 5, lane = threadIdx.x & 31;
    if (!x.both && x.half == 1 && w == 1) {                   // no rows for the second group
        st.stage += stages_of(x);
        st.keys0 += x.steps0;
        return;
    }
    const int row = (x.both ? w * kTile : 0) + in_group;
    const bool real = row < x.rows;
    const RowOf mine = row_of(a, sh, x, real ? row : 0);
    const int limit = real ? min(mine.limit, x.end) : 0;
    const uint32_t tmem = *(volatile uint32_t *)&sh->tmem + ((uint32_t)(warp * 32) << 16);
    const uint32_t to = tmem + 2 * kTile + w * kDim;
    const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);     // 0 would turn a hidden score into NaN
    float ref = -INFINITY;
    // The smallest limit of the item's rows.
    int least = x.end;
    if (x.entry >= 0) least = min(least, sh->plan[x.entry].len - sh->plan[x.entry].t + x.r0 / (int)a.group + 1);
    const uint32_t stage0 = st.stage;
    const int n = w == 0 ? x.steps0 : x.steps1, pos0 = w == 0 ? x.pos0 : x.pos1, order = x.both ? 0 : w;
    unsigned char *my_q = smem_q + w * query_bytes<kDim>();
    if (n > 0) {
        stage_queries<T, kDim>(a, my_q, x, mine, real, warp);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->q_full[w]);
    }
    const int page_shift = min((int)c.page_shift, 6);            // of the part of a page that is in a step
    const uint32_t whole = (1u << (kStep >> page_shift)) - 1u;
    bool looked = false;                                        // some values were looked at: the group agrees on it
    // A step: maximum, then exponentials of the first 32 scores; their registers are free for the next step's, whose load runs under the
    // other 32 and under the store of the weights.
    uint32_t lo[32], hi[32], p[32];
    uint64_t part = 0ull;
    float base = 0.f;                                           // ref * scale, 0 while nothing was seen
    const uint64_t scale2 = two(scale, scale);
    auto scores = [&](int s) { return tmem + w * kTile + (s & 1) * kStep; };
    auto ready = [&](int s) {
        const bool ok = __all_sync(0xffffffffu, wait_bar(&sh->s_full[w][s & 1], st.s >> (s & 1) & 1u, sh, ctl, kErrAttnTile));
        st.s ^= 1u << (s & 1);
        tc_fence_after();
        return ok;
    };
    auto exps = [&](const uint32_t (&r)[32], int at) {
        const uint64_t base2 = two(-base, -base);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 e = of_two(fma_two(two(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), scale2, base2));
            const float e0 = ex2(e.x), e1 = ex2(e.y);
            part = add_two(part, two(e0, e1));
            p[at + i] = Elem<T>::pack(e0, e1);
        }
    };
    if (n > 0) {
        if (!ready(0)) return;
        tc_ld32(scores(0), lo);
        tc_ld32(scores(0) + 32, hi);
        tc_landed(lo);
        tc_pin(hi);
    }
    for (int s = 0; s < n; ++s) {
        const int pos = pos0 + s * kStep;
        const uint32_t there = *(volatile uint32_t *)&sh->pages[order][((order == 0 ? st.keys0 : st.keys1) + s) % kPageWords];
        // Some row does not see some position: at the item's end, or where a page is not there.
        if (pos + kStep > least || there != whole) {
            const uint32_t vs = stage0 + v_stage(x, w, s);
            if (!__all_sync(0xffffffffu, wait_bar(&sh->ring_full[vs % kRing], (vs / kRing) & 1u, sh, ctl, kErrAttnTile))) return;
            unsigned char *v = ring + (size_t)(vs % kRing) * step_bytes<kDim>();
            looked = true;
            if (in_group < kStep) {                             // each thread looks after one position's values
                const uint32_t at = (uint32_t)in_group;
                if (pos + in_group >= x.end) {
#pragma unroll
                    for (int i = 0; i < kDim / 8; ++i) *reinterpret_cast<uint4 *>(v + swz(at, (uint32_t)i, kStep)) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                } else if (pos + in_group >= least) {
                    bool odd = false;
#pragma unroll 4
                    for (int i = 0; i < kDim / 8; ++i) {
                        const uint4 y = *reinterpret_cast<const uint4 *>(v + swz(at, (uint32_t)i, kStep));
                        const uint32_t z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            odd |= (z[k] & Elem<T>::kInfBits) == Elem<T>::kInfBits || (z[k] >> 16 & Elem<T>::kInfBits) == Elem<T>::kInfBits;
                    }
                    if (odd) *(volatile uint32_t *)&sh->odd[w] = 1u;
                }
            }
            const int seen = limit - pos;
#pragma unroll
            for (int i = 0; i < kStep; ++i)
                if (i >= seen || !(there >> (i >> page_shift) & 1u)) (i < 32 ? lo[i & 31] : hi[i & 31]) = 0xff800000u;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; i += 4)
#pragma unroll
            for (int k = 0; k < 4; ++k) top[k] = max_three(top[k], __uint_as_float(lo[i + k]), __uint_as_float(hi[i + k]));
        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        // (-inf) - (-inf) is no reason to move.
        if (__any_sync(0xffffffffu, (most - ref) * scale > kLag)) {
            const float now = (most - ref) * scale > kLag ? most : ref, down = ref == -INFINITY ? 0.f : ex2((ref - now) * scale);
            ref = now;
            base = ref == -INFINITY ? 0.f : ref * scale;
            part = mul_two(part, two(down, down));
            if (s > 0) {                                        // O stands still once the product before this step is done (the one before that is)
                if (!__all_sync(0xffffffffu, wait_bar(&sh->pv_done[w], (st.pv + s - 1) & 1u, sh, ctl, kErrAttnTile))) return;
                tc_fence_after();
#pragma unroll 1
                for (int i = 0; i < kDim; i += 16) {            // few registers: scores are waiting in most of them
                    uint32_t o[16];
                    tc_ld16(to + i, o);
                    tc_landed(o);
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * down);
                    tc_st16(to + i, o);
                }
            }
        }
        const bool more = s + 1 < n;
        exps(lo, 0);
        if (more) {
            if (!ready(s + 1)) return;
            tc_ld32(scores(s + 1), lo);
        }
        exps(hi, 16);
        if (more) tc_ld32(scores(s + 1) + 32, hi);
        tc_st32(scores(s), p);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[w][s & 1]);
        if (more) {                                             // here and not where they are used: registers may be moved in between
            tc_landed(lo);
            tc_pin(hi);
        }
    }
    const float2 sums = of_two(part);
    const float sum = sums.x + sums.y;
    st.stage = stage0 + stages_of(x);
    st.keys0 += x.steps0;
    if (!x.both) st.keys1 += x.steps1;
    if (n > 0) {
        if (!__all_sync(0xffffffffu, wait_bar(&sh->o_full[w], st.o, sh, ctl, kErrAttnTile))) return;
        st.o ^= 1u;
        st.pv += n;
        tc_fence_after();
    }
    const bool direct = x.slot0 < 0;
    bool again = false;
    if (looked) {                                               // were the values that somebody did not see all finite?
        if (!group_meet(sh, ctl, st, w)) return;
        again = *(volatile uint32_t *)&sh->odd[w] != 0u;
        if (!group_meet(sh, ctl, st, w)) return;
        if (in_group == 0) sh->odd[w] = 0;                      // nobody looks again before this warp's next queries are there
    }
    if (!again) {
        // Row r of the item belongs to group r / 16, the second workers' half to the slot behind.  Without steps the result is empty.
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const size_t slot = direct ? 0 : (size_t)(x.slot0 + row / kUnitRows * x.step + (x.half == 2 ? w : 0));
        const size_t place = slot * kUnitRows + row % kUnitRows;
        if (!direct && real) __stcg(a.part_ml + place, n > 0 ? make_float2(ref == -INFINITY ? -INFINITY : ref * scale, sum) : make_float2(-INFINITY, 0.f));
        // A thread has a row, a store instruction wants consecutive bytes: rows pass through the group's queries (nobody reads them any
        // more), each warp through its own 32.
        const unsigned long long to_row = direct ? (unsigned long long)(static_cast<T *>(a.out) + (size_t)mine.token * a.out_stride
                                                                        + (size_t)(x.head * (int)a.group + mine.sub) * kDim)
                                                 : (unsigned long long)(a.part + place * kDim);
        const uint32_t reals = __ballot_sync(0xffffffffu, real);
        auto out_rows = [&](auto width, int skip) {             // `width` 16-byte chunks of each row, from byte `skip` of it
            constexpr int kChunks = decltype(width)::value, kRows = 32 / kChunks;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int r = i * kRows + lane / kChunks;
                const uint4 y = *reinterpret_cast<const uint4 *>(my_q + swz((uint32_t)(warp * 32 + r), (uint32_t)(lane % kChunks), kTile));
                const unsigned long long p = __shfl_sync(0xffffffffu, to_row, r);
                if (reals >> r & 1u) __stcg(reinterpret_cast<uint4 *>(p + skip) + lane % kChunks, y);
            }
            __syncwarp();
        };
        if (direct) {
#pragma unroll 1
            for (int i = 0; i < kDim; i += 32) {
                uint32_t o[32];
                if (n > 0) tc_ld32(to + i, o);
                tc_landed(o);
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    uint32_t y[4];
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        y[m] = sum == 0.f ? 0u : Elem<T>::pack(__uint_as_float(o[k + 2 * m]) * inv, __uint_as_float(o[k + 2 * m + 1]) * inv);
                    *reinterpret_cast<uint4 *>(my_q + swz((uint32_t)in_group, (uint32_t)((i + k) / 8), kTile)) = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
            out_rows(std::integral_constant<int, kDim / 8>(), 0);
        } else if (n > 0) {
            constexpr int kPass = query_bytes<kDim>() / kTile / 4;          // elements of a row that fit at a time
#pragma unroll 1
            for (int at = 0; at < kDim; at += kPass) {
#pragma unroll 1
                for (int i = 0; i < kPass; i += 32) {
                    uint32_t o[32];
                    tc_ld32(to + at + i, o);
                    tc_landed(o);
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<uint4 *>(my_q + swz((uint32_t)in_group, (uint32_t)((i + k) / 4), kTile)) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
                out_rows(std::integral_constant<int, kPass / 4>(), at * 4);
            }
        }
    } else {
        // Hidden values that are not finite: the group's rows once more.
        const TileItem copy = x;                                // the call wants addresses: not those of what the loop keeps in registers
        Ring ring_copy = units;
        redo_rows<T, kDim>(c, a, map_k, map_v, sh, ctl, my_q, ring_copy, copy, w, warp, pos0, n);
        units = ring_copy;
        if (!group_meet(sh, ctl, st, w)) return;                // the next queries may come
    }
    tc_fence_before();
    if (!direct) {                                              // tell the merges how many row groups have their result
        __threadfence();
        if (!group_meet(sh, ctl, st, w)) return;
        const int mine_groups = x.half == 2 ? x.groups : max(min(x.groups - w * (kTile / kUnitRows), kTile / kUnitRows), 0);
        if (in_group == 64) atomicAdd(&a.counters[(size_t)(x.entry < 0 ? (int)a.n : x.entry) * c.heads + x.head], (uint32_t)mine_groups);
    }
}

} // namespace xpk
