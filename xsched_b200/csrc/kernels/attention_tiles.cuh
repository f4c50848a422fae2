// Tiles of an attention call (see attention.cu): up to 256 rows against 128 positions at a time on the tensor pipe.
//
// Two groups of four warps take 128 rows each (thread = row), or, where an item has at most 128 rows, the same rows and one
// half of the positions each.  Per tile and group:
//
//   S = Q K^T     tcgen05.mma M128 N128, Q and K from shared memory (K-major), S fp32 in tensor memory
//   P = exp2(..)  the group's threads read their rows of S, keep maximum and sum, and write P (16 bit) over S
//   O += P V      tcgen05.mma with P from tensor memory and V from shared memory (dimension-major: V lies as it is stored)
//
// One thread issues the MMAs of both groups in turn, so that one group's exponentials run under the other's products;
// another fills a ring of four stages (a tile of K or of V, 32 KB) by TMA, page by page.  MMAs of one thread execute in the
// order of issue: S of tile j + 1 may overwrite P of tile j once P V of tile j has been issued.  The barrier that says
// "S is there" therefore also says that the P V before it is done, and the group may touch O.
//
// O is not rescaled whenever the maximum grows: p is taken relative to a reference that follows the maximum only when it
// falls 2^8 behind, so p stays below 2^8 (fp16 holds 2^15) and almost every tile leaves O alone.
//
// Bound by the tensor pipe (4 * 128 * 128 * head_dim flop per group and tile: 0.55 us at 128) and by the exponentials
// (16 a clock and SM: 0.55 us) alike; K and V of a tile are fetched once for 256 rows.
#pragma once
#include "attention_units.cuh"

namespace xpk {

constexpr float kLag = 8.f;                                  // log2 units that the reference may fall behind the maximum

// ---- instructions ------------------------------------------------------------------------------------------------
__device__ __forceinline__ void attn_commit(void *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void attn_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void attn_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
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
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// V as B operand with the dimension contiguous: atoms of 64 dimensions x 8 positions (1024 B, 128-byte swizzle), the next
// eight positions behind it, the next 64 dimensions a whole tile of 128 positions further.
__device__ __forceinline__ uint64_t make_v_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)((kTile * 128u) >> 4) << 16;              // leading byte offset: between blocks of 64 dimensions
    d |= (uint64_t)(1024u >> 4) << 32;                       // stride byte offset: between groups of eight positions
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
template <class T> __host__ __device__ constexpr uint32_t mma_type() { return sizeof(T) == 2 ? 1u : 0u; }
template <> __host__ __device__ constexpr uint32_t mma_type<__half>() { return 0u; }
// D fp32; N = 128 positions, both K-major; N = kDim, B with N contiguous.
template <class T> __host__ __device__ constexpr uint32_t idesc_s() {
    return (1u << 4) | (mma_type<T>() << 7) | (mma_type<T>() << 10) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
template <class T, int kDim> __host__ __device__ constexpr uint32_t idesc_o() {
    return (1u << 4) | (mma_type<T>() << 7) | (mma_type<T>() << 10) | (1u << 16) | ((uint32_t)(kDim >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
constexpr uint32_t kAttnTmemCols = 512;                      // S of both groups (128 each), O of both (head_dim each)

// ---- an item -----------------------------------------------------------------------------------------------------
struct TileItem {
    int entry;                  // -1: the prefix
    int head, r0, rows;         // first row (of the sequence, or of all sharing ones), rows (up to 256)
    int from, end;              // positions [from, end) are the item's
    int seq;                    // whose table names the pages
    bool both;                  // both groups take every tile
    int first[2], count[2];     // tiles of each group, counted from `from`
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
    x.half = halves(all);
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
    const int first = run * sh->tile_run, last = min(first + sh->tile_run, (most + kTile - 1) / kTile), count = max(last - first, 0);
    x.both = x.half == 1 && x.rows > kTile;
    x.first[0] = x.first[1] = first;
    x.count[0] = x.count[1] = count;
    if (x.half == 2) {
        x.count[0] = (count + 1) / 2;
        x.first[1] = first + x.count[0];
        x.count[1] = count - x.count[0];
    } else if (!x.both) {
        x.count[1] = 0;
    }
    const int base = x.entry < 0 ? sh->pre_part0 : sh->part0[x.entry];
    x.step = runs * x.half;
    x.slot0 = base < 0 ? -1 : base + (x.head * row_groups(all) + x.r0 / kUnitRows) * x.step + run * x.half;
    return x;
}

// Counts of phases that each role has gone through; they go on from item to item.
struct TileState {
    uint32_t stage;             // ring stages filled (loader) or consumed (issuer, workers: in the order of loading)
    uint32_t s, o;              // workers: tiles with scores and items with results of their group
    uint32_t q[2], p[2];        // issuer: items with queries and tiles with weights of each group
};

// The order in which tiles of K and V are used: f(tile, is_v, group) for each stage of the ring.
template <class F>
__device__ __forceinline__ bool in_order(const TileItem &x, F f) {
    if (x.both) {
        const int n = x.count[0];
        if (n > 0 && !f(x.first[0], false, 0)) return false;
        for (int j = 0; j < n; ++j) {
            if (!f(x.first[0] + j, true, 0)) return false;
            if (j + 1 < n && !f(x.first[0] + j + 1, false, 0)) return false;
        }
        return true;
    }
    for (int w = 0; w < 2; ++w)
        if (x.count[w] > 0 && !f(x.first[w], false, w)) return false;
    for (int j = 0; j < max(x.count[0], x.count[1]); ++j)
        for (int w = 0; w < 2; ++w) {
            if (j >= x.count[w]) continue;
            if (!f(x.first[w] + j, true, w)) return false;
            if (j + 1 < x.count[w] && !f(x.first[w] + j + 1, false, w)) return false;
        }
    return true;
}

// ---- loader (one thread) -----------------------------------------------------------------------------------------
template <int kDim>
__device__ __forceinline__ void load_tiles(const CacheView &c, const AttnArgs &a, const CUtensorMap *map_k, const CUtensorMap *map_v, AttnShared *sh,
                                           Ctl *ctl, unsigned char *ring, TileState &st, const TileItem &x) {
    const int32_t *row = c.table + (size_t)x.seq * c.width;
    const int per = kTile >> c.page_shift;                     // pages of a tile
    in_order(x, [&](int tile, bool is_v, int) {
        const uint32_t s = st.stage % kRing;
        if (!wait_bar(&sh->ring_empty[s], ((st.stage / kRing) & 1u) ^ 1u, sh, ctl, kErrAttnTile)) return false;
        unsigned char *dst = ring + (size_t)s * tile_bytes<kDim>();
        const int pos = x.from + tile * kTile;
        uint32_t there = 0;
        int ids[kTile / 16];
#pragma unroll
        for (int j = 0; j < kTile / 16; ++j) {
            if (j >= per) break;
            const int at = pos + (j << c.page_shift);
            int id = at < x.end ? row[at >> c.page_shift] : -1;
            if (id < 0 || (uint32_t)id >= c.pages) id = -1; else there |= 1u << j;
            ids[j] = id;
        }
        sh->stage_pages[s] = there;                            // read by the workers once the stage is full
        mbar_arrive_expect_tx(&sh->ring_full[s], tile_bytes<kDim>());
#pragma unroll
        for (int j = 0; j < kTile / 16; ++j) {
            if (j >= per) break;
            const int z = ids[j] < 0 ? -1 : (int)(a.layer * c.pages) + ids[j];        // outside the pool: zeros
#pragma unroll
            for (int h = 0; h < kDim / 64; ++h)
                tma_load_3d(dst + h * (kTile * 128) + ((size_t)j << c.page_shift) * 128, is_v ? map_v : map_k, &sh->ring_full[s], h * 64,
                            x.head * (int)c.page, z);
        }
        ++st.stage;
        return true;
    });
}

// ---- issuer (one thread) -----------------------------------------------------------------------------------------
template <class T, int kDim>
__device__ __forceinline__ void issue_tiles(AttnShared *sh, Ctl *ctl, unsigned char *smem_q, unsigned char *ring, TileState &st, const TileItem &x) {
    const uint32_t tmem = *(volatile uint32_t *)&sh->tmem;
    const uint32_t q0 = smem_u32(smem_q), r0 = smem_u32(ring);
    auto full = [&](uint32_t stage) { return wait_bar(&sh->ring_full[stage % kRing], (stage / kRing) & 1u, sh, ctl, kErrAttnTile); };
    auto scores = [&](int w, uint32_t stage) {                // S_w = Q_w K^T
        const uint32_t q = q0 + w * tile_bytes<kDim>(), k = r0 + (stage % kRing) * tile_bytes<kDim>();
#pragma unroll
        for (int i = 0; i < kDim / 16; ++i) {
            const uint32_t off = (i / 4) * (kTile * 128) + (i % 4) * 32;
            attn_mma_ss(tmem + w * kTile, make_kmajor_sw128_desc(q + off), make_kmajor_sw128_desc(k + off), idesc_s<T>(), i > 0);
        }
        attn_commit(&sh->s_full[w]);
    };
    auto product = [&](int w, uint32_t stage, bool add) {     // O_w (+)= P_w V
        const uint32_t v = r0 + (stage % kRing) * tile_bytes<kDim>();
#pragma unroll
        for (int i = 0; i < kTile / 16; ++i)
            attn_mma_ts(tmem + 2 * kTile + w * kDim, tmem + w * kTile + i * 8, make_v_desc(v + i * 2048), idesc_o<T, kDim>(), add || i > 0);
    };
    auto queries = [&](int w) {
        const bool ok = wait_bar(&sh->q_full[w], st.q[w] & 1u, sh, ctl, kErrAttnTile);
        ++st.q[w];
        return ok;
    };
    auto weights = [&](int w) {
        const bool ok = wait_bar(&sh->p_full[w], st.p[w] & 1u, sh, ctl, kErrAttnTile);
        ++st.p[w];
        tc_fence_after();
        return ok;
    };
    if (x.both) {
        const int n = x.count[0];
        if (n == 0) return;
        for (int w = 0; w < 2; ++w)
            if (!queries(w)) return;
        if (!full(st.stage)) return;
        tc_fence_after();
        scores(0, st.stage);
        scores(1, st.stage);
        attn_commit(&sh->ring_empty[st.stage % kRing]);
        ++st.stage;
        for (int j = 0; j < n; ++j) {
            const uint32_t v = st.stage++, k = st.stage;
            const bool more = j + 1 < n;
            if (more) ++st.stage;
            for (int w = 0; w < 2; ++w) {
                if (!weights(w)) return;
                if (w == 0 && !full(v)) return;
                tc_fence_after();
                product(w, v, j > 0);
                if (w == 1) attn_commit(&sh->ring_empty[v % kRing]);
                if (more) {
                    if (w == 0 && !full(k)) return;
                    tc_fence_after();
                    scores(w, k);
                    if (w == 1) attn_commit(&sh->ring_empty[k % kRing]);
                } else {
                    attn_commit(&sh->o_full[w]);
                }
            }
        }
        return;
    }
    for (int w = 0; w < 2; ++w) {
        if (x.count[w] == 0) continue;
        if (!queries(w) || !full(st.stage)) return;
        tc_fence_after();
        scores(w, st.stage);
        attn_commit(&sh->ring_empty[st.stage % kRing]);
        ++st.stage;
    }
    for (int j = 0; j < max(x.count[0], x.count[1]); ++j)
        for (int w = 0; w < 2; ++w) {
            if (j >= x.count[w]) continue;
            if (!weights(w) || !full(st.stage)) return;
            tc_fence_after();
            product(w, st.stage, j > 0);
            attn_commit(&sh->ring_empty[st.stage % kRing]);
            ++st.stage;
            if (j + 1 < x.count[w]) {
                if (!full(st.stage)) return;
                tc_fence_after();
                scores(w, st.stage);
                attn_commit(&sh->ring_empty[st.stage % kRing]);
                ++st.stage;
            } else {
                attn_commit(&sh->o_full[w]);
            }
        }
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
    const unsigned long long at = real ? (unsigned long long)src : 0ull;
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll 4
    for (int i = 0; i < 32; i += kAtOnce) {
        const int r = i + lane / kLanes, chunk = lane % kLanes;
        const unsigned long long p = __shfl_sync(0xffffffffu, at, r);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (p != 0) v = __ldg(reinterpret_cast<const uint4 *>(p) + chunk);
        v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
        *reinterpret_cast<uint4 *>(dst + swz((uint32_t)(group_warp * 32 + r), (uint32_t)chunk, kTile)) = v;
    }
}

template <class T, int kDim>
__device__ __forceinline__ void work_tiles(const CacheView &c, const AttnArgs &a, AttnShared *sh, Ctl *ctl, unsigned char *smem_q, unsigned char *ring,
                                           TileState &st, const TileItem &x) {
    const int w = threadIdx.x >> 7, in_group = threadIdx.x & 127, warp = in_group >> 5, lane = threadIdx.x & 31;
    const int row = (x.both ? w * kTile : 0) + in_group;
    const bool real = row < x.rows;
    const RowOf mine = row_of(a, sh, x, real ? row : 0);
    const int limit = real ? min(mine.limit, x.end) : 0;
    const uint32_t tmem = *(volatile uint32_t *)&sh->tmem + ((uint32_t)(warp * 32) << 16);
    const uint32_t ts = tmem + w * kTile, to = tmem + 2 * kTile + w * kDim;
    const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);     // 0 would turn a hidden score into NaN
    float ref = -INFINITY, sum = 0.f;

    // The smallest limit of the item's rows, and the stage of the ring that holds the group's next values.
    int least = x.end;
    if (x.entry >= 0) least = min(least, sh->plan[x.entry].len - sh->plan[x.entry].t + x.r0 / (int)a.group + 1);
    const uint32_t stage0 = st.stage;
    const int n = x.count[w];
    if (n > 0) {
        stage_queries<T, kDim>(a, smem_q + w * tile_bytes<kDim>(), x, mine, real, warp);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->q_full[w]);
    }
    bool ok = true;
    for (int j = 0; j < n && ok; ++j) {
        ok = __all_sync(0xffffffffu, wait_bar(&sh->s_full[w], st.s & 1u, sh, ctl, kErrAttnTile));
        if (!ok) break;
        ++st.s;
        tc_fence_after();
        uint32_t r[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tc_ld32(ts + i * 32, *reinterpret_cast<uint32_t (*)[32]>(&r[i * 32]));
        tc_wait_ld();
        // Where the group's V of this tile lies in the ring, in the order of loading.
        const int pos = x.from + (x.first[w] + j) * kTile;
        uint32_t vstage;
        if (x.both) {
            vstage = stage0 + 1 + 2 * j;
        } else {
            // stages before V_w(j): the first keys of both groups, then per tile and group a V and, but for the last, a K
            vstage = stage0 + (x.count[0] > 0) + (x.count[1] > 0);
            const int before0 = w == 0 ? j : j + 1, before1 = j;
            vstage += min(before0, x.count[0]) + min(before0, max(x.count[0] - 1, 0));
            vstage += min(before1, x.count[1]) + min(before1, max(x.count[1] - 1, 0));
        }
        // Some row does not see some position: the item's last tiles, or a page that is not there.  The pages of a tile are
        // those of its V as well: the stage's word is read once V has arrived.
        const bool edge = pos + kTile > least;
        ok = __all_sync(0xffffffffu, wait_bar(&sh->ring_full[vstage % kRing], (vstage / kRing) & 1u, sh, ctl, kErrAttnTile));
        if (!ok) break;
        const uint32_t there = *(volatile uint32_t *)&sh->stage_pages[vstage % kRing];
        const uint32_t whole = (1u << (kTile >> c.page_shift)) - 1u;
        if (edge || there != whole) {
            unsigned char *v = ring + (size_t)(vstage % kRing) * tile_bytes<kDim>();
            const int at = pos + in_group;                    // each thread looks after one position's values
            if (at >= x.end) {
#pragma unroll
                for (int i = 0; i < kDim / 8; ++i) *reinterpret_cast<uint4 *>(v + swz((uint32_t)in_group, (uint32_t)i, kTile)) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            } else if (at >= least) {
                bool odd = false;
#pragma unroll 4
                for (int i = 0; i < kDim / 8; ++i) {
                    const uint4 y = *reinterpret_cast<const uint4 *>(v + swz((uint32_t)in_group, (uint32_t)i, kTile));
                    const uint32_t z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        odd |= (z[k] & Elem<T>::kInfBits) == Elem<T>::kInfBits || (z[k] >> 16 & Elem<T>::kInfBits) == Elem<T>::kInfBits;
                }
                if (odd) *(volatile uint32_t *)&sh->odd = 1u;
            }
            const int seen = limit - pos;
#pragma unroll
            for (int i = 0; i < 128; ++i)
                if (i >= seen || !(there >> (i >> c.page_shift) & 1u)) r[i] = 0xff800000u;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 4)
#pragma unroll
            for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], __uint_as_float(r[i + k]));
        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        float down = 1.f;
        if (most > ref && (ref == -INFINITY || (most - ref) * scale > kLag)) {
            down = ref == -INFINITY ? 0.f : ex2((ref - most) * scale);
            ref = most;
        }
        const float base = ref == -INFINITY ? 0.f : ref * scale;
        if (j > 0 && __any_sync(0xffffffffu, down != 1.f)) {
            sum *= down;
#pragma unroll 1
            for (int i = 0; i < kDim; i += 32) {
                uint32_t o[32];
                tc_ld32(to + i, o);
                tc_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * down);
                tc_st32(to + i, o);
            }
        }
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t p[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float e0 = ex2(fmaf(__uint_as_float(r[h * 64 + 2 * i]), scale, -base));
                const float e1 = ex2(fmaf(__uint_as_float(r[h * 64 + 2 * i + 1]), scale, -base));
                part[(2 * i) & 3] += e0;
                part[(2 * i + 1) & 3] += e1;
                p[i] = Elem<T>::pack(e0, e1);
            }
            tc_st32(ts + h * 32, p);
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[w]);
        sum += (part[0] + part[1]) + (part[2] + part[3]);
    }
    // All stages of the item have been asked for, whether or not this group used them.
    const int k0 = x.count[0], k1 = x.both ? 0 : x.count[1];
    st.stage = stage0 + 2 * (k0 + k1);
    if (!ok) return;

    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (n > 0) {
        ok = __all_sync(0xffffffffu, wait_bar(&sh->o_full[w], st.o & 1u, sh, ctl, kErrAttnTile));
        if (!ok) return;
        ++st.o;
        tc_fence_after();
    }
    const bool direct = x.slot0 < 0;
    // Row r of the item belongs to group r / 16, the second workers' half to the slot behind.  Without tiles the result is empty.
    if (w == 1 && !x.both && x.half == 1) return;            // no rows for the second group
    const size_t slot = direct ? 0 : (size_t)(x.slot0 + row / kUnitRows * x.step + (x.half == 2 ? w : 0));
    const size_t place = slot * kUnitRows + row % kUnitRows;
    if (!direct && real) __stcg(a.part_ml + place, n > 0 ? make_float2(ref == -INFINITY ? -INFINITY : ref * scale, sum) : make_float2(-INFINITY, 0.f));
    T *out = static_cast<T *>(a.out) + (size_t)mine.token * a.out_stride + (size_t)(x.head * (int)a.group + mine.sub) * kDim;
    float *part = a.part + place * kDim;
#pragma unroll 1
    for (int i = 0; i < kDim; i += 32) {
        uint32_t o[32];
        if (n > 0) {
            tc_ld32(to + i, o);
            tc_wait_ld();
        } else {
            if (!direct) break;
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0;
        }
        if (!real) continue;
        if (direct) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
                uint32_t y[4];
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    y[m] = sum == 0.f ? 0u : Elem<T>::pack(__uint_as_float(o[k + 2 * m]) * inv, __uint_as_float(o[k + 2 * m + 1]) * inv);
                *reinterpret_cast<uint4 *>(out + i + k) = make_uint4(y[0], y[1], y[2], y[3]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
                __stcg(reinterpret_cast<float4 *>(part + i + k), make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]),
                                                                           __uint_as_float(o[k + 3])));
        }
    }
    tc_fence_before();
}

// An item whose hidden values were not finite, once more by units (which add such values with selects).
template <class T, int kDim>
__device__ __forceinline__ void redo_item(const CacheView &c, const AttnArgs &a, const CUtensorMap *map_k, const CUtensorMap *map_v, AttnShared *sh,
                                          Ctl *ctl, Ring &r, const TileItem &x) {
    const int parts = x.half;
    for (int i = threadIdx.x >> 5; i < x.groups * parts; i += kWorkers) {
        const int g = i / parts, h = i % parts;
        Unit u;
        u.entry = x.entry;
        u.head = x.head;
        u.r0 = x.r0 + g * kUnitRows;
        u.rows = min(kUnitRows, x.rows - g * kUnitRows);
        u.from = x.from;
        u.first = x.first[h] * (kTile / kBlock);
        u.last = min((x.first[h] + x.count[h]) * (kTile / kBlock), (x.end - x.from + kBlock - 1) / kBlock);
        u.slot = x.slot0 < 0 ? -1 : x.slot0 + g * x.step + h;
        run_unit<T, kDim, 2>(c, a, map_k, map_v, sh, ctl, r, u);
    }
}

} // namespace xpk
