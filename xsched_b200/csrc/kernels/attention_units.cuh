// Units and merges of an attention call (see attention.cu).
//
// A unit is HBM-bound: 2 * 16 * head_dim * 2 bytes per block for 4 * 16 * 16 * head_dim flop.  Each warp has a ring of
// blocks of its own in shared memory, filled by TMA (128-byte swizzle) ahead of use.  Scores are computed transposed,
// S^T = K Q^T with mma.m16n8k16 (positions are M, 8 rows are N), so that up to 8 rows cost one MMA column block, and
// O^T = V^T P^T; the C fragment of S^T becomes the B fragment of P^T by transposing its 8x8 quarters (movmatrix).  P is rounded to the
// cache's 16-bit type for the second product, as in the tiles; sums and products are fp32.
#pragma once
#include "attention_plan.cuh"

namespace xpk {

// One warp's ring of blocks.  Its place and depth change with what the CTA is doing; a stage's phase goes with its barrier.
struct Ring {
    unsigned char *smem;
    unsigned long long *full;
    uint32_t stages;
    uint32_t loading, using_;      // next stage to fill and to read
    uint32_t phases, pending;      // bit s: parity to wait for at stage s; loads not yet waited for

    __device__ __forceinline__ void move(unsigned char *to, uint32_t depth) { smem = to; stages = depth; loading = using_ = 0; }
    __device__ __forceinline__ uint32_t take() {
        const uint32_t s = loading;
        loading = s + 1 == stages ? 0 : s + 1;
        ++pending;
        return s;
    }
    __device__ __forceinline__ uint32_t parity() const { return phases >> using_ & 1u; }
    __device__ __forceinline__ uint32_t give() {
        const uint32_t s = using_;
        phases ^= 1u << s;
        using_ = s + 1 == stages ? 0 : s + 1;
        --pending;
        return s;
    }
};

// What a unit covers: 16 rows of an entry for one key head, blocks [first, last) counted from its position `from`.
struct Unit {
    int entry, head, r0, rows, from, first, last;
    int slot;                  // partial result, -1: the output itself
};

template <class T, int kDim, int NT>
__device__ __forceinline__ void run_unit(const CacheView &c, const AttnArgs &a, const CUtensorMap *map_k, const CUtensorMap *map_v,
                                         AttnShared *sh, Ctl *ctl, Ring &ring, const Unit &w) {
    constexpr uint32_t kStage = unit_stage_bytes<kDim>(), kHalf = kStage / 2;
    constexpr int kSteps = kDim / 16;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const SeqPlan p = sh->plan[w.entry];
    const int head = w.head, rows = w.rows, r0 = w.r0;
    // A row sees positions below its limit; the last row's limit is the largest.
    const int most = p.len - p.t + (r0 + rows - 1) / (int)a.group + 1, least = p.len - p.t + r0 / (int)a.group + 1;
    const int first_block = w.first, last_block = min(w.last, (max(most - w.from, 0) + kBlock - 1) / kBlock);

    // Queries as B fragments: (dims 2t, 2t+1 and +8 of step ks) x (row g).
    uint32_t qf[NT][kSteps][2];
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = nt * 8 + g;
        const bool real = row < rows;
        const int tok = real ? (r0 + row) / (int)a.group : 0, sub = real ? (r0 + row) % (int)a.group : 0;
        const uint32_t *src = reinterpret_cast<const uint32_t *>(static_cast<const T *>(a.q) + (size_t)(p.row0 + tok) * a.q_stride
                                                                 + (size_t)(head * (int)a.group + sub) * kDim);
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
            qf[nt][ks][0] = real ? __ldg(src + ks * 8 + t) : 0u;
            qf[nt][ks][1] = real ? __ldg(src + ks * 8 + t + 4) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + 2 * t + e;
            limit[nt][e] = r < rows ? p.len - p.t + (r0 + r) / (int)a.group + 1 : 0;
        }
    }
    float o[NT][kSteps][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][k][e] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
    }

    // Page ids of 32 blocks at a time, one per lane; -1 where there is none.
    const int32_t *row_table = c.table + (size_t)p.seq * c.width;
    auto page_ids = [&](int base) {
        const int b = base + lane;
        int id = -1;
        if (b < last_block) {
            id = row_table[(w.from + b * kBlock) >> c.page_shift];
            if (id < 0 || (uint32_t)id >= c.pages) id = -1;
        }
        return id;
    };
    int load_base = first_block, load_ids = page_ids(load_base), next_load = first_block;
    int use_base = first_block, use_ids = load_ids;
    auto issue = [&]() {                                              // asks for the next block that exists
        while (next_load < last_block) {
            if (next_load - load_base >= 32) { load_base += 32; load_ids = page_ids(load_base); }
            const int id = __shfl_sync(0xffffffffu, load_ids, next_load - load_base);
            const int b = next_load++;
            if (id < 0) continue;
            const uint32_t s = ring.take();
            if (lane == 0) {
                unsigned char *dst = ring.smem + s * kStage;
                mbar_arrive_expect_tx(&ring.full[s], kStage);
                const int y = head * (int)c.page + ((w.from + b * kBlock) & (int)(c.page - 1)), z = (int)(a.layer * c.pages) + id;
#pragma unroll
                for (int x = 0; x < kDim; x += 64) {
                    tma_load_3d(dst + x * 2 * kBlock, map_k, &ring.full[s], x, y, z);
                    tma_load_3d(dst + kHalf + x * 2 * kBlock, map_v, &ring.full[s], x, y, z);
                }
            }
            return;
        }
    };
    for (uint32_t s = 0; s < ring.stages; ++s) issue();

    bool ok = true;
    for (int b = first_block; b < last_block; ++b) {
        if (b - use_base >= 32) { use_base += 32; use_ids = page_ids(use_base); }
        if (__shfl_sync(0xffffffffu, use_ids, b - use_base) < 0) continue;
        ok = __all_sync(0xffffffffu, wait_bar(&ring.full[ring.using_], ring.parity(), sh, ctl, kErrAttnLoad));
        if (!ok) break;
        const uint32_t s = ring.give();
        unsigned char *stage = ring.smem + s * kStage;
        const uint32_t ka = smem_u32(stage), va = ka + kHalf;
        const int pos0 = w.from + b * kBlock;
        bool selects = false;
        if (pos0 + kBlock > p.len) {                                   // values behind the end: anything, made zero
            for (int i = lane; i < kBlock * (kDim / 8); i += 32) {
                const uint32_t tok = i / (kDim / 8);
                if (pos0 + (int)tok >= p.len) *reinterpret_cast<uint4 *>(stage + kHalf + swz(tok, i % (kDim / 8), kBlock)) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        }
        if (pos0 + kBlock > least) {                                   // some row does not see some position of the block
            bool odd = false;
            for (int i = lane; i < kBlock * (kDim / 8); i += 32) {
                const uint32_t tok = i / (kDim / 8);
                if (pos0 + (int)tok < least) continue;
                const uint4 x = *reinterpret_cast<const uint4 *>(stage + kHalf + swz(tok, i % (kDim / 8), kBlock));
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    odd |= (w[k] & Elem<T>::kInfBits) == Elem<T>::kInfBits || (w[k] >> 16 & Elem<T>::kInfBits) == Elem<T>::kInfBits;
            }
            selects = __any_sync(0xffffffffu, odd);
        }

        float st[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) st[nt][0] = st[nt][1] = st[nt][2] = st[nt][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
            uint32_t kf[4];
            ldsm4(ka + swz((lane & 7) + (lane & 8), 2 * ks + (lane >> 4), kBlock), kf);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) Elem<T>::mma(st[nt], kf, qf[nt][ks][0], qf[nt][ks][1]);
        }
        uint32_t pf[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                // positions g and g + 8 of row 2t + e
                float lo = st[nt][e] * a.scale_log2, hi = st[nt][2 + e] * a.scale_log2;
                if (pos0 + g >= limit[nt][e]) lo = -INFINITY;
                if (pos0 + g + 8 >= limit[nt][e]) hi = -INFINITY;
                float top = fmaxf(lo, hi);
                // fmaxf passes NaN over, ex2 does not: a row that sees a NaN score becomes NaN, as it should.
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float now = fmaxf(m[nt][e], top), base = now == -INFINITY ? 0.f : now;
                const float down = ex2(m[nt][e] - base);
                m[nt][e] = now;
                lo = ex2(lo - base);
                hi = ex2(hi - base);
                l[nt][e] = fmaf(l[nt][e], down, lo + hi);
                st[nt][e] = lo;
                st[nt][2 + e] = hi;
                if (__any_sync(0xffffffffu, down != 1.f)) {
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) { o[nt][k][e] *= down; o[nt][k][2 + e] *= down; }
                }
            }
            pf[nt][0] = transpose8(Elem<T>::pack(st[nt][0], st[nt][1]));
            pf[nt][1] = transpose8(Elem<T>::pack(st[nt][2], st[nt][3]));
        }
        if (!selects) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t vf[4];
                ldsm4_t(va + swz((lane & 7) + (lane >> 4) * 8, 2 * k + ((lane >> 3) & 1), kBlock), vf);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) Elem<T>::mma(o[nt][k], vf, pf[nt][0], pf[nt][1]);
            }
        } else {
#pragma unroll 1
            for (int j = 0; j < kBlock; ++j) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float pj = __shfl_sync(0xffffffffu, j < 8 ? st[nt][e] : st[nt][2 + e], (j & 7) * 4 + t);
                        if (pos0 + j >= limit[nt][e]) continue;
#pragma unroll
                        for (int k = 0; k < kSteps; ++k)
#pragma unroll
                            for (int up = 0; up < 2; ++up) {
                                const uint32_t d = k * 16 + up * 8 + g;
                                const float v = Elem<T>::get(*reinterpret_cast<const uint16_t *>(stage + kHalf + swz(j, d >> 3, kBlock) + (d & 7) * 2));
                                o[nt][k][2 * up + e] = fmaf(pj, v, o[nt][k][2 * up + e]);
                            }
                    }
            }
        }
        __syncwarp();                                                  // the stage has been read
        issue();
    }
    if (!ok) return;

#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);

    if (w.slot < 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = nt * 8 + 2 * t + e;
                if (r >= rows) continue;
                const float inv = l[nt][e] == 0.f ? 0.f : 1.f / l[nt][e];
                T *dst = static_cast<T *>(a.out) + (size_t)(p.row0 + (r0 + r) / (int)a.group) * a.out_stride
                         + (size_t)(head * (int)a.group + (r0 + r) % (int)a.group) * kDim + g;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    dst[k * 16] = Elem<T>::put(o[nt][k][e] * inv);
                    dst[k * 16 + 8] = Elem<T>::put(o[nt][k][2 + e] * inv);
                }
            }
        return;
    }
    const size_t slot = (size_t)w.slot;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + 2 * t + e;
            if (r >= rows) continue;
            float *dst = a.part + (slot * kUnitRows + r) * kDim + g;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                __stcg(dst + k * 16, o[nt][k][e]);
                __stcg(dst + k * 16 + 8, o[nt][k][2 + e]);
            }
            if (g == 0) __stcg(a.part_ml + slot * kUnitRows + r, make_float2(m[nt][e], l[nt][e]));
        }
}

// The unit that ticket `ticket` stands for.
template <class T, int kDim>
__device__ __forceinline__ void unit_ticket(const CacheView &c, const AttnArgs &a, const CUtensorMap *map_k, const CUtensorMap *map_v,
                                            AttnShared *sh, Ctl *ctl, Ring &ring, int ticket) {
    int lo = 0, hi = (int)a.n - 1;                         // the last sequence with at most this many units before it
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sh->unit0[mid] <= ticket) lo = mid; else hi = mid - 1;
    }
    const SeqPlan p = sh->plan[lo];
    const int runs = runs_of(sh, a.group, lo), groups = row_groups(rows_of(p, a.group)), local = ticket - sh->unit0[lo], run = local % runs;
    Unit w;
    w.entry = lo;
    w.head = local / (runs * groups);
    w.r0 = local / runs % groups * kUnitRows;
    w.rows = (int)min(rows_of(p, a.group) - w.r0, (long long)kUnitRows);
    w.from = own_from(sh, lo);
    const int blocks = (p.len - w.from + kBlock - 1) / kBlock, each = (blocks + runs - 1) / runs;      // equally long
    w.first = run * each;
    w.last = min(w.first + each, blocks);
    w.slot = sh->part0[lo] < 0 ? -1 : sh->part0[lo] + local;
    if (w.rows > 8) run_unit<T, kDim, 2>(c, a, map_k, map_v, sh, ctl, ring, w);
    else run_unit<T, kDim, 1>(c, a, map_k, map_v, sh, ctl, ring, w);
    if (w.slot >= 0) {
        __threadfence();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) atomicAdd(&a.counters[(size_t)lo * c.heads + w.head], 1u);
    }
}

// ---- a merge ---------------------------------------------------------------------------------------------------
// Waits until `want` results are there; the whole warp.
__device__ __forceinline__ bool wait_count(const uint32_t *counter, uint32_t want, AttnShared *sh, Ctl *ctl) {
    if (ld_acquire(counter) >= want) return true;
    const unsigned long long t0 = global_ns();
    bool out = false;
    while (ld_acquire(counter) < want) {
        __nanosleep(64);
        if (*(volatile uint32_t *)&sh->abort != 0u || global_ns() - t0 > kWaitLimitNs) { out = true; break; }
    }
    if (!__any_sync(0xffffffffu, out)) return true;
    raise_error(ctl, kErrAttnMerge);
    *(volatile uint32_t *)&sh->abort = 1u;
    return false;
}

template <class T, int kDim>
__device__ __forceinline__ void run_merge(const CacheView &c, const AttnArgs &a, AttnShared *sh, Ctl *ctl, int merge) {
    constexpr int kVec = kDim / 32;
    const int lane = threadIdx.x & 31;
    const uint32_t out_rows = a.rows * a.q_heads;
    const uint32_t from = (uint32_t)merge * sh->merge_rows, to = min(from + (uint32_t)sh->merge_rows, out_rows);
    int entry = -1, head_seen = -1, runs = 0;
    for (uint32_t row = from; row < to; ++row) {
        const int tok = (int)(row / a.q_heads), qh = (int)(row % a.q_heads);
        if (entry < 0 || tok < sh->plan[entry].row0 || tok >= sh->plan[entry].row0 + sh->plan[entry].t) {
            int lo = -1, hi = (int)a.n;                               // the last entry that starts at or before the row
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (sh->plan[mid].row0 <= tok) lo = mid; else hi = mid;
            }
            entry = lo;
            head_seen = -1;
            if (entry < 0 || tok >= sh->plan[entry].row0 + sh->plan[entry].t) { entry = -1; continue; }
        }
        const SeqPlan p = sh->plan[entry];
        if (p.seq < 0 || sh->part0[entry] < 0) continue;
        const int head = qh / (int)a.group, r = (tok - p.row0) * (int)a.group + qh % (int)a.group;
        const bool with = shares(sh, entry);
        const int groups = row_groups(rows_of(p, a.group));
        if (head != head_seen) {
            runs = runs_of(sh, a.group, entry);
            if (!wait_count(&a.counters[(size_t)entry * c.heads + head], (uint32_t)(runs * groups), sh, ctl)) return;
            if (with && !wait_count(&a.counters[(size_t)a.n * c.heads + head], (uint32_t)(row_groups(sh->pre_rows) * pre_runs(sh)), sh, ctl)) return;
            head_seen = head;
        }
        // Results of the row, the prefix's runs first: slots at a step of one from two places.
        const int np = with ? pre_runs(sh) : 0, cr = sh->pre0[entry] + r;
        const size_t slot_p = with ? (size_t)sh->pre_part0 + ((size_t)head * row_groups(sh->pre_rows) + cr / kUnitRows) * np : 0;
        const size_t slot_o = (size_t)sh->part0[entry] + ((size_t)head * groups + r / kUnitRows) * runs;
        const size_t in_p = (size_t)(cr % kUnitRows), in_o = (size_t)(r % kUnitRows);
        const int all = np + runs;
        auto at = [&](int i) { return i < np ? (slot_p + i) * kUnitRows + in_p : (slot_o + (i - np)) * kUnitRows + in_o; };
        // Lane l keeps the maximum and sum of result l: most rows have no more than 32.
        float2 first = make_float2(-INFINITY, 0.f);
        if (lane < all) first = __ldcg(&a.part_ml[at(lane)]);
        float top = first.x;
        for (int i = lane + 32; i < all; i += 32) top = fmaxf(top, __ldcg(&a.part_ml[at(i)]).x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float base = top == -INFINITY ? 0.f : top;
        float acc[kVec], sum = 0.f;
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] = 0.f;
        for (int b = 0; b < all; b += 32) {
            float2 ml = first;
            if (b > 0) ml = b + lane < all ? __ldcg(&a.part_ml[at(b + lane)]) : make_float2(-INFINITY, 0.f);
            // A run in which the row saw nothing may have left its sum unwritten: it is passed over (weight -1).
            const float w = ml.x == -INFINITY && ml.y == 0.f ? -1.f : ex2(ml.x - base);
            if (!(w < 0.f)) sum = fmaf(w, ml.y, sum);
            const int here = min(32, all - b);
            // Sixteen results in flight: one after another they would cost an L2 round trip each.
            for (int i0 = 0; i0 < here; i0 += 16) {
                float x[16][kVec], wi[16];
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    const int i = min(i0 + u, 31);
                    wi[u] = __shfl_sync(0xffffffffu, w, i);
                    const bool real = i0 + u < here && !(wi[u] < 0.f);
                    if (!real) wi[u] = 0.f;
                    const float *src = a.part + at(real ? b + i : 0) * kDim + lane * kVec;
                    if constexpr (kVec == 4) {
                        const float4 y = real ? __ldcg(reinterpret_cast<const float4 *>(src)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        x[u][0] = y.x; x[u][1] = y.y; x[u][2] = y.z; x[u][3] = y.w;
                    } else {
                        const float2 y = real ? __ldcg(reinterpret_cast<const float2 *>(src)) : make_float2(0.f, 0.f);
                        x[u][0] = y.x; x[u][1] = y.y;
                    }
                }
#pragma unroll
                for (int u = 0; u < 16; ++u)
#pragma unroll
                    for (int v = 0; v < kVec; ++v) acc[v] = fmaf(wi[u], x[u][v], acc[v]);
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<T *>(a.out) + (size_t)tok * a.out_stride + (size_t)qh * kDim + lane * kVec);
#pragma unroll
        for (int v = 0; v < kVec; v += 2) dst[v / 2] = Elem<T>::pack(acc[v] * inv, acc[v + 1] * inv);
    }
}

} // namespace xpk
