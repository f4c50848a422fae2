// Attention over the paged key/value cache for single tokens, drafts and prompts.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp2(scale log2(e) (q . k_j - max)),   j below the row's limit
//
// A sequence's queries times the G = q_heads / kv_heads query heads that read one key head are its rows for that head
// (row r = query r / G, head r % G): they read the same keys, so a group of rows shares one pass over them.
//
// Work is cut into tickets that warps claim one at a time (pk_common.cuh), in this order:
//   units   (sequence, key head, 16 rows, a run of 16-position blocks): one warp streams the run's keys and values;
//   merges  a few output rows each, for sequences cut into several runs: weighted sum of the runs' results.
// The cut is a function of the lengths and the device's SM count alone, and a merge adds the runs in their order, so the
// result does not depend on which warp computed what, or on preemption.  A merge ticket waits (bounded) for the units it
// reads; those have smaller numbers, so they are already claimed by running warps.
//
// A unit is HBM-bound: 2 * 16 * head_dim * 2 bytes per block for 4 * 16 * 16 * head_dim flop.  Each warp has a ring of
// blocks of its own in shared memory, filled by TMA (128-byte swizzle) ahead of use.  Scores are computed transposed,
// S^T = K Q^T with mma.m16n8k16 (positions are M, 8 rows are N), so that up to 8 rows cost one MMA column block, and
// O^T = V^T P^T; the C fragment of S^T becomes the B fragment of P^T by transposing its 8x8 quarters (movmatrix).
//
// Positions that a row must not see may hold anything: scores are replaced before the maximum, values at or behind the
// sequence's end are zeroed in shared memory (0 * NaN), and a block whose hidden values are not finite is added with
// selects instead of MMAs.
#include "gemm_ptx.cuh"
#include "kv_cache.cuh"
#include <cuda_fp16.h>

namespace xpk {

constexpr int kAttnWarps = 8;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kBlock = 16;                                  // positions per block of a unit
constexpr int kUnitRows = 16;
constexpr int kUnitStages = 3;
constexpr int kMinRun = 4;                                  // blocks: a run shorter than 64 positions costs more to merge than it spreads
constexpr int kMergeRowsMost = 32;
constexpr uint32_t kErrAttnLoad  = 0x70000001u;
constexpr uint32_t kErrAttnMerge = 0x70000002u;

struct AttnArgs {
    const void *q;
    void *out;
    unsigned long long q_stride, out_stride;
    const int32_t *seqs, *starts;
    float scale_log2;
    uint32_t n, rows, q_heads, group, layer;
    uint32_t sms;                                           // of the device, whatever the grid: the cut depends on it
    float *part;                                            // [part_units][16][head_dim]
    float2 *part_ml;                                        // [part_units][16] maximum (log2 units), sum
    uint32_t *counters;                                     // [n][kv_heads] units done; zero between calls
};

struct SeqPlan {
    int row0, t, len, seq;                                  // first row, rows, positions held; seq < 0: nothing to do
};

struct AttnShared {
    SeqPlan plan[XPK_ATTENTION_MAX_SEQS];
    int unit0[XPK_ATTENTION_MAX_SEQS + 1];                  // first unit ticket of each sequence
    int part0[XPK_ATTENTION_MAX_SEQS];                      // its first partial result, -1: written directly
    unsigned long long full[kAttnWarps][kUnitStages];
    unsigned long long red[kAttnWarps];
    unsigned long long done;
    int run;                                                // blocks per run
    int units, merges, merge_rows;
    uint32_t abort, stop, last;
};

template <class T, int kDim> __host__ __device__ constexpr uint32_t stage_bytes() { return 2 * kBlock * kDim * 2; }
template <class T, int kDim> __host__ __device__ constexpr size_t attn_smem() {
    return 1024 + (size_t)kAttnWarps * kUnitStages * stage_bytes<T, kDim>() + sizeof(AttnShared);
}

// ---- instructions ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, void *bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%3, %4, %5}], [%2];"
                 :: "r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t ld_acquire(const uint32_t *p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

template <class T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
    static constexpr uint32_t kInfBits = 0x7f80u;           // exponent of infinities and NaN
    static __device__ __forceinline__ uint32_t pack(float a, float b) { __nv_bfloat162 y = __floats2bfloat162_rn(a, b); return *reinterpret_cast<uint32_t *>(&y); }
    static __device__ __forceinline__ float get(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Elem<__half> {
    static constexpr uint32_t kInfBits = 0x7c00u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) { __half2 y = __floats2half2_rn(a, b); return *reinterpret_cast<uint32_t *>(&y); }
    static __device__ __forceinline__ float get(uint16_t x) { return __half2float(*reinterpret_cast<__half *>(&x)); }
    static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// Byte offset of the 16-byte chunk `chunk` (8 elements) of row `row` in a box of `rows` x kDim elements: two (one) boxes of
// 64 elements behind one another, 128-byte swizzle.
__device__ __forceinline__ uint32_t swz(uint32_t row, uint32_t chunk, uint32_t rows) {
    return (chunk >> 3) * rows * 128u + row * 128u + ((chunk ^ row) & 7u) * 16u;
}

__device__ __forceinline__ int unit_blocks(const SeqPlan &p) { return (p.len + kBlock - 1) / kBlock; }
__device__ __forceinline__ int unit_groups(const SeqPlan &p, uint32_t group) { return (int)(((long long)p.t * group + kUnitRows - 1) / kUnitRows); }
__device__ __forceinline__ int runs_of(const SeqPlan &p, int run) { return max(1, (unit_blocks(p) + run - 1) / run); }

// ---- the cut ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, AttnShared *sh) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh->red[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long s = 0;
    for (int w = 0; w < kAttnWarps; ++w) s += sh->red[w];
    return s;
}

// Every CTA works the same cut out of the same arrays.
__device__ __forceinline__ void make_plan(const CacheView &c, const AttnArgs &a, AttnShared *sh) {
    for (uint32_t i = threadIdx.x; i < a.n; i += kAttnThreads) {
        SeqPlan p;
        p.seq = a.seqs ? a.seqs[i] : (int)i;
        p.row0 = a.starts ? min(max(a.starts[i], 0), (int)a.rows) : (int)i;
        p.t = a.starts ? max(min(a.starts[i + 1], (int)a.rows) - p.row0, 0) : ((uint32_t)i < a.rows ? 1 : 0);
        p.len = held_by(c, p.seq);
        if (p.len < 0 || p.t == 0) p.seq = -1;
        sh->plan[i] = p;
    }
    __syncthreads();
    unsigned long long work = 0;
    for (uint32_t i = threadIdx.x; i < a.n; i += kAttnThreads) {
        const SeqPlan p = sh->plan[i];
        if (p.seq >= 0) work += (unsigned long long)unit_blocks(p) * unit_groups(p, a.group) * c.heads;
    }
    work = block_sum(work, sh);
    const unsigned long long target = (unsigned long long)a.sms * kAttnWarps * 2;
    const int run = max(kMinRun, (int)min((work + target - 1) / target, 0x7fffffffull / kBlock));
    // First tickets and first partial results: a running sum over the sequences, 32 at a time, by the first warp.
    if (threadIdx.x < 32) {
        int units = 0, parts = 0;
        for (uint32_t base = 0; base < a.n; base += 32) {
            const uint32_t i = base + threadIdx.x;
            int u = 0, r = 0;
            if (i < a.n && sh->plan[i].seq >= 0) {
                const SeqPlan p = sh->plan[i];
                const int runs = runs_of(p, run);
                u = unit_groups(p, a.group) * (int)c.heads * runs;
                r = runs > 1 ? u : 0;
            }
            int us = u, rs = r;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, us, d), y = __shfl_up_sync(0xffffffffu, rs, d);
                if ((int)threadIdx.x >= d) { us += x; rs += y; }
            }
            if (i < a.n) {
                sh->unit0[i] = units + us - u;
                sh->part0[i] = r > 0 ? parts + rs - r : -1;
            }
            units += __shfl_sync(0xffffffffu, us, 31);
            parts += __shfl_sync(0xffffffffu, rs, 31);
        }
        if (threadIdx.x == 0) {
            sh->unit0[a.n] = units;
            sh->run = run;
            sh->units = units;
            const uint32_t out_rows = a.rows * a.q_heads;
            int per = 1;
            while (per < kMergeRowsMost && (unsigned long long)per * a.sms * kAttnWarps < out_rows) per *= 2;
            sh->merge_rows = per;
            sh->merges = parts > 0 ? (int)((out_rows + per - 1) / per) : 0;
        }
    }
    __syncthreads();
}

// ---- a unit ----------------------------------------------------------------------------------------------------
template <class Quit>
__device__ __forceinline__ bool wait_full(void *bar, uint32_t parity, AttnShared *sh, Ctl *ctl, Quit quit) {
    uint32_t it = 0;
    unsigned long long t0 = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++it & 0xFFu) == 0) {
            if (quit()) return false;
            const unsigned long long now = global_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > kWaitLimitNs) {
                raise_error(ctl, kErrAttnLoad);
                *(volatile uint32_t *)&sh->abort = 1u;
                return false;
            }
        }
    }
    return true;
}

struct Ring {                 // one warp's ring of blocks
    unsigned char *smem;
    unsigned long long *full;
    uint32_t loaded, used;    // blocks asked for and consumed since the kernel began
};

template <class T, int kDim, int NT>
__device__ __forceinline__ void run_unit(const CacheView &c, const AttnArgs &a, const CUtensorMap *map_k, const CUtensorMap *map_v,
                                         AttnShared *sh, Ctl *ctl, Ring &ring, int entry, int unit) {
    constexpr uint32_t kStage = stage_bytes<T, kDim>(), kHalf = kStage / 2;
    constexpr int kSteps = kDim / 16;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const SeqPlan p = sh->plan[entry];
    const int runs = runs_of(p, sh->run), groups = unit_groups(p, a.group);
    const int local = unit - sh->unit0[entry];
    const int run = local % runs, rg = (local / runs) % groups, head = local / (runs * groups);
    const int rows = (int)min((long long)p.t * a.group - (long long)rg * kUnitRows, (long long)kUnitRows);
    const int r0 = rg * kUnitRows;                                    // first row of the group, counted in its sequence
    const int first_block = run * sh->run;
    // A row sees positions below its limit; the last row's limit is the largest.
    const int most = p.len - p.t + (r0 + rows - 1) / (int)a.group + 1, least = p.len - p.t + r0 / (int)a.group + 1;
    const int last_block = min(min(first_block + sh->run, unit_blocks(p)), (max(most, 0) + kBlock - 1) / kBlock);

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
            id = row_table[(b * kBlock) >> c.page_shift];
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
            if (lane == 0) {
                const uint32_t s = ring.loaded % kUnitStages;
                unsigned char *dst = ring.smem + s * kStage;
                mbar_arrive_expect_tx(&ring.full[s], kStage);
                const int y = head * (int)c.page + ((b * kBlock) & (int)(c.page - 1)), z = (int)(a.layer * c.pages) + id;
#pragma unroll
                for (int x = 0; x < kDim; x += 64) {
                    tma_load_3d(dst + x * 2 * kBlock, map_k, &ring.full[s], x, y, z);
                    tma_load_3d(dst + kHalf + x * 2 * kBlock, map_v, &ring.full[s], x, y, z);
                }
            }
            ++ring.loaded;
            return;
        }
    };
    for (int s = 0; s < kUnitStages; ++s) issue();

    bool ok = true;
    for (int b = first_block; b < last_block; ++b) {
        if (b - use_base >= 32) { use_base += 32; use_ids = page_ids(use_base); }
        if (__shfl_sync(0xffffffffu, use_ids, b - use_base) < 0) continue;
        const uint32_t s = ring.used % kUnitStages, phase = (ring.used / kUnitStages) & 1u;
        ok = __all_sync(0xffffffffu, wait_full(&ring.full[s], phase, sh, ctl, [&] { return *(volatile uint32_t *)&sh->abort != 0u; }));
        if (!ok) break;
        ++ring.used;
        unsigned char *stage = ring.smem + s * kStage;
        const uint32_t ka = smem_u32(stage), va = ka + kHalf;
        const int pos0 = b * kBlock;
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

    if (sh->part0[entry] < 0) {
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
    const size_t slot = (size_t)(sh->part0[entry] + local);
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
    __threadfence();
    __syncwarp();
    if (lane == 0) atomicAdd(&a.counters[(size_t)entry * c.heads + head], 1u);
}

// ---- a merge ---------------------------------------------------------------------------------------------------
template <class T, int kDim>
__device__ __forceinline__ void run_merge(const CacheView &c, const AttnArgs &a, AttnShared *sh, Ctl *ctl, int merge) {
    constexpr int kVec = kDim / 32;
    const int lane = threadIdx.x & 31;
    const uint32_t out_rows = a.rows * a.q_heads;
    const uint32_t from = (uint32_t)merge * sh->merge_rows, to = min(from + (uint32_t)sh->merge_rows, out_rows);
    int entry = -1;
    for (uint32_t row = from; row < to; ++row) {
        const int tok = (int)(row / a.q_heads), qh = (int)(row % a.q_heads);
        if (entry < 0 || tok < sh->plan[entry].row0 || tok >= sh->plan[entry].row0 + sh->plan[entry].t) {
            int lo = -1, hi = (int)a.n;                               // the last entry that starts at or before the row
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (sh->plan[mid].row0 <= tok) lo = mid; else hi = mid;
            }
            entry = lo;
            if (entry < 0 || tok >= sh->plan[entry].row0 + sh->plan[entry].t) { entry = -1; continue; }
        }
        const SeqPlan p = sh->plan[entry];
        if (p.seq < 0 || sh->part0[entry] < 0) continue;
        const int head = qh / (int)a.group, r = (tok - p.row0) * (int)a.group + qh % (int)a.group;
        const int runs = runs_of(p, sh->run), groups = unit_groups(p, a.group);
        const uint32_t want = (uint32_t)(runs * groups);
        const uint32_t *counter = &a.counters[(size_t)entry * c.heads + head];
        if (ld_acquire(counter) < want) {
            const unsigned long long t0 = global_ns();
            bool out = false;
            while (ld_acquire(counter) < want) {
                __nanosleep(64);
                if (*(volatile uint32_t *)&sh->abort != 0u || global_ns() - t0 > kWaitLimitNs) { out = true; break; }
            }
            if (__any_sync(0xffffffffu, out)) {
                raise_error(ctl, kErrAttnMerge);
                *(volatile uint32_t *)&sh->abort = 1u;
                return;
            }
        }
        const size_t slot0 = (size_t)sh->part0[entry] + ((size_t)head * groups + r / kUnitRows) * runs;
        const size_t in = (size_t)(r % kUnitRows);
        float top = -INFINITY;
        for (int i = lane; i < runs; i += 32) top = fmaxf(top, __ldcg(&a.part_ml[(slot0 + i) * kUnitRows + in]).x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float base = top == -INFINITY ? 0.f : top;
        float acc[kVec], sum = 0.f;
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] = 0.f;
        for (int b = 0; b < runs; b += 32) {
            float2 ml = make_float2(-INFINITY, 0.f);
            if (b + lane < runs) ml = __ldcg(&a.part_ml[(slot0 + b + lane) * kUnitRows + in]);
            const float w = ex2(ml.x - base);
            sum = fmaf(w, ml.y, sum);
            const int here = min(32, runs - b);
#pragma unroll 4
            for (int i = 0; i < here; ++i) {
                const float wi = __shfl_sync(0xffffffffu, w, i);
                const float *src = a.part + ((slot0 + b + i) * kUnitRows + in) * kDim + lane * kVec;
                if constexpr (kVec == 4) {
                    const float4 x = __ldcg(reinterpret_cast<const float4 *>(src));
                    acc[0] = fmaf(wi, x.x, acc[0]); acc[1] = fmaf(wi, x.y, acc[1]);
                    acc[2] = fmaf(wi, x.z, acc[2]); acc[3] = fmaf(wi, x.w, acc[3]);
                } else {
                    const float2 x = __ldcg(reinterpret_cast<const float2 *>(src));
                    acc[0] = fmaf(wi, x.x, acc[0]); acc[1] = fmaf(wi, x.y, acc[1]);
                }
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

// ---- the tickets -----------------------------------------------------------------------------------------------
template <class T, int kDim, bool kPreemptible>
__device__ __forceinline__ void work_off(Ctl *ctl, const CUtensorMap *map_k, const CUtensorMap *map_v, const CacheView &c, const AttnArgs &a,
                                         AttnShared *sh, unsigned char *smem) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    make_plan(c, a, sh);
    // Never zero: a task that was stopped before any CTA got here must not look complete.
    const unsigned long long total = max((unsigned long long)sh->units + (unsigned long long)sh->merges, 1ull);
    if (threadIdx.x == 0) *(volatile unsigned long long *)&ctl->total = total;       // the same from every CTA
    ClaimCtx ctx;
    ctx.nret = 0;                                          // no ticket is ever handed back
    ctx.base = *(volatile unsigned long long *)&ctl->base;
    ctx.fresh = total - ctx.base;
    ctx.cur = 0;
    Ring ring{smem + (size_t)warp * kUnitStages * stage_bytes<T, kDim>(), sh->full[warp], 0u, 0u};
    unsigned long long done = 0;
    while (true) {
        unsigned long long ticket = kNoTile;
        if (lane == 0) {
            bool stop = *(volatile uint32_t *)&sh->abort != 0u;
            if constexpr (kPreemptible) stop = stop || ld_flag(ctl->flag) != 0;
            if (!stop) ticket = resolve_ticket(ctl, ctx, take_ticket(ctl));
        }
        ticket = __shfl_sync(0xffffffffu, ticket, 0);
        if (ticket == kNoTile) break;
        if (ticket < (unsigned long long)sh->units) {
            const int unit = (int)ticket;
            int lo = 0, hi = (int)a.n - 1;                 // the last sequence whose first unit is at most this one
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (sh->unit0[mid] <= unit) lo = mid; else hi = mid - 1;
            }
            const SeqPlan &p = sh->plan[lo];
            if ((long long)p.t * a.group > 8) run_unit<T, kDim, 2>(c, a, map_k, map_v, sh, ctl, ring, lo, unit);
            else run_unit<T, kDim, 1>(c, a, map_k, map_v, sh, ctl, ring, lo, unit);
        } else {
            run_merge<T, kDim>(c, a, sh, ctl, (int)(ticket - (unsigned long long)sh->units));
        }
        ++done;
    }
    // Loads that a unit gave up on still land in this CTA's shared memory: wait for them.
    for (; ring.used != ring.loaded; ++ring.used)
        wait_full(&ring.full[ring.used % kUnitStages], (ring.used / kUnitStages) & 1u, sh, ctl, [] { return false; });
    if (lane == 0 && done) atomicAdd(&sh->done, done);
}

// ---- the kernel ------------------------------------------------------------------------------------------------
template <class T, int kDim, bool kPreemptible>
__global__ void __launch_bounds__(kAttnThreads, 1)
attention_kernel(Ctl *ctl, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, CacheView c, AttnArgs a,
                 unsigned long long launch_no) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    AttnShared *sh = reinterpret_cast<AttnShared *>(smem + (size_t)kAttnWarps * kUnitStages * stage_bytes<T, kDim>());
    note_start(ctl);
    if (threadIdx.x == 0) {
        for (int w = 0; w < kAttnWarps; ++w)
            for (int s = 0; s < kUnitStages; ++s) mbar_init(&sh->full[w][s], 1);
        sh->done = 0;
        sh->abort = 0;
        // Queued behind a launch that is being stopped: no set-up.
        sh->stop = kPreemptible && ld_flag(ctl->flag) != 0 ? 1u : 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    if (sh->stop == 0u) work_off<T, kDim, kPreemptible>(ctl, &map_k, &map_v, c, a, sh, smem);
    __syncthreads();
    if (threadIdx.x == 0) sh->last = cta_leave(ctl, sh->done) ? 1u : 0u;
    __syncthreads();
    if (sh->last == 0u) return;
    // The last CTA leaves the counters ready for the next call once the work is complete.
    const bool task = ctl->mailbox != nullptr;
    const bool whole = *(volatile unsigned long long *)&ctl->tiles_done >= *(volatile unsigned long long *)&ctl->total;
    if (whole || !task)
        for (uint32_t i = threadIdx.x; i < a.n * c.heads; i += kAttnThreads) a.counters[i] = 0;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        cta_fold(ctl, launch_no);
        if (!task)                                         // a call without a task keeps nothing, not even an error
            for (unsigned i = 0; i < kCtlResetBytes / 8; ++i) reinterpret_cast<unsigned long long *>(ctl)[i] = 0;
    }
}

// ---- host side -------------------------------------------------------------------------------------------------
template <class T, int kDim>
static cudaError_t prepare_one() {
    cudaError_t e = cudaFuncSetAttribute(attention_kernel<T, kDim, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)attn_smem<T, kDim>());
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(attention_kernel<T, kDim, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)attn_smem<T, kDim>());
}
cudaError_t attention_prepare() {
    cudaError_t e = prepare_one<__nv_bfloat16, 128>();
    if (e == cudaSuccess) e = prepare_one<__nv_bfloat16, 64>();
    if (e == cudaSuccess) e = prepare_one<__half, 128>();
    if (e == cudaSuccess) e = prepare_one<__half, 64>();
    return e;
}

// Where things lie in a call's scratch.
struct AttnScratch {
    size_t ctl, counters, ml, part, bytes;
    uint32_t part_units;
};
AttnScratch attention_scratch(const CacheView &c, uint32_t sms, uint32_t rows, uint32_t n, uint32_t q_heads) {
    AttnScratch s;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    (void)rows;
    (void)q_heads;
    // Sequences of several runs have less than 2 work / run of them in all (the run is at least work / target).
    s.part_units = 2 * 2 * sms * kAttnWarps + 1;
    s.ctl = 0;
    s.counters = up(sizeof(Ctl));
    s.ml = s.counters + up((size_t)n * c.heads * 4);
    s.part = s.ml + up((size_t)s.part_units * kUnitRows * sizeof(float2));
    s.bytes = s.part + (size_t)s.part_units * kUnitRows * c.dim * sizeof(float);
    return s;
}
size_t attention_scratch_bytes(const CacheView &c, uint32_t sms, uint32_t rows, uint32_t n, uint32_t q_heads) {
    return attention_scratch(c, sms, rows, n, q_heads).bytes;
}
// What xpkTaskReset clears: the counters (the partial results need no clearing).
void attention_counters(const CacheView &c, uint32_t sms, const xpkAttentionArgs &x, void **at, size_t *bytes) {
    const AttnScratch s = attention_scratch(c, sms, x.rows, x.n, x.q_heads);
    *at = (unsigned char *)x.scratch + s.counters;
    *bytes = (size_t)x.n * c.heads * 4;
}

cudaError_t launch_attention(bool preemptible, Ctl *ctl, const xpkKvCache_st *cache, const xpkAttentionArgs &x, unsigned long long launch_no,
                             int grid, cudaStream_t st) {
    const CacheView c = view_of(cache);
    const AttnScratch s = attention_scratch(c, (uint32_t)cache->sms, x.rows, x.n, x.q_heads);
    unsigned char *scratch = (unsigned char *)x.scratch;
    AttnArgs a;
    a.q = x.q;
    a.out = x.out;
    a.q_stride = x.q_stride;
    a.out_stride = x.out_stride;
    a.seqs = x.seqs;
    a.starts = x.starts;
    a.scale_log2 = x.scale * 1.4426950408889634f;
    a.n = x.n;
    a.rows = x.rows;
    a.q_heads = x.q_heads;
    a.group = x.q_heads / c.heads;
    a.layer = x.layer;
    a.sms = (uint32_t)cache->sms;
    a.part = (float *)(scratch + s.part);
    a.part_ml = (float2 *)(scratch + s.ml);
    a.counters = (uint32_t *)(scratch + s.counters);
    if (ctl == nullptr) ctl = (Ctl *)(scratch + s.ctl);
    const CUtensorMap &mk = *(const CUtensorMap *)cache->map_k, &mv = *(const CUtensorMap *)cache->map_v;
    const bool bf16 = cache->d.dtype == XPK_DTYPE_BF16;
#define XPK_ATTN(T, D)                                                                                                              \
    do {                                                                                                                            \
        if (preemptible) attention_kernel<T, D, true><<<grid, kAttnThreads, attn_smem<T, D>(), st>>>(ctl, mk, mv, c, a, launch_no); \
        else attention_kernel<T, D, false><<<grid, kAttnThreads, attn_smem<T, D>(), st>>>(ctl, mk, mv, c, a, launch_no);            \
    } while (0)
    if (bf16 && c.dim == 128) XPK_ATTN(__nv_bfloat16, 128);
    else if (bf16) XPK_ATTN(__nv_bfloat16, 64);
    else if (c.dim == 128) XPK_ATTN(__half, 128);
    else XPK_ATTN(__half, 64);
#undef XPK_ATTN
    return cudaGetLastError();
}

} // namespace xpk
