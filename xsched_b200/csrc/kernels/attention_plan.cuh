// The cut of an attention call into tickets (see attention.cu): what each CTA works out at its start.
#pragma once
#include "gemm_ptx.cuh"
#include "kv_cache.cuh"
#include <cuda_fp16.h>

namespace xpk {

constexpr int kWorkers = 8;                                 // warps that run units and merges; two groups of four for tiles
constexpr int kAttnThreads = (kWorkers + 4) * 32;           // and a third group: one warp loads, one issues MMAs
// Registers: 384 threads are launched with 168 each; the workers, whose rows of scores fill 128, take over what the helpers
// do not need: 2 * 208 + 88 = 3 * 168.
constexpr int kWorkerRegs = 208, kHelperRegs = 88;
static_assert(2 * kWorkerRegs + kHelperRegs <= 3 * 168, "more registers than the launch has");
constexpr int kBlock = 16;                                  // positions per block of a unit
constexpr int kUnitRows = 16;                               // rows of a unit, and of a partial result
constexpr int kUnitStages = 3;
constexpr int kTile = 128;                                  // positions per tile; rows per group of a tile item
constexpr int kItemRows = 2 * kTile;
constexpr int kRing = 4;                                    // stages of the tile ring; a stage holds a tile of keys or of values
constexpr int kMinRun = 4;                                  // blocks: a run shorter than 64 positions costs more to merge than it spreads
constexpr int kMinTiles = 2;                                // tiles: one for each group of workers
constexpr int kShareRows = 64;                              // sequences of more rows fill tiles by themselves
constexpr int kMergeRowsMost = 32;
constexpr uint32_t kErrAttnLoad  = 0x70000001u;
constexpr uint32_t kErrAttnMerge = 0x70000002u;
constexpr uint32_t kErrAttnTile  = 0x70000003u;

struct AttnArgs {
    const void *q;
    void *out;
    unsigned long long q_stride, out_stride;
    const int32_t *seqs, *starts, *shared_len;
    float scale_log2;
    uint32_t n, rows, q_heads, group, layer;
    uint32_t sms;                                           // of the device, whatever the grid: the cut depends on it
    float *part;                                            // [part_slots][16][head_dim]
    float2 *part_ml;                                        // [part_slots][16] maximum (log2 units), sum
    uint32_t *counters;                                     // [n + 1][kv_heads] results there; the last row: the prefix; zero between calls
    uint32_t part_slots;
};

struct SeqPlan {
    int row0, t, len, seq;                                  // first row, rows, positions held; seq < 0: nothing to do
};

struct AttnShared {
    SeqPlan plan[XPK_ATTENTION_MAX_SEQS];
    int unit0[XPK_ATTENTION_MAX_SEQS];                      // units before each sequence's
    int tile0[XPK_ATTENTION_MAX_SEQS];                      // tile items before each sequence's (the prefix's come first)
    int part0[XPK_ATTENTION_MAX_SEQS];                      // its first partial result, -1: written directly
    int pre0[XPK_ATTENTION_MAX_SEQS];                       // rows of sharing sequences before it
    uint32_t share[XPK_ATTENTION_MAX_SEQS / 32];            // which sequences share
    // tile pipeline
    unsigned long long ring_full[kRing], ring_empty[kRing];
    unsigned long long q_full[2], s_full[2], p_full[2], o_full[2], drain;
    int ticket;
    uint32_t tmem, odd, stage_pages[kRing];
    // units
    unsigned long long full[kWorkers][kUnitStages];
    unsigned long long red[kAttnThreads / 32];
    unsigned long long done;
    int run, tile_run;                                      // blocks (tiles) per run
    int units, tiles, merges, merge_rows;
    int shared, shared_seq, pre_rows, pre_part0, pre_tiles; // prefix: positions, whose table, rows, first result, its tile items
    int tile_ctas;                                          // CTAs that begin with tiles
    uint32_t abort, stop, last;
};

template <int kDim> __host__ __device__ constexpr uint32_t unit_stage_bytes() { return 2 * kBlock * kDim * 2; }
template <int kDim> __host__ __device__ constexpr uint32_t tile_bytes() { return kTile * kDim * 2; }
template <int kDim> __host__ __device__ constexpr size_t ring_bytes() {
    const size_t tiles = (size_t)(2 + kRing) * tile_bytes<kDim>(), units = (size_t)kWorkers * kUnitStages * unit_stage_bytes<kDim>();
    return tiles > units ? tiles : units;
}
template <int kDim> __host__ __device__ constexpr size_t attn_smem() { return 1024 + ring_bytes<kDim>() + sizeof(AttnShared); }
static_assert(attn_smem<128>() <= 232448, "shared memory of one CTA");

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


// ---- shapes that follow from a sequence's plan ------------------------------------------------------------------
__device__ __forceinline__ bool shares(const AttnShared *sh, int i) { return sh->share[i >> 5] >> (i & 31) & 1u; }
// First position that a sequence's own runs cover.
__device__ __forceinline__ int own_from(const AttnShared *sh, int i) { return shares(sh, i) ? sh->shared : 0; }
__device__ __forceinline__ long long rows_of(const SeqPlan &p, uint32_t group) { return (long long)p.t * group; }
__device__ __forceinline__ bool by_tiles(const SeqPlan &p, uint32_t group) { return rows_of(p, group) > kUnitRows; }
__device__ __forceinline__ int row_groups(long long rows) { return (int)((rows + kUnitRows - 1) / kUnitRows); }
__device__ __forceinline__ int row_tiles(long long rows) { return (int)((rows + kItemRows - 1) / kItemRows); }
// With at most 128 rows the two groups of workers take half of a run's tiles each, and leave a result each.
__device__ __forceinline__ int halves(long long rows) { return rows <= kTile ? 2 : 1; }
__device__ __forceinline__ int chunks(int positions, int each, int run) { return max(1, ((positions + each - 1) / each + run - 1) / run); }
__device__ __forceinline__ int tile_runs(const AttnShared *sh, int positions) { return chunks(positions, kTile, sh->tile_run); }
// Results that are left for each row by a sequence's own runs, and by the prefix.
__device__ __forceinline__ int runs_of(const AttnShared *sh, uint32_t group, int i) {
    const SeqPlan &p = sh->plan[i];
    const int own = p.len - own_from(sh, i);
    return by_tiles(p, group) ? tile_runs(sh, own) * halves(rows_of(p, group)) : chunks(own, kBlock, sh->run);
}
__device__ __forceinline__ int pre_runs(const AttnShared *sh) { return tile_runs(sh, sh->shared) * halves(sh->pre_rows); }

// ---- the cut ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, AttnShared *sh) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh->red[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long s = 0;
    for (int w = 0; w < kAttnThreads / 32; ++w) s += sh->red[w];
    return s;
}

// Every CTA works the same cut out of the same arrays.
__device__ __forceinline__ void make_plan(const CacheView &c, const AttnArgs &a, AttnShared *sh) {
    const uint32_t tid = threadIdx.x;
    int shared = a.shared_len ? max(*a.shared_len, 0) & ~(int)(c.page - 1) : 0;
    unsigned long long sharing = 0;
    for (uint32_t base = 0; base < a.n; base += kAttnThreads) {              // whole warps: ballots below
        const uint32_t i = base + tid;
        bool with = false;
        if (i < a.n) {
            SeqPlan p;
            p.seq = a.seqs ? a.seqs[i] : (int)i;
            p.row0 = a.starts ? min(max(a.starts[i], 0), (int)a.rows) : (int)i;
            p.t = a.starts ? max(min(a.starts[i + 1], (int)a.rows) - p.row0, 0) : (i < a.rows ? 1 : 0);
            p.len = held_by(c, p.seq);
            if (p.len < 0 || p.t == 0) p.seq = -1;
            sh->plan[i] = p;
            with = shared > 0 && p.seq >= 0 && rows_of(p, a.group) <= kShareRows && p.len - p.t >= shared;
        }
        const uint32_t bits = __ballot_sync(0xffffffffu, with);
        if ((tid & 31) == 0 && i < XPK_ATTENTION_MAX_SEQS) sh->share[i >> 5] = bits;
        sharing += with;
    }
    sharing = block_sum(sharing, sh);
    if (sharing < 2) shared = 0;
    // A second round without the prefix if its results do not fit the scratch.
    for (int round = 0; round < 2; ++round) {
        if (shared == 0)
            for (uint32_t i = tid; i < XPK_ATTENTION_MAX_SEQS / 32; i += kAttnThreads) sh->share[i] = 0;
        if (tid == 0) sh->shared = shared;
        __syncthreads();
        unsigned long long blocks = 0, tiles = 0, rows = 0;
        for (uint32_t i = tid; i < a.n; i += kAttnThreads) {
            const SeqPlan p = sh->plan[i];
            if (p.seq < 0) continue;
            const int own = p.len - own_from(sh, i);
            if (by_tiles(p, a.group)) tiles += (unsigned long long)((own + kTile - 1) / kTile) * row_tiles(rows_of(p, a.group)) * c.heads;
            else blocks += (unsigned long long)((own + kBlock - 1) / kBlock) * c.heads;
            if (shares(sh, i)) rows += (unsigned long long)rows_of(p, a.group);
        }
        blocks = block_sum(blocks, sh);
        tiles = block_sum(tiles, sh);
        rows = block_sum(rows, sh);
        tiles += (unsigned long long)((shared + kTile - 1) / kTile) * row_tiles(rows) * c.heads;
        if (tid == 0) {
            const unsigned long long target = (unsigned long long)a.sms * kWorkers * 2;
            sh->run = max(kMinRun, (int)min((blocks + target - 1) / target, 0x7fffffffull / kBlock));
            sh->tile_run = max(kMinTiles, (int)min((tiles + a.sms - 1) / a.sms, 0x7fffffffull / kTile));
            sh->pre_rows = (int)rows;
            // CTAs are dealt to tiles and units by the time each kind takes: a tile of 256 rows about 1.3 us of an SM, a block
            // 64 bytes an element over the SM's share of HBM (44 GB/s): 0.19 us at 128.
            const float tile_us = 1.3f * (float)tiles, block_us = 0.0015f * (float)c.dim * (float)blocks;
            sh->tile_ctas = tiles == 0 ? 0 : blocks == 0 ? 0x7fffffff : max(1, (int)((float)gridDim.x * tile_us / (tile_us + block_us) + 0.5f));
        }
        __syncthreads();
        // Tickets and partial results before each sequence: a running sum, 32 sequences at a time, by the first warp.
        if (tid < 32) {
            int units = 0, items = 0, parts = 0, pre = 0;
            if (shared > 0) items = row_tiles(sh->pre_rows) * (int)c.heads * tile_runs(sh, shared);
            const int pre_items = items;
            for (uint32_t base = 0; base < a.n; base += 32) {
                const uint32_t i = base + tid;
                int u = 0, x = 0, r = 0, s = 0;
                if (i < a.n && sh->plan[i].seq >= 0) {
                    const SeqPlan p = sh->plan[i];
                    const long long rs = rows_of(p, a.group);
                    const int runs = runs_of(sh, a.group, (int)i);
                    if (by_tiles(p, a.group)) x = row_tiles(rs) * (int)c.heads * (runs / halves(rs));
                    else u = (int)c.heads * runs;
                    if (runs > 1 || shares(sh, (int)i)) r = row_groups(rs) * (int)c.heads * runs;
                    if (shares(sh, (int)i)) s = (int)rs;
                }
                int us = u, xs = x, rsum = r, ss = s;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int y0 = __shfl_up_sync(0xffffffffu, us, d), y1 = __shfl_up_sync(0xffffffffu, xs, d);
                    const int y2 = __shfl_up_sync(0xffffffffu, rsum, d), y3 = __shfl_up_sync(0xffffffffu, ss, d);
                    if ((int)tid >= d) { us += y0; xs += y1; rsum += y2; ss += y3; }
                }
                if (i < a.n) {
                    sh->unit0[i] = units + us - u;
                    sh->tile0[i] = items + xs - x;
                    sh->part0[i] = r > 0 ? parts + rsum - r : -1;
                    sh->pre0[i] = pre + ss - s;
                }
                units += __shfl_sync(0xffffffffu, us, 31);
                items += __shfl_sync(0xffffffffu, xs, 31);
                parts += __shfl_sync(0xffffffffu, rsum, 31);
                pre += __shfl_sync(0xffffffffu, ss, 31);
            }
            if (tid == 0) {
                sh->units = units;
                sh->tiles = items;
                sh->pre_tiles = pre_items;
                sh->pre_part0 = parts;
                if (shared > 0) parts += row_groups(sh->pre_rows) * (int)c.heads * pre_runs(sh);
                sh->last = parts > (int)a.part_slots;          // borrowed as a flag until the end of the kernel
                const uint32_t out_rows = a.rows * a.q_heads;
                int per = 1;
                while (per < kMergeRowsMost && (unsigned long long)per * a.sms * kWorkers < out_rows) per *= 2;
                sh->merge_rows = per;
                sh->merges = parts > 0 ? (int)((out_rows + per - 1) / per) : 0;
            }
        }
        __syncthreads();
        if (sh->last == 0u || shared == 0) break;
        shared = 0;
        __syncthreads();
    }
    if (sh->shared > 0) {                                       // the first sharing sequence's table names the prefix's pages
        if (tid < 32) {
            const uint32_t mine = tid < XPK_ATTENTION_MAX_SEQS / 32 && tid * 32 < a.n ? sh->share[tid] : 0u;
            const uint32_t some = __ballot_sync(0xffffffffu, mine != 0u);
            const int word = __ffs(some) - 1;
            const uint32_t bits = __shfl_sync(0xffffffffu, mine, word);
            if (tid == 0) sh->shared_seq = sh->plan[word * 32 + __ffs(bits) - 1].seq;
        }
        __syncthreads();
    }
}

// ---- waits -------------------------------------------------------------------------------------------------------
// Bounded; false when it gave up or another warp has.
__device__ __forceinline__ bool wait_bar(void *bar, uint32_t parity, AttnShared *sh, Ctl *ctl, uint32_t code, bool heed_abort = true) {
    uint32_t it = 0;
    unsigned long long t0 = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++it & 0xFFu) == 0) {
            if (heed_abort && *(volatile uint32_t *)&sh->abort != 0u) return false;
            const unsigned long long now = global_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > kWaitLimitNs) {
                raise_error(ctl, code);
                *(volatile uint32_t *)&sh->abort = 1u;
                return false;
            }
        }
    }
    return true;
}

} // namespace xpk
