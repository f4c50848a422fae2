// The cut of an attention call into tickets (see attention.cu): what each CTA works out at its start.
#pragma once
#include "gemm_ptx.cuh"
#include "kv_cache.cuh"
#include <cuda_fp16.h>

namespace xpk {

constexpr int kWorkers = 8;                                 // warps that run units and merges; two groups of four for tiles
constexpr int kUnitThreads = kWorkers * 32;
constexpr int kAttnThreads = kUnitThreads + 128;            // and a third group for tiles: one warp loads, one issues MMAs
// Registers: 384 threads are launched with 168 each; the workers, whose rows of scores fill 128, take over what the helpers
// do not need: 2 * 216 + 72 = 3 * 168.  The forms with tiles spill all the same (724 bytes of stores at head_dim 128, 352 at 64: units and
// tiles in one kernel); the forms without take up to 224 registers and spill nothing.
constexpr int kWorkerRegs = 216, kHelperRegs = 72;
static_assert(2 * kWorkerRegs + kHelperRegs <= 3 * 168, "more registers than the launch has");
constexpr int kBlock = 16;                                  // positions per block of a unit
constexpr int kUnitRows = 16;                               // rows of a unit, and of a partial result
// Sequences of up to 32 rows go by units (two groups read the same keys, the second from L2), longer ones by tiles: 40 drafts of up to 24
// rows take 53 us, and 56 with the border at 16.
constexpr int kUnitRowsMost = 32;
constexpr int kUnitStages = 3;
// Units that each warp gets where there is enough work: each begins by waiting for memory, so more and shorter ones are slower (32 sequences
// apart: 112 us with two, 117 with three, 130 with five, before runs were made equally long).
constexpr int kUnitWaves = 2;
constexpr int kTile = 128;                                  // positions per tile; rows per group of a tile item
constexpr int kItemRows = 2 * kTile;
constexpr int kStep = 64;                                   // positions per product; tiles are counted in pairs of steps
constexpr int kRing = 8;                                    // stages of the tile ring; a stage holds a step's keys or values
constexpr int kMinRun = 4;                                  // blocks: a run shorter than 64 positions costs more to merge than it spreads
// Tiles of a run at least, two for each group of workers: 16 sequences on 4096 take 35 us, and 39 with runs of 2 (twice the results to merge).
constexpr int kMinTiles = 4;
// Sequences of more rows read the prefix by themselves: they fill half a group's tile.  12 sequences of 48 rows on a prefix of 8192 take
// 78 us together and 140 each for itself.
constexpr int kShareRows = 64;
constexpr int kMergeRowsMost = 32;
constexpr int kPageWords = 16;                              // more than the steps that a ring holds
constexpr int kSched = 2;                                   // items the loader may be ahead
// Time of a tile of 256 rows at head_dim 128 that the cut reckons with, from an earlier form of the loop.  It scales it by head_dim, which the
// tiles do not bear out: they take 3.0 us at 64 and at 128 (prompts of 1024 on 8192).
constexpr float kTileUs = 2.6f;
constexpr uint32_t kErrAttnLoad  = 0x70000001u;
constexpr uint32_t kErrAttnMerge = 0x70000002u;
constexpr uint32_t kErrAttnTile  = 0x70000003u;
constexpr uint32_t kErrAttnCut   = 0x70000004u;

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
    unsigned long long sums[5];                             // blocks, tiles, sharing rows, sharing sequences, row groups of units
    int4 warp_sums[kAttnThreads / 32];
    uint32_t first_sharing;
    // tile pipeline
    unsigned long long ring_full[kRing], ring_empty[kRing];
    unsigned long long item_full[kSched], item_empty[kSched];
    unsigned long long q_full[2], s_full[2][2], p_full[2][2], pv_done[2], o_full[2], group_bar[2], worker_bar, drain;
    int item[kSched];                                       // tickets handed to issuer and workers; -1: no more
    uint32_t tmem, odd[2], pages[2][kPageWords];            // pages of the last steps of each order of keys that are there (bits)
    // units
    unsigned long long full[kWorkers][kUnitStages];
    unsigned long long done;
    int run, tile_run;                                      // blocks (tiles) per run
    int half_rows;                                          // up to so many rows the two groups of workers take half of a run each
    int units, tiles, merges, merge_rows;
    int shared, shared_seq, pre_rows, pre_part0, pre_tiles; // prefix: positions, whose table, rows, first result, its tile items
    int tile_ctas;                                          // CTAs that begin with tiles
    uint32_t abort, stop, last;
};

template <int kDim> __host__ __device__ constexpr uint32_t unit_stage_bytes() { return 2 * kBlock * kDim * 2; }
template <int kDim> __host__ __device__ constexpr uint32_t query_bytes() { return kTile * kDim * 2; }       // of a group of workers
template <int kDim> __host__ __device__ constexpr uint32_t step_bytes() { return kStep * kDim * 2; }
template <int kDim> __host__ __device__ constexpr size_t ring_bytes() {
    const size_t tiles = (size_t)2 * query_bytes<kDim>() + (size_t)kRing * step_bytes<kDim>(), units = (size_t)kWorkers * kUnitStages * unit_stage_bytes<kDim>();
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
__device__ __forceinline__ bool by_tiles(const SeqPlan &p, uint32_t group) { return rows_of(p, group) > kUnitRowsMost; }
__device__ __forceinline__ int row_groups(long long rows) { return (int)((rows + kUnitRows - 1) / kUnitRows); }
__device__ __forceinline__ int row_tiles(long long rows) { return (int)((rows + kItemRows - 1) / kItemRows); }
// With at most 128 rows the two groups of workers take half of a run's tiles each, and leave a result each; where so many results
// do not fit the scratch (half_rows 0) the first group takes all of them.  Sequences of 64 rows by halves and without: 64 of 8000
// positions 542 and 581 us; but 256 of 500 positions 686 and 331 us, where the merges outweigh what halves gain.
__device__ __forceinline__ int halves(const AttnShared *sh, long long rows) { return rows <= sh->half_rows ? 2 : 1; }
__device__ __forceinline__ int chunks(int positions, int each, int run) { return max(1, ((positions + each - 1) / each + run - 1) / run); }
__device__ __forceinline__ int tiles_of(int positions) { return (positions + kTile - 1) / kTile; }
// Runs of about tile_run tiles, equally long: the last item to end should not be a short one's neighbour.
__device__ __forceinline__ int tile_runs(const AttnShared *sh, int positions) {
    return max(1, (tiles_of(positions) + sh->tile_run / 2) / sh->tile_run);
}
// Results that are left for each row by a sequence's own runs, and by the prefix.
__device__ __forceinline__ int runs_of(const AttnShared *sh, uint32_t group, int i) {
    const SeqPlan &p = sh->plan[i];
    const int own = p.len - own_from(sh, i);
    return by_tiles(p, group) ? tile_runs(sh, own) * halves(sh, rows_of(p, group)) : chunks(own, kBlock, sh->run);
}
__device__ __forceinline__ int pre_runs(const AttnShared *sh) { return tile_runs(sh, sh->shared) * halves(sh, sh->pre_rows); }

// ---- the cut ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// Every CTA works the same cut out of the same arrays, a thread per sequence.
__device__ __forceinline__ void make_plan(const CacheView &c, const AttnArgs &a, AttnShared *sh) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t threads = blockDim.x, warps = threads / 32;
    int shared = a.shared_len ? max(*a.shared_len, 0) & ~(int)(c.page - 1) : 0;
    if (tid < 5) sh->sums[tid] = 0;
    if (tid == 5) sh->first_sharing = 0xffffffffu;
    __syncthreads();
    for (uint32_t base = 0; base < a.n; base += threads) {              // whole warps: ballots below
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
        if (lane == 0 && i < XPK_ATTENTION_MAX_SEQS) {
            sh->share[i >> 5] = bits;
            if (bits != 0) {
                atomicAdd(&sh->sums[3], (unsigned long long)__popc(bits));
                atomicMin(&sh->first_sharing, i + __ffs(bits) - 1);
            }
        }
    }
    __syncthreads();
    if (sh->sums[3] < 2) shared = 0;
    // Results that do not fit the scratch: once more without the prefix, then without halves too.  What is left then is under
    // 64 results per SM, by sequences of several runs alone; the scratch has room for 160.
    bool halved = true;
    while (true) {
        if (shared == 0 && tid < XPK_ATTENTION_MAX_SEQS / 32) sh->share[tid] = 0;
        if (tid == 0) {
            sh->shared = shared;
            sh->half_rows = halved ? kTile : 0;
            sh->shared_seq = shared > 0 ? sh->plan[sh->first_sharing].seq : -1;
        }
        __syncthreads();
        unsigned long long blocks = 0, tiles = 0, rows = 0, groups = 0;
        for (uint32_t i = tid; i < a.n; i += threads) {
            const SeqPlan p = sh->plan[i];
            if (p.seq < 0) continue;
            const int own = p.len - own_from(sh, (int)i);
            if (by_tiles(p, a.group)) tiles += (unsigned long long)((own + kTile - 1) / kTile) * row_tiles(rows_of(p, a.group));
            else {
                blocks += (unsigned long long)((own + kBlock - 1) / kBlock) * row_groups(rows_of(p, a.group));
                groups += row_groups(rows_of(p, a.group));
            }
            if (shares(sh, (int)i)) rows += (unsigned long long)rows_of(p, a.group);
        }
        if (warp * 32 < a.n) {
            blocks = warp_sum(blocks);
            tiles = warp_sum(tiles);
            rows = warp_sum(rows);
            groups = warp_sum(groups);
            if (lane == 0) {
                atomicAdd(&sh->sums[0], blocks);
                atomicAdd(&sh->sums[1], tiles);
                atomicAdd(&sh->sums[2], rows);
                atomicAdd(&sh->sums[4], groups);
            }
        }
        __syncthreads();
        blocks = sh->sums[0] * c.heads;
        rows = sh->sums[2];
        tiles = (sh->sums[1] + (unsigned long long)((shared + kTile - 1) / kTile) * row_tiles((long long)rows)) * c.heads;
        // Units come out at work / run and about half a unit more for each row group; a few more than kUnitWaves rounds of all warps
        // would be a round of their own.
        const unsigned long long waves = (unsigned long long)a.sms * kWorkers * kUnitWaves, halves_of = sh->sums[4] * c.heads / 2;
        const unsigned long long target = max(waves - min(waves, halves_of), waves / 4);
        if (tid == 0) {
            sh->run = max(kMinRun, (int)min((blocks + target - 1) / target, 0x7fffffffull / kBlock));
            sh->pre_rows = (int)rows;
            // CTAs are dealt to tiles and units by the time each kind takes: a tile of 256 rows about kTileUs of an SM, a block
            // 64 bytes an element over the SM's share of HBM (44 GB/s): 0.19 us at 128.  Those that begin with tiles get one item each: two rounds of shorter
            // ones left more results to merge than they balanced (256 sequences on 16384: 259 against 224 us).
            const float tile_us = kTileUs * (float)tiles * ((float)c.dim / 128.f), block_us = 0.0015f * (float)c.dim * (float)blocks;
            const float share = tiles == 0 ? 0.f : blocks == 0 ? 1.f : tile_us / (tile_us + block_us);
            const unsigned long long items = max((unsigned long long)((float)a.sms * share), 1ull);
            sh->tile_run = max(kMinTiles, (int)min((tiles + items - 1) / items, 0x7fffffffull / kTile));
            sh->tile_ctas = tiles == 0 ? 0 : max(1, (int)((float)gridDim.x * share + 0.5f));
        }
        __syncthreads();
        // Tickets and partial results before each sequence: a scan in each warp, then over the warps.
        int4 carry = make_int4(0, 0, 0, 0);
        if (shared > 0) carry.y = row_tiles(sh->pre_rows) * (int)c.heads * tile_runs(sh, shared);
        const int pre_items = carry.y;
        for (uint32_t base = 0; base < a.n; base += threads) {
            const uint32_t i = base + tid;
            int4 v = make_int4(0, 0, 0, 0);                                  // units, tile items, results, sharing rows
            if (i < a.n && sh->plan[i].seq >= 0) {
                const SeqPlan p = sh->plan[i];
                const long long rs = rows_of(p, a.group);
                const int runs = runs_of(sh, a.group, (int)i), groups = row_groups(rs) * (int)c.heads;
                if (by_tiles(p, a.group)) v.y = row_tiles(rs) * (int)c.heads * (runs / halves(sh, rs));
                else v.x = groups * runs;
                if (runs > 1 || shares(sh, (int)i)) v.z = (int)min((long long)groups * runs, (long long)a.part_slots + 1);      // the sum cannot wrap
                if (shares(sh, (int)i)) v.w = (int)rs;
            }
            int4 s = v;
            if (base + warp * 32 < a.n) {
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int y0 = __shfl_up_sync(0xffffffffu, s.x, d), y1 = __shfl_up_sync(0xffffffffu, s.y, d);
                    const int y2 = __shfl_up_sync(0xffffffffu, s.z, d), y3 = __shfl_up_sync(0xffffffffu, s.w, d);
                    if ((int)lane >= d) { s.x += y0; s.y += y1; s.z += y2; s.w += y3; }
                }
            }
            if (lane == 31) sh->warp_sums[warp] = s;
            __syncthreads();
            int4 before = carry;
            for (uint32_t w = 0; w < warps && base + w * 32 < a.n; ++w) {
                const int4 y = sh->warp_sums[w];
                if (w < warp) { before.x += y.x; before.y += y.y; before.z += y.z; before.w += y.w; }
                carry.x += y.x; carry.y += y.y; carry.z += y.z; carry.w += y.w;
            }
            if (i < a.n) {
                sh->unit0[i] = before.x + s.x - v.x;
                sh->tile0[i] = before.y + s.y - v.y;
                sh->part0[i] = v.z > 0 ? before.z + s.z - v.z : -1;
                sh->pre0[i] = before.w + s.w - v.w;
            }
            __syncthreads();
        }
        int parts = carry.z;
        if (shared > 0) parts += row_groups(sh->pre_rows) * (int)c.heads * pre_runs(sh);
        const bool fits = parts <= (int)a.part_slots;                         // the same for all threads
        if (!fits && (shared > 0 || halved)) {
            __syncthreads();                                                  // the sum reads what the next round writes first
            halved = halved && shared > 0;
            shared = 0;
            if (tid < 3 || tid == 4) sh->sums[tid] = 0;
            continue;
        }
        // By the bound above the results fit now; if they ever did not, nothing is stored and a task reports it.
        if (!fits) carry.x = carry.y = parts = 0;
        if (tid == 0) {
            if (!fits) sh->abort = 1;
            sh->units = carry.x;
            sh->tiles = carry.y;
            sh->pre_tiles = pre_items;
            if (carry.y > 0 && carry.y < (int)gridDim.x && carry.x > 0) sh->tile_ctas = carry.y;          // one each: a second item would be the last to end
            sh->pre_part0 = carry.z;
            const uint32_t out_rows = a.rows * a.q_heads;
            int per = 1;
            while (per < kMergeRowsMost && (unsigned long long)per * a.sms * kWorkers < out_rows) per *= 2;
            sh->merge_rows = per;
            sh->merges = parts > 0 ? (int)((out_rows + per - 1) / per) : 0;
        }
        break;
    }
    __syncthreads();
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
