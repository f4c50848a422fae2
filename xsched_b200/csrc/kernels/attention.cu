// Attention over the paged key/value cache for single tokens, drafts and prompts.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp2(scale log2(e) (q . k_j - max)),   j below the row's limit
//
// A sequence's queries times the G = q_heads / kv_heads query heads that read one key head are its rows for that head
// (row r = query r / G, head r % G): they read the same keys, so a group of rows shares one pass over them.  Sequences that
// promise a common prefix and have few rows put their rows together for it: the prefix is one more pass, over all of them.
//
// Three kinds of tickets:
//   tiles   (256 rows, key head, a run of 128-position tiles) by a whole CTA on the tensor pipe: the prefix, and sequences
//           of more than 32 rows;
//   units   (16 rows, key head, a run of 16-position blocks) by one warp: sequences of up to 32 rows;
//   merges  a few output rows by one warp, where a row's result comes from several runs: their weighted sum.
// The cut is a function of the lengths and the device's SM count alone, and a merge adds the runs in their order, so the
// result does not depend on who computed what, or on preemption.  Merges are claimed when no tile and no unit is left and
// wait (bounded) for those that others still run.
//
// Positions that a row must not see may hold anything: scores are replaced before the maximum, values at or behind the
// sequence's end are zeroed in shared memory (0 * NaN), and where hidden values are not finite they are added with
// selects instead of MMAs.
#include "attention_tiles.cuh"

#include <algorithm>

namespace xpk {

// Claim counters in the control block's own words: they only grow while a task is unfinished, a claimed ticket is always
// finished, and a completed task's are cleared with the rest.
constexpr int kTileTickets = 0, kUnitTickets = 1, kMergeTickets = 2;

constexpr int kNone = -1, kStopped = -2;                     // every ticket is claimed; the flag was up (it may be down again)

template <bool kPreemptible>
__device__ __forceinline__ int claim(Ctl *ctl, const AttnShared *sh, int which, int total) {       // one thread
    if (*(const volatile uint32_t *)&sh->abort != 0u) return kStopped;
    if constexpr (kPreemptible) { if (ld_flag(ctl->flag) != 0) return kStopped; }
    const unsigned long long t = atomicAdd(&ctl->user[which], 1ull);
    return t < (unsigned long long)total ? (int)t : kNone;
}

// A ticket for a warp.  Tickets are never dealt by the warp's number: a CTA that has not got an SM yet would hold some, and two launches
// that share the SMs would wait for each other's.
template <bool kPreemptible>
__device__ __forceinline__ int warp_claim(Ctl *ctl, const AttnShared *sh, int which, int total) {
    int t = kNone;
    if ((threadIdx.x & 31) == 0) t = claim<kPreemptible>(ctl, sh, which, total);
    return __shfl_sync(0xffffffffu, t, 0);
}

// An item from the loader; all lanes of a warp.
__device__ __forceinline__ int next_item(AttnShared *sh, Ctl *ctl, uint32_t &seen) {
    const uint32_t slot = seen % kSched;
    if (!wait_bar(&sh->item_full[slot], (seen / kSched) & 1u, sh, ctl, kErrAttnTile)) return kStopped;
    ++seen;
    return *(volatile int *)&sh->item[slot];
}

// Some CTAs begin with tiles (tensor pipe), the others with units (HBM), so that both are busy; each goes on with the rest.
template <class T, int kDim, bool kPreemptible, bool kTiles>
__device__ __forceinline__ void workers(Ctl *ctl, const CUtensorMap *map_k, const CUtensorMap *map_v, const CacheView &c, const AttnArgs &a,
                                        AttnShared *sh, unsigned char *smem) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool tiles = kTiles && sh->tiles > 0, tiles_first = tiles && (int)blockIdx.x < sh->tile_ctas;
    unsigned char *const unit_ring = smem + (size_t)warp * kUnitStages * unit_stage_bytes<kDim>();
    Ring ring{unit_ring, sh->full[warp], kUnitStages, 0u, 0u, 0u, 0u};
    unsigned long long done = 0;
    bool stopped = false;                                   // somewhere tickets may be left
    for (int phase = 0; phase < 2; ++phase) {
        if ((phase == 0) != tiles_first) {
            while (sh->units > 0) {
                const int ticket = warp_claim<kPreemptible>(ctl, sh, kUnitTickets, sh->units);
                stopped = stopped || ticket == kStopped;
                if (ticket < 0) break;
                unit_ticket<T, kDim>(c, a, map_k, map_v, sh, ctl, ring, ticket);
                done += lane == 0;
            }
            if (tiles && !tiles_first) __syncthreads();      // the units' rings lie where the tiles will: the loader waits here too
        } else if constexpr (kTiles) {
            if (!tiles) continue;
            WorkState st = {};
            uint32_t seen = 0;
            while (true) {
                const uint32_t slot = seen % kSched;
                const int ticket = __shfl_sync(0xffffffffu, next_item(sh, ctl, seen), 0);
                stopped = stopped || ticket == kStopped;
                if (ticket < 0) break;
                const TileItem x = tile_ticket(a, c, sh, ticket);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->item_empty[slot]);
                work_tiles<T, kDim>(c, a, map_k, map_v, sh, ctl, smem, smem + 2 * query_bytes<kDim>(), st, ring, x);
                done += threadIdx.x == 0;
            }
            // Both groups are through with the tiles' memory before units use it.
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->worker_bar);
            wait_bar(&sh->worker_bar, 0u, sh, ctl, kErrAttnTile);
            __syncwarp();
            ring.move(unit_ring, kUnitStages);
        }
    }
    // Merges wait for every unit and tile: only once all of them are claimed, by warps that finish them, may one be begun.  Without
    // anything to do there is one merge of nothing, so that the call has a ticket to complete.
    while (!stopped) {
        const int ticket = warp_claim<kPreemptible>(ctl, sh, kMergeTickets, sh->merges);
        if (ticket < 0) break;
        run_merge<T, kDim>(c, a, sh, ctl, ticket);
        done += lane == 0;
    }
    // Loads that a unit gave up on still reach this CTA's shared memory: wait for them.
    while (ring.pending > 0) {
        wait_bar(&ring.full[ring.using_], ring.parity(), sh, ctl, kErrAttnLoad, false);
        ring.give();
    }
    if (done) atomicAdd(&sh->done, done);
}

template <class T, int kDim, bool kPreemptible>
__device__ __forceinline__ void helpers(Ctl *ctl, const CUtensorMap *page_k, const CUtensorMap *page_v, const CacheView &c, const AttnArgs &a,
                                        AttnShared *sh, unsigned char *smem) {
    if (sh->tiles == 0) return;
    if ((int)blockIdx.x >= sh->tile_ctas) __syncthreads();
    unsigned char *tiles = smem + 2 * query_bytes<kDim>();
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
    if (warp == kWorkers) {                                  // loader
        const int lane = threadIdx.x & 31;
        uint32_t stage = 0, given = 0, keys0 = 0, keys1 = 0, ends = 0;
        while (true) {
            int ticket = kNone;
            if (lane == 0) ticket = claim<kPreemptible>(ctl, sh, kTileTickets, sh->tiles);
            ticket = __shfl_sync(0xffffffffu, ticket, 0);
            const uint32_t slot = given % kSched;
            if (!__all_sync(0xffffffffu, wait_bar(&sh->item_empty[slot], ((given / kSched) & 1u) ^ 1u, sh, ctl, kErrAttnTile))) break;
            if (lane == 0) {
                *(volatile int *)&sh->item[slot] = ticket;
                mbar_arrive(&sh->item_full[slot]);
            }
            ++given;
            if (ticket < 0) break;
            const TileItem x = tile_ticket(a, c, sh, ticket);
            if (!load_steps<kDim>(c, a, page_k, page_v, sh, ctl, tiles, stage, keys0, keys1, x)) break;
            // Ahead into the next item only while every CTA still gets one: the last ones go to whoever is through.
            bool ok = true;
            for (int w = 0; w < 2; ++w) {
                if ((w == 0 ? x.steps0 : x.steps1) == 0) continue;
                if (ticket + (int)gridDim.x >= sh->tiles)
                    ok = ok && __all_sync(0xffffffffu, wait_bar(&sh->o_full[w], ends >> w & 1u, sh, ctl, kErrAttnTile));
                ends ^= 1u << w;
            }
            if (!ok) break;
        }
        // Loads that nobody waited for: before the memory goes.
        for (uint32_t s = stage > (uint32_t)kRing ? stage - kRing : 0u; s < stage; ++s)
            wait_bar(&sh->ring_full[s % kRing], (s / kRing) & 1u, sh, ctl, kErrAttnTile, false);
    } else if (warp == kWorkers + 1) {                       // issuer
        const uint32_t lead = elect_lead();
        IssueState st = {};
        uint32_t seen = 0;
        while (true) {
            const uint32_t slot = seen % kSched;
            const int ticket = __shfl_sync(0xffffffffu, next_item(sh, ctl, seen), 0);
            if (ticket < 0) break;
            const TileItem x = tile_ticket(a, c, sh, ticket);
            __syncwarp();
            if (lead) mbar_arrive(&sh->item_empty[slot]);
            const int n0 = __shfl_sync(0xffffffffu, x.steps0, 0), n1 = __shfl_sync(0xffffffffu, x.steps1, 0);
            const bool both = __shfl_sync(0xffffffffu, (int)x.both, 0) != 0;
            if (!issue_steps<T, kDim>(sh, ctl, smem, tiles, st, n0, n1, both, lead)) break;
        }
        attn_commit(&sh->drain, lead);
        wait_bar(&sh->drain, 0u, sh, ctl, kErrAttnTile, false);
    }
    __syncwarp();
}

template <class T, int kDim, bool kPreemptible, bool kTiles>
__device__ __forceinline__ void work_off(Ctl *ctl, const CUtensorMap *map_k, const CUtensorMap *map_v, const CUtensorMap *page_k, const CUtensorMap *page_v,
                                         const CacheView &c, const AttnArgs &a, AttnShared *sh, unsigned char *smem) {
    const int warp = threadIdx.x >> 5;
    make_plan(c, a, sh);
    const int merges = max(sh->merges, sh->tiles + sh->units == 0 ? 1 : 0);
    const bool tiles = kTiles && sh->tiles > 0;
    if (threadIdx.x == 0) {
        // Never zero: a task that was stopped before any CTA got here must not look complete.
        *(volatile unsigned long long *)&ctl->total = (unsigned long long)sh->tiles + sh->units + merges;       // the same from every CTA
        if (sh->abort != 0u) raise_error(ctl, kErrAttnCut);
    }
    if (tiles && warp == kWorkers + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&sh->tmem)), "r"(kAttnTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0) sh->merges = merges;
    if constexpr (!kTiles) {
        workers<T, kDim, kPreemptible, false>(ctl, map_k, map_v, c, a, sh, smem);
        return;
    } else if (warp < kWorkers) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kWorkerRegs));
        workers<T, kDim, kPreemptible, true>(ctl, map_k, map_v, c, a, sh, smem);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kHelperRegs));
        helpers<T, kDim, kPreemptible>(ctl, page_k, page_v, c, a, sh, smem);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (tiles && warp == kWorkers + 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(*(volatile uint32_t *)&sh->tmem), "r"(kAttnTmemCols) : "memory");
}

// kTiles: the call may have tiles.  The form without them is what calls run whose sequences have one query each and no prefix: eight warps
// instead of twelve, and registers for units alone.
template <class T, int kDim, bool kPreemptible, bool kTiles>
__global__ void __launch_bounds__(kTiles ? kAttnThreads : kUnitThreads, 1)
attention_kernel(Ctl *ctl, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap page_k, const __grid_constant__ CUtensorMap page_v,
                 const __grid_constant__ CacheView c, const __grid_constant__ AttnArgs a, unsigned long long launch_no) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    AttnShared *sh = reinterpret_cast<AttnShared *>(smem + ring_bytes<kDim>());
    note_start(ctl);
    if (threadIdx.x == 0) {
        for (int w = 0; w < kWorkers; ++w)
            for (int s = 0; s < kUnitStages; ++s) mbar_init(&sh->full[w][s], 1);
        for (int s = 0; s < kRing; ++s) { mbar_init(&sh->ring_full[s], 1); mbar_init(&sh->ring_empty[s], 1); }
        for (int s = 0; s < kSched; ++s) { mbar_init(&sh->item_full[s], 1); mbar_init(&sh->item_empty[s], 1 + kWorkers); }
        for (int w = 0; w < 2; ++w) {
            mbar_init(&sh->q_full[w], 4);
            mbar_init(&sh->pv_done[w], 1);
            mbar_init(&sh->o_full[w], 1);
            for (int b = 0; b < 2; ++b) { mbar_init(&sh->s_full[w][b], 1); mbar_init(&sh->p_full[w][b], 4); }
            sh->odd[w] = 0;
        }
        mbar_init(&sh->group_bar[0], 4);
        mbar_init(&sh->group_bar[1], 4);
        mbar_init(&sh->worker_bar, kWorkers);
        mbar_init(&sh->drain, 1);
        sh->done = 0;
        sh->abort = 0;
        // Queued behind a launch that is being stopped: no set-up.
        sh->stop = kPreemptible && ld_flag(ctl->flag) != 0 ? 1u : 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    if (sh->stop == 0u) work_off<T, kDim, kPreemptible, kTiles>(ctl, &map_k, &map_v, &page_k, &page_v, c, a, sh, smem);
    __syncthreads();
    if (threadIdx.x == 0) sh->last = cta_leave(ctl, sh->done) ? 1u : 0u;
    __syncthreads();
    if (sh->last == 0u) return;
    // The last CTA leaves the counters ready for the next call once the work is complete.
    const bool task = ctl->mailbox != nullptr;
    const bool whole = *(volatile unsigned long long *)&ctl->tiles_done >= *(volatile unsigned long long *)&ctl->total;
    if (whole || !task)
        for (uint32_t i = threadIdx.x; i < (a.n + 1) * c.heads; i += blockDim.x) a.counters[i] = 0;
    if (!task) {                                           // a call without a task keeps nothing, not even an error
        if (threadIdx.x < kCtlResetBytes / 8) reinterpret_cast<unsigned long long *>(ctl)[threadIdx.x] = 0;
        return;
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) cta_fold(ctl, launch_no);
}

// ---- host side -------------------------------------------------------------------------------------------------
template <class T, int kDim>
static cudaError_t prepare_one() {
    const void *forms[] = {(const void *)attention_kernel<T, kDim, true, true>, (const void *)attention_kernel<T, kDim, true, false>,
                           (const void *)attention_kernel<T, kDim, false, true>, (const void *)attention_kernel<T, kDim, false, false>};
    for (const void *f : forms) {
        const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)attn_smem<kDim>());
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
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
    uint32_t part_slots;
};
AttnScratch attention_scratch(const CacheView &c, uint32_t sms, uint32_t rows, uint32_t n, uint32_t q_heads) {
    AttnScratch s;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    // Sequences of several runs leave less than twice work / run results, and a run is at least work / target (for tiles: 16
    // slots a result, two halves).  With a prefix every sharing sequence leaves some: one per key head if it is of one row
    // group (all are where each has a single query of up to 16 heads), at most eight; the prefix itself 16 per item.  Sequences
    // of 33 to 128 rows leave two per row group even in one run; the kernel cuts them without halves if they do not suffice.
    const size_t group = q_heads / c.heads, most = std::min<size_t>(n, rows);
    const size_t base = 2 * (size_t)kUnitWaves * sms * kWorkers + 128 * (size_t)sms;
    const size_t own = c.heads * most * (rows <= n && group <= kUnitRows ? 1 : 8);
    const size_t pre_rows = std::min<size_t>((size_t)rows * group, most * kShareRows);
    const size_t pre = 16 * (c.heads * ((pre_rows + kItemRows - 1) / kItemRows) + 4 * (size_t)sms);
    // More than 2^16 slots (1/2 GB at 128) are not worth a prefix: the kernel does without it if they do not suffice.
    s.part_slots = (uint32_t)(base + std::min<size_t>(own + pre, 1u << 16));
    s.ctl = 0;
    s.counters = up(sizeof(Ctl));
    // As many counters as any call needs: what has to be zero lies at the same place for all calls that use the scratch in turn.
    s.ml = s.counters + up((size_t)(XPK_ATTENTION_MAX_SEQS + 1) * c.heads * 4);
    s.part = s.ml + up((size_t)s.part_slots * kUnitRows * sizeof(float2));
    s.bytes = s.part + (size_t)s.part_slots * kUnitRows * c.dim * sizeof(float);
    return s;
}
size_t attention_scratch_bytes(const CacheView &c, uint32_t sms, uint32_t rows, uint32_t n, uint32_t q_heads) {
    return attention_scratch(c, sms, rows, n, q_heads).bytes;
}
// What xpkTaskReset clears: the counters (the partial results need no clearing).
void attention_counters(const CacheView &c, uint32_t sms, const xpkAttentionArgs &x, void **at, size_t *bytes) {
    const AttnScratch s = attention_scratch(c, sms, x.rows, x.n, x.q_heads);
    *at = (unsigned char *)x.scratch + s.counters;
    *bytes = ((size_t)x.n + 1) * c.heads * 4;
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
    a.shared_len = x.shared_len;
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
    a.part_slots = s.part_slots;
    if (ctl == nullptr) ctl = (Ctl *)(scratch + s.ctl);
    const CUtensorMap &mk = *(const CUtensorMap *)cache->map_k, &mv = *(const CUtensorMap *)cache->map_v;
    const CUtensorMap &pk = *(const CUtensorMap *)cache->page_k, &pv = *(const CUtensorMap *)cache->page_v;
    const bool bf16 = cache->d.dtype == XPK_DTYPE_BF16;
    // The host does not know lengths, but a row for each sequence and nothing shared means units only.
    const bool tiles = a.starts != nullptr || a.shared_len != nullptr || a.group > (uint32_t)kUnitRowsMost;
#define XPK_ATTN(T, D)                                                                                                                          \
    do {                                                                                                                                        \
        auto *f = tiles ? (preemptible ? attention_kernel<T, D, true, true> : attention_kernel<T, D, false, true>)                             \
                        : (preemptible ? attention_kernel<T, D, true, false> : attention_kernel<T, D, false, false>);                          \
        f<<<grid, tiles ? kAttnThreads : kUnitThreads, attn_smem<D>(), st>>>(ctl, mk, mv, pk, pv, c, a, launch_no);                             \
    } while (0)
    if (bf16 && c.dim == 128) XPK_ATTN(__nv_bfloat16, 128);
    else if (bf16) XPK_ATTN(__nv_bfloat16, 64);
    else if (c.dim == 128) XPK_ATTN(__half, 128);
    else XPK_ATTN(__half, 64);
#undef XPK_ATTN
    return cudaGetLastError();
}

} // namespace xpk
