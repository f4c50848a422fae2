// Pages of the key/value cache: free, fork, extend (with copy on write), compact, copy.
//
// The state is three integer arrays (table, lens, refs); a page is free when its count is zero, so there is no free list
// to keep in order: new pages are the lowest free ones, found by a scan of refs.  Every decision is a function of the
// arrays and the list, never of the order in which threads arrive.
//
//   free     one CTA per listed sequence.  Whoever exchanges lens[seq] for 0 first owns the row (a sequence listed twice
//            gives its pages back once), clears it and decrements the counts.
//   fork     one CTA per entry copies the parent's row and increments the counts.  lens stays as it was until the last
//            CTA leaves (an exit counter) and writes all of them: every CTA judges its entry by the lengths from before.
//   extend   one CTA: pages needed per entry, prefix sum in list order, scan of refs for that many free pages, then
//            table, counts and lens; the pages to be copied go to a list that the copy kernel behind it reads.
//   compact  one CTA ranks the holes below the number of live pages and the live pages above it (equally many); a grid
//            behind it copies the pages and rewrites the rows.
//   copy     one warp moves 2 KB at a time, four 16-byte words per lane in flight; 64 warps an SM keep 128 KB in flight,
//            about three times what latency x bandwidth asks for.  HBM-bound: every byte read and written once.
#include "kv_cache.cuh"

namespace xpk {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr uint32_t kUnitBytes = 2048;                    // slabs are whole units: 16 positions x 64 elements x 2 bytes
constexpr uint32_t kTileUnits = 32;                      // 64 KB: what a preemptible copy claims

// ------------------------------------------------------------------------------------------------- free and fork
__global__ void __launch_bounds__(128) kv_free_kernel(CacheView c, const int32_t *__restrict__ seqs, uint32_t n) {
    __shared__ int s_len;
    for (uint32_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int seq = seqs[i];
        if (threadIdx.x == 0) {
            s_len = 0;
            if (seq >= 0 && (uint32_t)seq < c.seqs) s_len = atomicExch(&c.lens[seq], 0);
        }
        __syncthreads();
        const int pages = s_len > 0 ? (int)min((long long)pages_of(c, s_len), (long long)c.width) : 0;
        int32_t *row = c.table + (size_t)max(seq, 0) * c.width;
        for (int j = threadIdx.x; j < pages; j += blockDim.x) {
            const int p = row[j];
            row[j] = -1;
            if (p >= 0 && (uint32_t)p < c.pages) atomicSub(&c.refs[p], 1);
        }
        __syncthreads();
    }
}

// Whether the lengths from before the call let entry i through (duplicates apart).
__device__ __forceinline__ bool fork_fits(const CacheView &c, const int32_t *parents, const int32_t *children, uint32_t i) {
    const int ch = children[i];
    return ch >= 0 && (uint32_t)ch < c.seqs && c.lens[ch] <= 0 && held_by(c, parents[i]) > 0;
}

__global__ void __launch_bounds__(256) kv_fork_kernel(CacheView c, KvWork w, const int32_t *__restrict__ parents,
                                                      const int32_t *__restrict__ children, uint32_t n) {
    __shared__ uint32_t s_last;
    for (uint32_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int child = children[i], parent = parents[i];
        bool pass = fork_fits(c, parents, children, i);
        bool earlier = false;
        if (pass)
            for (uint32_t j = threadIdx.x; j < i; j += blockDim.x)
                earlier |= children[j] == child && fork_fits(c, parents, children, j);
        pass = pass && !__syncthreads_or(earlier);          // all threads of the CTA agree on `pass`
        const int len = pass ? held_by(c, parent) : 0;
        const int pages = pages_of(c, len);
        for (int j = threadIdx.x; j < pages; j += blockDim.x) {
            const int p = c.table[(size_t)parent * c.width + j];
            c.table[(size_t)child * c.width + j] = p;
            if (p >= 0 && (uint32_t)p < c.pages) atomicAdd(&c.refs[p], 1);
        }
        if (threadIdx.x == 0) w.taken[i] = len;
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) s_last = atomicAdd(w.exited, 1u) + 1u == gridDim.x;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int len = __ldcg(&w.taken[i]);
        if (len > 0) c.lens[children[i]] = len;
    }
    if (threadIdx.x == 0) *w.exited = 0;
}

// ------------------------------------------------------------------------------------------------ scans of one CTA
// Exclusive sum over the CTA's threads; `total` gets the sum of all.
template <class N>
__device__ __forceinline__ N block_scan(N v, N *s_warp, N &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    N x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const N y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();                                        // s_warp of the call before has been read
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    const N sum = lane < (int)(blockDim.x >> 5) ? s_warp[lane] : 0;
    N y = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const N z = __shfl_up_sync(0xffffffffu, y, d);
        if (lane >= d) y += z;
    }
    const N before = __shfl_sync(0xffffffffu, y - sum, warp);
    total = __shfl_sync(0xffffffffu, y, 31);
    return before + x - v;
}

// ------------------------------------------------------------------------------------------------------- extend
__global__ void __launch_bounds__(kPlanThreads) kv_extend_kernel(CacheView c, KvWork w, const int32_t *__restrict__ seqs,
                                                                 const int32_t *__restrict__ tokens, uint32_t n) {
    constexpr int kEach = XPK_KV_MAX_LIST / kPlanThreads;
    __shared__ int s_seq[XPK_KV_MAX_LIST], s_tail[XPK_KV_MAX_LIST], s_off[XPK_KV_MAX_LIST];
    __shared__ int s_warp[32], s_copied;
    __shared__ long long s_warp_need[32];
    const int tid = threadIdx.x;
    int held[kEach], grow[kEach];
    bool again[kEach];
    for (int e = 0; e < kEach; ++e) {
        const uint32_t i = e * kPlanThreads + tid;
        held[e] = grow[e] = 0;
        again[e] = false;
        if (i >= n) continue;
        const int seq = seqs[i];
        const int len = held_by(c, seq);
        int tail = -1;
        if (len >= 0) {
            held[e] = len;
            grow[e] = max(tokens[i], 0);
            if (grow[e] > 0 && (len & (c.page - 1)) != 0) {
                tail = c.table[(size_t)seq * c.width + (len >> c.page_shift)];
                if (tail < 0 || (uint32_t)tail >= c.pages) tail = -1;
            }
        }
        s_seq[i] = len >= 0 ? seq : -1;
        s_tail[i] = tail;
    }
    if (tid == 0) s_copied = 0;
    __syncthreads();
    for (int e = 0; e < kEach; ++e) {
        const int i = e * kPlanThreads + tid;
        if (i >= (int)n || s_seq[i] < 0) continue;
        for (int j = 0; j < i; ++j) again[e] |= s_seq[j] == s_seq[i];
    }
    __syncthreads();
    for (int e = 0; e < kEach; ++e) {
        const int i = e * kPlanThreads + tid;
        if (i < (int)n && again[e]) { s_seq[i] = -1; s_tail[i] = -1; }
    }
    __syncthreads();
    // Entries of one shared last page split off in list order; the last holder keeps it.
    bool split[kEach];
    for (int e = 0; e < kEach; ++e) {
        const int i = e * kPlanThreads + tid;
        split[e] = false;
        if (i >= (int)n || s_tail[i] < 0) continue;
        const int holders = c.refs[s_tail[i]];
        if (holders <= 1) continue;
        int rank = 0;
        for (int j = 0; j < i; ++j) rank += s_tail[j] == s_tail[i];
        split[e] = holders - rank > 1;
    }
    __syncthreads();
    int carry = 0, refused = 0;
    for (int e = 0; e < kEach; ++e) {
        const int i = e * kPlanThreads + tid;
        int need = 0;
        if (i < (int)n) {
            if (!split[e]) s_tail[i] = -1;                   // from here on: the page to copy
            if (s_seq[i] >= 0) {
                const long long has = ((long long)held[e] + grow[e] + c.page - 1) >> c.page_shift;
                if (has > (long long)c.width || (long long)held[e] + grow[e] > 0x7fffffffll) ++refused;
                else need = (int)has - pages_of(c, held[e]) + (split[e] ? 1 : 0);
            }
        }
        // In 64 bits: an entry may want as many pages as a table row has, 2^26, and 1024 of them are summed.  More than every page
        // there is stays more; offsets count only if no page is missing.
        long long total;
        const long long before = block_scan((long long)need, s_warp_need, total), most = (long long)c.pages + 1;
        if (i < (int)n) s_off[i] = (int)min(carry + before, most);
        carry = (int)min(carry + total, most);
    }
    int all_refused;
    block_scan(refused, s_warp, all_refused);
    // The lowest free pages, as many as are needed.
    int found = 0;
    if (all_refused == 0) {
        for (uint32_t base = 0; base < c.pages && found < carry; base += 4 * kPlanThreads) {
            const uint32_t p0 = base + 4 * tid;
            int free4[4], mine = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                free4[k] = p0 + k < c.pages ? c.refs[p0 + k] == 0 : 0;
                mine += free4[k];
            }
            int total;
            int at = found + block_scan(mine, s_warp, total);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (free4[k]) { if (at < carry) w.remap[at] = (int)(p0 + k); ++at; }
            found += total;
        }
    }
    __syncthreads();
    const int missing = max(0, carry - found);
    if (all_refused != 0 || missing != 0) {
        if (tid == 0) {
            w.report[kReportCopied] = 0;
            w.report[kReportMissing] = all_refused != 0 ? 0 : missing;
            w.report[kReportRefused] = all_refused;
        }
        return;
    }
    // Page r of the new ones belongs to the last entry whose offset is at most r.
    for (int r = tid; r < carry; r += kPlanThreads) {
        int lo = 0, hi = (int)n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s_off[mid] <= r) lo = mid; else hi = mid - 1;
        }
        const int page = w.remap[r], seq = s_seq[lo], had = pages_of(c, held_by(c, seq));
        const int local = r - s_off[lo], old = s_tail[lo];
        int32_t *row = c.table + (size_t)seq * c.width;
        c.refs[page] = 1;
        if (old >= 0 && local == 0) {
            row[had - 1] = page;
            atomicSub(&c.refs[old], 1);
            const int at = atomicAdd(&s_copied, 1);
            w.src[at] = old;
            w.dst[at] = page;
        } else {
            row[had + local - (old >= 0 ? 1 : 0)] = page;
        }
    }
    __syncthreads();
    for (int e = 0; e < kEach; ++e) {
        const int i = e * kPlanThreads + tid;
        if (i < (int)n && s_seq[i] >= 0) c.lens[s_seq[i]] = held[e] + grow[e];
    }
    if (tid == 0) {
        w.report[kReportCopied] = s_copied;
        w.report[kReportMissing] = 0;
        w.report[kReportRefused] = 0;
    }
}

// ------------------------------------------------------------------------------------------------------ compact
__global__ void __launch_bounds__(kPlanThreads) kv_compact_kernel(CacheView c, KvWork w) {
    __shared__ int s_warp[32];
    const int tid = threadIdx.x;
    int mine = 0, live;
    for (uint32_t p = tid; p < c.pages; p += kPlanThreads) mine += c.refs[p] > 0;
    block_scan(mine, s_warp, live);
    int holes = 0, movers = 0;
    for (uint32_t base = 0; base < c.pages; base += 4 * kPlanThreads) {
        const uint32_t p0 = base + 4 * tid;
        int hole = 0, move = 0;                                    // a bit for each of four pages
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t p = p0 + k;
            if (p >= c.pages) continue;
            const bool used = c.refs[p] > 0;
            if (p < (uint32_t)live) hole |= (used ? 0 : 1) << k;
            else move |= (used ? 1 : 0) << k;
        }
        int th, tm;
        int ah = holes + block_scan(__popc(hole), s_warp, th);
        int am = movers + block_scan(__popc(move), s_warp, tm);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (hole >> k & 1) w.dst[ah++] = (int)(p0 + k);
            if (move >> k & 1) w.src[am++] = (int)(p0 + k);
        }
        holes += th;
        movers += tm;
    }
    __syncthreads();
    for (int r = tid; r < movers; r += kPlanThreads) {
        const int from = w.src[r], to = w.dst[r];
        w.remap[from] = to;
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
    }
    if (tid == 0) {
        w.report[kReportCopied] = movers;
        w.report[kReportMissing] = 0;
        w.report[kReportRefused] = 0;
        w.report[kReportLive] = live;
    }
}

// --------------------------------------------------------------------------------------------------------- copy
struct CopyShape {
    uint32_t slab_units;      // units of one page in one layer of k (or v)
    uint32_t pair_units;      // slab_units * 2 * layers
    size_t slab_bytes, layer_bytes;
};
__host__ __device__ inline CopyShape copy_shape(const CacheView &c) {
    CopyShape s;
    s.slab_bytes = (size_t)c.heads * c.page * c.dim * 2;
    s.layer_bytes = s.slab_bytes * c.pages;
    s.slab_units = (uint32_t)(s.slab_bytes / kUnitBytes);
    s.pair_units = s.slab_units * 2 * c.layers;
    return s;
}

// One warp copies unit u of the pairs' units; which pages: src[u / pair_units] -> dst[..].
__device__ __forceinline__ void copy_unit(const CacheView &c, const CopyShape &s, const int32_t *src, const int32_t *dst, unsigned long long u) {
    const uint32_t pair = (uint32_t)(u / s.pair_units), in = (uint32_t)(u - (unsigned long long)pair * s.pair_units);
    const uint32_t slab = in / s.slab_units, off = in - slab * s.slab_units;
    const int from = src[pair], to = dst[pair];
    if (from < 0 || (uint32_t)from >= c.pages || to < 0 || (uint32_t)to >= c.pages || from == to) return;
    unsigned char *base = ((slab & 1) ? c.v : c.k) + (size_t)(slab >> 1) * s.layer_bytes + (size_t)off * kUnitBytes + (threadIdx.x & 31) * 16;
    const uint4 *a = reinterpret_cast<const uint4 *>(base + (size_t)from * s.slab_bytes);
    uint4 *b = reinterpret_cast<uint4 *>(base + (size_t)to * s.slab_bytes);
    uint4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __ldcs(a + 32 * k);
#pragma unroll
    for (int k = 0; k < 4; ++k) __stcs(b + 32 * k, x[k]);
}

// `count` on the device (the plan in front wrote it) or, if null, `n`.  kRemap: the rows are rewritten as well.
template <bool kRemap>
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(CacheView c, KvWork w, const int32_t *__restrict__ src, const int32_t *__restrict__ dst,
                                                               const int32_t *count, uint32_t n) {
    if constexpr (kRemap) {
        const int live = w.report[kReportLive];
        for (uint32_t seq = blockIdx.x; seq < c.seqs; seq += gridDim.x) {
            const int pages = pages_of(c, held_by(c, (int)seq));
            int32_t *row = c.table + (size_t)seq * c.width;
            for (int j = threadIdx.x; j < pages; j += kCopyThreads) {
                const int p = row[j];
                if (p >= live && (uint32_t)p < c.pages) row[j] = w.remap[p];
            }
        }
    }
    const CopyShape s = copy_shape(c);
    const unsigned long long total = (unsigned long long)(count ? (uint32_t)max(*count, 0) : n) * s.pair_units;
    const unsigned long long warps = (unsigned long long)gridDim.x * (kCopyThreads / 32);
    for (unsigned long long u = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); u < total; u += warps) copy_unit(c, s, src, dst, u);
}

template <bool kPreemptible>
__global__ void __launch_bounds__(kCopyThreads) kv_copy_task_kernel(Ctl *ctl, CacheView c, const int32_t *__restrict__ src,
                                                                    const int32_t *__restrict__ dst, uint32_t n, unsigned long long launch_no) {
    __shared__ unsigned long long s_tile;
    note_start(ctl);
    const CopyShape s = copy_shape(c);
    const unsigned long long total = (unsigned long long)n * s.pair_units;
    unsigned long long done = 0;
    while (true) {
        if (threadIdx.x == 0) s_tile = claim_tile<kPreemptible>(ctl);
        __syncthreads();
        const unsigned long long tile = s_tile;
        if (tile == kNoTile) break;
        for (uint32_t k = threadIdx.x >> 5; k < kTileUnits; k += kCopyThreads / 32) {
            const unsigned long long u = tile * kTileUnits + k;
            if (u < total) copy_unit(c, s, src, dst, u);
        }
        ++done;
        __syncthreads();
    }
    if (threadIdx.x == 0) cta_exit(ctl, done, launch_no);
}

// --------------------------------------------------------------------------------------------------- host side
cudaError_t launch_kv_free(const CacheView &c, const int32_t *seqs, uint32_t n, int sms, cudaStream_t st) {
    kv_free_kernel<<<min(n, (uint32_t)sms * 8), 128, 0, st>>>(c, seqs, n);
    return cudaGetLastError();
}
cudaError_t launch_kv_fork(const CacheView &c, const KvWork &w, const int32_t *parents, const int32_t *children, uint32_t n, int sms, cudaStream_t st) {
    kv_fork_kernel<<<min(n, (uint32_t)sms * 4), 256, 0, st>>>(c, w, parents, children, n);
    return cudaGetLastError();
}
constexpr int kCopyCtasPerSm = 8;
cudaError_t launch_kv_extend(const CacheView &c, const KvWork &w, const int32_t *seqs, const int32_t *tokens, uint32_t n, int sms, cudaStream_t st) {
    kv_extend_kernel<<<1, kPlanThreads, 0, st>>>(c, w, seqs, tokens, n);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    kv_copy_kernel<false><<<sms * kCopyCtasPerSm, kCopyThreads, 0, st>>>(c, w, w.src, w.dst, w.report + kReportCopied, 0);
    return cudaGetLastError();
}
cudaError_t launch_kv_compact(const CacheView &c, const KvWork &w, int sms, cudaStream_t st) {
    kv_compact_kernel<<<1, kPlanThreads, 0, st>>>(c, w);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    kv_copy_kernel<true><<<sms * kCopyCtasPerSm, kCopyThreads, 0, st>>>(c, w, w.src, w.dst, w.report + kReportCopied, 0);
    return cudaGetLastError();
}
cudaError_t launch_kv_copy(const CacheView &c, const KvWork &w, const int32_t *src, const int32_t *dst, uint32_t n, int sms, cudaStream_t st) {
    const unsigned long long ctas = ((unsigned long long)n * copy_shape(c).pair_units + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
    kv_copy_kernel<false><<<(int)min(ctas, (unsigned long long)sms * kCopyCtasPerSm), kCopyThreads, 0, st>>>(c, w, src, dst, nullptr, n);
    return cudaGetLastError();
}
unsigned long long kv_copy_tiles(const CacheView &c, uint32_t n) {
    return ((unsigned long long)n * copy_shape(c).pair_units + kTileUnits - 1) / kTileUnits;
}
cudaError_t launch_kv_copy_task(bool preemptible, Ctl *ctl, const CacheView &c, const int32_t *src, const int32_t *dst, uint32_t n,
                                unsigned long long launch_no, int sms, cudaStream_t st) {
    const int grid = (int)min(kv_copy_tiles(c, n), (unsigned long long)sms * kCopyCtasPerSm);
    if (preemptible) kv_copy_task_kernel<true><<<grid, kCopyThreads, 0, st>>>(ctl, c, src, dst, n, launch_no);
    else kv_copy_task_kernel<false><<<grid, kCopyThreads, 0, st>>>(ctl, c, src, dst, n, launch_no);
    return cudaGetLastError();
}

} // namespace xpk
