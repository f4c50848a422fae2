// Norms of queries and keys for each head, rotation by position, and the write of keys and values into their pages: one
// pass over the rows of a projection.
//
//   y = x / sqrt(mean(x^2) + eps) * w        per head, fp32
//   (a, b) <- (a cos t - b sin t, b cos t + a sin t),   t = position * inv_freq[j]
//
// HBM-bound: every element is read once and written once (2 + 2 bytes), 12 KB in and 12 KB out per row at 32 + 2 * 8
// heads of 128.  A thread holds 16 bytes (8 elements) of a head at a time, so a head is 16 (8) lanes of one warp and the mean
// is four (three) shuffles.  A CTA takes one row, or four where there are many; its places, and its rotary / 2 angles a row, which
// all heads share through shared memory, are worked out under the loads of the first words.
//
// Angles: a position of 900,000 times a frequency of 1 leaves an fp32 angle with an error of 0.03; so the product and its
// reduction to [-pi, pi] are fp64 and only the remainder is rounded (2e-7) before sincosf.  The pairs (j, j + rotary / 2)
// are rotary / 16 lanes apart, since rotary is a multiple of 16; neighbouring pairs are in one thread.
#include "kv_cache.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace xpk {

constexpr int kAppendThreads = 256;

template <class T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float2 open(uint32_t x) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&x)); }
    static __device__ __forceinline__ uint32_t close(float a, float b) { __nv_bfloat162 y = __floats2bfloat162_rn(a, b); return *reinterpret_cast<uint32_t *>(&y); }
};
template <> struct Pair<__half> {
    static __device__ __forceinline__ float2 open(uint32_t x) { return __half22float2(*reinterpret_cast<__half2 *>(&x)); }
    static __device__ __forceinline__ uint32_t close(float a, float b) { __half2 y = __floats2half2_rn(a, b); return *reinterpret_cast<uint32_t *>(&y); }
};

template <class T>
__device__ __forceinline__ void open8(const uint4 &x, float (&f)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 p = Pair<T>::open(w[k]);
        f[2 * k] = p.x;
        f[2 * k + 1] = p.y;
    }
}
template <class T>
__device__ __forceinline__ uint4 close8(const float (&f)[8]) {
    return make_uint4(Pair<T>::close(f[0], f[1]), Pair<T>::close(f[2], f[3]), Pair<T>::close(f[4], f[5]), Pair<T>::close(f[6], f[7]));
}

// The entry of `starts` [n + 1] that row r belongs to: the last one that starts at or before it (-1: none); the whole warp.
// Each look narrows it down by 32 with one load a lane: a halving search would wait for memory five times as often.
__device__ __forceinline__ int entry_of(const int32_t *starts, int n, int r) {
    const int lane = threadIdx.x & 31;
    int lo = -1, hi = n;                                        // starts[lo] <= r < starts[hi]
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
        const bool below = at < hi && starts[at] <= r;
        const int got = __popc(__ballot_sync(0xffffffffu, below));
        const int from = lo + got * step;
        hi = min(hi, from + step);
        lo = from;
    }
    return lo >= 0 && r < starts[lo + 1] ? lo : -1;
}

struct RowPlace {
    long long pos;              // of the row in its sequence, -1: nothing to do
    int page;                   // -1: not there
};

// kLanes = head_dim / 8 threads hold a head; kRows consecutive rows a CTA: where they go and their angles are found side by
// side, under the loads of the first row's words.
template <class T, int kLanes, int kRows>
__global__ void __launch_bounds__(kAppendThreads, 3) kv_append_kernel(CacheView c, xpkKvAppendArgs a) {
    constexpr int kDim = kLanes * 8;
    constexpr int kAhead = 3;                                   // 16-byte words a thread holds at once
    __shared__ float2 s_turn[kRows][kDim / 2];                  // cos, sin; a thread's are kept apart, so that lanes read side by side
    __shared__ RowPlace s_place[kRows];
    const uint32_t words = (a.q_heads + 2 * c.heads) * kLanes;  // 16-byte words of a row
    const int half = (int)a.rotary / 2;
    const uint32_t row0 = blockIdx.x * kRows;
    auto word = [&](uint32_t row, uint32_t w) {
        const uint4 *x = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.qkv) + (size_t)row * a.qkv_stride);
        return w < words && row < a.rows ? __ldcs(x + w) : make_uint4(0, 0, 0, 0);
    };
    uint4 got[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) got[k] = word(row0, threadIdx.x + k * kAppendThreads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < kRows) {
        const uint32_t row = row0 + warp;
        RowPlace at{-1, -1};
        if (row < a.rows) {
            const int entry = a.starts ? entry_of(a.starts, (int)a.n, (int)row) : (row < a.n ? (int)row : -1);
            if (entry >= 0) {
                const int seq = a.seqs ? a.seqs[entry] : entry;
                const int len = held_by(c, seq);
                const long long pos = a.starts ? (long long)len - a.starts[entry + 1] + (long long)row : (long long)len - 1;
                if (len >= 0 && pos >= 0) {
                    at.pos = pos;
                    at.page = c.table[(size_t)seq * c.width + (pos >> c.page_shift)];
                    if ((uint32_t)at.page >= c.pages) at.page = -1;
                }
            }
        }
        if (lane == 0) s_place[warp] = at;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < half * kRows; i += kAppendThreads) {
        const int r = i / half, j = i - r * half;
        const long long pos = s_place[r].pos;
        if (pos < 0) continue;
        const double t = (double)pos * a.inv_freq[j];
        const double turns = rint(t * 0.15915494309189533577);
        // 2 pi in two parts: turns times the first is exact enough to leave the angle's own rounding as the only error.
        const double left = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586232, t));
        float sn, cs;
        sincosf((float)left, &sn, &cs);
        // A thread turns eight elements: pairs 8 t .. 8 t + 7 of the halves, or the four neighbours' pairs 4 t .. 4 t + 3.
        s_turn[r][a.interleaved ? (j & 3) * (half / 4) + j / 4 : (j & 7) * (half / 8) + j / 8] = make_float2(cs, sn);
    }
    __syncthreads();
    // 256 threads are whole heads: a thread's eight elements lie at the same place of every head it gets, so its turns and its
    // weights are fetched once.
    const int in = (int)(threadIdx.x % kLanes) * 8;
    const bool turned = in < (int)a.rotary, lower = in < half;
    uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
    if (a.q_weight != nullptr) {
        wq = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q_weight) + in);
        wk = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.k_weight) + in);
    }
    const int partner = !turned || a.interleaved ? lane : lane + (lower ? half / 8 : -(half / 8));
#pragma unroll 1
    for (int r = 0; r < kRows; ++r) {
        const uint32_t row = row0 + r;
        const RowPlace at = s_place[r];
        const bool there = at.page >= 0;
        float2 turn[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            turn[i] = make_float2(1.f, 0.f);
            if (turned) turn[i] = a.interleaved ? s_turn[r][(i >> 1) * (half / 4) + in / 8] : s_turn[r][i * (half / 8) + (lower ? in : in - half) / 8];
            if (lower && !a.interleaved) turn[i].y = -turn[i].y;
        }
        T *const q_row = static_cast<T *>(a.q) + (size_t)row * a.q_stride + in;
        const size_t slot = (((((size_t)a.layer * c.pages + max(at.page, 0)) * c.heads) << c.page_shift) + (size_t)(max(at.pos, 0ll) & (c.page - 1))) * kDim + in;
        T *const k_row = reinterpret_cast<T *>(c.k) + slot, *const v_row = reinterpret_cast<T *>(c.v) + slot;
        const uint32_t head_step = (uint32_t)kDim << c.page_shift;       // elements between heads of a page
        for (uint32_t base = 0; base < words; base += kAhead * kAppendThreads) {
            uint4 next[kAhead];                                 // the words after these: of the row, or of the row behind it
            const bool last = base + kAhead * kAppendThreads >= words;
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                next[k] = last && r + 1 == kRows ? make_uint4(0, 0, 0, 0)
                                                 : word(last ? row + 1 : row, (last ? 0 : base + kAhead * kAppendThreads) + threadIdx.x + k * kAppendThreads);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const uint32_t w = base + threadIdx.x + k * kAppendThreads;
                const uint32_t head = w / kLanes;
                const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + c.heads;
                uint4 out = got[k];
                // Every lane of a warp with a query or a key takes part in the shuffles; its other lanes throw their results away.
                if (__any_sync(0xffffffffu, !is_v)) {
                    float f[8];
                    open8<T>(out, f);
                    if (a.q_weight != nullptr) {
                        float sum = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) sum = fmaf(f[i], f[i], sum);
#pragma unroll
                        for (int d = kLanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                        float g[8];
                        open8<T>(is_q ? wq : wk, g);
                        const float s = rsqrtf(sum * (1.f / kDim) + a.eps);
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i] = f[i] * s * g[i];
                    }
                    if (a.interleaved) {
                        if (turned) {
#pragma unroll
                            for (int i = 0; i < 8; i += 2) {
                                const float u = f[i], v = f[i + 1];
                                f[i] = u * turn[i].x - v * turn[i].y;
                                f[i + 1] = v * turn[i].x + u * turn[i].y;
                            }
                        }
                    } else if (half != 0) {
                        // The partner's eight elements are `half / 8` lanes up for the first half, down for the second.
                        float other[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, f[i], partner);
                        if (turned) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) f[i] = fmaf(f[i], turn[i].x, other[i] * turn[i].y);
                        }
                    }
                    if (!is_v) out = close8<T>(f);
                }
                if (w >= words || at.pos < 0) continue;         // the latter the same for the whole CTA
                if (is_q) __stcs(reinterpret_cast<uint4 *>(q_row + (size_t)head * kDim), out);
                else if (there) *reinterpret_cast<uint4 *>((is_v ? v_row + (size_t)(head - a.q_heads - c.heads) * head_step : k_row + (size_t)(head - a.q_heads) * head_step)) = out;
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) got[k] = next[k];
        }
    }
}

template <class T, int kLanes>
static void launch_rows(const CacheView &c, const xpkKvAppendArgs &a, int sms, cudaStream_t st) {
    // Four rows a CTA share one search, one set of look-ups and fill the threads with angles, where there are rows enough for every
    // SM to have several CTAs of them (11,100 rows, 273 MB in and out: 70 us against 84 with one row a CTA); fewer are spread, one a CTA.
    if (a.rows >= (uint32_t)sms * 8) kv_append_kernel<T, kLanes, 4><<<(a.rows + 3) / 4, kAppendThreads, 0, st>>>(c, a);
    else kv_append_kernel<T, kLanes, 1><<<a.rows, kAppendThreads, 0, st>>>(c, a);
}

cudaError_t launch_kv_append(const CacheView &c, const xpkKvAppendArgs &a, bool bf16, int sms, cudaStream_t st) {
    if (bf16 && c.dim == 128) launch_rows<__nv_bfloat16, 16>(c, a, sms, st);
    else if (bf16) launch_rows<__nv_bfloat16, 8>(c, a, sms, st);
    else if (c.dim == 128) launch_rows<__half, 16>(c, a, sms, st);
    else launch_rows<__half, 8>(c, a, sms, st);
    return cudaGetLastError();
}

} // namespace xpk
