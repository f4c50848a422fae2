// C ABI of the paged key/value cache and its operators (declared in include/xsched_b200/pk.h): checks of arguments, the
// handle, launches.
#include "kv_cache.cuh"

#include <cuda.h>
#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <new>

namespace xpk {
// kv_pages.cu
cudaError_t launch_kv_free(const CacheView &c, const int32_t *seqs, uint32_t n, int sms, cudaStream_t st);
cudaError_t launch_kv_fork(const CacheView &c, const KvWork &w, const int32_t *parents, const int32_t *children, uint32_t n, int sms, cudaStream_t st);
cudaError_t launch_kv_extend(const CacheView &c, const KvWork &w, const int32_t *seqs, const int32_t *tokens, uint32_t n, int sms, cudaStream_t st);
cudaError_t launch_kv_compact(const CacheView &c, const KvWork &w, int sms, cudaStream_t st);
cudaError_t launch_kv_copy(const CacheView &c, const KvWork &w, const int32_t *src, const int32_t *dst, uint32_t n, int sms, cudaStream_t st);
unsigned long long kv_copy_tiles(const CacheView &c, uint32_t n);
// kv_append.cu
cudaError_t launch_kv_append(const CacheView &c, const xpkKvAppendArgs &a, bool bf16, int sms, cudaStream_t st);
// attention.cu
cudaError_t attention_prepare();
size_t attention_scratch_bytes(const CacheView &c, uint32_t sms, uint32_t rows, uint32_t n, uint32_t q_heads);
void attention_counters(const CacheView &c, uint32_t sms, const xpkAttentionArgs &x, void **at, size_t *bytes);
cudaError_t launch_attention(bool preemptible, Ctl *ctl, const xpkKvCache_st *cache, const xpkAttentionArgs &x, unsigned long long launch_no,
                             int grid, cudaStream_t st);
} // namespace xpk

using xpk::DeviceGuard;
using xpk::aligned16;
using xpk::view_of;

namespace {

std::mutex g_kv_mtx;
bool g_attention_ready[64];

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A pool as [layers * pages][kv_heads * page_size][head_dim]; a box is `rows` positions of one page by 64 elements.
bool pool_map(void *out, const xpkKvCacheDesc &d, void *base, uint32_t rows) {
    EncodeTiledFn fn = (EncodeTiledFn)xpk::tensor_map_encoder();
    if (!fn) return false;
    const cuuint64_t dims[3] = {d.head_dim, (cuuint64_t)d.kv_heads * d.page_size, (cuuint64_t)d.layers * d.pages};
    const cuuint64_t strides[2] = {(cuuint64_t)d.head_dim * 2, dims[1] * d.head_dim * 2};
    const cuuint32_t box[3] = {64, rows, 1}, each[3] = {1, 1, 1};
    return fn((CUtensorMap *)out, d.dtype == XPK_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims,
              strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

xpkResult done(cudaError_t e, unsigned launches) {
    if (e != cudaSuccess) return XPK_ERR_CUDA;
    xpk::note_launches(launches);
    return XPK_SUCCESS;
}

// Clears new memory and waits for that alone: streams that do not wait for the default stream may use it once this returns.
bool cleared(void *at, size_t bytes) {
    cudaStream_t st;
    if (cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking) != cudaSuccess) return false;
    const bool ok = cudaMemsetAsync(at, 0, bytes, st) == cudaSuccess && cudaStreamSynchronize(st) == cudaSuccess;
    return cudaStreamDestroy(st) == cudaSuccess && ok;
}

void free_cache(xpkKvCache_st *c) {
    if (c->work) cudaFree(c->work);
    delete c;
}

// The rows of an append or an attention: a dense stride if none is given, 16-byte steps, no overlap of rows.
xpkResult row_stride(uint64_t *stride, uint64_t dense) {
    if (*stride == 0) *stride = dense;
    if (*stride < dense) return XPK_ERR_INVALID_VALUE;
    return *stride % 8 ? XPK_ERR_ALIGNMENT : XPK_SUCCESS;
}

xpkResult check_attention(const xpkKvCache_st *cache, xpkAttentionArgs *x) {
    const xpkKvCacheDesc &d = cache->d;
    if (!x->out || !x->q || !x->scratch || x->n == 0 || x->rows == 0 || x->q_heads == 0 || x->layer >= d.layers) return XPK_ERR_INVALID_VALUE;
    if (!std::isfinite(x->scale)) return XPK_ERR_INVALID_VALUE;
    if (x->q_heads % d.kv_heads) return XPK_ERR_NOT_SUPPORTED;
    if (x->n > XPK_ATTENTION_MAX_SEQS || (uint64_t)x->rows * x->q_heads > 0x7fffffffull) return XPK_ERR_TOO_LARGE;
    if (!aligned16(x->out) || !aligned16(x->q) || (reinterpret_cast<uintptr_t>(x->scratch) & 255u)) return XPK_ERR_ALIGNMENT;
    if (!aligned4(x->seqs) || !aligned4(x->starts) || !aligned4(x->shared_len)) return XPK_ERR_ALIGNMENT;
    xpkResult r = row_stride(&x->q_stride, (uint64_t)x->q_heads * d.head_dim);
    if (r == XPK_SUCCESS) r = row_stride(&x->out_stride, (uint64_t)x->q_heads * d.head_dim);
    if (r != XPK_SUCCESS) return r;
    if (x->scratch_bytes < xpk::attention_scratch_bytes(view_of(cache), cache->sms, x->rows, x->n, x->q_heads)) return XPK_ERR_INVALID_VALUE;
    return XPK_SUCCESS;
}

xpkResult attention_ready(int device) {
    std::lock_guard<std::mutex> lk(g_kv_mtx);
    if (device < 0 || device >= 64) return XPK_ERR_CUDA;
    if (!g_attention_ready[device]) {
        if (xpk::attention_prepare() != cudaSuccess) return XPK_ERR_CUDA;
        g_attention_ready[device] = true;
    }
    return XPK_SUCCESS;
}

} // namespace

extern "C" {

xpkResult xpkKvCacheCreate(xpkKvCache_t *cache, const xpkKvCacheDesc *desc) {
    if (!cache || !desc) return XPK_ERR_INVALID_VALUE;
    const xpkKvCacheDesc &d = *desc;
    if (!d.k || !d.v || !d.page_table || !d.lens || !d.refs) return XPK_ERR_INVALID_VALUE;
    if (d.layers == 0 || d.pages == 0 || d.kv_heads == 0 || d.seqs == 0 || d.table_width == 0) return XPK_ERR_INVALID_VALUE;
    if (d.dtype != XPK_DTYPE_BF16 && d.dtype != XPK_DTYPE_F16) return XPK_ERR_NOT_SUPPORTED;
    if (d.page_size != 16 && d.page_size != 32 && d.page_size != 64 && d.page_size != 128) return XPK_ERR_NOT_SUPPORTED;
    if (d.head_dim != 64 && d.head_dim != 128) return XPK_ERR_NOT_SUPPORTED;
    // Positions, page ids, pages over all layers and the units of a page over all layers are 32-bit signed in the kernels.
    if (d.pages > 0x7ffffff0u || (uint64_t)d.layers * d.pages > 0x7fffffffull || d.seqs > 0x7fffffffu || d.kv_heads > 65536u ||
        (uint64_t)d.table_width * d.page_size > (1ull << 30) ||
        (uint64_t)d.layers * d.kv_heads * d.page_size * d.head_dim * 4 / 2048 > 0x7fffffffull) return XPK_ERR_TOO_LARGE;
    if (!aligned16(d.k) || !aligned16(d.v)) return XPK_ERR_ALIGNMENT;
    if (!aligned4(d.page_table) || !aligned4(d.lens) || !aligned4(d.refs)) return XPK_ERR_ALIGNMENT;
    xpkKvCache_st *c = new (std::nothrow) xpkKvCache_st();
    if (!c) return XPK_ERR_CUDA;
    c->d = d;
    c->sms = xpk::device_sms();
    if (c->sms == 0 || cudaGetDevice(&c->device) != cudaSuccess) { free_cache(c); return XPK_ERR_CUDA; }
    const size_t bytes = xpk::kv_work_bytes(d.pages);
    if (cudaMalloc((void **)&c->work, bytes) != cudaSuccess || !cleared(c->work, bytes)) { free_cache(c); return XPK_ERR_CUDA; }
    if (!pool_map(c->map_k, d, d.k, 16) || !pool_map(c->map_v, d, d.v, 16) ||
        !pool_map(c->page_k, d, d.k, std::min(d.page_size, 64u)) || !pool_map(c->page_v, d, d.v, std::min(d.page_size, 64u))) { free_cache(c); return XPK_ERR_CUDA; }
    const xpkResult r = attention_ready(c->device);
    if (r != XPK_SUCCESS) { free_cache(c); return r; }
    *cache = c;
    return XPK_SUCCESS;
}

xpkResult xpkKvCacheDestroy(xpkKvCache_t cache) {
    if (!cache) return XPK_ERR_INVALID_VALUE;
    DeviceGuard on_device(cache->device);
    free_cache(cache);
    return XPK_SUCCESS;
}

xpkResult xpkKvFree(xpkKvCache_t cache, const int32_t *seqs, uint32_t n, void *stream) {
    if (!cache || !seqs || n == 0) return XPK_ERR_INVALID_VALUE;
    if (!aligned4(seqs)) return XPK_ERR_ALIGNMENT;
    DeviceGuard on_device(cache->device);
    return done(xpk::launch_kv_free(view_of(cache), seqs, n, cache->sms, (cudaStream_t)stream), 1);
}

xpkResult xpkKvFork(xpkKvCache_t cache, const int32_t *parents, const int32_t *children, uint32_t n, void *stream) {
    if (!cache || !parents || !children || n == 0) return XPK_ERR_INVALID_VALUE;
    if (n > XPK_KV_MAX_LIST) return XPK_ERR_TOO_LARGE;
    if (!aligned4(parents) || !aligned4(children)) return XPK_ERR_ALIGNMENT;
    DeviceGuard on_device(cache->device);
    return done(xpk::launch_kv_fork(view_of(cache), xpk::kv_work(cache->work, cache->d.pages), parents, children, n, cache->sms, (cudaStream_t)stream), 1);
}

xpkResult xpkKvExtend(xpkKvCache_t cache, const int32_t *seqs, const int32_t *tokens, uint32_t n, void *stream) {
    if (!cache || !seqs || !tokens || n == 0) return XPK_ERR_INVALID_VALUE;
    if (n > XPK_KV_MAX_LIST) return XPK_ERR_TOO_LARGE;
    if (!aligned4(seqs) || !aligned4(tokens)) return XPK_ERR_ALIGNMENT;
    DeviceGuard on_device(cache->device);
    return done(xpk::launch_kv_extend(view_of(cache), xpk::kv_work(cache->work, cache->d.pages), seqs, tokens, n, cache->sms, (cudaStream_t)stream), 2);
}

xpkResult xpkKvCompact(xpkKvCache_t cache, void *stream) {
    if (!cache) return XPK_ERR_INVALID_VALUE;
    DeviceGuard on_device(cache->device);
    return done(xpk::launch_kv_compact(view_of(cache), xpk::kv_work(cache->work, cache->d.pages), cache->sms, (cudaStream_t)stream), 2);
}

xpkResult xpkKvCopy(xpkKvCache_t cache, const int32_t *src, const int32_t *dst, uint32_t n, void *stream) {
    if (!cache || !src || !dst || n == 0) return XPK_ERR_INVALID_VALUE;
    if (!aligned4(src) || !aligned4(dst)) return XPK_ERR_ALIGNMENT;
    DeviceGuard on_device(cache->device);
    return done(xpk::launch_kv_copy(view_of(cache), xpk::kv_work(cache->work, cache->d.pages), src, dst, n, cache->sms, (cudaStream_t)stream), 1);
}

xpkResult xpkTaskCreateKvCopy(xpkTask_t *task, xpkKvCache_t cache, const int32_t *src, const int32_t *dst, uint32_t n, uint32_t flags,
                              uint32_t *flag_dev) {
    if (!task || !cache || !src || !dst || n == 0) return XPK_ERR_INVALID_VALUE;
    if (!aligned4(src) || !aligned4(dst)) return XPK_ERR_ALIGNMENT;
    DeviceGuard on_device(cache->device);
    xpkTask_st *t = new (std::nothrow) xpkTask_st();
    if (!t) return XPK_ERR_CUDA;
    const xpkResult r = xpk::task_common(t, XPK_KIND_KV_COPY, flags, xpk::kv_copy_tiles(view_of(cache), n), flag_dev);
    if (r != XPK_SUCCESS) { xpk::task_free(t); return r; }
    t->cache = cache;
    t->p1 = src; t->p2 = dst; t->n = n;
    *task = t;
    return XPK_SUCCESS;
}

xpkResult xpkKvResult(xpkKvCache_t cache, xpkKvReport *report, void *stream) {
    if (!cache || !report) return XPK_ERR_INVALID_VALUE;
    DeviceGuard on_device(cache->device);
    if (cudaMemcpyAsync(report, cache->work, sizeof(*report), cudaMemcpyDeviceToHost, (cudaStream_t)stream) != cudaSuccess) return XPK_ERR_CUDA;
    return cudaStreamSynchronize((cudaStream_t)stream) == cudaSuccess ? XPK_SUCCESS : XPK_ERR_CUDA;
}

xpkResult xpkKvAppend(xpkKvCache_t cache, const xpkKvAppendArgs *args, void *stream) {
    if (!cache || !args) return XPK_ERR_INVALID_VALUE;
    xpkKvAppendArgs a = *args;
    const xpkKvCacheDesc &d = cache->d;
    if (!a.q || !a.qkv || a.n == 0 || a.rows == 0 || a.q_heads == 0 || a.layer >= d.layers) return XPK_ERR_INVALID_VALUE;
    if (a.rotary != 0 && !a.inv_freq) return XPK_ERR_INVALID_VALUE;
    if (a.rotary % 16 || a.rotary > d.head_dim || (a.q_weight == nullptr) != (a.k_weight == nullptr)) return XPK_ERR_NOT_SUPPORTED;
    if (a.q_weight && !(a.eps >= 0.f && std::isfinite(a.eps))) return XPK_ERR_INVALID_VALUE;
    if (a.rows > 0x7fffffffu || a.n > 0x7fffffffu || a.q_heads > 65536u) return XPK_ERR_TOO_LARGE;
    if (!aligned16(a.q) || !aligned16(a.qkv) || !aligned16(a.q_weight) || !aligned16(a.k_weight)) return XPK_ERR_ALIGNMENT;
    if (!aligned4(a.seqs) || !aligned4(a.starts) || (reinterpret_cast<uintptr_t>(a.inv_freq) & 7u)) return XPK_ERR_ALIGNMENT;
    xpkResult r = row_stride(&a.q_stride, (uint64_t)a.q_heads * d.head_dim);
    if (r == XPK_SUCCESS) r = row_stride(&a.qkv_stride, ((uint64_t)a.q_heads + 2 * d.kv_heads) * d.head_dim);
    if (r != XPK_SUCCESS) return r;
    DeviceGuard on_device(cache->device);
    return done(xpk::launch_kv_append(view_of(cache), a, d.dtype == XPK_DTYPE_BF16, cache->sms, (cudaStream_t)stream), 1);
}

size_t xpkAttentionScratchBytes(xpkKvCache_t cache, uint32_t rows, uint32_t n, uint32_t q_heads) {
    if (!cache) return 0;
    return xpk::attention_scratch_bytes(view_of(cache), cache->sms, rows, n, q_heads);
}

xpkResult xpkAttention(xpkKvCache_t cache, const xpkAttentionArgs *args, void *stream) {
    if (!cache || !args) return XPK_ERR_INVALID_VALUE;
    xpkAttentionArgs x = *args;
    const xpkResult r = check_attention(cache, &x);
    if (r != XPK_SUCCESS) return r;
    DeviceGuard on_device(cache->device);
    return done(xpk::launch_attention(false, nullptr, cache, x, 0, cache->sms, (cudaStream_t)stream), 1);
}

xpkResult xpkTaskCreateAttention(xpkTask_t *task, xpkKvCache_t cache, const xpkAttentionArgs *args, uint32_t flags, uint32_t *flag_dev) {
    if (!task || !cache || !args) return XPK_ERR_INVALID_VALUE;
    xpkAttentionArgs x = *args;
    xpkResult r = check_attention(cache, &x);
    if (r != XPK_SUCCESS) return r;
    DeviceGuard on_device(cache->device);
    xpkTask_st *t = new (std::nothrow) xpkTask_st();
    if (!t) return XPK_ERR_CUDA;
    // How many tiles there are is known once a launch has read the lengths; until then: not complete.
    r = xpk::task_common(t, XPK_KIND_ATTENTION, flags, 1, flag_dev);
    if (r == XPK_SUCCESS) {
        t->cache = cache;
        t->attention = x;
        xpk::attention_counters(view_of(cache), cache->sms, x, &t->clear_at, &t->clear_bytes);
        // Once here, waited for, and once by the first launch on its own stream: what used the memory before may be queued there still.
        if (cudaMemset(t->clear_at, 0, t->clear_bytes) != cudaSuccess || cudaStreamSynchronize(cudaStreamLegacy) != cudaSuccess) r = XPK_ERR_CUDA;
        t->clear_first = true;
    }
    if (r != XPK_SUCCESS) { xpk::task_free(t); return r; }
    *task = t;
    return XPK_SUCCESS;
}

} // extern "C"
