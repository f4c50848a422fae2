// The paged key/value cache as kernels see it, and the host object behind xpkKvCache_t.
#pragma once
#include "pk_internal.cuh"

struct xpkKvCache_st {
    xpkKvCacheDesc d;
    int device = 0;
    int sms = 0;
    int32_t *work = nullptr;              // see KvWork
    alignas(64) unsigned char map_k[128], map_v[128];      // boxes of 16 positions x 64 elements
    alignas(64) unsigned char page_k[128], page_v[128];    // boxes of a page (64 positions at most) x 64 elements
};

namespace xpk {

struct CacheView {
    unsigned char *k, *v;
    int32_t *table, *lens, *refs;
    uint32_t layers, pages, heads, page, page_shift, dim, seqs, width;
};

inline CacheView view_of(const xpkKvCache_st *c) {
    const xpkKvCacheDesc &d = c->d;
    uint32_t shift = 0;
    while ((1u << shift) < d.page_size) ++shift;
    return {(unsigned char *)d.k, (unsigned char *)d.v, d.page_table, d.lens, d.refs,
            d.layers, d.pages, d.kv_heads, d.page_size, shift, d.head_dim, d.seqs, d.table_width};
}

// Positions that a sequence holds, never more than its table row can name; -1 for padding.
__device__ __forceinline__ int held_by(const CacheView &c, int seq) {
    if (seq < 0 || (uint32_t)seq >= c.seqs) return -1;
    const long long most = min((long long)c.width << c.page_shift, 0x7fffffffll);
    const int n = c.lens[seq];
    return (int)min((long long)max(n, 0), most);
}
__device__ __forceinline__ int pages_of(const CacheView &c, int n) { return (int)(((long long)n + c.page - 1) >> c.page_shift); }

// The handle's workspace: 16 words (report, exit counter), the fork's decisions, then three arrays of a word per page.
struct KvWork {
    int32_t *report;        // kReport*
    uint32_t *exited;       // CTAs that have left the running fork; 0 between calls
    int32_t *taken;         // [XPK_KV_MAX_LIST] fork: length that child i takes over, 0 = passed over
    int32_t *remap;         // [pages] compact: new id of a page that moves; extend: the free pages it hands out
    int32_t *src, *dst;     // [pages] pages to copy
};
inline size_t kv_work_bytes(uint32_t pages) { return (16 + XPK_KV_MAX_LIST + 3 * (size_t)pages) * sizeof(int32_t); }
inline KvWork kv_work(int32_t *w, uint32_t pages) {
    int32_t *a = w + 16 + XPK_KV_MAX_LIST;
    return {w, (uint32_t *)w + 8, w + 16, a, a + pages, a + 2 * (size_t)pages};
}

constexpr int kReportCopied = 0, kReportMissing = 1, kReportRefused = 2, kReportLive = 3;

} // namespace xpk
