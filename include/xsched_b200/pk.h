/*
 * pk.h — C ABI of the preemptible persistent-kernel library (libxpk.so) for sm_100a.
 *
 * This is the device-side half of XSched's Level-2 ("deactivate") preemption on B200.
 * The reference obtains Level-2 by patching a guardian prologue into every application
 * kernel (platforms/cuda/hal/src/level2/instrument.cpp:15-231,
 * platforms/cuda/hal/inject/inject.cu:43-140): each thread block checks a global exit
 * flag, records exit/restore flags per block, and the host relaunches from `preempt_idx`
 * (platforms/cuda/hal/src/level2/cuda_queue.cpp:29-41).  That guardian exists only as
 * sm35/sm70/sm86 machine code (platforms/cuda/hal/src/arch/arch.cpp:26-39), so on B200 the
 * reference has no Level-2 at all.  Here the same contract is provided cooperatively:
 * every kernel below is persistent, claims its work tile by tile, polls a device-visible
 * preempt flag at each tile boundary, and on preemption leaves a resumable cursor in a
 * control block.  Relaunching the same task continues from the cursor; the output of a
 * task preempted and resumed any number of times is bit-identical to an unpreempted run.
 *
 * All entry points take plain pointers and sizes.  Device pointers are raw CUDA device
 * addresses; streams are CUstream/cudaStream_t passed as void*.  Every function returns
 * an xpkResult; nothing here allocates behind the caller's back except xpkTaskCreate*
 * (one device control block of about 16.6 KB — claim state plus two lists of handed-back
 * tiles — and one 64-byte mapped host mailbox per task).
 */
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    XPK_SUCCESS            = 0,
    XPK_ERR_INVALID_VALUE  = 1,  /* null pointer, zero size, bad shape            */
    XPK_ERR_ALIGNMENT      = 2,  /* a device pointer is not 16-byte aligned       */
    XPK_ERR_CUDA           = 3,  /* a CUDA runtime/driver call failed             */
    XPK_ERR_NOT_SUPPORTED  = 4,  /* shape outside what the kernel was built for   */
    XPK_ERR_BUSY           = 5,  /* task still in flight                          */
    XPK_ERR_DEVICE_TIMEOUT = 6,  /* a bounded device-side wait gave up            */
    XPK_ERR_TOO_LARGE      = 7,  /* exceeds a static capacity                     */
} xpkResult;

/* Task status as published by the kernel in the mailbox. */
typedef enum {
    XPK_STATUS_IDLE      = 0,  /* created or reset, never launched                 */
    XPK_STATUS_RUNNING   = 1,  /* launched, final CTA has not yet published        */
    XPK_STATUS_COMPLETED = 2,  /* every tile done                                   */
    XPK_STATUS_PREEMPTED = 3,  /* stopped on the preempt flag; cursor is resumable */
    XPK_STATUS_ERROR     = 4,  /* a bounded wait expired; output undefined         */
} xpkStatus;

typedef enum {
    XPK_KIND_TRIAD  = 1,  /* a[i] = fmaf(s, c[i], b[i]), fp32, 128-bit accesses   */
    XPK_KIND_VECADD = 2,  /* c[i] = a[i] + b[i], fp32                              */
    XPK_KIND_SORT   = 3,  /* int32 ascending LSD radix sort, 8-bit digits          */
    XPK_KIND_GEMM   = 4,  /* bf16 C[M,N] = A[M,K] * B[N,K]^T, fp32 accumulate      */
    XPK_KIND_ATTENTION = 5, /* attention over a paged key/value cache              */
    XPK_KIND_KV_COPY = 6, /* copies of pages of a key/value cache                  */
} xpkKind;

/* Launch-time flags for xpkTaskCreate*. */
enum {
    XPK_FLAG_NONE           = 0,
    XPK_FLAG_NON_PREEMPTIBLE = 1, /* the twin: same tile loop and the same ticket claim, the
                                     preempt flag never read.  For kernels nothing needs to
                                     stop, and to measure what the check costs.            */
    XPK_FLAG_ABORT_INFLIGHT = 2, /* GEMM only: on preemption abandon tiles whose main
                                     loop is still running and recompute them on resume
                                     (keeps the preemption latency below one tile).     */
    XPK_FLAG_GEMM_ONE_CTA   = 4, /* GEMM only: run the form in which one CTA owns a 256x256
                                     tile (tcgen05 .cta_group::1).                         */
    XPK_FLAG_GEMM_CTA_PAIR  = 8, /* GEMM only: run the form in which the two SMs of a TPC
                                     share a 256x256 tile (tcgen05 .cta_group::2).  With
                                     neither flag the library chooses (XPK_GEMM_FORM=one|pair
                                     in the environment overrides its choice).  Both forms
                                     write the same bytes.                                 */
};

typedef struct xpkTask_st *xpkTask_t;

/* Snapshot returned by xpkTaskQuery; mirrors the mailbox the final CTA writes. */
typedef struct {
    uint32_t status;       /* xpkStatus                                             */
    uint32_t error;        /* 0, or a kernel-specific code naming the wait that expired */
    uint64_t tiles_done;   /* tiles completed over the task's life (the cursor)     */
    uint64_t tiles_total;  /* tiles in the task                                     */
    uint64_t launches;     /* kernel launches issued for this task since reset      */
    uint64_t preemptions;  /* launches that ended PREEMPTED                         */
} xpkTaskInfo;

/* ---- library / device --------------------------------------------------------------- */

/* Number of SMs of the current device (the persistent grids are sized from it). */
xpkResult xpkDeviceSmCount(int *sm_count);
const char *xpkResultString(xpkResult r);

/* ---- preempt flag -------------------------------------------------------------------
 * A flag is one 32-bit word in device memory.  One flag is normally shared by all tasks
 * of one hardware queue (that is what HwQueue::Deactivate raises — reference contract
 * preempt/include/xsched/preempt/hal/hw_queue.h:36-44).  Raise/clear are enqueued as a
 * 32-bit stream memory write on `ctrl_stream`, which should not be the stream the
 * persistent kernel occupies.                                                          */
xpkResult xpkFlagCreate(uint32_t **flag_dev);
xpkResult xpkFlagDestroy(uint32_t *flag_dev);
xpkResult xpkFlagSet(uint32_t *flag_dev, uint32_t value, void *ctrl_stream);
/* A stream write needs 6-14 us to reach device memory.  A flag (256 bytes from xpkFlagCreate, or any zeroed
 * 16-byte-aligned block whose first word is the flag) can be given an early-warning word in mapped host memory:
 * the caller stores a non-zero value there (a plain host store, on the GPU within about 2 us) immediately before
 * xpkFlagSet(flag, 1, ..), and zero before lowering the flag.  Kernels that run a relay (the GEMM, the triad and the vector add) copy the raised
 * word into the flag; every kernel still honours the flag itself.  The word is freed with the flag's owner
 * calling xpkFlagDetachRelay.                                                                          */
xpkResult xpkFlagAttachRelay(uint32_t *flag_dev, volatile uint32_t **relay_host);
xpkResult xpkFlagDetachRelay(uint32_t *flag_dev, volatile uint32_t *relay_host);

/* ---- task creation ------------------------------------------------------------------
 * `flag_dev` may be NULL: the task then owns a private flag (see xpkTaskFlag).
 * `tile_elems`/tile shape 0 selects the default.                                        */

/* a = b + s*c computed as one fused multiply-add per element.  n in elements. */
xpkResult xpkTaskCreateTriad(xpkTask_t *task, float *a, const float *b, const float *c,
                             float s, uint64_t n, uint32_t tile_elems, uint32_t flags,
                             uint32_t *flag_dev);

/* c = a + b. */
xpkResult xpkTaskCreateVecAdd(xpkTask_t *task, float *c, const float *a, const float *b,
                              uint64_t n, uint32_t tile_elems, uint32_t flags,
                              uint32_t *flag_dev);

/* Ascending sort of n int32 keys.  `keys` holds the input and, after completion, the
 * sorted output (4 passes: the data ends in the buffer it started in).  `tmp` is a
 * caller-provided buffer of n keys.  `scratch` is caller-provided device memory of at
 * least xpkSortScratchBytes(n) bytes, 256-byte aligned; the library clears what it needs. */
size_t    xpkSortScratchBytes(uint64_t n);
xpkResult xpkTaskCreateSort(xpkTask_t *task, int32_t *keys, int32_t *tmp, void *scratch,
                            uint64_t n, uint32_t flags, uint32_t *flag_dev);

/* bf16 GEMM, C[M,N] (row-major, bf16) = A[M,K] (row-major) * B[N,K]^T (row-major, i.e.
 * both operands K-major), fp32 accumulation in tensor memory.  M % 128 == 0,
 * N % 256 == 0, K % 64 == 0.  A tile (the unit of xpkTaskInfo.tiles_*) is 512x256 in the
 * pair form and 256x256 in the one-CTA form (XPK_FLAG_GEMM_*); the pair form launches whole
 * pairs of CTAs (an `sm_limit` is rounded down to an even number, at least 2).           */
xpkResult xpkTaskCreateGemm(xpkTask_t *task, void *C, const void *A, const void *B,
                            uint32_t M, uint32_t N, uint32_t K, uint32_t flags,
                            uint32_t *flag_dev);

/* ---- task control ------------------------------------------------------------------- *
 * A task belongs to the device that was current when it was created.  xpkTaskLaunch,
 * xpkTaskReset and xpkTaskDestroy (and xpkFlagSet, for the flag's device) make that device
 * current for the duration of the call and restore the caller's, so they may be called
 * from any thread; `stream` must be a stream of the task's device.                       */

/* Enqueue the task's kernel on `stream`.  A fresh or reset task starts at tile 0; a
 * PREEMPTED task continues from its cursor; a COMPLETED task has re-armed itself and runs
 * again from tile 0 (callers whose inputs changed in place, like the sort's keys, restore them
 * first).  Never blocks.  `sm_limit` > 0 caps the persistent grid to that many SMs (0 = all).          */
xpkResult xpkTaskLaunch(xpkTask_t task, void *stream, int sm_limit);

/* Read the mailbox (mapped host memory; no CUDA call, no synchronisation). */
xpkResult xpkTaskQuery(xpkTask_t task, xpkTaskInfo *info);

/* Spin (with back-off) on the mailbox until the launch issued most recently has
 * published COMPLETED, PREEMPTED or ERROR, or `timeout_us` elapses (XPK_ERR_BUSY).      */
xpkResult xpkTaskWait(xpkTask_t task, uint64_t timeout_us, xpkTaskInfo *info);

/* Device-clock stamps (%globaltimer, nanoseconds) of the launch whose result the mailbox holds: when its
 * first CTA started and when its last CTA left.  For latency break-downs; XPK_ERR_BUSY before any launch
 * has published.  The GPU clock is not the host's: callers calibrate an offset themselves.            */
xpkResult xpkTaskTimes(xpkTask_t task, uint64_t *start_ns, uint64_t *exit_ns);

/* Rewind the cursor to tile 0 (enqueued on `stream`, ordered after prior work on it).  Costs nothing on the
 * device for a task that was never launched or has completed; the sort's scratch is cleared in any case. */
xpkResult xpkTaskReset(xpkTask_t task, void *stream);

/* The flag this task polls (its own, or the shared one given at creation). */
xpkResult xpkTaskFlag(xpkTask_t task, uint32_t **flag_dev);
xpkResult xpkTaskKind(xpkTask_t task, uint32_t *kind);
xpkResult xpkTaskDestroy(xpkTask_t task);

/* ---- sorting without any allocation ---------------------------------------------------
 * (No counterpart in the reference, which has no sort kernel and no allocation-free entry points.)
 *
 * For callers that cannot allocate device or pinned memory at the point where they need a sort —
 * code running while a memory pool is frozen, a plugin that was handed two buffers and a stream and
 * nothing else, a latency-critical section where cudaMalloc's implicit device synchronisation is not
 * acceptable.  xpkTaskCreateSort needs a control block, a mailbox and caller-provided scratch; this
 * entry point needs none of them: its control block, digit histograms and look-back words live in a
 * fixed array inside the library's device image (about 4.2 MB, held by every GPU that loads the
 * library until the process exits).
 *
 * Sorts `n` int32 keys ascending, in place in `keys`, using `tmp` (n keys) as the second buffer, on
 * `stream`; asynchronous, the result is ready when the stream reaches this point.  Not preemptible.
 *   - n > XPK_SORT_NOALLOC_MAX_KEYS  -> XPK_ERR_TOO_LARGE; keys/tmp must be 16-byte aligned.
 *   - Calls no cudaMalloc/cudaFree/cudaHostAlloc and no library routine that allocates.
 *   - The first call on each device resolves the array's address (cudaGetSymbolAddress) and sets a
 *     kernel attribute; make that first call outside any stream capture.
 *   - `stream` must be a stream of the device that is current in the calling thread: the array
 *     that is used is the current device's copy.
 *   - There is no status channel: a bounded wait inside the kernel that gives up (none has been
 *     seen to) leaves the keys unsorted and is not reported; callers that need a status use the
 *     task form (xpkTaskCreateSort / xpkTaskWait).
 *   - All calls on one device share the one array.  It keeps the previous call's contents (the entry
 *     point clears what it needs), and two calls whose kernels overlap on the GPU — different
 *     streams, or different host threads without ordering between their streams — race on it:
 *     serialise them.                                                                      */
#define XPK_SORT_NOALLOC_MAX_KEYS (4ull << 20)
xpkResult xpkSortNoAlloc(int32_t *keys, int32_t *tmp, uint64_t n, void *stream);

/* ---- paged key/value cache -------------------------------------------------------------
 * (No counterpart in the reference, which has no model kernels.)
 *
 * The operators of a decode loop around one cache: room for new tokens, forks that share pages, copies, compaction;
 * the norms, rotation and write of new queries, keys and values; the attention that reads them, with a prefix that a
 * batch shares read once for all.  The arrays belong to the caller and stay where they are for the cache's life:
 *
 *   k, v        [layers][pages][kv_heads][page_size][head_dim], bf16 or fp16, 16-byte aligned
 *   page_table  [seqs][table_width] page ids, position p of a sequence lies on entry p / page_size
 *   lens        [seqs] positions that a sequence holds (0 = the slot is free)
 *   refs        [pages] how many table entries name a page (0 = the page is free)
 *
 * page_size is 16, 32, 64 or 128, head_dim 64 or 128, table_width * page_size at most 2^30.  The three integer arrays live on the device, and every call
 * reads what they hold when its kernels run, so a loop can be captured once and replayed while lengths grow.  Page ids
 * and sequence ids are checked by the kernels: a sequence outside [0, seqs) is padding and is passed over, a page
 * outside [0, pages) is treated as not there (never read, never written).
 *
 * Calls are asynchronous on `stream`, a stream of the cache's device (the device current at creation), which is made
 * current for the call.  Calls on one cache share the handle's workspace (fork, extend, compact) and the arrays above:
 * those that change them are ordered by the caller, on one stream or by events.                                    */
typedef enum {
    XPK_DTYPE_BF16 = 1,
    XPK_DTYPE_F16  = 2,
} xpkDtype;

typedef struct xpkKvCache_st *xpkKvCache_t;

typedef struct {
    void *k, *v;
    int32_t *page_table, *lens, *refs;
    uint32_t dtype;                                   /* xpkDtype */
    uint32_t layers, pages, kv_heads, page_size, head_dim, seqs, table_width;
} xpkKvCacheDesc;

/* Checks the description and allocates the handle's workspace (12 bytes per page and 8 KB on the device). */
xpkResult xpkKvCacheCreate(xpkKvCache_t *cache, const xpkKvCacheDesc *desc);
/* Tasks created on the cache go first. */
xpkResult xpkKvCacheDestroy(xpkKvCache_t cache);

/* At most this many entries in the lists of fork and extend. */
#define XPK_KV_MAX_LIST 2048

/* The listed sequences give their pages back and are empty afterwards (lens 0, their table entries -1).  A sequence
 * listed twice, and one that is empty, is passed over. */
xpkResult xpkKvFree(xpkKvCache_t cache, const int32_t *seqs, uint32_t n, void *stream);

/* children[i] becomes a copy of parents[i] that shares its pages (no page is copied here; extend copies the last one
 * when one of its holders grows).  A child has to be empty before the call: entries with a child that is not, with an
 * empty parent, or with a child that an earlier entry has taken are passed over. */
xpkResult xpkKvFork(xpkKvCache_t cache, const int32_t *parents, const int32_t *children, uint32_t n, void *stream);

/* Makes room for tokens[i] more positions of seqs[i] and adds them to lens.  New pages are the free ones of lowest
 * index, in the order of the list; a last page that is partly filled and that others hold too is copied (all layers)
 * to a new page first, except by the list's last holder once nobody else is left.  A sequence counts once, at its first
 * place in the list.  All or nothing: if pages are missing, or a sequence would pass the table's width, nothing changes;
 * xpkKvResult tells. */
xpkResult xpkKvExtend(xpkKvCache_t cache, const int32_t *seqs, const int32_t *tokens, uint32_t n, void *stream);

/* Moves the live pages of highest index into the holes below them until the pages in use are [0, live), ascending to
 * ascending, and rewrites table and refs.  Only the first ceil(lens / page_size) entries of a table row are looked at. */
xpkResult xpkKvCompact(xpkKvCache_t cache, void *stream);

/* Copies page src[i] to page dst[i] in all layers.  No page may be in both lists, or twice in dst. */
xpkResult xpkKvCopy(xpkKvCache_t cache, const int32_t *src, const int32_t *dst, uint32_t n, void *stream);
/* The same as a preemptible task; a tile is 64 KB. */
xpkResult xpkTaskCreateKvCopy(xpkTask_t *task, xpkKvCache_t cache, const int32_t *src, const int32_t *dst, uint32_t n,
                              uint32_t flags, uint32_t *flag_dev);

/* What the last extend or compact found, read back on `stream` (which it waits for). */
typedef struct {
    int32_t copied;    /* pages copied (extend) or moved (compact)                          */
    int32_t missing;   /* extend: pages short; nothing was changed when not 0              */
    int32_t refused;   /* extend: sequences that would pass the table's width (as above)   */
    int32_t live;      /* compact: pages in use                                             */
} xpkKvReport;
xpkResult xpkKvResult(xpkKvCache_t cache, xpkKvReport *report, void *stream);

/* Norms, rotation and write of new tokens, one pass over the rows of a projection.
 *
 * Row r of `qkv` holds q_heads queries, kv_heads keys and kv_heads values of head_dim elements each.  The rows
 * starts[i] .. starts[i+1] (ascending, starts[n] at most `rows`) are the last ones of sequence seqs[i] (after extend): row j of t has
 * position lens - t + j.  A sequence is listed once: of two entries, either one's keys and values may be what stays.  Queries and keys are divided by their root mean square over the head (eps added to the mean) and
 * multiplied by q_weight / k_weight [head_dim], in fp32 (NULL: no norm); then the first `rotary` elements are turned by
 * position * inv_freq[j] (angles in fp64): the pairs are (j, j + rotary / 2), or (2j, 2j + 1) with `interleaved`; one
 * rounding at the end.  Queries go to `q` [rows][q_heads][head_dim], keys and values to the cache's `layer`.
 * Rows of padded sequences, rows before position 0 and rows behind starts[n] stay as they are.  A key whose page is
 * missing is not written. */
typedef struct {
    void *q;
    const void *qkv;
    uint64_t q_stride, qkv_stride;      /* elements between rows; 0 = dense, else a multiple of 8                  */
    const int32_t *seqs;                /* [n]; NULL: sequence i                                                  */
    const int32_t *starts;              /* [n + 1] ascending; NULL: one row per sequence                          */
    const void *q_weight, *k_weight;
    const double *inv_freq;             /* [rotary / 2] on the device                                             */
    float eps;
    uint32_t n, rows, q_heads, layer, rotary, interleaved;   /* rotary: a multiple of 16 up to head_dim, 0 = none */
} xpkKvAppendArgs;
xpkResult xpkKvAppend(xpkKvCache_t cache, const xpkKvAppendArgs *args, void *stream);

/* Attention of the rows of `q` (laid out and assigned to sequences as above) to the positions of their own sequences
 * up to and with their own: out = softmax(scale * q k^T) v.  Scores, maxima, sums and accumulators are fp32; the weights are rounded
 * to the cache's type before they meet v, and the result once at the end.  Query heads h * q_heads / kv_heads ... read key head h.
 * A sequence may be listed more than once.
 *
 * `shared_len` (one word on the device, or NULL) promises that the first so many positions lie on the same pages in
 * all sequences of the call that are longer than that; those pages are then read once for all instead of once per
 * sequence.  The result is the one without it up to rounding.  A row that sees nothing is written as zeros; rows of
 * padded sequences and behind starts[n] stay as they are.
 *
 * `scratch`: xpkAttentionScratchBytes bytes, 256-byte aligned, zeroed once before its first use; a call leaves it ready
 * for the next one on the same cache, whatever its sizes.  Calls that may overlap on the GPU (other streams, other captured graphs)
 * need scratch of their own.
 * A call that was refused wrote nothing.  The call has no status channel: a bounded wait inside the kernel that gives up leaves
 * `out` undefined (the task form reports it).  n <= XPK_ATTENTION_MAX_SEQS. */
#define XPK_ATTENTION_MAX_SEQS 1024
typedef struct {
    void *out;
    const void *q;
    uint64_t out_stride, q_stride;      /* elements between rows; 0 = dense, else a multiple of 8                  */
    const int32_t *seqs, *starts;
    const int32_t *shared_len;
    void *scratch;
    uint64_t scratch_bytes;
    float scale;
    uint32_t n, rows, q_heads, layer;
} xpkAttentionArgs;
size_t    xpkAttentionScratchBytes(xpkKvCache_t cache, uint32_t rows, uint32_t n, uint32_t q_heads);
xpkResult xpkAttention(xpkKvCache_t cache, const xpkAttentionArgs *args, void *stream);
/* The same as a preemptible task.  Its scratch is its own; what has to be zero in it is cleared here and, unless that launch is
 * captured, by the first launch on its stream.  A stop takes effect between tickets: a run of positions for up to 256 rows that is under
 * way, and the one or two claimed behind it, are finished first, which takes longer the longer the context is (0.15 ms at a prefix of
 * 16384, 2.4 ms for a prompt on 131072 positions).  XPK_FLAG_ABORT_INFLIGHT has no effect.  Lengths and tables are not to change between a
 * launch that was preempted and the one that finishes it. */
xpkResult xpkTaskCreateAttention(xpkTask_t *task, xpkKvCache_t cache, const xpkAttentionArgs *args, uint32_t flags,
                                 uint32_t *flag_dev);

/* Kernels launched by this library in this process since load (all tasks, the sort kernels of xpkSortNoAlloc, and
 * the cache's calls). */
uint64_t xpkLaunchCount(void);

#ifdef __cplusplus
}
#endif
