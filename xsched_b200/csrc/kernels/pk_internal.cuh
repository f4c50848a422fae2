// Host-side pieces shared by the files that implement the C ABI (pk_api.cu: tasks; kv_api.cu: the paged key/value
// cache): the task object, the per-call device switch and the task's common part.
#pragma once
#include "xsched_b200/pk.h"
#include "pk_common.cuh"

#include <atomic>

struct xpkTask_st {
    uint32_t kind = 0;
    uint32_t flags = 0;
    int device = 0;
    int sm_count = 0;
    xpk::Ctl *ctl = nullptr;               // device
    xpk::Mailbox *mb_host = nullptr;       // mapped pinned host memory
    xpk::Mailbox *mb_dev = nullptr;        // device alias
    uint32_t *flag = nullptr;         // flag the kernels poll
    unsigned long long total = 0;
    // Written by whichever thread launches or resets the task (an XQueue worker, the scheduler's thread on a
    // relaunch), read by application threads in xpkTaskQuery / xpkTaskWait.
    std::atomic<unsigned long long> launches{0};        // launch counter echoed by the mailbox
    std::atomic<unsigned long long> reset_at{0};        // value of `launches` at the last reset
    std::atomic<cudaStream_t> last_stream{nullptr};     // stream of the most recent launch
    // operands
    void *p0 = nullptr; const void *p1 = nullptr; const void *p2 = nullptr;
    float s = 0.f;
    unsigned long long n = 0;
    unsigned long long tile_elems = 0;
    uint32_t *sort_hist = nullptr, *sort_state = nullptr;
    size_t sort_scratch_bytes = 0;
    uint32_t M = 0, N = 0, K = 0;
    bool gemm_pair = false;           // the two-CTA form (tensor maps with 128-row boxes)
    alignas(64) unsigned char map_a[128];
    alignas(64) unsigned char map_b[128];
    // tasks on a key/value cache
    xpkKvCache_t cache = nullptr;
    xpkAttentionArgs attention = {};
    void *clear_at = nullptr;         // what a reset clears besides the control block
    size_t clear_bytes = 0;
    std::atomic<bool> clear_first{false};  // and the first launch
};

namespace xpk {

// Makes the task's device current for the duration of a call and puts the caller's device back.  The
// entry points that take a task may be called from any thread (a worker thread that never called
// cudaSetDevice is on device 0), while the task's memory and streams belong to the device it was
// created on.
class DeviceGuard {
public:
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&prev_) != cudaSuccess) { prev_ = -1; return; }
        if (prev_ != device) { if (cudaSetDevice(device) == cudaSuccess) switched_ = true; }
    }
    ~DeviceGuard() { if (switched_) cudaSetDevice(prev_); }
    DeviceGuard(const DeviceGuard &) = delete;
    DeviceGuard &operator=(const DeviceGuard &) = delete;
private:
    int prev_ = -1;
    bool switched_ = false;
};

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Creates the control block and the mailbox of a task on the current device; on failure the caller frees the task.
xpkResult task_common(xpkTask_st *t, uint32_t kind, uint32_t flags, unsigned long long total, uint32_t *flag_dev);
void task_free(xpkTask_st *t);
// SMs of the current device (0: the query failed).
int device_sms();
void *tensor_map_encoder();          // cuTensorMapEncodeTiled of the loaded driver, or null
void note_launches(unsigned n);      // the library-wide launch counter

} // namespace xpk
