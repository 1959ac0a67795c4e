// ecu_kv4.h -- host side of the paged 4-bit K/V cache, shared by the
// translation units that use it.
#pragma once
#include "../../include/engine_cuda.h"

#include <atomic>
#include <cuda_runtime.h>
#include <cstdint>
#include <map>
#include <vector>

// Which sequence holds which page, and how many hold each page.  Pure host
// bookkeeping: every operation either succeeds or leaves everything as it
// was, and collects the page copies and device words that follow from it.
struct KvBook {
    int n_pages = 0, n_seq = 0, max_pages = 0;
    struct Seq { int len = 0; std::vector<int> page; };
    std::vector<Seq>      seq;
    std::vector<int>      ref;
    std::vector<uint64_t> taken;      // bit p: page p is held
    size_t                hint = 0;   // no free page lies in a word below
    int                   used = 0;

    struct Copy { int from, to; };
    struct Set { int at, value; };    // device words: table [n_seq][max_pages], then len [n_seq]
    std::vector<Copy> copies;         // of the last operation
    std::vector<Set>  sets;

    void init(int pages, int seqs, int per_seq);
    int  extend(const int *s, const int *n_new, int n);
    int  fork(const int *src, const int *dst, int n);
    int  truncate(const int *s, const int *len, int n);
    int  compact();
    int  fail();                      // takes the last operation back; -1

private:
    struct Undo { int kind, a, b; };
    std::vector<Undo> log_;
    std::vector<std::pair<int, int>> cell_;    // table cells (sequence, index) that changed
    std::vector<int>                 length_;  // sequences whose length changed
    std::vector<int>                 move_;    // of each page, where it goes while pages move; else -1
    bool                             compacted_ = false;       // the last operation is a compaction
    int  take();
    void hold(int p);
    void drop(int p);
    void begin();
    void finish();
    void move_pages(bool back);
    bool slot(int s, const char *what);
};

struct ecu_kv {
    int    n_layer = 0, n_head_kv = 0, head_dim = 0, device = -1, sms = 0;
    size_t page_bytes = 0, device_bytes = 0;
    uint8_t *data = nullptr;
    bool     own_data = false;
    int     *meta = nullptr;          // device: table, then len
    KvBook   book;
    // a stream's id -> its attention workspace (handles are reused, and the
    // per-thread default stream's names another stream in each thread)
    std::map<unsigned long long, void *> ws;
    void *spare = nullptr;            // the first stream's, allocated with the pool
    bool  broken = false;             // a change ended between its launches: tables and bookkeeping differ
    int   inject = -1;                // ecu_kv_inject_failure: the launch of the next change that fails
    int *table() const { return meta; }
    int *len() const { return meta ? meta + (size_t)book.n_seq * book.max_pages : nullptr; }
};

// The current device for the time of a call.
struct DeviceScope {
    int  old = -1;
    bool ok;
    explicit DeviceScope(int dev)
    {
        ok = cudaGetDevice(&old) == cudaSuccess && (old == dev || cudaSetDevice(dev) == cudaSuccess);
        if (old == dev) old = -1;
    }
    ~DeviceScope()
    {
        if (old >= 0) cudaSetDevice(old);
    }
};

// A kernel's dynamic shared memory limit, set once per kernel (`done`: a bit
// per device) on the current device `dev`.
template <typename F> cudaError_t ecu_allow_smem(F kern, size_t bytes, int dev, std::atomic<unsigned> &done)
{
    if (dev < 32 && (done.load(std::memory_order_relaxed) >> dev & 1u)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 32) done.fetch_or(1u << dev);
    return e;
}

// A launch that may begin while what comes before it in the stream ends (the
// kernel waits for that itself, pdl_wait, before it touches global memory).
template <typename... P, typename... A>
cudaError_t ecu_launch_early(void (*kern)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t s, const A &...args)
{
    cudaLaunchConfig_t  cfg = {};
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

void ecu_count_launches(int n);       // ecu_kernel_launches()

// ecu_attn_prompt with a status word of the caller's on the device (nullptr:
// the one that ecu_attn_prompt_status reads): ECU_STATUS_TIMEOUT is set in it
// where a wait gives up.
int ecu_attn_prompt_on(int *status, int dtype, const void *q, const void *k, const void *v, void *out, int n_head, int n_head_kv,
                       int head_dim, long q_stride, long k_stride, long v_stride, long out_stride, const int *cu_q, const int *cu_k,
                       int n_seq, float scale, int device, void *stream);

// ecu_set_wait_ns for the prompt attention's translation unit, on the current
// device.
int ecu_prompt_set_wait(unsigned long long ns);

// Positions 0..n-1 of a sequence as fp16 rows [n][n_head_kv * head_dim] in
// device memory, as the cache holds them.
int ecu_kv_rows(ecu_kv *kv, int layer, int seq, int n, void *k, void *v, cudaStream_t s);
