// ecu_attn_prompt.cu -- causal attention of packed prompts behind
// engine_cuda.h.
#include "ecu_attn_prompt.cuh"
#include "ecu_kv4.h"
#include "ecu_model.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <exception>
#include <numeric>
#include <vector>

#define PA_LIST 1024              // sequences of one launch

// Set where a wait of a caller's own call gave up (the engine's calls name
// their context's word), until ecu_attn_prompt_status reads it.
static __device__ int g_prompt_status;

static std::atomic<unsigned> g_stall{0};        // devices (bits) whose next call's waits run out

static int say(const char *why)
{
    ecu_set_error(nullptr, 0, "ecu_attn_prompt: %s", why);
    return -1;
}

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled()
{
    static const EncodeTiled f = [] {
        void                           *p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return f;
}

// Rows x heads x head_dim in boxes of 128 rows of 64 elements of one head.
static int make_map(CUtensorMap *m, int dtype, const void *p, int head_dim, int heads, long rows, long stride)
{
    const EncodeTiled f = encode_tiled();
    if (!f) return say("the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, 1, 128}, ones[3] = {1, 1, 1};
    const CUresult   r = f(m, dtype == ECU_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                           const_cast<void *>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        ecu_set_error(nullptr, 0, "ecu_attn_prompt: the rows cannot be mapped (%d)", (int)r);
        return -1;
    }
    return 0;
}

template <typename T, int HD, int N>
static int launch(const CUtensorMap (&m)[3], const PromptArgs &a, const int *cu_q, const int *cu_k, const int *order, int n,
                  int device, cudaStream_t s)
{
    PromptSeqs<N> list;
    list.n = n;
    long long ctas = 0;
    for (int i = 0; i < n; i++) {
        const int x = order[i];
        list.q0[i] = cu_q[x];
        list.nq[i] = cu_q[x + 1] - cu_q[x];
        list.k0[i] = cu_k[x];
        list.nk[i] = cu_k[x + 1] - cu_k[x];
        list.cta[i] = (int)ctas;
        ctas += (((long long)(list.nq[i] + 127) / 128 * a.n_rep + 1) / 2) * a.n_kv;
    }
    if (ctas > INT_MAX) return say("too many rows and heads");
    list.cta[n] = (int)ctas;
    auto kern = k_attn_prompt<T, HD, N>;
    static std::atomic<unsigned> done{0};
    cudaError_t e = ecu_allow_smem(kern, PaShape<HD>::smem, device, done);
    if (e == cudaSuccess) {
        e = ecu_launch_early(kern, (unsigned)ctas, PA_THREADS, PaShape<HD>::smem, s, m[0], m[1], m[2], a, list);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        ecu_set_error(nullptr, 0, "ecu_attn_prompt: launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    ecu_count_launches(1);
    return 0;
}

template <typename T>
static int launch_all(const CUtensorMap (&m)[3], const PromptArgs &a, int head_dim, const int *cu_q, const int *cu_k, int n_seq,
                      int device, cudaStream_t s)
{
    // sequences with query rows, the most keys first: their last tiles are the longest walks
    std::vector<int> order;
    for (int i = 0; i < n_seq; i++)
        if (cu_q[i + 1] > cu_q[i]) order.push_back(i);
    std::stable_sort(order.begin(), order.end(),
                     [&](int x, int y) { return cu_k[x + 1] - cu_k[x] > cu_k[y + 1] - cu_k[y]; });
    for (int i = 0; i < (int)order.size(); i += PA_LIST) {
        const int  c = std::min<int>(PA_LIST, (int)order.size() - i);
        const int *o = order.data() + i;
        const int  rc = head_dim == 128 ? (c <= 32 ? launch<T, 128, 32>(m, a, cu_q, cu_k, o, c, device, s) : launch<T, 128, PA_LIST>(m, a, cu_q, cu_k, o, c, device, s))
                                        : (c <= 32 ? launch<T, 64, 32>(m, a, cu_q, cu_k, o, c, device, s) : launch<T, 64, PA_LIST>(m, a, cu_q, cu_k, o, c, device, s));
        if (rc != 0) return rc;
    }
    return 0;
}

int ecu_prompt_set_wait(unsigned long long ns) { return set_wait_limit(ns) == cudaSuccess ? 0 : -1; }

// The status word's address on the current device; nullptr: it cannot be had.
static int *status_word(int device)
{
    static std::atomic<int *> at[32];
    void                     *p = device < 32 ? at[device].load() : nullptr;
    if (!p) {
        if (cudaGetSymbolAddress(&p, g_prompt_status) != cudaSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        if (device < 32) at[device] = (int *)p;
    }
    return (int *)p;
}

// Reads and clears the word in one step, so that no flag that another stream's
// call sets in between is lost.
static __global__ void k_take_status(int *out) { *out = atomicExch(&g_prompt_status, 0); }

extern "C" int ecu_attn_prompt_status(int device, void *stream)
{
    int ndev = 0;
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) {
        cudaGetLastError();
        ecu_set_error(nullptr, 0, "ecu_attn_prompt_status: CUDA device %d not available (%d devices)", device, ndev);
        return -1;
    }
    DeviceScope d(device);
    if (!d.ok) return say("the device cannot be used");
    const cudaStream_t      s = (cudaStream_t)stream;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    cudaError_t             e = cudaStreamIsCapturing(s, &cap);
    if (e == cudaSuccess && cap != cudaStreamCaptureStatusNone) return say("the status of a stream that is being captured is not known");
    int *taken = nullptr, flags = 0;
    if (e == cudaSuccess) e = cudaMallocAsync((void **)&taken, sizeof flags, s);
    if (e == cudaSuccess) {
        k_take_status<<<1, 1, 0, s>>>(taken);
        e = cudaGetLastError();
        if (e == cudaSuccess) e = cudaMemcpyAsync(&flags, taken, sizeof flags, cudaMemcpyDeviceToHost, s);
        cudaFreeAsync(taken, s);
        if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        ecu_set_error(nullptr, 0, "ecu_attn_prompt_status: %s", cudaGetErrorString(e));
        return -1;
    }
    if (!flags) return 0;
    ecu_set_error(nullptr, 0, "ecu_attn_prompt: a kernel gave up on a bounded wait (status %d)", flags);
    return -1;
}

extern "C" int ecu_inject_prompt_timeout(int device)
{
    if (device < 0 || device >= 32) return say("no such device to stall");
    g_stall.fetch_or(1u << device);
    return 0;
}

extern "C" int ecu_attn_prompt(int dtype, const void *q, const void *k, const void *v, void *out, int n_head, int n_head_kv,
                               int head_dim, long q_stride, long k_stride, long v_stride, long out_stride, const int *cu_q,
                               const int *cu_k, int n_seq, float scale, int device, void *stream)
{
    return ecu_attn_prompt_on(nullptr, dtype, q, k, v, out, n_head, n_head_kv, head_dim, q_stride, k_stride, v_stride, out_stride, cu_q,
                              cu_k, n_seq, scale, device, stream);
}

int ecu_attn_prompt_on(int *status, int dtype, const void *q, const void *k, const void *v, void *out, int n_head, int n_head_kv,
                       int head_dim, long q_stride, long k_stride, long v_stride, long out_stride, const int *cu_q, const int *cu_k,
                       int n_seq, float scale, int device, void *stream)
{
    if (dtype != ECU_F16 && dtype != ECU_BF16) return say("rows are ECU_F16 or ECU_BF16");
    if (head_dim != 64 && head_dim != 128) {
        ecu_set_error(nullptr, 0, "ecu_attn_prompt: head_dim %d is not built (64 or 128)", head_dim);
        return -1;
    }
    if (n_head_kv < 1 || n_head < 1 || n_head % n_head_kv || n_head > 65535) {
        ecu_set_error(nullptr, 0, "ecu_attn_prompt: %d query heads for %d KV heads", n_head, n_head_kv);
        return -1;
    }
    if (n_seq < 0 || (n_seq > 0 && !cu_q)) return say("null offsets or negative count");
    if (!(scale > 0.0f) || !std::isfinite(scale)) return say("the scale is not a positive finite number");
    if (n_seq == 0) return 0;
    if (!cu_k) cu_k = cu_q;
    if (cu_q[0] != 0 || cu_k[0] != 0) return say("offsets begin at 0");
    for (int i = 0; i < n_seq; i++)
        if (cu_q[i + 1] < cu_q[i] || cu_k[i + 1] < cu_k[i]) return say("offsets decrease");
    if (cu_q[n_seq] == 0) return 0;
    const long es = 2, qr = (long)n_head * head_dim, kr = (long)n_head_kv * head_dim;
    const bool keys = cu_k[n_seq] > 0;
    if (cu_q[n_seq] == 1) q_stride = out_stride = qr;       // one row: no stride
    if (cu_k[n_seq] <= 1) k_stride = v_stride = kr;
    if (!q || !out || (keys && (!k || !v))) return say("null rows");
    if ((cu_q[n_seq] > 1 && (q_stride < qr || out_stride < qr)) || (cu_k[n_seq] > 1 && (k_stride < kr || v_stride < kr)))
        return say("rows overlap: a stride below the row's heads");
    if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) ||
        ((q_stride * es | k_stride * es | v_stride * es | out_stride * es) & 15))
        return say("rows are not 16-byte aligned");
    int ndev = 0;
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) {
        cudaGetLastError();
        ecu_set_error(nullptr, 0, "ecu_attn_prompt: CUDA device %d not available (%d devices)", device, ndev);
        return -1;
    }
    DeviceScope d(device);
    if (!d.ok) return say("the device cannot be used");
    if (!status && !(status = status_word(device))) return say("the status word cannot be had");
    PromptArgs  a{v, out, v_stride, out_stride, n_head_kv, n_head / n_head_kv, scale, status, 0};
    CUtensorMap m[3];
    // a pointer that no row is read from is not mapped: q stands in
    if (make_map(m + 0, dtype, q, head_dim, n_head, cu_q[n_seq], q_stride) != 0 ||
        make_map(m + 1, dtype, keys ? k : q, head_dim, keys ? n_head_kv : 1, keys ? cu_k[n_seq] : 1, keys ? k_stride : qr) != 0 ||
        make_map(m + 2, dtype, keys ? v : q, head_dim, keys ? n_head_kv : 1, keys ? cu_k[n_seq] : 1, keys ? v_stride : qr) != 0)
        return -1;
    const cudaStream_t s = (cudaStream_t)stream;
    if (device < 32 && g_stall.load(std::memory_order_relaxed))
        a.stall = (int)(g_stall.fetch_and(~(1u << device)) >> device & 1u);
    try {
        return dtype == ECU_F16 ? launch_all<__half>(m, a, head_dim, cu_q, cu_k, n_seq, device, s)
                                : launch_all<__nv_bfloat16>(m, a, head_dim, cu_q, cu_k, n_seq, device, s);
    } catch (const std::exception &e) {
        return say(e.what());
    }
}
