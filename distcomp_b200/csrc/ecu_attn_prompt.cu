// ecu_attn_prompt.cu -- causal attention of packed prompts behind
// engine_cuda.h.
#include "ecu_kv4.cuh"
#include "ecu_kv4.h"
#include "ecu_model.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <exception>

#define PA_LIST 1024              // sequences of one launch

struct PromptArgs {
    const void *q, *k, *v;
    void       *out;
    long        q_stride, k_stride, v_stride, out_stride;
    int         n_rep, hd;
    float       scale;
};

template <int N> struct PromptSeqs {
    int n;
    int q0[N + 1], k0[N + 1];
};

// One CTA per (query row, head): a warp per key, lanes over dimensions.
template <typename T, int N>
__global__ void __launch_bounds__(128) k_attn_prompt_simple(const PromptArgs a, const PromptSeqs<N> list)
{
    __shared__ float part[4][130];
    const int r = list.q0[0] + blockIdx.x, head = blockIdx.y, g = head / a.n_rep, hd = a.hd, nb = hd / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int       lo = 0, hi = list.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (list.q0[mid] <= r) lo = mid;
        else hi = mid;
    }
    const int n = list.k0[lo + 1] - list.k0[lo] - (list.q0[lo + 1] - 1 - r);    // keys that the row sees
    const T  *q = (const T *)a.q + (size_t)r * a.q_stride + (size_t)head * hd;
    float     qv[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
    for (int b = 0; b < nb; b++) qv[b] = kv4_float(q[b * 32 + lane]);
    for (int p = warp; p < n; p += 4) {
        const T *k = (const T *)a.k + (size_t)(list.k0[lo] + p) * a.k_stride + (size_t)g * hd;
        const T *v = (const T *)a.v + (size_t)(list.k0[lo] + p) * a.v_stride + (size_t)g * hd;
        float    dot = 0.0f;
        for (int b = 0; b < nb; b++) dot = fmaf(qv[b], kv4_float(k[b * 32 + lane]), dot);
        const float x = warp_sum(dot) * a.scale, mn = fmaxf(m, x), f = expf(m - mn), e = expf(x - mn);
        m = mn;
        l = l * f + e;
        for (int b = 0; b < nb; b++) o[b] = o[b] * f + e * kv4_float(v[b * 32 + lane]);
    }
    for (int b = 0; b < nb; b++) part[warp][b * 32 + lane] = o[b];
    part[warp][128] = m;
    part[warp][129] = l;
    __syncthreads();
    float M = -INFINITY, L = 0.0f, w[4];
    for (int k = 0; k < 4; k++) M = fmaxf(M, part[k][128]);
    for (int k = 0; k < 4; k++) {
        w[k] = part[k][128] > -INFINITY ? expf(part[k][128] - M) : 0.0f;
        L += w[k] * part[k][129];
    }
    if ((int)threadIdx.x < hd) {
        float x = 0.0f;
        for (int k = 0; k < 4; k++) x += w[k] * part[k][threadIdx.x];
        ((T *)a.out)[(size_t)r * a.out_stride + (size_t)head * hd + threadIdx.x] = kv4_from<T>(n > 0 ? x / L : 0.0f);
    }
}

static int say(const char *why)
{
    ecu_set_error(nullptr, 0, "ecu_attn_prompt: %s", why);
    return -1;
}

template <typename T, int N>
static int launch(const PromptArgs &a, int n_head, const int *cu_q, const int *cu_k, int n, cudaStream_t s)
{
    PromptSeqs<N> list;
    list.n = n;
    for (int i = 0; i <= n; i++) {
        list.q0[i] = cu_q[i];
        list.k0[i] = cu_k[i];
    }
    if (cu_q[n] == cu_q[0]) return 0;
    k_attn_prompt_simple<T, N><<<dim3((unsigned)(cu_q[n] - cu_q[0]), (unsigned)n_head), 128, 0, s>>>(a, list);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        ecu_set_error(nullptr, 0, "ecu_attn_prompt: launch failed: %s", cudaGetErrorString(e));
        return -1;
    }
    ecu_count_launches(1);
    return 0;
}

extern "C" int ecu_attn_prompt(int dtype, const void *q, const void *k, const void *v, void *out, int n_head, int n_head_kv,
                               int head_dim, long q_stride, long k_stride, long v_stride, long out_stride, const int *cu_q,
                               const int *cu_k, int n_seq, float scale, int device, void *stream)
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
    if (!std::isfinite(scale)) return say("the scale is not finite");
    if (n_seq == 0) return 0;
    if (!cu_k) cu_k = cu_q;
    if (cu_q[0] != 0 || cu_k[0] != 0) return say("offsets begin at 0");
    for (int i = 0; i < n_seq; i++)
        if (cu_q[i + 1] < cu_q[i] || cu_k[i + 1] < cu_k[i]) return say("offsets decrease");
    if (cu_q[n_seq] == 0) return 0;
    const long es = 2, qr = (long)n_head * head_dim, kr = (long)n_head_kv * head_dim;
    const bool keys = cu_k[n_seq] > 0;
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
    PromptArgs a{q, k, v, out, q_stride, k_stride, v_stride, out_stride, n_head / n_head_kv, head_dim, scale};
    for (int i = 0; i < n_seq; i += PA_LIST) {
        const int m = std::min(PA_LIST, n_seq - i);
        const int *cq = cu_q + i, *ck = cu_k + i;
        const cudaStream_t s = (cudaStream_t)stream;
        int rc;
        if (dtype == ECU_F16) rc = m <= 64 ? launch<__half, 64>(a, n_head, cq, ck, m, s) : launch<__half, PA_LIST>(a, n_head, cq, ck, m, s);
        else rc = m <= 64 ? launch<__nv_bfloat16, 64>(a, n_head, cq, ck, m, s) : launch<__nv_bfloat16, PA_LIST>(a, n_head, cq, ck, m, s);
        if (rc != 0) return rc;
    }
    return 0;
}
