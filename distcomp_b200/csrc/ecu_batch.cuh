// ecu_batch.cuh -- many sequences over one model's weights, their K/V in a
// pool of 4-bit pages: kernels that tie the batched prompt (ecu_prefill.cuh)
// to the pool's operators (ecu_kv4.cuh) and to the prompt attention.
#pragma once
#include "ecu_attn.cuh"
#include "ecu_common.cuh"

#include <cuda_fp16.h>

// Row t of QKV (q | k | v of one token): biases, and RoPE of q and k at the
// row's own position (src/engine.c:367-378), in place.
static __global__ void k_bt_rope(float *QKV, int ld, int n_head, int n_kv, int hd, const int *pos, const float *cs,
                                 const float *bq, const float *bk, const float *bv)
{
    const int    t = blockIdx.x, half = hd / 2;
    float       *q = QKV + (size_t)t * ld, *k = q + (size_t)n_head * hd, *v = k + (size_t)n_kv * hd;
    const float *c = cs + (size_t)pos[t] * hd;
    auto turn = [&](float *x, const float *b, int i) {
        const int h = i / half, j = i % half;
        float     x0 = x[h * hd + j], x1 = x[h * hd + j + half];
        if (b) { x0 = __fadd_rn(x0, b[h * hd + j]); x1 = __fadd_rn(x1, b[h * hd + j + half]); }
        rope_pair(x0, x1, c[2 * j], c[2 * j + 1]);
        x[h * hd + j] = x0;
        x[h * hd + j + half] = x1;
    };
    for (int i = threadIdx.x; i < n_head * half; i += blockDim.x) turn(q, bq, i);
    for (int i = threadIdx.x; i < n_kv * half; i += blockDim.x) turn(k, bk, i);
    if (bv)
        for (int i = threadIdx.x; i < n_kv * hd; i += blockDim.x) v[i] = __fadd_rn(v[i], bv[i]);
}

// A value as fp16; one that fp16 does not reach says so (what is infinite or
// NaN to begin with stays that).
__device__ __forceinline__ __half bt_half(float v, bool &past)
{
    const __half h = __float2half_rn(v);
    past |= __hisinf(h) && fabsf(v) < INFINITY;
    return h;
}

// Rows of fp32 values, `ld` apart, as fp16 rows without gaps; and a look at
// the cache's rows k and v (n_kv elements each, a multiple of 8; nullptr: not
// wanted), whose values are finite or NaN: an infinity among them was a value
// that fp16 does not reach.  Such a value flags ECU_STATUS_RANGE.
static __global__ void k_bt_half(const float *X, int ld, size_t rows, int width, __half *out, const __half *k, const __half *v,
                                 size_t n_kv, int *status)
{
    const size_t first = blockIdx.x * (size_t)blockDim.x + threadIdx.x, step = (size_t)gridDim.x * blockDim.x;
    const size_t total = rows * (size_t)width, vecs = k ? n_kv / 8 : 0;
    bool         past = false;
    for (size_t e = first; e < total; e += step) out[e] = bt_half(X[e / width * ld + e % width], past);
    for (size_t e = first; e < 2 * vecs; e += step) {
        const uint4 w = reinterpret_cast<const uint4 *>(e < vecs ? k : v)[e < vecs ? e : e - vecs];
        for (uint32_t x : {w.x, w.y, w.z, w.w}) past |= (x & 0x7FFFu) == 0x7C00u || (x & 0x7FFF0000u) == 0x7C000000u;
    }
    if (past) atomicOr(status, ECU_STATUS_RANGE);
}

// k_pf_split of a batch's attention rows, which the cache lets reach 8 * 65504.
static __global__ void k_bt_split(const float *X, size_t count, __half *hi, __half *lo, int *status)
{
    bool past = false;
    for (size_t e = blockIdx.x * (size_t)blockDim.x + threadIdx.x; e < count; e += (size_t)gridDim.x * blockDim.x) {
        const float v = X[e];
        hi[e] = bt_half(v, past);
        lo[e] = __float2half_rn(__fsub_rn(v, __half2float(hi[e])));
    }
    if (past) atomicOr(status, ECU_STATUS_RANGE);
}

// Positions 0..n-1 of a dense cache plane [n_kv][n_ctx][hd] as fp16 rows
// [n][n_kv][hd].
static __global__ void k_bt_plane_half(const float *plane, int n_ctx, int n_kv, int hd, int n, __half *out, int *status)
{
    const size_t total = (size_t)n * n_kv * hd;
    bool         past = false;
    for (size_t e = blockIdx.x * (size_t)blockDim.x + threadIdx.x; e < total; e += (size_t)gridDim.x * blockDim.x) {
        const int   d = (int)(e % hd), g = (int)(e / hd % n_kv);
        out[e] = bt_half(plane[((size_t)g * n_ctx + e / ((size_t)hd * n_kv)) * hd + d], past);
    }
    if (past) atomicOr(status, ECU_STATUS_RANGE);
}
