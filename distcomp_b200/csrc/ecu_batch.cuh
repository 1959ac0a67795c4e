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

// Rows of fp32 values, `ld` apart, as fp16 rows without gaps (clamped to
// fp16's range, which q and k do not leave in earnest).
static __global__ void k_bt_half(const float *X, int ld, size_t rows, int width, __half *out)
{
    const size_t total = rows * (size_t)width;
    for (size_t e = blockIdx.x * (size_t)blockDim.x + threadIdx.x; e < total; e += (size_t)gridDim.x * blockDim.x) {
        const float v = X[e / width * ld + e % width];
        out[e] = __float2half_rn(fabsf(v) < INFINITY ? fminf(fmaxf(v, -65504.0f), 65504.0f) : v);
    }
}

// Positions 0..n-1 of a dense cache plane [n_kv][n_ctx][hd] as fp16 rows
// [n][n_kv][hd].
static __global__ void k_bt_plane_half(const float *plane, int n_ctx, int n_kv, int hd, int n, __half *out)
{
    const size_t total = (size_t)n * n_kv * hd;
    for (size_t e = blockIdx.x * (size_t)blockDim.x + threadIdx.x; e < total; e += (size_t)gridDim.x * blockDim.x) {
        const int   d = (int)(e % hd), g = (int)(e / hd % n_kv);
        const float v = plane[((size_t)g * n_ctx + e / ((size_t)hd * n_kv)) * hd + d];
        out[e] = __float2half_rn(fabsf(v) < INFINITY ? fminf(fmaxf(v, -65504.0f), 65504.0f) : v);
    }
}
