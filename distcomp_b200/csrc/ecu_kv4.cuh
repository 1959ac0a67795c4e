// ecu_kv4.cuh -- kernels of the paged 4-bit K/V cache (layout: engine_cuda.h).
#pragma once
#include "ecu_common.cuh"
#include "ecu_pipe.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#define KV4_PAGE 64

// Place of chunk b (32 dimensions, 16 bytes) among a position's nb chunks.
__host__ __device__ inline int kv4_place(int t, int b, int nb)
{
    return nb == 4 ? b ^ ((t >> 1) & 3) : nb == 2 ? b ^ ((t >> 2) & 1) : b;
}

template <typename T> __device__ __forceinline__ float  kv4_float(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T      kv4_from(float v);
template <> __device__ __forceinline__ float            kv4_from<float>(float v) { return v; }
template <> __device__ __forceinline__ __half           kv4_from<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16    kv4_from<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive elements; `wide`: the address is a multiple of 16 bytes.
template <typename T> __device__ __forceinline__ void kv4_load8(const T *p, bool wide, float (&x)[8])
{
    if (wide) {
        __align__(16) T v[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            reinterpret_cast<uint4 *>(v)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = kv4_float(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = kv4_float(p[i]);
    }
}

template <typename T> __device__ __forceinline__ void kv4_store8(T *p, bool wide, const float (&x)[8])
{
    __align__(16) T v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = kv4_from<T>(x[i]);
    if (wide) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<uint4 *>(v)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = v[i];
    }
}

// Sequences of one launch, by value: a launch keeps its own copy, so the
// caller's arrays may go and a captured launch replays what it was given.
template <int N> struct KvSeqs {
    int      n;
    uint16_t seq[N];
};

// ---------------------------------------------------------------- append ---
template <int N> struct KvRows {
    int      n;
    uint16_t seq[N];
    int      row0[N + 1];     // first row of each sequence; row0[n] = rows
};

struct KvAppendArgs {
    const void *k, *v;
    long        k_stride, v_stride;
    void       *k_out, *v_out;
    uint8_t    *layer;            // the layer's pages
    size_t      page_bytes;
    const int  *table, *len;
    int         max_pages, n_pages, n_kv, nb;
    bool        wide, wide_out;
};

// Four lanes to a block of 32 values, eight values each.  A block's value of
// largest magnitude is found with two shuffles on (magnitude, first place)
// keys.  The code is decided exactly: the quotient's rounding can only be off
// near k + 1/2, and (k + 1/2) * scale has 5 + 11 bits, exact in fp32, so one
// comparison on either side settles it.  Bound by memory: 2 * (4 or 2) bytes
// of row read and 1.125 written per pair of K and V values.
template <typename T, typename O, int N>
__global__ void __launch_bounds__(256) k_kv4_append(const KvAppendArgs a, const KvRows<N> rows)
{
    const int per_row = 2 * a.n_kv * a.nb;                       // blocks of a row: K then V
    const long long blk = ((long long)blockIdx.x * 256 + threadIdx.x) >> 2;
    const int c = threadIdx.x & 3;
    const long long r = blk / per_row;
    if (r >= rows.row0[rows.n]) return;                          // whole groups of four leave together
    const int in_row = (int)(blk - r * per_row), side = in_row >= a.n_kv * a.nb;
    const int hb = in_row - side * a.n_kv * a.nb, h = hb / a.nb, b = hb - h * a.nb;
    const T  *src = side ? (const T *)a.v + (size_t)r * a.v_stride : (const T *)a.k + (size_t)r * a.k_stride;
    float     x[8];
    kv4_load8(src + (size_t)hb * 32 + 8 * c, a.wide, x);
    // the sequence of row r: the last whose first row is not past it
    int lo = 0, hi = rows.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (rows.row0[mid] <= r) lo = mid;
        else hi = mid;
    }
    const int s = rows.seq[lo];
    const int pos = __ldg(a.len + s) - (rows.row0[lo + 1] - (int)r);

    const unsigned mask = 0xFu << (threadIdx.x & 28);
    float          m = x[0];
    int            at = 8 * c;
    bool           fine = true;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (fabsf(x[i]) > fabsf(m)) { m = x[i]; at = 8 * c + i; }
        fine = fine && fabsf(x[i]) < INFINITY;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const float m2 = __shfl_xor_sync(mask, m, o);
        const int   a2 = __shfl_xor_sync(mask, at, o);
        fine = __shfl_xor_sync(mask, (int)fine, o) && fine;
        if (fabsf(m2) > fabsf(m) || (fabsf(m2) == fabsf(m) && a2 < at)) { m = m2; at = a2; }
    }
    __half dh = __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f));
    if (!fine) dh = __ushort_as_half(0x7FFF);
    else if (__half2float(dh) == 0.0f) dh = __ushort_as_half(0);
    const float d = __half2float(dh);
    const bool  flat = !fine || d == 0.0f;
    const float sg = d < 0.0f ? -1.0f : 1.0f, ad = fabsf(d);
    uint32_t    w = 0;
    float       y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        int code = 8;
        if (!flat) {
            // floor(x / d + 8.5) with x, d -> x * sign(d), |d|
            const float u = x[i] * sg;
            float       k = floorf(__fadd_rn(fminf(fmaxf(__fdiv_rn(u, ad), -16.0f), 16.0f), 0.5f));
            if (u < (k - 0.5f) * ad) k -= 1.0f;
            else if (u >= (k + 0.5f) * ad) k += 1.0f;
            code = min(15, max(0, (int)k + 8));
        }
        w |= (uint32_t)code << (4 * i);
        y[i] = (float)(code - 8) * d;
    }
    const int nkvhd = a.n_kv * a.nb * 32;
    if (a.k_out) kv4_store8((O *)(side ? a.v_out : a.k_out) + (size_t)r * nkvhd + (size_t)hb * 32 + 8 * c, a.wide_out, y);
    if (pos < 0 || pos >= a.max_pages * KV4_PAGE) return;
    const int page = __ldg(a.table + (size_t)s * a.max_pages + pos / KV4_PAGE);
    if ((unsigned)page >= (unsigned)a.n_pages) return;           // no page: nothing to write to
    const int hd = a.nb * 32, t = pos % KV4_PAGE;
    uint8_t  *p = a.layer + (size_t)page * a.page_bytes + (size_t)h * 72 * hd;
    *reinterpret_cast<uint32_t *>(p + side * 32 * hd + t * (hd / 2) + kv4_place(t, b, a.nb) * 16 + 4 * c) = w;
    if (c == 0) *reinterpret_cast<__half *>(p + 64 * hd + side * 4 * hd + (t * a.nb + b) * 2) = dh;
}

// ----------------------------------------------------------- page upkeep ---
// Page copies (every layer) and single device words, by value.
template <int N> struct KvUpdate {
    int n_copy, n_set;
    int a[N], b[N];               // copies (from, to), then words (at, value)
};

#define KV4_COPY_VECS 8           // 16-byte words a thread copies

// Blocks below copy_blocks copy 256 * KV4_COPY_VECS words of one page of one
// layer; the others set words.  Sources and destinations never overlap.
template <int N>
__global__ void __launch_bounds__(256) k_kv4_update(uint8_t *data, size_t page_bytes, size_t layer_bytes, int n_layer,
                                                    int blocks_page, unsigned copy_blocks, int *meta,
                                                    const KvUpdate<N> u)
{
    if (blockIdx.x >= copy_blocks) {
        const int i = (int)(blockIdx.x - copy_blocks) * 256 + (int)threadIdx.x;
        if (i < u.n_set) meta[u.a[u.n_copy + i]] = u.b[u.n_copy + i];
        return;
    }
    const int per_copy = blocks_page * n_layer;
    const int i = blockIdx.x / per_copy, rest = blockIdx.x - i * per_copy, l = rest / blocks_page, part = rest - l * blocks_page;
    const uint4 *src = reinterpret_cast<const uint4 *>(data + l * layer_bytes + (size_t)u.a[i] * page_bytes);
    uint4       *dst = reinterpret_cast<uint4 *>(data + l * layer_bytes + (size_t)u.b[i] * page_bytes);
    const int    n = (int)(page_bytes / 16), at = part * 256 * KV4_COPY_VECS + (int)threadIdx.x;
    uint4        v[KV4_COPY_VECS];
#pragma unroll
    for (int k = 0; k < KV4_COPY_VECS; k++)
        if (at + k * 256 < n) v[k] = src[at + k * 256];
#pragma unroll
    for (int k = 0; k < KV4_COPY_VECS; k++)
        if (at + k * 256 < n) dst[at + k * 256] = v[k];
}

// ------------------------------------------------------------------ read ---
// Positions pos .. pos + n - 1 of one sequence as rows of KV heads; a thread
// per 8 values.  pages: the sequence's table row.
template <typename O>
__global__ void __launch_bounds__(256) k_kv4_read(const uint8_t *layer, size_t page_bytes, const int *pages, int pos, int n,
                                                  int n_kv, int nb, int n_pages, int side, O *out)
{
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const int       per_row = n_kv * nb * 4;
    const long long r = e / per_row;
    if (r >= n) return;
    const int in_row = (int)(e - r * per_row), c = in_row & 3, hb = in_row >> 2, h = hb / nb, b = hb - h * nb;
    const int at = pos + (int)r, t = at % KV4_PAGE, hd = nb * 32;
    const int page = min(max(__ldg(pages + at / KV4_PAGE), 0), n_pages - 1);
    const uint8_t *p = layer + (size_t)page * page_bytes + (size_t)h * 72 * hd;
    const uint32_t w = *reinterpret_cast<const uint32_t *>(p + side * 32 * hd + t * (hd / 2) + kv4_place(t, b, nb) * 16 + 4 * c);
    const float    d = __half2float(*reinterpret_cast<const __half *>(p + 64 * hd + side * 4 * hd + (t * nb + b) * 2));
    float          y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = (float)((int)((w >> (4 * i)) & 15) - 8) * d;
    kv4_store8(out + (size_t)r * n_kv * hd + (size_t)hb * 32 + 8 * c, true, y);
}

// ---------------------------------------------------------------- attend ---
struct KvAttendArgs {
    const void    *q;
    void          *out;
    long           q_stride, out_stride;
    const uint8_t *layer;
    size_t         page_bytes;
    const int     *table, *len;
    int            max_pages, n_pages, n_kv, n_rep;
    float          scale;
    float         *part;          // workspace: partials of rows that several CTAs share
    unsigned      *count;         //   and their tickets
};

// One CTA per (row, query head), a warp per position, lanes over dimensions.
template <typename T, int N>
__global__ void __launch_bounds__(128) k_kv4_attend_simple(const KvAttendArgs a, const KvSeqs<N> list, int hd)
{
    __shared__ float part[4][130];
    const int i = blockIdx.x, head = blockIdx.y, g = head / a.n_rep, s = list.seq[i];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nb = hd / 32;
    const int n = min(__ldg(a.len + s), a.max_pages * KV4_PAGE);
    const T  *q = (const T *)a.q + (size_t)i * a.q_stride + (size_t)head * hd;
    float     qv[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
    for (int b = 0; b < nb; b++) qv[b] = kv4_float(q[b * 32 + lane]);
    for (int p = warp; p < n; p += 4) {
        const int page = min(max(__ldg(a.table + (size_t)s * a.max_pages + p / KV4_PAGE), 0), a.n_pages - 1), t = p % KV4_PAGE;
        const uint8_t *c = a.layer + (size_t)page * a.page_bytes + (size_t)g * 72 * hd;
        const __half  *sc = reinterpret_cast<const __half *>(c + 64 * hd);
        float          dot = 0.0f, v[4];
        for (int b = 0; b < nb; b++) {
            const int at = t * (hd / 2) + kv4_place(t, b, nb) * 16 + lane / 2;
            const int kc = (c[at] >> (4 * (lane & 1))) & 15, vc = (c[32 * hd + at] >> (4 * (lane & 1))) & 15;
            dot = fmaf(qv[b], (float)(kc - 8) * __half2float(sc[t * nb + b]), dot);
            v[b] = (float)(vc - 8) * __half2float(sc[2 * hd + t * nb + b]);
        }
        const float x = warp_sum(dot) * a.scale, mn = fmaxf(m, x), f = expf(m - mn), e = expf(x - mn);
        m = mn;
        l = l * f + e;
        for (int b = 0; b < nb; b++) o[b] = o[b] * f + e * v[b];
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
        float v = 0.0f;
        for (int k = 0; k < 4; k++) v += w[k] * part[k][threadIdx.x];
        ((T *)a.out)[(size_t)i * a.out_stride + (size_t)head * hd + threadIdx.x] = kv4_from<T>(n > 0 ? v / L : 0.0f);
    }
}
