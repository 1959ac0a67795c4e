// ecu_kv4.cuh -- kernels of the paged 4-bit K/V cache (layout: engine_cuda.h).
#pragma once
#include "ecu_common.cuh"
#include "ecu_pipe.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

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
    unsigned    nb_inv;           // x / nb = x * nb_inv >> 16 for the blocks of a row
    bool        wide, wide_out;
};

// The larger, or NaN where either is.
__device__ __forceinline__ float kv4_max(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Eight of a block's 32 values (the other 24 with the group's other lanes):
// the scale, and this lane's word of codes and values as stored.
//
// With u = x * sign(scale) and d = |scale|, the code is 8 + the k of
// (k - 1/2) d <= u < (k + 1/2) d.  k is guessed from u * (1 / d) - 2^-18, which
// is never too high and too low by one at most, and settled by r = u - k d, one
// fma: where r is near d / 2 it is exact (u and k d are multiples of 2^-24 of
// the power of two below d, and |r| is below it), so the comparison with d / 2
// decides as exact arithmetic would.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&x)[8], unsigned mask, int c, __half &dh, float (&y)[8])
{
    // the largest value and the largest negated one say the sign, unless they
    // are equal: then the first of them does
    float p = x[0], q = -x[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        p = kv4_max(p, x[i]);
        q = kv4_max(q, -x[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        p = kv4_max(p, __shfl_xor_sync(mask, p, o));
        q = kv4_max(q, __shfl_xor_sync(mask, q, o));
    }
    float m = p > q ? p : -q;
    if (p == q) {                                                // (the same in the group's four lanes)
        int at = 64;                                             // 2 * place of the first, odd for a negative value
#pragma unroll
        for (int i = 7; i >= 0; i--)
            if (fabsf(x[i]) == p) at = 2 * (8 * c + i) + (x[i] < 0.0f);
        at = min(at, __shfl_xor_sync(mask, at, 1));
        at = min(at, __shfl_xor_sync(mask, at, 2));
        m = at & 1 ? -p : p;
    }
    const bool fine = fabsf(m) < INFINITY && p == p;
    dh = __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f));
    if (!fine) dh = __ushort_as_half(0x7FFF);
    else if (__half2float(dh) == 0.0f) dh = __ushort_as_half(0);
    const float d = __half2float(dh), sign = copysignf(1.0f, d);
    // a scale of zero: every guess is 0, and nothing reaches the half step
    const float inv = d != 0.0f ? __frcp_rn(d) : 0.0f, half = d != 0.0f ? 0.5f * fabsf(d) : INFINITY;
    uint32_t    w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        // rounded to a whole number by adding 1.5 * 2^23 and taking it off again
        float k = __fsub_rn(__fadd_rn(__fmaf_rn(x[i], inv, -3.814697265625e-6f), 12582912.0f), 12582912.0f);
        if (__fmul_rn(__fmaf_rn(-k, d, x[i]), sign) >= half) k += 1.0f;
        k = fminf(fmaxf(k, -8.0f), 7.0f);
        // 2^23 + 8 + k has the bits 0x4B000000 + code: eight of them, 4 bits apart, add up to the
        // word and 0xFB000000
        w += __float_as_uint(k + 8388616.0f) << (4 * i);
        y[i] = k * d;
    }
    return fine ? w - 0xFB000000u : 0x88888888u;
}

// Four lanes to a block of 32 dimensions, eight values of K and of V each.
// Read are 4 or 2 bytes a value, written 0.5625, and 4 or 2 where the values
// are handed back; what bounds it is instruction issue (39 a value): 8310 bf16
// rows of 8 heads of 128, handed back, 26 us, 3.0 TB/s.
template <typename T, typename O, int N>
__global__ void __launch_bounds__(256) k_kv4_append(const KvAppendArgs a, const KvRows<N> rows)
{
    pdl_wait();
    pdl_trigger();
    const unsigned per_row = a.n_kv * a.nb;                      // blocks of a row
    const unsigned blk = (blockIdx.x * 256u + threadIdx.x) >> 2; // below 2^31: the host sees to it
    const int      c = threadIdx.x & 3, r = (int)(blk / per_row);
    if (r >= rows.row0[rows.n]) return;                          // whole groups of four leave together
    const int hb = (int)(blk - r * per_row), h = (int)((unsigned)hb * a.nb_inv >> 16), b = hb - h * a.nb;
    float     x[2][8];
    kv4_load8((const T *)a.k + (size_t)r * a.k_stride + (size_t)hb * 32 + 8 * c, a.wide, x[0]);
    kv4_load8((const T *)a.v + (size_t)r * a.v_stride + (size_t)hb * 32 + 8 * c, a.wide, x[1]);
    // the sequence of row r: the last whose first row is not past it
    int lo = 0, hi = rows.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (rows.row0[mid] <= r) lo = mid;
        else hi = mid;
    }
    const int  s = rows.seq[lo], pos = __ldg(a.len + s) - (rows.row0[lo + 1] - r);
    const bool placed = pos >= 0 && pos < a.max_pages * KV4_PAGE;
    const int  page = placed ? __ldg(a.table + (size_t)s * a.max_pages + pos / KV4_PAGE) : -1;
    const int  hd = a.nb * 32, t = pos % KV4_PAGE;
    const bool wr = (unsigned)page < (unsigned)a.n_pages;        // no page: nothing to write to
    uint8_t   *p = a.layer + (size_t)(wr ? page : 0) * a.page_bytes + (size_t)h * 72 * hd;
    const unsigned mask = 0xFu << (threadIdx.x & 28);
#pragma unroll
    for (int side = 0; side < 2; side++) {
        float          y[8];
        __half         d;
        const uint32_t w = kv4_quantise(x[side], mask, c, d, y);
        if (a.k_out)
            kv4_store8((O *)(side ? a.v_out : a.k_out) + (size_t)r * per_row * 32 + (size_t)hb * 32 + 8 * c, a.wide_out, y);
        if (!wr) continue;
        *reinterpret_cast<uint32_t *>(p + side * 32 * hd + t * (hd / 2) + kv4_place(t, b, a.nb) * 16 + 4 * c) = w;
        if (c == 0) *reinterpret_cast<__half *>(p + 64 * hd + side * 4 * hd + (t * a.nb + b) * 2) = d;
    }
}

// ----------------------------------------------------------- page upkeep ---
// Page copies (every layer) and single device words, by value.
template <int N> struct KvUpdate {
    int n_copy, n_set;
    int a[N], b[N];               // copies (from, to), then words (at, value)
};

#define KV4_COPY_VECS 8           // 16-byte words a thread copies

// Blocks below copy_blocks copy 256 * KV4_COPY_VECS words of one page of one
// layer; the others set words.  Sources and destinations never overlap.  Bound
// by memory: 64 pages of 32 layers (8 heads of 128) in 42 us, 7.1 TB/s of reads
// and writes.
template <int N>
__global__ void __launch_bounds__(256) k_kv4_update(uint8_t *data, size_t page_bytes, size_t layer_bytes, int n_layer,
                                                    int blocks_page, unsigned copy_blocks, int *meta,
                                                    const KvUpdate<N> u)
{
    pdl_wait();
    pdl_trigger();
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
    bool           wide_q;
    float         *part;          // workspace: partials of rows that several CTAs share
    unsigned      *count;         //   and their tickets
};

// The attention is one pass over the cached rows with a running maximum and
// sum.  K and V are integer codes times a scale per 32 dimensions, so both
// products run on the tensor cores (mma.sync m16n8k16, fp16 operands, fp32
// sums) on the codes themselves, which fp16 holds exactly:
//
//   score[t][col] = sum_b Kscale[t][b] * (Kcode[t][b] . q[col][b])
//   O^T[d][col]  += sum_t Vcode[t][d] * (weight[t][col] * Vscale[t][b(d)])
//
// The columns are the query heads that share the KV head.  An fp32 query is
// two columns, its fp16 part and the fp16 part of the rest (22 bits), and so
// is its weight * Vscale; the two add up in one thread.  16-bit queries are
// one column (exact after scaling by a power of two), and so are their
// weights (one rounding to 11 bits, which fp16 and bf16 outputs do not see).
// To stay in fp16's range a query is scaled by the power of two that brings
// its largest element to 2^13, and a weight is 2^(score - M + KV4_BASE), where
// M follows the largest score + log2 of the tile's largest V scale whenever
// that has passed M by KV4_SLACK: weight * scale never passes 2^14, and loses
// nothing above 2^-32 of 2^KV4_BASE.  M is common to a warp, so following it
// takes shuffles and a rescaling of the sums: with the slack both are rare.
// In fp32 every unit's V product starts from zero and is added to the running
// sums outside: the tensor core cuts off where fp32 addition rounds, which
// 16-bit outputs do not see but long fp32 sums would.
//
// Unpacking a word of 8 codes: (w & 0xF000F) | 0x64006400 is 1024 + code in
// each half, (w & 0xF000F0) | ... 1024 + 16 * code; one fp16x2 subtraction or
// fma leaves code - 8.  ldmatrix gives a thread the K codes of 8 dimensions of
// one position, and transposed the V codes of 4 dimensions of two positions:
// both are the operand layouts of the products, in the stored order.
//
// Work is cut into units, 32 positions of one KV head of one sequence, and
// numbered sequence by sequence, head by head; a row (a sequence's KV head)
// opens with a place of its own, about what its queries cost.  Places are
// dealt out evenly: CTAs get equal runs of them, and within a CTA the warps
// do, whatever the lengths.
// Each warp streams its units through a ring of its own (16-byte asynchronous
// copies; no barrier between warps) and keeps its own softmax.  A row that several warps
// share is merged in shared memory, one that several CTAs share through the
// workspace by whichever CTA ends last, in the order of the CTAs, so that the
// result does not depend on timing.
//
// One sequence of 131089 positions, 8 KV heads of 128, fp32 queries: 43 us, of
// which 26 stream the 151 MB (5.8 TB/s), bound by the instructions that unpack
// and multiply (about 800 a unit and warp); 64 sequences of 1 to 4096: 50 us.
#define KV4_BASE 8.0f
#define KV4_SLACK 6.0f
#define KV4_UNIT 32
#define KV4_STAGES 2
#define KV4_MAX_CTAS 192

template <typename T> struct KvSplit { static constexpr int N = 1; };
template <> struct KvSplit<float> { static constexpr int N = 2; };

template <int NT> struct KvWarps { static constexpr int N = NT == 1 ? 16 : 8; };

template <typename T, int NB, int NT> struct KvShape {
    static constexpr int HD = NB * 32, P = KvSplit<T>::N, W = KvWarps<NT>::N;
    static constexpr int HG = 8 * NT / P;                 // query heads of a group
    static constexpr int STAGE = 36 * HD;                 // one unit: K codes, V codes, K scales, V scales
    static constexpr int ENTRY = HG * (HD + 2);           // a partial: per head the sums, M and the weights' sum
    static constexpr size_t heads = (size_t)W * ENTRY * 4, join = KV4_MAX_CTAS * HG * 4;
    // the rings; later the tail partials and what is joined across CTAs
    static constexpr size_t rings = (size_t)W * KV4_STAGES * STAGE, ring = rings > heads + join ? rings : heads + join;
    static constexpr size_t smem(int n) { return ring + heads + (size_t)(n + 1) * 4; }
};

__device__ __forceinline__ float kv4_ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void kv4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same from zero
__device__ __forceinline__ void kv4_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// Four nibbles of each half of w, minus 8, as fp16 pairs (low half, high
// half).  and-or as one lop3: left to itself the compiler makes two of it.
__device__ __forceinline__ uint32_t kv4_and_or(uint32_t x, uint32_t mask, uint32_t bits)
{
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
    return y;
}

struct KvMagic {
    uint32_t mask0, mask1, bits;
    __device__ __forceinline__ KvMagic()
    {
        // opaque, so that they stay in registers
        asm volatile("mov.u32 %0, 0x000F000F;\n\tmov.u32 %1, 0x00F000F0;\n\tmov.u32 %2, 0x64006400;" : "=r"(mask0), "=r"(mask1), "=r"(bits));
    }
    __device__ __forceinline__ void unpack(uint32_t w, uint32_t (&n)[4]) const
    {
        const __half2 off = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));     // 1032
        const __half2 six = __halves2half2(__ushort_as_half(0x2C00), __ushort_as_half(0x2C00));     // 1 / 16
        const __half2 low = __halves2half2(__ushort_as_half(0xD480), __ushort_as_half(0xD480));     // -72
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t x = w >> (8 * k), a = kv4_and_or(x, mask0, bits), b = kv4_and_or(x, mask1, bits);
            const __half2  p = __hsub2(*reinterpret_cast<const __half2 *>(&a), off);
            const __half2  q = __hfma2(*reinterpret_cast<const __half2 *>(&b), six, low);
            n[2 * k] = *reinterpret_cast<const uint32_t *>(&p);
            n[2 * k + 1] = *reinterpret_cast<const uint32_t *>(&q);
        }
    }
};

__device__ __forceinline__ uint32_t kv4_pack(__half lo, __half hi)
{
    return (uint32_t)__half_as_ushort(lo) | ((uint32_t)__half_as_ushort(hi) << 16);
}

__device__ __forceinline__ uint32_t kv4_turn(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Codes of blocks b, b + 1 (b + 1 < NB) or b alone for 16 positions:
// r[0], r[1] positions 0-7 and 8-15 of block b, r[2], r[3] of block b + 1.
template <bool TRANS, bool PAIR> __device__ __forceinline__ void kv4_ldsm(uint32_t (&r)[4], uint32_t addr)
{
    if (PAIR) {
        if (TRANS)
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
        else
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
    } else {
        if (TRANS)
            asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
                         : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
        else
            asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
                         : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
    }
}

__device__ __forceinline__ void kv4_cp16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// A place in the numbering: place u is sequence i of the list, row r of its
// KV heads and head groups, place j of the row's nu; place 0 opens the row
// (its queries are loaded), place j > 0 is unit j - 1.
struct KvCursor {
    int i, r, j, nu;
    int left;                                             // places of this warp's run from here on
};

template <typename T, int NB, int NT, int N>
__global__ void __launch_bounds__(KvWarps<NT>::N * 32, 1) k_kv4_attend(const KvAttendArgs a, const KvSeqs<N> list)
{
    using S = KvShape<T, NB, NT>;
    constexpr int HD = S::HD, P = S::P, W = S::W, HG = S::HG, STAGE = S::STAGE, ENTRY = S::ENTRY;
    constexpr int HL = NT * (P == 2 ? 1 : 2);             // query heads whose columns a thread holds
    extern __shared__ __align__(128) uint8_t smem[];
    float     *tails = reinterpret_cast<float *>(smem);   // after the loop: tail partials, in the ring's place
    float     *heads = reinterpret_cast<float *>(smem + S::ring);
    int       *pre = reinterpret_cast<int *>(smem + S::ring + S::heads);     // places of a row before sequence i
    __shared__ int       rid[2 * W];                      // the row of each warp's head and tail partial, -1: none
    __shared__ float     wgt[2 * W][HG], top_s[2 * W][HG];
    __shared__ unsigned  mates[2 * W], sums[W];
    __shared__ int       lead_s[2 * W], n_lead;
    __shared__ float     joinL[HG];
    __shared__ int       last_s[2], c0_s[2], np_s[2];     // of the rows shared with CTAs before and after
    float *joinW = tails + W * ENTRY;                     // the weights of a row's CTAs, behind the tails

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int n = list.n, n_grp = (a.n_rep + HG - 1) / HG, R = a.n_kv * n_grp;
    const int cap = a.max_pages * KV4_PAGE;
    uint8_t  *ring = smem + (size_t)warp * KV4_STAGES * STAGE;

    if (tid < 2 * W) rid[tid] = -1;
    pdl_wait();
    pdl_trigger();
    // places before each sequence: a scan over the list, PER sequences a thread
    {
        constexpr int PER = (N + W * 32 - 1) / (W * 32);
        int           c[PER], sum = 0;
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const int i = tid * PER + k;
            c[k] = i < n ? (min(max(__ldg(a.len + list.seq[i]), 0), cap) + KV4_UNIT - 1) / KV4_UNIT : 0;
        }
#pragma unroll
        for (int k = 0; k < PER; k++) {
            c[k] += c[k] > 0;
            sum += c[k];
        }
        int run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        if (lane == 31) sums[warp] = (unsigned)run;
        __syncthreads();
        run -= sum;
        for (int w = 0; w < warp; w++) run += (int)sums[w];
#pragma unroll
        for (int k = 0; k < PER; k++) {
            if (tid * PER + k <= n) pre[tid * PER + k] = run;
            run += c[k];
        }
        if (tid == W * 32 - 1 && n == W * 32 * PER) pre[n] = run;
    }
    __syncthreads();

    // an empty sequence's row is zeros
    for (int i = blockIdx.x; i < n; i += gridDim.x)
        if (pre[i + 1] == pre[i])
            for (int x = tid; x < a.n_kv * a.n_rep * HD; x += W * 32)
                ((T *)a.out)[(size_t)i * a.out_stride + x] = kv4_from<T>(0.0f);

    const int  total = pre[n] * R;                        // below 2^31: the host sees to it
    // CTAs with a run: none of them empty, since a shared row waits for a ticket from each
    const int  ctas = min((int)gridDim.x, total);
    const bool busy = (int)blockIdx.x < ctas;
    auto       begin_of = [&](int b) { return (int)((long long)total * b / ctas); };
    const int  cu0 = busy ? begin_of(blockIdx.x) : 0, cu1 = busy ? begin_of(blockIdx.x + 1) : 0;
    const int  u0 = cu0 + (int)((long long)(cu1 - cu0) * warp / W), u1 = cu0 + (int)((long long)(cu1 - cu0) * (warp + 1) / W);

    auto locate = [&](int u) {
        KvCursor p;
        int      lo = 0, hi = n;                          // the last sequence whose units begin at or before u
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] * R <= u) lo = mid;
            else hi = mid;
        }
        p.i = lo;
        p.nu = pre[lo + 1] - pre[lo];
        p.r = (u - pre[lo] * R) / p.nu;
        p.j = u - pre[lo] * R - p.r * p.nu;
        p.left = u1 - u;
        return p;
    };
    auto next = [&](KvCursor &p) {
        p.left--;
        if (++p.j < p.nu) return;
        p.j = 0;
        if (++p.r < R) return;
        p.r = 0;
        do p.i++;
        while (p.i < n && pre[p.i + 1] == pre[p.i]);
        p.nu = p.i < n ? pre[p.i + 1] - pre[p.i] : 1;
    };
    // the page of the first unit at or after p inside this warp's run; p moves there
    auto page_at = [&](KvCursor &p) {
        if (p.left > 0 && p.j == 0) next(p);
        return p.left > 0 ? __ldg(a.table + (size_t)list.seq[p.i] * a.max_pages + (p.j - 1) / (KV4_PAGE / KV4_UNIT)) : 0;
    };
    // the unit's pieces of its page, 16 bytes a lane and copy (from inside the pool whatever the table says)
    const bool     vside = lane >= 4 * NB;
    const uint32_t ring_lane = smem_addr(ring) + lane * 16;
    const uint8_t *code_lane = a.layer + lane * 16, *scale_lane = a.layer + 64 * HD + (vside ? 4 * HD : 0) + (lane - (vside ? 4 * NB : 0)) * 16;
    auto issue = [&](const KvCursor &p, int page, int k) {
        const size_t   at = (size_t)min(max(page, 0), a.n_pages - 1) * a.page_bytes + (unsigned)((n_grp == 1 ? p.r : p.r / n_grp) * 72 * HD);
        const int      half = (p.j - 1) & 1;
        const uint8_t *src = code_lane + at + half * 16 * HD;
        const uint32_t dst = ring_lane + k * STAGE;
#pragma unroll
        for (int x = 0; x < NB; x++) {
            kv4_cp16(dst + 512 * x, src + 512 * x);
            kv4_cp16(dst + 16 * HD + 512 * x, src + 32 * HD + 512 * x);
        }
        if (lane < 8 * NB) kv4_cp16(dst + 32 * HD, scale_lane + at + half * 2 * HD);
    };

    const KvMagic magic;
    uint32_t qf[NT][NB][4];                               // the query columns, as the products' B operands
    float    fac[HL];                                     // score * fac: in units of log2
    float    O[NT][NB][2][4], M[HL], l[HL];

    // row p's queries on their way into the cache, before load_q wants them
    auto fetch_q = [&](const KvCursor &p) {
        const int kvh = p.r / n_grp, grp = p.r - kvh * n_grp;
        const T  *q = (const T *)a.q + (size_t)p.i * a.q_stride + (size_t)(kvh * a.n_rep + grp * HG) * HD;
        for (int x = lane * (128 / (int)sizeof(T)); x < min(HG, a.n_rep - grp * HG) * HD; x += 32 * (128 / (int)sizeof(T)))
            asm volatile("prefetch.global.L1 [%0];" ::"l"(q + x));
    };
    // this lane's elements of the query columns of row p.r: column col is query
    // head HG * group + col / P
    auto read_q = [&](const KvCursor &p, float (&x)[NT][NB][8]) {
        const int kvh = p.r / n_grp, grp = p.r - kvh * n_grp;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int hh = grp * HG + (nt * 8 + g) / P;
            const T  *q = (const T *)a.q + (size_t)p.i * a.q_stride + (size_t)(kvh * a.n_rep + hh) * HD + 8 * c;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (hh < a.n_rep) kv4_load8(q + 32 * b, a.wide_q, x[nt][b]);
                else
#pragma unroll
                    for (int e = 0; e < 8; e++) x[nt][b][e] = 0.0f;
            }
        }
    };
    // them as the products' operands (column col: part col % P of its head's
    // query), and the row's softmax from nothing
    auto load_q = [&](const float (&xs)[NT][NB][8]) {
        float f[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int    col = nt * 8 + g;
            const float(&x)[NB][8] = xs[nt];
            float        m = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(x[b][e]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            // 2^sh brings m to [2^13, 2^14); held where both it and its inverse are normal numbers
            const int sh = min(126, max(-126, 140 - (int)((__float_as_uint(fmaxf(m, 1e-38f)) >> 23) & 255)));
            // (with the scale's sign, so that fac is not negative)
            const float up = copysignf(__uint_as_float((uint32_t)(sh + 127) << 23), a.scale);
            f[nt] = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - sh) << 23);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                __half h[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float y = x[b][e] * up;
                    h[e] = __float2half_rn(y);
                    if (P == 2 && (col & 1)) h[e] = __float2half_rn(y - __half2float(h[e]));
                }
#pragma unroll
                for (int k = 0; k < 4; k++) qf[nt][b][k] = kv4_pack(h[k], h[k + 4]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            if (P == 2) fac[nt] = __shfl_sync(0xffffffffu, f[nt], 8 * c);
            else {
                fac[2 * nt] = __shfl_sync(0xffffffffu, f[nt], 8 * c);
                fac[2 * nt + 1] = __shfl_sync(0xffffffffu, f[nt], 8 * c + 4);
            }
        }
#pragma unroll
        for (int h = 0; h < HL; h++) {
            M[h] = -INFINITY;
            l[h] = 0.0f;
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int k = 0; k < 4; k++) O[nt][b][0][k] = O[nt][b][1][k] = 0.0f;
    };
    // NB fp16 scales of one position, as pairs
    auto scales = [&](const uint8_t *base, int t, uint32_t (&w)[(NB + 1) / 2]) {
        if (NB == 4) {
            const uint2 v = *reinterpret_cast<const uint2 *>(base + t * 8);
            w[0] = v.x;
            w[(NB + 1) / 2 - 1] = v.y;
        } else if (NB == 2) {
            w[0] = *reinterpret_cast<const uint32_t *>(base + t * 4);
        } else {
            const uint16_t *p = reinterpret_cast<const uint16_t *>(base) + t * NB;
#pragma unroll
            for (int k = 0; k < (NB + 1) / 2; k++) w[k] = (uint32_t)p[2 * k] | (2 * k + 1 < NB ? (uint32_t)p[2 * k + 1] << 16 : 0u);
        }
    };
    auto half_of = [](uint32_t w, int k) {
        const __half2 h = *reinterpret_cast<const __half2 *>(&w);
        return k ? __high2float(h) : __low2float(h);
    };
    const int mt_row = (lane & 7) + ((lane >> 3) & 1) * 8, mt_blk = lane >> 4;     // this lane's row of an ldmatrix

    // One unit.  left: positions of it inside the sequence; CUT: not all are
    auto unit = [&](const uint8_t *st, int left, auto cut) {
        constexpr bool CUT = decltype(cut)::value;
        constexpr int  MT = KV4_UNIT / 16;
        const uint32_t kaddr = smem_addr(st), vaddr = kaddr + 16 * HD;
        float          sc[MT][2][HL];
        uint32_t       vs[MT][2][(NB + 1) / 2];
        float          top[HL];
        __half2        vm = __float2half2_rn(0.0f);
#pragma unroll
        for (int h = 0; h < HL; h++) top[h] = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float acc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int k = 0; k < 4; k++) acc[nt][k] = 0.0f;
            const int t = mt * 16 + g, t2 = mt * 16 + mt_row;
            uint32_t  ks0[(NB + 1) / 2], ks1[(NB + 1) / 2];
            scales(st + 32 * HD, t, ks0);
            scales(st + 32 * HD, t + 8, ks1);
            scales(st + 34 * HD, t, vs[mt][0]);
            scales(st + 34 * HD, t + 8, vs[mt][1]);
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                uint32_t r[4];
                if (b + 1 < NB) kv4_ldsm<false, true>(r, kaddr + t2 * (HD / 2) + kv4_place(t2, b + mt_blk, NB) * 16);
                else kv4_ldsm<false, false>(r, kaddr + t2 * (HD / 2) + kv4_place(t2, b, NB) * 16);
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    if (b + d >= NB) continue;
                    uint32_t x[4], y[4];
                    magic.unpack(r[2 * d], x);
                    magic.unpack(r[2 * d + 1], y);
                    const float s0 = half_of(ks0[(b + d) / 2], (b + d) & 1), s1 = half_of(ks1[(b + d) / 2], (b + d) & 1);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float e[4];
                        kv4_mma0(e, x[0], y[0], x[1], y[1], qf[nt][b + d][0], qf[nt][b + d][1]);
                        kv4_mma(e, x[2], y[2], x[3], y[3], qf[nt][b + d][2], qf[nt][b + d][3]);
                        acc[nt][0] = fmaf(s0, e[0], acc[nt][0]);
                        acc[nt][1] = fmaf(s0, e[1], acc[nt][1]);
                        acc[nt][2] = fmaf(s1, e[2], acc[nt][2]);
                        acc[nt][3] = fmaf(s1, e[3], acc[nt][3]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < HL; h++) {
                const int nt = P == 2 ? h : h >> 1, k = h & 1;
                sc[mt][0][h] = P == 2 ? acc[nt][0] + acc[nt][1] : acc[nt][k];
                sc[mt][1][h] = P == 2 ? acc[nt][2] + acc[nt][3] : acc[nt][2 + k];
                if (!CUT || t < left) top[h] = fmaxf(top[h], sc[mt][0][h]);
                if (!CUT || t + 8 < left) top[h] = fmaxf(top[h], sc[mt][1][h]);
            }
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int k = 0; k < (NB + 1) / 2; k++) {
                    if (CUT && t + 8 * x >= left) vs[mt][x][k] = 0u;      // whatever lies past the end
                    vm = __hmax2(vm, __habs2(*reinterpret_cast<const __half2 *>(&vs[mt][x][k])));
                }
        }
        // this thread's V scales are below 2^ve (scales below 2^-24 are zeros)
        float       vmax = fmaxf(__low2float(vm), __high2float(vm));
        const float ve = (float)max((int)(__float_as_uint(vmax) >> 23) - 126, -24);
        bool        calm = true;
#pragma unroll
        for (int h = 0; h < HL; h++) {
            top[h] *= fac[h];
            calm = calm && top[h] + ve <= M[h] + KV4_SLACK;
        }
        if (!__all_sync(0xffffffffu, calm)) {
            // M follows the largest score + log2 of the largest V scale
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
#pragma unroll
                for (int h = 0; h < HL; h++) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
            }
            const float vw = (float)max((int)(__float_as_uint(vmax) >> 23) - 126, -24);
            float       alpha[HL];
#pragma unroll
            for (int h = 0; h < HL; h++) {
                const float m = fmaxf(M[h], top[h] + vw);
                alpha[h] = kv4_ex2(M[h] - m);
                M[h] = m;
                l[h] *= alpha[h];
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        O[nt][b][0][k] *= alpha[P == 2 ? nt : 2 * nt + (k & 1)];
                        O[nt][b][1][k] *= alpha[P == 2 ? nt : 2 * nt + (k & 1)];
                    }
        }
#pragma unroll
        for (int h = 0; h < HL; h++) {
            const float base = KV4_BASE - M[h];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    sc[mt][x][h] = kv4_ex2(fmaf(sc[mt][x][h], fac[h], base));
                    if (CUT && mt * 16 + g + 8 * x >= left) sc[mt][x][h] = 0.0f;
                    l[h] += sc[mt][x][h];
                }
        }
#pragma unroll
        for (int b = 0; b < NB; b += 2) {
            uint32_t r[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                const int t2 = mt * 16 + mt_row;
                if (b + 1 < NB) kv4_ldsm<true, true>(r[mt], vaddr + t2 * (HD / 2) + kv4_place(t2, b + mt_blk, NB) * 16);
                else kv4_ldsm<true, false>(r[mt], vaddr + t2 * (HD / 2) + kv4_place(t2, b, NB) * 16);
            }
#pragma unroll
            for (int d = 0; d < 2; d++) {
                if (b + d >= NB) continue;
                float e[NT][2][4];
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    uint32_t x[4], y[4];
                    magic.unpack(r[mt][2 * d], x);
                    magic.unpack(r[mt][2 * d + 1], y);
                    const float v0 = half_of(vs[mt][0][(b + d) / 2], (b + d) & 1), v1 = half_of(vs[mt][1][(b + d) / 2], (b + d) & 1);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        uint32_t p0, p1;
                        if (P == 2) {
                            const float    w0 = sc[mt][0][nt] * v0, w1 = sc[mt][1][nt] * v1;
                            const __half2  hi = __floats2half2_rn(w0, w1);
                            const __half2  lo = __floats2half2_rn(w0 - __low2float(hi), w1 - __high2float(hi));
                            const uint32_t hb = *reinterpret_cast<const uint32_t *>(&hi), lb = *reinterpret_cast<const uint32_t *>(&lo);
                            p0 = __byte_perm(hb, lb, 0x5410);
                            p1 = __byte_perm(hb, lb, 0x7632);
                        } else {
                            const __half2 h0 = __floats2half2_rn(sc[mt][0][2 * nt] * v0, sc[mt][0][(2 * nt + 1) % HL] * v0);
                            const __half2 h1 = __floats2half2_rn(sc[mt][1][2 * nt] * v1, sc[mt][1][(2 * nt + 1) % HL] * v1);
                            p0 = *reinterpret_cast<const uint32_t *>(&h0);
                            p1 = *reinterpret_cast<const uint32_t *>(&h1);
                        }
                        const uint32_t b0 = kv4_turn(p0), b1 = kv4_turn(p1);
                        if (P == 1) {
                            kv4_mma(O[nt][b + d][0], x[0], x[1], y[0], y[1], b0, b1);
                            kv4_mma(O[nt][b + d][1], x[2], x[3], y[2], y[3], b0, b1);
                        } else if (mt == 0) {
                            kv4_mma0(e[nt][0], x[0], x[1], y[0], y[1], b0, b1);
                            kv4_mma0(e[nt][1], x[2], x[3], y[2], y[3], b0, b1);
                        } else {
                            kv4_mma(e[nt][0], x[0], x[1], y[0], y[1], b0, b1);
                            kv4_mma(e[nt][1], x[2], x[3], y[2], y[3], b0, b1);
                        }
                    }
                }
                if (P == 2)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            O[nt][b + d][0][k] += e[nt][0][k];
                            O[nt][b + d][1][k] += e[nt][1][k];
                        }
            }
        }
    };
    // f(head of the group, dimension, sum) for what this thread holds of the row
    auto each = [&](auto f) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const float *o = O[nt][b][s];
                    const int    d = 32 * b + 4 * g + 2 * s;
                    if (P == 2) {
                        f(nt * 4 + c, nt, d, o[0] + o[1]);
                        f(nt * 4 + c, nt, d + 1, o[2] + o[3]);
                    } else {
                        f(nt * 8 + 2 * c, 2 * nt, d, o[0]);
                        f(nt * 8 + 2 * c, 2 * nt, d + 1, o[2]);
                        f(nt * 8 + 2 * c + 1, (2 * nt + 1) % HL, d, o[1]);
                        f(nt * 8 + 2 * c + 1, (2 * nt + 1) % HL, d + 1, o[3]);
                    }
                }
    };
    auto store_part = [&](float *e) {
        each([&](int h, int, int d, float v) { e[h * (HD + 2) + d] = v; });
        if (g == 0)
#pragma unroll
            for (int h = 0; h < HL; h++) {
                const int hh = P == 2 ? h * 4 + c : (h >> 1) * 8 + 2 * c + (h & 1);
                e[hh * (HD + 2) + HD] = M[h];
                e[hh * (HD + 2) + HD + 1] = l[h];
            }
    };
    auto sum_l = [&] {
#pragma unroll
        for (int h = 0; h < HL; h++)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
    };

    bool tail = false;                                    // this warp ends inside a row that began in its run
    if (u0 < u1) {
        KvCursor at = locate(u0), ahead = at;
        KvCursor first[KV4_STAGES];
        int      page[KV4_STAGES + 1];
        float    xq[NT][NB][8];
        read_q(at, xq);                                   // (all of these loads are in flight together)
#pragma unroll
        for (int k = 0; k < KV4_STAGES; k++) {            // independent loads
            page[k] = page_at(ahead);
            first[k] = ahead;
            if (ahead.left > 0) next(ahead);
        }
        page[KV4_STAGES] = page_at(ahead);                // of the unit that is issued next
#pragma unroll
        for (int k = 0; k < KV4_STAGES; k++) {
            if (first[k].left > 0) issue(first[k], page[k], k);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        load_q(xq);
        int      j0 = at.j, k = 0, len = min(__ldg(a.len + list.seq[at.i]), cap);
        for (;;) {
            if (at.j > 0) {
                asm volatile("cp.async.wait_group %0;" ::"n"(KV4_STAGES - 1) : "memory");
                __syncwarp();
                const int left = len - (at.j - 1) * KV4_UNIT;
                if (left >= KV4_UNIT) unit(ring + (size_t)k * STAGE, left, std::false_type());
                else unit(ring + (size_t)k * STAGE, left, std::true_type());
                __syncwarp();
                if (ahead.left > 0) {
                    issue(ahead, page[KV4_STAGES], k);
                    next(ahead);
                    if (ahead.j == 0 && ahead.left > 0) fetch_q(ahead);
                    page[KV4_STAGES] = page_at(ahead);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                k = k + 1 == KV4_STAGES ? 0 : k + 1;
            }
            const bool row_end = at.j + 1 == at.nu, run_end = at.left == 1;
            if (!row_end && !run_end) {
                at.j++;
                at.left--;
                continue;
            }
            sum_l();
            const int row = at.i * R + at.r;
            if (j0 > 0) {
                store_part(heads + warp * ENTRY);
                if (lane == 0) rid[2 * warp] = row;
            } else if (!row_end) {
                tail = true;
                if (lane == 0) rid[2 * warp + 1] = row;
            } else {
                const int kvh = at.r / n_grp, grp = at.r - kvh * n_grp;
                T        *o = (T *)a.out + (size_t)at.i * a.out_stride + (size_t)kvh * a.n_rep * HD;
#pragma unroll
                for (int h = 0; h < HL; h++) l[h] = __frcp_rn(l[h]);
                each([&](int h, int hl, int d, float v) {
                    if (grp * HG + h < a.n_rep) o[(size_t)(grp * HG + h) * HD + d] = kv4_from<T>(v * l[hl]);
                });
            }
            if (run_end) break;
            next(at);
            j0 = 0;
            float x2[NT][NB][8];
            read_q(at, x2);
            load_q(x2);
            len = min(__ldg(a.len + list.seq[at.i]), cap);
        }
    }
    __syncthreads();                                      // every ring is idle
    if (tail) store_part(tails + warp * ENTRY);
    // meanwhile: the rows that this CTA shares with others, slot 0 the one that
    // began before its run, slot 1 the one that goes on after it, and their CTAs
    if (lane < 2 && warp == W - 1) {
        np_s[lane] = last_s[lane] = 0;
        if (busy) {
            const KvCursor p = locate(lane ? cu1 - 1 : cu0);
            const int      first = pre[p.i] * R + p.r * p.nu, end = first + p.nu;
            if ((lane ? first >= cu0 : first < cu0) && (first < cu0 || end > cu1)) {
                auto cta_of = [&](int u) {
                    int b = (int)((long long)u * ctas / total);
                    while (begin_of(b + 1) <= u) b++;
                    while (begin_of(b) > u) b--;
                    return b;
                };
                c0_s[lane] = cta_of(first);
                np_s[lane] = cta_of(end - 1) - c0_s[lane] + 1;
            }
        }
    }
    __syncthreads();

    // Rows that this CTA's warps share.  A partial's weight is 2^(its M - the
    // row's M); one without a unit (its sums are zeros) has none.  M follows
    // what is no NaN: a partial of NaN scores alone has M = -inf, weight 0 and
    // sums of NaN.
    auto entry = [&](int e) { return (e & 1) ? tails + (e >> 1) * ENTRY : heads + (e >> 1) * ENTRY; };
    auto weight = [](float M, float m, float l) { return l == 0.0f ? 0.0f : kv4_ex2(M - m); };
    auto write = [&](int row, int x, float v) {
        const int i = row / R, r = row - i * R, kvh = r / n_grp, grp = r - kvh * n_grp, h = grp * HG + x / HD;
        if (h < a.n_rep)
            ((T *)a.out)[(size_t)i * a.out_stride + (size_t)(kvh * a.n_rep + h) * HD + x % HD] = kv4_from<T>(v);
    };
    if (warp < HG) {                                      // a warp per head, a lane per partial
        const int      row = lane < 2 * W ? rid[lane % (2 * W)] : -1;
        const unsigned same = __match_any_sync(0xffffffffu, row);
        const float   *e = entry(lane % (2 * W)) + warp * (HD + 2) + HD;
        const float    M = row >= 0 ? e[0] : -INFINITY;
        // floats in the order of their bits as whole numbers
        const int      bits = __float_as_int(M), key = bits ^ ((bits >> 31) & 0x7FFFFFFF);
        const int      most = __reduce_max_sync(same, key);
        const float    m = __int_as_float(most ^ ((most >> 31) & 0x7FFFFFFF));
        if (lane < 2 * W) {
            wgt[lane][warp] = row >= 0 ? weight(M, m, e[1]) : 0.0f;
            top_s[lane][warp] = m;
            mates[lane] = same;
        }
        const bool     first = row >= 0 && __ffs(same) - 1 == lane;
        const unsigned lead = __ballot_sync(0xffffffffu, first);
        if (warp == 0 && first) lead_s[__popc(lead & ((1u << lane) - 1))] = lane;
        if (tid == 0) n_lead = __popc(lead);
    }
    __syncthreads();
    // a warp per row and head, or, of few rows, per 32 dimensions of one
    const int span = n_lead * HG >= W ? NB : 1, parts = NB / span;
    for (int task = warp; task < n_lead * HG * parts; task += W) {
        const int      e = lead_s[task / (HG * parts)], row = rid[e];
        const unsigned own = mates[e];                    // the row's places
        const int      end = 32 - __clz(own);
        const int i = row / R, nu = pre[i + 1] - pre[i], first = pre[i] * R + (row - i * R) * nu;
        const bool whole = first >= cu0 && first + nu <= cu1;
        const int  h = task / parts % HG, d0 = task % parts * 32 + lane;
        float      L = 0.0f, v[NB];
#pragma unroll
        for (int x = 0; x < NB; x++) v[x] = 0.0f;
#pragma unroll 4
        for (int k = e; k < end; k++) {
            const float  w = wgt[k][h];
            const float *from = entry(k) + h * (HD + 2);
            if (own >> k & 1u) {                          // (an unused place holds anything; a weight of 0 does
                                                          // not take a place out: 0 * NaN is NaN)
                L = fmaf(w, from[HD + 1], L);
#pragma unroll
                for (int x = 0; x < NB; x++)
                    if (x < span) v[x] = fmaf(w, from[d0 + 32 * x], v[x]);
            }
        }
        if (whole) {
            const float inv = 1.0f / L;
            const int   r = row - i * R, kvh = r / n_grp, hh = (r - kvh * n_grp) * HG + h;
            if (hh < a.n_rep)
#pragma unroll
                for (int x = 0; x < NB; x++)
                    if (x < span)
                        ((T *)a.out)[(size_t)i * a.out_stride + (size_t)(kvh * a.n_rep + hh) * HD + d0 + 32 * x] = kv4_from<T>(v[x] * inv);
        } else {                                          // sums [HG][HD], then M and the weights' sum of each head
            float *out = a.part + ((size_t)blockIdx.x * 2 + (first >= cu0)) * ENTRY;
#pragma unroll
            for (int x = 0; x < NB; x++)
                if (x < span) out[h * HD + d0 + 32 * x] = v[x];
            if (d0 == 0) {
                out[HG * HD + h] = top_s[e][h];
                out[HG * HD + HG + h] = L;
            }
        }
    }
    if (np_s[0] == 0 && np_s[1] == 0) return;
    __syncthreads();
    // a ticket for each shared row (released after, and acquired before, the partials)
    if (lane == 0 && warp < 2 && np_s[warp]) {
        unsigned t;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(t) : "l"(a.count + c0_s[warp]) : "memory");
        last_s[warp] = t == (unsigned)(np_s[warp] - 1);
    }
    __syncthreads();
    for (int s = 0; s < 2; s++) {
        if (!last_s[s]) continue;
        // GR partials at a time, four sums a thread, up to eight partials in flight
        constexpr int V4 = HG * HD / 4, GR = W * 32 / V4;
        const int     c0 = c0_s[s], np = np_s[s], grp = tid / V4, x4 = tid % V4;
        auto          part = [&](int b) { return a.part + ((size_t)(c0 + b) * 2 + (b == 0)) * ENTRY; };
        float4        v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int b = grp + k * GR;
            v[k] = grp < GR && b < np ? __ldcg(reinterpret_cast<const float4 *>(part(b)) + x4) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (warp < HG) {
            float m = -INFINITY, L = 0.0f;
            for (int b = lane; b < np; b += 32) m = fmaxf(m, __ldcg(part(b) + HG * HD + warp));
#pragma unroll
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            for (int b = lane; b < np; b += 32) {
                const float ln = __ldcg(part(b) + HG * HD + HG + warp), w = weight(__ldcg(part(b) + HG * HD + warp), m, ln);
                joinW[b * HG + warp] = w;
                L = fmaf(w, ln, L);
            }
            L = warp_sum(L);
            if (lane == 0) joinL[warp] = L;
        }
        __syncthreads();
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int b0 = 0; b0 < np; b0 += 8 * GR) {
            if (b0)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int b = b0 + grp + k * GR;
                    if (grp < GR && b < np) v[k] = __ldcg(reinterpret_cast<const float4 *>(part(b)) + x4);
                }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int b = b0 + grp + k * GR;
                if (grp < GR && b < np) {
                    const float w = joinW[b * HG + x4 * 4 / HD];
                    sum.x = fmaf(w, v[k].x, sum.x);
                    sum.y = fmaf(w, v[k].y, sum.y);
                    sum.z = fmaf(w, v[k].z, sum.z);
                    sum.w = fmaf(w, v[k].w, sum.w);
                }
            }
        }
        if (grp < GR) reinterpret_cast<float4 *>(heads)[tid] = sum;
        __syncthreads();
        const KvCursor p = locate(s ? cu1 - 1 : cu0);
        for (int x = tid; x < HG * HD; x += W * 32) {
            float y = 0.0f;
#pragma unroll
            for (int k = 0; k < GR; k++) y += heads[k * HG * HD + x];
            write(p.i * R + p.r, x, y / joinL[x / HD]);
        }
        if (tid == 0) a.count[c0] = 0;                    // as the next call finds it
        __syncthreads();
    }
}
