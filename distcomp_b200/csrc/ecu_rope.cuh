// ecu_rope.cuh -- rows turned by their positions and appended to the paged
// 4-bit cache (layout: engine_cuda.h) in one pass.
//
// Pair i of a head turns by the angle pos * w_i.  The angle is kept in whole
// turns: pos * (w_i / 2 pi * 2^64) modulo 2^64 is the fraction of a turn, exact
// however far the position, in one 64-bit product (2^-65 turns a position from
// w_i itself); no table, and no angle that grows.
//
// A 4-bit code changes by a whole step where the turned key crosses the border
// between two codes, so a key is turned and quantised in 64 bits: its code is
// that of the exact value but for one in about 10^14, and the same from every
// implementation.  A query is turned in 32 bits and rounded once.
#pragma once
#include "ecu_kv4.cuh"

// What a rotation needs, by value in the kernel's arguments.
struct RopeTurns {
    int                rot, interleaved;
    double             factor;
    unsigned long long turn[64];
};

struct RopeArgs {
    KvAppendArgs kv;
    const void  *q;               // nullptr: keys alone
    void        *q_out;
    long         q_stride, q_out_stride;
    const int   *depth;           // nullptr: rows stand one behind the other
    int          n_rep, heads;    // query heads a KV head, KV heads of a block
    int          rows;            // rows of a block
    bool         wide_q;
    RopeTurns    turns;
};

// Up to eight consecutive elements (n of them; the others zero).
template <typename T> __device__ __forceinline__ void rope_load(const T *p, int n, bool wide, float (&x)[8])
{
    if (n >= 8) {
        if (wide) {
            __align__(16) T v[8];
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) reinterpret_cast<uint4 *>(v)[i] = reinterpret_cast<const uint4 *>(p)[i];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = kv4_float(v[i]);
            return;
        }
        n = 8;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = i < n ? kv4_float(p[i]) : 0.0f;
}

template <typename T> __device__ __forceinline__ void rope_store(T *p, int n, bool wide, const float (&x)[8])
{
    if (n >= 8 && wide) {
        kv4_store8(p, true, x);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < n) p[i] = kv4_from<T>(x[i]);
}

__device__ __forceinline__ double kv4_shfl_xor(unsigned mask, double v, int o)
{
    return __hiloint2double(__shfl_xor_sync(mask, __double2hiint(v), o), __shfl_xor_sync(mask, __double2loint(v), o));
}

// kv4_quantise of values of 64 bits.
__device__ __forceinline__ uint32_t kv4_quantise64(const double (&x)[8], unsigned mask, int c, __half &dh, float (&y)[8])
{
    double m = 0.0;                                              // the value of largest magnitude, the first of equals
    bool   fine = true;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        fine = fine && fabs(x[i]) < INFINITY;
        if (fabs(x[i]) > fabs(m)) m = x[i];
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const double w = kv4_shfl_xor(mask, m, o);
        if (fabs(w) > fabs(m) || (fabs(w) == fabs(m) && (c & o))) m = w;      // (of equals that of the lower lane)
    }
    fine = (__ballot_sync(mask, fine) & mask) == mask;
    dh = __double2half(fmin(fmax(m * -0.125, -65504.0), 65504.0));
    if (!fine) dh = __ushort_as_half(0x7FFF);
    else if (__half2float(dh) == 0.0f) dh = __ushort_as_half(0);
    const double d = (double)__half2float(dh), inv = d != 0.0 ? 1.0 / d : 0.0, half = d != 0.0 ? 0.5 * fabs(d) : INFINITY;
    uint32_t     w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        // k of (k - 1/2) |d| <= u < (k + 1/2) |d|, u = x * sign(d): a guess, settled by the rest
        double       k = rint(x[i] * inv);
        const double r = copysign(1.0, d) * fma(-k, d, x[i]);
        if (r >= half) k += 1.0;
        else if (r < -half) k -= 1.0;
        k = fmin(fmax(k, -8.0), 7.0);
        w |= (uint32_t)(8 + (int)k) << (4 * i);
        y[i] = (float)(k * d);
    }
    return fine ? w : 0x88888888u;
}

// A block takes a.rows rows and a.heads KV heads with their query heads: the
// angles' cosines and sines into shared memory, then the queries turned, and
// the keys, which wait in shared memory (a block of 32 dimensions and its
// partners may lie in different threads), then codes for K and V, four lanes to
// a block of 32 dimensions.
template <typename T, typename O, int N>
__global__ void __launch_bounds__(256) k_kv4_append_rope(const __grid_constant__ RopeArgs a, const __grid_constant__ KvRows<N> rows)
{
    extern __shared__ __align__(16) double rope_sm[];
    __shared__ int s_seq[64], s_pos[64];
    pdl_wait();
    pdl_trigger();
    const int hd = a.kv.nb * 32, rot = a.turns.rot, half = rot / 2, tid = threadIdx.x;
    const int chunks = (a.kv.n_kv + a.heads - 1) / a.heads;
    const int r0 = (int)(blockIdx.x / chunks) * a.rows, h0 = (int)(blockIdx.x % chunks) * a.heads;
    const int nr = min(a.rows, rows.row0[rows.n] - r0), nh = min(a.heads, a.kv.n_kv - h0);
    double2  *cs = reinterpret_cast<double2 *>(rope_sm);         // [rows][half]
    double   *ks = rope_sm + 2 * a.rows * half;                  // [rows][heads][hd]
    // where each row stands
    if (tid < nr) {
        const int r = r0 + tid;
        int       lo = 0, hi = rows.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (rows.row0[mid] <= r) lo = mid;
            else hi = mid;
        }
        s_seq[tid] = rows.seq[lo];
        s_pos[tid] = __ldg(a.kv.len + rows.seq[lo]) - (rows.row0[lo + 1] - r);
    }
    for (int x = tid; x < nr * half; x += 256) {
        const int r = r0 + x / half, i = x % half;
        int       lo = 0, hi = rows.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (rows.row0[mid] <= r) lo = mid;
            else hi = mid;
        }
        const int       first = __ldg(a.kv.len + rows.seq[lo]) - (rows.row0[lo + 1] - rows.row0[lo]);
        const long long pos = (long long)first + (a.depth ? __ldg(a.depth + r) : r - rows.row0[lo]);
        const long long turn = (long long)((unsigned long long)pos * a.turns.turn[i]);
        double          s, c;
        sincospi((double)turn * 0x1p-63, &s, &c);
        cs[x] = make_double2(c * a.turns.factor, s * a.turns.factor);
    }
    __syncthreads();
    // slices: eight pairs each, then eight dimensions each of those that do not turn
    const int  n_pair = (half + 7) / 8, n_rest = (hd - rot + 7) / 8, per_head = n_pair + n_rest;
    const bool even = half % 8 == 0;                             // slices begin at multiples of eight elements
    const int  q_heads = a.q ? nh * a.n_rep : 0, all = q_heads + nh;
    for (int x = tid; x < nr * all * per_head; x += 256) {
        const int  sl = x % per_head, hh = x / per_head % all, r = x / (per_head * all);
        const bool is_q = hh < q_heads;
        const T   *p = is_q ? (const T *)a.q + (size_t)(r0 + r) * a.q_stride + (size_t)(h0 * a.n_rep + hh) * hd
                            : (const T *)a.kv.k + (size_t)(r0 + r) * a.kv.k_stride + (size_t)(h0 + hh - q_heads) * hd;
        T         *o = is_q ? (T *)a.q_out + (size_t)(r0 + r) * a.q_out_stride + (size_t)(h0 * a.n_rep + hh) * hd : nullptr;
        double    *kd = ks + ((size_t)r * a.heads + (hh - q_heads)) * hd;
        const bool wide = even && (is_q ? a.wide_q : a.kv.wide);
        float      u[8], v[8];
        if (sl >= n_pair) {
            const int d = rot + 8 * (sl - n_pair), n = hd - d;
            rope_load(p + d, n, wide, u);
            if (is_q) rope_store(o + d, n, wide, u);
            else
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < n) kd[d + i] = (double)u[i];
            continue;
        }
        const int      i0 = 8 * sl, n = min(8, half - i0);
        const double2 *t = cs + r * half + i0;
        if (a.turns.interleaved) {
            rope_load(p + 2 * i0, 2 * n, wide, u);
            rope_load(p + 2 * i0 + 8, 2 * n - 8, wide, v);
            if (is_q) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const double2 e = t[min(i, n - 1)];
                    const float   c = (float)e.x, s = (float)e.y;
                    float        &p0 = i < 4 ? u[2 * (i & 3)] : v[2 * (i & 3)], &p1 = i < 4 ? u[2 * (i & 3) + 1] : v[2 * (i & 3) + 1];
                    const float   y0 = fmaf(p0, c, -p1 * s), y1 = fmaf(p1, c, p0 * s);
                    p0 = y0;
                    p1 = y1;
                }
                rope_store(o + 2 * i0, 2 * n, wide, u);
                rope_store(o + 2 * i0 + 8, 2 * n - 8, wide, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (i >= n) continue;
                    const double2 e = t[i];
                    const double  p0 = i < 4 ? u[2 * (i & 3)] : v[2 * (i & 3)], p1 = i < 4 ? u[2 * (i & 3) + 1] : v[2 * (i & 3) + 1];
                    kd[2 * (i0 + i)] = fma(p0, e.x, -p1 * e.y);
                    kd[2 * (i0 + i) + 1] = fma(p1, e.x, p0 * e.y);
                }
            }
        } else {
            rope_load(p + i0, n, wide, u);
            rope_load(p + half + i0, n, wide, v);
            if (is_q) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const double2 e = t[min(i, n - 1)];
                    const float   c = (float)e.x, s = (float)e.y, y0 = fmaf(u[i], c, -v[i] * s), y1 = fmaf(v[i], c, u[i] * s);
                    u[i] = y0;
                    v[i] = y1;
                }
                rope_store(o + i0, n, wide, u);
                rope_store(o + half + i0, n, wide, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (i >= n) continue;
                    const double2 e = t[i];
                    kd[i0 + i] = fma((double)u[i], e.x, -(double)v[i] * e.y);
                    kd[half + i0 + i] = fma((double)v[i], e.x, (double)u[i] * e.y);
                }
            }
        }
    }
    __syncthreads();
    const int blocks = nh * a.kv.nb, groups = nr * blocks;       // of four lanes
    for (int g0 = 0; g0 < groups; g0 += 64) {
        const int      g = g0 + tid / 4, c = tid & 3;
        const unsigned mask = 0xFu << (tid & 28);
        if (g >= groups) continue;                               // whole groups of four
        const int  r = g / blocks, hb = g - r * blocks, h = hb / a.kv.nb, b = hb - h * a.kv.nb;
        const int  pos = s_pos[r], t = pos & (KV4_PAGE - 1);
        const bool placed = pos >= 0 && pos < a.kv.max_pages * KV4_PAGE;
        const int  page = placed ? __ldg(a.kv.table + (size_t)s_seq[r] * a.kv.max_pages + pos / KV4_PAGE) : -1;
        const bool wr = (unsigned)page < (unsigned)a.kv.n_pages; // no page: nothing to write to
        uint8_t   *p = a.kv.layer + (size_t)(wr ? page : 0) * a.kv.page_bytes + (size_t)(h0 + h) * 72 * hd;
        const size_t at = (size_t)(h0 + h) * hd + 32 * b + 8 * c, out = (size_t)(r0 + r) * a.kv.n_kv * hd + at;
        float      y[8], xv[8];
        __half     d;
        kv4_load8((const T *)a.kv.v + (size_t)(r0 + r) * a.kv.v_stride + at, a.kv.wide, xv);
        double     xk[8];
#pragma unroll
        for (int i = 0; i < 8; i++) xk[i] = ks[((size_t)r * a.heads + h) * hd + 32 * b + 8 * c + i];
#pragma unroll
        for (int side = 0; side < 2; side++) {
            const uint32_t w = side ? kv4_quantise(xv, mask, c, d, y) : kv4_quantise64(xk, mask, c, d, y);
            if (a.kv.k_out) kv4_store8((O *)(side ? a.kv.v_out : a.kv.k_out) + out, a.kv.wide_out, y);
            if (!wr) continue;
            *reinterpret_cast<uint32_t *>(p + side * 32 * hd + t * (hd / 2) + kv4_place(t, b, a.kv.nb) * 16 + 4 * c) = w;
            if (c == 0) *reinterpret_cast<__half *>(p + 64 * hd + side * 4 * hd + (t * a.kv.nb + b) * 2) = d;
        }
    }
}
