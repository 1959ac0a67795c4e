// ecu_rope.cuh -- rows turned by their positions and appended to the paged
// 4-bit cache (layout: engine_cuda.h) in one pass.
//
// Pair i of a head turns by the angle pos * w_i.  The angle is kept in whole
// turns: pos * (w_i / 2 pi * 2^64) modulo 2^64 is the fraction of a turn, exact
// however far the position, in one 64-bit product (2^-65 turns a position from
// w_i itself); no table, and no angle that grows.
//
// A 4-bit code changes by a whole step where the turned key crosses the border
// between two codes.  So a key is turned in pairs of floats (the products and
// their sum with what they round off, cosine and sine of 48 bits): about 2^-46
// of its pair's size, and its code is that of the exact value but for one in
// some 10^12, the same from every implementation.  What such a pair of floats
// cannot decide at a glance (a block whose largest values differ in sign alone,
// a scale halfway between two fp16 numbers, subnormal scales) is decided in
// 64-bit arithmetic.  A query is turned in 32 bits and rounded once.
//
// The latency of a block's phases bounds long calls (angles, turned pairs, codes:
// three barriers for four rows, with 44 % of the warps there could be): 8310 rows
// of 7 prompts (32 query and 8 KV heads of 128, bf16, the stored values handed
// back) take 73 us, where their 214 MB take 33 at the rate of a copy; 44 million
// warp instructions use 56 % of the issue slots.  Keys in 64-bit arithmetic
// throughout took 149.  One row of each of 64 sequences takes 13 us, the host's
// call.
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

// A key as it turned: h + l, |l| at most half a step of h.
struct RopePair {
    float h, l;
};

// x0 * c - x1 * s for c = ch + cl, s = sh + sl
__device__ __forceinline__ RopePair rope_turn(float x0, float x1, float ch, float cl, float sh, float sl)
{
    const float p = __fmul_rn(x0, ch), pe = __fmaf_rn(x0, ch, -p), q = __fmul_rn(x1, sh), qe = __fmaf_rn(x1, sh, -q);
    const float d = __fsub_rn(p, q), b = __fsub_rn(d, p), e = __fsub_rn(__fsub_rn(p, __fsub_rn(d, b)), __fadd_rn(q, b));
    const float r = __fadd_rn(e, __fadd_rn(__fsub_rn(pe, qe), __fmaf_rn(x0, cl, -__fmul_rn(x1, sl))));
    RopePair    y;
    y.h = __fadd_rn(d, r);
    y.l = __fsub_rn(r, __fsub_rn(y.h, d));
    return y;
}

// kv4_quantise of pairs of floats: the same decisions, with l where it counts.
__device__ __forceinline__ uint32_t kv4_quantise_pair(const float (&h)[8], const float (&l)[8], unsigned mask, int c, __half &dh, float (&y)[8])
{
    float p = h[0], q = -h[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        p = kv4_max(p, h[i]);
        q = kv4_max(q, -h[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        p = kv4_max(p, __shfl_xor_sync(mask, p, o));
        q = kv4_max(q, __shfl_xor_sync(mask, q, o));
    }
    const float m = p > q ? p : -q, size = fabsf(m);
    // (the same in the group's four lanes) equal in size; a scale m / 8 whose 13 bits below fp16's are 1000..., or one
    // below fp16's normal numbers, where those bits are others
    if (p == q || (__float_as_uint(m) & 0x1FFFu) == 0x1000u || size < 0.00048828125f) {
        double x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (double)h[i] + (double)l[i];
        return kv4_quantise64(x, mask, c, dh, y);
    }
    const bool fine = size < INFINITY;
    dh = __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.0f), 65504.0f));
    if (!fine) dh = __ushort_as_half(0x7FFF);
    const float d = __half2float(dh), sign = copysignf(1.0f, d), inv = __frcp_rn(d), half = 0.5f * fabsf(d);
    uint32_t    w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float k = __fsub_rn(__fadd_rn(__fmaf_rn(h[i], inv, -3.814697265625e-6f), 12582912.0f), 12582912.0f);
        // near the border the difference is exact, and l decides
        if (__fsub_rn(__fmul_rn(__fmaf_rn(-k, d, h[i]), sign), half) >= -l[i] * sign) k += 1.0f;
        k = fminf(fmaxf(k, -8.0f), 7.0f);
        w += __float_as_uint(k + 8388616.0f) << (4 * i);
        y[i] = k * d;
    }
    return fine ? w - 0xFB000000u : 0x88888888u;
}

// A block takes a.rows rows and a.heads KV heads with their query heads: the
// angles' cosines and sines into shared memory, then the queries turned, and
// the keys, which wait in shared memory (a block of 32 dimensions and its
// partners may lie in different threads), then codes for K and V.
template <typename T, typename O, int N>
__global__ void __launch_bounds__(256, 4) k_kv4_append_rope(const __grid_constant__ RopeArgs a, const __grid_constant__ KvRows<N> rows)
{
    extern __shared__ __align__(16) uint8_t rope_sm[];
    __shared__ int       s_seq[64], s_pos[64];
    __shared__ long long s_turn[64];
    const int hd = a.kv.nb * 32, rot = a.turns.rot, half = rot / 2, tid = threadIdx.x;
    const int chunks = (a.kv.n_kv + a.heads - 1) / a.heads;
    const int r0 = (int)(blockIdx.x / chunks) * a.rows, h0 = (int)(blockIdx.x % chunks) * a.heads;
    const int nr = min(a.rows, rows.row0[rows.n] - r0), nh = min(a.heads, a.kv.n_kv - h0);
    // Slices: eight pairs each, then eight dimensions each of those that do not turn.
    const int n_pair = (half + 7) / 8, n_rest = (hd - rot + 7) / 8;
    // cosines and sines, and what they round off: pair i of slice x of row r at [r][i][x], so that lanes of consecutive
    // slices meet different banks
    float2   *cs = reinterpret_cast<float2 *>(rope_sm), *cs_rest = cs + a.rows * 8 * n_pair;
    float    *kh = reinterpret_cast<float *>(cs_rest + a.rows * 8 * n_pair), *kl = kh + a.rows * a.heads * hd;      // [rows][heads][hd]
    pdl_wait();
    pdl_trigger();
    // where each row stands, and how far it turns
    if (tid < nr) {
        const int r = r0 + tid;
        int       lo = 0, hi = rows.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (rows.row0[mid] <= r) lo = mid;
            else hi = mid;
        }
        const int first = __ldg(a.kv.len + rows.seq[lo]) - (rows.row0[lo + 1] - rows.row0[lo]), at = r - rows.row0[lo];
        s_seq[tid] = rows.seq[lo];
        s_pos[tid] = first + at;
        s_turn[tid] = (long long)first + (a.depth ? __ldg(a.depth + r) : at);
    }
    __syncthreads();
    for (int x = tid; x < nr * half; x += 256) {
        const int r = x / half, i = x - r * half;
        double    s, c;
        sincospi((double)(long long)((unsigned long long)s_turn[r] * a.turns.turn[i]) * 0x1p-63, &s, &c);
        c *= a.turns.factor;
        s *= a.turns.factor;
        const float ch = (float)c, sh = (float)s;
        const int   at = (r * 8 + (i & 7)) * n_pair + (i >> 3);
        cs[at] = make_float2(ch, sh);
        cs_rest[at] = make_float2((float)(c - (double)ch), (float)(s - (double)sh));
    }
    __syncthreads();
    // Slices begin at multiples of eight elements, but for second halves of other lengths and what lies behind them.
    const bool apart = !a.turns.interleaved, even = !apart || half % 8 == 0, even_rest = rot % 8 == 0;
    const int  q_heads = a.q ? nh * a.n_rep : 0, all = q_heads + nh;
    auto from = [&](int r, int hh) {                              // row r's head hh: the queries', then the keys'
        return hh < q_heads ? (const T *)a.q + (size_t)(r0 + r) * a.q_stride + (size_t)(h0 * a.n_rep + hh) * hd
                            : (const T *)a.kv.k + (size_t)(r0 + r) * a.kv.k_stride + (size_t)(h0 + hh - q_heads) * hd;
    };
    auto to = [&](int r, int hh) { return (T *)a.q_out + (size_t)(r0 + r) * a.q_out_stride + (size_t)(h0 * a.n_rep + hh) * hd; };
    // The pairs' first and second values lie in slices u and v, or, interleaved, are every other one of both.
    struct Slice { int i0, n, d0, d1, n0, n1; };
    auto slice = [&](int sl) {
        Slice x;
        x.i0 = 8 * sl;
        x.n = min(8, half - x.i0);
        x.d0 = apart ? x.i0 : 2 * x.i0;
        x.d1 = apart ? half + x.i0 : 2 * x.i0 + 8;
        x.n0 = apart ? x.n : 2 * x.n;
        x.n1 = apart ? x.n : 2 * x.n - 8;
        return x;
    };
    // Queries: a thread keeps its slice of a row and takes heads in turn.
    const int combos = nr * n_pair, lanes = combos >= 256 ? 1 : combos ? 256 / combos : 0;
    for (int x = tid; x < combos * lanes && q_heads > 0; x += 256) {
        const int     hl = x / combos, combo = x - hl * combos, r = combo / n_pair, sl = combo - r * n_pair;
        const Slice   at = slice(sl);
        const float2 *t = cs + r * 8 * n_pair + sl;
        float2        e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = t[min(i, at.n - 1) * n_pair];
        for (int hh = hl; hh < q_heads; hh += lanes) {
            const T *p = from(r, hh);
            T       *o = to(r, hh);
            float    u[8], v[8];
            rope_load(p + at.d0, at.n0, a.wide_q, u);
            rope_load(p + at.d1, at.n1, even && a.wide_q, v);
            if (apart) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y0 = fmaf(u[i], e[i].x, -v[i] * e[i].y), y1 = fmaf(v[i], e[i].x, u[i] * e[i].y);
                    u[i] = y0;
                    v[i] = y1;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float      &p0 = i < 4 ? u[2 * (i & 3)] : v[2 * (i & 3)], &p1 = i < 4 ? u[2 * (i & 3) + 1] : v[2 * (i & 3) + 1];
                    const float y0 = fmaf(p0, e[i].x, -p1 * e[i].y), y1 = fmaf(p1, e[i].x, p0 * e[i].y);
                    p0 = y0;
                    p1 = y1;
                }
            }
            rope_store(o + at.d0, at.n0, a.wide_q, u);
            rope_store(o + at.d1, at.n1, even && a.wide_q, v);
        }
    }
    // Keys
    for (int x = tid; x < nr * nh * n_pair; x += 256) {
        const int     r = x / (nh * n_pair), in_row = x - r * (nh * n_pair), h = in_row / n_pair, sl = in_row - h * n_pair;
        const Slice   at = slice(sl);
        const float2 *t = cs + r * 8 * n_pair + sl, *rest = cs_rest + r * 8 * n_pair + sl;
        const T      *p = from(r, q_heads + h);
        const int     kd = (r * a.heads + h) * hd;
        float         u[8], v[8], ul[8], vl[8];
        rope_load(p + at.d0, at.n0, a.kv.wide, u);
        rope_load(p + at.d1, at.n1, even && a.kv.wide, v);
        auto turn = [&](float &p0, float &p1, float &q0, float &q1, int i) {
            const float2   e = t[min(i, at.n - 1) * n_pair], f = rest[min(i, at.n - 1) * n_pair];
            const RopePair y0 = rope_turn(p0, p1, e.x, f.x, e.y, f.y), y1 = rope_turn(p1, -p0, e.x, f.x, e.y, f.y);
            p0 = y0.h, q0 = y0.l;
            p1 = y1.h, q1 = y1.l;
        };
        if (apart)
#pragma unroll
            for (int i = 0; i < 8; i++) turn(u[i], v[i], ul[i], vl[i], i);
        else
#pragma unroll
            for (int i = 0; i < 4; i++) {
                turn(u[2 * i], u[2 * i + 1], ul[2 * i], ul[2 * i + 1], i);
                turn(v[2 * i], v[2 * i + 1], vl[2 * i], vl[2 * i + 1], 4 + i);
            }
        rope_store(kh + kd + at.d0, at.n0, true, u);
        rope_store(kl + kd + at.d0, at.n0, true, ul);
        rope_store(kh + kd + at.d1, at.n1, even, v);
        rope_store(kl + kd + at.d1, at.n1, even, vl);
    }
    for (int x = tid; x < nr * all * n_rest; x += 256) {
        const int r = x / (all * n_rest), in_row = x - r * all * n_rest, hh = in_row / n_rest, d = rot + 8 * (in_row - hh * n_rest), n = hd - d;
        const T  *p = from(r, hh);
        float     u[8];
        rope_load(p + d, n, even_rest && (hh < q_heads ? a.wide_q : a.kv.wide), u);
        if (hh < q_heads) rope_store(to(r, hh) + d, n, even_rest && a.wide_q, u);
        else
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < n) {
                    kh[(r * a.heads + hh - q_heads) * hd + d + i] = u[i];
                    kl[(r * a.heads + hh - q_heads) * hd + d + i] = 0.0f;
                }
    }
    __syncthreads();
    // Codes, four lanes to a block of 32 dimensions: blocks hb of row r in turn.
    const int blocks = nh * a.kv.nb, step_r = 64 / blocks, step_hb = 64 - step_r * blocks;
    int       r = tid / 4 / blocks, hb = tid / 4 - r * blocks;
    for (; r < nr; r += step_r, hb += step_hb) {
        if (hb >= blocks) {
            hb -= blocks;
            if (++r >= nr) break;
        }
        const int      c = tid & 3, h = (int)((unsigned)hb * a.kv.nb_inv >> 16), b = hb - h * a.kv.nb;
        const unsigned mask = 0xFu << (tid & 28);
        const size_t   at = (size_t)h0 * hd + 32 * hb + 8 * c, out = (size_t)(r0 + r) * a.kv.n_kv * hd + at;
        float          y[8], x[8], l[8];
        __half         d[2];
        uint32_t       w[2];
        kv4_load8((const T *)a.kv.v + (size_t)(r0 + r) * a.kv.v_stride + at, a.kv.wide, x);
        const int  pos = s_pos[r], t = pos & (KV4_PAGE - 1);
        const bool placed = pos >= 0 && pos < a.kv.max_pages * KV4_PAGE;
        const int  page = placed ? __ldg(a.kv.table + (size_t)s_seq[r] * a.kv.max_pages + pos / KV4_PAGE) : -1;
        w[1] = kv4_quantise(x, mask, c, d[1], y);
        if (a.kv.k_out) kv4_store8((O *)a.kv.v_out + out, a.kv.wide_out, y);
        const int kd = r * a.heads * hd + 32 * hb + 8 * c;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 fh = *reinterpret_cast<const float4 *>(kh + kd + i), fl = *reinterpret_cast<const float4 *>(kl + kd + i);
            x[i] = fh.x, x[i + 1] = fh.y, x[i + 2] = fh.z, x[i + 3] = fh.w;
            l[i] = fl.x, l[i + 1] = fl.y, l[i + 2] = fl.z, l[i + 3] = fl.w;
        }
        w[0] = kv4_quantise_pair(x, l, mask, c, d[0], y);
        if (a.kv.k_out) kv4_store8((O *)a.kv.k_out + out, a.kv.wide_out, y);
        if ((unsigned)page >= (unsigned)a.kv.n_pages) continue;   // no page: nothing to write to
        uint8_t *p = a.kv.layer + (size_t)page * a.kv.page_bytes + (size_t)(h0 + h) * 72 * hd;
#pragma unroll
        for (int side = 0; side < 2; side++) {
            *reinterpret_cast<uint32_t *>(p + side * 32 * hd + t * (hd / 2) + kv4_place(t, b, a.kv.nb) * 16 + 4 * c) = w[side];
            if (c == 0) *reinterpret_cast<__half *>(p + 64 * hd + side * 4 * hd + (t * a.kv.nb + b) * 2) = d[side];
        }
    }
}
