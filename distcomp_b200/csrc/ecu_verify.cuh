// ecu_verify.cuh -- drafted tokens held against the target's probabilities.
//
// A sequence's rows are a tree, row 0 its root.  From the root on, the rows
// that hang on the current one are tried in order; with P = softmax(logits / T)
// of the current row, f = P at first and F the sum of f, row j with token x is
// accepted where u_j q(x) F < f(x) (q: the distribution it was drawn from; 1
// where there was none), and becomes the current row.  A rejected one leaves
// f <- max(f / F - q, 0), or f(x) <- 0.  Where none is left, the next token is
// the first x whose running sum of f passes u F: so tokens are distributed as
// the target's own.
//
// Which tokens those are is decided by comparing sums, so everything that is
// compared is held in 64 bits: a running sum of 32 bits would let about one
// draw in a hundred of a vocabulary of 128256 fall to a neighbour.
//
// A cluster of CTAs walks one sequence's tree; its warps hold equal runs of the
// vocabulary, and sums meet through distributed shared memory.  A row is read
// once: its largest logit, whether it is a distribution at all, and the sum of
// 2^((l - c) / T log2 e) come out of one pass, c being the row's first logit (64
// bits hold 2^+-1000 around it; where that is not enough, a second pass takes
// the largest).  The exponential is a table of 2^(k/256) and four terms of its
// series: ten operations of 64 bits a logit.
//
// Latency bounds it: the rows of a path come one behind the other, each a pass
// and an exchange between the cluster's CTAs.  A chain of 5 drafts over 128256
// fp32 logits takes 14 us (of a row's 0.5 MB on 8 CTAs), 48 trees of 4 to 16
// rows (bf16) 48 to 54 us: 51 MB through L2, 57 % of the issue slots and 22 % of
// the fp64 units' time.  The 64 registers that two CTAs an SM leave spill 80 to
// 124 bytes a thread, and the table is read at a random place a lane.  Two passes
// over a row, the maximum first and then exp()'s sums, took 44 and 191.
#pragma once
#include "ecu_kv4.cuh"

#include <cooperative_groups.h>

#define VER_WARPS 16
#define VER_MAX_CTAS 8            // of a cluster
#define VER_ROWS 64               // rows of a tree

struct VerifyArgs {
    const void  *logits;
    long         stride, draft_stride;
    const float *draft;           // nullptr: tokens were not drawn
    const int   *token, *parent;
    const float *u, *u_next, *temperature;
    int         *kept, *n_kept, *next;
    int          vocab, seq0;     // seq0: the launch's first sequence
    bool         wide;
};

template <int N> struct VerifyRows {
    int n;
    int row0[N + 1];
};

// The largest value so far and its first place; -1 where a NaN or an infinity was among them.
struct VerTop {
    float v;
    int   at;
};
struct __align__(16) VerWord {
    double sum;
    VerTop top;
};
__device__ __forceinline__ double warp_total(double v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __hiloint2double(__shfl_xor_sync(0xffffffffu, __double2hiint(v), o), __shfl_xor_sync(0xffffffffu, __double2loint(v), o));
    return v;
}

__device__ __forceinline__ VerTop ver_top(VerTop a, VerTop b)
{
    if (a.at < 0 || b.at < 0) return VerTop{0.0f, -1};
    return b.v > a.v || (b.v == a.v && b.at < a.at) ? b : a;
}

// Of n sums (at most 128) that begin at `before`, the first positive one that the
// running sum passes the mark in, and the sum before it; where none does
// (rounding), or `end` says so already, the last positive one.  By a warp.
struct VerDraw {
    int    at;
    double before;
    bool   end;
};
__device__ __forceinline__ VerDraw ver_find(const double *sums, int n, double before, double mark, bool end, int lane)
{
    double w[4], in = 0.0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        w[k] = 4 * lane + k < n ? sums[4 * lane + k] : 0.0;
        in += w[k];
    }
    const double mine = in;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double v = __hiloint2double(__shfl_up_sync(0xffffffffu, __double2hiint(in), o), __shfl_up_sync(0xffffffffu, __double2loint(in), o));
        if (lane >= o) in += v;
    }
    double run = before + (in - mine), at = run;
    int    hit = -1, any = -1;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (w[k] > 0.0) {
            any = 4 * lane + k;
            if (hit < 0 && !end && run + w[k] > mark) {
                hit = any;
                at = run;
            }
        }
        run += w[k];
    }
    const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, any >= 0);
    VerDraw        d{-1, 0.0, hits == 0};
    const int      from = hits ? __ffs(hits) - 1 : some ? 31 - __clz(some) : 0;
    d.at = __shfl_sync(0xffffffffu, hits ? hit : any, from);
    d.before = __hiloint2double(__shfl_sync(0xffffffffu, __double2hiint(at), from), __shfl_sync(0xffffffffu, __double2loint(at), from));
    return d;
}

#define VER_TABLE 256

// 2^t; t < -1000: 0, t > 1000: infinity.  t = k / 256 + f with |f| <= 1/512, and
// 2^f by its series up to f^4 (the next term is below 2^-54).
__device__ __forceinline__ double ver_ex2(double t, const double *table)
{
    const double magic = 26388279066624.0;                // 1.5 * 2^44: a sum's last bit is 1/256
    const double m = t + magic, f = t - (m - magic);
    const int    k = __double2loint(m);
    double       p = fma(f, 0.009618129107628477, 0.05550410866482158);
    p = fma(f, p, 0.2402265069591007);
    p = fma(f, p, 0.6931471805599453);
    const double w = table[k & (VER_TABLE - 1)];
    p = fma(w, f * p, w);
    p = __hiloint2double(__double2hiint(p) + ((k >> 8) << 20), __double2loint(p));
    return t < -1000.0 ? 0.0 : t > 1000.0 ? INFINITY : p;
}

// f(x, logit) for this lane's elements of [x0, x1), x0 a multiple of eight.
template <typename T, typename F> __device__ __forceinline__ void ver_each(const T *row, int x0, int x1, bool wide, int lane, F f)
{
    constexpr int V = 16 / (int)sizeof(T), U = 16 / V;    // elements of 16 bytes; loads in flight together
    int           x = x0;
    if (wide) {
        for (; x + V <= x1; x += 32 * V * U) {
            uint4 w[U];
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int at = x + (32 * i + lane) * V;
                w[i] = at + V <= x1 ? __ldg(reinterpret_cast<const uint4 *>(row + at)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int at = x + (32 * i + lane) * V;
                const T  *v = reinterpret_cast<const T *>(&w[i]);
                if (at + V <= x1)
#pragma unroll
                    for (int k = 0; k < V; k++) f(at + k, kv4_float(v[k]));
            }
        }
        x = x1 - (x1 - x0) % V;                           // (fewer than V are left)
    }
    for (x += lane; x < x1; x += 32) f(x, kv4_float(row[x]));
}

template <typename T, int N>
__global__ void __launch_bounds__(VER_WARPS * 32, 2) k_draft_verify(const VerifyArgs a, const __grid_constant__ VerifyRows<N> rows)
{
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    const int CL = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    __shared__ VerWord  x_word[2][VER_WARPS];             // what this CTA's warps tell the cluster, two exchanges in turn
    __shared__ VerTop   b_top[VER_MAX_CTAS * VER_WARPS];  // what all warps said
    __shared__ double   b_sum[VER_MAX_CTAS * VER_WARPS], p_sum[VER_WARPS];
    __shared__ double   F_s[VER_ROWS + 1];                // f's sums at the current row, before each rejection
    __shared__ int      gone_s[VER_ROWS], tok_s[VER_ROWS], par_s[VER_ROWS];
    __shared__ float    u_s[VER_ROWS];
    __shared__ double   table[VER_TABLE];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid < VER_TABLE) table[tid] = exp2((double)tid / VER_TABLE);
    pdl_wait();
    pdl_trigger();
    const int i = (int)blockIdx.x / CL, r0 = rows.row0[i], n = rows.row0[i + 1] - r0, W = CL * VER_WARPS;
    const int seq = a.seq0 + i;
    if (n == 0) {                                         // (the whole cluster)
        if (rank == 0 && tid == 0) {
            a.n_kept[seq] = 0;
            a.next[seq] = -1;
        }
        return;
    }
    if (tid < n) {
        tok_s[tid] = __ldg(a.token + r0 + tid);
        par_s[tid] = __ldg(a.parent + r0 + tid);
        u_s[tid] = __ldg(a.u + r0 + tid);
    }
    __syncthreads();                                      // the table's warps are not its only readers
    const float  temp = a.temperature ? __ldg(a.temperature + seq) : 1.0f;
    const bool   greedy = !(temp > 0.0f);
    const double inv = greedy ? 1.0 : 1.4426950408889634 / (double)temp;
    // this warp's run of the vocabulary, a multiple of 8 but for the last
    const int per = ((a.vocab + W - 1) / W + 7) & ~7, me = rank * VER_WARPS + warp;
    const int x0 = min(a.vocab, me * per), x1 = min(a.vocab, x0 + per);
    int       turn = 0;

    const T     *lg = nullptr;
    const float *dr = nullptr;
    VerTop       top{-INFINITY, 0x7FFFFFFF};
    double       from = 0.0;                              // c
    bool         bad = false;
    int          n_gone = 0, n_res = 0;                   // tokens taken out, subtractions

    // every warp's sum, at every CTA, and their total, in the order of the warps by every thread alike
    auto exchange = [&](double sum) {
        if (lane == 0) x_word[turn][warp].sum = sum;
        cl.sync();
        for (int k = tid; k < W; k += VER_WARPS * 32) b_sum[k] = cl.map_shared_rank(&x_word[turn][0], k / VER_WARPS)[k % VER_WARPS].sum;
        __syncthreads();
        turn ^= 1;
    };
    auto total = [&] {
        double s = 0.0;
        for (int k = lane; k < W; k += 32) s += b_sum[k];
        return warp_total(s);
    };
    auto weight = [&](float l) { return l == -INFINITY ? 0.0 : ver_ex2(((double)l - from) * inv, table); };
    // f(x) as the rejections so far left it
    auto f_at = [&](int x, float l) {
        for (int k = 0; k < n_gone; k++)
            if (gone_s[k] == x) return 0.0;
        double f = weight(l);
        if (n_res) {
            const double q = (double)__ldg(dr + x);
            for (int k = 0; k < n_res; k++) f = fmax(f / F_s[k] - q, 0.0);
        }
        return f;
    };
    auto f_of = [&](int x) { return f_at(x, kv4_float(lg[x])); };
    auto sum_f = [&] {
        double s = 0.0;
        ver_each(lg, x0, x1, a.wide, lane, [&](int x, float l) { s += f_at(x, l); });
        exchange(warp_total(s));
        return total();
    };
    // Row j becomes the current one: its largest logit, whether it is a distribution, f's sum.
    auto open_row = [&](int j) {
        lg = (const T *)a.logits + (size_t)(r0 + j) * a.stride;
        dr = a.draft ? a.draft + (size_t)(r0 + j) * a.draft_stride : nullptr;
        const float first = kv4_float(lg[0]);
        from = fabsf(first) < INFINITY ? (double)first : 0.0;
        n_gone = n_res = 0;
        top = VerTop{-INFINITY, 0x7FFFFFFF};
        int    b = 0;
        double s0 = 0.0, s1 = 0.0;
        ver_each(lg, x0, x1, a.wide, lane, [&](int x, float l) {
            b |= !(l < INFINITY);                         // NaN or an infinity
            if (l > top.v || (l == top.v && x < top.at)) top = VerTop{l, x};
            if (!greedy) {
                const double w = weight(l);
                if (x & 1) s1 += w;
                else s0 += w;
            }
        });
        const double s = warp_total(s0 + s1);
        auto reduce = [&] {
#pragma unroll
            for (int o = 16; o; o >>= 1) top = ver_top(top, VerTop{__shfl_xor_sync(0xffffffffu, top.v, o), __shfl_xor_sync(0xffffffffu, top.at, o)});
        };
        if (b) top.at = -1;
        reduce();
        if (lane == 0) x_word[turn][warp] = VerWord{s, top};
        cl.sync();                                        // (b_sum and b_top are read no more)
        for (int k = tid; k < W; k += VER_WARPS * 32) {
            const VerWord w = cl.map_shared_rank(&x_word[turn][0], k / VER_WARPS)[k % VER_WARPS];
            b_sum[k] = w.sum;
            b_top[k] = w.top;
        }
        __syncthreads();
        turn ^= 1;
        top = VerTop{-INFINITY, 0x7FFFFFFF};
        for (int k = lane; k < W; k += 32) top = ver_top(top, b_top[k]);
        reduce();
        bad = top.at < 0 || top.v == -INFINITY;
        double F = total();
        if (!bad && !greedy && !(F >= 0x1p-100 && F < INFINITY)) {        // the first logit lies too far from the largest
            from = (double)top.v;
            __syncthreads();
            F = sum_f();
        }
        return F;
    };

    int    cur = 0, held = 1;
    double F = open_row(0), whole = F;                    // f's sum; that of the row as it was
    if (rank == 0 && tid < n) a.kept[r0 + tid] = tid == 0 ? 0 : -1;
    __syncthreads();
    for (int j = 1; j < n && !bad; j++) {
        if (par_s[j] != cur) continue;
        const int x = tok_s[j];
        if ((unsigned)x >= (unsigned)a.vocab) continue;   // no such token: never accepted
        bool take;
        if (greedy) take = x == top.at;
        else {
            const double f = f_of(x), q = dr ? (double)__ldg(dr + x) : 1.0;
            take = (double)u_s[j] * q * F < f;
            if (!take) {
                // a difference that has lost digits (little is left, in all or, next to all, of its warp's run) is summed anew
                const bool anew = dr || !(F - f > whole * 0x1p-10) || !(b_sum[x / per] - f > whole * 0x1p-40);
                __syncthreads();                          // b_sum, F_s and gone_s are read no more
                if (dr) {
                    if (tid == 0) F_s[n_res] = F;
                    n_res++;
                } else {
                    if (tid == 0) {
                        gone_s[n_gone] = x;
                        b_sum[x / per] -= f;
                    }
                    n_gone++;
                    F -= f;
                }
                __syncthreads();
                if (anew) F = whole = sum_f();
            }
        }
        if (!take) continue;
        cur = j;
        if (rank == 0 && tid == 0) a.kept[r0 + held] = j;
        held++;
        F = whole = open_row(j);
    }
    if (rank == 0 && tid == 0) a.n_kept[seq] = held;
    if (bad || greedy) {
        if (rank == 0 && tid == 0) a.next[seq] = bad ? -1 : top.at;
        cl.sync();                                        // no CTA leaves while others read its shared memory
        return;
    }
    if (!(F > 0.0)) {                                     // a rejection of all there was: the target's own distribution
        n_gone = n_res = 0;
        __syncthreads();
        F = sum_f();
    }
    // the warp whose run holds the draw
    const double mark = (double)__ldg(a.u_next + seq) * F;
    const VerDraw draw = ver_find(b_sum, W, 0.0, mark, false, lane);
    const int     owner = draw.at;
    // its CTA's warps share the run once more: their sums, and the one that holds the draw (or the last weight)
    if (owner >= 0 && owner / VER_WARPS == rank) {
        const int o0 = min(a.vocab, owner * per), o1 = min(a.vocab, o0 + per), part = ((o1 - o0 + VER_WARPS - 1) / VER_WARPS + 3) & ~3;
        const int p0 = min(o1, o0 + warp * part), p1 = min(o1, p0 + part);
        double    mine = 0.0;
        for (int x = p0 + lane; x < p1; x += 32) mine += f_of(x);
        mine = warp_total(mine);
        if (lane == 0) p_sum[warp] = mine;
        __syncthreads();
        const VerDraw part_draw = ver_find(p_sum, VER_WARPS, draw.before, mark, draw.end, lane);
        const bool    end = part_draw.end;
        if (part_draw.at < 0 && tid == 0) a.next[seq] = top.at;
        if (part_draw.at == warp) {
            // four tokens a lane in turn: their sum, the sums before them, and the first that passes the mark
            int    pick = -1;
            double run = part_draw.before;
            for (int b = p0; b < p1; b += 128) {
                double f[4], in = 0.0;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int x = b + 4 * lane + k;
                    f[k] = x < p1 ? f_of(x) : 0.0;
                    in += f[k];
                }
                const double mine = in;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double v = __hiloint2double(__shfl_up_sync(0xffffffffu, __double2hiint(in), o), __shfl_up_sync(0xffffffffu, __double2loint(in), o));
                    if (lane >= o) in += v;
                }
                double at = run + (in - mine);
                int    hit = -1, any = -1;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    at += f[k];
                    if (f[k] > 0.0) {
                        any = b + 4 * lane + k;
                        if (hit < 0 && !end && at > mark) hit = any;
                    }
                }
                const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, any >= 0);
                if (hits) {
                    pick = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
                    break;
                }
                if (some) pick = __shfl_sync(0xffffffffu, any, 31 - __clz(some));      // where none passes: the last
                run += __hiloint2double(__shfl_sync(0xffffffffu, __double2hiint(in), 31), __shfl_sync(0xffffffffu, __double2loint(in), 31));
            }
            if (lane == 0) a.next[seq] = pick;
        }
    }
    cl.sync();
}
