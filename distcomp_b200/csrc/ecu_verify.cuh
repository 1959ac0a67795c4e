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
// vocabulary, and sums meet through distributed shared memory.
#pragma once
#include "ecu_kv4.cuh"

#include <cooperative_groups.h>

#define VER_WARPS 16
#define VER_MAX_CTAS 16           // of a cluster
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

// The largest value so far and its first place; a NaN or an infinity shows in `bad`.
struct VerTop {
    float v;
    int   at;
};
__device__ __forceinline__ VerTop ver_top(VerTop a, VerTop b)
{
    return b.v > a.v || (b.v == a.v && b.at < a.at) ? b : a;
}

template <typename T, int N>
__global__ void __launch_bounds__(VER_WARPS * 32) k_draft_verify(const VerifyArgs a, const __grid_constant__ VerifyRows<N> rows)
{
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    const int CL = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    __shared__ double   x_sum[2][VER_WARPS];              // what this CTA's warps tell the cluster, two exchanges in turn
    __shared__ float    x_top[2][VER_WARPS];
    __shared__ int      x_at[2][VER_WARPS], x_bad[2][VER_WARPS];
    __shared__ double   b_sum[VER_MAX_CTAS * VER_WARPS];
    __shared__ float    b_top[VER_MAX_CTAS * VER_WARPS];
    __shared__ int      b_at[VER_MAX_CTAS * VER_WARPS], b_bad[VER_MAX_CTAS * VER_WARPS];
    __shared__ double   F_s[VER_ROWS + 1];                // f's sums at the current row, before each rejection
    __shared__ int      gone_s[VER_ROWS], tok_s[VER_ROWS], par_s[VER_ROWS];
    __shared__ float    u_s[VER_ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
    const float  temp = a.temperature ? __ldg(a.temperature + seq) : 1.0f;
    const bool   greedy = !(temp > 0.0f);
    const double inv = greedy ? 1.0 : 1.0 / (double)temp;
    // this warp's run of the vocabulary, a multiple of 8 but for the last
    const int per = ((a.vocab + W - 1) / W + 7) & ~7, me = rank * VER_WARPS + warp;
    const int x0 = min(a.vocab, me * per), x1 = min(a.vocab, x0 + per);
    int       turn = 0;

    const T     *lg = nullptr;
    const float *dr = nullptr;
    VerTop       top{-INFINITY, 0x7FFFFFFF};
    bool         bad = false;
    int          n_gone = 0, n_res = 0;                   // tokens taken out, subtractions

    // every warp's value, at every CTA
    auto exchange = [&](double sum) {
        if (lane == 0) x_sum[turn][warp] = sum;
        cl.sync();
        for (int k = tid; k < W; k += VER_WARPS * 32) b_sum[k] = cl.map_shared_rank(&x_sum[turn][0], k / VER_WARPS)[k % VER_WARPS];
        __syncthreads();
        turn ^= 1;
    };
    auto total = [&] {                                    // in the order of the warps, by every thread alike
        double s = 0.0;
        for (int k = lane; k < W; k += 32) s += b_sum[k];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += kv4_shfl_xor(0xffffffffu, s, o);
        __syncthreads();                                  // b_sum may be written again
        return s;
    };
    auto weight = [&](float l) { return l == -INFINITY ? 0.0 : exp(((double)l - (double)top.v) * inv); };
    // f(x) as the rejections so far left it
    auto f_of = [&](int x) {
        for (int k = 0; k < n_gone; k++)
            if (gone_s[k] == x) return 0.0;
        double f = weight(kv4_float(lg[x]));
        if (n_res) {
            const double q = (double)__ldg(dr + x);
            for (int k = 0; k < n_res; k++) f = fmax(f / F_s[k] - q, 0.0);
        }
        return f;
    };
    auto sum_f = [&] {
        double s = 0.0;
        for (int x = x0 + lane; x < x1; x += 32) s += f_of(x);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += kv4_shfl_xor(0xffffffffu, s, o);
        exchange(s);
    };
    auto open_row = [&](int j) {                          // row j becomes the current one: its largest value
        lg = (const T *)a.logits + (size_t)(r0 + j) * a.stride;
        dr = a.draft ? a.draft + (size_t)(r0 + j) * a.draft_stride : nullptr;
        top = VerTop{-INFINITY, 0x7FFFFFFF};
        int b = 0;
        for (int x = x0 + lane; x < x1; x += 32) {
            const float v = kv4_float(lg[x]);
            b |= !(v < INFINITY);                         // NaN or an infinity
            if (v > top.v) top = VerTop{v, x};
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            top = ver_top(top, VerTop{__shfl_xor_sync(0xffffffffu, top.v, o), __shfl_xor_sync(0xffffffffu, top.at, o)});
            b |= __shfl_xor_sync(0xffffffffu, b, o);
        }
        if (lane == 0) {
            x_top[turn][warp] = top.v;
            x_at[turn][warp] = top.at;
            x_bad[turn][warp] = b;
        }
        cl.sync();
        for (int k = tid; k < W; k += VER_WARPS * 32) {
            b_top[k] = cl.map_shared_rank(&x_top[turn][0], k / VER_WARPS)[k % VER_WARPS];
            b_at[k] = cl.map_shared_rank(&x_at[turn][0], k / VER_WARPS)[k % VER_WARPS];
            b_bad[k] = cl.map_shared_rank(&x_bad[turn][0], k / VER_WARPS)[k % VER_WARPS];
        }
        __syncthreads();
        turn ^= 1;
        top = VerTop{-INFINITY, 0x7FFFFFFF};
        b = 0;
        for (int k = lane; k < W; k += 32) {
            top = ver_top(top, VerTop{b_top[k], b_at[k]});
            b |= b_bad[k];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            top = ver_top(top, VerTop{__shfl_xor_sync(0xffffffffu, top.v, o), __shfl_xor_sync(0xffffffffu, top.at, o)});
            b |= __shfl_xor_sync(0xffffffffu, b, o);
        }
        __syncthreads();
        bad = b || top.v == -INFINITY;
        n_gone = n_res = 0;
    };

    int    cur = 0, held = 1;
    double F = 0.0;
    open_row(0);
    bool have = false;                                    // F is f's sum
    if (rank == 0 && tid < n) a.kept[r0 + tid] = tid == 0 ? 0 : -1;
    __syncthreads();
    for (int j = 1; j < n && !bad; j++) {
        if (par_s[j] != cur) continue;
        const int x = tok_s[j];
        if ((unsigned)x >= (unsigned)a.vocab) continue;   // no such token: never accepted
        bool take;
        if (greedy) take = x == top.at;
        else {
            if (!have) {
                sum_f();
                F = total();
                have = true;
            }
            const double f = f_of(x), q = dr ? (double)__ldg(dr + x) : 1.0;
            take = (double)u_s[j] * q * F < f;
            if (!take) {
                if (dr) {
                    if (tid == 0) F_s[n_res] = F;
                    n_res++;
                } else {
                    if (tid == 0) gone_s[n_gone] = x;
                    n_gone++;
                }
                __syncthreads();
                have = false;
            }
        }
        if (!take) continue;
        cur = j;
        if (rank == 0 && tid == 0) a.kept[r0 + held] = j;
        held++;
        open_row(j);
        have = false;
    }
    if (rank == 0 && tid == 0) a.n_kept[seq] = held;
    if (bad || greedy) {
        if (rank == 0 && tid == 0) a.next[seq] = bad ? -1 : top.at;
        cl.sync();                                        // no CTA leaves while others read its shared memory
        return;
    }
    sum_f();
    F = total();
    if (!(F > 0.0)) {                                     // a rejection of all there was: the target's own distribution
        n_gone = n_res = 0;
        sum_f();
        F = total();
    }
    // the warp whose run holds the draw
    const double mark = (double)__ldg(a.u_next + seq) * F;
    double       before = 0.0, s = 0.0;
    int          owner = -1, last = -1;
    for (int k = 0; k < W; k++) {                         // the same at every thread
        const double w = b_sum[k];
        if (w > 0.0) last = k;
        if (owner < 0 && w > 0.0 && s + w > mark) {
            owner = k;
            before = s;
        }
        s += w;
    }
    const bool past = owner < 0;                          // rounding: the last token that has any weight
    if (past) owner = last;
    if (owner == me) {
        int    pick = -1;
        double run = before;
        for (int b = x0; b < x1; b += 32) {
            const int    x = b + lane;
            const double f = x < x1 ? f_of(x) : 0.0;
            double       in = f;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double v = __hiloint2double(__shfl_up_sync(0xffffffffu, __double2hiint(in), o), __shfl_up_sync(0xffffffffu, __double2loint(in), o));
                if (lane >= o) in += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, f > 0.0 && run + in > mark && !past), any = __ballot_sync(0xffffffffu, f > 0.0);
            if (hit) {
                pick = b + __ffs(hit) - 1;
                break;
            }
            if (any) pick = b + 31 - __clz(any);          // where none passes: the last
            run += __hiloint2double(__shfl_sync(0xffffffffu, __double2hiint(in), 31), __shfl_sync(0xffffffffu, __double2loint(in), 31));
        }
        if (lane == 0) a.next[seq] = pick;
    }
    cl.sync();
}
