// ecu_tree.cuh -- attention of several drafted positions per sequence, a tree
// of them, over the paged 4-bit cache (layout: engine_cuda.h).
//
// A column is one query head of one drafted row; the columns of a KV head read
// the same K and V.  One pass over the cached positions with a running maximum
// and sum, the products on the tensor cores (mma.sync m16n8k16, fp16 operands,
// fp32 sums) on the integer codes, which fp16 holds exactly:
//
//   score[col][t] = sum_b Kscale[t][b] * (q[col][b] . Kcode[t][b])
//   O[col][d]    += sum_t (weight[col][t] * Vscale[t][b(d)]) * Vcode[t][d]
//
// The columns are the products' rows, 16 to a tile: then the scores lie in the
// registers as the second product wants its weights.  An fp32 query is two rows
// of a tile, g its fp16 part and g + 8 the fp16 part of the rest (22 bits), and
// so are its weights; they add up in one thread.  The weights of 16-bit queries
// are one fp16 number each (off by 2^-11 of a weight at most, as their outputs are
// rounded by 2^-11, and of bf16 by 2^-8): a second part would double the second
// product's rows, and with them the tiles of a call.  The weights' sum is
// of the unrounded ones.  Ranges, the power of two that
// a query is scaled by and the maximum that is followed lazily are those of
// ecu_kv4.cuh's attention.
//
// Positions before the drafted ones are seen by every row; of the drafted ones
// those of its mask.  What a row does not see is taken out by selection, not by
// adding -inf or weighing 0: a NaN there has no effect.
//
// Work is cut into units, 32 positions of one KV head and up to `wc` tiles of 16
// columns of one sequence.  A CTA's 12 warps are wc by 12 / wc: a group of wc
// warps reads a unit together (16-byte asynchronous copies, a ring a group),
// each for its own tile, and the groups take the units of a row in turn.
// Places (units, and a few for each row's beginning and end) are dealt evenly to
// one CTA an SM; a row's groups are merged in shared memory, and a row that
// several CTAs share is joined from their partial sums by a second launch, in
// the order of the CTAs.
//
// Short calls are bound by latency: 6 drafts of one sequence of 900 positions
// (32 query and 8 KV heads of 128, fp32) take 16 us (the host's call alone 12),
// 17 sequences of up to 3000 positions (16 and 4 heads of 64, fp16) 35: a step of
// the groups takes about 3 us (64-wide heads 1.7), a row's queries, merge and
// output 5 to 8, a join 12.  Many columns are bound by the scales between the
// products, which the tensor cores do not apply: 32 sequences of 1 to 4096
// positions (64 and 8 heads of 128) take 444 us in fp32, 545 before the fp32 sums
// were packed and rows' own places counted.  In 16 bits such calls run on
// ecu_tree_tc.cuh's kernel instead.  At 128-wide heads the 168 registers that 12
// warps leave spill 144 bytes a thread in 16 bits, 92 in fp32, at 96-wide ones 12
// and none.
#pragma once
#include "ecu_kv4.cuh"

#define TREE_ROWS 64              // drafted rows of a sequence: bits of a mask
#define TREE_WARPS 12
#define TREE_OPEN 12              // places of a row beside its units
#define TREE_MAX_WC 4

struct TreeArgs {
    const void    *q;
    void          *out;
    long           q_stride, out_stride;
    const uint8_t *layer;
    size_t         page_bytes;
    const int     *table, *len;
    const long long *mask;        // nullptr: each row sees those before it
    int            max_pages, n_pages, n_kv, n_rep, wc;
    int            group;         // columns of a row: wc tiles of them
    int            open;          // places of a row beside its units
    int            entry;         // columns of a partial
    float          scale;
    bool           wide_q, wide_out;
    float         *part;          // workspace: partials of rows that several CTAs share
};

template <typename T, int NB> struct TreeShape {
    static constexpr int HD = NB * 32, P = KvSplit<T>::N, C = 16 / P;       // columns of a tile
    static constexpr int STAGE = 36 * HD;                                   // one unit
    static constexpr int LD = HD + 4;                                       // a column of a warp's partial
    static constexpr int EC = TREE_MAX_WC * C;                              // columns of a partial: sums, then M, then the weights' sum of each
    static constexpr size_t ring = (size_t)24 * STAGE, parts = (size_t)TREE_WARPS * C * LD * 4;
    static constexpr size_t smem(int n) { return ring + parts + (size_t)(n + 1) * 4; }
};

// Two fp32 values in one register pair, for the packed fp32 units.
__device__ __forceinline__ uint64_t tree_two(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void     tree_untwo(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t tree_fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t tree_add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Places of one sequence's rows (KV heads times groups of columns).
struct TreePlan {
    int nu, rows, n_cg;           // units of a row, rows, groups of columns
};
// unit: positions of a unit; group: columns of a row
__host__ __device__ inline TreePlan tree_plan(int len, int n_new, int n_kv, int n_rep, int group, int unit)
{
    TreePlan p;
    p.nu = n_new > 0 && len > 0 ? (len + unit - 1) / unit : 0;
    p.n_cg = (n_new * n_rep + group - 1) / group;
    p.rows = p.nu ? n_kv * p.n_cg : 0;
    return p;
}
__host__ __device__ inline int tree_places(const TreePlan &p, int open) { return p.rows * (p.nu + open); }

// pre[i]: places before sequence i, by the first NT threads of a block that
// meets as a whole.
template <int NT, int N>
__device__ __forceinline__ void tree_scan(const TreeArgs &a, const KvRows<N> &rows, int unit, int *pre, int *sums)
{
    constexpr int PER = (N + NT - 1) / NT;
    const int     tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = rows.n;
    int           c[PER], sum = 0, run = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int i = tid * PER + k;
        c[k] = 0;
        if (i < n && tid < NT) {
            const int len = min(max(__ldg(a.len + rows.seq[i]), 0), a.max_pages * KV4_PAGE);
            c[k] = tree_places(tree_plan(len, rows.row0[i + 1] - rows.row0[i], a.n_kv, a.n_rep, a.group, unit), a.open);
        }
        sum += c[k];
    }
    if (tid < NT) {
        run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        if (lane == 31) sums[warp] = run;
    }
    __syncthreads();
    if (tid < NT) {
        run -= sum;
        for (int w = 0; w < warp; w++) run += sums[w];
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const int i = tid * PER + k;
            if (i < n) pre[i] = run;
            run += c[k];
            if (i == n - 1) pre[n] = run;
        }
    }
    __syncthreads();
}

// A row: sequence i, KV head r / n_cg, group of columns r % n_cg; its first
// place, and the units [j0, j1) of it that fall to the CTA with the places
// [cu0, cu1).  first() and next() walk the rows that have units there: places
// are a.open (what its beginning and end cost) and then one a unit.
template <int N> struct TreeWalk {
    const TreeArgs  &a;
    const KvRows<N> &rows;
    const int       *pre;
    int              unit, total, cu0, cu1;
    int              i, r, nu, n_rows, n_cg, place, j0, j1;

    __device__ __forceinline__ TreeWalk(const TreeArgs &a_, const KvRows<N> &rows_, const int *pre_, int unit_, int cta, int ctas)
        : a(a_), rows(rows_), pre(pre_), unit(unit_), total(pre_[rows_.n])
    {
        cu0 = (int)((long long)total * cta / ctas);
        cu1 = (int)((long long)total * (cta + 1) / ctas);
        int lo = 0, hi = rows.n;                          // the last sequence whose places begin at or before cu0
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= cu0) lo = mid;
            else hi = mid;
        }
        i = lo;
        enter();
        r = (cu0 - place) / (nu + a.open);
        place += r * (nu + a.open);
        range();
        while (place < cu1 && j1 <= j0) next();           // (its units end before the run, or begin behind it)
    }
    __device__ __forceinline__ int  len() const { return min(max(__ldg(a.len + rows.seq[i]), 0), a.max_pages * KV4_PAGE); }
    __device__ __forceinline__ void range()
    {
        j0 = max(0, cu0 - place - a.open);
        j1 = min(nu, cu1 - place - a.open);
    }
    __device__ __forceinline__ void enter()
    {
        const TreePlan p = tree_plan(len(), rows.row0[i + 1] - rows.row0[i], a.n_kv, a.n_rep, a.group, unit);
        nu = p.nu;
        n_rows = p.rows;
        n_cg = p.n_cg;
        r = 0;
        place = pre[i];
    }
    __device__ __forceinline__ bool here() const { return place < cu1 && j1 > j0; }
    __device__ __forceinline__ void next()
    {
        place += nu + a.open;
        if (++r == n_rows) {
            do i++;
            while (i < rows.n && pre[i + 1] == pre[i]);
            if (i < rows.n) enter();
            else place = total;
        }
        range();
    }
    __device__ __forceinline__ int page(int j) const { return __ldg(a.table + (size_t)rows.seq[i] * a.max_pages + j); }
};

// A sequence without positions: zeros.
template <typename T, int N> __device__ __forceinline__ void tree_zeros(const TreeArgs &a, const KvRows<N> &rows, const int *pre, int hd)
{
    for (int i = blockIdx.x; i < rows.n; i += gridDim.x)
        if (pre[i + 1] == pre[i])
            for (int r = rows.row0[i]; r < rows.row0[i + 1]; r++)
                for (int x = threadIdx.x; x < a.n_kv * a.n_rep * hd; x += blockDim.x) ((T *)a.out)[(size_t)r * a.out_stride + x] = kv4_from<T>(0.0f);
}

template <typename T, int NB, int N>
__global__ void __launch_bounds__(TREE_WARPS * 32, 1) k_kv4_tree(const __grid_constant__ TreeArgs a, const __grid_constant__ KvRows<N> rows)
{
    using S = TreeShape<T, NB>;
    constexpr int HD = S::HD, P = S::P, C = S::C, STAGE = S::STAGE, LD = S::LD, RR = P == 2 ? 1 : 2;
    extern __shared__ __align__(128) uint8_t smem[];
    float *parts = reinterpret_cast<float *>(smem + S::ring);
    int   *pre = reinterpret_cast<int *>(smem + S::ring + S::parts);
    __shared__ float ml_s[2][2][TREE_WARPS][C];           // each warp's M and weights' sums, of two rows in turn
    __shared__ int   sums[TREE_WARPS];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int WC = a.wc, WP = TREE_WARPS / WC, wc = warp % WC, wp = warp / WC;
    pdl_wait();
    pdl_trigger();
    tree_scan<TREE_WARPS * 32>(a, rows, KV4_UNIT, pre, sums);
    tree_zeros<T>(a, rows, pre, HD);
    const int ctas = min((int)gridDim.x, pre[rows.n]);
    if ((int)blockIdx.x >= ctas) return;
    TreeWalk<N> row(a, rows, pre, KV4_UNIT, blockIdx.x, ctas);

    // ---- the group's copies: cursor `ahead` runs before the products
    const int      gt = WC * 32, gtid = wc * 32 + lane, A = WC == 1 ? 2 : 3, ST = WC == 1 ? 2 : 4;
    uint8_t       *ring = smem + (size_t)wp * ST * STAGE;
    const uint32_t ring_at = smem_addr(ring);
    TreeWalk<N>    ahead = row;
    int            aj = ahead.j0 + wp;
    auto settle = [&] {                                   // ahead's unit, in whichever row it lies
        while (ahead.place < ahead.cu1 && aj >= ahead.j1) {
            ahead.next();
            aj = ahead.j0 + wp;
        }
    };
    auto page_at = [&] { return ahead.place < ahead.cu1 ? ahead.page(aj / (KV4_PAGE / KV4_UNIT)) : 0; };
    settle();
    int  page = page_at();
    auto issue = [&](int slot) {
        if (ahead.place < ahead.cu1) {
            const size_t   at = (size_t)min(max(page, 0), a.n_pages - 1) * a.page_bytes + (size_t)(ahead.r / ahead.n_cg) * (72 * HD);
            const uint8_t *src = a.layer + at;
            const int      half = aj & 1;
            const uint32_t dst = ring_at + slot * STAGE;
            for (int x = gtid; x < STAGE / 16; x += gt) {
                int off;
                if (x < 2 * HD) off = (x >= HD ? 32 * HD - 16 * HD : 0) + half * 16 * HD;
                else off = 64 * HD - 32 * HD + half * 2 * HD + (x >= 2 * HD + HD / 8 ? 2 * HD : 0);
                kv4_cp16(dst + 16 * x, src + off + 16 * x);
            }
            aj += WP;
            settle();
            page = page_at();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto meet = [&] {
        if (WC == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + wp), "r"(gt) : "memory");
    };
    for (int k = 0; k < A; k++) issue(k);
    int slot = 0, slot_in = A % ST;

    const KvMagic magic;
    const int     mt_row = (lane & 7) + ((lane >> 3) & 1) * 8, mt_blk = lane >> 4;
    uint32_t      qf[NB][2][4];
    float         O[NB][4][4], M[RR], l[RR], fac[RR];
    unsigned long long seen[RR];
    auto half_of = [](uint32_t w, int k) {
        const __half2 h = *reinterpret_cast<const __half2 *>(&w);
        return k ? __high2float(h) : __low2float(h);
    };

    // One unit at position t0.  CUT: some of its positions are drafted, or behind the end
    auto unit = [&](const uint8_t *st, int t0, int base, int len, auto cut) {
        constexpr bool CUT = decltype(cut)::value;
        const uint32_t kaddr = smem_addr(st), vaddr = kaddr + 16 * HD;
        float          sc[4][2 * RR];                     // [tile of 8 positions][row][position 2c + e]
        uint32_t       vs[4][NB];                         // V scales of this thread's two positions of each tile
        float          top[RR];
        uint32_t       live[RR];                          // CUT: bit 2 * tile + e
        __half2        vm = __float2half2_rn(0.0f);
        float          vrow[RR];
#pragma unroll
        for (int x = 0; x < RR; x++) {
            top[x] = -INFINITY;
            vrow[x] = 0.0f;
            live[x] = 0u;
        }
        if (CUT)
#pragma unroll
            for (int nt = 0; nt < 4; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int t = t0 + 8 * nt + 2 * c + e;
#pragma unroll
                    for (int x = 0; x < RR; x++)
                        if (t < len && (t < base || (seen[x] >> (t - base) & 1u))) live[x] |= 1u << (2 * nt + e);
                }
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
            uint64_t acc[2][2];                           // pairs of positions 2c, 2c + 1
            uint32_t ks[2][NB];
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const uint32_t *kp = reinterpret_cast<const uint32_t *>(st + 32 * HD + (16 * kt + 8 * y + 2 * c) * NB * 2);
                const uint32_t *vp = reinterpret_cast<const uint32_t *>(st + 34 * HD + (16 * kt + 8 * y + 2 * c) * NB * 2);
#pragma unroll
                for (int k = 0; k < NB; k++) {
                    ks[y][k] = kp[k];
                    vs[2 * kt + y][k] = vp[k];
                }
                acc[y][0] = acc[y][1] = 0ull;
            }
            const int t2 = kt * 16 + mt_row;
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                uint32_t r[4];
                if (b + 1 < NB) kv4_ldsm<false, true>(r, kaddr + t2 * (HD / 2) + kv4_place(t2, b + mt_blk, NB) * 16);
                else kv4_ldsm<false, false>(r, kaddr + t2 * (HD / 2) + kv4_place(t2, b, NB) * 16);
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    if (b + d >= NB) continue;
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        uint32_t x[4];
                        float    e[4];
                        magic.unpack(r[2 * d + y], x);
                        const uint32_t(&q0)[4] = qf[b + d][0], (&q1)[4] = qf[b + d][1];
                        kv4_mma0(e, q0[0], q0[1], q0[2], q0[3], x[0], x[1]);
                        kv4_mma(e, q1[0], q1[1], q1[2], q1[3], x[2], x[3]);
                        const float s0 = half_of(ks[y][(b + d) / 2], (b + d) & 1), s1 = half_of(ks[y][(NB + b + d) / 2], (NB + b + d) & 1);
                        const uint64_t s2 = tree_two(s0, s1);
                        acc[y][0] = tree_fma2(s2, tree_two(e[0], e[1]), acc[y][0]);
                        acc[y][1] = tree_fma2(s2, tree_two(e[2], e[3]), acc[y][1]);
                    }
                }
            }
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int nt = 2 * kt + y;
                float     row[2][2];
                tree_untwo(acc[y][0], row[0][0], row[0][1]);
                tree_untwo(acc[y][1], row[1][0], row[1][1]);
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int x = 0; x < RR; x++) {
                        const float s = P == 2 ? row[0][e] + row[1][e] : row[x][e];
                        sc[nt][2 * x + e] = s;
                        if (!CUT || (live[x] >> (2 * nt + e) & 1u)) top[x] = fmaxf(top[x], s);
                    }
#pragma unroll
                for (int k = 0; k < NB; k++) {
                    const __half2 h = __habs2(*reinterpret_cast<const __half2 *>(&vs[nt][k]));
                    if (!CUT) vm = __hmax2(vm, h);
                    else
#pragma unroll
                        for (int x = 0; x < RR; x++) {    // half 2k of a position pair's 2 NB scales belongs to position 2k / NB
                            if (live[x] >> (2 * nt + (2 * k) / NB) & 1u) vrow[x] = fmaxf(vrow[x], __low2float(h));
                            if (live[x] >> (2 * nt + (2 * k + 1) / NB) & 1u) vrow[x] = fmaxf(vrow[x], __high2float(h));
                        }
                }
            }
        }
        // the V scales are below 2^ve (scales below 2^-24 are zeros)
        auto exponent = [](float v) { return (float)max((int)(__float_as_uint(v) >> 23) - 126, -24); };
        if (!CUT)
#pragma unroll
            for (int x = 0; x < RR; x++) vrow[x] = fmaxf(__low2float(vm), __high2float(vm));
        auto still = [&](int x) { return top[x] + exponent(vrow[x]) <= M[x] + KV4_SLACK || (CUT && live[x] == 0u); };
        bool calm = true;
#pragma unroll
        for (int x = 0; x < RR; x++) {
            top[x] *= fac[x];
            calm = calm && still(x);
        }
        if (!__all_sync(0xffffffffu, calm)) {
            // M follows the largest score + log2 of the largest V scale
#pragma unroll
            for (int x = 0; x < RR; x++) {
                const unsigned asked = __ballot_sync(0xffffffffu, !still(x)) >> (lane & 28) & 15u;
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    vrow[x] = fmaxf(vrow[x], __shfl_xor_sync(0xffffffffu, vrow[x], o));
                    top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], o));
                }
                // (of this row alone, and where one of its own lanes asked for it: no row's bits depend on what shares its tile)
                const float m = top[x] + exponent(vrow[x]);
                const bool  grow = asked && m > M[x] + KV4_SLACK;
                const float alpha = grow ? kv4_ex2(kv4_rel(M[x]) - kv4_rel(m)) : 1.0f;
                if (grow) M[x] = m;
                l[x] *= alpha;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        O[b][j][2 * x] *= alpha;
                        O[b][j][2 * x + 1] *= alpha;
                        if (P == 2) {
                            O[b][j][2] *= alpha;
                            O[b][j][3] *= alpha;
                        }
                    }
            }
        }
#pragma unroll
        for (int x = 0; x < RR; x++) {
            // (17 short sequences take 35.8 us for 35.3 with scores as they may be, past KV4_FAR, 32 in fp32 444 for 434)
            float off = KV4_BASE - M[x], times = fac[x];
            if (kv4_far(M[x])) {
                off = -M[x];
                times = 1.0f;
#pragma unroll
                for (int nt = 0; nt < 4; nt++)
#pragma unroll
                    for (int e = 0; e < 2; e++) sc[nt][2 * x + e] *= fac[x];
            }
#pragma unroll
            for (int nt = 0; nt < 4; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float p = kv4_ex2(fmaf(sc[nt][2 * x + e], times, off));
                    if (CUT && !(live[x] >> (2 * nt + e) & 1u)) p = 0.0f;
                    sc[nt][2 * x + e] = p;
                    l[x] += p;
                }
        }
#pragma unroll
        for (int b = 0; b < NB; b += 2) {
            uint32_t r[2][4];
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const int t2 = kt * 16 + mt_row;
                if (b + 1 < NB) kv4_ldsm<true, true>(r[kt], vaddr + t2 * (HD / 2) + kv4_place(t2, b + mt_blk, NB) * 16);
                else kv4_ldsm<true, false>(r[kt], vaddr + t2 * (HD / 2) + kv4_place(t2, b, NB) * 16);
            }
#pragma unroll
            for (int d = 0; d < 2; d++) {
                if (b + d >= NB) continue;
                float e[4][4];
#pragma unroll
                for (int kt = 0; kt < 2; kt++) {
                    uint32_t x[4], y[4], w[4];
                    magic.unpack(r[kt][2 * d], x);
                    magic.unpack(r[kt][2 * d + 1], y);
#pragma unroll
                    for (int s = 0; s < 2; s++) {         // the two tiles of 8 positions
                        const int   nt = 2 * kt + s;
                        const float v0 = half_of(vs[nt][(b + d) / 2], (b + d) & 1), v1 = half_of(vs[nt][(NB + b + d) / 2], (NB + b + d) & 1);
                        // (the scale of a position that is not seen may be NaN)
                        auto times = [&](int z, int y, float v) { return CUT && !(live[z] >> (2 * nt + y) & 1u) ? 0.0f : sc[nt][2 * z + y] * v; };
                        if (P == 2) {
                            const float   w0 = times(0, 0, v0), w1 = times(0, 1, v1);
                            const __half2 hi = __floats2half2_rn(w0, w1);
                            const __half2 lo = __floats2half2_rn(w0 - __low2float(hi), w1 - __high2float(hi));
                            w[2 * s] = *reinterpret_cast<const uint32_t *>(&hi);
                            w[2 * s + 1] = *reinterpret_cast<const uint32_t *>(&lo);
                        } else {
#pragma unroll
                            for (int z = 0; z < 2; z++) {
                                const __half2 h = __floats2half2_rn(times(z % RR, 0, v0), times(z % RR, 1, v1));
                                w[2 * s + z] = *reinterpret_cast<const uint32_t *>(&h);
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (P == 1) kv4_mma(O[b + d][j], w[0], w[1], w[2], w[3], x[j], y[j]);
                        else if (kt == 0) kv4_mma0(e[j], w[0], w[1], w[2], w[3], x[j], y[j]);
                        else kv4_mma(e[j], w[0], w[1], w[2], w[3], x[j], y[j]);
                    }
                }
                if (P == 2)                               // (the tensor core cuts off where fp32 addition rounds)
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int k = 0; k < 4; k += 2)
                            tree_untwo(tree_add2(tree_two(O[b + d][j][k], O[b + d][j][k + 1]), tree_two(e[j][k], e[j][k + 1])), O[b + d][j][k], O[b + d][j][k + 1]);
            }
        }
    };

    int which = 0;
    for (; row.here(); row.next(), which ^= 1) {
        float(&ml)[2][TREE_WARPS][C] = ml_s[which];
        const int len = row.len(), r0 = rows.row0[row.i], n_new = rows.row0[row.i + 1] - r0, base = len - n_new;
        const int kvh = row.r / row.n_cg, cg = row.r - kvh * row.n_cg, cols = n_new * a.n_rep;
        const int col0 = (cg * WC + wc) * C;              // this warp's first column
        const bool mine = col0 < cols;
        // ---- this warp's queries, scaled into fp16's range, and its softmax from nothing
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int   col = col0 + g + (P == 1 ? 8 * x : 0), t = col / a.n_rep, h = col - t * a.n_rep;
            const bool  there = col < cols;
            float       v[NB][8], m = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (there) kv4_load8((const T *)a.q + (size_t)(r0 + t) * a.q_stride + (size_t)(kvh * a.n_rep + h) * HD + 32 * b + 8 * c, a.wide_q, v[b]);
                else
#pragma unroll
                    for (int k = 0; k < 8; k++) v[b][k] = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(v[b][k]));
            }
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            // 2^sh brings m to [2^13, 2^14); held where both it and its inverse are normal numbers
            const int   sh = min(126, max(-126, 140 - (int)((__float_as_uint(fmaxf(m, 1e-38f)) >> 23) & 255)));
            const float up = copysignf(__uint_as_float((uint32_t)(sh + 127) << 23), a.scale);
            if (x < RR) {
                fac[x] = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - sh) << 23);
                M[x] = -INFINITY;
                l[x] = 0.0f;
                seen[x] = !there ? 0ull : a.mask ? (unsigned long long)__ldg(a.mask + r0 + t) : (2ull << t) - 1;
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                __half h8[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float y = v[b][k] * up;
                    h8[k] = __float2half_rn(y);
                    if (P == 2 && x == 1) h8[k] = __float2half_rn(y - __half2float(h8[k]));
                }
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    qf[b][s][x] = kv4_pack(h8[2 * s], h8[2 * s + 4]);
                    qf[b][s][2 + x] = kv4_pack(h8[2 * s + 1], h8[2 * s + 5]);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int k = 0; k < 4; k++) O[b][j][k] = 0.0f;
        for (int j = row.j0 + wp; j < row.j1; j += WP) {
            if (WC == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
            else asm volatile("cp.async.wait_group 2;" ::: "memory");
            meet();
            if (WC > 1) issue(slot_in);                   // (the group is done with the unit that lay there)
            if (mine) {
                const int t0 = j * KV4_UNIT;
                if (t0 + KV4_UNIT <= base) unit(ring + slot * STAGE, t0, base, len, std::false_type());
                else unit(ring + slot * STAGE, t0, base, len, std::true_type());
            }
            if (WC == 1) {
                __syncwarp();
                issue(slot);
            }
            slot = slot + 1 == ST ? 0 : slot + 1;
            slot_in = slot_in + 1 == ST ? 0 : slot_in + 1;
        }
        // ---- the row's end: the groups' partials, each relative to the largest M
#pragma unroll
        for (int x = 0; x < RR; x++) {
            M[x] = kv4_rel(M[x]);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            if (c == 0) {
                ml[0][warp][g + 8 * x] = M[x];
                ml[1][warp][g + 8 * x] = l[x];
            }
        }
        __syncthreads();
        // M follows what is no NaN: a partial of NaN scores alone has M = -inf, weight 0 and sums of NaN
        auto weigh = [](float m, float top, float sum) { return sum == 0.0f ? 0.0f : kv4_ex2(m - top); };
        auto most = [&](int w0, int col) {
            float m = -INFINITY;
            for (int k = 0; k < WP; k++) m = fmaxf(m, ml[0][k * WC + w0][col]);
            return m;
        };
#pragma unroll
        for (int x = 0; x < RR; x++) {
            const float f = weigh(M[x], most(wc, g + 8 * x), l[x]);
            float      *to = parts + (size_t)(warp * C + g + 8 * x) * LD + 8 * c;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float4 v;
                    float *vp = reinterpret_cast<float *>(&v);
#pragma unroll
                    for (int j = 0; j < 4; j++) vp[j] = f * (P == 2 ? O[b][j][e] + O[b][j][2 + e] : O[b][j][2 * x + e]);
                    *reinterpret_cast<float4 *>(to + 32 * b + 4 * e) = v;
                }
        }
        __syncthreads();
        const bool complete = row.j0 == 0 && row.j1 == row.nu;
        float     *entry = a.part + ((size_t)blockIdx.x * 2 + (row.j0 == 0)) * (S::EC * (HD + 2));
        for (int x = tid; x < WC * C * (HD / 4); x += TREE_WARPS * 32) {
            const int d4 = x % (HD / 4), cc = x / (HD / 4), w0 = cc / C, cw = cc - w0 * C, col = cg * WC * C + cc;
            if (col >= cols) continue;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = 0; k < WP; k++) {
                const float4 v = *reinterpret_cast<const float4 *>(parts + (size_t)((k * WC + w0) * C + cw) * LD + 4 * d4);
                s.x += v.x;
                s.y += v.y;
                s.z += v.z;
                s.w += v.w;
            }
            const float m = most(w0, cw);
            float       L = 0.0f;
            for (int k = 0; k < WP; k++) {
                const float lk = ml[1][k * WC + w0][cw];
                L = fmaf(weigh(ml[0][k * WC + w0][cw], m, lk), lk, L);
            }
            if (complete) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;       // a row that sees nothing: zeros
                const int   t = col / a.n_rep, h = col - t * a.n_rep;
                T          *o = (T *)a.out + (size_t)(r0 + t) * a.out_stride + (size_t)(kvh * a.n_rep + h) * HD + 4 * d4;
                o[0] = kv4_from<T>(s.x * inv);
                o[1] = kv4_from<T>(s.y * inv);
                o[2] = kv4_from<T>(s.z * inv);
                o[3] = kv4_from<T>(s.w * inv);
            } else {
                reinterpret_cast<float4 *>(entry)[cc * (HD / 4) + d4] = s;
                if (d4 == 0) {
                    entry[S::EC * HD + cc] = m;
                    entry[S::EC * (HD + 1) + cc] = L;
                }
            }
        }
        // (the next row writes into the other half of ml_s, and into parts behind its first barrier)
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Rows that several CTAs share: a block per CTA and `slice` columns, which has
// work where a row begins in that CTA and goes on behind it; a warp takes columns
// in turn.
template <typename T, int NB, int N>
__global__ void __launch_bounds__(256) k_kv4_tree_join(const __grid_constant__ TreeArgs a, const __grid_constant__ KvRows<N> rows, int unit, int grid, int slice)
{
    constexpr int  HD = NB * 32;
    __shared__ int pre[N + 1], sums[8];
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = rows.n, EC = a.entry;
    pdl_wait();
    pdl_trigger();
    tree_scan<256>(a, rows, unit, pre, sums);
    const int total = pre[n], ctas = min(grid, total), slices = (a.group + slice - 1) / slice, cta = blockIdx.x / slices;
    if (cta >= ctas) return;
    auto begin_of = [&](int b) { return (int)((long long)total * b / ctas); };
    const int cu0 = begin_of(cta), cu1 = begin_of(cta + 1);
    // the row of the run's last place
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= cu1 - 1) lo = mid;
        else hi = mid;
    }
    const int      len = min(max(__ldg(a.len + rows.seq[lo]), 0), a.max_pages * KV4_PAGE), r0 = rows.row0[lo], n_new = rows.row0[lo + 1] - r0;
    const TreePlan p = tree_plan(len, n_new, a.n_kv, a.n_rep, a.group, unit);
    const int      r = (cu1 - 1 - pre[lo]) / (p.nu + a.open), begin = pre[lo] + r * (p.nu + a.open) + a.open, end = begin + p.nu;
    if (begin < cu0 || begin >= cu1 || end <= cu1) return;
    int last = (int)((long long)(end - 1) * ctas / total);          // the CTA of the row's last unit
    while (begin_of(last + 1) <= end - 1) last++;
    while (begin_of(last) > end - 1) last--;
    const int np = last - cta + 1, kvh = r / p.n_cg, cg = r - kvh * p.n_cg;
    auto      entry = [&](int b) { return a.part + ((size_t)(cta + b) * 2 + (b == 0)) * ((size_t)EC * (HD + 2)); };
    const int cc0 = (blockIdx.x % slices) * slice;
    for (int cc = cc0 + warp; cc < min(cc0 + slice, a.group); cc += 8) {
        const int col = cg * a.group + cc;
        if (col >= n_new * a.n_rep) return;
        float m = -INFINITY, L = 0.0f;
        for (int b = lane; b < np; b += 32) m = fmaxf(m, __ldcg(entry(b) + EC * HD + cc));
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int b0 = 0; b0 < np; b0 += 32) {
            float w = 0.0f;
            if (b0 + lane < np) {
                const float l = __ldcg(entry(b0 + lane) + EC * (HD + 1) + cc);
                w = l == 0.0f ? 0.0f : kv4_ex2(__ldcg(entry(b0 + lane) + EC * HD + cc) - m);
                L = fmaf(w, l, L);
            }
            const int k1 = min(32, np - b0);
#pragma unroll 4
            for (int k = 0; k < k1; k++) {
                const float f = __shfl_sync(0xffffffffu, w, k);
                if (lane < HD / 4) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(entry(b0 + k)) + cc * (HD / 4) + lane);
                    s.x = fmaf(f, v.x, s.x);
                    s.y = fmaf(f, v.y, s.y);
                    s.z = fmaf(f, v.z, s.z);
                    s.w = fmaf(f, v.w, s.w);
                }
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if (lane >= HD / 4) continue;
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        const int   t = col / a.n_rep, h = col - t * a.n_rep;
        T          *o = (T *)a.out + (size_t)(r0 + t) * a.out_stride + (size_t)(kvh * a.n_rep + h) * HD + 4 * lane;
        o[0] = kv4_from<T>(s.x * inv);
        o[1] = kv4_from<T>(s.y * inv);
        o[2] = kv4_from<T>(s.z * inv);
        o[3] = kv4_from<T>(s.w * inv);
    }
}
