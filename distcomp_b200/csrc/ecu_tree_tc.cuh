// ecu_tree_tc.cuh -- the attention of ecu_tree.cuh for many columns of 16-bit
// queries, on tcgen05.
//
// A row of work is up to 128 columns of one KV head of one sequence, a unit 128
// positions: S = Q K^T (fp32, tensor memory), P = 2^(S scale - M) rounded to
// fp16 over S's place, O += P V (fp32, tensor memory).  Roles by warp:
//   0-15  softmax, four threads a column (32 positions each); O's rescaling and
//         the output at a row's end
//   16-19 K, 20-23 V: codes and scales become fp16 operands in shared memory;
//         16-19 the queries into tensor memory at a row's beginning
//   24    issues the products
//   25    copies the units' pages as they lie into shared memory
//   26    looks for large scales in them, and tells the others what a unit is
//   (27 idle: registers move by groups of four warps, from the 72 a thread
//   that the block starts with to what each role wants)
// A chain of short steps bounds it (a unit's scores, their softmax, their
// product with V), not any one unit of the SM: so the roles are many and run
// apart, on two units' operands.  64 drafts behind 131025 positions (32 query
// and 8 KV heads of 128, bf16) take 228 us: 603 TFLOP/s, the tensor pipe 31 % and
// the issue slots 67 % in use, 152 MB read once at 0.65 TB/s; 32 sequences of 1 to
// 4096 positions with 1 to 24 drafts (64 and 8 heads) 137 us, of which the
// products take 22 % of the tensor pipe (columns that no row fills among them).
// The kernel on mma.sync takes 769 and 381.
// K and V are (code - 8) * scale rounded to fp16, as the batch's prompts take
// them (a score is off by 2^-11 of its products' size at most, an eighth of what
// the rounding of bf16 queries leaves; exact keys, with a second operand for
// their rest, took 1.4 times as long), the weights are rounded to fp16.
// Where a scale passes 2^12 (values past 2^15), the row's K and V are taken 2^-4
// smaller from that unit on, O with them.
// Positions that only some rows see (the drafted ones): their scores are taken
// out by selection; a NaN among their values is zeroed in the operand, noted,
// and given back at the row's end to the columns that see it.
//
// Tensor memory: S of units in turn at columns 0 and 128 (P in the first 16 of
// each 32), O at 256, the queries of rows in turn at 384 and 448.  Shared
// memory: tiles of 128 positions of 64 dimensions (128 bytes, 128-byte
// swizzle), HD / 64 of them side by side; within 8 dimensions the order is 0, 4,
// 1, 5, 2, 6, 3, 7, as codes unpack, in K and Q alike, and undone in the output.
#pragma once
#include "ecu_attn_prompt.cuh"
#include "ecu_tree.cuh"

#define TT_THREADS 896
// Registers a thread at launch (7 groups of four warps: 504 between them), and
// then 4 * 80 for the softmax, 2 * 64, 48.  More than there are would wait
// forever, so the launch looks at what the kernel was compiled to
// (tree_tc_fits).
#define TT_REGS 72
static_assert(4 * 80 + 2 * 64 + 48 <= 7 * TT_REGS, "the groups' registers are those of the launch");
#define TT_UNIT 128
#define TT_COLS 128
#define TT_OPEN 6                 // places of a row beside its units
#define TT_BASE 9.0f              // weights are 2^(t - M + TT_BASE) ...
#define TT_SLACK 6.0f             // ... and M follows when t has passed it by so much: below 2^15, and fp16 down to 2^-33
#define TT_SHIFT 4
#define TT_RING 4

template <int HD> struct TreeTc {
    static constexpr int NB = HD / 32, B = HD / 64, TILE = B * PA_BOX;
    static constexpr size_t tiles = (size_t)4 * TILE;             // K and V of two units
    static constexpr int    PAGES = 144 * HD;                     // a unit's two pages as they lie, of TT_RING units
    static constexpr size_t smem(int n) { return 1024 + tiles + TT_RING * PAGES + (size_t)(n + 1) * 4; }
};

// Does any of the 128 threads at barrier `id` say so?
__device__ __forceinline__ bool tt_any(int id, bool mine)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                 "barrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((uint32_t)mine), "r"(id) : "memory");
    return any != 0;
}

// What the roles know of a unit; warp 26 writes it, for eight units in turn (a
// unit that far ahead is copied only after this one's products).
struct TtUnit {
    int r0, n_new, len;           // the sequence's first row, its drafted rows, its positions
    int kvh, cg, j;               // KV head, group of 128 columns, place of the unit
    int row;                      // number of its row in the CTA
    int flags;
};
#define TT_FIRST 1                // of its row's units in this CTA
#define TT_LAST 2
#define TT_MORE 4                 // another unit follows
#define TT_WHOLE 8                // all of the row's units are this CTA's
#define TT_BEGINS 16              // the row's first unit is
#define TT_SHIFTED 32             // operands are taken 2^-TT_SHIFT smaller

template <typename T, int HD, int N>
__global__ void __launch_bounds__(TT_THREADS, 1) k_kv4_tree_tc(const __grid_constant__ TreeArgs a, const __grid_constant__ KvRows<N> rows,
                                                              int *status, int stall)
{
    using S = TreeTc<HD>;
    constexpr int NB = S::NB, B = S::B, TILE = S::TILE, CH = NB;     // chunks of K, or of V, a thread
    extern __shared__ uint8_t raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    uint8_t *pages_s = sm + S::tiles;
    int     *pre = reinterpret_cast<int *>(pages_s + TT_RING * S::PAGES);
    __shared__ __align__(8) uint64_t k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2], raw_full[TT_RING], raw_ready[TT_RING], raw_free[TT_RING], pv_done, drain;
    __shared__ uint32_t              tmem_s;
    __shared__ int                   dead, sums[TT_THREADS / 32];
    __shared__ float                 part_s[4][TT_COLS], fac_s[8][TT_COLS];     // fac_s: of eight rows in turn
    __shared__ unsigned long long    bad_s[8][NB];                              // drafted positions whose V block is NaN
    __shared__ __align__(16) TtUnit  unit_s[8];
    __shared__ int                   any_s;                                     // the CTA has units
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (warp == 24) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(k_full + s, 4);
            mbar_init(k_free + s, 1);
            mbar_init(v_full + s, 4);
            mbar_init(v_free + s, 1);
            mbar_init(s_full + s, 1);
            mbar_init(p_full + s, 16);
        }
        for (int s = 0; s < TT_RING; s++) {
            mbar_init(raw_full + s, 1);
            mbar_init(raw_ready + s, 1);
            mbar_init(raw_free + s, 8);
        }
        mbar_init(&pv_done, 1);
        mbar_init(&drain, 1);
        mbar_init_fence();
        dead = 0;
    }
    pdl_wait();
    pdl_trigger();
    tree_scan<512>(a, rows, TT_UNIT, pre, sums);
    tree_zeros<T>(a, rows, pre, HD);
    const int ctas = min((int)gridDim.x, pre[rows.n]);
    if (tid == 800) any_s = (int)blockIdx.x < ctas && TreeWalk<N>(a, rows, pre, TT_UNIT, blockIdx.x, ctas).here();
    pa_fence_before();
    __syncthreads();
    pa_fence_after();
    const uint32_t tmem = tmem_s;
    // every wait is bounded; one that gives up lets the others give up too, and
    // the block's end flags the status
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (!pa_wait(bar, parity, &dead)) atomicExch(&dead, 1);
    };
    auto gone = [&] { return *reinterpret_cast<volatile int *>(&dead) != 0; };
    const uint32_t dk = smem_addr(sm), dv = dk + 2 * TILE;        // K of unit u at u & 1, V behind both

    if (!any_s) {
    } else if (warp >= 24) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 24) {
            const uint32_t ids = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
            const uint32_t ido = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((128u >> 4) << 24);
            const uint64_t kd = pa_desc(dk, 16), vd = pa_desc(dv, PA_BOX);
            auto until = [&](uint64_t *bar, uint32_t parity) {
                if (!pa_wait(bar, parity, &dead, status)) atomicExch(&dead, 1);
                __syncwarp();
            };
            auto qk = [&](int u, int row) {                   // unit u, the CTA's row-th row
                const uint32_t q = tmem + 384 + 64 * (row & 1);
                const uint64_t k = kd + (uint64_t)((u & 1) * (TILE >> 4));
#pragma unroll
                for (int x = 0; x < HD / 16; x++)
                    pa_mma_ts(tmem + 128 * (u & 1), q + 8 * x, k + (uint64_t)(((x / 4) * PA_BOX + (x % 4) * 32) >> 4), ids, x > 0);
                pa_commit(s_full + (u & 1));
                pa_commit(k_free + (u & 1));
            };
            auto pv = [&](int u, bool more) {
#pragma unroll
                for (int x = 0; x < 8; x++)
                    pa_mma_ts(tmem + 256, tmem + 128 * (u & 1) + 32 * (x / 2) + 8 * (x % 2), vd + (uint64_t)(((u & 1) * TILE + x * 2048) >> 4), ido, more || x > 0);
                pa_commit(v_free + (u & 1));
                pa_commit(&pv_done);
            };
            until(k_full + 0, 0);
            pa_fence_after();
            qk(0, 0);
            for (int u = 0, flags = TT_MORE; flags & TT_MORE; u++) {
                flags = unit_s[u & 7].flags;
                if (flags & TT_MORE) {                    // the next unit's scores, before this one's weights are waited for
                    until(k_full + ((u + 1) & 1), (uint32_t)((u + 1) >> 1) & 1u);
                    if (__any_sync(0xffffffffu, gone())) break;
                    pa_fence_after();
                    qk(u + 1, unit_s[(u + 1) & 7].row);
                }
                until(v_full + (u & 1), (uint32_t)(u >> 1) & 1u);
                until(p_full + (u & 1), (uint32_t)(u >> 1) & 1u);
                if (__any_sync(0xffffffffu, gone())) break;
                pa_fence_after();
                pv(u, !(flags & TT_FIRST));
            }
            pa_commit(&drain);
            // no product in flight when tensor memory is given back
            if (!mbar_drain(&drain, 0, wait_limit_ns())) atomicExch(&dead, 1);
        } else if (warp == 25) {
            // ---- the pages, as far ahead as the ring lets them
            int issued = 0;
            for (TreeWalk<N> w(a, rows, pre, TT_UNIT, blockIdx.x, ctas); w.here() && !__any_sync(0xffffffffu, gone()); w.next()) {
                const size_t head = (size_t)(w.r / w.n_cg) * (72 * HD);
                int          left = w.len() - w.j0 * TT_UNIT, page[2], next[2];
                auto         table = [&](int j, int left, int(&p)[2]) {
                    p[0] = left > 0 ? w.page(2 * j) : 0;
                    p[1] = left > KV4_PAGE ? w.page(2 * j + 1) : 0;
                };
                table(w.j0, left, page);
                for (int j = w.j0; j < w.j1; j++, issued++, left -= TT_UNIT) {
                    const int at = issued % TT_RING, both = left > KV4_PAGE;
                    table(j + 1, left - TT_UNIT, next);
                    if (issued >= TT_RING) wait(raw_free + at, (uint32_t)(issued / TT_RING - 1) & 1u);
                    if (__any_sync(0xffffffffu, gone())) break;
                    if (lane == 0) {
                        mbar_expect_tx(raw_full + at, both ? 144 * HD : 72 * HD);
                        for (int p = 0; p <= both; p++)
                            bulk_g2s(pages_s + at * S::PAGES + p * 72 * HD, a.layer + (size_t)min(max(page[p], 0), a.n_pages - 1) * a.page_bytes + head, 72 * HD, raw_full + at);
                    }
                    __syncwarp();
                    page[0] = next[0];
                    page[1] = next[1];
                }
            }
            // nothing on its way into shared memory when the block ends
            if (lane == 0)
                for (int x = max(0, issued - TT_RING); x < issued; x++)
                    if (!mbar_drain(raw_full + x % TT_RING, (uint32_t)(x / TT_RING) & 1u, wait_limit_ns())) atomicExch(&dead, 1);
            __syncwarp();
        } else if (warp == 26) {
            // ---- what the units are
            int         u = 0, row = 0;
            TreeWalk<N> w(a, rows, pre, TT_UNIT, blockIdx.x, ctas);
            for (bool on = true; on && !__any_sync(0xffffffffu, gone()); row++) {
                const int r0 = rows.row0[w.i], n_new = rows.row0[w.i + 1] - r0, len = w.len(), kvh = w.r / w.n_cg, cg = w.r - kvh * w.n_cg;
                const int j0 = w.j0, j1 = w.j1, how = (j0 == 0 && j1 == w.nu ? TT_WHOLE : 0) | (j0 == 0 ? TT_BEGINS : 0);
                int       shift = 0;
                w.next();
                on = w.here();
                for (int j = j0; j < j1; j++, u++) {
                    const uint8_t *raw_u = pages_s + u % TT_RING * S::PAGES + 64 * HD;
                    wait(raw_full + u % TT_RING, (uint32_t)(u / TT_RING) & 1u);
                    if (__any_sync(0xffffffffu, gone())) break;
                    // A scale past 2^12 (a NaN is none) of a position inside the sequence?  A page's scales are those of K and
                    // then those of V, 16 bytes of them 8 / NB positions.
                    __half2   most = __float2half2_rn(0.0f);
                    const int here = len - j * TT_UNIT;   // positions of the sequence from the unit's first on
#pragma unroll
                    for (int x = lane; x < HD; x += 32) {
                        const int   p = x / (HD / 2), in = x % (HD / 2) % (HD / 4);
                        const uint4 v = *reinterpret_cast<const uint4 *>(raw_u + p * 72 * HD + x % (HD / 2) * 16);
                        uint32_t    s2[4] = {v.x, v.y, v.z, v.w};
                        if (here < TT_UNIT) {             // (behind the end lies whatever does)
                            const int in_seq = (here - p * KV4_PAGE - in * (8 / NB)) * NB;
#pragma unroll
                            for (int k = 0; k < 4; k++) s2[k] &= (2 * k < in_seq ? 0xFFFFu : 0u) | (2 * k + 1 < in_seq ? 0xFFFF0000u : 0u);
                        }
#pragma unroll
                        for (int k = 0; k < 4; k++) most = __hmax2(most, __habs2(*reinterpret_cast<const __half2 *>(&s2[k])));
                    }
                    if (__any_sync(0xffffffffu, __low2float(most) >= 4096.0f || __high2float(most) >= 4096.0f)) shift = TT_SHIFTED;
                    if (lane < NB && j == j0) bad_s[row & 7][lane] = 0ull;
                    __syncwarp();
                    if (lane == 0) {
                        unit_s[u & 7] = {r0, n_new, len, kvh, cg, j, row,
                                         (j == j0 ? TT_FIRST : 0) | (j == j1 - 1 ? TT_LAST : 0) | (j < j1 - 1 || on ? TT_MORE : 0) | how | shift};
                        if (!(stall && u == 0)) mbar_arrive(raw_ready + u % TT_RING);
                    }
                }
            }
        }
    } else if (warp >= 16) {
        // ---- operands of K (warps 16-19) or V (20-23)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // Chunk i of a thread is 16 bytes of codes: position t + STEP i of the unit, block b (the same of all i).
        constexpr int  STEP = TT_UNIT / CH;
        const bool     is_v = warp >= 20;
        const int      me = tid & 127, t = me / NB, b = kv4_place(t, me % NB, NB);
        const uint8_t *code_at = pages_s + (is_v ? 32 * HD : 0) + t * (HD / 2) + (me % NB) * 16;
        const uint8_t *scale_at = pages_s + (is_v ? 68 * HD : 64 * HD) + (t * NB + b) * 2;
        // Its words of eight dimensions go to `to` ^ (16 * word) of a tile.  Blocks 2 and 3, in the other box, take their
        // words in the order 2, 3, 0, 1: eight threads, two positions of four blocks, then store to all eight 16-byte
        // columns of the banks.
        uint8_t       *tile = sm + (is_v ? 2 * TILE : 0);
        const uint32_t to = (b / 2) * PA_BOX + t * 128 + ((((b & 1) * 4) ^ (b & 2) ^ (t & 7)) * 16);
        const KvMagic  magic;
        uint64_t      *full = is_v ? v_full : k_full, *free = is_v ? v_free : k_free;
        for (int u = 0, flags = TT_MORE; flags & TT_MORE; u++) {
            wait(raw_ready + u % TT_RING, (uint32_t)(u / TT_RING) & 1u);
            if (u >= 2) wait(free + (u & 1), (uint32_t)((u >> 1) - 1) & 1u);
            if (__any_sync(0xffffffffu, gone())) break;   // (what a unit is, is known only where its wait ended well)
            const TtUnit &x = unit_s[u & 7];
            flags = x.flags;
            const int     left = x.len - x.j * TT_UNIT - t;       // positions of the sequence from t on
            const __half2 by = __half2half2(__ushort_as_half((unsigned short)((flags & TT_SHIFTED ? 15 - TT_SHIFT : 15) << 10)));
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const int      from = u % TT_RING * S::PAGES + STEP * i / KV4_PAGE * 72 * HD, in = STEP * i % KV4_PAGE;
                const uint4    c = *reinterpret_cast<const uint4 *>(code_at + from + in * (HD / 2));
                uint32_t       s = *reinterpret_cast<const unsigned short *>(scale_at + from + in * NB * 2);
                if (left <= STEP * i) s = 0u;             // behind the end: zeros
                if (is_v && (s & 0x7FFFu) > 0x7C00u && x.n_new + STEP * i >= left) {       // a drafted position's NaN
                    atomicOr(&bad_s[x.row & 7][b], 1ull << (x.n_new + STEP * i - left));
                    s = 0u;
                }
                const __half2  scale = __hmul2(__half2half2(__ushort_as_half((unsigned short)s)), by);
                const bool     turn = b & 2;
                const uint32_t code[4] = {turn ? c.z : c.x, turn ? c.w : c.y, turn ? c.x : c.z, turn ? c.y : c.w};
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    uint32_t n[4];
                    magic.unpack(code[y], n);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const __half2 p = __hmul2(*reinterpret_cast<const __half2 *>(&n[k]), scale);
                        n[k] = *reinterpret_cast<const uint32_t *>(&p);
                    }
                    *reinterpret_cast<uint4 *>(tile + (u & 1) * TILE + STEP * 128 * i + (to ^ 16 * y)) = make_uint4(n[0], n[1], n[2], n[3]);
                }
            }
            if (!is_v && flags & TT_FIRST) {              // the row's queries, a column a thread
                const int   cw = (warp & 3) * 32 + lane, col = x.cg * TT_COLS + cw, t = col / a.n_rep;
                const bool  there = t < x.n_new;
                const T    *q = (const T *)a.q + (size_t)(x.r0 + (there ? t : 0)) * a.q_stride + (size_t)(x.kvh * a.n_rep + (there ? col - t * a.n_rep : 0)) * HD;
                float       m = 0.0f, v[8];
#pragma unroll 2
                for (int d = 0; d < HD; d += 8) {
                    kv4_load8(q + d, a.wide_q, v);
#pragma unroll
                    for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(v[k]));
                }
                // 2^sh brings m to [2^13, 2^14); held where both it and its inverse are normal numbers
                const int   sh = min(126, max(-126, 140 - (int)((__float_as_uint(fmaxf(m, 1e-38f)) >> 23) & 255)));
                const float up = there ? copysignf(__uint_as_float((uint32_t)(sh + 127) << 23), a.scale) : 0.0f;
                fac_s[x.row & 7][cw] = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - sh) << 23);
                const uint32_t tq = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 384 + 64 * (x.row & 1);
#pragma unroll 1
                for (int d = 0; d < HD; d += 32) {
                    uint32_t o[16];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        kv4_load8(q + d + 8 * e, a.wide_q, v);
#pragma unroll
                        for (int k = 0; k < 4; k++) o[4 * e + k] = there ? kv4_pack(__float2half_rn(v[k] * up), __float2half_rn(v[k + 4] * up)) : 0u;
                    }
                    pa_st16(tq + d / 2, o);
                }
                pa_st_wait();
                pa_fence_before();
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(full + (u & 1));
                mbar_arrive(raw_free + u % TT_RING);
            }
        }
    } else {
        // ---- softmax.  The four warps of 32 columns meet in every unit, and leave together where a wait gave up.
        asm volatile("setmaxnreg.inc.sync.aligned.u32 80;");
        constexpr int  HQ = HD / 4;
        const int      qf = warp >> 2, cw = (warp & 3) * 32 + lane, team = 1 + (warp & 3);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, to = tmem + lanes + 256 + HQ * qf;
        float          m = -INFINITY, l = 0.0f, fac = 0.0f;       // M in units of t = S * fac * 2^shift; this quarter's weights' sum
        bool           shifted = false;
        unsigned long long mask = 0ull;
        // Unit u's weights in the place of its scores.  CUT: some of this quarter's 32 positions are not seen by all rows, or
        // lie behind the end; live has those that this column sees.  False where a wait gave up.
        auto unit = [&](int u, int flags, uint32_t live, auto cut) {
            constexpr bool CUT = decltype(cut)::value;
            const uint32_t ts = tmem + lanes + 128 * (u & 1) + 32 * qf;
            const bool     now = flags & TT_SHIFTED, turn = now != shifted;      // (once a row at most)
            uint32_t       s[2][16];
#pragma unroll
            for (int c = 0; c < 2; c++) pa_ld16(s[c], ts + 16 * c);
            pa_ld_wait();
#pragma unroll
            for (int c = 0; c < 2; c++) pa_pin(s[c]);
            if (CUT)
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int x = 0; x < 16; x++)
                        if (!(live >> (16 * c + x) & 1u)) s[c][x] = 0xFF800000u;
            float top[2];
#pragma unroll
            for (int q = 0; q < 2; q++) {
                auto v = [&](int x) { return __uint_as_float(s[q][x]); };
                top[q] = pa_max3(v(0), v(1), v(2));
#pragma unroll
                for (int x = 3; x < 15; x += 2) top[q] = pa_max3(top[q], v(x), v(x + 1));
                top[q] = pa_max(top[q], v(15));
            }
            float       sl = fac * (now ? (float)(1 << TT_SHIFT) : 1.0f);
            float       mx = pa_max(top[0], top[1]);
            mx = mx == -INFINITY ? mx : mx * sl;          // (0 * infinity is none)
            // not (mx within the slack of m): a NaN grows, and turns its whole row into NaN
            auto grows = [&] { return !(mx <= m) && !(mx - m <= TT_SLACK); };
            if (tt_any(team, grows() || turn || gone())) {
                part_s[qf][cw] = mx;
                if (tt_any(team, gone())) return false;
                mx = pa_max(pa_max3(part_s[0][cw], part_s[1][cw], part_s[2][cw]), part_s[3][cw]);
                const bool grow = grows(), first = flags & TT_FIRST;
                // (past 2^23, rounding the scores first, as ecu_tree.cuh's kernel does there, took 233 us for 223 at 131025
                // positions; this takes 227)
                const float less = grow ? pa_near(mx) : 1.0f;
                float       f = grow && !first ? kv4_ex2((m - mx) * less) : 1.0f;
                if (grow) m = mx * less;
                fac *= less;
                sl *= less;
                l *= f;
                if (turn) f *= 1.0f / (1 << TT_SHIFT);
                shifted = now;
                if (!first) {
                    wait(&pv_done, (uint32_t)(u - 1) & 1u);                  // the sums so far are complete
                    pa_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HQ; c += 16) {
                        uint32_t o[16];
                        pa_ld16(o, to + c);
                        pa_ld_wait();
                        pa_pin(o);
#pragma unroll
                        for (int x = 0; x < 16; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                        pa_st16(to + c, o);
                    }
                }
            }
            const float    mb = m == -INFINITY ? 0.0f : fmaf(m, 0.0f, TT_BASE - m);      // (an infinite maximum makes the row NaN)
            const uint64_t sl2 = pa_two(sl, sl), mb2 = pa_two(mb, mb);
            uint64_t       sum[2] = {pa_two(0.0f, 0.0f), pa_two(0.0f, 0.0f)};
            uint32_t       p[16];
#pragma unroll
            for (int x = 0; x < 16; x++) {
                const uint32_t *v = &s[x >> 3][2 * (x & 7)];
                const uint64_t  t2 = pa_fma2(pa_two(__uint_as_float(v[0]), __uint_as_float(v[1])), sl2, mb2);
                float           e0, e1;
                pa_untwo(t2, e0, e1);
                if (x % PA_FMA == PA_FMA - 1) {
                    e0 = pa_ex2_fma<4>(e0);
                    e1 = pa_ex2_fma<4>(e1);
                } else {
                    e0 = kv4_ex2(e0);
                    e1 = kv4_ex2(e1);
                }
                if (CUT) {                                // (what is not seen may be infinite times nothing)
                    e0 = live >> (2 * x) & 1u ? e0 : 0.0f;
                    e1 = live >> (2 * x) & 2u ? e1 : 0.0f;
                }
                sum[x & 1] = pa_add2(sum[x & 1], pa_two(e0, e1));
                p[x] = pa_pair(__half(), e0, e1);
            }
            pa_st16(ts, p);                               // over scores that this thread alone has read
            float a0, a1;
            pa_untwo(pa_add2(sum[0], sum[1]), a0, a1);
            l += a0 + a1;
            pa_st_wait();
            return true;
        };
        for (int u = 0, flags = TT_MORE; flags & TT_MORE; u++) {
            const TtUnit &x = unit_s[u & 7];
            wait(s_full + (u & 1), (uint32_t)(u >> 1) & 1u);
            flags = x.flags;
            // (what a unit is, is known only where its wait ended well: the warps' votes see to that)
            const bool some = x.cg * TT_COLS + (warp & 3) * 32 < x.n_new * a.n_rep;      // the warp's columns
            pa_fence_after();
            if (some && flags & TT_FIRST && !gone()) {
                const int t = (x.cg * TT_COLS + cw) / a.n_rep;
                mask = 0ull;
                if (t < x.n_new) mask = (a.mask ? (unsigned long long)__ldg(a.mask + x.r0 + t) : (2ull << t) - 1) & (~0ull >> (64 - x.n_new));
                fac = fac_s[x.row & 7][cw];
                m = -INFINITY;
                l = 0.0f;
                shifted = flags & TT_SHIFTED;
            }
            const int lo = x.len - x.n_new - (x.j * TT_UNIT + 32 * qf);      // positions of this quarter that every row sees
            if (!some) {
                if (tt_any(team, gone()) && tt_any(team, gone())) break;
            } else if (lo >= 32) {
                if (!unit(u, flags, 0u, std::false_type())) break;
            } else if (!unit(u, flags, (uint32_t)(lo >= 0 ? (1ull << lo) - 1 | mask << lo : lo > -64 ? mask >> -lo : 0ull), std::true_type()))
                break;
            pa_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + (u & 1));
            if (!(flags & TT_LAST)) continue;
            // ---- the row's end: this thread's half of its column's dimensions
            // (a parity tells a phase from the one before it alone: unit u - 1's first, which may still be on its way; unit
            // u - 2's products are behind unit u's scores)
            if (u > 0) wait(&pv_done, (uint32_t)(u - 1) & 1u);
            wait(&pv_done, (uint32_t)u & 1u);
            if (x.cg * TT_COLS + (warp & 3) * 32 >= x.n_new * a.n_rep) continue;
            pa_fence_after();
            named_bar(team, 128);
            part_s[qf][cw] = l;
            named_bar(team, 128);
            const float L = (part_s[0][cw] + part_s[1][cw]) + (part_s[2][cw] + part_s[3][cw]);
            const int   col = x.cg * TT_COLS + cw, t = col / a.n_rep;
            const bool  complete = flags & TT_WHOLE, there = t < x.n_new;
            const float up = shifted ? (float)(1 << TT_SHIFT) : 1.0f;
            const float inv = !complete ? up : L == 0.0f ? 0.0f : up / L;      // a row that sees nothing: zeros
            float      *entry = a.part + ((size_t)blockIdx.x * 2 + (flags & TT_BEGINS ? 1 : 0)) * ((size_t)TT_COLS * (HD + 2));
            T          *out = (T *)a.out + (size_t)(x.r0 + t) * a.out_stride + (size_t)(x.kvh * a.n_rep + col - t * a.n_rep) * HD + HQ * qf;
#pragma unroll 1
            for (int c = 0; c < HQ; c += 16) {
                uint32_t o[16];
                pa_ld16(o, to + c);
                pa_ld_wait();
                pa_pin(o);
                const bool nan = bad_s[x.row & 7][(HQ * qf + c) / 32] & mask;       // a NaN of a drafted position that the row sees
                float      y[16];
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const int from = (x & 8) + ((x & 7) < 4 ? 2 * (x & 7) : 2 * (x & 7) - 7);      // where dimension x lies
                    y[x] = nan ? NAN : __uint_as_float(o[from]) * inv;
                }
                if (!there) continue;
                if (complete) {
                    kv4_store8(out + c, a.wide_out, *reinterpret_cast<float(*)[8]>(y));
                    kv4_store8(out + c + 8, a.wide_out, *reinterpret_cast<float(*)[8]>(y + 8));
                } else
#pragma unroll
                    for (int x = 0; x < 16; x += 4)
                        *reinterpret_cast<float4 *>(entry + (size_t)cw * HD + HQ * qf + c + x) = make_float4(y[x], y[x + 1], y[x + 2], y[x + 3]);
            }
            if (!complete && there && qf == 0) {
                entry[TT_COLS * HD + cw] = fac == 0.0f ? m : m * (fac_s[x.row & 7][cw] / fac);
                entry[TT_COLS * (HD + 1) + cw] = L;
            }
            named_bar(team, 128);                         // part_s is free again
        }
    }
    pa_fence_before();
    __syncthreads();
    if (tid == 0 && gone()) atomicOr(status, ECU_STATUS_TIMEOUT);
    if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}
