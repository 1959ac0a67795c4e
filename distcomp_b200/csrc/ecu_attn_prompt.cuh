// ecu_attn_prompt.cuh -- causal attention of packed prompts on tcgen05.
//
// A CTA works on two query tiles of 128 rows (a "pair": query heads of one KV
// head, so that both read the same K and V) and walks their keys 128 at a
// time:  S = Q K^T (fp32, tensor memory), P = exp2(S * scale * log2 e - m)
// rounded to 16 bits over S's place, O += P V (fp32, tensor memory).  The two
// tiles take turns: while one's softmax runs, the tensor core computes the
// other's products.  Roles by warp:
//   0-7, 8-15 softmax of tile 0 and 1, two threads per row (64 keys each, so
//             that a tile's softmax is short beside the other tile's
//             products); O's rescaling and the output at the end
//   16        copies: Q once, K and V tiles through a ring (TMA)
//   17        issues the products (one thread)
//   18, 19    clean V tiles that some row sees only in part: an element that
//             is not finite would turn 0 * element into NaN for rows that do
//             not see it.  Such elements are zeroed in shared memory, their
//             keys noted, and added to the rows that do see them at the end.
// The maximum that P is taken relative to follows the running one only when
// that has grown by more than 2^8 (P stays far inside fp16's range, and the
// sums are fp32), so O is rescaled a few times per row at most, and a row's
// two threads exchange maxima only then: a vote between their two warps.
// The exponentials of a pair of tiles, 32768 at 16 a clock, take as long as
// its products at full rate; an eighth of them is computed on the FMA units
// instead (2^x = 2^n p(f) for |f| <= 1/2, p the polynomial of least relative
// error by the Remez exchange, whose extremes are equal: 7.5e-5 of degree 3 for
// bf16, whose own step is 2^-8, 2.7e-6 of degree 4 for fp16).
//
// 8192 tokens, 32 heads of 128 over 8: 549 us, 1001 TFLOP/s; the walk's turn of
// two tiles takes 1.5 times its products' time, the softmax of a tile being
// longer than the other tile's products, and a pair 7 us beside its walk.
//
// Tensor memory: S of tile t at column 128 t (P in the first 32 of each 64), O at
// 256 + HD t.  Shared memory: tiles of 128 rows of 64 elements (128 bytes,
// 128-byte swizzle), HD / 64 of them side by side; Q and K are K-major
// operands, V (keys x dimensions) is read MN-major.
#pragma once
#include "ecu_kv4.cuh"
#include "ecu_pipe.cuh"

#include <cuda.h>

#define PA_THREADS 640
#define PA_FMA 8                           // every PA_FMA-th pair of exponentials goes to the FMA units
#define PA_BOX 16384                       // 128 rows x 128 bytes

template <int HD> struct PaShape {
    static constexpr int B = HD / 64;              // boxes of a tile
    static constexpr int TILE = B * PA_BOX;
    // at hd 64 more stages than the walk needs: one CTA an SM, which takes all of tensor memory
    static constexpr int STAGES = HD == 128 ? 4 : 6;
    static constexpr size_t smem = 1024 + (size_t)(2 + STAGES) * TILE;
};

struct PromptArgs {
    const void *v;
    void       *out;
    long        v_stride, out_stride;
    int         n_kv, n_rep;
    float       scale;
    int        *status;           // ECU_STATUS_TIMEOUT where a wait gave up
    int         stall;            // 1: the first keys are never copied, so that a wait runs out
};

// Sequences of one launch by value, the longest first: where their rows lie
// and the CTA that begins them.
template <int N> struct PromptSeqs {
    int n;
    int q0[N], nq[N], k0[N], nk[N], cta[N + 1];
};

__device__ __forceinline__ void pa_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// The products and their commits are issued by one elected thread, but by a
// whole warp's control flow: elect.sync's predicate on the instruction itself
// keeps the descriptors in uniform registers (behind any other predicate or
// branch every operand of every product is moved there first, for each thread
// that might issue it).
__device__ __forceinline__ void pa_commit(uint64_t *bar)
{
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar))
                 : "memory");
}

__device__ __forceinline__ void pa_tma(uint32_t dst, const CUtensorMap *map, int x, int head, int row, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(head), "r"(row), "r"(smem_addr(bar))
                 : "memory");
}

// Shared-memory operand: K-major rows 128 B apart, groups of 8 rows 1024 B
// (SBO); MN-major: 64 elements a row, groups of 8 k 1024 B apart (SBO), the
// next 64 elements a box further (LBO).  Version 1, 128-byte swizzle.
__device__ __forceinline__ uint64_t pa_desc(uint32_t addr, uint32_t lbo)
{
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void pa_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xFFFFFFFF;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}

__device__ __forceinline__ void pa_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xFFFFFFFF;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}

// Waits that sleep: up to 20 us at a time inside the barrier's own wait, so
// that waiting warps leave the issue slots to the others.
__device__ __forceinline__ bool pa_try(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_addr(bar)), "r"(parity), "r"(20000u) : "memory");
    return ok != 0;
}

// False when the limit of every wait ran out, or another's has: *dead says so
// of this CTA's, *status (nullptr: not looked at) of another CTA's or
// kernel's.  It is looked at after a millisecond, a thousand times what a tile
// takes: one limit, and not one per CTA, passes before a grid ends.
__device__ __forceinline__ bool pa_wait(uint64_t *bar, uint32_t parity, int *dead, int *status = nullptr)
{
    if (pa_try(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!pa_try(bar, parity)) {
        if (*reinterpret_cast<volatile int *>(dead)) return false;
        const uint64_t dt = globaltimer_ns() - t0;
        if (dt > wait_limit_ns()) return false;
        if (status && dt > 1000000 && *reinterpret_cast<volatile int *>(status) != 0) return false;
    }
    return true;
}

#define PA_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define PA_W8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])

// 16 columns of this thread's row (its warp's 32 lanes)
__device__ __forceinline__ void pa_ld16(uint32_t (&v)[16], uint32_t addr)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : PA_R8(v, 0), PA_R8(v, 8)
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void pa_st16(uint32_t addr, const uint32_t (&v)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
                 PA_W8(v, 0), PA_W8(v, 8)
                 : "memory");
}

__device__ __forceinline__ void pa_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// the loaded values are used after the wait only
template <int N> __device__ __forceinline__ void pa_pin(uint32_t (&v)[N])
{
#pragma unroll
    for (int x = 0; x < N; x++) asm volatile("" : "+r"(v[x]));
}
__device__ __forceinline__ void pa_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t pa_pair(__half, float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pa_pair(__nv_bfloat16, float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Two fp32 values in one register pair, for the packed fp32 units.
__device__ __forceinline__ uint64_t pa_two(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void pa_untwo(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t pa_fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t pa_add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// max that a NaN survives
__device__ __forceinline__ float pa_max(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float pa_max3(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^t on the FMA units: t = n + f with |f| <= 1/2, n added to the polynomial's
// exponent.  Below -126 it is zero, as ex2's: what a row does not see has
// t = -inf, and 2^-126 times a large bf16 value would count.  So the result is
// formed 2^64 too large, with t held at -190, and the last product flushes it.
template <int DEG> __device__ __forceinline__ float pa_ex2_fma(float t)
{
    t = fmaxf(t, -190.0f);
    const float r = __fadd_rn(t, 12582976.0f);                   // 1.5 * 2^23 + 64: n + 64 in the low bits
    const float f = __fsub_rn(t, __fsub_rn(r, 12582976.0f));
    float       p;
    if (DEG == 3) {
        p = fmaf(f, 0.055171668529510498f, 0.24261112511157990f);
        p = fmaf(f, p, 0.69326096773147583f);
        p = fmaf(f, p, 0.99992805719375610f);
    } else {
        p = fmaf(f, 0.0095701021f, 0.0559178628f);
        p = fmaf(f, p, 0.2402474433f);
        p = fmaf(f, p, 0.6931217909f);
        p = fmaf(f, p, 0.9999992847f);
    }
    float y;
    asm("mul.ftz.f32 %0, %1, 0f1F800000;" : "=f"(y) : "f"(__uint_as_float(__float_as_uint(p) + (__float_as_uint(r) << 23))));
    return y;
}

// Does any of the 64 threads at barrier `id` say so?
__device__ __forceinline__ bool pa_any(int id, bool mine)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                 "barrier.cta.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((uint32_t)mine), "r"(id) : "memory");
    return any != 0;
}

template <typename T> struct PaBits;     // exponent mask of two elements, and what carries it into the sign when it is full
template <> struct PaBits<__half> { static constexpr uint32_t exp = 0x7C007C00u, one = 0x04000400u, fmt = 0; };
template <> struct PaBits<__nv_bfloat16> { static constexpr uint32_t exp = 0x7F807F80u, one = 0x00800080u, fmt = 1; };

template <typename T, int HD, int N>
__global__ void __launch_bounds__(PA_THREADS, 1)
k_attn_prompt(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
              const PromptArgs a, const PromptSeqs<N> list)
{
    using S = PaShape<HD>;
    constexpr int ST = S::STAGES, B = S::B;
    extern __shared__ uint8_t raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = sm + 2 * S::TILE;
    __shared__ __align__(8) uint64_t q_full[2], full[ST], empty[ST], s_full[2], p_full[2], due[4], clean[4], drain;
    __shared__ uint32_t              tmem_s, bad[4][4];       // keys of the partly seen tiles with cleaned elements
    __shared__ int                   any_bad, dead;
    __shared__ float                 half_s[2][2][128];       // what a row's two threads tell each other
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // this CTA's pair: the sequence, the KV head, the two items (tile, head); the
    // latest tiles, which have most keys, come first
    int lo = 0, hi = list.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (list.cta[mid] <= (int)blockIdx.x) lo = mid;
        else hi = mid;
    }
    const int nq = list.nq[lo], nk = list.nk[lo], q0 = list.q0[lo], k0 = list.k0[lo];
    const int items = (nq + 127) / 128 * a.n_rep, pairs = (items + 1) / 2;
    const int at = (int)blockIdx.x - list.cta[lo], kvh = at % a.n_kv, item = 2 * (pairs - 1 - at / a.n_kv);
    const int n_tile = min(2, items - item);
    auto tile_of = [&](int t) { return (item + t) / a.n_rep; };
    auto head_of = [&](int t) { return kvh * a.n_rep + (item + t) % a.n_rep; };
    auto seen = [&](int row) { return min(nk, max(0, row + 1 + nk - nq)); };    // keys that a row sees
    // key tiles: n in all, those below n_plain seen whole by every row; the rows
    // of a pair end at most 255 keys apart, so at most 3 are seen in part
    const int n = (seen(min(tile_of(n_tile - 1) * 128 + 128, nq) - 1) + 127) / 128;
    const int n_plain = seen(tile_of(0) * 128) / 128;

    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // one tile of K (x even) or V of key tile x / 2 into the ring's place x % ST
    auto copy_kv = [&](int x) {
        mbar_expect_tx(full + x % ST, S::TILE);
        for (int b = 0; b < B; b++)
            pa_tma(smem_addr(ring + x % ST * S::TILE + b * PA_BOX), (x & 1) ? &mv : &mk, b * 64, kvh, k0 + x / 2 * 128, full + x % ST);
        // the cleaners may look at the stage's barrier only now that it
        // counts this tile: its phase's parity would fit an earlier one too
        if ((x & 1) && x / 2 >= n_plain) mbar_arrive(due + (x / 2 - n_plain));
    };
    if (tid == 512) {                                     // the first copies are on their way before the block meets
        for (const CUtensorMap *m : {&mq, &mk, &mv}) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
        for (int s = 0; s < ST; s++) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init(q_full + t, 1);
            mbar_init(s_full + t, 1);
            mbar_init(p_full + t, 8);
        }
        for (int j = 0; j < 4; j++) {
            mbar_init(due + j, 1);
            mbar_init(clean + j, 2);
        }
        mbar_init(&drain, 1);
        mbar_init_fence();
        any_bad = dead = 0;
        pdl_wait();
        if (n > 0) {
            for (int t = 0; t < n_tile; t++) {
                mbar_expect_tx(q_full + t, S::TILE);
                for (int b = 0; b < B; b++)
                    pa_tma(smem_addr(sm + t * S::TILE + b * PA_BOX), &mq, b * 64, head_of(t), q0 + tile_of(t) * 128, q_full + t);
                if (t == 0 && !a.stall) copy_kv(0);
            }
            for (int x = 1; x < min(ST, 2 * n); x++) copy_kv(x);
        }
    }
    if (tid < 16) bad[tid >> 2][tid & 3] = 0;
    pdl_wait();
    pdl_trigger();
    pa_fence_before();
    __syncthreads();
    pa_fence_after();
    const uint32_t tmem = tmem_s;
    // every wait is bounded; one that gives up lets the others give up too, and
    // the block's end flags the status (which the softmax warps do not look at:
    // that made 8192 tokens 1.2 % slower)
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (!pa_wait(bar, parity, &dead)) atomicExch(&dead, 1);
    };
    auto watch = [&](uint64_t *bar, uint32_t parity) {
        if (!pa_wait(bar, parity, &dead, a.status)) atomicExch(&dead, 1);
    };
    auto gone = [&] { return *reinterpret_cast<volatile int *>(&dead) != 0; };

    if (warp == 16) {
        if (lane == 0) {
            int x = min(ST, 2 * n);
            for (; x < 2 * n; x++) {
                watch(empty + x % ST, (uint32_t)(x / ST - 1) & 1u);
                if (gone()) break;
                copy_kv(x);
            }
            // nothing may still be on its way into shared memory when the block
            // ends, whoever has given up by then or does so later
            bool landed = true;
            for (int t = 0; t < n_tile && n > 0; t++) landed &= mbar_drain(q_full + t, 0, wait_limit_ns());
            for (int y = max(a.stall, x - ST); y < x; y++) landed &= mbar_drain(full + y % ST, (uint32_t)(y / ST) & 1u, wait_limit_ns());
            if (!landed) atomicExch(&dead, 1);
        }
        __syncwarp();
    } else if (warp == 17) {
        if (n > 0) {
            // fp32 sums, M = 128; S: N = 128 keys; O: N = HD dimensions, V MN-major
            const uint32_t ids = (1u << 4) | (PaBits<T>::fmt << 7) | (PaBits<T>::fmt << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
            const uint32_t ido = (1u << 4) | (PaBits<T>::fmt << 7) | (PaBits<T>::fmt << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((128u >> 4) << 24);
            const uint64_t qd = pa_desc(smem_addr(sm), 16), kd = pa_desc(smem_addr(ring), 16), vd = pa_desc(smem_addr(ring), PA_BOX);
            auto qk = [&](int t, int s) {
                const uint64_t q = qd + (uint64_t)(t * (S::TILE >> 4)), k = kd + (uint64_t)(s * (S::TILE >> 4));
#pragma unroll
                for (int x = 0; x < HD / 16; x++) {
                    const uint64_t off = (uint64_t)(((x / 4) * PA_BOX + (x % 4) * 32) >> 4);
                    pa_mma_ss(tmem + 128 * t, q + off, k + off, ids, x > 0);
                }
            };
            auto pv = [&](int t, int s, bool more) {
                const uint64_t v = vd + (uint64_t)(s * (S::TILE >> 4));
#pragma unroll
                for (int x = 0; x < 8; x++)
                    pa_mma_ts(tmem + 256 + HD * t, tmem + 128 * t + 64 * (x / 4) + 8 * (x % 4), v + (uint64_t)(x * 2048 >> 4), ido, more || x > 0);
            };
            // (all lanes wait, and are together again for what follows)
            auto until = [&](uint64_t *bar, uint32_t parity) {
                watch(bar, parity);
                __syncwarp();
            };
            until(full + 0, 0);
            for (int t = 0; t < n_tile; t++) {
                until(q_full + t, 0);
                pa_fence_after();
                qk(t, 0);
                pa_commit(s_full + t);
            }
            pa_commit(empty + 0);
            for (int j = 0; j < n; j++) {
                const int iv = 2 * j + 1, sv = iv % ST, ik = iv + 1, sk = ik % ST;
                until(full + sv, (uint32_t)(iv / ST) & 1u);
                if (j >= n_plain) until(clean + (j - n_plain), 0);
                for (int t = 0; t < n_tile; t++) {
                    until(p_full + t, (uint32_t)j & 1u);
                    if (__any_sync(0xffffffffu, gone())) break;
                    pa_fence_after();
                    pv(t, sv, j > 0);
                    if (t + 1 == n_tile) pa_commit(empty + sv);
                    if (j + 1 < n) {
                        if (t == 0) until(full + sk, (uint32_t)(ik / ST) & 1u);
                        qk(t, sk);
                        if (t + 1 == n_tile) pa_commit(empty + sk);
                    }
                    pa_commit(s_full + t);    // the next scores, or at the end the sums, and all before
                }
                if (__any_sync(0xffffffffu, gone())) break;
            }
            pa_commit(&drain);
            // no product in flight when tensor memory is given back
            if (!mbar_drain(&drain, 0, wait_limit_ns())) atomicExch(&dead, 1);
        }
        __syncwarp();
    } else if (warp >= 18) {
        const int me = tid - 576;
        for (int j = n_plain; j < n; j++) {
            const int iv = 2 * j + 1;
            wait(due + (j - n_plain), 0);
            wait(full + iv % ST, (uint32_t)(iv / ST) & 1u);
            if (__any_sync(0xffffffffu, gone())) break;
            uint4 *v = reinterpret_cast<uint4 *>(ring + (iv % ST) * S::TILE);
            for (int i = me; i < S::TILE / 16; i += 64) {
                uint4     x = v[i];
                uint32_t *w = reinterpret_cast<uint32_t *>(&x);
                uint32_t  full_exp = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) full_exp |= (w[e] & PaBits<T>::exp) + PaBits<T>::one;
                if (full_exp & 0x80008000u) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t f = (w[e] & PaBits<T>::exp) + PaBits<T>::one;
                        w[e] &= (f & 0x8000u ? 0u : 0xFFFFu) | (f & 0x80000000u ? 0u : 0xFFFF0000u);
                    }
                    v[i] = x;
                    const int key = (i % (PA_BOX / 16)) / 8;
                    atomicOr(&bad[j - n_plain][key >> 5], 1u << (key & 31));
                    any_bad = 1;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(clean + (j - n_plain));
        }
    } else {
        // Nothing here leaves the loop early, whatever gave up: the two warps of
        // 32 rows meet at their barrier in every turn.
        const int      t = warp >> 3, hf = (warp >> 2) & 1, r = (warp & 3) * 32 + lane, pair = 1 + 4 * t + (warp & 3);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + lanes + 128 * t, to = tmem + lanes + 256 + HD * t;
        if (t < n_tile) {
            const int   row = tile_of(t) * 128 + r, vis = seen(row);
            const float sl = a.scale * 1.4426950408889634f;
            float       m = -INFINITY, l = 0.0f;          // the maximum that P is relative to; this half's weights' sum
            for (int j = 0; j < n; j++) {
                wait(s_full + t, (uint32_t)j & 1u);
                pa_fence_after();
                uint32_t s[4][16];
#pragma unroll
                for (int c = 0; c < 4; c++) pa_ld16(s[c], ts + 64 * hf + 16 * c);
                pa_ld_wait();
#pragma unroll
                for (int c = 0; c < 4; c++) pa_pin(s[c]);
                if (j >= n_plain) {
                    const int left = vis - j * 128 - 64 * hf;
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int x = 0; x < 16; x++)
                            if (16 * c + x >= left) s[c][x] = 0xFF800000u;
                }
                float top[4];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    auto v = [&](int x) { return __uint_as_float(s[q][x]); };
                    top[q] = pa_max3(v(0), v(1), v(2));
#pragma unroll
                    for (int x = 3; x < 15; x += 2) top[q] = pa_max3(top[q], v(x), v(x + 1));
                    top[q] = pa_max(top[q], v(15));
                }
                float mx = pa_max(pa_max3(top[0], top[1], top[2]), top[3]);
                // not (mx within 2^8 of m): a NaN grows, and turns its whole row into NaN
                auto grows = [&] { return !(mx <= m) && !((mx - m) * sl <= 8.0f); };
                if (pa_any(pair, grows())) {
                    half_s[t][hf][r] = mx;
                    named_bar(pair, 64);
                    mx = pa_max(mx, half_s[t][hf ^ 1][r]);
                    const bool  grow = grows();
                    const float f = grow && j > 0 ? kv4_ex2((m - mx) * sl) : 1.0f;
                    if (grow) m = mx;
                    l *= f;
                    if (j > 0)
#pragma unroll 1
                        for (int c = 0; c < HD / 2; c += 16) {
                            uint32_t o[16];
                            pa_ld16(o, to + HD / 2 * hf + c);
                            pa_ld_wait();
                            pa_pin(o);
#pragma unroll
                            for (int x = 0; x < 16; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                            pa_st16(to + HD / 2 * hf + c, o);
                        }
                }
                // (an infinite maximum, or product with the scale, makes the row NaN in every weight)
                const float    mb = m == -INFINITY ? 0.0f : fmaf(m * sl, 0.0f, m * sl);
                const uint64_t sl2 = pa_two(sl, sl), mb2 = pa_two(-mb, -mb);
                uint64_t       sum[2] = {pa_two(0.0f, 0.0f), pa_two(0.0f, 0.0f)};
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t p[16];
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        const uint32_t *v = &s[2 * h + (x >> 3)][2 * (x & 7)];
                        const uint64_t  t2 = pa_fma2(pa_two(__uint_as_float(v[0]), __uint_as_float(v[1])), sl2, mb2);
                        float           e0, e1;
                        pa_untwo(t2, e0, e1);
                        if (x % PA_FMA == PA_FMA - 1) {
                            e0 = pa_ex2_fma<PaBits<T>::fmt ? 3 : 4>(e0);
                            e1 = pa_ex2_fma<PaBits<T>::fmt ? 3 : 4>(e1);
                        } else {
                            e0 = kv4_ex2(e0);
                            e1 = kv4_ex2(e1);
                        }
                        sum[x & 1] = pa_add2(sum[x & 1], pa_two(e0, e1));
                        p[x] = pa_pair(T(), e0, e1);
                    }
                    pa_st16(ts + 64 * hf + 16 * h, p);    // over scores that this thread alone has read
                }
                float a0, a1;
                pa_untwo(pa_add2(sum[0], sum[1]), a0, a1);
                l += a0 + a1;
                pa_st_wait();
                pa_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + t);
            }
            // the output: this thread's half of the row's dimensions
            if (n > 0) wait(s_full + t, (uint32_t)n & 1u);
            for (int j = n_plain; j < n; j++) wait(clean + (j - n_plain), 0);
            pa_fence_after();
            named_bar(pair, 64);
            half_s[t][hf][r] = l;
            named_bar(pair, 64);
            const float inv = gone() ? NAN : 1.0f / (half_s[t][0][r] + half_s[t][1][r]);
            // through the place of the tile's queries, 16-byte chunk j of row r at
            // j ^ (r & 7), so that rows leave whole: 2.5 us a pair where every
            // thread writes its own row
            uint8_t *rows_s = sm + t * S::TILE + (size_t)(warp & 3) * 32 * HD * 2;
#pragma unroll 1
            for (int c = 0; c < HD / 2; c += 16) {
                uint32_t o[16];
                if (n > 0) {
                    pa_ld16(o, to + HD / 2 * hf + c);
                    pa_ld_wait();
                    pa_pin(o);
                }
                {
                    float y[16];
#pragma unroll
                    for (int x = 0; x < 16; x++) y[x] = vis > 0 ? __uint_as_float(o[x]) * inv : 0.0f;
                    if (any_bad)                          // cleaned elements of keys that the row sees
                        for (int w = 0; w < 16; w++)
                            for (uint32_t left = bad[w >> 2][w & 3]; left; left &= left - 1) {
                                const int key = (n_plain + (w >> 2)) * 128 + (w & 3) * 32 + __ffs(left) - 1;
                                if (key >= vis) continue;
                                const T *v = (const T *)a.v + (size_t)(k0 + key) * a.v_stride + (size_t)kvh * HD + HD / 2 * hf + c;
#pragma unroll
                                for (int x = 0; x < 16; x++) {
                                    const float e = kv4_float(v[x]);
                                    if (!(fabsf(e) < INFINITY)) y[x] += e;
                                }
                            }
#pragma unroll
                    for (int x = 0; x < 16; x += 8) {
                        uint4 w;
                        w.x = pa_pair(T(), y[x], y[x + 1]);
                        w.y = pa_pair(T(), y[x + 2], y[x + 3]);
                        w.z = pa_pair(T(), y[x + 4], y[x + 5]);
                        w.w = pa_pair(T(), y[x + 6], y[x + 7]);
                        *reinterpret_cast<uint4 *>(rows_s + lane * HD * 2 + (((HD / 2 * hf + c + x) / 8 ^ (lane & 7)) * 16)) = w;
                    }
                }
            }
            named_bar(pair, 64);
            T *out = (T *)a.out + (size_t)(q0 + tile_of(t) * 128 + (warp & 3) * 32) * a.out_stride + (size_t)head_of(t) * HD;
            const int rows = nq - tile_of(t) * 128 - (warp & 3) * 32;       // of these 32
#pragma unroll
            for (int x = hf * 32 + lane; x < 32 * HD / 8; x += 64) {
                const int y = x / (HD / 8), j = x % (HD / 8);
                if (y < rows) *reinterpret_cast<uint4 *>(out + (size_t)y * a.out_stride + j * 8) = *reinterpret_cast<const uint4 *>(rows_s + y * HD * 2 + ((j ^ (y & 7)) * 16));
            }
        }
    }
    pa_fence_before();
    __syncthreads();
    if (tid == 512 && gone()) atomicOr(a.status, ECU_STATUS_TIMEOUT);
    if (warp == 17) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}
