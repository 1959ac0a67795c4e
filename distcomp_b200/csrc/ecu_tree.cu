// ecu_tree.cu -- the attention of drafted rows over the paged 4-bit cache behind
// engine_cuda.h.
#include "ecu_draft.h"
#include "ecu_tree.cuh"
#include "ecu_tree_tc.cuh"

#include <algorithm>
#include <climits>
#include <cmath>
#include <exception>

#define CK(call)                                                                        \
    do {                                                                                \
        cudaError_t e_ = (call);                                                        \
        if (e_ != cudaSuccess) {                                                        \
            cudaGetLastError();                                                         \
            ecu_set_error(nullptr, 0, "%s failed: %s", #call, cudaGetErrorString(e_)); \
            return -1;                                                                  \
        }                                                                               \
    } while (0)

static std::atomic<unsigned> g_stall{0};        // devices (bits) whose next call's waits run out
static std::atomic<unsigned> g_regs{0};         // ... whose next call finds the kernel on tensor memory compiled to other registers

// The device's bit of a mask, taken out of it.
static int injected(std::atomic<unsigned> &mask, int device)
{
    if (device >= 32 || !mask.load(std::memory_order_relaxed)) return 0;
    return (int)(mask.fetch_and(~(1u << device)) >> device & 1u);
}

// Two partials a CTA, of up to 128 columns
extern "C" size_t ecu_kv_tree_ws_bytes(const ecu_kv *kv)
{
    return kv && kv->device >= 0 ? (size_t)kv->sms * 2 * TT_COLS * (kv->head_dim + 2) * sizeof(float) : 0;
}

int ecu_draft_set_wait(unsigned long long ns) { return set_wait_limit(ns) == cudaSuccess ? 0 : -1; }

extern "C" int ecu_inject_tree_timeout(int device)
{
    if (device < 0 || device >= 32) return say("ecu_inject_tree_timeout", "no such device to stall");
    g_stall.fetch_or(1u << device);
    return 0;
}

extern "C" int ecu_inject_tree_registers(int device)
{
    if (device < 0 || device >= 32) return say("ecu_inject_tree_registers", "no such device");
    g_regs.fetch_or(1u << device);
    return 0;
}

// The pool's own workspace for a stream: by the stream's id, since handles are
// reused and the per-thread default stream's names another in each thread.
static int tree_workspace(ecu_kv *kv, cudaStream_t s, void **ws)
{
    unsigned long long id = 0;
    CK(cudaStreamGetId(s, &id));
    const size_t bytes = ecu_kv_tree_ws_bytes(kv);
    if (kv->tree_ws.size() >= KV4_STREAMS && !kv->tree_ws.count(id)) {       // streams come and go: start over
        CK(cudaDeviceSynchronize());
        for (auto &w : kv->tree_ws) {
            cudaFree(w.second);
            kv->device_bytes -= bytes;
        }
        kv->tree_ws.clear();
    }
    auto at = kv->tree_ws.find(id);
    if (at == kv->tree_ws.end()) {
        void *p = nullptr;
        CK(cudaMalloc(&p, bytes));
        try {
            at = kv->tree_ws.emplace(id, p).first;
        } catch (...) {
            cudaFree(p);
            throw;
        }
        kv->device_bytes += bytes;
    }
    *ws = at->second;
    return 0;
}

// The rows' plan over the sequences as they are: how many, how many CTAs have
// work for two units (of their groups), whether all are of one length.
struct TreeTotal { long long rows = 0, want = 0; double units = 0.0; bool even = true; };
template <int N> static TreeTotal tree_total(const ecu_kv *kv, const TreeArgs &a, const KvRows<N> &r, int group, int unit, int per_cta)
{
    TreeTotal t;
    int       last = -1;
    for (int i = 0; i < r.n; i++) {
        const TreePlan p = tree_plan(kv->book.seq[r.seq[i]].len, r.row0[i + 1] - r.row0[i], a.n_kv, a.n_rep, group, unit);
        if (!p.rows) continue;
        t.rows += p.rows;
        t.units += (double)p.rows * p.nu;
        t.want += (long long)p.rows * std::max(1, p.nu / per_cta);
        t.even = t.even && (last < 0 || last == p.nu);
        last = p.nu;
    }
    return t;
}

// How a launch cuts its rows: its CTAs, whether rows are shared and so joined,
// and how long that takes: `start`, `step` for each of a CTA's units, `row` for
// each of its rows, `join` where there is a second launch (us, measured).
struct TreeWay { int grid; bool shared, even; double us; };
static TreeWay tree_way(const TreeTotal &t, int sms, bool captured, double start, double step, double row, double join)
{
    auto us = [&](int grid, bool shared) {
        return start + std::max(1.0, t.units / grid) * step + (double)t.rows / grid * row + (shared ? join : 0.0);
    };
    // One CTA an SM; fewer where a CTA would find less than two units a group.
    // (A captured launch's sequences grow: nothing of its plan may depend on them.)
    TreeWay w;
    w.grid = captured ? sms : (int)std::max(1ll, std::min<long long>(sms, t.want));
    w.even = !captured && t.even;
    // Few rows of one length get as many CTAs each, whose parts are equal when a row's beginning takes no place.
    if (w.even && t.rows <= w.grid) w.grid -= (int)(w.grid % t.rows);
    w.shared = !w.even || t.rows % w.grid != 0;
    w.us = us(w.grid, w.shared);
    if (!w.even || !w.shared) return w;
    // Or whole rows of one length, as many a CTA, and no join.
    int whole = (int)std::min<long long>(sms, t.rows);
    while (t.rows % whole) whole--;
    const double alone = us(whole, false);
    if (alone < w.us) w = {whole, false, true, alone};
    return w;
}

// Is the kernel on tensor memory compiled to the registers that its roles share (more than the launch has would wait
// forever)?  If not, the other kernel takes its calls.
template <typename T, int HD, int N> static bool tree_tc_fits(int device)
{
    static std::atomic<int> regs{0};
    cudaFuncAttributes      f;
    if (!regs.load(std::memory_order_relaxed)) {
        if (cudaFuncGetAttributes(&f, k_kv4_tree_tc<T, HD, N>) == cudaSuccess) regs.store(f.numRegs, std::memory_order_relaxed);
        else cudaGetLastError();
    }
    return regs.load(std::memory_order_relaxed) == TT_REGS && !injected(g_regs, device);
}

template <typename T, int NB, int N, typename F>
static int tree_start(TreeArgs a, const KvRows<N> &r, const TreeWay &w, long long rows, int unit, cudaStream_t s, F launch)
{
    if (w.even && rows <= w.grid) a.open = 0;
    if (launch(a, w.grid) != 0) return -1;
    if (!w.shared) return 0;
    // Columns of a block of the join: one a warp where rows have many parts (1 sequence of 4000 positions, 128 columns a KV
    // head: 39, 47 and 57 us with 8, 16 and 32), else two (17 of 2000: 104, 102 and 108).
    const int slice = rows * 4 <= w.grid ? 8 : 16;
    return launched("ecu_kv_attend_tree", ecu_launch_early(k_kv4_tree_join<T, NB, N>, (unsigned)w.grid * ((a.group + slice - 1) / slice), 256, 0, s, a, r, unit, w.grid, slice));
}

template <typename T, int NB, int N>
static int tree_launch(ecu_kv *kv, TreeArgs a, const int *seq, int first, const int *n_new, int n, bool captured, cudaStream_t s)
{
    using S = TreeShape<T, NB>;
    KvRows<N> r;
    fill_rows(r, seq, first, n_new, n);
    if (r.row0[n] == 0) return 0;
    // Tiles of a group: the width that is estimated to take least.  (A step of the groups, 32 positions each, takes 3.0 us
    // at 128-wide heads and 1.7 at 64, a row's queries, merge and output 5 to 8.5, a join 12 to 18.  Narrow groups spread few
    // rows over more CTAs, wide ones read the cache less often: one sequence of 2000 positions with 16 drafts of 4 query
    // heads, bf16, 26, 32, 35 and 40 us with 1 to 4 tiles; 32 of 1 to 4096 positions of 8 query heads, fp32, 545, 468, 440
    // and 437.)
    const double size = S::C * S::HD / 1024.0;
    TreeWay      best{};
    long long    best_rows = 0;
    for (int wc = TREE_MAX_WC; wc >= 1; wc--) {
        const int       groups = TREE_WARPS / wc;
        const TreeTotal t = tree_total(kv, a, r, S::C * wc, KV4_UNIT, 2 * groups);
        TreeTotal       steps = t;                        // the groups take a row's units in turn
        steps.units /= groups;
        const TreeWay w = tree_way(steps, kv->sms, captured, 3.0, 0.4 + 0.65 * NB, 2.3 + 3.1 * size, 8.0 + 3.0 * size + 1.5 * wc);
        if (!best.grid || w.us < best.us) {
            best = w;
            best_rows = t.rows;
            a.wc = wc;
        }
    }
    if constexpr (sizeof(T) == 2 && NB % 2 == 0) {
        // A unit of 128 positions and up to 128 columns, however many it has, takes 1.85 us (of 64-wide heads 1.6), the first
        // and the last some 14 more.  (4 sequences of 16384 positions, 4 query heads a KV head, 32 / 64 columns: 79 against 83 /
        // 82 against 130 us, 64-wide 70 against 57 / 71 against 85.  Over 570 calls of 1 to 32 sequences of up to 4096
        // positions, these estimates take 1 to 3 % longer than the best of all choices, counts of units alone 14 to 17.)
        const TreeTotal t = tree_total(kv, a, r, TT_COLS, TT_UNIT, 1);
        const TreeWay   w = tree_way(t, kv->sms, captured, 17.0, NB == 4 ? 1.85 : 1.6, 0.0, 13.0);
        if (w.us < best.us && tree_tc_fits<T, NB * 32, N>(kv->device)) {
            a.group = a.entry = TT_COLS;
            a.open = TT_OPEN;
            auto kern = k_kv4_tree_tc<T, NB * 32, N>;
            int *status = ecu_prompt_status_word(kv->device);
            if (!status) return say("ecu_kv_attend_tree", "the status word cannot be had");
            const int stall = injected(g_stall, kv->device);
            return tree_start<T, NB>(a, r, w, t.rows, TT_UNIT, s, [&](const TreeArgs &a, int grid) {
                static std::atomic<unsigned> done{0};
                CK(ecu_allow_smem(kern, TreeTc<NB * 32>::smem(N), kv->device, done));
                return launched("ecu_kv_attend_tree", ecu_launch_early(kern, (unsigned)grid, TT_THREADS, TreeTc<NB * 32>::smem(n), s, a, r, status, stall));
            });
        }
    }
    a.group = S::C * a.wc;
    a.entry = S::EC;
    a.open = TREE_OPEN;
    auto kern = k_kv4_tree<T, NB, N>;
    return tree_start<T, NB>(a, r, best, best_rows, KV4_UNIT, s, [&](const TreeArgs &a, int grid) {
        static std::atomic<unsigned> done{0};
        CK(ecu_allow_smem(kern, S::smem(N), kv->device, done));
        return launched("ecu_kv_attend_tree", ecu_launch_early(kern, (unsigned)grid, TREE_WARPS * 32, S::smem(n), s, a, r));
    });
}

template <typename T, int NB> static int tree_list(ecu_kv *kv, TreeArgs a, const int *seq, const int *n_new, int n, bool captured, cudaStream_t s)
{
    // at most 2^31 - 1 places in a launch, however the sequences may grow
    const TreePlan  p = tree_plan(kv->book.max_pages * KV4_PAGE, TREE_ROWS, a.n_kv, a.n_rep, TreeShape<T, NB>::C, KV4_UNIT);
    const long long places = (long long)p.rows * (p.nu + std::max(TREE_OPEN, TT_OPEN));
    if (places > INT_MAX) return say("ecu_kv_attend_tree", "too many positions and heads a sequence");
    const int most = (int)std::min<long long>(KV4_LIST, INT_MAX / places);
    for (int i = 0; i < n; i += most) {
        const int  m = std::min(most, n - i);
        const int *q = seq ? seq + i : nullptr;
        if ((m <= 64 ? tree_launch<T, NB, 64>(kv, a, q, i, n_new + i, m, captured, s)
                     : tree_launch<T, NB, KV4_LIST>(kv, a, q, i, n_new + i, m, captured, s)) != 0)
            return -1;
        size_t rows = 0;
        for (int j = 0; j < m; j++) rows += n_new[i + j];
        a.q = (const T *)a.q + rows * a.q_stride;
        a.out = (T *)a.out + rows * a.out_stride;
        if (a.mask) a.mask += rows;
    }
    return 0;
}

template <typename T> static int tree_dim(ecu_kv *kv, const TreeArgs &a, const int *seq, const int *n_new, int n, bool captured, cudaStream_t s)
{
    switch (kv->head_dim / 32) {
    case 1: return tree_list<T, 1>(kv, a, seq, n_new, n, captured, s);
    case 2: return tree_list<T, 2>(kv, a, seq, n_new, n, captured, s);
    case 3: return tree_list<T, 3>(kv, a, seq, n_new, n, captured, s);
    default: return tree_list<T, 4>(kv, a, seq, n_new, n, captured, s);
    }
}

extern "C" int ecu_kv_attend_tree(ecu_kv *kv, int layer, int dtype, const void *q, void *out, int n_head, long q_stride, long out_stride,
                                  const int *seq, const int *n_new, int n, const uint64_t *mask, float scale, void *ws, void *stream)
{
    const char *what = "ecu_kv_attend_tree";
    if (!kv || n < 0 || (n > 0 && !n_new)) return say(what, "null argument or negative count");
    if (layer < 0 || layer >= kv->n_layer) {
        ecu_set_error(nullptr, 0, "%s: layer %d of %d", what, layer, kv->n_layer);
        return -1;
    }
    const size_t es = dtype_bytes(dtype);
    if (!es) return say(what, "unknown element type");
    if (n_head < 1 || n_head % kv->n_head_kv || n_head / kv->n_head_kv > 4096 || n_head > INT_MAX / kv->head_dim) {
        ecu_set_error(nullptr, 0, "%s: %d query heads for %d KV heads", what, n_head, kv->n_head_kv);
        return -1;
    }
    if (!std::isfinite(scale)) return say(what, "the scale is not finite");
    if (whole(kv, what) != 0) return -1;
    try {
        const long long rows = rows_ok(kv, seq, n_new, n, TREE_ROWS, what);
        if (rows < 0) return -1;
        if (rows == 0) return 0;
        const long row = (long)n_head * kv->head_dim;
        if (!q || !out) return say(what, "null rows");
        if (rows > 1 && (q_stride < row || out_stride < row)) return say(what, "rows overlap: a stride below n_head * head_dim");
        if (((uintptr_t)q | (uintptr_t)out) % es || ((uintptr_t)ws & 15) || ((uintptr_t)mask & 7))
            return say(what, "rows, masks or workspace are not aligned");
        if (kv->device < 0) return say(what, "the pool has no device");
        DeviceScope d(kv->device);
        if (!d.ok) return say(what, "the pool's device cannot be used");
        const cudaStream_t s = (cudaStream_t)stream;
        const int          cap = capturing(s, what);
        if (cap < 0) return -1;
        if (!ws) {
            if (cap) return say(what, "a captured call needs a workspace of its own");
            if (tree_workspace(kv, s, &ws) != 0) return -1;
        }
        TreeArgs a = {};
        a.q = q;
        a.out = out;
        a.q_stride = q_stride;
        a.out_stride = out_stride;
        a.layer = kv->data + (size_t)layer * kv->book.n_pages * kv->page_bytes;
        a.page_bytes = kv->page_bytes;
        a.table = kv->table();
        a.len = kv->len();
        a.mask = (const long long *)mask;
        a.max_pages = kv->book.max_pages;
        a.n_pages = kv->book.n_pages;
        a.n_kv = kv->n_head_kv;
        a.n_rep = n_head / kv->n_head_kv;
        a.scale = scale;
        a.wide_q = !(((uintptr_t)q | (uintptr_t)(q_stride * (long)es)) & 15);
        a.wide_out = !(((uintptr_t)out | (uintptr_t)(out_stride * (long)es)) & 15);
        a.part = (float *)ws;
        if (dtype == ECU_F16) return tree_dim<__half>(kv, a, seq, n_new, n, cap, s);
        if (dtype == ECU_BF16) return tree_dim<__nv_bfloat16>(kv, a, seq, n_new, n, cap, s);
        return tree_dim<float>(kv, a, seq, n_new, n, cap, s);
    } catch (const std::exception &e) {
        return say(what, e.what());
    }
}
