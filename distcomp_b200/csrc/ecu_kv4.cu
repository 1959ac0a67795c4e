// ecu_kv4.cu -- the paged 4-bit K/V cache behind engine_cuda.h: the pool,
// the rows written into it and the attention that reads it.
#include "ecu_kv4.cuh"
#include "ecu_kv4.h"
#include "ecu_model.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <exception>
#include <memory>
#include <optional>

#define CK(call)                                                                        \
    do {                                                                                \
        cudaError_t e_ = (call);                                                        \
        if (e_ != cudaSuccess) {                                                        \
            cudaGetLastError();                                                         \
            ecu_set_error(nullptr, 0, "%s failed: %s", #call, cudaGetErrorString(e_)); \
            return -1;                                                                  \
        }                                                                               \
    } while (0)


// The driver takes a thread's default stream down when the thread ends.  Where
// work was under way on it then, that thread's end and the process's next calls
// have waited for one another for good, the GPU idle (five runs in five of
// test_attend_keeps_a_workspace_a_stream behind the tests before it; none in
// eleven with the wait here, which comes before the driver's own part).
namespace {
struct ThreadEnd {
    unsigned long long devices = 0;
    ~ThreadEnd()
    {
        for (int d = 0; d < 64; d++)
            if (devices >> d & 1u && cudaSetDevice(d) == cudaSuccess) cudaStreamSynchronize(cudaStreamPerThread);
    }
};
}
void ecu_on_thread_stream()
{
    static thread_local ThreadEnd end;
    int                           d = 0;
    if (cudaGetDevice(&d) == cudaSuccess && d < 64) end.devices |= 1ull << d;
}

static bool shape_ok(int n_head_kv, int head_dim)
{
    return n_head_kv > 0 && n_head_kv <= 4096 && (head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128);
}

// ------------------------------------------------------------------ pool ---

template <int N> static int update_launch(ecu_kv *kv, size_t &c0, size_t &s0, cudaStream_t s)
{
    KvUpdate<N> u;
    const auto &B = kv->book;
    u.n_copy = (int)std::min<size_t>(N, B.copies.size() - c0);
    for (int i = 0; i < u.n_copy; i++) {
        u.a[i] = B.copies[c0 + i].from;
        u.b[i] = B.copies[c0 + i].to;
    }
    u.n_set = (int)std::min<size_t>(N - u.n_copy, B.sets.size() - s0);
    for (int i = 0; i < u.n_set; i++) {
        u.a[u.n_copy + i] = B.sets[s0 + i].at;
        u.b[u.n_copy + i] = B.sets[s0 + i].value;
    }
    c0 += u.n_copy;
    s0 += u.n_set;
    if (kv->device < 0) return 0;
    const int      blocks_page = (int)((kv->page_bytes / 16 + 256 * KV4_COPY_VECS - 1) / (256 * KV4_COPY_VECS));
    const unsigned copy_blocks = (unsigned)u.n_copy * kv->n_layer * blocks_page;
    return launched("ecu_kv", ecu_launch_early(k_kv4_update<N>, copy_blocks + (u.n_set + 255) / 256, 256, 0, s, kv->data, kv->page_bytes,
                                               kv->page_bytes * B.n_pages, kv->n_layer, blocks_page, copy_blocks, kv->meta, u));
}

// What the last operation changed, on the device.  The lists travel as kernel
// arguments: 128 entries in a 1 KB argument, longer ones 2000 at a time.  A
// launch that fails takes the operation back where it is the first; where it
// is not, the device's tables are neither the old nor the new ones, and the
// pool refuses what comes after.
static int update(ecu_kv *kv, cudaStream_t s)
{
    size_t c0 = 0, s0 = 0;
    const size_t nc = kv->book.copies.size(), ns = kv->book.sets.size();
    const int    fail_at = kv->inject;
    kv->inject = -1;
    for (int i = 0; c0 < nc || s0 < ns; i++) {
        const int rc = i == fail_at ? say("ecu_kv", "launch failed: injected")
                                    : nc - c0 + ns - s0 <= 128 ? update_launch<128>(kv, c0, s0, s) : update_launch<2000>(kv, c0, s0, s);
        if (rc == 0) continue;
        if (i == 0) kv->book.fail();
        else kv->broken = true;
        return -1;
    }
    return 0;
}

// The checks that every change of the pool begins with.
static int change_ok(ecu_kv *kv, const void *list, const void *list2, int n, cudaStream_t s, const char *what)
{
    if (!kv || n < 0 || (n > 0 && (!list || !list2))) return say(what, "null argument or negative count");
    if (whole(kv, what) != 0) return -1;
    if (kv->device < 0) return 0;
    // a launch that failed later would leave the bookkeeping ahead of the device
    DeviceScope d(kv->device);
    if (!d.ok) return say(what, "the pool's device cannot be used");
    const int c = capturing(s, what);
    if (c > 0) return say(what, "the pool's bookkeeping cannot be captured");
    int dev = -1;
    if (c == 0 && (cudaStreamGetDevice(s, &dev) != cudaSuccess || dev != kv->device)) {
        cudaGetLastError();
        return say(what, "the stream is not one of the pool's device");
    }
    return c;
}

extern "C" {

size_t ecu_kv4_page_bytes(int n_head_kv, int head_dim)
{
    return shape_ok(n_head_kv, head_dim) ? (size_t)72 * head_dim * n_head_kv : 0;
}

void ecu_kv_close(ecu_kv *kv)
{
    if (!kv) return;
    if (kv->device >= 0) {
        DeviceScope d(kv->device);
        for (auto &w : kv->ws) cudaFree(w.second);
        for (auto &w : kv->tree_ws) cudaFree(w.second);
        if (kv->spare) cudaFree(kv->spare);
        if (kv->meta) cudaFree(kv->meta);
        if (kv->own_data && kv->data) cudaFree(kv->data);
    }
    delete kv;
}

int ecu_kv_open(ecu_kv **out, int n_layer, int n_head_kv, int head_dim, int n_pages, int n_seq, int max_pages, int device,
                void *data, char *err, size_t errlen)
{
    if (err && errlen) err[0] = '\0';
    if (!out) { ecu_set_error(err, errlen, "null argument"); return -1; }
    *out = nullptr;
    if (!shape_ok(n_head_kv, head_dim)) {
        ecu_set_error(err, errlen, "a 4-bit cache of %d KV heads of %d dimensions is not built (32, 64, 96 or 128)", n_head_kv,
                      head_dim);
        return -1;
    }
    if (n_layer < 1 || n_layer > 65535 || n_pages < 1 || n_seq < 1 || n_seq > 65535 || max_pages < 1 ||
        max_pages > INT_MAX / (2 * ECU_KV4_PAGE) || (long long)n_seq * (max_pages + 1) > INT_MAX) {
        ecu_set_error(err, errlen, "a pool of %d layers, %d pages, %d sequences of %d pages", n_layer, n_pages, n_seq, max_pages);
        return -1;
    }
    size_t bytes = 0;
    if (__builtin_mul_overflow(ecu_kv4_page_bytes(n_head_kv, head_dim), (size_t)n_pages * n_layer, &bytes)) {
        ecu_set_error(err, errlen, "a pool of %d layers of %d pages is too large", n_layer, n_pages);
        return -1;
    }
    if (data && ((uintptr_t)data & 15)) { ecu_set_error(err, errlen, "the pages' memory is not 16-byte aligned"); return -1; }
    try {
        std::unique_ptr<ecu_kv, void (*)(ecu_kv *)> kv(new ecu_kv(), ecu_kv_close);
        kv->n_layer = n_layer;
        kv->n_head_kv = n_head_kv;
        kv->head_dim = head_dim;
        kv->page_bytes = ecu_kv4_page_bytes(n_head_kv, head_dim);
        kv->book.init(n_pages, n_seq, max_pages);
        if (device != -1) {
            int ndev = 0;
            if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) {
                cudaGetLastError();
                ecu_set_error(err, errlen, "CUDA device %d not available (%d devices)", device, ndev);
                return -1;
            }
            DeviceScope d(device);
            if (!d.ok) { ecu_set_error(err, errlen, "cudaSetDevice(%d) failed", device); return -1; }
            kv->device = device;
            cudaDeviceGetAttribute(&kv->sms, cudaDevAttrMultiProcessorCount, device);
            kv->sms = std::min(kv->sms, KV4_MAX_CTAS);
            const size_t words = (size_t)n_seq * max_pages + n_seq;
            void *p = nullptr;
            if (cudaMalloc(&p, words * sizeof(int)) == cudaSuccess) {
                kv->meta = (int *)p;
                kv->data = (uint8_t *)data;
                if (!data && cudaMalloc(&p, bytes) == cudaSuccess) {
                    kv->data = (uint8_t *)p;
                    kv->own_data = true;
                }
            }
            if (cudaMalloc(&p, ecu_kv_ws_bytes(kv.get())) == cudaSuccess) kv->spare = p;
            if (!kv->meta || !kv->data || !kv->spare) {
                cudaGetLastError();
                ecu_set_error(err, errlen, "out of device memory for a pool of %zu bytes", bytes);
                return -1;
            }
            kv->device_bytes = words * sizeof(int) + (data ? 0 : bytes) + ecu_kv_ws_bytes(kv.get());
            cudaMemset(kv->spare, 0, ecu_kv_ws_bytes(kv.get()));
            // -1 in the table, 0 in the lengths
            cudaMemset(kv->meta, 0xFF, (size_t)n_seq * max_pages * sizeof(int));
            cudaMemset(kv->len(), 0, (size_t)n_seq * sizeof(int));
            if (kv->own_data) cudaMemset(kv->data, 0, bytes);
            if (cudaDeviceSynchronize() != cudaSuccess) {
                ecu_set_error(err, errlen, "clearing the pool failed: %s", cudaGetErrorString(cudaGetLastError()));
                return -1;
            }
        }
        *out = kv.release();
        return 0;
    } catch (const std::exception &e) {
        ecu_set_error(err, errlen, "out of memory for the pool's bookkeeping (%s)", e.what());
        return -1;
    }
}

int ecu_kv_get_info(const ecu_kv *kv, ecu_kv_info *i)
{
    if (!kv || !i) return -1;
    *i = {kv->n_layer, kv->n_head_kv, kv->head_dim, kv->book.n_pages, kv->book.n_seq, kv->book.max_pages, kv->device,
          kv->book.used, kv->page_bytes, kv->device_bytes, kv->data, kv->table(), kv->len()};
    return 0;
}

int ecu_kv_len(const ecu_kv *kv, int seq, int *pages, int n)
{
    if (!kv || slots_ok(kv, &seq, 1, "ecu_kv_len") != 0) return -1;
    const auto &q = kv->book.seq[seq];
    for (int i = 0; pages && i < n && i < (int)q.page.size(); i++) pages[i] = q.page[i];
    return q.len;
}

#define KV_CHANGE(name_, list, list2, op)                                                            \
    if (change_ok(kv, list, list2, n, (cudaStream_t)stream, name_) != 0) return -1;                  \
    try {                                                                                           \
        std::optional<DeviceScope> d;                                                               \
        if (kv->device >= 0) d.emplace(kv->device);                                                 \
        if (d && !d->ok) return say(name_, "the pool's device cannot be used");                      \
        const int r = (op);                                                                         \
        return r < 0 ? r : update(kv, (cudaStream_t)stream) != 0 ? -1 : r;                           \
    } catch (const std::exception &e) {                                                             \
        kv->book.fail();                                                                            \
        return say(name_, e.what());                                                                 \
    }

int ecu_kv_extend(ecu_kv *kv, const int *seq, const int *n_new, int n, void *stream)
{
    KV_CHANGE("ecu_kv_extend", seq, n_new, kv->book.extend(seq, n_new, n))
}

int ecu_kv_fork(ecu_kv *kv, const int *src, const int *dst, int n, void *stream)
{
    KV_CHANGE("ecu_kv_fork", src, dst, kv->book.fork(src, dst, n))
}

int ecu_kv_truncate(ecu_kv *kv, const int *seq, const int *len, int n, void *stream)
{
    KV_CHANGE("ecu_kv_truncate", seq, len, kv->book.truncate(seq, len, n))
}

int ecu_kv_free(ecu_kv *kv, const int *seq, int n, void *stream)
{
    KV_CHANGE("ecu_kv_free", seq, seq, kv->book.truncate(seq, nullptr, n))
}

int ecu_kv_compact(ecu_kv *kv, void *stream)
{
    const int n = 0;
    KV_CHANGE("ecu_kv_compact", nullptr, nullptr, kv->book.compact())
}

} // extern "C"

struct KvMove { int from, to; uint16_t at; };

// What is left of the moves and of the last operation's device words, as much
// as a launch carries: a sequence's moves that do not fit go on in the next.
template <int N>
static int keep_launch(ecu_kv *kv, const std::vector<KvMove> &moves, const std::vector<int> &first, size_t &i, size_t &j, size_t &w, cudaStream_t s)
{
    KvMoves<N> m;
    m.n = m.n_set = 0;
    m.first[0] = 0;
    int k = 0;
    while (k < N && j < moves.size()) {
        const int take = std::min<int>(N - k, first[i + 1] - (int)j);
        for (int x = 0; x < take; x++, k++, j++) {
            m.from[k] = moves[j].from;
            m.to[k] = moves[j].to;
            m.at[k] = moves[j].at;
        }
        m.first[++m.n] = k;
        if ((int)j == first[i + 1]) i++;
    }
    for (; m.n_set < 2 * N && w < kv->book.sets.size(); m.n_set++, w++) {
        m.word[m.n_set] = kv->book.sets[w].at;
        m.value[m.n_set] = kv->book.sets[w].value;
    }
    if (kv->device < 0) return 0;
    const long long blocks = (long long)m.n * kv->n_layer + (m.n_set + 255) / 256;
    return launched("ecu_kv_keep", ecu_launch_early(k_kv4_move<N>, (unsigned)blocks, 256, 0, s, kv->data, kv->page_bytes,
                                                    kv->page_bytes * kv->book.n_pages, kv->n_layer, kv->n_head_kv, kv->head_dim / 32, kv->meta, m));
}

extern "C" int ecu_kv_keep(ecu_kv *kv, const int *seq, const int *n_new, const int *kept, const int *n_kept, int n, void *stream)
{
    const char *what = "ecu_kv_keep";
    if (change_ok(kv, seq, n_new, n, (cudaStream_t)stream, what) != 0) return -1;
    if (n > 0 && !n_kept) return say(what, "null argument or negative count");
    if (slots_ok(kv, seq, n, what) != 0) return -1;
    bool changing = false;
    try {
        std::vector<bool>   seen((size_t)kv->book.n_seq, false);
        std::vector<KvMove> moves;
        std::vector<int>    first{0}, len;
        for (int i = 0; i < n; i++) {
            const auto &q = kv->book.seq[seq[i]];
            if (seen[seq[i]]) {
                ecu_set_error(nullptr, 0, "%s: sequence %d comes twice", what, seq[i]);
                return -1;
            }
            seen[seq[i]] = true;
            if (n_new[i] < 0 || n_new[i] > q.len || n_kept[i] < 0 || n_kept[i] > n_new[i] || (n_kept[i] > 0 && !kept)) {
                ecu_set_error(nullptr, 0, "%s: %d rows of %d new ones of sequence %d of %d positions", what, n_kept[i], n_new[i], seq[i], q.len);
                return -1;
            }
            const int base = q.len - n_new[i];
            for (int t = 0; t < n_kept[i]; t++, kept++) {
                if (*kept < t || *kept >= n_new[i] || (t > 0 && *kept <= kept[-1])) {
                    ecu_set_error(nullptr, 0, "%s: the kept rows of sequence %d are not rising numbers below %d", what, seq[i], n_new[i]);
                    return -1;
                }
                if (*kept == t) continue;
                const int a = base + *kept, b = base + t, to = q.page[b / ECU_KV4_PAGE];
                if (kv->book.ref[to] > 1) {
                    ecu_set_error(nullptr, 0, "%s: positions of sequence %d lie in a page that other sequences hold", what, seq[i]);
                    return -1;
                }
                moves.push_back({q.page[a / ECU_KV4_PAGE], to, (uint16_t)(a % ECU_KV4_PAGE | b % ECU_KV4_PAGE << 8)});
            }
            if ((int)moves.size() > first.back()) first.push_back((int)moves.size());
            len.push_back(base + n_kept[i]);
        }
        std::optional<DeviceScope> d;
        if (kv->device >= 0) d.emplace(kv->device);
        if (d && !d->ok) return say(what, "the pool's device cannot be used");
        // (The moves name their pages themselves, and those given back are taken
        // only by later calls.)
        changing = true;
        if (kv->book.truncate(seq, len.data(), n) != 0) return -1;
        changing = false;
        const int fail_at = kv->inject;
        kv->inject = -1;
        size_t i = 0, j = 0, w = 0;
        for (int k = 0; j < moves.size() || w < kv->book.sets.size(); k++) {
            const bool small = moves.size() - j <= 64 && kv->book.sets.size() - w <= 128;
            const int  rc = k == fail_at ? say(what, "launch failed: injected")
                            : small      ? keep_launch<64>(kv, moves, first, i, j, w, (cudaStream_t)stream)
                                         : keep_launch<512>(kv, moves, first, i, j, w, (cudaStream_t)stream);
            if (rc == 0) continue;
            if (k == 0) kv->book.fail();
            else kv->broken = true;
            return -1;
        }
        return 0;
    } catch (const std::exception &e) {
        if (changing) kv->book.fail();
        return say(what, e.what());
    }
}

extern "C" {

int ecu_kv_inject_failure(ecu_kv *kv, int launch)
{
    if (!kv || launch < 0) return say("ecu_kv_inject_failure", "null argument or negative number");
    kv->inject = launch;
    return 0;
}

} // extern "C"

// ---------------------------------------------------------------- append ---

template <typename T, typename O, int N>
static int append_launch(ecu_kv *kv, const KvAppendArgs &a, const int *seq, int first, const int *n_new, int n, cudaStream_t s)
{
    KvRows<N> r;
    r.n = n;
    r.row0[0] = 0;
    for (int i = 0; i < n; i++) {
        r.seq[i] = (uint16_t)(seq ? seq[i] : first + i);
        r.row0[i + 1] = r.row0[i] + n_new[i];
    }
    const long long threads = (long long)r.row0[n] * a.n_kv * a.nb * 4;
    if (threads == 0) return 0;
    return launched("ecu_kv_append", ecu_launch_early(k_kv4_append<T, O, N>, (unsigned)((threads + 255) / 256), 256, 0, s, a, r));
}

template <typename T, typename O>
static int append_list(ecu_kv *kv, KvAppendArgs a, const int *seq, const int *n_new, int n, cudaStream_t s)
{
    const size_t row = (size_t)kv->n_head_kv * kv->head_dim;
    for (int i = 0; i < n; i += KV4_LIST) {
        const int  m = std::min(KV4_LIST, n - i);
        const int *q = seq ? seq + i : nullptr;
        if ((m <= 64 ? append_launch<T, O, 64>(kv, a, q, i, n_new + i, m, s)
                     : append_launch<T, O, KV4_LIST>(kv, a, q, i, n_new + i, m, s)) != 0)
            return -1;
        size_t rows = 0;
        for (int j = 0; j < m; j++) rows += n_new[i + j];
        a.k = (const T *)a.k + rows * a.k_stride;
        a.v = (const T *)a.v + rows * a.v_stride;
        if (a.k_out) {
            a.k_out = (O *)a.k_out + rows * row;
            a.v_out = (O *)a.v_out + rows * row;
        }
    }
    return 0;
}

template <typename T>
static int append_out(ecu_kv *kv, const KvAppendArgs &a, int out_dtype, const int *seq, const int *n_new, int n, cudaStream_t s)
{
    if (out_dtype == ECU_F32) return append_list<T, float>(kv, a, seq, n_new, n, s);
    if (out_dtype == ECU_F16) return append_list<T, __half>(kv, a, seq, n_new, n, s);
    return append_list<T, __nv_bfloat16>(kv, a, seq, n_new, n, s);
}

extern "C" int ecu_kv_append(ecu_kv *kv, int layer, int dtype, const void *k, const void *v, long k_stride, long v_stride,
                             const int *seq, const int *n_new, int n, int out_dtype, void *k_out, void *v_out, void *stream)
{
    const char *what = "ecu_kv_append";
    if (!kv || n < 0 || (n > 0 && !n_new)) return say(what, "null argument or negative count");
    if (layer < 0 || layer >= kv->n_layer) {
        ecu_set_error(nullptr, 0, "%s: layer %d of %d", what, layer, kv->n_layer);
        return -1;
    }
    const size_t es = dtype_bytes(dtype), os = dtype_bytes(out_dtype);
    if (!es || !os) return say(what, "unknown element type");
    if (whole(kv, what) != 0) return -1;
    if (slots_ok(kv, seq, n, what) != 0) return -1;
    const long row = (long)kv->n_head_kv * kv->head_dim;
    try {
        long long         rows = 0;
        std::vector<bool> seen((size_t)kv->book.n_seq, false);
        for (int i = 0; i < n; i++) {
            const int   s = seq ? seq[i] : i;
            const auto &q = kv->book.seq[s];
            if (seen[s]) {
                ecu_set_error(nullptr, 0, "%s: sequence %d comes twice", what, s);
                return -1;
            }
            seen[s] = true;
            if (n_new[i] < 0 || n_new[i] > q.len) {
                ecu_set_error(nullptr, 0, "%s: %d rows for sequence %d of %d positions", what, n_new[i], s, q.len);
                return -1;
            }
            for (int j = (q.len - n_new[i]) / ECU_KV4_PAGE; n_new[i] > 0 && j < (int)q.page.size(); j++)
                if (kv->book.ref[q.page[j]] > 1) {
                    ecu_set_error(nullptr, 0, "%s: positions of sequence %d lie in a page that other sequences hold", what, s);
                    return -1;
                }
            rows += n_new[i];
        }
        if (rows == 0) return 0;
        if (rows > INT_MAX / (row / 8)) return say(what, "too many rows");            // a thread for eight values
        if (!k || !v || (!k_out) != (!v_out)) return say(what, "null rows, or one of k_out and v_out alone");
        if (rows > 1 && (k_stride < row || v_stride < row)) return say(what, "rows overlap: a stride below n_head_kv * head_dim");
        if (((uintptr_t)k | (uintptr_t)v) % es || (k_out && ((uintptr_t)k_out | (uintptr_t)v_out) % os))
            return say(what, "rows are not aligned to their elements");
        if (kv->device < 0) return say(what, "the pool has no device");
        DeviceScope d(kv->device);
        if (!d.ok) return say(what, "the pool's device cannot be used");
        KvAppendArgs a;
        a.k = k;
        a.v = v;
        a.k_stride = k_stride;
        a.v_stride = v_stride;
        a.k_out = k_out;
        a.v_out = v_out;
        a.layer = kv->data + (size_t)layer * kv->book.n_pages * kv->page_bytes;
        a.page_bytes = kv->page_bytes;
        a.table = kv->table();
        a.len = kv->len();
        a.max_pages = kv->book.max_pages;
        a.n_pages = kv->book.n_pages;
        a.n_kv = kv->n_head_kv;
        a.nb = kv->head_dim / 32;
        a.nb_inv = (65536 + a.nb - 1) / a.nb;             // exact below 32768: at most 4096 heads of 4 blocks
        a.wide = !(((uintptr_t)k | (uintptr_t)v | (uintptr_t)(k_stride * (long)es) | (uintptr_t)(v_stride * (long)es)) & 15);
        a.wide_out = !(((uintptr_t)k_out | (uintptr_t)v_out) & 15);
        const cudaStream_t s = (cudaStream_t)stream;
        if (dtype == ECU_F32) return append_out<float>(kv, a, out_dtype, seq, n_new, n, s);
        if (dtype == ECU_F16) return append_out<__half>(kv, a, out_dtype, seq, n_new, n, s);
        return append_out<__nv_bfloat16>(kv, a, out_dtype, seq, n_new, n, s);
    } catch (const std::exception &e) {
        return say(what, e.what());
    }
}

extern "C" int ecu_kv_read(ecu_kv *kv, int layer, int seq, int pos, int n, float *k, float *v, void *stream)
{
    const char *what = "ecu_kv_read";
    if (!kv) return say(what, "null argument");
    if (layer < 0 || layer >= kv->n_layer || slots_ok(kv, &seq, 1, what) != 0 || pos < 0 || n < 0 ||
        (long long)pos + n > kv->book.seq[seq].len)
        return say(what, "no such layer, sequence or positions");
    if (whole(kv, what) != 0) return -1;
    if (kv->device < 0) return say(what, "the pool has no device");
    if (n == 0) return 0;
    const cudaStream_t s = (cudaStream_t)stream;
    const int          c = capturing(s, what);
    if (c) return c < 0 ? -1 : say(what, "a host copy cannot be captured");
    DeviceScope d(kv->device);
    if (!d.ok) return say(what, "the pool's device cannot be used");
    const size_t   count = (size_t)n * kv->n_head_kv * kv->head_dim;
    const uint8_t *lay = kv->data + (size_t)layer * kv->book.n_pages * kv->page_bytes;
    float         *buf = nullptr;
    CK(cudaMallocAsync((void **)&buf, count * sizeof(float), s));
    int rc = 0;
    for (int side = 0; side < 2 && rc == 0; side++) {
        float *host = side ? v : k;
        if (!host) continue;
        k_kv4_read<float><<<(unsigned)((count / 8 + 255) / 256), 256, 0, s>>>(
            lay, kv->page_bytes, kv->table() + (size_t)seq * kv->book.max_pages, pos, n, kv->n_head_kv, kv->head_dim / 32,
            kv->book.n_pages, side, buf);
        rc = launched(what, cudaGetLastError());
        if (rc == 0 && (cudaMemcpyAsync(host, buf, count * sizeof(float), cudaMemcpyDeviceToHost, s) != cudaSuccess ||
                        cudaStreamSynchronize(s) != cudaSuccess)) {
            ecu_set_error(nullptr, 0, "%s: %s", what, cudaGetErrorString(cudaGetLastError()));
            rc = -1;
        }
    }
    cudaFreeAsync(buf, s);
    return rc;
}

int ecu_kv_rows(ecu_kv *kv, int layer, int seq, int n, void *k, void *v, cudaStream_t s)
{
    const size_t   vecs = (size_t)n * kv->n_head_kv * kv->head_dim / 8;
    const uint8_t *lay = kv->data + (size_t)layer * kv->book.n_pages * kv->page_bytes;
    for (int side = 0; side < 2; side++) {
        k_kv4_read<__half><<<(unsigned)((vecs + 255) / 256), 256, 0, s>>>(
            lay, kv->page_bytes, kv->table() + (size_t)seq * kv->book.max_pages, 0, n, kv->n_head_kv, kv->head_dim / 32,
            kv->book.n_pages, side, (__half *)(side ? v : k));
        if (launched("ecu_kv_rows", cudaGetLastError()) != 0) return -1;
    }
    return 0;
}

// ---------------------------------------------------------------- attend ---

// Heads of a group: one 8-column tile, two where an fp32 query has more than
// 4 heads on its KV head (two groups would read the cache twice).
static int attend_tiles(int dtype, int n_rep) { return dtype == ECU_F32 && n_rep > 4 ? 2 : 1; }

template <typename T, int NB, int NT, int N>
static int attend_launch(ecu_kv *kv, const KvAttendArgs &a, const int *seq, int first, int n, bool whole, cudaStream_t s)
{
    using S = KvShape<T, NB, NT>;
    KvSeqs<N> list;
    list.n = n;
    const long long rows_seq = (long long)kv->n_head_kv * ((a.n_rep + S::HG - 1) / S::HG);
    long long       units = 0, rows = 0;
    for (int i = 0; i < n; i++) {
        list.seq[i] = (uint16_t)(seq ? seq[i] : first + i);
        const long long u = (kv->book.seq[list.seq[i]].len + KV4_UNIT - 1) / KV4_UNIT;
        units += (u + (u > 0)) * rows_seq;
        rows += u ? rows_seq : 0;
    }
    // one CTA per SM, fewer where the warps would find less than a unit each;
    // a CTA per row at least, so that few short rows are merged inside a CTA.
    // A captured call is replayed at lengths to come: every SM.
    const long long want = std::max((units + S::W - 1) / S::W, rows);
    const int       grid = whole ? kv->sms : (int)std::max(1ll, std::min<long long>(kv->sms, want));
    const size_t    smem = S::smem(n);
    auto            kern = k_kv4_attend<T, NB, NT, N>;
    static std::atomic<unsigned> done{0};
    CK(ecu_allow_smem(kern, S::smem(N), kv->device, done));
    return launched("ecu_kv_attend", ecu_launch_early(kern, (unsigned)grid, S::W * 32, smem, s, a, list));
}

template <typename T, int NB, int NT>
static int attend_list(ecu_kv *kv, KvAttendArgs a, const int *seq, int n, bool whole, cudaStream_t s)
{
    // at most 2^31 - 1 places in a launch, however the sequences may grow
    const long long places = (long long)kv->n_head_kv * ((a.n_rep + KvShape<T, NB, NT>::HG - 1) / KvShape<T, NB, NT>::HG) *
                             ((long long)kv->book.max_pages * (KV4_PAGE / KV4_UNIT) + 1);
    if (places > INT_MAX) return say("ecu_kv_attend", "too many positions and heads a sequence");
    const int most = (int)std::min<long long>(KV4_LIST, INT_MAX / places);
    for (int i = 0; i < n; i += most) {
        const int  m = std::min(most, n - i);
        const int *q = seq ? seq + i : nullptr;
        if ((m <= 64 ? attend_launch<T, NB, NT, 64>(kv, a, q, i, m, whole, s)
                     : attend_launch<T, NB, NT, KV4_LIST>(kv, a, q, i, m, whole, s)) != 0)
            return -1;
        a.q = (const T *)a.q + (size_t)m * a.q_stride;
        a.out = (T *)a.out + (size_t)m * a.out_stride;
    }
    return 0;
}

template <typename T, int NT>
static int attend_dim(ecu_kv *kv, const KvAttendArgs &a, const int *seq, int n, bool whole, cudaStream_t s)
{
    switch (kv->head_dim / 32) {
    case 1: return attend_list<T, 1, NT>(kv, a, seq, n, whole, s);
    case 2: return attend_list<T, 2, NT>(kv, a, seq, n, whole, s);
    case 3: return attend_list<T, 3, NT>(kv, a, seq, n, whole, s);
    default: return attend_list<T, 4, NT>(kv, a, seq, n, whole, s);
    }
}

// Tickets of each CTA's row, then two partials a CTA of at most 8 heads.
static size_t count_bytes(const ecu_kv *kv) { return ((size_t)kv->sms * sizeof(unsigned) + 255) & ~(size_t)255; }

extern "C" size_t ecu_kv_ws_bytes(const ecu_kv *kv)
{
    return kv && kv->device >= 0 ? count_bytes(kv) + (size_t)kv->sms * 2 * 8 * (kv->head_dim + 2) * sizeof(float) : 0;
}

extern "C" int ecu_kv_attend(ecu_kv *kv, int layer, int dtype, const void *q, void *out, int n_head, long q_stride,
                             long out_stride, const int *seq, int n, float scale, void *ws, void *stream)
{
    const char *what = "ecu_kv_attend";
    if (!kv || n < 0) return say(what, "null argument or negative count");
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
    if (slots_ok(kv, seq, n, what) != 0) return -1;
    if (n == 0) return 0;
    const long row = (long)n_head * kv->head_dim;
    if (!q || !out) return say(what, "null rows");
    if (n > 1 && (q_stride < row || out_stride < row)) return say(what, "rows overlap: a stride below n_head * head_dim");
    if (((uintptr_t)q | (uintptr_t)out) % es || ((uintptr_t)ws & 15)) return say(what, "rows or workspace are not aligned");
    if (kv->device < 0) return say(what, "the pool has no device");
    DeviceScope d(kv->device);
    if (!d.ok) return say(what, "the pool's device cannot be used");
    const cudaStream_t s = (cudaStream_t)stream;
    const int          cap = capturing(s, what);
    if (cap < 0) return -1;
    if (!ws) {
        if (cap) return say(what, "a captured call needs a workspace of its own");
        try {
            unsigned long long id = 0;
            CK(cudaStreamGetId(s, &id));
            const size_t bytes = ecu_kv_ws_bytes(kv);
            if (kv->ws.size() >= KV4_STREAMS && !kv->ws.count(id)) {        // streams come and go: start over
                CK(cudaDeviceSynchronize());
                for (auto &w : kv->ws) {
                    if (!w.second) continue;
                    if (!kv->spare) std::swap(kv->spare, w.second);
                    else {
                        cudaFree(w.second);
                        kv->device_bytes -= bytes;
                    }
                }
                kv->ws.clear();
            }
            void *&own = kv->ws[id];
            if (!own) std::swap(own, kv->spare);
            if (!own) {
                void        *p = nullptr;
                CK(cudaMalloc(&p, bytes));
                const cudaError_t e = cudaMemsetAsync(p, 0, bytes, s);       // ahead of the call that takes it
                if (e != cudaSuccess) {
                    cudaGetLastError();
                    cudaFree(p);
                    ecu_set_error(nullptr, 0, "%s: clearing a workspace failed: %s", what, cudaGetErrorString(e));
                    return -1;
                }
                own = p;
                kv->device_bytes += bytes;
            }
            ws = own;
        } catch (const std::exception &e) {
            return say(what, e.what());
        }
    }
    KvAttendArgs a;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.layer = kv->data + (size_t)layer * kv->book.n_pages * kv->page_bytes;
    a.page_bytes = kv->page_bytes;
    a.table = kv->table();
    a.len = kv->len();
    a.max_pages = kv->book.max_pages;
    a.n_pages = kv->book.n_pages;
    a.n_kv = kv->n_head_kv;
    a.n_rep = n_head / kv->n_head_kv;
    a.scale = scale;
    a.wide_q = !(((uintptr_t)q | (uintptr_t)(q_stride * (long)es)) & 15);
    a.count = (unsigned *)ws;
    a.part = (float *)((uint8_t *)ws + count_bytes(kv));
    if (dtype == ECU_F16) return attend_dim<__half, 1>(kv, a, seq, n, cap, s);
    if (dtype == ECU_BF16) return attend_dim<__nv_bfloat16, 1>(kv, a, seq, n, cap, s);
    return attend_tiles(dtype, a.n_rep) == 2 ? attend_dim<float, 2>(kv, a, seq, n, cap, s) : attend_dim<float, 1>(kv, a, seq, n, cap, s);
}
