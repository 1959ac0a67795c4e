// ecu_draft.cu -- a step with drafted tokens behind engine_cuda.h: rows turned
// by their positions and appended, and the drafts' verification.  (The attention
// is in ecu_tree.cu, ecu_kv_keep, a change of the pool, in ecu_kv4.cu.)
#include "ecu_draft.h"
#include "ecu_rope.cuh"
#include "ecu_verify.cuh"

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

// -------------------------------------------------------------- rotation ---

static int set_turns(ecu_rope *r, int rot, int interleaved, const double *freq, double factor, const char *what)
{
    if (!r || !freq) return say(what, "null argument");
    if (rot < 0 || rot > 128 || rot % 2) {
        ecu_set_error(nullptr, 0, "%s: %d turning dimensions (an even number up to 128)", what, rot);
        return -1;
    }
    if (!std::isfinite(factor)) return say(what, "the factor is not finite");
    ecu_rope t = {};
    t.rot = rot;
    t.interleaved = interleaved != 0;
    t.factor = factor;
    for (int i = 0; i < rot / 2; i++) {
        if (!std::isfinite(freq[i])) return say(what, "a frequency is not finite");
        // radians a position as a fraction of a turn: 64 bits behind the point
        long double f = (long double)freq[i] / (2.0L * 3.14159265358979323846264338327950288L);
        f -= floorl(f);
        const long double w = roundl(f * 18446744073709551616.0L);
        t.turn[i] = w >= 18446744073709551616.0L ? 0 : (uint64_t)w;
    }
    *r = t;
    return 0;
}

extern "C" int ecu_rope_set(ecu_rope *r, int rot, int interleaved, const double *freq, double factor)
{
    return set_turns(r, rot, interleaved, freq, factor, "ecu_rope_set");
}

extern "C" int ecu_rope_init(ecu_rope *r, int rot, int interleaved, double base, int scaling, double factor, double context, double slow,
                             double fast)
{
    const char *what = "ecu_rope_init";
    if (rot < 2 || rot > 128 || rot % 2) {
        ecu_set_error(nullptr, 0, "%s: %d turning dimensions (an even number up to 128)", what, rot);
        return -1;
    }
    if (!(base > 1.0) || !std::isfinite(base)) return say(what, "the base is not a number above 1");
    if (scaling < ECU_ROPE_PLAIN || scaling > ECU_ROPE_YARN) return say(what, "unknown scaling");
    if (scaling != ECU_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return say(what, "the scaling factor is not a number from 1 on");
    if (scaling >= ECU_ROPE_BANDS && (!(context >= 1.0) || !std::isfinite(context) || !(slow > 0.0) || !(fast > slow) || !std::isfinite(fast)))
        return say(what, "the original context or the bounds slow < fast are not valid");
    const double pi = 3.14159265358979323846;
    double       f[64], attention = 1.0, lo = 0.0, hi = 1.0;
    if (scaling == ECU_ROPE_YARN) {
        // the pair that turns so many times over the original context
        auto pair = [&](double turns) { return rot * std::log(context / (turns * 2.0 * pi)) / (2.0 * std::log(base)); };
        lo = std::max(std::floor(pair(fast)), 0.0);
        hi = std::min(std::ceil(pair(slow)), rot - 1.0);
        if (hi == lo) hi += 0.001;
        attention = 0.1 * std::log(factor) + 1.0;
    }
    for (int i = 0; i < rot / 2; i++) {
        const double x = std::pow(base, -2.0 * i / rot);
        double       w = 1.0;                             // how much of the pair's own frequency stays
        if (scaling == ECU_ROPE_LINEAR) w = 0.0;
        else if (scaling == ECU_ROPE_BANDS) w = std::min(1.0, std::max(0.0, (context * x / (2.0 * pi) - slow) / (fast - slow)));
        else if (scaling == ECU_ROPE_YARN) w = 1.0 - std::min(1.0, std::max(0.0, (i - lo) / (hi - lo)));
        f[i] = scaling == ECU_ROPE_PLAIN ? x : w * x + (1.0 - w) * (x / factor);
    }
    return set_turns(r, rot, interleaved, f, attention, what);
}

template <typename T, typename O, int N>
static int rope_launch(ecu_kv *kv, RopeArgs a, const int *seq, int first, const int *n_new, int n, cudaStream_t s)
{
    KvRows<N> r;
    fill_rows(r, seq, first, n_new, n);
    const int total = r.row0[n], hd = kv->head_dim;
    if (total == 0) return 0;
    // a block takes whole rows, or, of few rows, a part of their heads: enough
    // blocks for every SM first, then up to 8 KV heads and some 40 KB of keys
    a.heads = std::min(a.kv.n_kv, 8);
    while (a.heads > 1 && (long long)total * ((a.kv.n_kv + a.heads - 1) / a.heads) < kv->sms) a.heads = (a.heads + 1) / 2;
    const int chunks = (a.kv.n_kv + a.heads - 1) / a.heads, per_row = (a.turns.rot / 2 + 7) / 8 * 128 + a.heads * hd * 8;
    a.rows = std::max(1, std::min({64, 40960 / per_row, (int)((long long)total * chunks / (4 * kv->sms))}));
    const long long blocks = (long long)((total + a.rows - 1) / a.rows) * chunks;
    if (blocks > INT_MAX) return say("ecu_kv_append_rope", "too many rows");
    return launched("ecu_kv_append_rope",
                    ecu_launch_early(k_kv4_append_rope<T, O, N>, (unsigned)blocks, 256, (size_t)a.rows * per_row, s, a, r));
}

template <typename T, typename O> static int rope_list(ecu_kv *kv, RopeArgs a, const int *seq, const int *n_new, int n, cudaStream_t s)
{
    const size_t row = (size_t)kv->n_head_kv * kv->head_dim;
    for (int i = 0; i < n; i += KV4_LIST) {
        const int  m = std::min(KV4_LIST, n - i);
        const int *q = seq ? seq + i : nullptr;
        if ((m <= 64 ? rope_launch<T, O, 64>(kv, a, q, i, n_new + i, m, s) : rope_launch<T, O, KV4_LIST>(kv, a, q, i, n_new + i, m, s)) != 0)
            return -1;
        size_t rows = 0;
        for (int j = 0; j < m; j++) rows += n_new[i + j];
        a.kv.k = (const T *)a.kv.k + rows * a.kv.k_stride;
        a.kv.v = (const T *)a.kv.v + rows * a.kv.v_stride;
        if (a.q) {
            a.q = (const T *)a.q + rows * a.q_stride;
            a.q_out = (T *)a.q_out + rows * a.q_out_stride;
        }
        if (a.depth) a.depth += rows;
        if (a.kv.k_out) {
            a.kv.k_out = (O *)a.kv.k_out + rows * row;
            a.kv.v_out = (O *)a.kv.v_out + rows * row;
        }
    }
    return 0;
}

template <typename T> static int rope_out(ecu_kv *kv, const RopeArgs &a, int out_dtype, const int *seq, const int *n_new, int n, cudaStream_t s)
{
    if (out_dtype == ECU_F32) return rope_list<T, float>(kv, a, seq, n_new, n, s);
    if (out_dtype == ECU_F16) return rope_list<T, __half>(kv, a, seq, n_new, n, s);
    return rope_list<T, __nv_bfloat16>(kv, a, seq, n_new, n, s);
}

extern "C" int ecu_kv_append_rope(ecu_kv *kv, int layer, const ecu_rope *rope, int dtype, const void *q, const void *k, const void *v,
                                  int n_head, long q_stride, long k_stride, long v_stride, const int *seq, const int *n_new, int n,
                                  const int *depth, void *q_out, long q_out_stride, int out_dtype, void *k_out, void *v_out, void *stream)
{
    const char *what = "ecu_kv_append_rope";
    if (!kv || !rope || n < 0 || (n > 0 && !n_new)) return say(what, "null argument or negative count");
    if (layer < 0 || layer >= kv->n_layer) {
        ecu_set_error(nullptr, 0, "%s: layer %d of %d", what, layer, kv->n_layer);
        return -1;
    }
    const size_t es = dtype_bytes(dtype), os = dtype_bytes(out_dtype);
    if (!es || !os) return say(what, "unknown element type");
    if (rope->rot < 0 || rope->rot > kv->head_dim || rope->rot % 2) {
        ecu_set_error(nullptr, 0, "%s: %d turning dimensions of %d", what, rope->rot, kv->head_dim);
        return -1;
    }
    if (q && (n_head < 1 || n_head % kv->n_head_kv || n_head > INT_MAX / kv->head_dim)) {
        ecu_set_error(nullptr, 0, "%s: %d query heads for %d KV heads", what, n_head, kv->n_head_kv);
        return -1;
    }
    if (!q != !q_out) return say(what, "one of q and q_out alone");
    if (whole(kv, what) != 0) return -1;
    const long row = (long)kv->n_head_kv * kv->head_dim, q_row = (long)n_head * kv->head_dim;
    try {
        const long long rows = rows_ok(kv, seq, n_new, n, INT_MAX, what);
        if (rows < 0) return -1;
        for (int i = 0; i < n; i++) {
            const int   s = number_of(0, seq, i);
            const auto &b = kv->book.seq[s];
            for (int j = (b.len - n_new[i]) / ECU_KV4_PAGE; n_new[i] > 0 && j < (int)b.page.size(); j++)
                if (kv->book.ref[b.page[j]] > 1) {
                    ecu_set_error(nullptr, 0, "%s: positions of sequence %d lie in a page that other sequences hold", what, s);
                    return -1;
                }
        }
        if (rows == 0) return 0;
        if (rows > INT_MAX / 2) return say(what, "too many rows");
        if (!k || !v || (!k_out) != (!v_out)) return say(what, "null rows, or one of k_out and v_out alone");
        if (rows > 1 && (k_stride < row || v_stride < row || (q && (q_stride < q_row || q_out_stride < q_row))))
            return say(what, "rows overlap: a stride below their width");
        if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v) % es || (k_out && ((uintptr_t)k_out | (uintptr_t)v_out) % os) ||
            ((uintptr_t)depth & 3))
            return say(what, "rows are not aligned to their elements");
        if (q == q_out && q && rows > 1 && q_stride != q_out_stride) return say(what, "queries in place keep their stride");
        if (kv->device < 0) return say(what, "the pool has no device");
        DeviceScope d(kv->device);
        if (!d.ok) return say(what, "the pool's device cannot be used");
        RopeArgs a = {};
        a.kv.k = k;
        a.kv.v = v;
        a.kv.k_stride = k_stride;
        a.kv.v_stride = v_stride;
        a.kv.k_out = k_out;
        a.kv.v_out = v_out;
        a.kv.layer = kv->data + (size_t)layer * kv->book.n_pages * kv->page_bytes;
        a.kv.page_bytes = kv->page_bytes;
        a.kv.table = kv->table();
        a.kv.len = kv->len();
        a.kv.max_pages = kv->book.max_pages;
        a.kv.n_pages = kv->book.n_pages;
        a.kv.n_kv = kv->n_head_kv;
        a.kv.nb = kv->head_dim / 32;
        a.kv.nb_inv = (65536 + a.kv.nb - 1) / a.kv.nb;    // exact below 32768: at most 8 heads of 4 blocks
        a.kv.wide = !(((uintptr_t)k | (uintptr_t)v | (uintptr_t)(k_stride * (long)es) | (uintptr_t)(v_stride * (long)es)) & 15);
        a.kv.wide_out = !(((uintptr_t)k_out | (uintptr_t)v_out) & 15);
        a.q = q;
        a.q_out = q_out;
        a.q_stride = q_stride;
        a.q_out_stride = q_out_stride;
        a.depth = depth;
        a.n_rep = q ? n_head / kv->n_head_kv : 0;
        a.wide_q = !(((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)(q_stride * (long)es) | (uintptr_t)(q_out_stride * (long)es)) & 15);
        a.turns.rot = rope->rot;
        a.turns.interleaved = rope->interleaved;
        a.turns.factor = rope->factor;
        for (int i = 0; i < 64; i++) a.turns.turn[i] = rope->turn[i];
        const cudaStream_t s = (cudaStream_t)stream;
        if (dtype == ECU_F32) return rope_out<float>(kv, a, out_dtype, seq, n_new, n, s);
        if (dtype == ECU_F16) return rope_out<__half>(kv, a, out_dtype, seq, n_new, n, s);
        return rope_out<__nv_bfloat16>(kv, a, out_dtype, seq, n_new, n, s);
    } catch (const std::exception &e) {
        return say(what, e.what());
    }
}

// ---------------------------------------------------------------- verify ---

template <typename T, int N>
static int verify_launch(VerifyArgs a, const int *n_row, int n, int sms, cudaStream_t s)
{
    VerifyRows<N> r;
    r.n = n;
    r.row0[0] = 0;
    for (int i = 0; i < n; i++) r.row0[i + 1] = r.row0[i] + n_row[i];
    // CTAs of a sequence: as many as keep all sequences in flight together, two
    // CTAs an SM, and find a few hundred tokens a warp
    const int cl = std::max(1, std::min(VER_MAX_CTAS, std::min(2 * sms / n, a.vocab / (VER_WARPS * 64))));
    cudaLaunchConfig_t  cfg = {};
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cl;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(n * cl));
    cfg.blockDim = dim3(VER_WARPS * 32);
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    if (s == cudaStreamPerThread) ecu_on_thread_stream();
    return launched("ecu_draft_verify", cudaLaunchKernelEx(&cfg, k_draft_verify<T, N>, a, r));
}

template <typename T> static int verify_list(VerifyArgs a, const int *n_row, int n, int sms, cudaStream_t s)
{
    for (int i = 0; i < n; i += KV4_LIST) {
        const int m = std::min(KV4_LIST, n - i);
        a.seq0 = i;
        if ((m <= 64 ? verify_launch<T, 64>(a, n_row + i, m, sms, s) : verify_launch<T, KV4_LIST>(a, n_row + i, m, sms, s)) != 0) return -1;
        size_t rows = 0;
        for (int j = 0; j < m; j++) rows += n_row[i + j];
        a.logits = (const T *)a.logits + rows * a.stride;
        if (a.draft) a.draft += rows * a.draft_stride;
        a.token += rows;
        a.parent += rows;
        a.u += rows;
        a.kept += rows;
    }
    return 0;
}

extern "C" int ecu_draft_verify(int dtype, const void *logits, long stride, int n_vocab, const float *draft, long draft_stride,
                                const int *token, const int *parent, const int *n_row, int n, const float *u, const float *u_next,
                                const float *temperature, int *kept, int *n_kept, int *next, int device, void *stream)
{
    const char  *what = "ecu_draft_verify";
    const size_t es = dtype_bytes(dtype);
    if (!es) return say(what, "unknown element type");
    if (n < 0 || (n > 0 && (!n_row || !u_next || !n_kept || !next)) || n_vocab < 1) return say(what, "null argument, negative count or no vocabulary");
    if (n_vocab > 1 << 30) return say(what, "a vocabulary of more than 2^30 tokens");       // (tokens are counted in an int, past the end too)
    long long rows = 0;
    for (int i = 0; i < n; i++) {
        if (n_row[i] < 0 || n_row[i] > VER_ROWS) {
            ecu_set_error(nullptr, 0, "%s: %d rows of sequence %d (64 at most)", what, n_row[i], i);
            return -1;
        }
        rows += n_row[i];
    }
    if (n == 0) return 0;
    if (rows > INT_MAX / 2) return say(what, "too many rows");
    if (rows > 0 && (!logits || !token || !parent || !u || !kept)) return say(what, "null rows");
    if (rows > 1 && (stride < n_vocab || (draft && draft_stride < n_vocab))) return say(what, "rows overlap: a stride below n_vocab");
    if ((uintptr_t)logits % es ||
        (((uintptr_t)draft | (uintptr_t)token | (uintptr_t)parent | (uintptr_t)u | (uintptr_t)u_next | (uintptr_t)temperature |
          (uintptr_t)kept | (uintptr_t)n_kept | (uintptr_t)next) & 3))
        return say(what, "rows are not aligned to their elements");
    int ndev = 0;
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) {
        cudaGetLastError();
        ecu_set_error(nullptr, 0, "%s: CUDA device %d not available (%d devices)", what, device, ndev);
        return -1;
    }
    DeviceScope d(device);
    if (!d.ok) return say(what, "the device cannot be used");
    int sms = 0;
    CK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    VerifyArgs a = {};
    a.logits = logits;
    a.stride = stride;
    a.draft = draft;
    a.draft_stride = draft_stride;
    a.token = token;
    a.parent = parent;
    a.u = u;
    a.u_next = u_next;
    a.temperature = temperature;
    a.kept = kept;
    a.n_kept = n_kept;
    a.next = next;
    a.vocab = n_vocab;
    a.wide = !(((uintptr_t)logits | (uintptr_t)(stride * (long)es)) & 15);
    const cudaStream_t s = (cudaStream_t)stream;
    if (dtype == ECU_F32) return verify_list<float>(a, n_row, n, sms, s);
    if (dtype == ECU_F16) return verify_list<__half>(a, n_row, n, sms, s);
    return verify_list<__nv_bfloat16>(a, n_row, n, sms, s);
}
