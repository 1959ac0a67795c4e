/*
 * engine_cuda.h -- C ABI of the B200 (sm_100a) llama token loop.
 *
 * Drop-in for distcomp's CPU engine (src/engine.h:74-101) and its GGUF block
 * dequant (src/gguf.h:86).  Plain C types only: no CUDA or torch types cross
 * this boundary; streams are passed as `void *` (a cudaStream_t, or NULL for
 * the context's own stream).
 *
 * Contract kept from the reference:
 *   - errors are int 0 / -1; open functions write a message into err[errlen]
 *     (src/engine.c:23-27), ecu_last_error() returns the last one per thread;
 *   - a context serves one stage: EMBED, a contiguous LAYERS range or HEAD
 *     (src/engine.h:23-27); ECU_STAGE_FULL is an addition that runs all three
 *     back to back on one device;
 *   - ecu_forward has llm_forward's `out` contract (src/engine.h:83-88):
 *       EMBED  out[0..n_embd)  = embedding row of `token`
 *       LAYERS out in and out  = the state after this stage's layers
 *       HEAD   out[0..n_embd)  = normed state, out[n_embd] = argmax token
 *       FULL   as HEAD, from `token` alone;
 *   - a context is single-threaded, like llm_ctx.
 * Weights are uploaded (and repacked for coalesced loads, values unchanged)
 * once at open; the caller's file buffer may be released afterwards.
 */
#ifndef DC_ENGINE_CUDA_H
#define DC_ENGINE_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    ECU_STAGE_EMBED  = 0,   /* src/engine.h:24 LLM_STAGE_EMBED  */
    ECU_STAGE_LAYERS = 1,   /* src/engine.h:25 LLM_STAGE_LAYERS */
    ECU_STAGE_HEAD   = 2,   /* src/engine.h:26 LLM_STAGE_HEAD   */
    ECU_STAGE_FULL   = 3,   /* new: embed + all layers + head on one device */
    ECU_STAGE_SPAN   = 4    /* new: a layer range with the embedding and/or the
                               head folded in (ecu_ctx_open_span) */
};

/* ecu_ctx_open_span flags */
#define ECU_SPAN_EMBED 1u   /* the step starts from a token: embedding row first */
#define ECU_SPAN_HEAD  2u   /* the step ends with the output head: argmax token */
#define ECU_SPAN_FFN_FIRST 4u   /* layer `first` contributes its FFN half only (RMSNorm,
                                   gate/up, SwiGLU, down + residual) */
#define ECU_SPAN_ATTN_LAST 8u   /* layer `last` contributes its attention half only
                                   (RMSNorm, Q/K/V, attention, attn_output + residual):
                                   a pipeline may cut a layer between its halves */

typedef struct ecu_model ecu_model;   /* host view of a GGUF file (borrowed bytes) */
typedef struct ecu_ctx   ecu_ctx;     /* one stage resident on one device           */

/* Geometry of an open context (the fields of llm_ctx, src/engine.h:46-70). */
typedef struct {
    int   n_layer, n_embd, n_head, n_head_kv, n_ff, head_dim, n_vocab, n_rep, n_ctx;
    int   stage, first, last, pos, device;
    float rms_eps, rope_base;
    size_t device_bytes;      /* weights + KV cache + work buffers on the device */
} ecu_info;

/* ---- GGUF view --------------------------------------------------------- */

/* Parse a GGUF v2/v3 image held by the caller (replaces gguf_open,
 * src/gguf.h:52).  Tensor data stay in `file` until a context is opened. */
int  ecu_model_open(ecu_model **out, const void *file, size_t size, char *err, size_t errlen);

/* Assemble a model from tensor views and metadata instead of a file image,
 * as dcd's shard role does when it builds a gguf_file from received tensors
 * (src/daemon.c:963-1019). */
/* The same from a GGUF file on disk: mapped read-only, so that a context
 * opened from it reads (pages in) only its stage's tensors, and the model
 * owns the mapping until ecu_model_close.  Replaces the reference's whole-
 * file fread (src/shard.c:84-104, llm_open_file) for stage nodes. */
int  ecu_model_open_file(ecu_model **out, const char *path, char *err, size_t errlen);

ecu_model *ecu_model_new(void);
int  ecu_model_set_str(ecu_model *m, const char *key, const char *val);
int  ecu_model_set_u32(ecu_model *m, const char *key, unsigned long val);
int  ecu_model_set_f32(ecu_model *m, const char *key, float val);
int  ecu_model_add_tensor(ecu_model *m, const char *name, unsigned n_dims, const uint64_t *dims,
                          unsigned ggml_type, const void *data, size_t nbytes);
void ecu_model_close(ecu_model *m);
/* Number of tensors, and lookup by name (gguf_tensor_find, src/gguf.h:72). */
size_t ecu_model_n_tensors(const ecu_model *m);
int  ecu_model_tensor(const ecu_model *m, const char *name, unsigned *ggml_type,
                      unsigned *n_dims, uint64_t dims[4], const void **data, size_t *nbytes);

/* ---- engine (src/engine.h:72-101) -------------------------------------- */

/* Device bytes a stage needs at context length n_ctx (0 = the model's);
 * the device counterpart of llm_ctx_floats (src/engine.h:74).  0 on error. */
size_t ecu_ctx_bytes(const ecu_model *m, int stage, int first, int last, int n_ctx);

/* Open a stage on CUDA device `device` (replaces llm_ctx_open,
 * src/engine.h:79).  The same geometry and error rules as the reference. */
int  ecu_ctx_open(ecu_ctx **out, const ecu_model *m, int stage, int first, int last, int n_ctx,
                  int device, char *err, size_t errlen);
/* A pipeline stage that folds the reference's EMBED / LAYERS / HEAD stages
 * of one node into one context (src/shard.c:358-437 gives a node's layer
 * range; its entry node also embeds, its exit node also runs the head):
 * layers first..last (first > last: none) plus the embedding and/or the
 * head by `flags`; with ECU_SPAN_FFN_FIRST / ECU_SPAN_ATTN_LAST the range
 * starts at layer first's FFN half / ends with layer last's attention half
 * (a layer cut between two GPUs: the residual stream is all that crosses).
 * One persistent step per token runs all of it.  Forward
 * contract: input a token with ECU_SPAN_EMBED, else a state in out;
 * output the state, plus out[n_embd] = the argmax with ECU_SPAN_HEAD.  The
 * position advances every step.  ecu_ctx_info reports ECU_STAGE_SPAN. */
int  ecu_ctx_open_span(ecu_ctx **out, const ecu_model *m, int first, int last, unsigned flags, int n_ctx,
                       int device, char *err, size_t errlen);
void ecu_ctx_close(ecu_ctx *c);
int  ecu_ctx_info(const ecu_ctx *c, ecu_info *info);
/* How the context runs a step: "persistent" (one cooperative kernel per
 * token, every phase of the stage inside it) or "kernels: <reason>" (one
 * kernel per operation, and why the persistent kernel does not apply).
 * No reference counterpart (the CPU engine has one implementation). */
const char *ecu_ctx_path(const ecu_ctx *c);

/* One token through the stage, host `out` (replaces llm_forward,
 * src/engine.h:88).  -1 for a token outside the vocabulary (EMBED/FULL) or
 * an exhausted context (LAYERS/FULL). */
int  ecu_forward(ecu_ctx *c, int token, float *out);
/* Rewind the KV cache (replaces llm_reset, src/engine.h:90). */
void ecu_reset(ecu_ctx *c);
/* Exactly one layer at the current position, position unchanged
 * (replaces llm_layer_once, src/engine.h:94). */
int  ecu_layer_once(ecu_ctx *c, int layer_idx, float *out);
/* The first n layers of the stage (0 = all), then pos++ (replaces
 * llm_step_layers, src/engine.h:98). */
int  ecu_step_layers(ecu_ctx *c, int n, float *out);
/* Argmax of the last HEAD/FULL logits, lowest index on ties (replaces
 * llm_pick, src/engine.h:101). */
int  ecu_pick(const ecu_ctx *c);
/* Copy the last logits to host memory (n floats, n <= n_vocab). */
int  ecu_get_logits(const ecu_ctx *c, float *out, size_t n);
/* Set the cache position directly (what engine_stages.c does with lay.pos). */
int  ecu_set_pos(ecu_ctx *c, int pos);

/* ---- device-resident chaining (no host hop between stages) ------------- */

/* Device pointer of the stage's state buffer (n_embd + 1 floats).  LAYERS
 * and HEAD read their input there; every stage leaves its output there. */
float *ecu_state_ptr(ecu_ctx *c);
/* ecu_forward without host copies: input/output in ecu_state_ptr(c),
 * enqueued on `stream` (NULL = the context's stream), not synchronised.
 * The token is read from host memory at enqueue time. */
int  ecu_forward_dev(ecu_ctx *c, int token, void *stream);
/* Device address of the context's current token (one int).  EMBED and FULL
 * steps read their input token there; HEAD and FULL steps write their argmax
 * there.  A pipeline hands the token from the last stage to the first by
 * writing this address (a device copy or an NCCL receive), the way the
 * reference's shard.c sends the argmax back to the entry node. */
int *ecu_token_ptr(ecu_ctx *c);
/* One step from device-resident input only: the token at ecu_token_ptr(c)
 * (EMBED/FULL) or the state at ecu_state_ptr(c) (LAYERS/HEAD), output left
 * in the state buffer (and the token word for HEAD/FULL), position advanced.
 * Enqueued on `stream` (NULL = the context's stream), not synchronised; a
 * token outside the vocabulary is reported by the next ecu_sync.  -1 when
 * the context is exhausted. */
int  ecu_step_dev(ecu_ctx *c, void *stream);
/* A second context of the same stage on the same device that shares the
 * first one's uploaded weights and keeps its own KV cache, position, work
 * buffers and stream: one per concurrent sequence (the reference keeps one
 * llm_ctx per process, src/daemon.c:757; a GPU stage serving several
 * interleaved sequences needs one cache each).  The weights are freed when
 * the last context holding them closes. */
int  ecu_ctx_fork(ecu_ctx **out, ecu_ctx *base, char *err, size_t errlen);

/* ---- tensor parallelism (the alternative partition to shard.c's layer
 * ranges, src/shard.c:358-437): one FULL context per GPU, rank r of w owns
 * query/KV heads [r*n/w, ..), the matching rows of the fused Q/K/V, rows
 * [r*n_embd/w, ..) of attn_output and ffn_down, FFN channels [r*n_ff/w, ..)
 * and a vocabulary slice of the head.  Every projection keeps its whole
 * input, so each output element is computed by one rank with the one-GPU
 * arithmetic (bit-identical results); the ranks exchange outputs inside the
 * persistent step through each other's memory (NVLink peer stores).  Steps
 * must be issued on every rank in the same order (ecu_forward / decode);
 * a rank that falls more than ~2 s behind makes the others' step fail with
 * a timeout status. */
#define ECU_TP_HANDLE_BYTES 64
int  ecu_ctx_open_tp(ecu_ctx **out, const ecu_model *m, int n_ctx, int device, int tp_rank, int tp_world,
                     char *err, size_t errlen);
/* This rank's shareable handle (ECU_TP_HANDLE_BYTES) for the other ranks. */
int  ecu_tp_handle(ecu_ctx *c, unsigned char *out);
/* Map every rank's handle (world * ECU_TP_HANDLE_BYTES, rank order; this
 * rank's own entry is ignored).  Call once, on every rank, before a step. */
int  ecu_tp_connect(ecu_ctx *c, const unsigned char *handles);
/* out4 = {rank, world, first vocabulary row, end row} of this context's head
 * slice (ecu_get_logits returns that slice). */
int  ecu_tp_slice(const ecu_ctx *c, int *out4);
/* ---- pipeline links: the stages of a layer pipeline (one context per GPU
 * and sequence, typically spans) hand the state and the token to each
 * other inside their persistent steps, as tagged words written straight
 * into the next stage's memory over NVLink, instead of a host or NCCL hop
 * between steps (the reference sends them over UDP, src/shard.c:664-723).
 * Each stage's step then only needs launching, in the same sequence order
 * on every GPU: a step waits (bounded, ~2 s, then the status reports a
 * timeout) until its input has arrived.  Contexts with the persistent step
 * only, not tensor-parallel ones; every stage of a pipeline opened from the
 * same model.  Use ecu_step_dev on linked contexts. */
#define ECU_LINK_HANDLE_BYTES 64
/* This context's shareable handle (ECU_LINK_HANDLE_BYTES), for the stage
 * before it (another process: CUDA IPC). */
int  ecu_link_handle(ecu_ctx *c, unsigned char *out);
/* Send this context's output to the stage whose handle this is: its output
 * state, or with the head its argmax token (to the first stage). */
int  ecu_link_next(ecu_ctx *c, const unsigned char *handle);
/* The same for a context of this process (next may be on the same device;
 * then its steps must follow this one's on one stream). */
int  ecu_link_next_local(ecu_ctx *c, ecu_ctx *next);
/* This context's input arrives over a link: the state for a stage without
 * the embedding, else the token.  Once set, ecu_forward is refused. */
int  ecu_link_input(ecu_ctx *c);
/* A linked first stage's input token for its next step from the host (the
 * token the prompt's last position picked), enqueued on `stream` (NULL =
 * the context's stream) before that step. */
int  ecu_link_feed(ecu_ctx *c, int token, void *stream);

/* Greedy decode on a FULL context without host round trips: feeds
 * prompt[0..n_prompt) token by token, then generates n_gen tokens, each one
 * fed back on the device.  out_tokens receives the n_gen generated ids.
 * Returns 0, or -1 when the context runs out. */
int  ecu_generate(ecu_ctx *c, const int *prompt, int n_prompt, int n_gen, int *out_tokens);
/* A prompt of n tokens through a FULL context at once (the reference feeds
 * prompts token by token, src/shard.c:911-917, one llm_forward each): every
 * layer runs its n tokens as one batch (GEMMs on the tensor cores with
 * split-fp16 operands, about fp32 accuracy; causal attention over the
 * cache), the cache gets the n positions, and the last token goes through
 * the head: out = normed state (n_embd) + the picked token, as ecu_forward's
 * out for that token, and the context's position advances by n.  Results
 * agree with the token-by-token path within the 1e-3 bar, not bit for bit.
 * Shapes the batched kernels do not cover (unfused projections, head_dim
 * other than 64/128, n_ctx > 8192) and tensor-parallel ranks run the
 * per-token step instead.  Scratch for the batch is allocated on first use
 * and grows with the longest prompt. */
int  ecu_prefill(ecu_ctx *c, const int *tokens, int n, float *out);

/* The batched prompt for one stage of a layer pipeline (src/shard.c:358-437
 * splits the model into EMBED, LAYERS ranges and HEAD; the reference feeds
 * the prompt through them token by token, src/shard.c:911-917).  x: device
 * memory the caller owns, n rows of n_embd floats (the n prompt positions).
 * EMBED: x = the embedding rows of tokens[0..n).  LAYERS: x goes through the
 * stage's layers in place (ecu_prefill's kernels), the stage's KV cache
 * gets positions pos..pos+n-1 and its position advances by n.  HEAD: the
 * last row of x through the head, out = normed state + picked token as
 * ecu_forward's (tokens may be NULL).  SPAN: those of its parts in that
 * order, the position advancing by n.  Every stage's rows agree bit for bit
 * with a FULL context's ecu_prefill of the same prompt.  Synchronises the
 * context's stream before returning. */
int  ecu_prefill_rows(ecu_ctx *c, const int *tokens, int n, float *x, float *out);
/* Decode steps on a FULL context continuing from the token in the state
 * buffer, on the context's stream, without synchronising; used to time the
 * device-side loop.  Returns 0 or -1. */
int  ecu_decode_async(ecu_ctx *c, int n_steps);
/* Wait for the context's stream; returns -1 if a kernel reported an error. */
int  ecu_sync(ecu_ctx *c);
/* The context's CUDA stream (as void *). */
void *ecu_stream(ecu_ctx *c);

/* ---- block dequant on the device (replaces gguf_dequant, src/gguf.h:86) - */

/* Dequantise elements [off, off+n) of a tensor of `total` elements and ggml
 * type `ggml_type` whose raw GGUF blocks are at host pointer `raw`, on
 * device `device`, into host `dst`.  Same rejection rules as the reference
 * (range, block-aligned off, supported types).  Bit-exact with it. */
int  ecu_dequant(unsigned ggml_type, const void *raw, size_t total, size_t off, size_t n,
                 float *dst, int device);
/* The same from a context's uploaded (repacked) copy of tensor `name`,
 * proving the device layout holds the file's values. */
int  ecu_dequant_tensor(ecu_ctx *c, const char *name, size_t off, size_t n, float *dst);

/* ---- single-GEMV entry point (the quantised matvec of src/engine.c:348) - */

/* y[o] = sum_i W[i + o*n_in] x[i] for a raw GGUF weight at host pointer
 * `w_raw` on `device`; x and y are host arrays.  Uploads per call: for
 * tests and one-off use, not the token loop. */
int  ecu_matvec(unsigned ggml_type, const void *w_raw, int n_in, int n_out, const float *x,
                float *y, int device);

/* ---- without device allocation ------------------------------------------ */

/* y = W x over raw GGUF blocks already in device memory (n_out rows of
 * n_in inputs, the file's block order), and *d_token = the first maximum of
 * y with llm_pick's rules, enqueued on `stream` (NULL = the legacy default
 * stream) without synchronising.  All pointers are device pointers the
 * caller owns.  No counterpart in the reference: it is for callers that
 * cannot allocate device memory -- a shard node held to a fixed memory
 * budget, a host that hands out device memory from its own pool, a loop
 * that cannot take cudaMalloc's device synchronisation.  It allocates
 * nothing: its scratch is one fixed 16 KiB array inside the library, which
 * limits n_out to 524288 rows (more returns -1 with a message).  Every
 * call looks that array's device address up with cudaGetSymbolAddress
 * (which allocates nothing), so the address stays right across a context
 * torn down and created again; make the first call on a device before any
 * stream capture.  Every call shares the array, so calls that may overlap
 * on the GPU (two streams, two threads) race: serialise them. */
int  ecu_matvec_argmax_noalloc(unsigned ggml_type, const void *d_w, int n_in, int n_out,
                               const float *d_x, float *d_y, int *d_token, void *stream);

/* ---- a K/V cache in pages of 4-bit rows, shared by many sequences -------- */

/* The contexts above keep one dense fp32 cache each (the reference keeps one
 * llm_ctx per process, src/daemon.c:757); a server of many sequences keeps
 * theirs in one pool of pages instead, at 4.5 bits a value (fp32 contexts:
 * 32), and forks share the pages of their common prefix.
 *
 * A page holds ECU_KV4_PAGE positions of every KV head of one layer; page p
 * of layer l lies at data + (l * n_pages + p) * ecu_kv4_page_bytes().  One
 * page id names the same positions in every layer.  Per KV head a page has
 * 72 * head_dim bytes: K codes of the 64 positions (head_dim / 2 bytes each),
 * V codes, K scales, V scales (fp16, [64][head_dim / 32]).  A position's
 * codes are 16-byte chunks, one per block of 32 dimensions, two codes a byte
 * in order, the low nibble first; chunk b of position t lies at place
 * b ^ ((t >> 1) & 3) for head_dim 128, b ^ ((t >> 2) & 1) for 64, b for 32
 * and 96 (so that eight positions' chunks fall into different banks of
 * shared memory, where pages are copied whole).  A value is
 * (code - 8) * scale: the values of GGUF's Q4_0 blocks.  The scale is
 * fp16(m / -8), m the block's value of largest magnitude (the first of
 * equals; at most 65504 in magnitude), a code floor(x / scale + 8.5) clamped
 * to 0..15, decided exactly; a block with a value that is not finite reads
 * as NaN, one whose scale rounds to zero as zeros. */
#define ECU_KV4_PAGE 64

/* element types of the rows that the operators below read and write */
enum { ECU_F32 = 0, ECU_F16 = 1, ECU_BF16 = 2 };

typedef struct ecu_kv ecu_kv;

/* Bytes of one page of one layer; 0 for a shape that is not covered
 * (head_dim 32, 64, 96 and 128 are). */
size_t ecu_kv4_page_bytes(int n_head_kv, int head_dim);

/* A pool of n_pages pages for up to n_seq sequences (slots 0..n_seq-1, all
 * empty) of up to max_pages pages each.  data: n_layer * n_pages pages of
 * device memory that the caller keeps (16-byte aligned, its contents left as
 * they are), or NULL: the pool allocates them.  The bookkeeping (which
 * sequence holds which page, how many hold a page) is on the host, its table
 * and lengths are mirrored in device memory at fixed addresses.  device -1:
 * the bookkeeping alone, without a GPU (to plan capacity).  A pool is
 * single-threaded, like a context.  A thread that has calls enqueued on its own
 * default stream (cudaStreamPerThread) waits for them where it ends. */
int  ecu_kv_open(ecu_kv **out, int n_layer, int n_head_kv, int head_dim, int n_pages, int n_seq, int max_pages,
                 int device, void *data, char *err, size_t errlen);
void ecu_kv_close(ecu_kv *kv);

typedef struct {
    int    n_layer, n_head_kv, head_dim, n_pages, n_seq, max_pages, device;
    int    used;              /* pages that some sequence holds */
    size_t page_bytes, device_bytes;
    void  *data;              /* the pages */
    int   *table, *len;       /* device: page ids [n_seq][max_pages] (-1: none), positions [n_seq] */
} ecu_kv_info;
int  ecu_kv_get_info(const ecu_kv *kv, ecu_kv_info *info);
/* Positions of a sequence (-1: no such slot); its page ids into
 * pages[0..n) (NULL: none wanted). */
int  ecu_kv_len(const ecu_kv *kv, int seq, int *pages, int n);

/* The next four, and ecu_kv_compact, change sequences in the list's order;
 * each either does all of it or, with -1, nothing.  (Long changes take several
 * launches, about 2000 page copies and table words each.  Where one after the
 * first fails, which no valid call brings about, the pool refuses every later
 * call but those that read its bookkeeping, and ecu_kv_close.)  What they
 * change on the device is enqueued on
 * `stream` (NULL: the legacy default stream); calls on the same pool from
 * different streams are ordered by the caller, and a stream that is being
 * captured is refused (the bookkeeping would not be replayed).
 *
 * extend: sequence seq[i] grows by n_new[i] positions; pages are taken
 * lowest free id first.  Where its last page is partly filled and other
 * sequences hold it too, the sequence gets a copy of its own first (every
 * layer).  New positions' rows are what ecu_kv_append writes.
 * fork: dst[i], an empty slot, becomes a copy of src[i], sharing its pages.
 * truncate: sequence seq[i] keeps its first len[i] positions (at most its
 * length); pages past them are given back.  ecu_kv_free: all of them. */
int  ecu_kv_extend(ecu_kv *kv, const int *seq, const int *n_new, int n, void *stream);
int  ecu_kv_fork(ecu_kv *kv, const int *src, const int *dst, int n, void *stream);
int  ecu_kv_truncate(ecu_kv *kv, const int *seq, const int *len, int n, void *stream);
int  ecu_kv_free(ecu_kv *kv, const int *seq, int n, void *stream);
/* Moves pages so that those in use are pages 0..used-1: the k-th lowest page
 * at or above `used` goes to the k-th lowest hole below it (every layer), and
 * the tables follow.  Returns the number of pages moved, or -1. */
int  ecu_kv_compact(ecu_kv *kv, void *stream);

/* The rows of n sequences' newest positions, quantised into layer `layer`'s
 * pages: sequence seq[i] (NULL: slots 0..n-1; no slot twice) gets n_new[i]
 * rows, its positions len - n_new[i] .. len - 1, from consecutive rows of k
 * and v (device, `dtype`, a row's KV heads one after the other, rows k_stride
 * / v_stride elements apart).  The positions' pages must be the sequence's
 * own (freshly extended ones are).  k_out, v_out (or NULL): the values as the
 * cache holds them, `out_dtype`, rows of n_head_kv * head_dim without gaps,
 * apart from k and v.
 * The lengths are read on the device when the call runs, so a captured call
 * appends to the then newest positions (whose pages must then be the
 * sequence's own: that is checked when the call is made, not at a replay). */
int  ecu_kv_append(ecu_kv *kv, int layer, int dtype, const void *k, const void *v, long k_stride, long v_stride,
                   const int *seq, const int *n_new, int n, int out_dtype, void *k_out, void *v_out, void *stream);

/* Attention of one query row per sequence over all of its positions in layer
 * `layer`: out row i = softmax(scale * q_h K^T) V for the n_head query heads
 * (head h reads KV head h / (n_head / n_head_kv)) of sequence seq[i] (NULL:
 * slots 0..n-1; a slot may come twice).  q and out: device, `dtype`, a row's
 * heads one after the other, rows q_stride / out_stride elements apart.  An
 * empty sequence's row becomes zeros.  Sums and the softmax are fp32; of fp32
 * queries, and of their weights, 22 bits count.  A position that is not finite
 * in K makes its head's rows NaN, one in V its block of 32 dimensions, however
 * little it weighs.  The lengths are read on the device when the call runs.
 * ws: ecu_kv_ws_bytes() bytes of device memory, zeroed once before their
 * first use, that no other call uses at the same time; NULL: the pool's own
 * for this stream, which a stream that is being captured must not take (made
 * on its first call; past 16 streams the device is synchronised and they are
 * made anew).  out and q do not overlap. */
int    ecu_kv_attend(ecu_kv *kv, int layer, int dtype, const void *q, void *out, int n_head, long q_stride,
                     long out_stride, const int *seq, int n, float scale, void *ws, void *stream);
size_t ecu_kv_ws_bytes(const ecu_kv *kv);
/* Positions pos .. pos + n - 1 of a sequence as fp32 rows [n][n_head_kv *
 * head_dim] in host memory (K and V as the cache holds them; either may be
 * NULL): the cache's ecu_dequant_tensor.  Synchronises `stream`. */
int    ecu_kv_read(ecu_kv *kv, int layer, int seq, int pos, int n, float *k, float *v, void *stream);

/* ---- steps with drafted tokens ------------------------------------------- */

/* A step may check several drafted tokens of a sequence at once: extend the
 * sequence by them, write their rows (ecu_kv_append_rope), attend to the cache
 * and to each other along a tree (ecu_kv_attend_tree), hold them against the
 * target's probabilities (ecu_draft_verify), and keep what was accepted
 * (ecu_kv_keep).  These calls are for programs that run a model's layers
 * themselves: ecu_batch_feed takes no trees and hands back a sequence's last row
 * alone.  The drafted rows are a sequence's newest positions; row 0 is
 * the token that was picked last, every other row hangs on an earlier one.  No
 * counterpart in the reference, which feeds one token a step
 * (src/shard.c:911-917). */
#define ECU_DRAFT_ROWS 64     /* of a sequence, at most */

/* A rotation: the first `rot` dimensions of a head turn in pairs, (i, i + rot/2)
 * or, interleaved, (2i, 2i + 1), by the angle pos * w_i; both results are
 * multiplied by `factor`.  turn[i] is w_i / 2 pi as a 64-bit fraction, so that
 * pos * turn[i] modulo 2^64 is the fraction of a turn, however far the
 * position.  Filled by the two functions below; rot 0 turns nothing. */
typedef struct {
    int      rot, interleaved;
    double   factor;
    uint64_t turn[64];
} ecu_rope;
/* w_i = base^(-2i/rot), and of those, for contexts longer than the trained
 * `context`:  LINEAR  w_i / factor;  BANDS  pairs of fewer than `slow` turns
 * over `context` w_i / factor, of more than `fast` w_i, between them a blend
 * linear in the number of turns;  YARN  the same blend linear in the pair's
 * number i, between the (rounded) numbers at which pairs turn `fast` and `slow`
 * times, and the result's factor 0.1 ln(factor) + 1. */
enum { ECU_ROPE_PLAIN = 0, ECU_ROPE_LINEAR = 1, ECU_ROPE_BANDS = 2, ECU_ROPE_YARN = 3 };
int  ecu_rope_init(ecu_rope *r, int rot, int interleaved, double base, int scaling, double factor, double context,
                   double slow, double fast);
/* The caller's own frequencies, radians a position, rot / 2 of them. */
int  ecu_rope_set(ecu_rope *r, int rot, int interleaved, const double *freq, double factor);

/* ecu_kv_append of keys that are turned by their positions on the way, and of
 * the queries beside them (q NULL: none): q_out row r = row r of q, turned.
 * Row r of a sequence that gets n_new[i] rows is written at position len -
 * n_new[i] + r and turned by the position len - n_new[i] + depth[r] (depth:
 * device, one number for each row of the call; NULL: r), len read on the device
 * when the call runs.  A key is turned to some 46 bits and quantised from
 * them, so that its code is that of the exact value (but for about one in
 * 10^12); one that passes fp32's range on the way (values near 2^127) reads as
 * NaN.  A query is turned in 32 bits and rounded once to `dtype`.  q_out may be
 * q with its stride; else it is apart from the rows read.  Everything else as
 * in ecu_kv_append. */
int  ecu_kv_append_rope(ecu_kv *kv, int layer, const ecu_rope *rope, int dtype, const void *q, const void *k,
                        const void *v, int n_head, long q_stride, long k_stride, long v_stride, const int *seq,
                        const int *n_new, int n, const int *depth, void *q_out, long q_out_stride, int out_dtype,
                        void *k_out, void *v_out, void *stream);

/* Attention of the newest n_new[i] (at most ECU_DRAFT_ROWS) positions of each
 * sequence seq[i] (NULL: slots 0..n-1; no slot twice) in layer `layer`: a row
 * sees every position before them, and of them those whose bit is set in its
 * mask (mask: device, one word for each row of the call, bit j its sequence's
 * j-th drafted row; NULL: itself and those before it).  q and out: rows of
 * consecutive sequences one after the other, as in ecu_kv_attend.  A row that
 * sees nothing becomes zeros.  A position that a row sees and that is not
 * finite in K makes the row NaN, one in V its block of 32 dimensions; positions
 * that it does not see have no effect (but for values past 2^15, see below).
 * ws: ecu_kv_tree_ws_bytes() bytes of
 * device memory that no other call uses at the same time; NULL: the pool's own
 * for this stream, as in ecu_kv_attend, but of the first stream too made on its
 * first call (some 20 MB).  out and q do not overlap.  The lengths
 * are read on the device when the call runs, so a captured call follows its
 * sequences.  Sums and the softmax
 * are fp32; of fp32 queries, and of their weights, 22 bits count; the weights of
 * 16-bit queries are rounded to fp16's 11.  Calls of many columns (rows times
 * query heads of a KV head, some 32 and more) of 16-bit queries and 64- or
 * 128-wide heads see keys and values rounded to 11 bits too, as the prompts of
 * a batch do.  Whether a call does goes by an estimate of its time over all of
 * its sequences, as does how they are cut among the SMs: so a sequence's last
 * bits are the same in every call of the same lists and lengths, but may differ
 * beside other sequences, and in a captured call.  Where a call of many columns
 * meets a position whose values pass 2^15, a drafted one that a row does not see
 * too, all rows of the sequence take keys and values from that unit of 128
 * positions on with scales rounded to multiples of 2^-20 (a value is off by
 * 2^-18 more at most).  Rows of large scores stay finite; where a row's largest
 * passes some 2^22 in size, in a call of many columns, its scores count as if
 * divided by the power of two that brings it below (their own rounding is of that
 * size).
 * Every wait in the kernel is bounded (ecu_set_wait_ns): where one gives up, the
 * call's rows mean nothing, and ecu_attn_prompt_status reports it. */
int    ecu_kv_attend_tree(ecu_kv *kv, int layer, int dtype, const void *q, void *out, int n_head, long q_stride,
                          long out_stride, const int *seq, const int *n_new, int n, const uint64_t *mask, float scale,
                          void *ws, void *stream);
size_t ecu_kv_tree_ws_bytes(const ecu_kv *kv);

/* Drafted tokens held against the target's probabilities with given random
 * numbers.  Sequence i has n_row[i] (at most ECU_DRAFT_ROWS) consecutive rows:
 * logits [n_vocab] (at most 2^30; `dtype`, rows `stride` elements apart), the token of each
 * row and its parent, an earlier row of the sequence (row 0's are not looked
 * at).  From row 0 on, rows are tried in order: one that hangs on the current
 * row, with token x, is accepted where u[row] q(x) F < f(x), and becomes the
 * current one.  f is softmax(logits / temperature) of the current row, F its
 * sum, q the distribution that its children were drawn from: row `current` of
 * draft (fp32, rows draft_stride apart), or 1 where draft is NULL (the drafter
 * does not draw).  A rejected row leaves f <- max(f / F - q, 0), or f(x) <- 0.
 * At the end next[i] is the first x with f(x) > 0 whose running sum passes
 * u_next[i] F; where nothing is left of f (so that no later row was accepted
 * either) f is softmax(logits / temperature) again for that.  A temperature (one a sequence; NULL: 1) that is not above 0
 * takes the first of the largest logits instead, and accepts it alone.
 * Everything compared is 64-bit.  A token outside the vocabulary is not tried.
 * A row whose logits hold a NaN or +infinity, or -infinity alone, ends the walk
 * with next[i] = -1 when it becomes the current one.
 * kept: the accepted rows, numbered within their sequence, row 0 first, in the
 * first n_kept[i] of the sequence's n_row[i] words, -1 in the others; a
 * sequence without rows has n_kept 0 and next -1.  All but n_row are device
 * memory. */
int  ecu_draft_verify(int dtype, const void *logits, long stride, int n_vocab, const float *draft, long draft_stride,
                      const int *token, const int *parent, const int *n_row, int n, const float *u, const float *u_next,
                      const float *temperature, int *kept, int *n_kept, int *next, int device, void *stream);

/* Of the newest n_new[i] positions of sequence seq[i] (no slot twice) the
 * n_kept[i] rows named in `kept` (host, the sequences' lists one after the
 * other; rising numbers below n_new[i]) stay, moved together behind the
 * positions before them in every layer; the others are given back as by
 * ecu_kv_truncate.  Positions that rows move to must lie in the sequence's own
 * pages.  A change of the pool like those above. */
int  ecu_kv_keep(ecu_kv *kv, const int *seq, const int *n_new, const int *kept, const int *n_kept, int n, void *stream);

/* ---- packed prompts ------------------------------------------------------- */

/* Causal attention of packed prompts, on the tensor cores: sequence s has
 * query rows cu_q[s] .. cu_q[s+1]-1 and key/value rows cu_k[s] .. cu_k[s+1]-1
 * (host arrays of n_seq + 1 non-decreasing offsets from 0; cu_k NULL: the
 * queries').  The last query sees every key of its sequence, each earlier one
 * one key less; a row that sees none becomes zeros.  q, k, v, out: device,
 * `dtype` (ECU_F16 or ECU_BF16), 16-byte aligned, a row's heads one after the
 * other, rows a multiple of 8 elements apart; head_dim 64 or 128; scale > 0.  What lies
 * behind the last row, or in keys that a row does not see (NaN and infinities
 * too), has no effect.  Sums and the softmax are fp32, relative to weights of
 * up to 2^8 (bf16 values near 2^127 / 2^8 / keys can pass fp32's range); the
 * weights are rounded to `dtype` before their product with V; scores past some
 * 2^22 count as in ecu_kv_attend_tree's calls of many columns.  out overlaps
 * none of the others.
 * Every wait in the kernel is bounded (ecu_set_wait_ns): one that gives up
 * leaves rows of NaN, which ecu_attn_prompt_status reports. */
int  ecu_attn_prompt(int dtype, const void *q, const void *k, const void *v, void *out, int n_head, int n_head_kv,
                     int head_dim, long q_stride, long k_stride, long v_stride, long out_stride, const int *cu_q,
                     const int *cu_k, int n_seq, float scale, int device, void *stream);
/* Waits for the stream; -1 where a wait of an ecu_attn_prompt or
 * ecu_kv_attend_tree call on `device` has given up since this was last asked
 * (until then, waits of later calls that take longer than a millisecond give up
 * with it), or the status cannot be read.  The calls inside ecu_batch_feed and ecu_prefill report
 * through those. */
int  ecu_attn_prompt_status(int device, void *stream);

/* ---- many sequences over one model (serving) ---- */

/* Sequences with the weights of a FULL context and their K/V in a pool of
 * 4-bit pages: prompts and single tokens of any of them in one call.  No
 * counterpart in the reference, which serves one sequence a process
 * (src/daemon.c:757).  For models of head_dim 64 or 128 whose embedding and
 * feed-forward widths are multiples of 8 and whose Q, K and V, and gate and
 * up, share a format of the fast layouts (as the persistent step wants), of
 * any n_ctx; others are refused, and so are tensor-parallel and staged
 * contexts.  n_seq slots of the base's n_ctx positions, n_pages pages
 * of ECU_KV4_PAGE positions between them.  The base may be closed first. */
typedef struct ecu_batch ecu_batch;
int  ecu_batch_open(ecu_batch **out, ecu_ctx *base, int n_seq, int n_pages, char *err, size_t errlen);
void ecu_batch_close(ecu_batch *b);
/* The batch's pool, to fork, truncate and free its sequences and to compact
 * it (ecu_kv_*), on the batch's stream. */
ecu_kv *ecu_batch_kv(ecu_batch *b);
void   *ecu_batch_stream(ecu_batch *b);
/* Sequence seq[i] (no slot twice) takes the next n_tok[i] >= 1 of `tokens`
 * at its end; picked[i] is the token that its last position's head picks
 * (llm_pick's rule), logits (NULL: none wanted; host, n rows of n_vocab) that
 * head's output.  The rows of all sequences go through the layers together
 * (ecu_prefill's GEMMs; a few single tokens alone as the decode step's
 * matrix-vector products); a sequence with one token attends through
 * ecu_kv_attend, the others through ecu_attn_prompt (in fp16: 11 bits of each
 * operand and weight), all to keys and values as the cache holds them.  So a
 * prompt leaves nearly the same state however it is cut, but not the same
 * bits: where a key or value lies at the border of two 4-bit codes, the
 * paths' rounding can decide it either way, and later layers follow.  Against
 * the fp32 cache of ecu_forward the states differ by the cache's 4-bit
 * rounding.  Prompts' queries, keys and values, and the
 * attention rows of more than 16 single tokens, go through fp16: a finite one
 * past 65504 in magnitude fails the feed (fed alone, single tokens reach what
 * the cache holds, 8 * 65504).  On an error the sequences keep what they
 * held.  Synchronises the batch's stream. */
int  ecu_batch_feed(ecu_batch *b, const int *seq, const int *n_tok, int n, const int *tokens, int *picked, float *logits);

/* ---- failure-path testing ------------------------------------------------ */

/* No counterpart in the reference, whose failure paths are host retries and
 * aborts (src/shard.c:533-545).  Every wait inside the engine's kernels (a
 * tagged word from another CTA or rank, a bulk copy's barrier) is bounded:
 * after the limit it sets the context's status word and lets the kernel run
 * to its end, and the step returns -1.  ecu_set_wait_ns sets that limit on
 * `device` (default 2 s; between launches).  ecu_inject_wait_timeout makes
 * the next persistent step of `c` wait, in its first GEMV phase with a
 * tagged input, for an input word that no phase writes: its waits run out,
 * that step returns -1 with the timeout in ecu_last_error, and the context
 * steps normally again afterwards (reset it: that step's cache row is not
 * valid).  -1 for a context on the per-kernel step.  ecu_inject_late_warp:
 * in the next persistent step of `c` (4 query heads of 128 a KV head, one
 * GPU) one warp of every block comes 10 us late to each phase, which changes
 * nothing but the step's time.
 * ecu_inject_prompt_timeout: the next prompt attention on `device`
 * (ecu_attn_prompt, or inside ecu_batch_feed or ecu_prefill) never copies its
 * first keys, so that its waits run out: ecu_attn_prompt_status, or the call
 * around it, returns -1.  ecu_inject_tree_timeout: the same of the next
 * ecu_kv_attend_tree that runs on the tensor memory.  ecu_inject_tree_registers:
 * the next one that would finds its kernel compiled to other registers than
 * its roles share, and runs on the other.  ecu_kv_inject_failure: of the
 * launches with which the next change of the pool updates the device (a pool
 * without one counts them alike), number `launch`, from 0, fails. */
int  ecu_set_wait_ns(int device, unsigned long long ns);
int  ecu_inject_wait_timeout(ecu_ctx *c);
int  ecu_inject_late_warp(ecu_ctx *c);
int  ecu_inject_prompt_timeout(int device);
int  ecu_inject_tree_timeout(int device);
int  ecu_inject_tree_registers(int device);
int  ecu_kv_inject_failure(ecu_kv *kv, int launch);

/* ---- measurement --------------------------------------------------------- */

/* Quantised-matvec microbenchmark (the reference's matvec,
 * src/engine.c:277-357, timed on the device): `copies` device copies of one
 * n_out x n_in matrix of raw GGUF blocks (host array w_raw, repacked into
 * the layouts the engine keeps), then `rounds` replays of a CUDA graph of
 * one launch of y = W_c x per copy, back to back; *ms_per_launch = CUDA
 * event time / launches.  Enough copies to exceed the L2 make every launch
 * stream its matrix from HBM.  y (host) = the last launch's output. */
int  ecu_matvec_bench(unsigned ggml_type, const void *w_raw, int n_in, int n_out, const float *x,
                      float *y, int device, int copies, int rounds, double *ms_per_launch);

/* The same matrices streamed through the persistent step's GEMV phases: one
 * cooperative launch runs one phase per copy (y = W_c x, plain x, each CTA's
 * rows through its shared-memory ring, the next copy's rows already in
 * flight while a phase ends), `rounds` launches timed with CUDA events;
 * *ms_per_matvec = time / (rounds * copies).  The decode step consumes its
 * weight matrices this way.  Q4_0 / Q8_0 / Q4_K with n_in a multiple of
 * 1024 (the fast layouts); -1 otherwise. */
int  ecu_matvec_stream_bench(unsigned ggml_type, const void *w_raw, int n_in, int n_out, const float *x,
                             float *y, int device, int copies, int rounds, double *ms_per_matvec);

/* Per-kernel-kind totals of a profiling replay. */
typedef struct {
    char   kind[32];          /* "gemv_gate_up", "attention", ...               */
    int    launches;
    double total_ms;          /* sum of CUDA-event durations of those launches  */
    double bytes_per_launch;  /* algorithmic bytes: weights as stored in the
                                 file + vectors read and written                 */
} ecu_kprof;

/* One persistent step with every CTA's time (globaltimer ns) at the start
 * and at the end of each phase: out[(p + 1) * grid + cta] = the end of
 * phase p, out[cta] = the start; n_words >= (phases + 1) * grid (*grid =
 * the CTA count, the SM count).  kinds (optional) receives the phases'
 * names, comma-separated.  Returns the number of phases, or -1.  The
 * position advances as in a step.  For measuring the CTAs' skew at phase
 * boundaries. */
int  ecu_profile_cta_ns(ecu_ctx *c, unsigned long long *out, size_t n_words, int *grid, char *kinds,
                        size_t kinds_len);
/* Run n_steps decode steps of a FULL (or LAYERS) context without the graph,
 * with a pair of CUDA events around every kernel on the context's stream,
 * and aggregate the durations per kernel kind into out[0..max_kinds).  The
 * steps are real decode steps (the position advances).  Returns the number
 * of kinds written, or -1. */
int  ecu_profile_steps(ecu_ctx *c, int n_steps, ecu_kprof *out, int max_kinds);

/* ---- misc -------------------------------------------------------------- */

const char *ecu_last_error(void);
/* Number of kernels this process has launched through the engine. */
uint64_t ecu_kernel_launches(void);
/* Library version string. */
const char *ecu_version(void);

#ifdef __cplusplus
}
#endif
#endif
