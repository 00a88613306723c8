/*
 * quanta_hip.h — C-ABI of the MI355X (gfx950) quantized matmul path.
 *
 * Drop-in boundary under the reference's L1 kernels (engine/src/ops.h) and its shortlist head
 * (engine/src/model.cpp:240-334). Plain pointers and sizes only. Every function returns a status
 * (QH_OK = 0); on failure qh_last_error() gives a message for the calling thread.
 *
 * Memory: every tensor, activation and output pointer below is a DEVICE pointer unless the
 * parameter name ends in _host. `stream` is a hipStream_t (NULL = the null stream). Calls only
 * enqueue work; nothing synchronises unless the function says so. Functions are reentrant and may
 * be called from any host thread; the only shared state is the per-device init record.
 *
 * Block layouts are the .qnt layouts, unchanged (reference engine/src/model_file.h:16-38,
 * scripts/export.py:10-13):
 *   Q8_0 [rows][cols]: int8 quants [rows*cols], then fp16 scales [rows*cols/32]
 *   Q4_0 [rows][cols]: packed nibbles [rows*cols/2] (per 32-block, byte j = (q[j]+8) | (q[j+16]+8)<<4),
 *                      then fp16 scales [rows*cols/32]
 *   quantized activation (QuantVec, ops.h:47-51): int8 q[cols], f32 d[cols/32]
 * Results are bit-identical to the reference's scalar kernels (ops_ref.cpp) on the same inputs.
 */
#ifndef QUANTA_HIP_H
#define QUANTA_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. */
enum {
    QH_OK = 0,
    QH_ERR_ARG = 1,         /* null pointer, bad count or range */
    QH_ERR_DTYPE = 2,       /* dtype not allowed for this call */
    QH_ERR_SHAPE = 3,       /* cols % 32 != 0, mismatched tensors, size limits */
    QH_ERR_ALIGN = 4,       /* device pointer not 16-byte aligned */
    QH_ERR_HIP = 5,         /* a HIP runtime call failed */
    QH_ERR_NOMEM = 6,       /* workspace too small / allocation failed */
    QH_ERR_UNSUPPORTED = 7  /* e.g. top_k beyond the supported maximum */
};

/* Tensor dtypes, numbered as the .qnt file stores them (reference model_file.h:16, DType). */
enum { QH_F32 = 0, QH_F16 = 1, QH_Q8_0 = 2, QH_Q4_0 = 3 };

/* A device-only layout, never a .qnt dtype: a Q8_0 [rows][cols] head as nibble planes (qh_head_planes), the same
 * int8 values q = 16 h + l with h = floor(q / 16) in [-8, 7] and l = q - 16 h in [0, 15], in as many bytes as the
 * Q8_0 tensor: the high plane [rows][cols/2] (Q4_0 blocks of the codes h + 8), the low plane [rows][cols/2] (Q4_0
 * blocks of l, no offset), then the Q8_0 fp16 scales [rows][cols/32] unchanged. The shortlist head screens with the
 * high plane alone (reference research/head_deep.py:68-78, docs/PROGRESS.md:121-130). */
enum { QH_Q8_0_PLANES = 16 };

/* Quantization block size (reference model_file.h:17, QK). */
#define QH_QK 32

/* Device view of a .qnt tensor (reference model_file.h:27-38, Tensor): `data` is the device
 * address of the quant section; for Q8_0 / Q4_0 the fp16 scales follow at data + quant bytes. */
typedef struct qh_tensor {
    int32_t dtype;
    int32_t rows;
    int32_t cols;
    const void* data;
} qh_tensor;

/* Message of the last failed call on this thread ("" if none). */
const char* qh_last_error(void);

/* Library version string. */
const char* qh_version(void);

/* Selects `device` for the calling thread and records its properties (idempotent).
 * Replaces: nothing (the reference has no device); called once before the others. */
int qh_init(int device);

/* Size in bytes of the quant section (reference model_file.cpp:29-38, Tensor::quant_bytes). */
size_t qh_quant_bytes(int dtype, int rows, int cols);

/* Quant section plus scale section. */
size_t qh_tensor_bytes(int dtype, int rows, int cols);

/* Checks a tensor view: dtype, shape, cols % 32 and 16-byte alignment of `data`. */
int qh_validate_tensor(const qh_tensor* W);

/* Thin device-memory helpers so C/C++ callers need no HIP headers. */
int qh_malloc(void** ptr, size_t bytes);

/* Forced allocation failure, for tests of the error paths: after `after` more device allocations by the library
 * (qh_malloc and the decoder's own buffers), the next one fails with QH_ERR_NOMEM before any HIP call, and the hook
 * disarms itself; after < 0 disarms it. Process-wide. No counterpart in the reference: it is the fault hook its
 * failure handling is tested with (an allocation failure maps to an error code, nothing is leaked). */
int qh_fault_alloc(int after);
int qh_free(void* ptr);
int qh_memcpy_h2d(void* dst, const void* src_host, size_t bytes, void* stream); /* async */
int qh_memcpy_d2h(void* dst_host, const void* src, size_t bytes, void* stream); /* synchronous */
int qh_memset(void* dst, int value, size_t bytes, void* stream);
int qh_stream_sync(void* stream);
int qh_stream_create(void** stream); /* non-blocking stream at the default priority */
int qh_stream_destroy(void* stream);

/* Per-32-block int8 quantization of n_tok activation rows of length n (x is [n_tok][n] f32):
 * q [n_tok][n] int8, d [n_tok][n/32] f32.
 * Replaces: void quantize_q8(const float* x, int n, QuantVec& out)   (reference ops.h:52,
 *           implementation ops_ref.cpp:69-83), once per token row. */
int qh_quantize_q8(const float* x, int n_tok, int n, int8_t* q, float* d, void* stream);

/* Decode GEMV: out[r] = W[r,:] . x for r in [r0, r1) (out indexed by absolute row), W Q8_0 or Q4_0,
 * x = (xq [cols] int8, xd [cols/32] f32). Per row: int32 block dots, then the serial chain
 * acc = fma(float(s_b) * dw_b, dx_b, acc) in block order.
 * Replaces: void matvec_q(float* out, const Tensor& W, const QuantVec& x, int r0, int r1)
 *           (reference ops.h:61, MatvecQFn ops.h:57; implementation ops_ref.cpp:85-120). */
int qh_matvec_q(float* out, const qh_tensor* W, const int8_t* xq, const float* xd, int r0, int r1,
                void* stream);

/* GEMV over unquantized weights: out[r] = W[r,:] . x for r in [r0, r1), W F32 or F16 ([rows][cols] row-major, cols
 * a multiple of 32), x [cols] f32. Per row the serial chain acc = fma(w_i, x_i, acc) from +0 in column order (the
 * reference build's contraction of acc += w * x; an F16 weight is converted exactly).
 * Replaces: void matvec_ref(float* out, const Tensor& W, const float* x, int r0, int r1) for F32 / F16 W
 *           (reference ops.h:43, implementation ops_ref.cpp:8-27: Model::linear's path for an unquantized W,
 *           model.cpp:154-156). */
int qh_matvec_ref(float* out, const qh_tensor* W, const float* x, int r0, int r1, void* stream);

/* Prefill matmul for n tokens: out[t*ldo + r] for t in [0, n), r in [r0, r1); xq is [n][cols]
 * int8, xd is [n][cols/32] f32 (the n QuantVecs back to back). Every (row, token) value is
 * bit-identical to qh_matvec_q on that token (int8 MFMA, K = 32 per instruction = one block).
 * Replaces: void matmul_q(float* out, int ldo, const Tensor& W, const QuantVec* x, int n, int r0,
 *           int r1) (reference ops.h:69, MatmulQFn ops.h:68; implementation ops_ref.cpp:122-160). */
int qh_matmul_q(float* out, int ldo, const qh_tensor* W, const int8_t* xq, const float* xd, int n, int r0,
                int r1, void* stream);

/* Workspace bytes qh_argmax needs for n logits (0 if n <= 0); no initialisation needed. */
size_t qh_argmax_workspace_bytes(int n);

/* First index of the maximum of logits[0, n) written to *index (device int32). Calls that overlap must not
 * share a workspace.
 * Replaces: the greedy branch of Sampler::sample, std::max_element (reference sampler.cpp:35-37). */
int qh_argmax(const float* logits, int n, int32_t* index, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------ Exact Shortlist Head */

/* Which logits the caller needs (reference model.h:24-29, HeadQuery). `must` is a DEVICE array of
 * n_must ids. top_k must be in [1, QH_HEAD_MAX_TOPK]. */
typedef struct qh_head_query {
    int32_t top_k;
    int32_t n_valid; /* ids >= n_valid are ignored; 0 = whole vocab */
    const int32_t* must;
    int32_t n_must;
} qh_head_query;

#define QH_HEAD_MAX_TOPK 256 /* seeds = top_k + 8 (the sampler's survivor limit, QH_SAMPLE_MAX_TOPK) */

/* Device-side summary of one shortlist call. */
typedef struct qh_head_stats {
    int32_t top1;       /* first argmax of logits over [0, n_valid) (greedy token) */
    int32_t n_rows;     /* 8-bit rows rescored (reference Model::last_head_rows) */
    int32_t n_seeds;    /* seeds rescored first */
    int32_t n_cand;     /* candidates: upper bound >= tau */
    int32_t n_must;     /* must ids rescored */
    int32_t seed_tie;   /* 1 if the last seed's coarse score ties an unselected eligible row */
    float tau;          /* k-th best exact seed logit (-inf if fewer than k seeds) */
    float top1_logit;   /* logits[top1] */
} qh_head_stats;

/* Outputs of qh_shortlist_head, all device buffers owned by the caller. */
typedef struct qh_head_out {
    float* logits;        /* [V]: exact logit for rescored rows, -inf elsewhere */
    float* coarse;        /* [V]: 4-bit score (reference Model::head_coarse) */
    float* upper;         /* [V]: coarse + error bound (reference Model::head_upper) */
    int32_t* rows;        /* [V + n_must]: rescored rows: seeds (best coarse first), then candidates
                             (unordered), then must ids */
    qh_head_stats* stats; /* one record */
} qh_head_out;

/* Workspace bytes qh_shortlist_head needs for a V x D head and top_k (0 if unsupported: D must be a multiple
 * of 64 and at most 4096, V at most 1,048,576 on a 256-CU GPU). The workspace needs no initialisation (each call
 * resets what it uses); calls that overlap must not share one. */
size_t qh_shortlist_workspace_bytes(int V, int D, int top_k);

/* Exact Shortlist Head on one quantized hidden state (xq [D] int8, xd [D/32] f32):
 * 4-bit screen of all V rows with bound = fma(sum_b fma(err_b, xnorm_b), 1.001, 1e-5); seeds = the
 * top_k+8 best eligible coarse scores (lower row first on ties), rescored exactly; tau = k-th best
 * exact seed; candidates {r < n_valid, not seed or must, upper[r] >= tau} and must ids rescored
 * exactly; then the greedy argmax. head8 Q8_0 [V][D], head4 Q4_0 [V][D], err F16 [V][D/32].
 * Replaces: void Model::shortlist_head(const HeadQuery&) (reference model.cpp:240-334) followed by
 *           the greedy sample (sampler.cpp:35-37). */
int qh_shortlist_head(const qh_tensor* head8, const qh_tensor* head4, const qh_tensor* err, const int8_t* xq,
                      const float* xd, const qh_head_query* query, const qh_head_out* out, void* workspace,
                      size_t workspace_bytes, void* stream);

/* Bytes of the scratch array qh_shortlist_head_noalloc works in: one array in each GPU's memory, held by the library
 * until the process ends. Enough for the 151,936-row Qwen2.5 head (0.78 MB, the same at every top_k) and
 * for heads up to about 800,000 rows of 896. */
#define QH_NOALLOC_SCRATCH_BYTES ((size_t)4 << 20)

/* qh_shortlist_head with the same arguments and results but no workspace argument, and no device allocation of any
 * kind: its workspace is the library's scratch array on the current GPU. Fails with QH_ERR_NOMEM, launching nothing,
 * when qh_shortlist_workspace_bytes(V, D, top_k) exceeds QH_NOALLOC_SCRATCH_BYTES. Every call on one GPU works in that
 * GPU's one array, which keeps the last call's contents (the kernels reset what they read, so nothing of one call
 * reaches the next): calls in order on one stream are fine, calls that overlap on one GPU (two streams, or two host
 * threads without an order between them) race and give wrong results. The first call on a device runs qh_init for it
 * (device checks and the scratch array's address); under HIP graph capture, call qh_init for the device (or this entry
 * point once, eagerly) before the capture begins, so that the captured call only launches kernels.
 * No counterpart in the reference (its Model allocates the head's state on the host at load): for callers that cannot
 * allocate device memory, such as code under HIP graph capture, tight serving loops and harnesses that forbid
 * hipMalloc. */
int qh_shortlist_head_noalloc(const qh_tensor* head8, const qh_tensor* head4, const qh_tensor* err, const int8_t* xq,
                              const float* xd, const qh_head_query* query, const qh_head_out* out, void* stream);

/* The nibble-plane layout of a Q8_0 [V][D] head (D a multiple of 64): writes qh_tensor_bytes(QH_Q8_0_PLANES, V, D)
 * bytes (the Q8_0 tensor's size) at `planes`, a 16-byte aligned DEVICE buffer that must not overlap head8's data.
 * The caller may free the Q8_0 copy afterwards: the planes hold the same values, so the exact rows (and an embedding
 * lookup) can be read from them.
 * Replaces: the research layout "the Q8 ints stored as two nibble planes" (reference research/head_deep.py:8-10,
 *           68-78; docs/PROGRESS.md:121-130); the reference engine keeps the Q8_0 head and a separate Q4_0 copy. */
int qh_head_planes(const qh_tensor* head8, void* planes, void* stream);

/* The Exact Shortlist Head over a nibble-plane head alone (planes: QH_Q8_0_PLANES [V][D]), with no extra copy:
 * the screen reads the high plane and the scales (coarse = the chain acc = fma(float(sum_i (16 h_i + 8) x_i) * d_b,
 * dx_b, acc), the values at the midpoints of their high-nibble buckets; bound = fma(sum_b fma(d_b, (8 dx_b) *
 * sum_i |x_i|), 1.001, 1e-5), since |q - (16 h + 8)| = |l - 8| <= 8), then the same seeds, tau, candidates, must ids
 * and greedy argmax as qh_shortlist_head; exact rows are rebuilt from both planes, so every rescored logit is
 * bit-identical to the full Q8_0 head's. Outputs and workspace as qh_shortlist_head
 * (qh_shortlist_workspace_bytes(V, D, top_k)).
 * Replaces: the scope's nibble-plane shortlist variant (reference research/head_deep.py:68-78 "hi4, analytic
 *           bound", docs/PROGRESS.md:121-130) run through Model::shortlist_head's procedure (model.cpp:240-334). */
int qh_shortlist_planes(const qh_tensor* planes, const int8_t* xq, const float* xd, const qh_head_query* query,
                        const qh_head_out* out, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------ sampler */

/* The reference's SamplerParams (sampler.h) without the seed: the generator state lives in device memory. */
typedef struct qh_sampler_params {
    float temperature;    /* <= 0: greedy (first maximum after the penalty) */
    int32_t top_k;        /* 0 = disabled */
    float top_p;          /* 1 = disabled */
    float min_p;          /* 0 = disabled */
    float repeat_penalty; /* 1 = disabled; divides positive logits, multiplies negative ones (HF semantics) */
    int32_t repeat_window; /* how many recent history ids the penalty looks at; 0 = all */
} qh_sampler_params;

#define QH_SAMPLE_MAX_TOPK 256       /* survivors of the top-k cut qh_sample handles without a workspace */
#define QH_SAMPLE_MAX_VOCAB 262144   /* n_valid limit (the history bitmap lives in LDS) */

/* The generator state a reference Sampler constructed with a nonzero seed starts from (sampler.cpp:10-13). */
uint64_t qh_sampler_state(uint64_t seed);

/* One draw of Sampler::sample (sampler.cpp:22-85) on DEVICE logits: repetition penalty over the distinct ids of the
 * history window, then greedy, or top-k, softmax with temperature, min-p, top-p and a draw from the xorshift64*
 * generator whose state is the DEVICE uint64 *state (advanced by one draw when temperature > 0). The chosen id goes
 * to the DEVICE int32 *out_id. The logits are not modified (the reference samples from its own copy).
 *   rows / head_stats: the shortlist head's row list and stats (qh_shortlist_head's out.rows / out.stats), the only
 *                      ids whose logits are finite; NULL / NULL to consider every id below n_valid.
 *   history[0, n_hist): DEVICE token history (the session's prompt and generated ids), NULL when n_hist is 0.
 * Requires 1 <= n_valid <= QH_SAMPLE_MAX_VOCAB and, with temperature > 0, min(top_k or n_valid, n_valid) <=
 * QH_SAMPLE_MAX_TOPK (qh_sample_ws takes any number, and over full logits of tens of thousands of ids is several times
 * as fast for any top_k). Ties between equal logits in the top-k go to the lower id
 * (unspecified in the reference).
 * Replaces: Sampler::sample (reference sampler.cpp:22-85) and Sampler's generator (sampler.cpp:10-21). */
int qh_sample(const float* logits, int32_t n_valid, const int32_t* rows, const qh_head_stats* head_stats,
              const int32_t* history, int32_t n_hist, const qh_sampler_params* params, uint64_t* state,
              int32_t* out_id, void* stream);

/* qh_sample with a DEVICE workspace of qh_sample_workspace_bytes(n_valid) bytes (16-byte aligned). Over full logits
 * (rows NULL) of 8,192 ids and more the whole GPU first finds the largest of each group of 256 ids, and one workgroup
 * then reads only the groups that can hold a survivor: 151,936 ids at top_k 20 take 20 us, 72 without a workspace
 * (greedy draws from 16,384 ids on: 6 and 32). It also lifts the QH_SAMPLE_MAX_TOPK limit: any top_k, top_k 0 (every id
 * a survivor) included. More survivors than that are sorted by a device-wide radix sort (4 passes over the logit half);
 * the softmax sum, top-p, total and draw then run in the reference's order and stop where the remaining terms can no
 * longer change a rounded result. Any call may write the workspace: calls that share one must not overlap. Replaces: Sampler::sample (reference sampler.cpp:22-85) with top_k 0 or large. */
size_t qh_sample_workspace_bytes(int32_t n_valid);
int qh_sample_ws(const float* logits, int32_t n_valid, const int32_t* rows, const qh_head_stats* head_stats,
                 const int32_t* history, int32_t n_hist, const qh_sampler_params* params, uint64_t* state,
                 int32_t* out_id, void* ws, size_t ws_bytes, void* stream);

/* ------------------------------------------------------------------ 8-bit paged key / value cache */

/* A key / value cache in 8 bits for many sequences, in pages that sequences may share. A block is 16 tokens of one KV
 * head, keys and values apart: int8 codes and one f32 scale d, which stand for code * d. A page holds page_tokens tokens
 * of every KV head (its layout is the library's own; qh_kv8_read gives values back). One page number names the same
 * tokens in every layer. All memory is the caller's; the calls below only enqueue work, take no memory of their own and
 * can be captured in a HIP graph (the lists they read are DEVICE arrays, read when the work runs). Calls that change one
 * cache have to be in order; calls that overlap must not share a workspace.
 * No counterpart in the reference, whose cache holds one sequence in f16 or f32 (model.cpp:96-104, 197-204). */
#define QH_KV8_BLOCK 16
#define QH_KV8_MAX_SEQS 32768
#define QH_KV8_MAX_PAGES (1 << 20)

typedef struct qh_kv8_cache {
    void* pages;     /* [n_layers][n_pages][qh_kv8_page_bytes(page_tokens, n_kv_heads, head_dim)], 16-byte aligned */
    int32_t* table;  /* [n_seqs][seq_pages]: the page of a sequence's tokens [j * page_tokens, (j + 1) * page_tokens) */
    int32_t* lens;   /* [n_seqs]: tokens of the sequence */
    int32_t* refs;   /* [n_pages]: how many sequences hold the page; 0: free */
    int32_t* status; /* one: QH_KV8_* bits that calls on this cache have set (cleared by qh_kv8_reset or the caller) */
    int32_t n_layers, n_pages;
    int32_t page_tokens; /* a power of two, 16 to 256 */
    int32_t n_kv_heads; /* at most 256 */
    int32_t head_dim; /* 64 or 128 */
    int32_t n_seqs, seq_pages;
} qh_kv8_cache;

/* Bits of *status. */
enum {
    QH_KV8_NO_PAGES = 1, /* resize or fork: too few free pages */
    QH_KV8_BAD_LIST = 2, /* a sequence number or length out of range, or a sequence named twice: the call did nothing */
    QH_KV8_SHARED = 4    /* append: tokens in a page that other sequences hold were not stored */
};

/* Bytes of one page (0 for an unsupported shape). */
size_t qh_kv8_page_bytes(int page_tokens, int n_kv_heads, int head_dim);

/* Every page free, every sequence empty, status 0 (page contents are left). A new cache's state arrays need it. */
int qh_kv8_reset(const qh_kv8_cache* c, void* stream);

/* Workspace bytes of qh_kv8_resize, qh_kv8_fork and qh_kv8_compact (16-byte aligned, no initialisation). */
size_t qh_kv8_pages_workspace_bytes(const qh_kv8_cache* c);

/* Sequence seqs[i] gets length lens[i] (DEVICE arrays of n; each sequence once), for every i of the list at once. First
 * the shorter ones give back the pages past their new length (0: all of them); then the longer ones take the lowest free
 * pages, in the list's order. A last page that is partly filled and also held by other sequences is replaced by a copy of
 * it when its sequence grows, so that new tokens go into the sequence's own page. With fewer free pages than the longer
 * ones need, none of them grows and QH_KV8_NO_PAGES is set. Tokens between the old and the new length have no values
 * until qh_kv8_append stores them. */
int qh_kv8_resize(const qh_kv8_cache* c, const int32_t* seqs, const int32_t* lens, int n, void* workspace,
                  size_t workspace_bytes, void* stream);

/* Sequence dst[i] becomes a fork of src[i] (DEVICE arrays of n; each dst once and in no place of src): its pages are
 * given back, and it holds src[i]'s tokens: src[i]'s pages, shared (copy 0), or copies of them in the lowest free pages
 * (copy 1; with too few of them every listed dst stays empty and QH_KV8_NO_PAGES is set). */
int qh_kv8_fork(const qh_kv8_cache* c, const int32_t* src, const int32_t* dst, int n, int copy, void* workspace,
                size_t workspace_bytes, void* stream);

/* Sequence dst[i] takes what src[i] held before the call, for every i of the list at once (DEVICE arrays of n; each dst once;
 * dst NULL: sequence i): a beam search's sequences become those of the beams that are continued. src may name sequences of
 * dst, any number of times, and -1 leaves its dst empty. Pages are shared; pages that no sequence holds afterwards are free.
 * qh_kv8_resize then gives each sequence room for its next token, with a copy of a partly filled last page that others hold.
 * Workspace: 16-byte aligned, no initialisation; NULL where the size is 0. */
size_t qh_kv8_reorder_workspace_bytes(const qh_kv8_cache* c);
int qh_kv8_reorder(const qh_kv8_cache* c, const int32_t* src, const int32_t* dst, int n, void* workspace,
                   size_t workspace_bytes, void* stream);

/* Moves the pages in use to the front: with L of them, those numbered L and above move, in order, to the free numbers
 * below L, in every layer, and the tables follow. *live (DEVICE, may be NULL) = L: the pages from L on are free. */
int qh_kv8_compact(const qh_kv8_cache* c, int32_t* live, void* workspace, size_t workspace_bytes, void* stream);

/* The ragged batch of the calls below: n entries over n_tok rows. Entry b is the rows [start[b], start[b + 1]) (start:
 * DEVICE [n + 1], ascending; NULL: n == n_tok and one row each), the LAST tokens of sequence seqs[b] (DEVICE [n]; NULL:
 * sequence b), whose length qh_kv8_resize has set before: row i of m is at position lens - m + i. Rows outside
 * the entries are neither read nor written. Entries whose sequence number is out of range are empty sequences. Rows are
 * ld elements apart, a row's heads contiguous; dtype QH_F32 or QH_F16. Bases and row strides: multiples of 16 bytes. */

/* Stores k and v, rows of [n_kv_heads][head_dim], into layer `layer`: per block d = max|x| / 127 (rounded to f32) and
 * the codes nearest to x / d, halves away from zero. A block that holds earlier tokens keeps the larger of its scale and
 * the new ones', and where that grows its codes are rounded to it. An infinite or NaN value makes its block's scale NaN,
 * so that all 16 tokens of that head read as NaN. A scale never falls: where qh_kv8_resize has cut tokens off inside a block,
 * the tokens that stay keep the rounding, or the NaN, that those brought, until the block is stored from its first token
 * again. Each sequence in one entry at most, and its tokens in order: a block's
 * earlier tokens have to be there. Tokens in a page that other sequences hold are left out (QH_KV8_SHARED). */
int qh_kv8_append(const qh_kv8_cache* c, int layer, const void* k, const void* v, int dtype, int64_t ldk, int64_t ldv,
                  const int32_t* start, const int32_t* seqs, int n, int n_tok, void* stream);

/* The stored values of the entries' tokens: code * d rounded to f32, then to dtype. Tokens without a page read as 0; rows
 * before a sequence's first position are left as they are. */
int qh_kv8_read(const qh_kv8_cache* c, int layer, void* k, void* v, int dtype, int64_t ldk, int64_t ldv,
                const int32_t* start, const int32_t* seqs, int n, int n_tok, void* stream);

/* Workspace bytes of a qh_kv8_attention call with n entries over n_tok rows (16-byte aligned, no initialisation; a smaller
 * batch can need more, as it is split further). 0 where it needs none: workspace may be NULL then. */
size_t qh_kv8_attention_workspace_bytes(const qh_kv8_cache* c, int n_heads, int n, int n_tok);

/* Attention of query rows q [n_heads][head_dim] over their sequences: out = sum_j p_j v_j with p = softmax(scale *
 * q . k_j) over the positions j that the row sees: up to its own (causal 1), or the whole sequence (causal 0, for states
 * that are not the queries' own: an entry may then have more rows than the sequence has tokens). Query head h reads KV
 * head h / (n_heads / n_kv_heads). Tokens without a page are left out. A row that sees nothing (an empty
 * sequence, or a position below 0) is 0. out may not
 * overlap q. One kind of kernel takes the whole batch, by its rows and entries together: prompts and single tokens are faster
 * in a call each. A row of q that is not finite gives NaN, and so does a visible token that reads as NaN. Sums in f32; f32
 * queries and weights go through the matrix instructions as two f16 each, and so do the weights of f16 calls, but for
 * prompts (more than 32 rows of a KV head's queries to an entry), whose weights are rounded to one f16: a caller who wants two
 * there too passes the queries in f32. A weight is also held
 * to 2^-31 of the largest product of a token's weight and its block's value scale among the tokens that the row sees and whose
 * stored values are not all zero (storing rounded off up to 2^-1 of that product). Tokens that a row does not see, or gives no
 * weight to, take nothing from it, as long as that product is above 2^-80 of the sequence's largest value scale; below, as
 * where zeros have all the weight, it loses bits. */
int qh_kv8_attention(const qh_kv8_cache* c, int layer, const void* q, void* out, int dtype, int n_heads, int64_t ldq,
                     int64_t ldo, const int32_t* start, const int32_t* seqs, int n, int n_tok, int causal, float scale,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Which kernels a qh_kv8_attention call of this shape takes, by its sizes alone (single: start NULL); for profiles, and for
 * tests that have to reach each of them. */
enum {
    QH_KV8_WHOLE = 0,  /* a workgroup takes a row tile's sequence whole */
    QH_KV8_SHARES = 1, /* the tiles of all sequences in equal shares, which are joined */
    QH_KV8_TILES = 2   /* many rows: a workgroup to a tile of them */
};
typedef struct qh_kv8_plan {
    int32_t kernel;   /* QH_KV8_WHOLE, QH_KV8_SHARES or QH_KV8_TILES */
    int32_t rows;     /* of a workgroup's row tile */
    int32_t waves;    /* of a workgroup */
    int32_t splits;   /* QH_KV8_SHARES: shares; QH_KV8_TILES: workgroups over a row tile's positions, at most; else 1 */
    int32_t launches; /* of the kernel, over the batch's entries in turn */
} qh_kv8_plan;
int qh_kv8_attention_plan(const qh_kv8_cache* c, int n_heads, int n, int n_tok, int single, qh_kv8_plan* plan);

/* ------------------------------------------------------------------ rows of a step of many sequences */

/* Root-mean-square norm of n_tok rows of n, with a residual's addition before it: h = x + res, rounded to dtype (QH_F32 or
 * QH_F16; res NULL: h = x), goes to sum (NULL: nowhere), and h / sqrt(mean(h^2) + eps) * w to the outputs that are given:
 * y, rows of dtype, and / or q [n_tok][n] with d [n_tok][n / 32], the blocks that qh_quantize_q8 makes of the result in f32
 * (n a multiple of 32 then). w is f32 [n]. Squares are summed and results computed in 64 bits, rounded to f32, and f16 rows from
 * there. Rows are ld elements apart, on any alignment of their type (q: 16 bytes). sum may be x or res, with its row stride; the
 * outputs overlap nothing else. n at most QH_NORM_MAX; n_tok below 2^24, of rows of
 * more than 2,048 below 2^23, of more than 8,192 below 2^22. A NaN makes its row NaN; an infinity makes its own place NaN and the
 * rest of the row 0 (in blocks: as qh_quantize_q8 takes those).
 * No counterpart among the reference's kernels by itself: its rmsnorm (ops_ref.cpp:194-199) sums in f32 in order, which the
 * decoder's own kernels keep to the bit. */
#define QH_NORM_MAX 32768
int qh_rmsnorm(const void* x, const void* res, const float* w, int dtype, int64_t ldx, int64_t ldr, int n_tok, int n,
               double eps, void* sum, int64_t lds, void* y, int64_t ldy, int8_t* q, float* d, void* stream);

/* How far a rotary position turns the pairs of a head: pair i of rot_dim / 2 by theta^(-2 i / rot_dim) radians a position,
 * changed by `scaling` for contexts longer than the trained one:
 *   QH_ROPE_PLAIN  as it is
 *   QH_ROPE_LINEAR all divided by factor
 *   QH_ROPE_BASE   theta * factor^(rot_dim / (rot_dim - 2)) in theta's place: the slowest pair is divided by factor, the first
 *                  by nothing (rot_dim 2: as it is)
 *   QH_ROPE_PARTS  by parts: pairs that turn at most `low` times over `context` positions are divided by factor, those that
 *                  turn `high` times or more are left, with a ramp linear in the TURNS between them, as the schedule is
 *                  published. Programs that ramp linearly in the pair's index between those two ends turn the pairs between
 *                  them otherwise: for a model that was made with one, give qh_rope that table. What cosines and sines are
 *                  multiplied by (often 0.1 log(factor) + 1) is qh_rope's `magnitude` */
enum { QH_ROPE_PLAIN = 0, QH_ROPE_LINEAR = 1, QH_ROPE_BASE = 2, QH_ROPE_PARTS = 3 };
typedef struct qh_rope_desc {
    double theta;
    int32_t rot_dim; /* even, 2 to QH_ROPE_MAX_DIM */
    int32_t scaling; /* QH_ROPE_* */
    double factor, context, low, high; /* factor > 0; by parts: context > 0, 0 <= low < high */
} qh_rope_desc;
#define QH_ROPE_MAX_DIM 256

/* The pairs' turns (of 2 pi) per position in 64 bits: rot_dim / 2 of them into turns_host, which the caller uploads once.
 * Host only. Another schedule is as good: qh_rope takes any table. */
int qh_rope_turns(const qh_rope_desc* r, double* turns_host);

/* The rows' side of qh_rope: n_heads heads of head_dim one after the other (q's and k's at most 4,096 together), rows ld (out:
 * ldo) elements apart. out may be x (then ldo is ld); they do not overlap otherwise. */
typedef struct qh_rope_rows {
    const void* x;
    void* out;
    int64_t ld, ldo;
    int32_t n_heads;
} qh_rope_rows;

/* Rotary positions: every head of q's and k's rows (k NULL: q alone) has its first rot_dim dims turned in pairs (a, b) ->
 * (a cos - b sin, a sin + b cos) by the angle 2 pi pos[t] turns[i], cos and sin times `magnitude`; the others are copied. A
 * pair is the dims i and i + rot_dim / 2, or (interleaved 1) 2 i and 2 i + 1. pos: DEVICE int32 [n_tok], of either sign;
 * turns: DEVICE [rot_dim / 2]. Angles are taken in 64 bits less their whole turns: with qh_rope_turns' table they are off by up to
 * some 2^-51 of the angle (2^-49 where rot_dim is no power of two), by the table's rounding and the product's: below f32's step up
 * to 10^8 positions, 5e-7 radians at int32's ends. Rows of dtype QH_F32 or QH_F16 on any alignment of their type; head_dim at most
 * QH_ROPE_MAX_DIM.
 * Replaces: the rotation in Model::forward (reference model.cpp:187-196), for many sequences' tokens; the decoder's own
 * kernels keep the reference's f32 table to the bit. */
int qh_rope(const double* turns, int rot_dim, int interleaved, float magnitude, int head_dim, const qh_rope_rows* q,
            const qh_rope_rows* k, int dtype, const int32_t* pos, int n_tok, void* stream);

/* Attention of prompts over their own keys and values, as the projections give them, before (or without) their rounding into
 * a cache: out = sum_j p_j v_j with p = softmax(scale * q . k_j) over the keys j that a row sees. Entry b of n has the query rows
 * [start[b], start[b + 1]) of n_tok and the keys and values [kstart[b], kstart[b + 1]) of n_keys (DEVICE int32 [n + 1] each,
 * ascending; kstart NULL: start, and n_keys is n_tok). With causal 1 the rows are the entry's last positions: row i of m sees
 * the keys up to keys - m + i, so that new tokens behind kept ones see those too; with causal 0 every row sees every key of its
 * entry (states that are not the rows' own). Query head h reads KV head h / (n_heads / n_kv_heads). head_dim is 64 or 128; rows
 * of dtype QH_F32 or QH_F16, ld elements apart on any alignment of their type, a row's heads contiguous. A row that sees
 * nothing is 0; rows outside the entries are neither read nor written. Keys and values that a row does not see have no part in
 * it, whatever they hold. A NaN or an infinity that it sees stays in its dim where it is a value's, however small its weight, and
 * makes the row NaN where it is the query's; of a key's it becomes NaN, or what the formula gives. (Values that are not finite
 * are read once more: such a call takes up to twice its time.) f16: weights are rounded to f16 once. f32: products keep 22 bits and
 * more of every value from 2^-110 up, whatever the others are; of smaller ones what is above 2^-133; and a result of small values
 * is off by up to keys^2 * 2^-137 besides (6e-36 for 1,000 keys). Sums in f32 (a row that sees a score past f32's range may be NaN),
 * in an order that follows the whole call: a sequence's rows have the same bits in every call of the same shape and starts, but
 * not in another batch. out overlaps no input. The workspace is 16-byte aligned and needs no initialisation (NULL where the size
 * is 0); calls that overlap must not share one.
 * No counterpart in the reference, whose prompts attend to its cache in chunks (Model::forward_batch, model.cpp:387-405). */
size_t qh_attention_workspace_bytes(int dtype, int n_heads, int n_kv_heads, int head_dim, int n, int n_tok, int n_keys);
int qh_attention(const void* q, const void* k, const void* v, void* out, int dtype, int n_heads, int n_kv_heads,
                 int head_dim, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo, const int32_t* start,
                 const int32_t* kstart, int n, int n_tok, int n_keys, int causal, float scale, void* workspace,
                 size_t workspace_bytes, void* stream);

/* Beam search's selection. logits: DEVICE rows [n_prompts * beams][n_valid] of dtype QH_F32 or QH_F16, ld elements apart, on
 * any alignment of their type; scores: DEVICE f32 [n_prompts * beams], what each beam has so far (NULL: 0). A candidate is a
 * beam b of a prompt and an id v, with the score scores[b] + logits[b][v] - log sum_u exp(logits[b][u]); sums, exponentials
 * and the comparison of candidates are 64-bit, and equal ones go to the lower b, then the lower v. With m the largest logit of the
 * beam, that is (logits[b][v] - m) + (scores[b] - log sum_u exp(logits[b][u] - m)): beside a score of 2^53 times the logits'
 * differences and more, all ids of a beam are equal. For each prompt its k best
 * candidates, best first, into DEVICE arrays [n_prompts][k]: parent (the row, prompt * beams + b), token and score (f32). A
 * logit of -infinity is no candidate, and neither is any of a row whose score is not finite or whose logits hold a NaN or
 * +infinity or are all -infinity (a beam that ended gets the score -infinity); where there are fewer than k, the places
 * behind them have parent and token -1 and the score -infinity (which is also what a score past f32's range rounds to). beams
 * at most QH_BEAM_MAX_BEAMS, fewer than 2^17 rows, k at most QH_BEAM_MAX_K, n_valid at most QH_SAMPLE_MAX_VOCAB. The workspace
 * is 16-byte aligned and needs no initialisation; calls that overlap must not share one.
 * No counterpart in the reference, which samples one sequence (Sampler::sample, sampler.cpp:22-85). */
#define QH_BEAM_MAX_BEAMS 256
#define QH_BEAM_MAX_K 256
size_t qh_beam_workspace_bytes(int dtype, int n_prompts, int beams, int n_valid);
int qh_beam_select(const void* logits, int dtype, int64_t ld, const float* scores, int n_prompts, int beams, int n_valid,
                   int k, int32_t* parent, int32_t* token, float* score, void* workspace, size_t workspace_bytes,
                   void* stream);

/* ------------------------------------------------------------------ GPU-resident decoder */

/* FLAG_HADAMARD_DOWN (reference engine/src/model_file.h:19-21): the down projection's input is rotated by the
 * block-diagonal 256 x 256 Walsh-Hadamard transform (model.cpp:216-220), the weights having been rotated offline. */
#define QH_FLAG_HADAMARD_DOWN 1u

/* Model shape (reference engine/src/model_file.h:40-45, HParams, with its flags) and the load options: the context
 * length of the KV cache and kv_f32, an f32 cache in place of fp16 (Model::load's kv_f16 = false, the CLI's --kv-f32,
 * model.cpp:96-104). */
typedef struct qh_model_desc {
    int32_t vocab_size, dim, n_layers, n_heads, n_kv_heads, head_dim, ffn_dim, ctx_len, qkv_bias;
    float rope_theta, norm_eps;
    uint32_t flags;  /* QH_FLAG_* */
    int32_t kv_f32;  /* 0: fp16 cache (the reference's default); 1: f32 cache */
} qh_model_desc;

typedef struct qh_decoder qh_decoder;

/* Device addresses of the decoder's results and state, valid until qh_decoder_destroy. */
typedef struct qh_decoder_state {
    float* logits;          /* [vocab]: the last head call's logits (-inf outside the shortlist) */
    float* hidden;          /* [dim]: the last head call's final normed hidden state */
    int8_t* xq;             /* [dim]: its int8 quantization (first dim bytes) */
    float* xd;              /* [dim / 32]: its block scales */
    qh_head_stats* stats;   /* the last shortlist call's summary (top1, n_rows, ...) */
    int32_t* top1_full;     /* the greedy token of the last full-head call */
    int32_t* pos;           /* next position */
    int32_t* n_out;         /* tokens written to the output list since qh_decoder_begin */
    int32_t* token;         /* the token the next step consumes */
    uint16_t* kcache;       /* [n_layers][n_kv_heads][head_dim / 8][ctx_len][8] fp16 bits: chunks of 8 dimensions
                               (position p, KV head h, dimension i at ((h * (head_dim / 8) + i / 8) * ctx_len + p) * 8
                               + i % 8 within its layer) */
    uint16_t* vcache;       /* [n_layers][ceil(ctx_len / 8)][n_kv_heads * head_dim][8] fp16 bits: blocks of 8
                               positions, each dimension's 8 values contiguous (position p, column c at
                               ((p / 8) * kv_dim + c) * 8 + p % 8 within its layer) */
    int32_t* status;        /* 0, or bit 0: a step ran at a position >= ctx_len (it wrote nothing to the cache);
                               bit 1: a prompt token was outside [0, vocab); bit 2: the cache that
                               qh_decoder_bind_kv8 named had no place for a forward's tokens, which were not stored and
                               attended to nothing. Cleared by qh_decoder_prefill. */
    int32_t* history;       /* [ctx_len + 1]: the token history (the session's history_, session.cpp:13-52): the
                               prompt ids of every prefill since position 0, then each chosen id */
    int32_t* history_len;   /* its length */
    uint64_t* rng_state;    /* the sampler's xorshift64* state */
    float* kcache_f32;      /* with kv_f32 (kcache and vcache NULL then): [n_layers][ctx_len][n_kv_heads * head_dim],
                               the reference's own layout (model.cpp:96-104); NULL otherwise */
    float* vcache_f32;      /* the same for V */
} qh_decoder_state;

/* Creates a decoder over device tensors, in this order (reference model.cpp:14-33, 47-58):
 *   model.embed_tokens.weight ([vocab][dim], also the LM head when tied), model.norm.weight (F32 [1][dim]);
 *   per layer: input_layernorm (F32), q_proj, k_proj, v_proj, o_proj, q/k/v biases (F32, or data NULL without
 *   qkv_bias), post_attention_layernorm (F32), gate_proj, up_proj, down_proj;
 *   then quanta.head_q4 (Q4_0 [vocab][dim]) and quanta.head_err (F16 [vocab][dim/32]), or both with data NULL;
 *   optionally (n_tensors 5 + 12 n_layers) lm_head.weight ([vocab][dim]), the LM head of an untied model; data NULL
 *   there, or n_tensors 4 + 12 n_layers, means tied.
 * Every matrix (the embedding and LM head included) may be Q8_0, Q4_0, F32 or F16, each on its own, as the exporter
 * writes them (F32 / F16 ones run matvec_ref's float chain on the f32 activation, model.cpp:150-157); the LM head is
 * Q8_0 when the shortlist head tensors are given (model.cpp:49-58).
 * Allocates an fp16 KV cache (f32 with hp->kv_f32) for ctx_len positions and the work buffers. dim, ctx_len <= 8192,
 * head_dim 64 or 128, n_heads * head_dim == dim, ffn_dim % 256 == 0 with QH_FLAG_HADAMARD_DOWN. The tensors must
 * stay alive while the decoder is used.
 * Replaces: Model::load (reference model.cpp:10-106) after the .qnt file is read and uploaded. */
int qh_decoder_create(const qh_model_desc* hp, const qh_tensor* tensors, int n_tensors, qh_decoder** out);
int qh_decoder_destroy(qh_decoder* d);

/* n prompt tokens (device array) at positions [pos0, pos0 + n): every layer in 32-token chunks, then the head for
 * the last token (top_k > 0: shortlist head with n_valid = vocab; 0: full 8-bit head). The next position becomes
 * pos0 + n. Replaces: Model::forward_batch (reference model.cpp:349-433). */
int qh_decoder_prefill(qh_decoder* d, const int32_t* tokens, int n, int pos0, int top_k, void* stream);

/* Starts a greedy generation: the last head call's greedy token becomes the first output (out_dev[0]) and the next
 * input, as Session::generate samples its first token from the prompt's logits (reference session.cpp:33-52). */
int qh_decoder_begin(qh_decoder* d, int top_k, int32_t* out_dev, int out_cap, void* stream);

/* One greedy decode step entirely on the device: forward of the current token at the current position, head,
 * greedy token appended to the output list and made the next input, position + 1. The launch sequence does not
 * depend on host state, so it can be captured in a HIP graph once and replayed for every step.
 * Replaces: one iteration of Session::generate with the greedy sampler (reference session.cpp:39-49, model.cpp:165-228,
 * sampler.cpp:35-37). */
int qh_decoder_step(qh_decoder* d, int top_k, void* stream);

int qh_decoder_views(qh_decoder* d, qh_decoder_state* v);

/* The prefill stack: how many prompt tokens later qh_decoder_prefill calls take through each layer's norms and
 * matmuls at once. 32 (the default) is the reference's chunk (Model::kBatch, model.h:52; forward_batch,
 * model.cpp:349-361); a multiple of 32 up to 1024 runs the same arithmetic on larger batches (the matmul tile kernels
 * at M up to `stack`; attention of the whole stack at once over an fp16 cache, in 32-token sub-chunks in order over an
 * f32 one), so every hidden state, cache row and logit is bit-identical to the 32-token chunks. Reallocates the
 * decoder's work buffers: it synchronises the device, the pointers qh_decoder_views gave (xq / xd) change and their
 * contents are lost, and a step captured in a HIP graph before the call must be captured again. With an fp16 cache of
 * more than 1,024 positions a stack above 32 also takes a workspace for attention scores: 264 bytes per position, KV
 * head and group of 64 (token, query head) pairs of it, at most 256 MB, and less (down to one such group) where memory
 * is short, in more passes. On failure the previous stack stays.
 * Replaces: nothing (the reference's chunk is a compile-time constant); a scheduling choice of the GPU path. */
int qh_decoder_set_prefill_stack(qh_decoder* d, int stack);

/* Later prefill and step calls keep their keys and values in sequence `seq` of the 8-bit cache c (n_layers, n_kv_heads
 * and head_dim of the model; its state arrays in order, its memory alive while it is bound) instead of the decoder's own
 * cache, and attend to that sequence: results then carry the 8-bit rounding and are no longer the reference's bits. A
 * prefill at pos0 (at most the sequence's length) first shortens the sequence to pos0; a step continues it, so its
 * position has to be the sequence's length. Both take pages from the cache as the sequence grows, copying a last page that
 * other sequences hold. So a prompt is read once and its continuations are forks: qh_kv8_fork, then for each fork this call
 * and a prefill of the prompt's last token. Tokens that have no place (no free page, another position, past the context or
 * the table row) set *status. Synchronises the device and allocates workspaces at the first call and where the cache's size
 * changes (a failure leaves the decoder as it was); the sequence is read on the device, so a step captured in a HIP graph
 * follows a later call that names another sequence of the same cache, and has to be captured again for another cache.
 * c NULL: the decoder's own cache again (with what it held).
 * No counterpart in the reference, whose Model owns one sequence. */
int qh_decoder_bind_kv8(qh_decoder* d, const qh_kv8_cache* c, int seq);

/* Stages of a decode step, as qh_decoder_step_timed names them: per layer l, id l * QH_STAGES_PER_LAYER + one of
 * QH_STAGE_QKV (rmsnorm + q/k/v projections; in layer 0 also what makes room in a bound 8-bit cache),
 * QH_STAGE_ATTENTION, QH_STAGE_O (o projection + residual), QH_STAGE_GATE_UP (rmsnorm + gate/up projections + SwiGLU),
 * QH_STAGE_DOWN (down projection + residual); then QH_STAGE_FINAL_NORM, QH_STAGE_HEAD and, when a sampler picks the token,
 * QH_STAGE_PICK. With the fused kernels (the default) and the decoder's own cache each per-layer stage is one kernel. */
enum {
    QH_STAGE_QKV = 0,
    QH_STAGE_ATTENTION = 1,
    QH_STAGE_O = 2,
    QH_STAGE_GATE_UP = 3,
    QH_STAGE_DOWN = 4,
    QH_STAGES_PER_LAYER = 8,
    QH_STAGE_FINAL_NORM = 1 << 20,
    QH_STAGE_HEAD = (1 << 20) + 1,
    QH_STAGE_PICK = (1 << 20) + 2
};

/* One qh_decoder_step with every kernel it launches timed on the device by the dispatch's own start and stop
 * timestamps (no extra packets between the kernels): for the i-th kernel, us_host[i] microseconds and stage_host[i]
 * its stage id; *n_host = the number of kernels. Host arrays; synchronises the stream. When the step launches more
 * than cap kernels the result is QH_ERR_NOMEM with *n_host set to the number it launched (the capacity it needs) and
 * us_host / stage_host unset; the step itself has run all the same (the decoder has advanced one token), so a caller
 * that retries with a larger cap takes the next step.
 * No counterpart in the reference (its CLI times whole tokens); for profiling. */
int qh_decoder_step_timed(qh_decoder* d, int top_k, void* stream, float* us_host, int32_t* stage_host, int cap,
                          int32_t* n_host);

/* The head queries of later prefill / begin / step calls, as Session::head_query builds them from the session's
 * sampler parameters (session.cpp:63-79): top_k = (temperature <= 0 ? 1 : p->top_k), the full head when that is 0,
 * and, when p->repeat_penalty != 1, the last p->repeat_window ids of the token history (all when 0) as must ids. The
 * calls' own top_k argument is then ignored. NULL restores plain queries (the calls' top_k, no must ids). With the
 * shortlist head tensors, top_k is at most QH_HEAD_MAX_TOPK (QH_ERR_UNSUPPORTED above).
 * Replaces: Session::set_sampler and Session::head_query (reference session.h, session.cpp:63-79). */
int qh_decoder_set_query(qh_decoder* d, const qh_sampler_params* p);

/* The token qh_decoder_begin and qh_decoder_step choose: NULL (the default) takes the head's greedy top-1; with p,
 * one qh_sample draw over the head's logits (its row list when the shortlist ran) with the token history, from the
 * generator state `seed | 1` (seed nonzero). The state lives on the device and advances with each draw, so a captured
 * step keeps sampling on replay.
 * Replaces: the Sampler that Session::generate calls (reference sampler.cpp:10-85, session.cpp:32-52). */
int qh_decoder_set_sampler(qh_decoder* d, const qh_sampler_params* p, uint64_t seed);

#ifdef __cplusplus
}
#endif

#endif /* QUANTA_HIP_H */
