/* ccdecode.h — C ABI of the MI355X batched ragged decode pass.
 *
 * The library replaces the GPU side of the reference's Runner
 * (web/model/stage.js): one context owns a contiguous range of positions
 * (0 = embedding, 1..L = blocks, L+1 = final norm + LM head), its q8 weights,
 * an int8 paged KV pool, session frames (slots) with page tables, and all
 * scratch. cc_step runs one packed pass over prepared jobs — the reference's
 * Runner.#pass (web/model/stage.js:1314-1481) — and returns per-row top-M
 * candidates or the f16 rows handed downstream.
 *
 * Host policy (queueing, batching rules, admission, eviction, cuts, boundary
 * logs) stays with the caller, as it does in the reference's Runner; the
 * caller is the JS shim (chattorrent_amd/node/runner.js) over the N-API addon,
 * or Python over ctypes. Every entry point returns a cc_status; on failure
 * cc_last_error() holds the message. A context is not reentrant: calls on one
 * context must not overlap (the reference runs jobs one at a time,
 * web/model/stage.js:5, :646-654).
 *
 * Plain C types only. Host buffers are owned by the caller for the duration of
 * the call; the library copies through its own pinned staging.
 */
#ifndef CCDECODE_H
#define CCDECODE_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Error classes of the reference's Runner, kept per job
 * (web/model/stage.js:930-941 busy, :948-958 / :1073-1079 cold,
 * :1067-1072 stale, :339-345 nospec, :1225-1259 bad job, :1114-1117 pool too
 * small; device loss: web/engine.js:703-744). */
typedef enum cc_status {
    CC_OK = 0,
    CC_BUSY = 1,      /* capacity refusal (no frame / page free now) */
    CC_COLD = 2,      /* the session's cache is not here (evicted or behind) */
    CC_STALE = 3,     /* a duplicate job behind the cache */
    CC_NOSPEC = 4,    /* no speculative replay state (hybrid models only) */
    CC_EARG = 5,      /* a malformed job or call */
    CC_EPOOL = 6,     /* the KV pool cannot hold this context at all */
    CC_EOOM = 7,      /* device allocation failed */
    CC_EDEVICE = 8    /* a HIP error; the context should be destroyed */
} cc_status;

/* Model dimensions: loader.js dimsFromManifest (web/model/loader.js:146-201),
 * checked like model.js checkDims (web/model/model.js:22-40). */
typedef struct cc_dims {
    int32_t hidden, n_layer, n_heads, n_kv_heads, head_dim, ffn, vocab;
    int32_t q8_group;       /* weights: one scale per this many values along K (32) */
    float rms_eps;
    double rope_theta;
    int32_t rope_scaling;   /* 0 none, 1 llama3 (kernels.js:1998-2014) */
    double rs_factor, rs_low_freq, rs_high_freq, rs_orig_max_pos;
    int32_t tied;           /* LM head reads the embedding table */
    /* Hybrid (Qwen3.5-architecture) checkpoints — dimsFromManifest,
     * web/model/loader.js:146-201. rot_dim: RoPE width (partial rotary,
     * kernels.js:1080-1129); 0 means head_dim. hybrid != 0: full_attention
     * blocks also carry attn_gate, q_norm and k_norm (loader.js:543-565), and
     * n_heads*head_dim may differ from hidden. layer_kinds: n_layer entries,
     * CC_FULL_ATTENTION or CC_LINEAR_ATTENTION (NULL: every block full; the
     * array is copied by cc_create). lin_*: Gated DeltaNet's key heads, value
     * heads, key and value head widths, conv width (linear_num_key_heads ..
     * linear_conv_kernel_dim). */
    int32_t rot_dim;
    int32_t hybrid;
    const uint8_t* layer_kinds;
    int32_t lin_nk, lin_nv, lin_dk, lin_dv, lin_conv;
    /* The MTP draft head (model.js:529-576, loader.js:628-638): the
     * vocabulary rows it drafts over (manifest mtp.draft_vocab); 0: none. A
     * context holding the head holds it. */
    int32_t mtp_vocab;
} cc_dims;
enum { CC_FULL_ATTENTION = 0, CC_LINEAR_ATTENTION = 1 };

/* Runner options (web/model/stage.js:107-110). lo/hi: the position range
 * held; n_max: context window; t_max: the most rows one pass carries; slots:
 * full contexts the KV pool holds (pages = slots * ceil(n_max/page));
 * sessions: frames (page tables). */
typedef struct cc_opts {
    int32_t lo, hi;
    int32_t n_max;
    int32_t t_max;
    int32_t slots;
    int32_t sessions;
    int32_t page_tokens;    /* 64 (web/split.js:75) */
    int32_t max_jobs;       /* the most jobs one pass packs */
    int32_t device;
} cc_opts;

typedef struct cc_ctx cc_ctx;

/* Tensor ids for cc_upload / cc_fill_random (HF names). layer = -1 for the
 * model-level tensors. */
enum {
    CC_T_Q = 0, CC_T_K = 1, CC_T_V = 2, CC_T_O = 3, CC_T_GATE = 4, CC_T_UP = 5, CC_T_DOWN = 6,
    CC_T_LN1 = 7, CC_T_LN2 = 8, CC_T_WTE = 9, CC_T_NORM = 10, CC_T_LM_HEAD = 11,
    /* a hybrid checkpoint's full_attention extras (loader.js:543-565):
     * attn_gate q8 [n_heads*head_dim, hidden]; q_norm, k_norm f32 [head_dim] */
    CC_T_ATTN_GATE = 12, CC_T_Q_NORM = 13, CC_T_K_NORM = 14,
    /* linear_attention blocks (loader.js:567-590, tools/convert_hf.py:188-219):
     * in_proj_q/k q8 [keyDim, hidden], in_proj_v/z q8 [valueDim, hidden],
     * in_proj_b/a q8 [nV, hidden], conv1d_q/k f32 [keyDim, conv],
     * conv1d_v f32 [valueDim, conv], gate_params f32 [2*nV] (A_log, then
     * dt_bias), gated_norm f32 [Dv], out_proj q8 [hidden, valueDim] */
    CC_T_IN_Q = 15, CC_T_IN_K = 16, CC_T_IN_V = 17, CC_T_IN_Z = 18, CC_T_IN_B = 19, CC_T_IN_A = 20,
    CC_T_CONV_Q = 21, CC_T_CONV_K = 22, CC_T_CONV_V = 23, CC_T_GATE_PARAMS = 24, CC_T_GATED_NORM = 25,
    CC_T_OUT_PROJ = 26,
    /* the MTP head (loader.js:633-634): enorm, hnorm, mtp_norm f32 [hidden];
     * fc_e, fc_h q8 [hidden, hidden]; embed_draft, head_draft q8
     * [mtp_vocab, hidden]. Its full-attention block's tensors are the block
     * ids above at layer CC_LAYER_MTP. */
    CC_T_MTP_ENORM = 27, CC_T_MTP_HNORM = 28, CC_T_MTP_FC_E = 29, CC_T_MTP_FC_H = 30, CC_T_MTP_NORM = 31,
    CC_T_MTP_EMBED = 32, CC_T_MTP_HEAD = 33
};
enum { CC_LAYER_MTP = -2 };
enum { CC_SCALES_F16 = 0, CC_SCALES_F32 = 1 };

/* new Runner(device, d, w, {...}) — web/model/stage.js:107-238. */
cc_status cc_create(const cc_dims* dims, const cc_opts* opts, cc_ctx** out);
void cc_destroy(cc_ctx* ctx);
const char* cc_last_error(const cc_ctx* ctx);

/* uploadQ8(device, int8Bytes, scales, group) — web/model/kernels.js:122-126;
 * norms (tensor LN1/LN2/NORM) are f32 `data` with n = hidden and no scales,
 * and so are the hybrid f32 tensors (Q_NORM .. GATED_NORM, n = their size).
 * q8 tensors: `data` int8 [N, K] row-major, `scales` [N, ceil(K/group)] as
 * f16 bits or f32 (rounded to the device's f16 scale). `group` is any
 * multiple of 32 (the reference's converter writes 64,
 * tools/convert_hf.py:493): a scale covering group/32 of the device's
 * 32-wide groups is given to each of them, which is exact. */
cc_status cc_upload(cc_ctx* ctx, int32_t layer, int32_t tensor, const void* data, size_t n,
                    const void* scales, size_t ns, int32_t scale_dtype, int32_t group);

/* Synthetic weights on the device from the counter-based generator shared
 * with the test oracle (no reference counterpart: the reference's random
 * models are randomWeights, web/model/model.js:697-717). On a hybrid model
 * (and for the MTP head) this is for timing only: the Gated DeltaNet's f32
 * parameters take fixed values (conv taps 0.25, A_log -1, dt_bias 0) that
 * the oracle does not mirror; parity tests upload their weights. */
cc_status cc_fill_random(cc_ctx* ctx, uint64_t seed);

/* One prepared job of a pass (the fields #prepare hands #pass,
 * web/model/stage.js:1195-1308). `ids` when the pass enters at position 0,
 * else `hidden` (n*hidden f16 bits). `sampled`: rows the head samples — 1
 * (the last row) or n (a verify); 0 when the pass does not reach the head. */
typedef struct cc_job {
    int32_t slot;
    int32_t past;
    int32_t n;
    int32_t sampled;
    const int32_t* ids;
    const uint16_t* hidden;
    /* Speculative decoding through linear_attention blocks (stage.js:1248-1283,
     * model.js:447-470 restoreSpec / snapSpec). snap != 0: a verify job
     * (n <= 8 rows); its blocks keep the state it starts from and its rows'
     * projections. rollback != 0: the session's last job here was a verify
     * from `base`; this job continues at past = base + keep (0 <= keep <= that
     * verify's n): the blocks go back to the verify's starting state and
     * re-run its first `keep` rows before this job's own. Zero-initialised
     * fields mean neither. */
    int32_t snap;
    int32_t rollback;
    int32_t keep;
    /* The job's session drafts with the MTP head (stage.js:1287-1293): at a
     * context holding it, the MTP layer's KV rows past..past+n-1 are filled
     * from the job's `ids` (given whatever the entry position) paired with
     * the trunk's hidden rows one position earlier; a job that samples
     * nothing keeps its last row for the next job (stage.js:1408-1421). */
    int32_t mtp;
} cc_job;

/* Runner.#pass — web/model/stage.js:1314-1481. Runs positions [at, to) for
 * `njobs` jobs packed in order. Pages for rows past..past+n-1 are taken from
 * the pool on the device in job order (model.js ensurePages replayed).
 * Outputs: when `to` is past the last block (the head), `top_vals`/`top_ids`
 * receive `topk` candidates per sampled row (sampled rows in job order, best
 * first, ties to the lower id); otherwise `hidden_out` receives every row as
 * f16 bits [T, hidden]. `status` (optional, njobs) is set per job. A pass
 * that fails leaves the outputs alone; only if the device itself stops while
 * a large pass's rows are leaving it (CC_EDEVICE) may hidden_out hold a part
 * of them. */
cc_status cc_step(cc_ctx* ctx, const cc_job* jobs, int32_t njobs, int32_t at, int32_t to,
                  int32_t topk, float* top_vals, uint32_t* top_ids, uint16_t* hidden_out,
                  int32_t* status);

/* `steps` greedy passes of Runner.#pass (web/model/stage.js:1314-1481) run
 * back to back on the device, the route's closed decode loop
 * (web/route.js:865-952) without a host round trip between passes: every
 * job is one row, sampled; pass k runs each job at past + k with the token
 * pass k-1 sampled (column 0 of its candidates; pass 0 takes jobs[j].ids[0]),
 * and packs its rows and attention work on the device. Each pass takes the
 * pages its jobs newly need, job by job, as a cc_step of that pass would, so
 * the frames' page tables and the pool end as after `steps` cc_step calls
 * (CC_BUSY, before anything runs, when the pool cannot supply them).
 * Outputs: top_vals / top_ids [steps][njobs][topk], best first. Each pass's
 * results equal cc_step's for the same jobs. A context holding every position of a full-attention model
 * without an MTP head. */
cc_status cc_decode_steps(cc_ctx* ctx, const cc_job* jobs, int32_t njobs, int32_t steps, int32_t topk,
                          float* top_vals, uint32_t* top_ids);

/* After sampling `token` from row `row` of the last pass (Runner.#mtpAfter,
 * web/model/stage.js:296-320): the session keeps that row's hidden state
 * (row -1: keep the one it has) and, for k_drafts > 0 (at most 7), the MTP
 * head chains that many drafts after `token` at positions pos..
 * (model.js:567-576 mtpChain: each step's argmax over the draft vocabulary,
 * lowest id on a tie, is the next step's token). The MTP layer's KV rows
 * written there are speculative; the next job's fill rewrites them. Pages
 * are taken for pos + k_drafts tokens. `drafts` receives k_drafts ids. */
cc_status cc_mtp_draft(cc_ctx* ctx, int32_t slot, int32_t row, int32_t token, int32_t pos, int32_t k_drafts,
                       uint32_t* drafts);

/* Runner.#release / freePages — web/model/stage.js:842-874,
 * web/model/model.js:204-211: the slot's pages return to the pool. */
cc_status cc_release(cc_ctx* ctx, int32_t slot);

/* Frame pages the slot holds (the frame's `owned` length). */
int32_t cc_slot_pages(const cc_ctx* ctx, int32_t slot);
int32_t cc_free_pages(const cc_ctx* ctx);

/* Fill rows 0..tokens-1 of a slot with random int8 KV (codes uniform in
 * ±127, one f16 scale ~U(0.005, 0.02) per token and kv head), taking pages
 * as a job would. `key` names the chat in the generator index. */
cc_status cc_fill_random_kv(cc_ctx* ctx, int32_t slot, int32_t tokens, uint64_t seed, uint64_t key);

/* Debug readback in the reference's row layout (web/model/kernels.js:999-1022:
 * D/4 code words then D/QB f32 scales per row): rows t0..t1-1 of one kv head,
 * which = 0 for K, 1 for V, `layer` a held block index. */
cc_status cc_read_kv(cc_ctx* ctx, int32_t layer, int32_t which, int32_t slot, int32_t head,
                     int32_t t0, int32_t t1, uint32_t* out);
cc_status cc_write_kv(cc_ctx* ctx, int32_t layer, int32_t which, int32_t slot, int32_t head,
                      int32_t t0, int32_t t1, const uint32_t* rows);
cc_status cc_read_pages(cc_ctx* ctx, int32_t slot, uint32_t* out, int32_t n);

/* The last pass's full logits rows [rows, vocab] f32 (the sampled rows of a
 * pass that reached the head), for parity checks: the reference reads back
 * whole rows when a sampler needs them (web/model/stage.js:1428-1436). */
cc_status cc_read_logits(cc_ctx* ctx, int32_t rows, float* out);

/* Stats (Runner.counts / vramBytes, web/model/stage.js:219-259). */
typedef struct cc_stats {
    uint64_t vram_bytes;
    uint64_t weight_bytes;
    uint64_t kv_bytes;
    uint64_t scratch_bytes;
    int64_t passes;
    int64_t rows;
    double last_pass_ms;
} cc_stats;
cc_status cc_stats_get(const cc_ctx* ctx, cc_stats* out);

/* Per-kernel timing with HIP events on the context's stream (the
 * reference's gpuprof.js level 2, web/model/gpuprof.js:1-12, re-done for
 * HIP). While enabled, each cc_step, after its own work, launches each class
 * below again for every block of the step, back-to-back between one event
 * pair (so no marker sits between launches); cc_profile_read returns the
 * summed milliseconds, the launch count and the algorithmic HBM bytes of
 * those launches (q8 weights at 1.0625 B per weight; KV rows at
 * D + 4*D/32 B). The launches are the step's own kernels: with few rows a
 * matmul's time includes forming its operand where it did so itself. The
 * step's results are unchanged. Enabling resets the sums. */
enum { CC_K_QKV = 0, CC_K_O = 1, CC_K_GU = 2, CC_K_DOWN = 3, CC_K_HEAD = 4, CC_K_ATTN = 5, CC_K_COUNT = 6 };
cc_status cc_profile(cc_ctx* ctx, int32_t enable);
cc_status cc_profile_read(const cc_ctx* ctx, int32_t kind, double* ms, int64_t* launches, double* bytes);

/* ---- Kernel-level entry points (one reference kernel each), used by the
 * parity tests to hold each GPU kernel to the oracle on identical inputs. All
 * pointers are host memory. ---- */

/* matmulNobias for q8 — web/model/kernels.js:1874-1914. Y[M,N] = X[M,K] W^T. */
cc_status cc_op_matmul_q8(cc_ctx* ctx, const float* X, int32_t M, int32_t K,
                          const int8_t* W, const uint16_t* scales_f16, int32_t N, float* Y);
/* store_kv — web/model/kernels.js:1960-1973, into `slot`'s pages of block
 * `layer`: src [T_new, nKV*D] f32; rope != 0 rotates (K), else V. */
cc_status cc_op_store_kv(cc_ctx* ctx, int32_t layer, int32_t which, int32_t slot,
                         const float* src, int32_t T_new, int32_t T_past);
/* round_f16 — web/model/kernels.js:2100-2105. In place on n floats. */
cc_status cc_op_round_f16(cc_ctx* ctx, float* a, int64_t n);
/* topkRows — web/model/kernels.js:2129-2144: rows x V logits → M pairs. */
cc_status cc_op_topk(cc_ctx* ctx, const float* logits, int32_t rows, int32_t V, int32_t M,
                     float* vals, uint32_t* ids);
/* No counterpart in the reference: an allocation-free cc_op_topk for callers
 * that cannot allocate device memory (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc). `logits` [rows, V] f32,
 * `vals` and `ids` [rows, M] are DEVICE pointers the caller owns; the stages'
 * keys go to a static 4 MiB scratch array per GPU (TOPK_SCRATCH_KEYS keys),
 * and calls needing more are refused with CC_EARG. The first stage keeps
 * rows * ceil(V/4096) * M keys and the next one far fewer: at M = 1 and
 * V = 2^20 a call needs rows * 257 keys, so up to 2040 rows fit; at M = 256
 * and V = 262144, 30 rows.
 * Runs asynchronously on
 * `stream` (a hipStream_t; NULL: the context's stream): the caller
 * synchronises before reading `vals`/`ids`. Calls no hipMalloc, hipFree or
 * allocating routine. Every call on one GPU shares that GPU's scratch, so
 * calls that overlap on one GPU (different streams or contexts) race. */
cc_status cc_topk_noalloc(cc_ctx* ctx, const float* logits, int32_t rows, int32_t V, int32_t M, float* vals,
                          uint32_t* ids, void* stream);
/* rmsnorm — web/model/kernels.js:1927-1932. */
cc_status cc_op_rmsnorm(cc_ctx* ctx, const float* x, const float* w, int32_t T, int32_t H,
                        float* y);
/* attend (web/model/model.js:321-351) for one job of block `layer` whose K/V
 * rows are already stored: q [n, nH*D] f32 (before RoPE) -> out [n, nH*D]. */
cc_status cc_op_attend(cc_ctx* ctx, int32_t layer, int32_t slot, const float* q, int32_t n,
                       int32_t past, float* out);

/* ---- Operators on the caller's device buffers: one decode step of long
 * chats, from the paged cache to the token, for callers that run their own
 * blocks or sample rows themselves. They stand beside cc_topk_noalloc: every
 * buffer is device memory of the context's GPU that the caller owns, nothing
 * is allocated or copied, and a call runs asynchronously on `stream` (a
 * hipStream_t; NULL: the context's stream), in kernels alone, so it can be
 * captured into a HIP graph (its jobs and pointers are then the captured
 * ones). The context gives the GPU and holds the error message; calls on one
 * context from two threads must not overlap. Calls on several streams may
 * overlap on the GPU as long as they share no workspace and no rows that one
 * of them writes. No counterpart in the reference, whose cache ops are inside
 * its pass and whose sampler runs on the host (web/model/sampling.js). ---- */

/* A paged int8 cache, K and V of one layer. Each (page of 64 tokens, kv head)
 * is a block of 64*D code bytes (code + 128) and then 64*D/32 f32 scales, one
 * per token and 32 channels; `k` and `v` are [n_pages][n_kv_heads] blocks:
 *   K: token t, channel d at t*D + (D/4)*((d%32)/8) + 8*(d/32) + d%8, scale of
 *      group g at t*D/32 + g;
 *   V: with u = 16*((t%16)/4) + 4*(t/16) + t%4, code at ((u/16)*D + d)*16 +
 *      u%16, scale at ((u/16)*D/32 + g)*16 + u%16.
 * page_table [slots][max_pages]: a slot's pages in token order (an index of
 * n_pages or more is no page: rows are not stored there, and its tokens are
 * masked). rope [rope_rows][rot_dim/2][2]: cos and sin of each position, f32.
 * bounds (may be NULL): key bounds, n_pages * cc_bounds_bytes(cache) bytes:
 * per page and kv head 2*D int8 codes, channel d's largest (w = 0) and
 * smallest (w = 1) key of the page's 64 tokens at (2w + (d%32)/16)*(D/2) +
 * 16*(d/32) + d%16, then, after all kv heads' codes, f32 scales
 * [n_kv_heads][D/32]. k, v and bounds are 16-byte aligned; D (head_dim) is 64,
 * 128 or 256; rot_dim is even, at most D; max_pages at most 32768. */
typedef struct cc_cache {
    int32_t n_kv_heads, head_dim, rot_dim;
    int32_t n_pages, max_pages, slots, rope_rows;
    void* k;
    void* v;
    void* bounds;
    const uint32_t* page_table;
    const float* rope;
} cc_cache;
/* The context's own cache of block `layer` (bounds NULL: the caller may set
 * its own). Its pages are the context's to give: cc_step, cc_fill_random_kv
 * and cc_release change the page table on the context's stream. The context's
 * own passes (cc_step, cc_decode_steps, cc_mtp_draft) and cc_op_attend take a
 * row's index for its position. Once a slot's rows were placed otherwise
 * (cc_kv_append_at) or given up (cc_kv_evict) they compute wrong attention for
 * it, with no error: go on with the operators, or release the slot. */
cc_status cc_cache_of(cc_ctx* ctx, int32_t layer, cc_cache* out);
/* Bytes of key bounds a page takes; 0 for a head_dim that is not supported. */
size_t cc_bounds_bytes(const cc_cache* cache);

/* `n` rows of a slot from position `past`. The rows of a call's jobs lie
 * behind each other in job order. Host memory, read during the call. */
typedef struct cc_rows {
    int32_t slot, past, n;
} cc_rows;

/* Stores the jobs' rows: k, rotated to its position, and v, both f32 [rows]
 * [n_kv_heads * D] with ldk and ldv floats from row to row, in 32-channel
 * groups of int8 codes as store_kv rounds them (web/model/kernels.js:1024-1073:
 * the pass's own bits). Where the cache has bounds, a page whose last row is
 * among them gets its key bounds, from its 64 rows as the cache holds them:
 * per 32 channels B = (largest magnitude)/127, the largest key of a channel as
 * ceil(key/B), the smallest as floor(key/B), both within +-127. The page's
 * earlier rows are those stored before. The slots' pages must be in the page
 * table. CC_EARG: a slot twice in a call, rows past max_pages*64 or rope_rows. */
cc_status cc_kv_append(cc_ctx* ctx, const cc_cache* cache, const cc_rows* jobs, int32_t njobs, const float* k,
                       int64_t ldk, const float* v, int64_t ldv, void* stream);
/* Key bounds of the pages that lie within the jobs' rows as a whole, from what
 * the cache holds: for rows that another path stored (cc_step). */
cc_status cc_kv_bounds(cc_ctx* ctx, const cc_cache* cache, const cc_rows* jobs, int32_t njobs, void* stream);

/* Attention of the jobs' rows over selected pages. Row i of a job is at
 * position past + i and sees the tokens up to its own (stored before). q f32
 * [rows][n_heads * D] before RoPE, ldq floats from row to row; out alike, with
 * ldo, in memory of its own. Query head h reads kv head h / (n_heads / n_kv_heads).
 * A row sees P = (past + i)/64 + 1 pages. Up to `budget` it reads them all.
 * Else each kv head of it reads `budget` of them: the first `sink`, the last
 * `recent`, and the best of the others by score, ties to the lower page. With
 * the rotated query in 8 bits as store_kv rounds a key (codes c, scales T per
 * 32 channels) and a page's bounds (hi, lo, B), a query head's score is the
 *   sum over groups g of T_g * B_g * sum over d in g of max(c*hi, c*lo),
 * and the kv head's the largest over its query heads, rounded to f32.
 * out = softmax(q . k / sqrt(D)) v over the tokens read. How many workgroups
 * share a row's pages follows from the rows of the call, so a row's last bits
 * may differ between calls of few and of many rows; which pages it reads does
 * not. An output value's error is relative to the largest |v| of its 32
 * channels among the tokens read.
 * 0 <= sink, 1 <= recent, sink + recent <= budget. cache->bounds is needed
 * where a row sees more than `budget` pages: the pages before the row's last
 * `recent` have theirs. `workspace`: cc_attend_workspace bytes (for a
 * call of up to `rows` rows; 0: it would be refused), 16-byte aligned, of any
 * contents; two calls that may overlap need two. */
size_t cc_attend_workspace(cc_ctx* ctx, const cc_cache* cache, int32_t rows, int32_t n_heads, int32_t budget);
cc_status cc_attend_pages(cc_ctx* ctx, const cc_cache* cache, const cc_rows* jobs, int32_t njobs, int32_t n_heads,
                          int32_t budget, int32_t sink, int32_t recent, const float* q, int64_t ldq, float* out,
                          int64_t ldo, void* workspace, size_t workspace_bytes, void* stream);

/* A cache held within a bound: rows whose positions are not their indices,
 * what attention gives each row of the cache, and giving up the rows that get
 * the least.
 *
 * Positions of the rows of a call, `pos` [rows][n_axes] in device memory, on 1
 * to 4 axes (time, height and width of an image's patches; text has the same
 * position on each). Pair j of rotary channels turns by axis axis_of[j]
 * (rot_dim/2 bytes of HOST memory, read during the call; NULL: the first axis).
 * A position outside the rope table is taken as the table's nearest. */
typedef struct cc_positions {
    int32_t n_axes;
    const int32_t* pos;
    const uint8_t* axis_of;
} cc_positions;

/* The marks of a cache's rows, [n_pages][n_kv_heads][64] each, 16-byte aligned:
 * the attention weight that a row has gathered, and its token's number in the
 * chat (0 is the chat's first token). */
typedef struct cc_marks {
    float* weight;
    int32_t* token;
} cc_marks;

/* cc_kv_append at positions `at` (NULL: each row's index, as there) instead of
 * the rows' indices: row past + i of a slot may hold any token. Where marks is
 * given the rows' weights become 0 and their tokens first[j] + i (`first`: host
 * memory, one of each job; NULL: past). The key bounds of pages that a call
 * completes are made as there. */
cc_status cc_kv_append_at(cc_ctx* ctx, const cc_cache* cache, const cc_positions* at, const cc_marks* marks,
                          const cc_rows* jobs, int32_t njobs, const int32_t* first, const float* k, int64_t ldk,
                          const float* v, int64_t ldv, void* stream);

/* Attention of the jobs' rows, at positions `at` (NULL: their indices), over
 * all rows of their slot up to their own: row i of a job sees the rows 0 ..
 * past + i. q, out, n_heads as in cc_attend_pages. Where marks is given and
 * observe > 0, the weights w of the slot's rows r = 0 .. past + n - 1 become
 *   fade * w[r] + the sum over the job's last `observe` rows i that see r, and
 *   over the query heads of the kv head, of softmax(q_i . k / sqrt(D))[r]
 * (0 <= fade <= 1; 0: what was there does not matter). One job a slot, and no
 * page in two of the call's slots (its marks are one page's). The order of the
 * sums follows from the call's jobs alone: the same call gives the same bits. A
 * row that sees no row (its pages are outside the cache) gives 0 and adds
 * nothing. An output value's error is relative to the largest finite |v| of its
 * 32 channels among the rows that the job sees; a row that sees one that is no
 * finite number has NaN in these 32 channels. A query row and head with a value
 * that is no number, or that sees such a key, has NaN in its output and, if it
 * counts, in the weights of the rows that it sees, and in no others. Keys and
 * values of the cache are below 2^96. `workspace`: cc_weigh_workspace
 * bytes for the same jobs (0: the call would be refused), 16-byte aligned, of
 * any contents; two calls that may overlap need two. */
size_t cc_weigh_workspace(cc_ctx* ctx, const cc_cache* cache, const cc_rows* jobs, int32_t njobs, int32_t n_heads,
                          int32_t observe);
cc_status cc_attend_weigh(cc_ctx* ctx, const cc_cache* cache, const cc_positions* at, const cc_marks* marks,
                          const cc_rows* jobs, int32_t njobs, int32_t n_heads, int32_t observe, float fade, const float* q,
                          int64_t ldq, float* out, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream);

/* Of a slot's `rows` rows each kv head is to keep `keep`, and the slot's chat
 * has seen `seen` tokens. Host memory, read during the call. */
typedef struct cc_keep {
    int32_t slot, rows, keep, seen;
} cc_keep;

/* Gives up rows - keep rows of each kv head of the jobs' slots (none where rows
 * <= keep). Kept are the rows whose token is among the chat's first `sink`
 * (token < sink) or latest `recent` (token >= seen - recent; where these are
 * more than `keep`, the lower rows of them), then those with the largest
 * weight, ties to the lower row; a weight that is no number, and a row whose
 * page is outside the cache, counts least. The rows below `keep` that stay,
 * stay where they are; in row order, the i-th row from `keep` on that stays
 * moves to the i-th row below `keep` that goes, with its codes, scales and
 * marks, and rows from `keep` on are left as they were. So a slot's kv heads
 * hold different tokens in its rows 0 .. keep - 1, in no order; the pages
 * behind them are the caller's again, and cc_kv_append, cc_attend_pages and a
 * context's own passes (see cc_cache_of), which take a row's index for its
 * position, no longer fit the slot. Key bounds
 * are not touched (cc_kv_bounds makes them anew). 1 <= keep, sink >= 0, recent
 * >= 0; one job a slot, and no page that another slot reads (its rows are
 * written over). `workspace`: cc_evict_workspace bytes (may be 0 even for a
 * call that is not refused), as above. */
size_t cc_evict_workspace(const cc_cache* cache, const cc_keep* jobs, int32_t njobs);
cc_status cc_kv_evict(cc_ctx* ctx, const cc_cache* cache, const cc_marks* marks, const cc_keep* jobs, int32_t njobs,
                      int32_t sink, int32_t recent, void* workspace, size_t workspace_bytes, void* stream);

/* What a call asks of each of its rows: device arrays [rows], or NULL where
 * none asks for it. The meaning is the reference's sampler's
 * (web/model/sampling.js:57-215) with two more cuts, biases and masks, but:
 * an id that a list repeats is penalised once for its counts' sum (there once
 * an entry); a count of 0 is no entry (there rep and pres apply); a row with
 * no token left gives -1 (there its first or last token); and the draw's sums
 * are of f64 weights as cc_sample says (there the walk adds their f32 copies,
 * so a u within about 2^-23 of a border may fall to the other side).
 *   temp       0 or below: greedy
 *   top_k      0 or below, or vocab and more: off
 *   top_p      1 and more: off;  min_p  0: off (at most 1 counts)
 *   rep, freq, pres   penalties of the tokens in the row's history (1, 0 and 0:
 *              none); one token's frequency penalty is at most freq_cap
 *   pen_at [rows+1], pen_ids [n_pen], pen_counts [n_pen] or NULL: row r's
 *              history is the entries [pen_at[r], pen_at[r+1]); an entry counts
 *              pen_counts, or 1, and an id's entries add up, to 2^32 - 1 at
 *              most (0 or below: no entry)
 *   bias_at [rows+1], bias_ids, bias [n_bias]: added to the row's logits; of an
 *              id's entries the last counts
 *   mask [n_masks][mask_words], mask_of [rows]: bit t%32 of word t/32 allows
 *              token t to the rows of that mask (mask_of out of range: every
 *              token); mask_words >= ceil(vocab/32)
 *   u          the random numbers, in [0, 1)
 * Ids outside the vocabulary and entries outside the lists are passed over. */
typedef struct cc_sampling {
    const float* temp;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* rep;
    const float* freq;
    const float* pres;
    float freq_cap;
    const int32_t* pen_at;
    const int32_t* pen_ids;
    const int32_t* pen_counts;
    int32_t n_pen;
    const int32_t* bias_at;
    const int32_t* bias_ids;
    const float* bias;
    int32_t n_bias;
    const uint32_t* mask;
    int32_t mask_words, n_masks;
    const int32_t* mask_of;
    const double* u;
} cc_sampling;

/* The rows' logits with penalties, biases and masks: with c a token's count
 * in the row's history, x > 0 ? x / rep : x * rep, less pres + min(freq * c,
 * freq_cap), where c > 0; plus its bias; -inf where the mask bars it (whatever
 * the logit, NaN too). In f64 steps, rounded to f32 once; untouched logits keep
 * their bits. logits f32 [rows][vocab], ld floats from row to row; out alike
 * with ldo, and may be logits itself (same ld), or else shares no memory with
 * it. vocab at most 2^20. */
cc_status cc_logits_adjust(cc_ctx* ctx, const float* logits, int64_t ld, int32_t rows, int32_t vocab,
                           const cc_sampling* sampling, float* out, int64_t ldo, void* stream);
/* Draws a token of each row of logits, which stay as they are. Of the adjusted
 * row a (a NaN counts as -inf), s = f32(a / temp), a finite value stays finite;
 * kept are, in this order, the s that reach the top_k-th largest, of those the
 * s that reach the largest value above (and with) which lies top_p of their
 * weight exp(s), and of those exp(s - max) >= min_p; equal values are kept or
 * cut together. The token is the first, in id order, at which the running sum
 * of the kept weights is above u times their sum. Weights are held to 2^-42 of
 * the row's largest one and summed exactly; in a row without cuts, to 2^-42 of
 * the largest among the same 4096 tokens, and each 4096 tokens' sum to 2^-42
 * of the row's largest. A row's result does not depend on the call's other
 * rows. ids gets the token, probs (may be NULL) the probability it was drawn
 * with. Greedy: the first maximum of a, 1. A row with nothing above -inf:
 * -1, 0. `workspace`: cc_sample_workspace bytes
 * (0: the shape would be refused), 16-byte aligned, of any contents; two calls
 * that may overlap need two. */
size_t cc_sample_workspace(int32_t rows, int32_t vocab, const cc_sampling* sampling);
cc_status cc_sample(cc_ctx* ctx, const float* logits, int64_t ld, int32_t rows, int32_t vocab,
                    const cc_sampling* sampling, int32_t* ids, float* probs, void* workspace, size_t workspace_bytes,
                    void* stream);

/* cc_sample over the last pass's `rows` sampled rows (those cc_read_logits
 * reads), for samplers that need whole rows: the token is drawn where the
 * logits are, where the reference reads the rows back (web/model/stage.js:
 * 1428-1436). `sampling` holds HOST pointers here, read during the call; ids
 * and probs (may be NULL) are host memory, written when the call returns. */
cc_status cc_sample_pass(cc_ctx* ctx, int32_t rows, const cc_sampling* sampling, int32_t* ids, float* probs);

#ifdef __cplusplus
}
#endif
#endif
