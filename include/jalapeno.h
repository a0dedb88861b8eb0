/*
 * jalapeno.h -- C ABI of the B200 speculative-decoding engine for Qwen3.
 *
 * This ABI replaces the reference engine crate's public Rust API
 * (fawwaz46/jalapenos-at-home, engine/src/lib.rs:16-21) and its native GPU
 * bridge (engine/src/gpu.rs:19-42 -> engine/src/gpu.m:21-128).  Each entry
 * point names the reference item it stands in for.
 *
 * Conventions
 *  - Every call returns jl_status; JL_OK is 0.  On failure,
 *    jl_last_error() returns a thread-local message (never NULL).
 *  - Token ids are uint32_t (the reference uses usize; Qwen3's vocabulary
 *    fits in 32 bits).
 *  - The caller owns every host buffer it passes; the library owns device
 *    memory.  Handles are not thread safe: use one handle from one thread at
 *    a time.  Different handles are independent (one model per GPU replica).
 *  - There is no CPU fallback: calls that compute fail with
 *    JL_ERR_NO_DEVICE when no CUDA device is present.
 */
#ifndef JALAPENO_H
#define JALAPENO_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum jl_status {
    JL_OK = 0,
    JL_ERR_INVALID_ARG = 1, /* reference: assert!/panic on bad arguments */
    JL_ERR_FORMAT = 2,      /* reference: Err(...) from try_load / Mxfp4::validate */
    JL_ERR_OOM = 3,         /* reference: "could not allocate GPU memory" panic */
    JL_ERR_CUDA = 4,        /* reference: gpu_finish() returning -1 (gpu.m:114-128) */
    JL_ERR_TIMEOUT = 5,     /* a bounded device wait gave up */
    JL_ERR_IO = 6,          /* reference: io::Error from try_load */
    JL_ERR_NO_DEVICE = 7    /* no CUDA device: this engine has no CPU path */
} jl_status;

/* Thread-local description of the last failure on this thread. */
const char* jl_last_error(void);
/* Library version string, e.g. "0.1.0 sm_100a". */
const char* jl_version(void);
/* Number of visible CUDA devices (0 when none); never fails. */
int jl_device_count(void);

/* ------------------------------------------------------------------------
 * Weights on the host: engine::load / try_load (engine/src/lib.rs:85-202),
 * Tensor / Mxfp4 / Weights (lib.rs:27-71, mxfp4.rs:5-26).  Needs no GPU.
 * ---------------------------------------------------------------------- */

typedef struct jl_weights jl_weights;

typedef enum jl_dtype { JL_BF16 = 0, JL_MXFP4 = 1 } jl_dtype;

typedef struct jl_tensor_view {
    const char* name;        /* HF name without the .mxfp4_* suffix */
    jl_dtype dtype;
    int ndim;                /* 1 or 2 */
    size_t shape[2];         /* logical shape: [rows, cols] (cols in elements) */
    const uint16_t* bf16;    /* JL_BF16: shape product bf16 values, else NULL */
    const uint8_t* packed;   /* JL_MXFP4: rows*cols/2 bytes, low nibble = even index */
    const uint8_t* scales;   /* JL_MXFP4: rows*cols/32 E8M0 bytes (bias 127) */
} jl_tensor_view;

/* Reads every *.safetensors file of `dir` (sorted by name), with the
 * reference loader's validation: header <= 1e8 bytes, offsets in range,
 * BF16 tensors (U16 allowed in "jalapenos-mxfp4-v1" files), .mxfp4_packed /
 * .mxfp4_scales pairs, no duplicates, no orphaned scales, no NaN scale. */
jl_status jl_weights_load(const char* dir, jl_weights** out);
void jl_weights_free(jl_weights* w);
size_t jl_weights_count(const jl_weights* w);
/* i-th tensor in name order. */
jl_status jl_weights_at(const jl_weights* w, size_t i, jl_tensor_view* view);
jl_status jl_weights_get(const jl_weights* w, const char* name, jl_tensor_view* view);

/* ------------------------------------------------------------------------
 * Models on the GPU: Model::load / load_with_prefill (engine/src/model.rs:
 * 54-108) with Backend::Gpu, GpuModel::new (engine/src/gpu.rs:336-428).
 * ---------------------------------------------------------------------- */

typedef struct jl_model jl_model;
typedef struct jl_cache jl_cache;

typedef enum jl_kv_dtype { JL_KV_BF16 = 0, JL_KV_F32 = 1 } jl_kv_dtype;

typedef struct jl_model_options {
    int device;              /* CUDA device ordinal (default 0) */
    jl_kv_dtype kv_dtype;    /* KV cache element type (default bf16) */
    size_t kv_pool_tokens;   /* KV page pool capacity in tokens; 0 = context limit + 1024 */
    size_t max_pass_rows;    /* largest rows per forward pass; 0 = 4096 */
} jl_model_options;

/* Fills `o` with the defaults above. */
void jl_model_options_default(jl_model_options* o);

/* Loads config.json (num_hidden_layers, max_position_embeddings,
 * eos_token_id) and every .safetensors file of `dir`, uploads to the GPU.  bf16 and MXFP4
 * tensors may be mixed; a tied lm_head (absent or equal to the embedding
 * table) is stored once.  Every header is checked before any payload is
 * read (the checks and messages of jl_weights_load); payloads then go from
 * the files to the device through two 16 MB pinned buffers, so host memory
 * never holds the checkpoint.  opts may be NULL.
 * Replaces Model::load (engine/src/model.rs:55-57). */
jl_status jl_model_load(const char* dir, const jl_model_options* opts, jl_model** out);

/* Architecture of a seeded synthetic model (no file I/O): the same tensors a
 * checkpoint written from the seeded stream would hold.  Used by benchmarks
 * and tests; weights are generated on the GPU. */
typedef struct jl_synth_config {
    int layers, hidden, q_heads, kv_heads, inter, vocab;
    int tied;                /* 1: lm_head is the embedding table */
    int max_positions;       /* config.json max_position_embeddings */
    int eos;                 /* config.json eos_token_id */
    uint64_t seed;
    int mxfp4;               /* 1: q/k/v/o/gate/up/down quantized to MXFP4 */
    int mxfp4_embed;         /* 1: embedding and lm_head quantized too */
} jl_synth_config;
jl_status jl_model_synthesize(const jl_synth_config* cfg, const jl_model_options* opts,
                              jl_model** out);
void jl_model_free(jl_model* m);

typedef struct jl_model_info {
    int layers, hidden, q_heads, kv_heads, inter, vocab, max_positions, eos;
    int tied;
    int mxfp4_projections;   /* 1 when the layer projections are MXFP4 */
    int mxfp4_head;          /* 1 when the output table is MXFP4 */
    size_t weight_bytes;     /* bytes of weights resident on the GPU */
    size_t pass_bytes;       /* weight bytes one single-row forward pass reads */
    size_t kv_bytes_per_token;
} jl_model_info;
jl_status jl_model_info_get(const jl_model* m, jl_model_info* info);

/* Copies one weight tensor back to the host in its device format (for
 * tests).  bf16: rows*cols*2 bytes; MXFP4: packed then scales. */
jl_status jl_model_read_tensor(const jl_model* m, const char* name, void* dst, size_t cap,
                               size_t* written);

/* ------------------------------------------------------------------------
 * KV cache: Model::cache / KvCache::truncate (engine/src/model.rs:37-52,
 * 124-133), GpuCache (engine/src/gpu.rs:272-300).  Pages of the model's
 * pool are taken as the sequence grows; truncation only moves the length.
 * ---------------------------------------------------------------------- */

jl_status jl_cache_create(jl_model* m, jl_cache** out);
void jl_cache_free(jl_cache* c);
size_t jl_cache_len(const jl_cache* c);
/* len must not exceed the current length (KvCache::truncate asserts). */
jl_status jl_cache_truncate(jl_cache* c, size_t len);

/* A new cache that continues from the first `len` positions of `c` (at most
 * its length).  The two share full pages, and the page that `len` ends in is
 * copied; a cache that later writes into a shared page (after a truncation)
 * first gets a copy of its own, so neither sees the other's tokens.  Pages go
 * back to the pool with the last cache that holds them.  No counterpart in the
 * reference, whose caches are contiguous. */
jl_status jl_cache_fork(jl_cache* c, size_t len, jl_cache** out);
/* After jl_predict_tree: keeps `n` of the tree's nodes, a path from a child of
 * the committed positions down (each entry a child of the one before it), moves
 * their keys and values together and adds them to the length.  n == 0 keeps
 * none.  Any other pass on the cache, a truncation or this call drops the rest
 * of the tree. */
jl_status jl_cache_compact(jl_cache* c, const uint32_t* path, size_t n);

/* ------------------------------------------------------------------------
 * Forward passes: Model::predict / next_token / hidden (model.rs:143-240),
 * GpuModel::run (gpu.rs:544-634).  One host sync per call.
 * ---------------------------------------------------------------------- */

/* Appends `n` tokens to `c` and predicts after the last row (all == 0, one
 * id) or after every row (all != 0, n ids).  out_logits (nullable) receives
 * [rows_predicted, vocab] f32 logits. */
jl_status jl_predict(jl_model* m, jl_cache* c, const uint32_t* ids, size_t n, int all,
                     uint32_t* out_ids, float* out_logits);
/* jl_predict for a speculative loop's draft step: n = 1 or 2 tokens,
 * predicting after the last, through the kernels the loop's draft passes
 * run (on a model whose layer projections are all MXFP4, CUDA-core
 * projections with rounding of their own; otherwise the same pass as
 * jl_predict).  Stands in for the draft's proposal passes of
 * generate_scheduled (engine/src/speculative.rs:84-92, 136-138, which call
 * Model::predict); it lets callers check those kernels' logits. */
jl_status jl_predict_draft(jl_model* m, jl_cache* c, const uint32_t* ids, size_t n,
                           uint32_t* out_id, float* out_logits);
/* Verifies a tree of drafted tokens in one pass: node i holds ids[i] and
 * follows node parents[i] (an earlier node, or -1: the committed positions), and
 * out_ids[i] is the model's next token after the committed positions and node
 * i's path.  A chain (parents -1, 0, 1, ..) predicts what jl_predict with `all`
 * set does, up to the rounding of other kernels (logits within 2e-4 relative L2
 * on a bf16 pool): where a row's two best logits are nearer than that, the two
 * calls may name different tokens, and decoding by trees may leave the stream
 * that jl_generate or jl_generate_speculative gives.  1..JL_TREE_MAX_NODES nodes, at most max_pass_rows, and
 * length + n within the context limit.  The length stays; jl_cache_compact
 * keeps a path.  The reference verifies chains only (speculative.rs:95-97).
 * out_logits (nullable) receives [n, vocab] f32 logits. */
jl_status jl_predict_tree(jl_model* m, jl_cache* c, const uint32_t* ids, const int32_t* parents, size_t n,
                          uint32_t* out_ids, float* out_logits);
/* Model::next_token (model.rs:203-205): predict after a fresh prompt. */
jl_status jl_next_token(jl_model* m, const uint32_t* ids, size_t n, uint32_t* out_id);
/* Model::hidden (model.rs:143-154): residual stream after `layers` layers
 * for `n` tokens on a fresh cache, [n, hidden] f32. */
jl_status jl_hidden(jl_model* m, const uint32_t* ids, size_t n, size_t layers, float* out);

/* ------------------------------------------------------------------------
 * Generation: Model::generate (model.rs:268-285), generate_speculative /
 * generate_scheduled (speculative.rs:32-143), DraftSchedule (scheduler.rs).
 * ---------------------------------------------------------------------- */

/* Greedy decode.  out receives prompt + generated ids (capacity `cap`,
 * which must be >= n + count); *out_len is set to their number. */
jl_status jl_generate(jl_model* m, const uint32_t* prompt, size_t n, size_t count,
                      uint32_t* out, size_t cap, size_t* out_len);

typedef struct jl_schedule {
    uint32_t gamma;          /* initial draft length */
    uint32_t max_gamma;      /* adaptive upper bound (== gamma when fixed) */
    int adaptive;
} jl_schedule;
/* DraftSchedule::fixed (scheduler.rs:9-16): gamma must be positive. */
jl_status jl_schedule_fixed(uint32_t gamma, jl_schedule* out);
/* DraftSchedule::adaptive (scheduler.rs:18-27): 0 < initial <= maximum. */
jl_status jl_schedule_adaptive(uint32_t initial, uint32_t maximum, jl_schedule* out);

typedef struct jl_round_stats {
    uint32_t gamma, drafted, accepted, next_gamma; /* RoundStats (speculative.rs:13-19) */
} jl_round_stats;

typedef enum jl_spec_mode {
    JL_SPEC_DEVICE = 0,      /* whole loop on the GPU in one CUDA graph, one host sync */
    JL_SPEC_HOST = 1         /* reference control flow on the host, one sync per pass */
} jl_spec_mode;

typedef struct jl_spec_options {
    jl_spec_mode mode;
    /* Oracle-draft mode (benchmarks): when oracle_stream is non-NULL, the
     * draft model still runs every pass but its prediction for position P is
     * replaced by oracle_stream[P] (P < oracle_len), or with probability
     * oracle_p by a uniform id drawn from (oracle_seed, P). */
    const uint32_t* oracle_stream;
    size_t oracle_len;
    double oracle_p;
    uint64_t oracle_seed;
} jl_spec_options;
void jl_spec_options_default(jl_spec_options* o);

typedef struct jl_spec_result {
    /* caller-provided outputs */
    uint32_t* tokens;        /* prompt + generated ids, capacity tokens_cap */
    size_t tokens_cap;
    jl_round_stats* rounds_out; /* per-round stats, capacity rounds_cap (nullable) */
    size_t rounds_cap;
    /* filled by the call (SpeculativeResult, speculative.rs:21-30) */
    size_t n_tokens;
    size_t drafted, accepted, rounds;
    size_t prefill_passes, draft_passes, verify_passes;
    double prefill_ms;       /* both prefills, GPU time */
    double decode_ms;        /* everything after prefill, GPU time */
    double draft_ms, verify_ms; /* per phase (JL_SPEC_HOST only; 0 otherwise) */
} jl_spec_result;

/* The projections of one layer as the forward pass runs them: the
 * reference's public matmul (engine/src/lib.rs:240-266, y = x . W^T) applied
 * to `rows` f32 input rows, in the fused forms this engine uses.
 *   JL_PROJ_QKV     y = [x.Wq^T | x.Wk^T | x.Wv^T]   (q_width + 2*kv_width)
 *   JL_PROJ_O       y = x . Wo^T                      (hidden)
 *   JL_PROJ_GATE_UP y = silu(x.Wgate^T) * (x.Wup^T)   (intermediate, lib.rs:459-463)
 *   JL_PROJ_DOWN    y = x . Wdown^T                   (hidden)
 *   JL_PROJ_HEAD    y = x . Whead^T                   (vocab; layer ignored)
 * Inputs are NOT normalised first.  rows must be at most 16. */
typedef enum jl_projection {
    JL_PROJ_QKV = 0, JL_PROJ_O = 1, JL_PROJ_GATE_UP = 2, JL_PROJ_DOWN = 3, JL_PROJ_HEAD = 4
} jl_projection;
jl_status jl_project(jl_model* m, int layer, jl_projection which, const float* x, size_t rows,
                     float* y);

/* jl_project for callers that cannot allocate device memory when they call
 * it (a host running under a fixed device-memory reservation, or code that
 * cannot take cudaMalloc's implicit synchronisation).  No counterpart in the
 * reference: it exists for this engine's C ABI only.
 *   x: device pointer, rows x input width f32; y: device pointer, rows x
 *   output width f32 (widths as for jl_project); stream: a cudaStream_t of
 *   m's device, or NULL for the model's own stream.
 * MXFP4 projections on the tensor-core path only; rows 1..8.  All scratch
 * comes from one fixed 4 MiB device array per device (no allocation of any
 * kind); a projection whose scratch would exceed it is rejected with
 * JL_ERR_INVALID_ARG.  Calls share that array, so calls that overlap on
 * the GPU race.  Creating or loading a model on a device sets the array up
 * (module load, address lookup, a pinned flag word), so no call loads or
 * allocates anything.
 * Returns after the projection has finished (the stream is synchronised). */
jl_status jl_project_noalloc(jl_model* m, int layer, jl_projection which, const float* x,
                             size_t rows, float* y, void* stream);

/* ------------------------------------------------------------------------
 * Operators of tree-shaped speculation on device memory the caller owns.
 * The reference drafts chains (speculative.rs:79-97) and grows its caches in
 * place; these operators serve hosts that draft a tree of tokens, fork a
 * sequence, or keep their own pages in the engine's layout.
 *
 * Conventions of this section
 *  - Pointers are device pointers unless the text says otherwise, all on the
 *    device that holds the pool; calls run there whichever device is current
 *    (and leave the current device as it was).
 *  - Calls are asynchronous on `stream`, a cudaStream_t (NULL: the device's
 *    legacy default stream).  They allocate nothing, keep nothing from one
 *    call for the next and can be captured into a CUDA graph.  Calls on
 *    different streams are independent as long as their buffers are.
 *  - A sequence's position p lies in page page_table[p / 64] of the pool, at
 *    row p % 64.  Page ids outside [0, pages) and positions past the table
 *    are never dereferenced: reads of them act as masked positions, writes
 *    are skipped.
 *  - `status` (nullable) points to a device int that the kernels OR bits
 *    into: 1 a page id outside the pool, 2 an index or length out of range
 *    (the part out of range was skipped), 4 a bounded device wait gave up
 *    (the outputs of that call are not valid).
 * ---------------------------------------------------------------------- */

/* Pages of keys and values, [page][kv_head][64][128] of `dtype` for K and
 * for V, 16-byte aligned.  Calls that work on every layer find layer l's
 * pages layer_stride bytes times l behind k and v. */
typedef struct jl_kv_pages {
    void* k;
    void* v;
    size_t layer_stride;     /* a multiple of 16; ignored with one layer */
    int layers;              /* 1 for the calls that work on one layer */
    int pages;
    int kv_heads;
    jl_kv_dtype dtype;
} jl_kv_pages;

/* Per-head RMSNorm and rotation of queries and keys, and the append of keys
 * and values to the cache, in one pass over the q|k|v rows of a projection
 * (lib.rs:291-321, 363-396).  A row's rotation (pos) and its place in the
 * sequence (slot) are separate: the nodes of a drafted tree at one depth
 * share a position, and each has a slot of its own.
 *   y = x / sqrt(mean(x^2) + eps) * w, then for i < 64
 *   (y[i], y[i + 64]) -> (y[i] cos - y[i + 64] sin, y[i + 64] cos + y[i] sin)
 * in f32, rounded once into q or the pool; values are stored as they come.
 * A row whose pos lies outside [0, positions) is skipped whole (status 2).
 * Two rows must not append to the same place. */
typedef struct jl_norm_rope {
    jl_kv_pages pool;          /* one layer */
    int rows, q_heads;
    jl_kv_dtype dtype;         /* type of the qkv and q rows */
    const void* qkv;           /* [rows][qkv_ld]: q heads, k heads, v heads, 128 each; 16-byte aligned */
    size_t qkv_ld;             /* elements from row to row, a multiple of 8 */
    void* q;                   /* [rows][q_ld]: the rotated queries; may be qkv itself with q_ld == qkv_ld */
    size_t q_ld;               /* a multiple of 8 */
    const uint16_t* q_norm;    /* bf16 [128]; NULL: queries are rotated without a norm */
    const uint16_t* k_norm;    /* bf16 [128]; NULL: keys are rotated without a norm */
    float eps;
    const float* rope;         /* [positions][64][2]: cos and sin of each angle */
    int positions;
    const int32_t* pos;        /* [rows] rotation position */
    const int32_t* slot;       /* [rows] position in the sequence; negative: no append.  NULL: pos */
    const int32_t* seq;        /* [rows] sequence (row of page_table).  NULL: sequence 0 */
    const int32_t* page_table; /* [seqs][max_pages] */
    int seqs, max_pages;
    int32_t* status;
} jl_norm_rope;
jl_status jl_qk_norm_rope(const jl_norm_rope* a, void* stream);

/* Most nodes a tree may have. */
#define JL_TREE_MAX_NODES 256
/* Workspace that is enough for every jl_tree_attention call. */
#define JL_TREE_WORKSPACE_BYTES ((size_t)48 << 20)

/* Attention of the nodes of drafted trees over the paged cache
 * (lib.rs:401-441 for rows that do not form a chain).  Sequence s has the
 * query rows row_start[s] .. row_start[s + 1] - 1, one per node, and ctx[s]
 * committed positions that every node sees; node j's key and value lie at
 * position ctx[s] + j and are seen by the nodes whose mask has bit j (a
 * node's own bit included: nothing is added to the mask).  Without a mask
 * the nodes form a chain: node i sees nodes 0..i, as in a prompt, a decode
 * step or a linear verify pass.
 *   out = sum over seen p of softmax(q . k_p * scale) v_p, rounded once into
 *   the output type; lse = log of the sum of exp(q . k_p * scale).
 * Scores, maxima and sums are f32; q . k_p * scale must stay below 2^30.  The
 * exponential is off by 2^-22 of itself, and weights below 2^-126 of the row's
 * largest are zero.  f32 rows: q, k, v and the weights keep 24 bits.  bf16 rows:
 * the weights keep 17 bits and an f32 pool's values 16, both rounded to nearest.
 * The tensor core's additions cut off, so long sums are carried on in f32 outside
 * it: what is lost stays below 6e-6 of the weighted mean of |v| for f32 rows, and
 * below 4e-5 before the rounding for bf16 rows, whatever the length.
 * A row that sees nothing gets zeros and an lse of -infinity.  Whatever lies
 * in positions that a row does not see, infinities and NaN included, does
 * not reach its output; a value that is not finite in a position that it sees
 * makes that dim of its output infinite or NaN, whatever the position's
 * weight.  Rows from row_start[seqs] on are not written.
 * The sum is split between CTAs by the width of the page table and the
 * lengths of the whole batch, in a fixed order: the same inputs give the same
 * bits, but a row's last bits may differ in another batch or with another
 * max_pages.  A table no wider than the batch needs is fastest. */
typedef struct jl_tree_attn {
    jl_kv_pages pool;          /* one layer */
    int rows, q_heads;         /* q_heads a multiple of pool.kv_heads, at most 128 per kv head */
    jl_kv_dtype dtype;         /* type of the q and out rows */
    const void* q;             /* [rows][q_ld], 16-byte aligned */
    size_t q_ld;               /* elements from row to row, a multiple of 8 */
    void* out;                 /* [rows][out_ld]; may be q itself with out_ld == q_ld */
    size_t out_ld;             /* a multiple of 8 */
    float* lse;                /* [rows][q_heads], or NULL */
    int seqs;
    int max_nodes;             /* largest tree of the batch, 1..JL_TREE_MAX_NODES; CTAs are set
                                  aside for its rows in every sequence, so no larger than needed */
    const int32_t* row_start;  /* [seqs + 1] */
    const int32_t* ctx;        /* [seqs] */
    const uint64_t* mask;      /* [rows][mask_words]: bit j % 64 of word j / 64, or NULL */
    int mask_words;            /* at least max_nodes / 64, rounded up */
    const int32_t* page_table; /* [seqs][max_pages] */
    int max_pages;
    float scale;               /* 0: 1 / sqrt(128) */
    void* workspace;           /* 256-byte aligned, not shared by calls that may overlap */
    size_t workspace_bytes;    /* at least what jl_tree_attention_workspace says */
    int32_t* status;
} jl_tree_attn;
jl_status jl_tree_attention(const jl_tree_attn* a, void* stream);
/* Bytes of workspace the call needs (from its sizes alone; pointers may be
 * NULL except pool.k, which names the device; seqs or max_pages 0: for any), at most
 * JL_TREE_WORKSPACE_BYTES. */
jl_status jl_tree_attention_workspace(const jl_tree_attn* a, size_t* bytes);

/* Moves positions of sequences together in every layer: position ctx[s] + i
 * takes what position ctx[s] + path[s][i] held before the call, for
 * i < path_len[s] (the accepted path of a drafted tree; any order, entries
 * may repeat).  Positions behind it keep what they held. */
typedef struct jl_kv_compaction {
    jl_kv_pages pool;
    int seqs;
    const int32_t* ctx;        /* [seqs] */
    const int32_t* path;       /* [seqs][path_ld] node indices */
    int path_ld;               /* 1..JL_TREE_MAX_NODES */
    const int32_t* path_len;   /* [seqs], each at most path_ld */
    const int32_t* page_table; /* [seqs][max_pages]; a page that one sequence writes to is no other's */
    int max_pages;
    int32_t* status;
} jl_kv_compaction;
jl_status jl_kv_compact(const jl_kv_compaction* a, void* stream);

/* Copies n pages in every layer: the first rows[i] rows (1..64; rows NULL:
 * all 64) of page src[i] to page dst[i], K and V.  src, dst and rows are
 * host arrays, read before the call returns.  A page may be the source of
 * several copies; a page that is the destination of two, or both source and
 * destination, is an error. */
jl_status jl_kv_copy_pages(const jl_kv_pages* pool, const int32_t* src, const int32_t* dst,
                           const int32_t* rows, size_t n, void* stream);

/* ------------------------------------------------------------------------
 * Profiling.
 * ---------------------------------------------------------------------- */

/* Model::time_pass (engine/src/model.rs:242-266, the CLI's --time-rows):
 * prefills `prompt`, then times `reps` + 2 passes of `rows` tokens that
 * predict after every row (rolling the cache back after each), drops the
 * first two and returns the median wall and GPU milliseconds. */
jl_status jl_time_pass(jl_model* m, const uint32_t* prompt, size_t n, size_t rows, size_t reps,
                       double* wall_ms, double* gpu_ms);

/* Launches one projection kernel of `layer` for `rows` input rows `iters`
 * times back to back on the model's stream and returns the mean device time
 * per launch (CUDA events) and the weight bytes each launch reads.  On a
 * model whose decode pass is fused (every projection MXFP4), O, GATE_UP and
 * DOWN time the fused kernel that pass runs, on the input pieces a previous
 * pass left behind, and HEAD with a bf16 table the final norm + tensor-core
 * table + argmax kernels; otherwise the standalone projection.  No reference
 * counterpart: it feeds the per-kernel roofline report. */
jl_status jl_time_projection(jl_model* m, int layer, jl_projection which, int rows, int iters,
                             double* ms_per_launch, size_t* weight_bytes);

/* jl_time_pass for one row taking the path a speculative loop's draft step
 * takes (on a model whose draft steps have a path of their own; otherwise
 * the same as jl_time_pass with rows = 1).  No reference counterpart: it
 * feeds the profile of a speculative round. */
jl_status jl_time_pass_draft(jl_model* m, const uint32_t* prompt, size_t n, size_t reps,
                             double* wall_ms, double* gpu_ms);

/* Kernels one forward pass of `rows` rows (with its next-token prediction)
 * launches: `draft_step` nonzero for a speculative loop's draft step.  No
 * reference counterpart: it feeds the launch count of the benchmark. */
jl_status jl_pass_kernels(const jl_model* m, size_t rows, int draft_step, size_t* kernels);

/* Runs one device wait that nothing completes, bounded by `polls` polls
 * (1..2^20) of the poll loop every pass kernel's waits use, which then sets
 * the same error bit: returns JL_ERR_TIMEOUT with the bounded-wait message
 * and leaves the model usable.  No reference counterpart: it tests the
 * timeout path without faulting or hanging the GPU. */
jl_status jl_wait_probe(jl_model* m, uint32_t polls);

/* Chooses the kernel of prompt attention for the prompt passes recorded
 * after the call: tensor_cores = 1 (the default) runs it on tcgen05 MMAs
 * wherever the model allows (fused MXFP4 model, bf16 KV pool, GQA group of
 * 1, 2, 4 or 8), 0 keeps the CUDA-core kernel.  *active (may be NULL)
 * receives 1 when prompts now run on tensor cores.  No reference
 * counterpart: it lets tests compare the two kernels on identical inputs. */
jl_status jl_model_prompt_attention(jl_model* m, int tensor_cores, int* active);

/* Kernel phase timeline, from the diagnostic build of this library
 * (`make -C jalapenos-at-home_b200 timeline` -> lib/libjalapeno_timeline.so):
 * the decode-pass kernels stamp the GPU's nanosecond clock at fixed points
 * of their critical path.  jl_timeline_read copies the stamps of the last
 * recorded pass (jl_time_pass / jl_time_pass_draft record one pass and
 * replay it), launches x JL_TIMELINE_CTAS x JL_TIMELINE_POINTS values, 0
 * where a CTA or point did not stamp; `stamps` NULL returns the launch
 * count only.  JL_ERR_INVALID_ARG from the normal build.  No reference
 * counterpart: it backs the per-kernel phase profiles. */
#define JL_TIMELINE_CTAS 512
#define JL_TIMELINE_POINTS 8
jl_status jl_timeline_read(uint64_t* stamps, size_t cap, size_t* launches);
/* Kernel of launch i of that pass (NULL past the last). */
const char* jl_timeline_kernel(size_t launch);

/* generate_scheduled: both models share token ids; the target has the
 * final say, so the output equals jl_generate(target, ...) whenever the
 * forward pass is row-count invariant (it is here). opts may be NULL. */
jl_status jl_generate_speculative(jl_model* target, jl_model* draft, const uint32_t* prompt,
                                  size_t n, size_t count, const jl_schedule* schedule,
                                  const jl_spec_options* opts, jl_spec_result* result);

/* ------------------------------------------------------------------------
 * A batch of independent sequences on one GPU, decoded in lockstep rounds
 * (the benchmark configuration with a per-GPU batch of sequences).  The
 * reference engine has no batch call: it decodes one sequence per call
 * (model.rs:268-285, speculative.rs:43-143), and each sequence here gets
 * exactly the tokens and counters that call gives it alone.  Weights are
 * read once per round for the whole batch.
 * ---------------------------------------------------------------------- */
#define JL_MAX_BATCH 64

typedef struct jl_batch_stats {
    double prefill_ms;       /* every sequence's prefill, GPU time */
    double decode_ms;        /* the batched loop, GPU time */
    size_t rounds;           /* lockstep rounds */
    size_t target_passes;    /* target passes of up to 16 rows */
    size_t draft_passes;     /* draft passes of up to 16 rows */
} jl_batch_stats;

/* Greedy decode of `batch` sequences (1..JL_MAX_BATCH): prompts[i] holds
 * prompt_lens[i] ids.  results[i].tokens (capacity tokens_cap, at least
 * prompt_lens[i] + count or the context limit) receives prompt + generated
 * ids and n_tokens its length; the other result fields are zero except
 * verify_passes (passes the sequence took part in), prefill_ms and
 * decode_ms (the whole batch's).  stats may be NULL. */
jl_status jl_generate_batch(jl_model* m, size_t batch, const uint32_t* const* prompts,
                            const size_t* prompt_lens, size_t count, jl_spec_result* results,
                            jl_batch_stats* stats);

/* jl_generate_speculative for each of `batch` sequences: schedules[i] and
 * opts[i] (opts may be NULL; its mode is ignored, the loop runs on the
 * device) belong to sequence i, and results[i] is filled as that call
 * fills it, with prefill_ms and decode_ms the whole batch's.  batch x
 * (largest max_gamma + 1) must not exceed 512.  stats may be NULL. */
jl_status jl_generate_speculative_batch(jl_model* target, jl_model* draft, size_t batch,
                                        const uint32_t* const* prompts, const size_t* prompt_lens,
                                        size_t count, const jl_schedule* schedules,
                                        const jl_spec_options* opts, jl_spec_result* results,
                                        jl_batch_stats* stats);

#ifdef __cplusplus
}
#endif
#endif /* JALAPENO_H */
