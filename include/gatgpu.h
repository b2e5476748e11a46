/*
 * gatgpu.h -- C ABI of the MI355X (gfx950) three-layer multi-head GAT forward.
 *
 * One opaque context per device owns every device buffer: the destination-row
 * CSR graph, its degree schedule, three layers of weights and the per-layer
 * activations.  Host buffers stay owned by the caller.  No function throws;
 * each returns 0 (GATGPU_OK) or a negative error class, and
 * gatgpu_last_error() describes the failure.  A context is used by one host
 * thread at a time.
 *
 * The entry points replace the per-layer "paths" of the reference harness:
 *   run_path(path, g, p, q, s, input, w, hidden, panel, t, policy)
 *     baseline/bench/main.cpp:21-25 (path whitelist main.cpp:30)
 *   X_layer(const Graph&, const Param&, const Prepared&, [const Schedule&,]
 *           const std::vector<float>& input, Workspace&, bool hidden, Times&)
 *     baseline/include/gat.hpp:107-117
 * The graph container (u64 rowptr, u32 col, f32 x; baseline/include/gat.hpp:32-39)
 * and the weight layout (W[in][heads*dim] row-major, head h = columns
 * [h*dim,(h+1)*dim), aL/aR[heads*dim]; baseline/include/gat.hpp:42-48) are
 * taken unchanged.
 */
#ifndef GATGPU_H
#define GATGPU_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct gatgpu_ctx gatgpu_ctx;

/* Return codes.  The reference throws std::runtime_error for each of these
 * (baseline/src/common.cpp:6-49); its harness maps them to "FAIL msg", exit 1
 * (baseline/bench/main.cpp:184). */
enum {
    GATGPU_OK = 0,
    GATGPU_EINVAL = -1,     /* malformed argument, CSR, shape or option       */
    GATGPU_ESTATE = -2,     /* call order: graph/layer/input not set yet      */
    GATGPU_ENODEV = -3,     /* no usable HIP device / wrong architecture      */
    GATGPU_ENOMEM = -4,     /* device allocation failed                       */
    GATGPU_EDEVICE = -5,    /* a HIP call or kernel launch failed             */
    GATGPU_ENONFINITE = -6, /* NaN/Inf in features or weights                 */
    GATGPU_EOVERFLOW = -7   /* size product overflows (common.cpp:6-9)        */
};

/* Precision of a forward.  FP32: FP32 X, W, Z and softmax state (the
 * reference's ref_fp32 / standard_fp32).  BF16: RNE-rounded bf16 X and W,
 * FP32 MFMA accumulation, L/R from the FP32 accumulators, Z stored bf16,
 * FP32 score/max/exp/denominator/output accumulation (standard_bf16 with a
 * bf16 copy of Z; baseline/IMPLEMENTATION_CONTRACT.md sections 3.2-3.3).
 * On transform-first layers of 8 heads x 32 features R is instead the FP32
 * dot of the stored bf16 Z row with a_r, formed both in the projection and,
 * per edge, in the aggregation from the Z row it gathers anyway, so no R
 * values are gathered; the row max stays exact over those R values. */
enum { GATGPU_FP32 = 0, GATGPU_BF16 = 1 };

/* Dataflow of one layer.  TRANSFORM_FIRST projects Z = X W then aggregates Z
 * rows (standard_layer, baseline/src/baseline_standard.cpp:98-108).
 * AGGREGATE_FIRST gathers the layer's input rows instead of Z
 * (tfs_online_fused, implementation/src/gat_tfs_online.cpp:200-283); bf16
 * only, in <= 128, and head_dim 32 with 1, 2, 4 or 8 heads or 8 heads of 64.
 * For 8 heads it runs in the sum form of tfs_online_fused: U_h = sum_j p_jh X_j
 * per row (FP32 sums of the bf16 rows, p entering as hi + lo bf16), then
 * (U_h / den_h) W_h on the MFMA units, with U_h / den_h entering as hi + lo
 * bf16 for FP32 outputs and as one bf16 for bf16-stored hidden outputs (the
 * rounding of a bf16 projection input); otherwise each gathered row is projected
 * and p (X_j W_h) summed, in the neighbour-step order of
 * baseline/src/baseline_tfs.cpp:16-110.  AUTO selects the sum form where it
 * applies (bf16) and the layer's bf16 Z table (n x heads x head_dim x 2 bytes)
 * exceeds 256 MB, and transform-first elsewhere.  gatgpu_model_forward with
 * AGGREGATE_FIRST uses it on the layers that support it and transform-first
 * on the others. */
/* TFS_B1 is the faithful neighbour-step TFS ("tfs_bf16",
 * baseline/src/baseline_tfs.cpp:16-110, max_prescan first): per step the
 * weighted source row p X_j is rounded to bf16 and multiplied by W_h with FP32
 * sums, the exact row max taken before any exponent.  Same shape limits as
 * AGGREGATE_FIRST; used for dataflow comparisons, not selected by AUTO. */
enum { GATGPU_AUTO = 0, GATGPU_TRANSFORM_FIRST = 1, GATGPU_AGGREGATE_FIRST = 2, GATGPU_TFS_B1 = 3 };

/* Stage selectors for gatgpu_get_stage (Workspace fields, gat.hpp:96-106). */
enum {
    GATGPU_STAGE_Z = 0,    /* [n][heads*dim] projected features (TF only)   */
    GATGPU_STAGE_LEFT = 1, /* [n][heads]                                     */
    GATGPU_STAGE_RIGHT = 2,/* [n][heads]                                     */
    GATGPU_STAGE_MAX = 3,  /* [n][heads] exact row max M = leaky(L + max R)  */
    GATGPU_STAGE_DEN = 4,  /* [n][heads] sum of exp(score - M)               */
    GATGPU_STAGE_OUT = 5,  /* [n][heads*dim] normalised (+ELU) layer output  */
    GATGPU_STAGE_XBF = 6   /* [n][in] the layer input rounded to bf16, as
                              convert() writes Workspace::xbf (common.cpp:
                              85-93): bf16 layers whose FP32 input the layer
                              rounds itself -- by the convert kernel, by the
                              projection (kept only with option
                              GATGPU_OPT_KEEP_INPUT_BF16) or into the
                              aggregate-first gather table.  Absent for a
                              chained bf16 input: that is the previous
                              layer's OUT stage, rounded in its epilogue.  */
};

/* Per-layer stage times in milliseconds, measured with HIP events on the
 * context's stream.  Field names follow gat::Times (baseline/include/gat.hpp:68-76).
 * normalize and activation are fused into the aggregation kernel on the GPU,
 * so their time is inside aggregate_ms and their fields read 0. */
typedef struct gatgpu_times {
    double convert_ms;
    double projection_ms;
    double lr_ms;
    double max_prescan_ms;
    double aggregate_ms;
    double normalize_ms;
    double activation_ms;
    double total_ms;
} gatgpu_times;

/* Options (gatgpu_set_option).  Thresholds are in-degrees. */
enum {
    GATGPU_OPT_BLOCK_ROW_MIN_DEGREE = 1, /* rows below are never split (default
                                            512, or 128 on graphs below 1M
                                            edges as long as options 1 to 3
                                            are at their defaults, 512 here;
                                            0: no such limit)                */
    GATGPU_OPT_SPLIT_ROW_MIN_DEGREE = 2, /* rows at/above are split over waves
                                            (default per kernel: 1024 sum form,
                                            1536 8-head, 2048 one-head; 512 on
                                            graphs below 16M edges, 128 in the
                                            8-head and one-head kernels below
                                            1M with the defaults; chunks
                                            doubled until the heaviest row has
                                            <= 96 of them, the degree with them
                                            (8-head) or at least 2 chunks (the
                                            others); a value applies to all,
                                            0 restores them)                  */
    GATGPU_OPT_SPLIT_CHUNK_EDGES = 3,    /* edges per split chunk (default per
                                            kernel: 256, 512, 1024; 256 below
                                            16M edges, 128 where rows of 128
                                            are split; scaled as above; a value
                                            >= 64 applies to all, 0 restores) */
    /* 4 is not a key: rows of small degree take one wave each like the rest
       (or share one with rows of equal degree, where a row needs fewer lanes). */
    GATGPU_OPT_KEEP_INPUT_BF16 = 5,      /* 1: bf16 transform-first layers also
                                            store the input rows their
                                            projection rounds (stage XBF);
                                            0 (default): they are rounded in
                                            registers only                    */
    GATGPU_OPT_FUSE_NEXT_PROJECTION = 6  /* 2: gatgpu_model_forward runs the
                                            projection of a bf16 one-head
                                            output layer (<= 60 classes over
                                            8 x 32 inputs) inside the previous
                                            layer's aggregation, on its output
                                            rows staged in LDS: Z, L and R of
                                            the output layer are bit-equal to
                                            the unfused run, and the hidden
                                            layer's OUT stage is not stored
                                            (gatgpu_stage_size gives 0, and a
                                            per-layer forward of the output
                                            layer chained on it fails).
                                            1 (default): the same on graphs of
                                            at least 16M edges, where it is the
                                            faster form; smaller graphs run
                                            unfused.
                                            0: every layer stores its output  */
};

/* ---- lifetime -------------------------------------------------------- */
/* Opens `device` (HIP ordinal), checks it is a gfx950, creates the stream. */
int gatgpu_create(int device, gatgpu_ctx** out);
/* Frees every device buffer; accepts NULL. */
int gatgpu_destroy(gatgpu_ctx* ctx);
/* Message of the last failure on ctx (or of the last failed create when ctx
 * is NULL).  Valid until the next call on the same context. */
const char* gatgpu_last_error(const gatgpu_ctx* ctx);

/* ---- static inputs (untimed, like load_graph/prepare: baseline/README.md:52) ---- */
/* The host checks of gatgpu_set_graph without a context or device
 * (Graph::validate, baseline/src/common.cpp:23-30): row[0] == 0, row[n] == e,
 * monotone rows, col[k] < n, 0 < n <= INT32_MAX, e <= 2^40, and every
 * in-degree below 2^32 (GATGPU_EOVERFLOW).  Rows are checked before sources.
 * The message is gatgpu_last_error(NULL). */
int gatgpu_validate_graph(uint64_t n, uint64_t e, const uint64_t* row, const uint32_t* col);
/* Validates (as gatgpu_validate_graph) and uploads the CSR, then builds the
 * degree schedule on the GPU.  Replaces load_graph + Graph::validate
 * (baseline/src/common.cpp:23-39) and degree_schedule (common.cpp:120-125). */
int gatgpu_set_graph(gatgpu_ctx* ctx, uint64_t n, uint64_t e, const uint64_t* row,
                     const uint32_t* col);
/* Uploads one layer (0..2) of weights and prepares its bf16 copy.  Replaces
 * Param::validate + prepare (common.cpp:45-49, 97-119): 0 < heads <= 8,
 * 0 < dim <= 64, 0 < in, all values finite. */
int gatgpu_set_layer(gatgpu_ctx* ctx, int layer, int in, int heads, int dim, const float* w,
                     const float* al, const float* ar);
/* Uploads the node features x[n][din] (Graph::x); all values finite. */
int gatgpu_set_input(gatgpu_ctx* ctx, uint64_t n, int din, const float* x);

/* ---- schedule -------------------------------------------------------- */
/* Copies the degree permutation (perm[sorted] = original row, ascending
 * (degree, id)) and neighbor_steps (sum over 16-row tiles of the last row's
 * degree), both computed on the GPU.  Either pointer may be NULL.
 * Replaces degree_schedule (baseline/src/common.cpp:120-125) and degree_perm
 * (implementation/src/gat_tfs_online.cpp:180-189). */
int gatgpu_degree_schedule(gatgpu_ctx* ctx, uint32_t* perm, uint64_t* neighbor_steps);
/* Copies the CSR in degree-sorted order: prow[k] = sum of degrees of
 * perm[0..k), pcol[prow[k]..prow[k+1]) = col[row[perm[k]]..row[perm[k]+1]). */
int gatgpu_permuted_csr(gatgpu_ctx* ctx, uint64_t* prow, uint32_t* pcol);
/* choose_R (implementation/src/gat_tfs_online.cpp:191-199) from the device
 * max degree: 128 if rho<32, 64 if rho<1024, 32 if rho<20000, else 16. */
int gatgpu_choose_R(gatgpu_ctx* ctx, int* r_out);

/* ---- forward --------------------------------------------------------- */
/* One layer (0..2).  `input` NULL chains from the device-resident output of
 * layer-1 run with the same precision (layer 0 reads the graph features);
 * non-NULL uploads a host FP32 [n][in] matrix first (outside the timing),
 * as run_path takes any `input` vector.  hidden != 0 applies ELU
 * (layers 0 and 1 of the model).  times may be NULL.
 * Replaces standard_layer / ref_layer / tfs_layer (gat.hpp:107-117) and
 * reference / tfs_online_fused (implementation/src/gat_online.cpp:167,
 * implementation/src/gat_tfs_online.cpp:200-202). */
int gatgpu_layer_forward(gatgpu_ctx* ctx, int layer, int precision, int dataflow, int hidden,
                         const float* input, gatgpu_times* times);
/* The three layers chained on device (hidden = layer < 2), timed from the
 * first kernel of layer 0 to the last of layer 2 with HIP events (the model
 * timer of baseline/bench/main.cpp:171-174).  logits (NULL allowed) receives
 * layer 2's FP32 [n][dim] output after the timer stops.  times (NULL allowed)
 * points at 3 per-layer records; total_ms (NULL allowed) gets the model time.
 * The per-stage events are recorded only when times is given: with total_ms
 * alone the forward carries two events, its first and its last.
 * dataflow applies to every layer (AUTO decides per layer; AGGREGATE_FIRST
 * falls back to transform-first on layers it does not support). */
int gatgpu_model_forward(gatgpu_ctx* ctx, int precision, int dataflow, float* logits,
                         gatgpu_times* times, double* total_ms);
/* ---- fixed-p operator ----------------------------------------------- */
/* Uploads a fixture's attention weights for `layer`: p[e][heads] (the
 * unnormalised exp weights, original CSR edge order) and den[n][heads].
 * Checks them as load_fixture does (baseline/src/common.cpp:186-193): all
 * finite, p in [0, 1], den equal to the row's sum of p within 1e-5 relative,
 * den > 0 on a non-empty row.  p is permuted to degree-sorted order on the
 * device.  set_graph and set_layer(layer) drop the fixture.  The GATFIX1 file
 * (common.cpp:171-194) is read by the host harness. */
int gatgpu_set_fixed_p(gatgpu_ctx* ctx, int layer, const float* p, const float* den);
/* The fixed-p operator of the reference harness (baseline/bench/main.cpp:
 * 103-150, "standard_op"): projection Z = XW in `precision`, then
 * out = (sum_e p[e] Z[col[e]]) * (den > 0 ? 1/den : 0) with the fixture's p
 * and den and no activation (standard_aggregate with fixed_p and finish,
 * baseline/src/baseline_standard.cpp:52-97).  dataflow TFS_B1 is the
 * reference's "tfs_op" of the same mode (tfs_aggregate with fixed_p,
 * baseline_tfs.cpp:16-110), AGGREGATE_FIRST the FP32-product variant; both
 * bf16 only.  input as in gatgpu_layer_forward.  Stages: Z (transform-first),
 * LEFT, RIGHT from the projection, DEN = the fixture's den, MAX zero, OUT FP32. */
int gatgpu_fixed_p_forward(gatgpu_ctx* ctx, int layer, int precision, int dataflow, const float* input,
                           gatgpu_times* times);

/* Copies a stage of the last forward of `layer` as FP32 (bf16 stages are
 * widened exactly). */
int gatgpu_get_stage(gatgpu_ctx* ctx, int layer, int which, float* host_out);
/* Size in floats of a stage buffer (0 if absent). */
int gatgpu_stage_size(gatgpu_ctx* ctx, int layer, int which, uint64_t* count);

/* Wall-clock times (ms) of the static steps, outside every forward timer
 * (the reference prints them as STATIC degree_sort_ms / model_prepare_ms and
 * COLD startup_before_inference_ms, baseline/bench/main.cpp:56,168-169;
 * baseline/README.md:52).  Each field holds its step's last run. */
typedef struct gatgpu_static_times {
    double graph_check_ms;   /* set_graph: host CSR validation (Graph::validate)      */
    double graph_h2d_ms;     /* set_graph: rowptr and col upload                     */
    double degree_sort_ms;   /* set_graph: degree schedule on the device (sort,
                                permuted CSR, relabelling, split tables)             */
    double model_prepare_ms; /* set_layer: checks, bf16 W, B_LR, fragment packing
                                and upload, summed over the layers set             */
    double input_h2d_ms;     /* set_input: feature checks and upload                 */
    double input_permute_ms; /* set_input: features gathered into degree order       */
    double logits_d2h_ms;    /* model_forward: the logits copied to the host         */
} gatgpu_static_times;
int gatgpu_get_static_times(gatgpu_ctx* ctx, gatgpu_static_times* out);

/* ---- allocation-free layer ------------------------------------------- */
/* No counterpart in the reference.  For callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops): the
 * transform-first gatgpu_layer_forward of `layer` on device-resident rows,
 * with every intermediate (bf16 input rows, Z, L, R, max, den, split-row
 * partial sums and arrival counters, and room for the output, which is taken
 * where `out` is not 16-byte aligned and copied from there) in one static
 * device array of GATGPU_STATIC_SCRATCH_BYTES per GPU, held until the process
 * ends.  It calls no allocator.
 *   x   device FP32 [n][in], original node order
 *   out device FP32 [n][heads*dim], original node order: the values
 *       gatgpu_get_stage(OUT) returns after gatgpu_layer_forward with the
 *       same input, precision and hidden (bf16 hidden outputs widened)
 * Graph, layer weights and options come from the context (set-up calls,
 * which do allocate).  The work is enqueued on the context's stream
 * (gatgpu_stream) and the call returns without waiting; the stages of the
 * context are not touched.  Rejects (GATGPU_EOVERFLOW, before any launch) a
 * layer whose intermediates exceed the array.  (On a graph below 1M edges a
 * layer that fits only with the 512-edge split takes that: the same values up
 * to the order of the sums.)  Every call on one GPU shares
 * that GPU's array: calls that overlap on one GPU (several contexts or host
 * threads, or streams not ordered against each other) race. */
#define GATGPU_STATIC_SCRATCH_BYTES (64u << 20)
int gatgpu_layer_forward_static(gatgpu_ctx* ctx, int layer, int precision, int hidden, const float* x,
                                float* out);
/* Bytes of the static array gatgpu_layer_forward_static would use for
 * `layer` of the context's graph.  GATGPU_ESTATE (and *bytes untouched) if
 * the graph or the layer's weights are not set. */
int gatgpu_static_scratch_need(gatgpu_ctx* ctx, int layer, int precision, int hidden, uint64_t* bytes);

/* ---- attention among the rows of segments ------------------------------ */
/* No counterpart in the reference.  Beside the attention over a graph's edges:
 * softmax attention in which every row of a segment (a graph or document of a
 * packed batch, or one sequence with its cached keys) attends to the keys of
 * its own segment, on device-resident rows, with its gradient.
 *
 * Segment s has q_len[s] query rows from q_begin[s] and k_len[s] key rows from
 * k_begin[s] of the caller's arrays.  Query i stands at position
 * pos = i + k_len - q_len among the keys.  For head h and the key/value head
 * h / (heads / kv_heads):
 *   x = scale q.k      y = cap > 0 ? cap tanh(x / cap) : x      s = y + bias
 *   out = sum_j p_j v_j,  p = softmax of s over the keys that the query sees
 *   lse = log sum exp s
 * GATGPU_MASK_FULL: every key is seen.  GATGPU_MASK_PREFIX: key j is seen if
 * j <= pos or j < prefix[s] (causal with a visible prefix).
 * GATGPU_BIAS_LINEAR: bias = -slope[h] |pos - j|, slope constant.
 * GATGPU_BIAS_TABLE: bias = table[h][min(d, buckets - 1)] with one byte d of
 * distance per pair (a shortest path, say); d = GATGPU_HIDDEN: not seen.  A
 * table entry of -infinity hides its pairs as well, and so does any of -1e6 or
 * below (beside a key of an ordinary score it weighs 0 anyway; the log-sum of a
 * row of nothing else has FP32 steps of 1/16 and more, too wide to form weights
 * from again).
 * A row that sees no key of finite score gets out = 0, lse = -infinity, and no
 * gradient.  Keys that are not seen add nothing, whatever they hold (NaN
 * included); a NaN or infinity in a seen value reaches that row's output.
 * Sums of weights times values are formed in FP32 before they are divided by
 * the weights' sum, with weights of up to 2^8: values beyond 1e30 may overflow.
 *
 * Storage: GATGPU_FP32 (products in FP32) or GATGPU_BF16 (bf16 rows, FP32
 * scores, softmax state and sums; the weights and, backward, the score
 * gradients are rounded to bf16 as operands of their products).  dim: a
 * multiple of 8, at most 128.  heads <= 64.
 *
 * All work is enqueued on the context's stream (gatgpu_stream) and calls return
 * without waiting; neither forward nor backward allocates, waits or copies, so
 * both can be captured into a HIP graph.  A captured call refers to its plan's
 * tables, the buffers and the workspace: keep them until the last replay, and
 * give graphs that may run at once workspaces of their own.  The same holds for
 * calls: two that overlap need two workspaces.  Arrays must lie on the context's
 * device.  Rows that belong to no segment are neither read nor written. */
enum { GATGPU_MASK_FULL = 0, GATGPU_MASK_PREFIX = 1 };
enum { GATGPU_BIAS_NONE = 0, GATGPU_BIAS_LINEAR = 1, GATGPU_BIAS_TABLE = 2 };
#define GATGPU_HIDDEN 255

typedef struct gatgpu_attention gatgpu_attention; /* a plan: shape and segments */
typedef struct gatgpu_attention_shape {
    int precision;        /* GATGPU_FP32 or GATGPU_BF16                          */
    int heads, kv_heads;  /* heads is a multiple of kv_heads                     */
    int dim;
    int mask, bias;
    int buckets;          /* GATGPU_BIAS_TABLE: 1 to 64                          */
    float scale;          /* > 0                                                 */
    float cap;            /* 0: none                                             */
} gatgpu_attention_shape;

/* Plans the segments (a host array each; prefix NULL: 0) and uploads the
 * tables of tiles.  Query rows of two segments must not overlap
 * (GATGPU_EINVAL); key rows may (a shared prefix in a cache), but such a plan
 * has no backward pass.  Lengths may be 0; q_len * heads / kv_heads and k_len
 * are at most 2^30.  The plan belongs to ctx and is destroyed before it. */
int gatgpu_attention_create(gatgpu_ctx* ctx, const gatgpu_attention_shape* shape, uint64_t segments,
                            const uint64_t* q_begin, const uint32_t* q_len, const uint64_t* k_begin,
                            const uint32_t* k_len, const uint32_t* prefix, gatgpu_attention** out);
/* Waits for the context's stream and frees the plan; accepts NULL. */
int gatgpu_attention_destroy(gatgpu_attention* plan);
/* Bytes of device workspace (16-byte aligned) a forward / backward call needs;
 * either may be NULL. */
int gatgpu_attention_workspace(const gatgpu_attention* plan, uint64_t* forward, uint64_t* backward);
/* Layout of the pair distances: segment s has q_len[s] rows of ld[s] bytes
 * (k_len rounded up to 16) from offset[s] on, `bytes` in all; any may be NULL.
 * (Offsets are those of tight packing in the order of the segments.) */
int gatgpu_attention_distances(const gatgpu_attention* plan, uint64_t* bytes, uint64_t* offset, uint32_t* ld);

/* Device arrays of one call.  Rows of `heads` (or kv_heads) vectors of dim
 * elements side by side; strides in elements, 16-byte aligned like the bases,
 * at least the row's width (so q, k and v may be parts of one array's rows).
 * Arrays of query rows may be NULL where every q_len is 0, arrays of key rows
 * where every k_len is.  What a call writes must share no memory with what it
 * reads or else writes. */
typedef struct gatgpu_attention_io {
    const void *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;
    const float* bias;    /* LINEAR: slope[heads]; TABLE: table[heads][buckets]  */
    const uint8_t* dist;  /* TABLE: pair distances, 16-byte aligned              */
    void* out;
    uint64_t out_stride;
    float* lse;           /* [row][heads], row as in out; forward: may be NULL   */
    void* rest;           /* bf16, may be NULL: an array of out's size and stride,
                             which a forward call leaves for its backward call
                             (rows for which it needs nothing may stay as they
                             were).  It holds the next 16 bits of out, encoded.
                             With it the weights enter out as two bf16 each, so
                             that dout.out has 16 bits, and as three with a
                             table: FP32's.  Without it an error of out's
                             rounding, 2^-8 of dout.out, stays in the score
                             gradients.  Required when dbias is given         */
    const void* dout;
    uint64_t dout_stride;
    void *dq, *dk, *dv;
    uint64_t dq_stride, dk_stride, dv_stride;
    float* dbias;         /* TABLE: [heads][buckets], may be NULL                */
} gatgpu_attention_io;

/* Reads q, k, v, bias, dist; writes out, and lse and rest where given. */
int gatgpu_attention_forward(gatgpu_attention* plan, const gatgpu_attention_io* io, void* workspace, uint64_t bytes);
/* Gradients of a forward call: reads what it read, its out, lse and rest, and
 * dout; writes dq, dk and dv of every row of a segment, and dbias.  Sums run in
 * one fixed order: equal inputs give equal bits. */
int gatgpu_attention_backward(gatgpu_attention* plan, const gatgpu_attention_io* io, void* workspace, uint64_t bytes);

/* ---- layer norm -------------------------------------------------------- */
/* No counterpart in the reference (which has no norm between layers).
 *   h = x + residual, rounded to the storage type and written to sum (without
 *   a residual: h = x);  n = (h - mean) rstd over the row's columns, rstd =
 *   1 / sqrt(variance + eps);  y = n gamma + beta, through ELU if elu != 0
 * and the gradients of x (= residual), gamma and beta.  Device arrays; rows of
 * `width` elements at strides in elements, any alignment (16-byte aligned rows of
 * whole 16 bytes are somewhat faster); gamma, beta, mean, rstd and their gradients are
 * FP32.  Stream, capture, device and workspace: as gatgpu_attention_forward.
 * y may be x or residual, sum x or residual, dx dy or dsum (same stride). */
typedef struct gatgpu_norm_io {
    int precision;        /* of the rows: GATGPU_FP32 or GATGPU_BF16             */
    int elu;
    uint64_t rows;
    uint32_t width;
    float eps;            /* >= 0                                                */
    const void* x;
    uint64_t x_stride;
    const void* residual; /* NULL: none                                          */
    uint64_t residual_stride;
    void* sum;            /* with a residual: h, may be NULL in a forward call
                             that no backward follows                            */
    uint64_t sum_stride;
    const float *gamma, *beta; /* NULL: 1 and 0                                  */
    void* y;
    uint64_t y_stride;
    float *mean, *rstd;   /* [rows]; forward: may be NULL                        */
    const void* dy;
    uint64_t dy_stride;
    const void* dsum;     /* gradient that reaches h beside y's, NULL: none      */
    uint64_t dsum_stride;
    void* dx;
    uint64_t dx_stride;
    float *dgamma, *dbeta; /* [width], may be NULL                               */
} gatgpu_norm_io;

int gatgpu_norm_forward(gatgpu_ctx* ctx, const gatgpu_norm_io* io);
/* Reads h (sum where a residual is given, else x), mean, rstd, gamma, beta, dy
 * and dsum; writes dx, dgamma and dbeta (sums in one fixed order). */
int gatgpu_norm_backward(gatgpu_ctx* ctx, const gatgpu_norm_io* io, void* workspace, uint64_t bytes);
/* Bytes of workspace of a backward call that gives dgamma or dbeta. */
int gatgpu_norm_workspace(gatgpu_ctx* ctx, uint64_t rows, uint32_t width, uint64_t* bytes);
/* Layer norm of the model's own layers: from now on the output of `layer` is
 * norm(aggregation), through ELU where the layer is hidden, in every forward of
 * the layer (gatgpu_layer_forward, gatgpu_model_forward,
 * gatgpu_layer_forward_static); its OUT stage is that, in FP32.  gamma, beta:
 * host FP32 [heads*dim], finite.  gamma and beta NULL: no norm any more.  The
 * fixed-p operator has none.  set_layer(layer) drops it. */
int gatgpu_set_norm(gatgpu_ctx* ctx, int layer, const float* gamma, const float* beta, float eps);

/* ---- norms and rotation of queries and keys ----------------------------- */
/* No counterpart in the reference.  In front of either attention, for each row and
 * head:
 *   n = x / sqrt(mean(x^2) + eps),  t = n gamma   (norm == 0: t = x)
 *   y = t with the pairs (a, b) of its first `rot` columns turned by the angle
 *       position freq[i]:  y_a = t_a cos - t_b sin,  y_b = t_b cos + t_a sin
 * and the gradients of x and gamma.  GATGPU_PAIRS_HALVES: pair i is the columns
 * (i, i + rot / 2); GATGPU_PAIRS_NEIGHBOURS: (2 i, 2 i + 1).  Angles are formed in
 * 64 bits, so positions may be far; their sines and cosines (times gamma in a forward
 * call), products and sums are FP32, y and the gradients are rounded once.  Squares
 * that would leave FP32 are formed of x times a power of two.  A NaN or infinity stays
 * in its own row and head, as does the NaN of a vector of zeros with eps 0.
 * Device arrays: rows of `heads` (kv_heads) vectors of dim elements side by side,
 * strides in elements, 16-byte aligned like the bases.  q_out may be q, k_out k, and
 * dq dq_out, dk dk_out (same strides); else what a call writes shares no memory with
 * what it reads or else writes.  Stream, capture, device and workspace: as
 * gatgpu_attention_forward. */
enum { GATGPU_PAIRS_HALVES = 0, GATGPU_PAIRS_NEIGHBOURS = 1 };
typedef struct gatgpu_rotate_io {
    int precision;        /* of the rows: GATGPU_FP32 or GATGPU_BF16             */
    int heads, kv_heads;  /* heads 1 to 1024, kv_heads 0 (no k) to 1024          */
    int dim;              /* a multiple of 8, at most 256                        */
    int norm;
    int rot;              /* even, 0 (no rotation) to dim                        */
    int pairs;
    float eps;            /* >= 0                                                */
    uint64_t rows;
    const void *q, *k;
    uint64_t q_stride, k_stride;
    const float *gamma_q, *gamma_k; /* [dim], NULL: 1; not read if norm == 0     */
    const uint32_t* position;       /* [rows]; not read if rot == 0              */
    const double* freq;             /* [rot / 2] radians a position, 8-byte aligned */
    void *q_out, *k_out;
    uint64_t q_out_stride, k_out_stride;
    const void *dq_out, *dk_out;    /* gradients of q_out and k_out              */
    uint64_t dq_out_stride, dk_out_stride;
    void *dq, *dk;                  /* gradients of q and k                      */
    uint64_t dq_stride, dk_stride;
    float *dgamma_q, *dgamma_k;     /* [dim], may be NULL; with norm only        */
} gatgpu_rotate_io;

/* Reads q, k, gamma, position and freq; writes q_out and k_out. */
int gatgpu_rotate_forward(gatgpu_ctx* ctx, const gatgpu_rotate_io* io);
/* Reads what the forward call read, dq_out and dk_out; writes dq, dk, dgamma_q and
 * dgamma_k (sums in one fixed order). */
int gatgpu_rotate_backward(gatgpu_ctx* ctx, const gatgpu_rotate_io* io, void* workspace, uint64_t bytes);
/* Bytes of workspace of a backward call that gives dgamma_q or dgamma_k. */
int gatgpu_rotate_workspace(gatgpu_ctx* ctx, const gatgpu_rotate_io* io, uint64_t* bytes);

/* ---- paged cache ---------------------------------------------------------- */
/* No counterpart in the reference.  A cache of keys and values in pages of `page`
 * tokens, for requests that grow token by token.  A request's tokens lie in the
 * blocks of its row of a block table: token t in page table[r][t / page] at offset
 * t % page, its slot being page index * page + offset.  A step over a packed batch
 * (request r has rows q_begin[r] to q_begin[r + 1]) is
 *   gatgpu_blocks_assign     pages, slots, positions and lengths from the lengths
 *   gatgpu_rotate_forward    queries and keys (position from the call before)
 *   gatgpu_cache_append      keys and values into their slots
 *   gatgpu_cache_attention   the rows' attention over their requests' pages
 * with every length in device memory, so that one captured graph serves steps of any
 * lengths (rows behind the last request's are left alone).  Stream, capture, device
 * and workspace: as gatgpu_attention_forward.  Whatever the arrays of lengths,
 * slots and pages hold, nothing outside the given arrays is read or written. */
#define GATGPU_NO_PAGE 0xffffffffu /* in a table: no page; as a slot: no token */

/* Block tables.  All arrays but the counts below are uint32 on the device.
 * Assign: request r has cached[r] tokens and gets fresh[r] more, for which it takes
 *   pages from the end of the free list, in the order of requests and blocks: the
 *   k-th page taken is free[free_count - 1 - k].  Request r is served if
 *   cached + fresh <= blocks * page, if the pages of requests 0 to r together are there
 *   (or r needs none; requests too long for the table count none), and if its rows end
 *   within `rows`.  Writes
 *     table     the taken pages, in the places of their blocks (nothing else)
 *     stored    tokens in the cache after the step: cached + fresh, of a request that is
 *               not served cached.  May be cached
 *     k_len     cached + fresh, of a request that is not served 0
 *     q_begin   [requests + 1] sums of fresh, beginning with 0 (2^32 - 1 where they pass that)
 *     slot      of each row; GATGPU_NO_PAGE behind the last request's rows, in those of a
 *               request that is not served, and where its table has no page
 *     position  of each row, 0 in the same places but the last
 *     free_left pages left in the list.  May be free_count
 *     unserved  requests that are not served
 * Release: the pages of the blocks that hold cached[r] tokens are put behind the
 *   list's free_count pages, in the order of requests and blocks (entries of `pages` or
 *   more are no pages); free_left: what the list holds then, at most `pages`.
 * A page belongs to one request, and to it once; equal inputs give equal lists. */
typedef struct gatgpu_blocks_io {
    uint32_t requests;     /* at most 2^20                                        */
    uint32_t page;         /* tokens: 16, 32, 64, 128 or 256                      */
    uint32_t pages;        /* of the cache, and of the free list; pages * page < 2^32 */
    uint32_t rows;         /* of slot and position; release: not read             */
    uint32_t blocks;       /* of a table row; blocks * page < 2^32                */
    uint64_t table_stride; /* entries from row to row, at least blocks            */
    const uint32_t *cached, *fresh; /* [requests]; release: cached                */
    uint32_t *table, *free;
    const uint32_t* free_count;     /* [1]                                        */
    uint32_t* free_left;            /* [1]                                        */
    uint32_t *stored, *k_len, *q_begin, *slot, *position, *unserved; /* release: not written */
} gatgpu_blocks_io;
int gatgpu_blocks_assign(gatgpu_ctx* ctx, const gatgpu_blocks_io* io, void* workspace, uint64_t bytes);
int gatgpu_blocks_release(gatgpu_ctx* ctx, const gatgpu_blocks_io* io, void* workspace, uint64_t bytes);
/* Bytes of workspace of either call. */
int gatgpu_blocks_workspace(gatgpu_ctx* ctx, const gatgpu_blocks_io* io, uint64_t* bytes);

/* The cache's device arrays, 16-byte aligned, for the caller to allocate.  Elements
 * are e4m3 bytes (8-bit floats of 3 mantissa bits, at most 448) times the scale of
 * their page and head, a power of two from 2^-64 to 2^64. */
typedef struct gatgpu_cache {
    uint32_t pages;  /* at least 1; pages * page < 2^32                           */
    uint32_t page;   /* tokens: 16, 32, 64, 128 or 256                            */
    int kv_heads;    /* 1 to 64                                                   */
    int dim;         /* a multiple of 16, at most 128                             */
    uint8_t* k;      /* [pages][kv_heads][page][dim]                              */
    uint8_t* v;      /* [pages][kv_heads][dim][page]                              */
    float *k_scale, *v_scale; /* [pages][kv_heads]                                */
} gatgpu_cache;

/* Keys and values of new tokens into their slots.  The tokens of a page are
 * neighbouring rows of one call, in the order of their slots, without gaps.  Those
 * before the first of them in the page keep their values, those behind the last are
 * no tokens any more.  The page's scale becomes the smallest power of two that holds
 * the largest magnitude m of its new tokens (m <= 448 scale), but no less than it was
 * if tokens stay; where it grows, their bytes are rounded again.  Values round to the
 * nearest e4m3 value, ties to even, beyond 448 * 2^64 to that; NaN and infinities become NaN
 * and leave the scale alone.  A slot of pages * page or more is no token: its row is
 * not read. */
typedef struct gatgpu_append_io {
    int precision;        /* of the rows: GATGPU_FP32 or GATGPU_BF16             */
    uint64_t rows;        /* < 2^27                                              */
    const void *k, *v;    /* rows of kv_heads vectors, 16-byte aligned           */
    uint64_t k_stride, v_stride;
    const uint32_t* slot; /* [rows]                                              */
} gatgpu_append_io;
int gatgpu_cache_append(gatgpu_ctx* ctx, const gatgpu_cache* cache, const gatgpu_append_io* io);

/* Attention of the rows over their requests' pages.  Row i of request r, of q_len =
 * q_begin[r + 1] - q_begin[r] rows, stands at position k_len[r] - q_len + i and sees
 * the tokens up to it that have a page (a table entry of `pages` or more hides its
 * block's); heads / kv_heads query heads share a key/value head:
 *   s = scale q.k,  out = sum p v,  p = softmax of s,  lse = log sum exp s
 * A row that sees no token of finite score gets out = 0 and lse = -infinity.  What is
 * not seen adds nothing, whatever its bytes hold; a NaN in a seen value reaches that
 * row's output.  Rows of no request are neither read nor written; of a request's rows
 * those beyond the first `most` are not computed.  k_len beyond blocks * page counts
 * as that, q_begin beyond rows as rows.
 * GATGPU_BF16: q and out bf16; GATGPU_FP32: both FP32.  Scores, softmax state and sums
 * are FP32; so is the weights' sum, and lse.  Where weights meet the values they are
 * fp16: one is off by at most 2^-11 of it (FP32 calls, in two parts: 2^-22), or its
 * product with its page's scale by 2^-31 of the largest such product of the row,
 * whichever is more.  Sums run in one fixed order: equal inputs give equal bits. */
typedef struct gatgpu_cache_attention_io {
    int precision;
    int heads;             /* a multiple of kv_heads, at most 64                 */
    float scale;           /* > 0                                                */
    uint64_t rows;         /* of q, out and lse: < 2^31 / heads                  */
    uint32_t requests;     /* at most 2^20                                       */
    uint32_t most;         /* rows of a request                                  */
    uint32_t blocks;       /* of a table row; blocks * page < 2^32               */
    uint64_t table_stride; /* entries from row to row, at least blocks           */
    const void* q;
    uint64_t q_stride;
    const uint32_t* q_begin; /* [requests + 1], not decreasing                   */
    const uint32_t* k_len;   /* [requests]                                       */
    const uint32_t* table;
    void* out;
    uint64_t out_stride;
    float* lse;            /* [row][heads], may be NULL                          */
} gatgpu_cache_attention_io;
int gatgpu_cache_attention(gatgpu_ctx* ctx, const gatgpu_cache* cache, const gatgpu_cache_attention_io* io,
                           void* workspace, uint64_t bytes);
/* Bytes of workspace for a call of these sizes (arrays need not be set). */
int gatgpu_cache_attention_workspace(gatgpu_ctx* ctx, const gatgpu_cache* cache, const gatgpu_cache_attention_io* io,
                                     uint64_t* bytes);

/* ---- misc ------------------------------------------------------------ */
int gatgpu_set_option(gatgpu_ctx* ctx, int key, int64_t value);
/* Blocks until all work on the context's stream is done. */
int gatgpu_synchronize(gatgpu_ctx* ctx);
/* The context's HIP stream (hipStream_t) for callers that order their own
 * work against it. */
void* gatgpu_stream(gatgpu_ctx* ctx);

#ifdef __cplusplus
}
#endif
#endif /* GATGPU_H */
