/*
 * deepep_amd — C ABI of the MI355X (gfx950) dispatch / combine / W4A8-MoE hot path.
 *
 * Conventions
 *   - every function returns 0 on success, a negative DPEP_E* code otherwise, and never throws;
 *     dpep_last_error() returns a thread-local message for the last failure on this thread;
 *   - every pointer is a DEVICE pointer unless its name ends in _host;
 *   - `stream` is a hipStream_t passed as void* (NULL = the null stream); every call only
 *     enqueues work on that stream and returns without synchronising;
 *   - output buffers are allocated by the caller; the library owns only the workspace;
 *   - one call at a time per workspace (the host layer keeps the reference's per-buffer lock).
 *
 * Each entry point cites the reference interface it replaces (paths relative to the reference
 * checkout).
 */
#ifndef DEEPEP_AMD_H
#define DEEPEP_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DPEP_OK 0
#define DPEP_EINVAL (-1)  /* bad argument (maps to ValueError, like std::invalid_argument in csrc/ops) */
#define DPEP_ERUNTIME (-2) /* HIP failure (maps to RuntimeError, like std::runtime_error in csrc/ops) */

#define DPEP_MAX_TOPK 32
#define DPEP_MAX_LOCAL_EXPERTS 1024

const char* dpep_last_error(void);
int dpep_version(void);

/* Workspace: one hipMalloc'd HBM block standing in for the reference's symmetric SHMEM workspace
 * (csrc/runtime/session.cpp:40-140, Runtime(...) in csrc/bindings/module.cpp:54-71).  Holds the
 * layout scratch (per-chunk histograms) and the MegaMoE intermediates of one EP rank's share. */
int dpep_workspace_create(size_t bytes, void** ws);
int dpep_workspace_destroy(void* ws);
int dpep_workspace_capacity(void* ws, size_t* bytes);
/* Switches of a workspace for tests and diagnosis; no counterpart in the reference.  Keys:
 *   "layout_one_launch"             0: dpep_layout always takes two launches (count, assign); 1 (default): one
 *                                   launch whose workgroups exchange their histograms, where the input is small enough
 *   "layout_exchange_ticks"         bound of a workgroup's wait for the others' histograms in 10 ns ticks (default 2 s)
 *   "layout_exchange_extra_rows"    1: the workgroups wait for one histogram more than there are workgroups, so that
 *                                   the wait runs out (exercises the error path)
 *   "layout_payload_looks"          how often a payload in the layout's grid looks for a word of the layout's, one or two
 *                                   microseconds apart, before it works its rows out from the ids itself (0 to 64, the default)
 *   "gemm_zero_fill"                1 (default): workgroups of dpep_megamoe_forward's first GEMM that get no tile zero
 *                                   the output rows of tokens no local expert serves; 0: the weighted reduce writes them
 *   "megamoe_served_only"           1: dpep_megamoe_forward leaves the rows of y whose token no local expert serves
 *                                   untouched (one rank's share of an EP job, where other ranks produce those rows);
 *                                   0 (default): they are zeroed
 *   "gemm_tile_rows"                0 (default): dpep_megamoe_forward chooses the row-tile height of its grouped GEMMs
 *                                   from the expected rows per expert; 64, 128 or 192: that height for both, 32: the
 *                                   kernel for few rows per expert for both
 *   "gemm_few_rows_waves"           its waves per workgroup when forced: 4 (default) or 1
 *   "gemm_paired"                   with 128 forced: 0 (default) the kernel that the other heights take too, 1 the one with
 *                                   two workgroups to a CU, 2 that one with its weights past the caches
 *   "gemm_column_waves"             1 (default): the GEMM whose waves split a tile's columns, where it takes the sizes;
 *                                   0: always the 2 x 2 form */
int dpep_workspace_tune(void* ws, const char* key, long long value);
/* Scratch bytes dpep_layout needs for T*K routes and L local experts
 * (notify_layout() workspace_bytes, csrc/ops/notify.cpp:98-110). */
size_t dpep_layout_workspace_bytes(int num_tokens, int num_topk, int num_local_experts);

/* Routing layout: validity, per-expert counts, prefix sums and the stable permutation.
 * Replaces notify() (csrc/ops/notify.cpp:112-190 -> notify_full_kernel, csrc/kernels/notify/notify.cpp:2026)
 * and the count/prefix half of expand() (csrc/direct/ops/expand.cpp:52-219).
 *   topk_idx      int64 [T,K]; a route is valid for this rank iff 0 <= e < num_experts and
 *                 expert_begin <= e < expert_begin + num_local
 *   counts        int32 [L]    rows per local expert (expert_totals slice / actual_expert_counts)
 *   psum          int32 [L]    inclusive prefix (psum_num_recv_tokens_per_expert)
 *   offsets       int32 [L+1]  exclusive prefix with leading 0 (expert_offsets)
 *   route_to_row  int32 [T*K]  row of route (t,s), -1 if it produces no row (recv_to_expanded_idx)
 *   row_to_route  int32 [T*K]  first R entries valid: flat route id t*K+s of each row (weight_return_meta)
 *   num_rows      int32 [1]    R */
int dpep_layout(void* ws, const int64_t* topk_idx, int num_tokens, int num_topk, int num_experts,
                int expert_begin, int num_local, int32_t* counts, int32_t* psum, int32_t* offsets,
                int32_t* route_to_row, int32_t* row_to_route, int32_t* num_rows, void* stream);

/* dpep_layout for callers that cannot allocate: code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc.  It has no counterpart in the reference (whose notify always works in its pre-allocated symmetric
 * workspace).  Same inputs, outputs and results as dpep_layout, but no workspace: the histograms live in a device
 * array inside the library (84 KiB per GPU, held until the process ends), and the call allocates nothing - no
 * hipMalloc, hipFree or pinned memory, on the first call or any later one.  Always the two-launch form (count, then
 * assign); it reports nothing to the host, so R is read from num_rows on the device.  Limits: those of dpep_layout
 * (at most DPEP_MAX_LOCAL_EXPERTS local experts, T*K < 2^31), checked before anything is launched.  All calls on one
 * GPU share that GPU's array: calls whose kernels overlap on one GPU (different streams) race; calls on one stream
 * do not.  Nothing in the array has to be zero or is kept between calls. */
int dpep_layout_static(const int64_t* topk_idx, int num_tokens, int num_topk, int num_experts, int expert_begin,
                       int num_local, int32_t* counts, int32_t* psum, int32_t* offsets, int32_t* route_to_row,
                       int32_t* row_to_route, int32_t* num_rows, void* stream);

/* Host side of the layout's single synchronisation: blocks until the most recent dpep_layout launched on ws has
 * run, then returns R and (optionally) the rows per local expert.  Replaces the device-to-host read-back that sizes
 * the outputs of a fresh dispatch (deep_ep/backends/mesh_clos/elastic.py:1476, `.cpu()` of the notify outputs):
 * the layout kernel writes these few words straight into pinned host memory owned by the workspace and this
 * call polls them, which costs a few microseconds less than a copy plus a stream wait.
 *   counts_host   int32 [num_local] host memory, may be NULL; num_local must equal the launched layout's
 *   num_rows_host int32 [1] host memory
 *   timeout_us    DPEP_ERUNTIME if the kernel has not reported by then (a layout launch that failed never will)
 * One layout may be outstanding per workspace; the call does not wait for anything but the layout kernel. */
int dpep_layout_wait(void* ws, int32_t* counts_host, int num_local, int32_t* num_rows_host, long long timeout_us);
/* 1 if the most recent layout launched on ws has reported (dpep_layout_wait would not have to wait), else 0. */
int dpep_layout_ready(void* ws);
/* Stores value in *word (8-byte aligned, GPU-accessible memory such as hipMallocSignalMemory's) behind everything the stream was
 * given before: what other streams' hipStreamWaitValue64 wait for. */
int dpep_stream_raise(void* word, uint64_t value, void* stream);

/* Expand-permute payload dispatch: out[row(t,s)] = x[t] for every route with a row.
 * Replaces dispatch() (csrc/ops/dispatch.cpp:82-211 -> dispatch_kernel, csrc/kernels/dispatch/dispatch.cpp:628)
 * and the scatter half of expand() (csrc/direct/kernels/expand/expand.cpp:334-520).
 *   row_bytes     bytes per payload row (BF16: 2H, FP8: H); must be a multiple of 16
 *   scales        optional fp32 [T, scale_cols] side rows moved with the payload (FP8 per-128 scales)
 *   topk_weights  optional fp32 [T,K]; out_weights[row] = topk_weights[t,s]
 *   num_rows      R (host value from dpep_layout_wait), or -1 when the host does not know R yet: the launch then
 *                 does not depend on R, out / out_scales / out_weights must hold T*K rows and the first R are
 *                 written.  A caller that allocates at capacity can thus queue layout and dispatch back to back
 *                 and read R (to narrow its outputs) while they run. */
int dpep_dispatch_copy(const void* x, const float* scales, const float* topk_weights,
                       const int32_t* route_to_row, const int32_t* row_to_route, int num_tokens,
                       int num_topk, int num_rows, int row_bytes, int scale_cols, void* out,
                       float* out_scales, float* out_weights, void* stream);

/* How dpep_dispatch_copy, dpep_dispatch_quant_fp8 and dpep_cast_to_fp8 store their payload rows; process-wide, no
 * counterpart in the reference (its rows leave through the transport).  Returns the policy in force before the call
 * (DPEP_STORE_QUERY changes nothing), or DPEP_EINVAL.
 *   DPEP_STORE_STREAMING  (default) non-temporal stores: the rows go to HBM past the caches, the kernel's time is the
 *                         time of its traffic and nothing is left for the next kernel to write back
 *   DPEP_STORE_THROUGH    write-through stores: the memory-side cache takes the rows first, so the kernel itself ends
 *                         sooner when that cache is clean and the kernel that follows pays for the write-back, unless it
 *                         is the reader of those rows and finds them there
 *   DPEP_STORE_CACHED     plain stores */
#define DPEP_STORE_THROUGH 0
#define DPEP_STORE_STREAMING 1
#define DPEP_STORE_CACHED 2
#define DPEP_STORE_QUERY 3
int dpep_dispatch_store_policy(int policy);

/* Fused per-128-element FP8 e4m3fn quantisation + expand-permute: the reference's caller-side
 * per_token_cast_to_fp8 (deep_ep/utils/math.py:45-61) followed by the FP8 dispatch above, in one pass.
 *   x             bf16 [T,H], H % 128 == 0
 *   out           fp8  [R,H]; out_scales fp32 [R, H/128]
 *   num_rows      R or -1, as for dpep_dispatch_copy */
int dpep_dispatch_quant_fp8(const void* x, const float* topk_weights, const int32_t* route_to_row,
                            const int32_t* row_to_route, int num_tokens, int num_topk, int num_rows,
                            int hidden, void* out, float* out_scales, float* out_weights, void* stream);

/* Routing layout and payload dispatch of a small batch (at most 2048 routes: a decode step) in ONE launch.
 * Replaces the low-latency dispatch (csrc/ops/low_latency.cpp:80-216 -> dispatch_low_latency, csrc/kernels/dispatch/
 * low_latency.cpp:73), which likewise derives the rows inside the payload kernel instead of running notify first; for
 * larger batches dpep_layout followed by dpep_dispatch_copy / dpep_dispatch_quant_fp8 produce the same results.
 * Every workgroup works out the rows of its own token from the whole routing table (which fits its LDS), so nothing
 * waits for a layout kernel.  Arguments as for dpep_layout plus dpep_dispatch_copy (quantize == 0: x of row_bytes
 * bytes per token, optional scales and weights) or dpep_dispatch_quant_fp8 (quantize != 0: x BF16, row_bytes = 2H,
 * H % 128 == 0, out FP8 + out_scales FP32 [.,H/128]).  out / out_scales / out_weights must hold T*K rows; the first R are
 * written.  The per-expert counts and R also go to the workspace's host mailbox: dpep_layout_wait works as after
 * dpep_layout. */
int dpep_layout_dispatch_small(void* ws, const int64_t* topk_idx, const void* x, const float* scales,
                               const float* topk_weights, int num_tokens, int num_topk, int num_experts, int expert_begin,
                               int num_local, int row_bytes, int scale_cols, int quantize, int32_t* counts, int32_t* psum,
                               int32_t* offsets, int32_t* route_to_row, int32_t* row_to_route, int32_t* num_rows, void* out,
                               float* out_scales, float* out_weights, void* stream);

/* One fresh dispatch as ElasticBuffer makes it (notify + dispatch, deep_ep/backends/mesh_clos/elastic.py:648-1008): the layout
 * and, queued behind it or in the same grid before the host knows R, the payload; for a small batch both in one launch (see above).  The
 * payload outputs hold capacity_rows rows, of which the first min(R, capacity_rows) are written: a caller that finds
 * R > capacity_rows allocates R rows and calls dpep_dispatch_copy / dpep_dispatch_quant_fp8 with the same maps.  One that does
 * so whenever DPEP_ROWS_KEPT says that the outputs are too small, or mostly unused, sets report_to_host to
 * DPEP_REPORT_ALL_OR_NONE: the outputs are then left as they are in these cases (a small batch may write part of them), and the
 * launch ends at once.  capacity_rows is then taken for DPEP_CAPACITY of the rows that the caller expects (with other values
 * the even share of the routes is what is expected); the expectation decides how the work is split, never what is computed. */
#define DPEP_REPORT_ALL_OR_NONE 2
#define DPEP_CAPACITY(rows) ((rows) + (rows) / 8 + 256)
#define DPEP_ROWS_KEPT(rows, capacity) ((rows) <= (capacity) && (capacity) - (rows) <= (rows) / 2 + 1024)
typedef struct dpep_fresh_dispatch {
    const int64_t* topk_idx;    /* [T,K] */
    int64_t* topk_idx_copy;     /* [T,K] receives a copy of topk_idx (the handle's own), or NULL */
    const void* x;              /* [T] rows of row_bytes bytes */
    const float* scales;        /* [T,scale_cols] 4-byte words moved with the rows, or NULL */
    const float* topk_weights;  /* [T,K] or NULL */
    int32_t* counts;            /* layout outputs as for dpep_layout */
    int32_t* psum;
    int32_t* offsets;
    int32_t* route_to_row;
    int32_t* row_to_route;
    int32_t* num_rows;
    int32_t* send_counts;       /* [E]: rows of experts 0..e that are local to this rank, or NULL */
    void* out;                  /* payload outputs, capacity_rows rows each; out_scales and out_weights NULL where unused */
    float* out_scales;
    float* out_weights;
    int32_t num_tokens, num_topk, num_experts, expert_begin, num_local;
    int32_t row_bytes, scale_cols;
    int32_t quantize;           /* != 0: x is BF16 and is quantised per 128 columns (scales NULL, out FP8, out_scales [.,H/128]) */
    int32_t capacity_rows;
    int32_t report_to_host;     /* != 0: counts and R also go to the host mailbox (dpep_layout_wait); see above for 2 */
} dpep_fresh_dispatch;
int dpep_dispatch_fresh(void* ws, const dpep_fresh_dispatch* call, void* stream);

/* Stand-alone per-128 quantiser (deep_ep/utils/math.py:45-61): x bf16 [T,H] -> fp8 [T,H], fp32 [T,ceil(H/128)].
 * H % 16 == 0; a last block shorter than 128 is quantised as if padded with zeros (math.py:52-53). */
int dpep_cast_to_fp8(const void* x, int num_tokens, int hidden, void* out, float* out_scales, void* stream);

/* The dequantiser the reference checks its FP8 path with: out = bf16(fp32(code) * scale), one scale per block of 128
 * columns (per_token_cast_back, deep_ep/utils/math.py:64-79).  scales: fp32 [T, ceil(H/128)], or, scales_are_e8m0_bytes
 * != 0, one exponent byte per block (the reference's int32 scale tensors hold four of them each, math.py:74-76).
 * H % 16 == 0; the last block of a row may be short.  codes e4m3fn [T,H] -> out bf16 [T,H]. */
int dpep_cast_back(const void* codes, const void* scales, int scales_are_e8m0_bytes, int num_tokens, int hidden, void* out,
                   void* stream);

/* Combine: out[t] = bf16_rne( sum over slots in order, skipping -1, of fp32(y[row]) (* w[row]) ).
 * Replaces combine() (csrc/ops/combine.cpp:198-326 -> combine_kernel, csrc/kernels/combine/combine.cpp:2965)
 * with row_weights == NULL, and aggregate() / the low-latency combine
 * (csrc/direct/ops/aggregate.cpp:44-143, csrc/direct/kernels/aggregate/aggregate_impl.h:166-226,
 * csrc/kernels/combine/low_latency.cpp:41) with row_weights != NULL.
 *   y             bf16 [R,H], H % 8 == 0
 *   row_weights   optional fp32 [R]: multiply each row before the add (separate mul and add)
 *   return_in     optional fp32 [R]: weight-return channel; return_out[t,s] = return_in[row], 0 without a row
 *   out           bf16 [T,H];  return_out fp32 [T,K] */
int dpep_combine(const void* y, const float* row_weights, const int32_t* route_to_row, int num_tokens,
                 int num_topk, int num_rows, int hidden, void* out, const float* return_in,
                 float* return_out, void* stream);

/* dpep_combine (half != 0: dpep_combine_fp16) of a y that holds num_rows rows of which about expected_rows are in use, as
 * in the low-latency path's capacity layout: the expectation decides how the work is split, never what is computed. */
int dpep_combine_expecting(const void* y, int half, const float* row_weights, const int32_t* route_to_row, int num_tokens, int num_topk,
                           int num_rows, int expected_rows, int hidden, void* out, const float* return_in, float* return_out,
                           void* stream);

/* dpep_combine that writes only the tokens that own at least one row and leaves the others' rows of `out` untouched.
 * For one rank's receive share of an EP job most candidate tokens own no row here, and in the reference nothing is
 * produced for them on this rank at all (a rank returns rows only for the routes it served,
 * csrc/kernels/combine/combine.cpp:2965); dpep_combine zero-fills them, which is what a single-rank caller needs. */
int dpep_combine_served(const void* y, const float* row_weights, const int32_t* route_to_row, int num_tokens,
                        int num_topk, int num_rows, int hidden, void* out, const float* return_in,
                        float* return_out, void* stream);

/* The same combine for IEEE half rows and output (the low-latency path accepts BF16 or FP16 expert outputs and
 * returns the same dtype: deep_ep/backends/mesh_clos/elastic.py:596-606; oracle expected_combine,
 * tests/elastic/test_ep_low_latency.py:449-463): fp32 accumulation in slot order, one RNE rounding to half. */
int dpep_combine_fp16(const void* y, const float* row_weights, const int32_t* route_to_row, int num_tokens,
                      int num_topk, int num_rows, int hidden, void* out, const float* return_in,
                      float* return_out, void* stream);

/* MXFP8 activation quantiser, block 32 (quantize_input, experiments/megamoe/python/
 * deep_ep_experimental/megamoe/reference.py:44-54; device ComputeMxScale/QuantizeMxFp8Data).
 *   x bf16 [B,H], H % 32 == 0 -> codes e4m3 [B,H], scales e8m0 [B,H/32] */
int dpep_mx_quant(const void* x, int rows, int hidden, void* codes, uint8_t* scales, void* stream);

/* Host-only check of the grouped GEMM's copy/wait schedule; no counterpart in the reference (it is how this build
 * shows, without a GPU, that for a workgroup that walks `tiles_per_workgroup` tiles of `tile_rows` (64, 128 or 192)
 * rows and `ktiles` k tiles of 128 every asynchronous copy is covered by a counted wait before it is read, under
 * in-order completion of vector-memory operations: an item's operands before its MFMAs, the next tile's gather
 * indices before the copy cursor switches tiles), and that a ring slot of scale bytes is refilled only when the span of k
 * tiles it held has been read to the end.  epilogue_stores = stores a tile end issues (they only make the
 * counted waits stricter).  without_drain: bit 0 replays the schedule WITHOUT the cursor's wait at tile switches (what a
 * kernel that trusted every index fetch would do): the check then has to fail for tiles shorter than the copies run ahead;
 * bit 1 replays rings of two scale slots instead of the kernel's three: the check then has to fail where k is no multiple
 * of 512 and a workgroup has several tiles; that they do fail is how the tests know that the check can.
 * Returns 0, or DPEP_EINVAL with the first violation in dpep_last_error(). */
int dpep_megamoe_schedule_check(int tile_rows, int tiles_per_workgroup, int ktiles, int epilogue_stores, int without_drain);
/* The same check for the kernel that runs where K is a multiple of 512 (its waves split the tile's columns and load their
 * weights straight into registers; k tiles come in fours).  slack = operations the replayed wait allows in flight beyond
 * the kernel's own count: with slack > 0 the check has to fail, which is how the tests know that it can. */
int dpep_megamoe_schedule_check_column_waves(int tile_rows, int tiles_per_workgroup, int ktiles, int epilogue_stores, int slack);
/* The same check for the kernel with two workgroups to a CU (128 rows; k tiles in fours, those of padding included), whose
 * weights have a cursor of their own: also that it asks for the right item's.  first_slack, second_slack: as slack, for the
 * waits in front of an item's first and second k step. */
int dpep_megamoe_schedule_check_paired(int tiles_per_workgroup, int ktiles, int epilogue_stores, int first_slack, int second_slack);

/* Which grouped GEMM kernel a forward of these sizes takes on this workspace (NULL: one with default settings), for the
 * first or (second != 0) the second GEMM: its row-tile height (64, 128, 192, or 32 for the kernel for few rows per expert)
 * and its waves per workgroup.  Host arithmetic only; no counterpart in the reference. */
int dpep_megamoe_gemm_choice(void* ws, int num_tokens, int hidden, int intermediate, int num_topk, int num_experts, int num_local,
                             int num_shared, int second, int32_t* tile_rows, int32_t* waves);
#define DPEP_GEMM_TWO_BY_TWO 0       /* 64, 128 or 192 rows: 2 x 2 waves, weights through LDS */
#define DPEP_GEMM_COLUMN_WAVES 1     /* the same heights: the waves split the columns, weights straight to registers */
#define DPEP_GEMM_PAIRED 2           /* 128 rows, two workgroups to a CU */
#define DPEP_GEMM_PAIRED_STREAMED 3  /* the same, weights past the caches */
#define DPEP_GEMM_FEW_ROWS 4         /* 32 rows, activations through LDS; four waves to a workgroup, or one */
#define DPEP_GEMM_ONE_WAVE 5         /* 32 rows, one wave to a workgroup, no LDS */
/* The same question, answered with the kernel's name. */
int dpep_megamoe_gemm_kernel(void* ws, int num_tokens, int hidden, int intermediate, int num_topk, int num_experts, int num_local,
                             int num_shared, int second, int32_t* kernel);

/* Bytes of workspace dpep_megamoe_forward needs (buffer_size(), experiments/megamoe/csrc/forward.cpp:480).
 * num_shared = number of shared experts (0..8) whose rows (every token, each) are held next to the routed ones. */
size_t dpep_megamoe_workspace_bytes(int num_tokens, int num_topk, int hidden, int intermediate, int num_local,
                                    int num_shared);

/* What the grouped GEMM works on for a logical hidden or intermediate size: whole 256-column tiles and whole spans of
 * scales, at least 512 (dim <= 512 -> 512, else the next multiple of 256).  Prepared weights are padded to it when
 * they are prepared (zero codes, scale 1.0), input rows by a copy inside the forward; 0 for dim < 1.
 * (The reference accepts hidden % 64 == 0 and intermediate_hidden % 128 == 0, api.py:93-105.) */
int dpep_megamoe_padded_dim(int dim);

/* Shape of the prepared form of one raw weight tensor [L,N,K/2] + [L,N,K/32]: packed [L,padded_n,padded_k/2] and scales
 * [L,padded_n,scale_cols] (the scales are stored in spans of four k tiles = k 512, the last span padded).
 * N % 64 == 0 (gate_up: N = 2I with I % 128 == 0, both halves padded separately), K % 64 == 0.
 * (Part of the transform_weights_for_mega_moe contract below.) */
int dpep_megamoe_prepared_shape(int n, int k, int gate_up, int* padded_n, int* padded_k, int* scale_cols);

/* One-off weight re-layout (transform_weights_for_mega_moe, experiments/megamoe/python/.../api.py:311-379):
 * raw packed FP4 [L,N,K/2] + e8m0 [L,N,K/32]  ->  the tile order the GEMM kernel streams, padded as
 * dpep_megamoe_prepared_shape says (out_packed and out_scales have those sizes).  Byte shuffle only.
 * gate_up != 0 (first GEMM, N = 2I, gate rows then up rows) interleaves gate and up in groups of 32 output columns so
 * SwiGLU is lane-local (the counterpart of _interleave_gate_up_128, api.py:285-293). */
int dpep_megamoe_prepare_weights(const uint8_t* w_packed, const uint8_t* w_scales, int num_local, int n,
                                 int k, int gate_up, uint8_t* out_packed, uint8_t* out_scales, void* stream);

/* Diagnosis, no counterpart in the reference: what the idle workgroups of the most recent dpep_megamoe_forward's first
 * GEMM did (see "gemm_zero_fill").  Waits for `stream`, then reports the number of filler waves of that launch (0: the
 * launch had a tile for every workgroup, or zero fill is off) and the tokens they looked at before they were told to
 * stop.  The sizes are those of the forward call. */
int dpep_megamoe_fill_report(void* ws, int num_tokens, int num_topk, int hidden, int intermediate, int num_local,
                             int num_shared, int32_t* fillers_host, int64_t* tokens_filled_host, void* stream);

/* Fused W4A8 MoE forward for one rank's local experts (Plan::forward, experiments/megamoe/csrc/forward.cpp:340-478
 * -> mega_moe_kernel_do, kernel_launch.hpp:8-13):
 * layout -> gather rows -> GMM1 (MXFP8 x MXFP4) -> bf16 -> SwiGLU -> MXFP8 requant -> GMM2 -> bf16 ->
 * route-weighted fp32 reduce per token -> bf16.
 *   x_codes e4m3 [B,H], x_scales e8m0 [B,H/32], topk_idx int32 [B,K] (distinct, in [0,E)), topk_weights fp32 [B,K]
 *   H % 64 == 0, I % 128 == 0 (hidden / intermediate as the caller sees them)
 *   w1/s1: prepared GMM1 weights of the raw [L,2I,H/2] and scales; w2/s2: prepared GMM2 weights of the raw [L,H,I/2]
 *   and scales (sizes: dpep_megamoe_prepared_shape)
 *   shared_w1/s1/w2/s2: the same for num_shared shared experts ([S,2I,H/2] ...; sw1/sw2/ss1/ss2 of
 *   mega_moe_kernel_do), NULL when num_shared == 0.  A shared expert processes every token and its output is
 *   added with weight 1 after the routed experts' (golden.py:160-164).
 *   y bf16 [B,H]; expert_token_nums int32 [L] (routed experts only) */
int dpep_megamoe_forward(void* ws, const void* x_codes, const uint8_t* x_scales, const int32_t* topk_idx,
                         const float* topk_weights, const uint8_t* w1, const uint8_t* s1, const uint8_t* w2,
                         const uint8_t* s2, const uint8_t* shared_w1, const uint8_t* shared_s1,
                         const uint8_t* shared_w2, const uint8_t* shared_s2, int num_shared, int num_tokens, int hidden,
                         int intermediate, int num_topk, int num_experts, int expert_begin, int num_local, void* y,
                         int32_t* expert_token_nums, void* stream);

/* The same forward with its arguments in a struct, and with the choice of BF16 input rows, which the forward then quantises
 * itself (dpep_mx_quant's arithmetic, in the launch that also works out the layout): x_bf16 [B,H] instead of x_codes / x_scales,
 * and scratch for the codes [B, dpep_megamoe_padded_dim(H)] and their scale bytes [B, dpep_megamoe_padded_dim(H) / 32]. */
typedef struct dpep_megamoe_call {
    const void* x_codes;
    const uint8_t* x_scales;
    const void* x_bf16;
    uint8_t* x_codes_scratch;
    uint8_t* x_scales_scratch;
    const int32_t* topk_idx;
    const float* topk_weights;
    const uint8_t *w1, *s1, *w2, *s2;
    const uint8_t *shared_w1, *shared_s1, *shared_w2, *shared_s2;
    void* y;
    int32_t* expert_token_nums;
    int32_t num_shared, num_tokens, hidden, intermediate, num_topk, num_experts, expert_begin, num_local;
} dpep_megamoe_call;
int dpep_megamoe_run(void* ws, const dpep_megamoe_call* call, void* stream);

/* ---- Operators around dispatch and combine: router, balance loss, 4-bit products.  The reference takes routes and experts as given, so
 * these have no counterpart there. ---- */
#define DPEP_TYPE_F32 0
#define DPEP_TYPE_BF16 1
#define DPEP_TYPE_F16 2
#define DPEP_SCORE_SOFTMAX 0
#define DPEP_SCORE_SIGMOID 1
#define DPEP_MAX_ROUTER_TOKENS (1 << 30)
#define DPEP_MAX_SEQUENCES ((1 << 22) - 1)
#define DPEP_W4_MAX_N (1 << 30)
#define DPEP_W4_MAX_K 16384
#define DPEP_W4_MAX_ROWS 65535
#define DPEP_W4_MAX_ROUTES 2048

/* A layer's router.  Scores: softmax over the row, or each logit's sigmoid.  Experts are chosen by key: the logit (softmax), or the
 * sigmoid plus the expert's bias, rounded to fp32; an expert whose logit is -inf is never chosen, a NaN ranks with +inf.  With
 * num_groups > 1 the num_experts / num_groups experts of a group stand together: the num_topk_groups groups of the largest key
 * (softmax), or of the largest sum of two keys (sigmoid), stay in the choice.  Ties go to the lowest index.
 *   num_experts  1..1024;  num_topk  1..DPEP_MAX_TOPK, at most the experts of num_topk_groups groups;  num_groups  1..64, a divisor of num_experts
 *   normalize    != 0: the chosen experts' scores are divided by their sum (sigmoid: plus 1e-20)
 *   scale        factor of the weights, 1e-30 to 1e30 in magnitude
 *   logits_type  DPEP_TYPE_*;  index_bytes  of an expert id: 8, or 4 */
typedef struct dpep_router {
    int32_t num_experts, num_topk, num_groups, num_topk_groups;
    int32_t score, normalize;
    float scale;
    int32_t logits_type, index_bytes;
} dpep_router;
/* Expert ids and weights of every token, best first; -1 and 0 where fewer than num_topk experts are left.
 *   logits [T,E];  bias optional fp32 [E] (sigmoid only);  token_mask optional bytes [T], 0: padding, which gets no route
 *   topk_idx int64 or int32 [T,K];  topk_weights fp32 [T,K] */
int dpep_route(const dpep_router* r, const void* logits, const float* bias, const uint8_t* token_mask, int num_tokens, void* topk_idx,
               float* topk_weights, void* stream);

/* Balance loss of every sequence, and its counts.  A token without a route (ids outside 0..E-1) is padding.  In a sequence of N other
 * tokens with R routes, c_e of them to expert e: loss = sum_e (E c_e / R) (sum_t p_te / N), p a token's softmax, or its sigmoids over
 * (their sum + 1e-20); 0 for a sequence without tokens.  Sums are taken in an order that depends on the sizes alone.  T*K < 2^31, here and in
 * the loss's gradient; B at most DPEP_MAX_SEQUENCES.
 *   sequence_offsets  int32 [B+1] ascending from 0 to T, or NULL: one sequence
 *   losses fp32 [B];  counts int32 [B,E];  tokens int32 [B] (N);  scratch  dpep_balance_scratch_bytes, 4-byte aligned */
size_t dpep_balance_scratch_bytes(int num_experts, int num_tokens, int num_sequences);
int dpep_balance_loss(const dpep_router* r, const void* logits, const void* topk_idx, int num_tokens, const int32_t* sequence_offsets, int num_sequences,
                      float* losses, int32_t* counts, int32_t* tokens, void* scratch, void* stream);
/* dpep_route and the dpep_balance_loss of its routes, in one pass over the logits. */
int dpep_route_balance(const dpep_router* r, const void* logits, const float* bias, const uint8_t* token_mask, int num_tokens, const int32_t* sequence_offsets,
                       int num_sequences, void* topk_idx, float* topk_weights, float* losses, int32_t* counts, int32_t* tokens, void* scratch, void* stream);

/* Gradient of the logits, in their type, from the gradient of the route weights (grad_weights, as dpep_combine's return channel gives
 * it; entries without a route are not read into it), of the balance losses (grad_losses, with what dpep_balance_loss was given and
 * returned), or of both.  The choice itself and the counts have no gradient.  Ids of a token are taken for distinct.
 *   topk_weights  dpep_route's, needed where they are normalised */
typedef struct dpep_router_gradients {
    const void* logits;
    const void* topk_idx;
    const float* topk_weights;
    const float* grad_weights;
    const int32_t* sequence_offsets;
    const int32_t* counts;
    const int32_t* tokens;
    const float* grad_losses;
    void* grad_logits;
    int32_t num_sequences;
} dpep_router_gradients;
int dpep_router_backward(const dpep_router* r, const dpep_router_gradients* g, int num_tokens, void* stream);

/* Matrices [L,N,K] in 4 bits: value (q - zero) * scale, q two to a byte along K (low nibble: even k), one scale and zero point for each
 * `group` values of a row.
 *   packed [L,N,K/2], 16-byte aligned;  scales [L,N,K/group] in the type of the rows multiplied;  zeros bytes [L,N,K/group] (0..15), or
 *   NULL: 8;  group 32, 64 or a multiple of 128, a divisor of K;  K at most 16384
 * x is multiplied by 16 + q and (16 + zero) times its group's sum taken off again, in fp32: a row of x that holds an infinity or a NaN, or
 * values whose sums pass the range of fp32, gets results that are not finite. */
typedef struct dpep_w4 {
    const uint8_t* packed;
    const void* scales;
    const uint8_t* zeros;
    int32_t n, k, group;
} dpep_w4;
/* y[m] = W x[m]: x, y of `type` (BF16 or FP16), x [M,K] 16-byte aligned, y [M,N], which overlaps neither x nor the weights, sums
 * in fp32, rounded once.  M at most 65535; meant for a few rows: beyond about 16 the time grows with M. */
int dpep_w4_matvec(const dpep_w4* w, int type, const void* x, int num_rows, void* y, void* stream);
/* An expert layer for few tokens (T*K <= 2048 routes): y[t] = sum over the slots s of topk_weights[t,s] * W2[e] (silu(g) * u) with
 * (g, u) = W1[e] x[t], e = topk_idx[t,s] - expert_begin; slots whose expert is not one of the num_local do not count, a token without
 * a slot that does gets zeros.  The rows between the products keep 16 bits of mantissa.
 *   gate_up [L,2I,H]: gate rows, then up rows;  down [L,H,I];  x [T,H] 16-byte aligned;  topk_idx [T,K] of index_bytes 8 or 4;  y [T,H],
 *   which may be x, but overlaps topk_idx nowhere
 *   scratch  dpep_w4_experts_scratch_bytes, 16-byte aligned */
size_t dpep_w4_experts_scratch_bytes(int num_tokens, int num_topk, int hidden, int intermediate);
int dpep_w4_experts(const dpep_w4* gate_up, const dpep_w4* down, int type, const void* x, const void* topk_idx, int index_bytes, const float* topk_weights,
                    int num_tokens, int num_topk, int expert_begin, int num_local, void* y, void* scratch, void* stream);

/* What every token passes through beside the routed experts: norm, dense gated block, products in 8-bit integers.  The reference has
 * none of it.  "type" is DPEP_TYPE_*. */

/* Root-mean-square norm of the rows, after the residual's addition.  s = x, or x + residual rounded to `type`;
 * rstd = (mean of s^2 + eps)^-1/2;  v = s rstd weight, in fp32.
 *   x, residual (or NULL), stream_out (s; needed with a residual, may be x or the residual, NULL without one), y (v rounded, or NULL) [T,H] of
 *   `type`;  weight [H] of weight_type (`type` or fp32);  rstd fp32 [T] or NULL
 *   quantize  v in 8 bits, each value rounded from fp32 once:
 *     DPEP_QUANT_FP8    codes e4m3 [T,H], scales fp32 [T,ceil(H/128)]: as dpep_cast_to_fp8 (H a multiple of 16)
 *     DPEP_QUANT_MXFP8  codes e4m3 [T,H], scales e8m0 bytes [T,H/32]: as dpep_mx_quant (H a multiple of 32), and the scale NaN (255) for a
 *                       block of 32 that holds a NaN or an infinity
 *     DPEP_QUANT_INT8   codes int8 [T,H], scales fp32 [T]: as dpep_quantize_tokens (H a multiple of 16)
 * The squares are added up in fp32: a row whose sum passes its range (values of 1.8e19 / sqrt(H) and more) has rstd 0 and v 0, one whose mean square is below
 * it and eps 0 an infinite rstd; what is not finite in a row stays in that row's results.
 * H is a multiple of 8, at most DPEP_NORM_MAX_HIDDEN; pointers to rows are 16-byte aligned; T below 2^23.  Outputs overlap no input but for stream_out, nor
 * one another. */
#define DPEP_NORM_MAX_HIDDEN 16384
#define DPEP_NORM_MAX_TOKENS 0x7fffff
#define DPEP_QUANT_NONE 0
#define DPEP_QUANT_FP8 1
#define DPEP_QUANT_MXFP8 2
#define DPEP_QUANT_INT8 3
typedef struct dpep_norm {
    const void* x;
    const void* residual;
    const void* weight;
    void* stream_out;
    void* y;
    float* rstd;
    void* codes;
    void* scales;
    float eps;
    int32_t type, weight_type, quantize, num_tokens, hidden;
} dpep_norm;
int dpep_rms_norm(const dpep_norm* n, void* stream);
/* Its gradients, from that of y and (optional) that of s from elsewhere, with xh = s rstd and c the row's mean of grad_y weight xh:
 *   grad_x = rstd (grad_y weight - xh c) + grad_stream, of x and of the residual alike;  grad_weight[h] = sum over t of grad_y xh, fp32
 *   stream = s;  grad_x of `type` may be grad_y or grad_stream;  scratch dpep_rms_norm_backward_scratch_bytes, 16-byte aligned
 * Outputs and scratch overlap no other input, nor one another.  Sums are taken in an order that depends on the sizes alone. */
typedef struct dpep_norm_gradients {
    const void* grad_y;
    const void* stream;
    const void* weight;
    const float* rstd;
    const void* grad_stream;
    void* grad_x;
    float* grad_weight;
    int32_t type, weight_type, num_tokens, hidden;
} dpep_norm_gradients;
size_t dpep_rms_norm_backward_scratch_bytes(int num_tokens, int hidden);
int dpep_rms_norm_backward(const dpep_norm_gradients* g, void* scratch, void* stream);

/* The gated feed-forward block y = (silu(x Wg^T) * (x Wu^T)) Wd^T.
 *   gate_up [2I,H]: gate rows, then up rows;  down [H,I];  x, y [T,H]; all of `type` (BF16 or FP16), H and I multiples of 8 from 8 to
 *   DPEP_FFN_MAX_DIM, rows 16-byte aligned
 *   kept  fp32 [T,2I], the gate and up products for the backward, or NULL
 * Sums in fp32; the rows between the products are rounded to `type`, as the matrix cores take them.  Outputs and scratch (dpep_gated_ffn*_scratch_bytes,
 * 16-byte aligned) overlap no input, nor one another. */
#define DPEP_FFN_MAX_DIM 65536
#define DPEP_FFN_MAX_TOKENS 0x1fffff
typedef struct dpep_ffn {
    const void* gate_up;
    const void* down;
    int32_t type, hidden, inter;
} dpep_ffn;
size_t dpep_gated_ffn_scratch_bytes(int num_tokens, int hidden, int inter);
int dpep_gated_ffn(const dpep_ffn* f, const void* x, int num_tokens, void* y, float* kept, void* scratch, void* stream);
/* Gradients of x and of both matrices (of `type`), from that of y. */
size_t dpep_gated_ffn_backward_scratch_bytes(int num_tokens, int hidden, int inter);
int dpep_gated_ffn_backward(const dpep_ffn* f, const void* grad_y, const void* x, const float* kept, int num_tokens, void* grad_x, void* grad_gate_up,
                            void* grad_down, void* scratch, void* stream);

/* Tokens in 8-bit integers: scale = max(|x|) / 127 of the row (at least 1e-20 / 127), code = x * (127 / max(|x|)) rounded to nearest even.
 *   x [T,K] of `type`, 16-byte aligned, K a multiple of 16;  codes int8 [T,K] 16-byte aligned;  scales fp32 [T]
 * A row that holds a NaN gets a NaN for its scale; one that holds infinities gets infinity, 127 with their sign for their codes and 0 for the others'. */
int dpep_quantize_tokens(const void* x, int type, int num_tokens, int k, int8_t* codes, float* scales, void* stream);
/* y[t,n] = x_scales[t] scales[n] sum_k x[t,k] codes[n,k]: integer sums, exact; scaled in fp32, rounded once to `type`.
 *   codes int8 [N,K], x int8 [T,K]: 16-byte aligned, K a multiple of 16 up to DPEP_W8_MAX_K;  scales fp32 [N];  x_scales fp32 [T];  y [T,N];
 *   scratch  dpep_w8_matmul_scratch_bytes, 16-byte aligned;  y and scratch overlap no input, nor one another
 * ceil(T/256) ceil(N/256) is below 2^23 (results of 550 G and more do not fit the card). */
#define DPEP_W8_MAX_K 65536
#define DPEP_W8_MAX_N 0x1fffff
#define DPEP_W8_MAX_ROWS 0x1fffff
typedef struct dpep_w8 {
    const int8_t* codes;
    const float* scales;
    int32_t n, k;
} dpep_w8;
size_t dpep_w8_matmul_scratch_bytes(int num_rows, int n, int k);
int dpep_w8_matmul(const dpep_w8* w, const int8_t* x, const float* x_scales, int num_rows, int type, void* y, void* scratch, void* stream);

/* How calls of these sizes make their products, for tests and diagnosis.  Host arithmetic only.
 *   operation  DPEP_PRODUCTS_FFN: of rows, a = H and b = I, the gate and up product and the down product;  _FFN_BACKWARD: dh, then the gradients of x, gate_up and
 *              down;  _W8: of rows, a = N and b = K, one
 *   choices    room for 4.  Returns how many there are, or an error below zero */
#define DPEP_PRODUCTS_FFN 0
#define DPEP_PRODUCTS_FFN_BACKWARD 1
#define DPEP_PRODUCTS_W8 2
typedef struct dpep_product_choice {
    int32_t way;      /* 0 a stream of the matrix, tiles of 128 in a ring (1) or two workgroups to a compute unit (2), tiles of 256 (3) */
    int32_t parts;    /* of k; where there are more than one another kernel adds up their sums */
    int32_t stream_groups, stream_blocks, stream_stages; /* of a stream: groups of 16 columns and blocks of 16 rows of a workgroup, stages of its rings */
    int32_t together; /* in one launch with the other two */
    int64_t workgroups;
} dpep_product_choice;
int dpep_product_choices(int operation, int rows, int a, int b, dpep_product_choice* choices);

#ifdef __cplusplus
}
#endif
#endif
