/*
 * kim-kvcache B200 — C ABI of the sm_100a token-loop kernels.
 *
 * These entry points replace the reference's internal CUDA launch layer and
 * its cuBLAS calls:
 *   src/cuda/kv/kernels.cuh:31-143          cuda_detail::launch* (KV pages, attention)
 *   src/cuda/model/kernels.cuh:11-117       cuda_model_detail::launch* (norm, RoPE, ...)
 *   src/cuda/model/runner_support.cpp:196-274  cublasGemmEx wrappers (dense projections)
 *
 * Conventions: plain pointers to device memory, sizes in elements unless
 * named *_bytes, `stream` is a cudaStream_t (NULL = legacy default stream).
 * Every function returns 0 on a successful launch, KK_EINVAL for rejected
 * arguments (nothing is launched), or a CUDA runtime error code.
 * FP16 tensors are passed as uint16_t bit patterns.
 *
 * KV page layout (same as the reference, include/kim-kv/core/kv_layout.h:73-90):
 * a page holds every layer of its tokens as [layer][K/V][token][kv_head][dim];
 * micro pages hold 8 tokens, extent pages 64; pools are arrays of pages.
 */
#ifndef KK_KERNELS_H
#define KK_KERNELS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define KK_KAPI __attribute__((visibility("default")))
#else
#define KK_KAPI
#endif

#define KK_EINVAL 1000
/* Native error code of a transaction or step that failed because one of its
 * kernels reported an error (a descriptor outside its pool, a bounded device
 * wait that ran out) instead of the CUDA runtime. */
#define KK_EDEVICE 1002

typedef struct kk_kv_pools {
    void* micro;               /* micro_capacity pages of layers*2*T*kv_heads*head_dim fp16,
                                  T = micro_page_tokens (8 when 0) */
    void* extent;              /* extent_capacity pages of layers*2*64*kv_heads*head_dim fp16 */
    uint32_t micro_capacity;
    uint32_t extent_capacity;
    uint32_t layers;
    uint32_t kv_heads;
    uint32_t head_dim;
    uint32_t micro_page_tokens; /* tokens per micro page: 0 or 8 (the two-pool runtime), or
                                   16/32/64 for a fixed-page backend's pool (reference
                                   EngineBackendState(config, tokens_per_page, capacity),
                                   src/cuda/engine/backend.cpp:91-106); the extent pool is then
                                   unused (extent_capacity 0) */
} kk_kv_pools;

/* One block-table entry as the kernels read it (reference DeviceBlockDescriptor,
 * include/kim-kv/engine/engine_kv.h:100-117, without the generation). */
typedef struct kk_page_desc {
    uint32_t slot;
    uint32_t logical_token_begin;
    uint16_t valid_tokens;
    uint8_t kind;              /* 0 micro, 1 extent */
    uint8_t reserved0;
    uint32_t reserved1;
} kk_page_desc;

/* Destination of one lane's new token (reference CudaEngineTransaction::writeLayer
 * slot mapping, src/cuda/engine/transaction.cpp:158-194). */
typedef struct kk_kv_slot {
    uint32_t slot;
    uint16_t page_token;
    uint8_t kind;
    uint8_t active;            /* 0: lane skipped */
} kk_kv_slot;

/* Partial-tail copy-on-write: first `tokens` tokens of src -> dst. */
typedef struct kk_kv_copy {
    uint32_t src_slot;
    uint32_t dst_slot;
    uint16_t tokens;
    uint8_t src_kind;
    uint8_t dst_kind;
} kk_kv_copy;

/* One lane of a ragged decode-attention batch (reference DevicePagedDecodeBatchItem,
 * include/kim-kv/engine/engine_kv.h:172-181). */
typedef struct kk_attn_lane {
    uint32_t desc_offset;      /* first entry of this lane in the descriptor array */
    uint32_t desc_count;
    uint32_t token_count;      /* attended tokens, current token included */
    uint32_t item_offset;      /* filled by kk_attention_plan */
    uint32_t item_count;       /* filled by kk_attention_plan */
    uint32_t query_row;        /* row of query / output used by this lane */
    uint32_t first_item_shared; /* filled by the planners: 1 when the lane's first item
                                   begins in an earlier lane */
    uint32_t reserved;
} kk_attn_lane;

/* A split-KV work item: a run [desc_begin, desc_end) of the descriptor array.
 * Items of kk_attention_plan lie inside one lane (flags 0); items of
 * kk_attention_plan_balanced may continue from `lane` into the following
 * lanes when their descriptors are contiguous (flags KK_ATTN_ITEM_MULTI_LANE),
 * and may cut a full 64-token extent page in half: the item's first
 * descriptor then starts at token KK_ATTN_ITEM_SKIP(flags) and its last one
 * ends at token KK_ATTN_ITEM_LIMIT(flags) (0: at its valid count), so two
 * consecutive items share that descriptor. Only extent descriptors may be cut. */
#define KK_ATTN_ITEM_MULTI_LANE 1u
#define KK_ATTN_ITEM_SKIP(flags) (((flags) >> 8) & 0xffu)
#define KK_ATTN_ITEM_LIMIT(flags) (((flags) >> 16) & 0xffu)
#define KK_ATTN_EXTENT_HALF 32u
typedef struct kk_attn_item {
    uint32_t lane;             /* first lane of the item */
    uint32_t desc_begin;
    uint32_t desc_end;
    uint32_t reserved;         /* flags */
} kk_attn_item;

/* ---- K1: fused GQA paged decode attention ------------------------------------
 * Replaces launchPagedDecodeAttention / launchPagedDecodeAttentionBatch
 * (src/cuda/attention/paged_decode_kernels.cu:533-617): QK^T, online softmax and
 * PV in one pass that walks micro and extent entries directly, all lanes and
 * KV heads of a layer in one launch, split over the context with a combine.
 * head_dim must be 64; kv_heads in {1,2,4,8}; q_heads/kv_heads <= 16.
 * query/output rows: [q_heads][head_dim] fp16 at row stride *_stride elements. */
KK_KAPI uint32_t kk_attention_plan(const kk_page_desc* host_descs, kk_attn_lane* host_lanes,
    uint32_t num_lanes, uint32_t target_tokens, kk_attn_item* host_items, uint32_t max_items);
/* Token-balanced plan (no counterpart in the reference): cuts the batch's
 * token stream, lane after lane, into about num_parts runs of equal token
 * count at page granularity (use the SM count: one run per SM). Runs may span
 * lanes; a lane split across runs is combined by the split-KV combine. Fills
 * item_offset/item_count/first_item_shared of every lane; returns the item count (items beyond
 * max_items are counted, not written). Served by the TMA kernel only. */
KK_KAPI uint32_t kk_attention_plan_balanced(const kk_page_desc* host_descs,
    kk_attn_lane* host_lanes, uint32_t num_lanes, uint32_t num_parts, kk_attn_item* host_items,
    uint32_t max_items);
KK_KAPI uint64_t kk_attention_workspace_bytes(uint32_t num_lanes, uint32_t num_items,
    uint32_t q_heads, uint32_t head_dim);
/* Zero-fills the per-lane completion counters of a fresh workspace (once). */
KK_KAPI int kk_attention_workspace_init(void* workspace, uint32_t num_lanes, void* stream);
KK_KAPI int kk_paged_decode_attention(const kk_kv_pools* pools, uint32_t layer,
    uint32_t q_heads, const kk_page_desc* descs, const kk_attn_lane* lanes, uint32_t num_lanes,
    const kk_attn_item* items, uint32_t num_items, const uint16_t* query, uint32_t query_stride,
    uint16_t* output, uint32_t output_stride, float scale, void* workspace,
    uint64_t workspace_bytes, void* stream);

/* kk_paged_decode_attention without a caller workspace. No counterpart in
 * the reference, which allocates attention scratch per call.
 *
 * It is for callers that cannot allocate device memory for the workspace:
 *  - hosts that reach the library through an FFI (cgo, JNI, ctypes) with only
 *    raw stream handles and no device allocator of their own;
 *  - serving loops that must not call cudaMalloc per step, because it
 *    synchronizes the device and its latency is unbounded.
 *
 * The completion counters and partial softmax states live in one fixed
 * device array of KK_ATTN_SCRATCH_BYTES (4 MiB) per device, created with the
 * library's module. A call that needs more,
 * kk_attention_workspace_bytes(num_lanes, num_items, q_heads, 64) >
 * KK_ATTN_SCRATCH_BYTES, is rejected with KK_ENOSCRATCH and launches
 * nothing. For scale: 64 lanes x 148 items x 32 query heads need 2.5 MB.
 *
 * The per-lane completion counters at the start of the scratch must be zero
 * when a kernel starts. This entry point zeroes them on `stream` before every
 * launch. Nothing else needs initial values.
 *
 * The first call on each device (the device that owns `stream`) looks up the
 * scratch address; make it before any stream capture. Arguments are checked
 * before anything is queued: a rejected call writes nothing. Calls that can overlap on one device (different
 * streams, or several host threads) share the one scratch array and race:
 * serialize them on one stream, or use kk_paged_decode_attention with a
 * workspace per stream. Other arguments, results and errors are those of
 * kk_paged_decode_attention. */
#define KK_ATTN_SCRATCH_BYTES (4u << 20)
#define KK_ENOSCRATCH 1001
KK_KAPI int kk_paged_decode_attention_noalloc(const kk_kv_pools* pools, uint32_t layer,
    uint32_t q_heads, const kk_page_desc* descs, const kk_attn_lane* lanes, uint32_t num_lanes,
    const kk_attn_item* items, uint32_t num_items, const uint16_t* query, uint32_t query_stride,
    uint16_t* output, uint32_t output_stride, float scale, void* stream);

/* Kernel used by kk_paged_decode_attention (process-wide; default AUTO). No
 * counterpart in the reference (it has one attention implementation).
 *  KK_ATTN_AUTO   : the TMA kernel where supported (kv_heads in {1,2,4,8},
 *                   which is every shape the direct-load kernel serves);
 *  KK_ATTN_DIRECT : always the direct-load kernel (warps load K/V rows into
 *                   registers);
 *  KK_ATTN_TMA    : always the TMA kernel (persistent, warp-specialised, K/V
 *                   staged through a 3-stage shared-memory ring); calls it
 *                   cannot serve return KK_EINVAL.
 * The direct-load kernel rejects multi-lane items (device status
 * kErrBadArgument = 3, items skipped).
 * Both produce the same results within FP32 rounding of the softmax sums.
 * Returns 0 or KK_EINVAL for an unknown value. */
#define KK_ATTN_AUTO 0
#define KK_ATTN_DIRECT 1
#define KK_ATTN_TMA 2
KK_KAPI int kk_attention_set_variant(int variant);

/* ---- K8: decode attention of lanes that share a prefix ----------------------------
 * No counterpart in the reference, whose forks each read the shared pages
 * (paged_decode_kernels.cu:533-617 walks every lane's whole table). Lanes whose
 * block tables begin with the same pages (forks of one prompt, the positions
 * of one prompt chunk) form a group; the group's pages are read once for all of
 * its query rows, each lane's remaining pages for that lane alone, and the
 * softmax parts are joined exactly. Same results as kk_paged_decode_attention
 * over the whole tables, up to FP32 rounding of the softmax sums and 2^-21 of a
 * weight (2^-32 of the row's largest one, if that is more).
 *
 * Host side, once per step (the plan serves every layer):
 *   kk_prefix_groups finds the groups and cuts the shared pages off the lanes'
 *   tables; kk_prefix_attention_plan makes the work list; descriptors, lanes,
 *   groups and items are copied to the device.
 * head_dim must be 64; q_heads / kv_heads <= 16. */
typedef struct kk_prefix_group {
    uint32_t desc_offset;      /* the shared pages' descriptors */
    uint32_t desc_count;
    uint32_t token_count;
    uint32_t lane_begin;       /* lanes [lane_begin, lane_begin + lane_count) share them */
    uint32_t lane_count;
    uint32_t part_row;         /* filled by the plan: first partial row, */
    uint32_t part_count;       /* splits of the prefix, */
    uint32_t row_tiles;        /* tiles of 128 query rows per KV head */
} kk_prefix_group;

typedef struct kk_prefix_item {
    uint32_t owner;            /* group (row_tiles != 0) or lane (row_tiles == 0) */
    uint32_t kv_head;
    uint32_t desc_begin;       /* run of the descriptor array */
    uint32_t desc_end;
    uint32_t part;
    uint16_t row_tile;         /* first tile of query rows */
    uint16_t row_tiles;        /* 1 or 2; 0: a lane's own pages */
    uint32_t token_tiles;      /* 128-token tiles of the run */
    uint32_t part_row;         /* first partial row that the item writes */
    uint32_t lane_begin;       /* the group's lanes */
    uint32_t lane_count;
    uint32_t query_row;        /* the lane's (row_tiles == 0) */
    uint32_t reserved;
} kk_prefix_item;

typedef struct kk_prefix_plan {
    uint32_t num_items;        /* shared items first, then lanes' own */
    uint32_t num_shared;
    uint32_t tasks_per_cta;    /* lanes' own items per thread block */
    uint32_t num_lanes;
    uint32_t num_groups;
    uint32_t num_descs;
    uint32_t q_heads;
    uint32_t kv_heads;
    uint64_t part_rows;        /* partial softmax rows in the workspace */
} kk_prefix_plan;

/* Finds runs of at least max(2, min_lanes) consecutive lanes whose tables
 * begin with the same pages (slot, kind and valid tokens) for at least
 * min_tokens tokens, writes a group for each and moves the shared descriptors
 * out of those lanes (desc_offset, desc_count, token_count). A group takes all
 * pages that its lanes have in common. Of all ways to cut the lanes into runs
 * the one with the largest sum of (lanes - 1) * (shared tokens + 1375) is taken
 * (1375: what a group costs besides its tokens). Only neighbours are grouped: a
 * caller puts lanes of one prefix next to each other (query_row leaves their
 * rows where they are). A small group can cost more than it saves (36 pairs that
 * share 300 tokens, 4 KV heads: 19.0 us, 14.6 without groups; 30 times four lanes
 * that share 3,000, 8 KV heads: 90 us, 174 without): min_lanes and min_tokens
 * leave those out. Returns the groups written, the first max_groups. */
KK_KAPI uint32_t kk_prefix_groups(const kk_page_desc* host_descs, kk_attn_lane* host_lanes,
    uint32_t num_lanes, uint32_t min_lanes, uint32_t min_tokens, kk_prefix_group* host_groups,
    uint32_t max_groups);
/* Splits the groups' pages and the lanes' own pages into items for num_sms
 * SMs. Fills item_offset, item_count and reserved (1 + group, 0: none) of
 * every lane, the part fields of every group, the items (those beyond
 * max_items are counted, not written) and the plan. Groups may come from
 * kk_prefix_groups or be made by the caller; a lane belongs to one group at
 * most. KK_EINVAL: a range outside its array, a lane in two groups, head
 * counts that are not served, or more than 2^32 - 1 partial rows. */
KK_KAPI int kk_prefix_attention_plan(const kk_page_desc* host_descs, uint32_t num_descs,
    kk_attn_lane* host_lanes, uint32_t num_lanes, kk_prefix_group* host_groups, uint32_t num_groups,
    uint32_t q_heads, uint32_t kv_heads, uint32_t num_sms, kk_prefix_item* host_items,
    uint32_t max_items, kk_prefix_plan* plan);
/* Workspace of a call (16-byte aligned, no initial values). Calls that can
 * overlap need one each. */
KK_KAPI uint64_t kk_prefix_attention_workspace_bytes(const kk_prefix_plan* plan);

typedef struct kk_prefix_attn_desc {
    kk_kv_pools pools;
    uint32_t layer;
    uint32_t q_heads;
    float scale;
    uint32_t reserved;
    kk_prefix_plan plan;
    const kk_page_desc* descs;      /* device copies of the plan's arrays */
    const kk_attn_lane* lanes;
    const kk_prefix_group* groups;
    const kk_prefix_item* items;
    const uint16_t* query;          /* rows lane.query_row: [q_heads][64] at query_stride */
    uint16_t* output;
    uint64_t query_stride;
    uint64_t output_stride;
    void* workspace;
    uint64_t workspace_bytes;
} kk_prefix_attn_desc;
/* A lane that has no tokens at all gets zeros. Descriptors outside their pool
 * or over their page contribute nothing and are reported by kk_device_status,
 * as are items that do not fit the plan. query, output and workspace are
 * 16-byte aligned, the plan's arrays 4-byte, strides multiples of 8. Two lanes
 * must not name the same query row. */
KK_KAPI int kk_prefix_attention(const kk_prefix_attn_desc* desc, void* stream);

/* ---- K2: batched KV append / copy-on-write -----------------------------------
 * kk_kv_write replaces launchWriteLayerToken (paged_decode_kernels.cu:65-99) and
 * launchAppendTokens (src/cuda/kv/page_kernels.cu:77-127) for one token per
 * lane: writes K and V of layers [layer_begin, +layer_count) for every active
 * lane. key/value element (lane, layer, head, dim) lives at
 * lane*lane_stride + layer*layer_stride + head*head_dim + dim.
 * kk_kv_copy_tokens replaces launchCopyLayerTokens / launchCopyPageTokens
 * (paged_decode_kernels.cu:29-63, page_kernels.cu:46-75). */
KK_KAPI int kk_kv_write(const kk_kv_pools* pools, uint32_t layer_begin, uint32_t layer_count,
    const kk_kv_slot* slots, uint32_t num_lanes, const uint16_t* key, const uint16_t* value,
    uint64_t lane_stride, uint64_t layer_stride, void* stream);
KK_KAPI int kk_kv_copy_tokens(const kk_kv_pools* pools, uint32_t layer_begin,
    uint32_t layer_count, const kk_kv_copy* copies, uint32_t num_copies, void* stream);

/* Rotating append of a ragged batch (no counterpart in the reference, whose
 * appends copy already rotated tokens, page_kernels.cu:77-127): one pass over
 * `rows` token rows of any number of sequences rotates queries and keys to
 * their positions and writes keys and values of one layer into the pages.
 * Row r: pairs (d, d + rotary_dim/2) of every query and key head, d <
 * rotary_dim/2, turn by positions[r] * theta^(-2d / rotary_dim); the other
 * dims are copied. The angle is reduced in 64-bit fixed point and is off by
 * less than 4e-6 rad at any 32-bit position; products are FP32, rounded once to
 * FP16.
 * A row whose slot is inactive is skipped: its query_out row and every page
 * stay as they were. A slot outside its pool, or a position outside cos_sin's
 * table, skips the row too and is reported by kk_device_status. Two active
 * rows of one call must not name the same (slot, token).
 * head_dim % 8 == 0, rotary_dim % 16 == 0, rotary_dim <= min(head_dim, 256);
 * pointers 16-byte aligned (cos_sin: 8, slots and positions: 4), strides multiples of 8 and not below
 * the row they step over. query_out may be query itself (same stride). */
typedef struct kk_kv_append_desc {
    kk_kv_pools pools;
    uint32_t layer;
    uint32_t rows;              /* 0: nothing is launched */
    uint32_t q_heads;           /* 0: no queries (query, query_out ignored) */
    uint32_t rotary_dim;        /* 0: no rotation (theta, positions, cos_sin ignored) */
    float theta;                /* >= 1 */
    uint32_t table_positions;   /* rows of cos_sin */
    const float* cos_sin;       /* optional [table_positions][rotary_dim / 2] pairs (cos, sin)
                                   used in place of theta */
    const kk_kv_slot* slots;    /* [rows] */
    const uint32_t* positions;  /* [rows] */
    const uint16_t* query;      /* [rows][q_heads][head_dim] at query_stride, and so on */
    const uint16_t* key;
    const uint16_t* value;
    uint16_t* query_out;
    uint64_t query_stride;
    uint64_t key_stride;
    uint64_t value_stride;
    uint64_t query_out_stride;
} kk_kv_append_desc;
KK_KAPI int kk_kv_append_rope(const kk_kv_append_desc* desc, void* stream);

/* Promotion copy: the 8 micro pages micro_slots[0..7] (all layers) become the
 * extent page extent_slot, tokens 8k..8k+7 <- micro page k (replaces
 * launchPromotion, src/cuda/kv/page_kernels.cu:129-182). */
KK_KAPI int kk_kv_promote(const kk_kv_pools* pools, const uint32_t* micro_slots_host,
    uint32_t extent_slot, void* stream);
/* K6 data path between pages and a contiguous KV tensor
 * [layer][K|V][token][head][dim] fp16 (16-byte aligned).
 * kk_kv_gather replaces gatherAsync / launchGather (src/cuda/kv/gather.cpp:9-107,
 * page_kernels.cu:184-242): every descriptor's valid tokens are copied to
 * out at their logical positions; tokens of [0, total_tokens) not covered by
 * any descriptor are left untouched. Descriptors must not overlap.
 * kk_kv_scatter is the inverse for appended tokens (appendAsync segment
 * copies, launchAppendTokens, page_kernels.cu:77-127): `in` holds the
 * [layer][K|V][token_count][head][dim] values of logical tokens
 * [first_token, first_token + token_count), written into the pages that the
 * descriptors map there. One CTA per (descriptor, layer, K|V). A descriptor
 * outside its pool is skipped and reported by kk_device_status. */
KK_KAPI int kk_kv_gather(const kk_kv_pools* pools, const kk_page_desc* descs, uint32_t num_descs,
    uint32_t total_tokens, uint16_t* out, void* stream);
KK_KAPI int kk_kv_scatter(const kk_kv_pools* pools, const kk_page_desc* descs, uint32_t num_descs,
    uint32_t first_token, uint32_t token_count, const uint16_t* in, void* stream);
/* Deterministic pseudo-random FP16 fill (uniform in [-scale, scale)) for
 * synthetic KV pages and test tensors; same (seed, index) -> same value. */
KK_KAPI int kk_fill_fp16(uint16_t* data, uint64_t count, uint64_t seed, float scale,
    void* stream);

/* ---- K3: norms, RoPE, SiLU gate, residual -------------------------------------
 * Replace launchRmsNorm(Batch), launchRope(Batch), launchSwiGlu, launchResidualAdd,
 * launchEmbedding(Batch) (src/cuda/model/kernels.cu:16-218). */
KK_KAPI int kk_rmsnorm(const uint16_t* x, const uint16_t* weight, uint16_t* y, uint32_t rows,
    uint32_t cols, float eps, void* stream);
KK_KAPI int kk_embed_rmsnorm(const uint16_t* embed, const uint32_t* tokens,
    const uint16_t* weight, uint16_t* hidden, uint16_t* y, uint32_t rows, uint32_t cols,
    float eps, void* stream);
KK_KAPI int kk_rope(uint16_t* q, uint32_t q_stride, uint16_t* k, uint32_t k_stride,
    const uint32_t* positions, uint32_t rows, uint32_t q_heads, uint32_t kv_heads,
    uint32_t head_dim, float theta, void* stream);
KK_KAPI int kk_silu_mul(const uint16_t* gate, const uint16_t* up, uint16_t* out, uint32_t rows,
    uint32_t cols, void* stream);
KK_KAPI int kk_residual_add(uint16_t* hidden, const uint16_t* update, uint64_t count,
    void* stream);

/* ---- K4/K5: tcgen05 weight-streaming GEMM with fused epilogues ---------------
 * Y[n][m] = sum_k W[m][k] * X[n][k] for m < M, n < N (N <= 64): FP16 operands,
 * FP32 accumulation in tensor memory, split-K across a thread-block cluster with
 * a distributed-shared-memory reduction, then one of the epilogues below.
 * Replaces cublasGemmEx in gemmBatch / logitsGemmBatch
 * (src/cuda/model/runner_support.cpp:196-274) plus the elementwise kernel that
 * follows each projection. K % 8 == 0. */
enum kk_epilogue {
    KK_EPI_STORE_F16 = 0,    /* out[n*out_stride+m] = half(acc) */
    KK_EPI_STORE_F32 = 1,    /* out[n*out_stride+m] = acc */
    KK_EPI_RESIDUAL = 2,     /* out[...] = hadd(out[...], half(acc)) */
    KK_EPI_SILU_PAIRS = 3,   /* rows 2i / 2i+1 = gate_i / up_i: out[n*out_stride+i] =
                                half(silu(half(g)) * half(u)) */
    KK_EPI_QKV_ROPE = 4,     /* rows [0,q_rows): q, RoPE'd into out; next kv_rows: k,
                                RoPE'd into the KV page slot; next kv_rows: v into the page */
    KK_EPI_ARGMAX = 5,       /* fp32 logits (optional) + greedy argmax per column */
};

typedef struct kk_gemm_desc {
    const uint16_t* weight;    /* [M][K] fp16 row-major */
    uint32_t M;
    uint32_t K;
    const uint16_t* x;         /* [x_rows][x_stride] fp16 */
    uint32_t N;
    uint32_t x_stride;
    uint32_t x_rows;           /* allocated rows of x (>= N) */
    uint32_t epilogue;
    void* out;
    uint32_t out_stride;
    uint32_t split_k;          /* 0 = choose automatically */
    /* KK_EPI_QKV_ROPE */
    const uint32_t* positions; /* [N] */
    const kk_kv_slot* slots;   /* [N] */
    kk_kv_pools pools;
    uint32_t layer;
    uint32_t q_rows;
    uint32_t kv_rows;
    uint32_t head_dim;
    float rope_theta;
    /* KK_EPI_ARGMAX */
    uint32_t* tokens;          /* [N] greedy ids */
    void* argmax_workspace;    /* kk_argmax_workspace_bytes(M, N) bytes, zeroed once */
    uint32_t weight_layout;    /* KK_W_ROW_MAJOR, or KK_W_PACKED: weight holds
                                  kk_gemm_pack_weight output for (M, K) */
    /* Fused RMSNorm of the input rows (replaces a separate rmsNormBatchKernel,
     * src/cuda/model/kernels.cu:48-124, at the same FP16 rounding point): when
     * norm_input is set, every X tile is normalised in shared memory before
     * the tensor cores read it, X'[n][k] = half(x[n][k] * r[n] * g[k]) with
     * r[n] = 1 / sqrt(mean_k norm_input[n][k]^2 + norm_eps) and g =
     * norm_weight (1 when NULL); then Y = X' W^T. With x = norm_input this is
     * the reference's half(RMSNorm(x)) followed by the projection. */
    const uint16_t* norm_input; /* [N][norm_stride] fp16, 16-byte aligned, or NULL */
    uint32_t norm_stride;
    float norm_eps;
    const uint16_t* norm_weight; /* [K] fp16, 16-byte aligned, or NULL */
    /* KK_EPI_QKV_ROPE: optional table of the rotation factors, [rope_positions]
     * [head_dim / 2] pairs (cos, sin) of position * theta^(-2d / head_dim),
     * 8-byte aligned; NULL computes them in the kernel (sincosf). The runner
     * fills it once on the host, with the host math library the reference's
     * model uses, for every position up to max_position_embeddings. */
    const float* rope_cos_sin;
    uint32_t rope_positions;
} kk_gemm_desc;

#define KK_W_ROW_MAJOR 0
#define KK_W_PACKED 1
/* Weight packing (no counterpart in the reference, whose cuBLAS calls read the
 * row-major tensors): W [M][K] row-major (K % 8 == 0, 16-byte aligned) ->
 * 128x64 tiles of 16 KB, each contiguous and pre-swizzled, so that the GEMM
 * streams one tile per untiled bulk copy. Rows and columns are zero-padded to
 * multiples of 128 and 64. Done once at weight load. */
KK_KAPI uint64_t kk_gemm_packed_bytes(uint32_t M, uint32_t K);
KK_KAPI int kk_gemm_pack_weight(const uint16_t* weight, uint32_t M, uint32_t K,
    uint16_t* packed, void* stream);
/* The same with every column k scaled by col_scale[k] (fp16, 16-byte aligned)
 * before packing, W'[m][k] = half(W[m][k] * col_scale[k]): folds an RMSNorm
 * weight into the projection that consumes the normalised rows. */
KK_KAPI int kk_gemm_pack_weight_scaled(const uint16_t* weight, uint32_t M, uint32_t K,
    const uint16_t* col_scale, uint16_t* packed, void* stream);

KK_KAPI uint64_t kk_argmax_workspace_bytes(uint32_t M, uint32_t N);
KK_KAPI int kk_gemm(const kk_gemm_desc* desc, void* stream);

/* ---- K7: penalties, biases and grammar masks on logits, greedy token -----------
 * No counterpart in the reference (its LM head takes the argmax of the raw
 * logits). Row r of FP32 logits x becomes, token by token, in this order:
 *   1. v in the row's history (prompt or output), repetition p:
 *        x = x > 0 ? x / p : x * p;
 *   2. v given n >= 1 times in the output part of the history:
 *        x = x - frequency * n, then x = x - presence;
 *   3. v in the row's bias list: x = x + bias (of several entries for v the
 *      last one counts);
 *   4. v's mask bit clear: x = -inf, whatever x was (NaN included).
 * Every operation is rounded to FP32 by itself. tokens[r] is the token of the
 * highest logit, the lowest id among equals; NaN and -inf are never chosen, and
 * a row that leaves nothing else gets KK_NO_TOKEN. Results do not depend on
 * the order in which threads run.
 * Strides are in elements; rows may start at any multiple of 4 bytes. vocab is
 * at most 400,000 where a history or biases are given, 10 million with a mask
 * alone, 2^30 with none of them.
 * Ids outside the vocabulary are ignored. Offsets that decrease or pass their
 * array and mask rows outside the masks are reported by kk_device_status; the
 * row's history or biases are then left out, respectively the row is masked
 * entirely. Bias ids that descend within a row are reported too; what that row
 * gets of its biases is not specified. Arrays are 4-byte aligned; history_size
 * and bias_size are at most 2^32 - 256. */
#define KK_NO_TOKEN 0xffffffffu
#define KK_NO_MASK 0xffffffffu
typedef struct kk_logits_desc {
    const float* logits;             /* [rows][vocab] at logits_stride */
    float* out;                      /* may be logits itself (same stride); NULL: not written */
    uint32_t* tokens;                /* [rows], or NULL */
    uint64_t logits_stride;
    uint64_t out_stride;
    uint32_t rows;
    uint32_t vocab;
    /* Penalties: row r's token ids are history[history_offsets[r] .. [r + 1]),
     * the first prompt_counts[r] of them the prompt (NULL: none). A NULL
     * factor array is neutral (1, 0, 0); all three NULL: no history is read. */
    const uint32_t* history;
    const uint32_t* history_offsets; /* [rows + 1] */
    const uint32_t* prompt_counts;   /* [rows] */
    const float* repetition;         /* [rows] */
    const float* presence;
    const float* frequency;
    uint64_t history_size;           /* entries of history */
    /* Biases: row r's pairs are those at bias_offsets[r] .. [r + 1), ids
     * ascending. NULL offsets: none. */
    const uint32_t* bias_tokens;
    const float* bias_values;
    const uint32_t* bias_offsets;    /* [rows + 1] */
    uint64_t bias_size;
    /* Grammar masks: bit v % 32 of word v / 32 of a mask set: v is allowed.
     * Row r uses mask mask_rows[r] (KK_NO_MASK: all allowed; NULL: mask r).
     * NULL mask: none. */
    const uint32_t* mask;            /* [num_masks] rows of mask_stride words */
    const uint32_t* mask_rows;       /* [rows] */
    uint32_t mask_stride;
    uint32_t num_masks;
} kk_logits_desc;
KK_KAPI int kk_logits_process(const kk_logits_desc* desc, void* stream);

/* Reads and clears the device-side status words of all kernel modules
 * (synchronises the stream). 0 = no kernel recorded an error. These words
 * collect the errors of the entry points above; the runtime's own launches
 * (kk_runtime.h: the runner's fused step, the backend's per-layer
 * transactions) report into per-step and per-stream words of their own and
 * fail the affected transactions at commit. */
KK_KAPI int kk_device_status(void* stream);

/* Test hook for the bounded waits of K1 (no counterpart in the reference,
 * whose failure injection is host-side only): from the next launch on, CTA 0
 * of every TMA attention launch on the current device drops its stage number
 * `stage` (issues no copy and no arrival for it), so that the consumers'
 * bounded wait runs out after `wait_limit_ns` and the kernel reports
 * kErrWaitTimeout and returns. stage 0xFFFFFFFF and wait_limit_ns 0 restore
 * the defaults (no stage dropped, 2 s). Call it with no kernel in flight. */
KK_KAPI int kk_debug_attention_fault(uint32_t stage, uint64_t wait_limit_ns);

/* Programmatic dependent launch for subsequent launches on this thread (0/1). */
KK_KAPI void kk_set_pdl(int enabled);

#ifdef __cplusplus
}
#endif

#endif /* KK_KERNELS_H */
