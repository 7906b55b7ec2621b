// K2 — batched KV append and copy-on-write over the page pools.
//
// kk_kv_write: one launch writes the new token's K and V of a range of layers
// for every lane (the reference issues one tiny launch per lane per layer,
// src/cuda/engine/transaction.cpp:195-204). One warp moves one (lane, layer,
// K|V) row of kv_heads*head_dim FP16 values with 16-byte accesses.
// kk_kv_copy_tokens: partial-tail copy-on-write of the first `tokens` tokens
// of a page into a fresh page, for a range of layers (reference
// copyLayerTokensKernel / copyPageTokensKernel, paged_decode_kernels.cu:29-63,
// page_kernels.cu:46-75). Both are bandwidth-bound byte movers.
// kk_kv_append_rope: rotary embedding of a layer's new queries and keys, with
// the keys and values written into their pages by the same pass.
#include "../../../include/kk_kernels.h"
#include "kernels_internal.h"
#include "launch.cuh"

#include <cmath>
#include <limits>

namespace kk {

__device__ unsigned int g_pages_status;

namespace {

struct PoolView {
    __half* micro;
    __half* extent;
    std::uint64_t micro_page;
    std::uint64_t extent_page;
    std::uint32_t micro_slots;
    std::uint32_t extent_slots;
    std::uint32_t row;         // kv_heads * head_dim elements per token per K|V
    std::uint32_t layers;
    std::uint32_t micro_cap;   // tokens per micro page
    unsigned int* status;      // error word of the launch (null: the module's word)
};

__device__ __forceinline__ void report(PoolView const& v, unsigned int code)
{
    atomicCAS(v.status != nullptr ? v.status : &g_pages_status, kErrNone, code);
}

PoolView view(kk_kv_pools const& p)
{
    PoolView v{};
    v.micro = static_cast<__half*>(p.micro);
    v.extent = static_cast<__half*>(p.extent);
    v.row = p.kv_heads * p.head_dim;
    v.micro_cap = microPageTokens(p);
    v.micro_page = std::uint64_t(p.layers) * 2u * v.micro_cap * v.row;
    v.extent_page = std::uint64_t(p.layers) * 2u * 64u * v.row;
    v.micro_slots = p.micro == nullptr ? 0 : p.micro_capacity;
    v.extent_slots = p.extent == nullptr ? 0 : p.extent_capacity;
    v.layers = p.layers;
    return v;
}

// Start of the (layer, component) block of a page; nullptr if out of bounds.
__device__ __forceinline__ __half* block_of(PoolView const& v, std::uint32_t kind,
    std::uint32_t slot, std::uint32_t layer, std::uint32_t component)
{
    bool const micro = kind == 0;
    if (micro ? slot >= v.micro_slots : slot >= v.extent_slots) {
        report(v, kErrBadDescriptor);
        return nullptr;
    }
    std::uint32_t const cap = micro ? v.micro_cap : 64u;
    __half* page = micro ? v.micro + std::uint64_t(slot) * v.micro_page
                         : v.extent + std::uint64_t(slot) * v.extent_page;
    return page + (std::uint64_t(layer) * 2u + component) * cap * v.row;
}

// grid: (num_lanes, layer_count, 2); one warp per row, 8 elements per thread step.
__global__ void kv_write_kernel(PoolView v, std::uint32_t layer_begin, kk_kv_slot const* slots,
    __half const* key, __half const* value, std::uint64_t lane_stride, std::uint64_t layer_stride)
{
    pdl_wait();
    std::uint32_t const lane_idx = blockIdx.x;
    std::uint32_t const layer_off = blockIdx.y;
    std::uint32_t const component = blockIdx.z;
    kk_kv_slot const s = slots[lane_idx];
    if (!s.active) {
        return;
    }
    std::uint32_t const cap = s.kind == 0 ? v.micro_cap : 64u;
    if (s.page_token >= cap) {
        report(v, kErrBadDescriptor);
        return;
    }
    __half* dst = block_of(v, s.kind, s.slot, layer_begin + layer_off, component);
    if (dst == nullptr) {
        return;
    }
    dst += std::uint64_t(s.page_token) * v.row;
    __half const* src = (component == 0 ? key : value) + lane_idx * lane_stride
        + layer_off * layer_stride;
    for (std::uint32_t i = threadIdx.x * 8u; i < v.row; i += blockDim.x * 8u) {
        *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<uint4 const*>(src + i);
    }
}

// grid: (num_copies, layer_count, 2): copies tokens*row contiguous elements.
__global__ void kv_copy_kernel(PoolView v, std::uint32_t layer_begin, kk_kv_copy const* copies,
    std::uint32_t const* count)
{
    pdl_wait();
    if (count != nullptr && blockIdx.x >= *count) {
        return;
    }
    kk_kv_copy const c = copies[blockIdx.x];
    std::uint32_t const layer = layer_begin + blockIdx.y;
    std::uint32_t const component = blockIdx.z;
    std::uint32_t const src_cap = c.src_kind == 0 ? v.micro_cap : 64u;
    std::uint32_t const dst_cap = c.dst_kind == 0 ? v.micro_cap : 64u;
    if (c.tokens > src_cap || c.tokens > dst_cap) {
        report(v, kErrBadDescriptor);
        return;
    }
    __half const* src = block_of(v, c.src_kind, c.src_slot, layer, component);
    __half* dst = block_of(v, c.dst_kind, c.dst_slot, layer, component);
    if (src == nullptr || dst == nullptr) {
        return;
    }
    std::uint64_t const n = std::uint64_t(c.tokens) * v.row;
    for (std::uint64_t i = threadIdx.x * 8u; i < n; i += blockDim.x * 8u) {
        *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<uint4 const*>(src + i);
    }
}

// ---- kk_kv_append_rope --------------------------------------------------------

constexpr std::uint32_t kMaxRotaryDim = 256;
constexpr int kAppendThreads = 256;
constexpr std::uint32_t kAppendWave = 148 * 5;  // CTAs that the SMs hold at once
constexpr std::uint32_t kTailBatch = 3;  // copies in flight per thread (one: 16.0 us, three: 14.6, for 4,999 half rotated rows)
constexpr std::uint32_t kAppendMaxRows = 8;  // rows per CTA, at most

struct AppendArgs {
    PoolView pools;
    std::uint32_t layer;
    std::uint32_t rows;
    std::uint32_t rows_per_cta;
    std::uint32_t q_heads;
    std::uint32_t kv_heads;
    std::uint32_t head_dim;
    std::uint32_t rotary_half;
    std::uint32_t table_positions;
    float2 const* cos_sin;
    kk_kv_slot const* slots;
    std::uint32_t const* positions;
    __half const* query;
    __half const* key;
    __half const* value;
    __half* query_out;
    std::uint64_t query_stride;
    std::uint64_t key_stride;
    std::uint64_t value_stride;
    std::uint64_t query_out_stride;
    // theta^(-2d / rotary_dim) / (2 pi) turns per position, as 0.64 fixed point.
    std::uint64_t turns[kMaxRotaryDim / 2];
};

// Rotates queries and keys of rows_per_cta token rows per CTA and writes keys
// and values into their pages. A byte mover: every input element is read once
// and every output written once, 16 bytes at a time, so HBM bounds it. A step
// is 8 pairs (16 + 16 bytes) of one rotated head, or 8 copied elements. The
// (cos, sin) of a row are computed once for all of its heads and kept in shared
// memory; a thread's first steps are requested before them, so that the loads
// run under that arithmetic. Angles: position * turns in 64-bit fixed point
// drops whole turns exactly, and the top 32 bits of what is left are the
// angle to 2^-32 turns at any position. Five CTAs per SM: the registers that
// the compiler takes without that bound leave four (74.8 us in place of 73.6 for
// 16,384 rows, 19.8 in place of 16.3 for 4,999).
// kWhole: every dim of a head is rotated. Inputs then go around L1 (16,384 rows:
// 69.5 us in place of 72.5); beside copied dims that costs more than it gives (4,999
// half rotated rows: 13.9 us in place of 12.7). The loop over copied dims, which
// then has no turns, stays: without it the compiler spills (75.4 us).
template <bool kWhole>
__global__ void __launch_bounds__(kAppendThreads, 5) kv_append_rope_kernel(const __grid_constant__ AppendArgs a)
{
    // (cos, sin) of a row's pairs, two to a 16-byte entry: [row][entry of a step][step], so
    // that the steps of neighbouring threads read neighbouring entries. (In the order
    // of the pairs, four-way bank conflicts: 80 us in place of 73.6 for 16,384 rows.)
    __shared__ float4 s_cs[kAppendMaxRows * (kMaxRotaryDim / 4)];
    __shared__ __half* s_dst[kAppendMaxRows];  // key of the row's token in its page; null: row skipped
    __shared__ std::uint32_t s_value[kAppendMaxRows];  // elements from there to its value
    pdl_launch_dependents();
    pdl_wait();
    std::uint32_t const row0 = blockIdx.x * a.rows_per_cta;
    std::uint32_t const left = a.rows - row0;
    std::uint32_t const n_rows = left < a.rows_per_cta ? left : a.rows_per_cta;
    std::uint32_t const tid = threadIdx.x;
    std::uint32_t const half = a.rotary_half;
    std::uint32_t const chunks = half / 8u;                   // steps per rotated head
    std::uint32_t const row_steps = (a.q_heads + a.kv_heads) * chunks;
    std::uint32_t const steps = n_rows * row_steps;
    std::uint32_t const row_copies = a.pools.row / 8u;
    std::uint32_t const copies = n_rows * row_copies;

    struct Step {
        std::uint32_t row;   // within the CTA
        std::uint32_t head;  // queries first, then keys
        std::uint32_t pair;  // first of its 8 pairs
    };
    auto locate = [&](std::uint32_t i) {
        std::uint32_t const row = i / row_steps;
        std::uint32_t const rest = i - row * row_steps;
        std::uint32_t const head = rest / chunks;
        return Step{row, head, (rest - head * chunks) * 8u};
    };
    auto source = [&](Step const& s) {
        std::uint64_t const row = row0 + s.row;
        return (s.head < a.q_heads ? a.query + row * a.query_stride + s.head * a.head_dim
                                   : a.key + row * a.key_stride + (s.head - a.q_heads) * a.head_dim) + s.pair;
    };
    auto value_source = [&](std::uint32_t i) {
        std::uint32_t const row = i / row_copies;
        return a.value + (row0 + row) * a.value_stride + (i - row * row_copies) * 8u;
    };

    auto load = [](__half const* src) {
        uint4 const* const p = reinterpret_cast<uint4 const*>(src);
        return kWhole ? __ldcg(p) : *p;
    };
    Step cur{};
    uint4 lo{}, hi{}, val{};
    if (tid < steps) {
        cur = locate(tid);
        __half const* src = source(cur);
        lo = load(src);
        hi = load(src + half);
    }
    if (tid < copies) {
        val = load(value_source(tid));
    }

    if (tid < n_rows) {
        kk_kv_slot const slot = a.slots[row0 + tid];
        __half* dst = nullptr;
        std::uint32_t const cap = slot.kind == 0 ? a.pools.micro_cap : 64u;
        if (slot.active) {
            if (slot.page_token >= cap || slot.kind > 1u) {
                report(a.pools, kErrBadDescriptor);
            } else if (a.cos_sin != nullptr && a.positions[row0 + tid] >= a.table_positions) {
                report(a.pools, kErrBadArgument);
            } else {
                dst = block_of(a.pools, slot.kind, slot.slot, a.layer, 0);
                if (dst != nullptr) {
                    dst += std::uint64_t(slot.page_token) * a.pools.row;
                }
            }
        }
        s_dst[tid] = dst;
        s_value[tid] = cap * a.pools.row;
    }
    for (std::uint32_t i = tid; i < n_rows * half; i += kAppendThreads) {
        std::uint32_t const row = i / half;
        std::uint32_t const d = i - row * half;
        std::uint32_t const position = a.positions[row0 + row];
        float2 cs;
        if (a.cos_sin != nullptr) {
            cs = position < a.table_positions ? a.cos_sin[std::uint64_t(position) * half + d] : make_float2(1.f, 0.f);
        } else {
            std::uint64_t const turn = position * a.turns[d];  // modulo one turn
            // Half turns in [-1, 1).
            sincospif(static_cast<float>(static_cast<std::int32_t>(turn >> 32)) * 0x1p-31f, &cs.y, &cs.x);
        }
        reinterpret_cast<float2*>(s_cs)[((row * 4u + d % 8u / 2u) * chunks + d / 8u) * 2u + d % 2u] = cs;
    }
    __syncthreads();

    for (std::uint32_t i = tid; i < steps;) {
        std::uint32_t const next = i + kAppendThreads;
        Step const s = cur;
        uint4 const xa = lo, xb = hi;
        if (next < steps) {
            cur = locate(next);
            __half const* src = source(cur);
            lo = load(src);
            hi = load(src + half);
        }
        i = next;
        __half* dst = s_dst[s.row];
        if (dst == nullptr) {
            continue;
        }
        __half2 const* pa = reinterpret_cast<__half2 const*>(&xa);
        __half2 const* pb = reinterpret_cast<__half2 const*>(&xb);
        float4 const* cs = &s_cs[s.row * 4u * chunks + s.pair / 8u];
        uint4 ya, yb;
        __half2* qa = reinterpret_cast<__half2*>(&ya);
        __half2* qb = reinterpret_cast<__half2*>(&yb);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float2 const fa = __half22float2(pa[e]);
            float2 const fb = __half22float2(pb[e]);
            float4 const c = cs[e * chunks];  // (cos, sin) of two pairs
            qa[e] = __floats2half2_rn(fa.x * c.x - fb.x * c.y, fa.y * c.z - fb.y * c.w);
            qb[e] = __floats2half2_rn(fb.x * c.x + fa.x * c.y, fb.y * c.z + fa.y * c.w);
        }
        dst = s.head < a.q_heads
            ? a.query_out + (row0 + s.row) * a.query_out_stride + s.head * a.head_dim + s.pair
            : dst + (s.head - a.q_heads) * a.head_dim + s.pair;
        *reinterpret_cast<uint4*>(dst) = ya;
        *reinterpret_cast<uint4*>(dst + half) = yb;
    }
    for (std::uint32_t i = tid; i < copies;) {
        std::uint32_t const row = i / row_copies;
        std::uint32_t const e = (i - row * row_copies) * 8u;
        uint4 const x = val;
        i += kAppendThreads;
        if (i < copies) {
            val = load(value_source(i));
        }
        __half* dst = s_dst[row];
        if (dst != nullptr) {
            *reinterpret_cast<uint4*>(dst + s_value[row] + e) = x;
        }
    }
    // Dims behind the rotated ones.
    std::uint32_t const tail = a.head_dim - 2u * half;
    std::uint32_t const head_copies = tail / 8u;
    std::uint32_t const row_tails = (a.q_heads + a.kv_heads) * head_copies;
    std::uint32_t const tails = n_rows * row_tails;
    for (std::uint32_t i0 = tid; i0 < tails; i0 += kAppendThreads * kTailBatch) {
        uint4 x[kTailBatch];
        __half* to[kTailBatch];
#pragma unroll
        for (std::uint32_t k = 0; k < kTailBatch; ++k) {
            std::uint32_t const i = i0 + k * kAppendThreads;
            to[k] = nullptr;
            if (i < tails) {
                std::uint32_t const row = i / row_tails;
                std::uint32_t const rest = i - row * row_tails;
                std::uint32_t const head = rest / head_copies;
                std::uint32_t const e = 2u * half + (rest - head * head_copies) * 8u;
                __half* const dst = s_dst[row];
                if (dst != nullptr) {
                    to[k] = head < a.q_heads ? a.query_out + (row0 + row) * a.query_out_stride + head * a.head_dim + e
                                             : dst + (head - a.q_heads) * a.head_dim + e;
                    x[k] = *reinterpret_cast<uint4 const*>(source(Step{row, head, e}));
                }
            }
        }
#pragma unroll
        for (std::uint32_t k = 0; k < kTailBatch; ++k) {
            if (to[k] != nullptr) {
                *reinterpret_cast<uint4*>(to[k]) = x[k];
            }
        }
    }
}

struct PromoteSlots {
    std::uint32_t micro[8];
};

// grid (8 source pages, layers, 2): 8 tokens x row elements per block.
__global__ void kv_promote_kernel(PoolView v, PromoteSlots src, std::uint32_t extent_slot)
{
    pdl_wait();
    std::uint32_t const k = blockIdx.x;
    std::uint32_t const layer = blockIdx.y;
    std::uint32_t const component = blockIdx.z;
    __half const* from = block_of(v, 0, src.micro[k], layer, component);
    __half* to = block_of(v, 1, extent_slot, layer, component);
    if (from == nullptr || to == nullptr) {
        return;
    }
    to += std::uint64_t(8u * k) * v.row;
    std::uint64_t const n = 8ull * v.row;
    for (std::uint64_t i = threadIdx.x * 8u; i < n; i += blockDim.x * 8u) {
        *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<uint4 const*>(from + i);
    }
}

// K6 gather / scatter between pages and a contiguous KV tensor
// [layer][K|V][token][head][dim] (the reference's gatherKernel and
// appendTokensKernel, src/cuda/kv/page_kernels.cu:77-127, :184-242, which
// search the descriptor list per element). Here one CTA moves one page's
// (layer, K|V) block: valid_tokens contiguous rows, 16-byte accesses.
// Scatter copies only the tokens of [first, first + count) into the pages.
// grid (descriptors, layers * 2).
__global__ void kv_gather_kernel(PoolView v, kk_page_desc const* descs, std::uint32_t total_tokens,
    __half* out, __half const* in, std::uint32_t first, std::uint32_t count)
{
    pdl_wait();
    kk_page_desc const d = descs[blockIdx.x];
    std::uint32_t const layer = blockIdx.y / 2u;
    std::uint32_t const component = blockIdx.y % 2u;
    bool const micro = d.kind == 0;
    std::uint32_t const cap = micro ? v.micro_cap : 64u;
    std::uint32_t const begin = d.logical_token_begin;
    std::uint32_t const end = begin + d.valid_tokens;
    __half* page = block_of(v, micro ? 0 : 1, d.slot, layer, component);
    bool const bad = page == nullptr || d.valid_tokens > cap || d.kind > 1
        || (in == nullptr ? end > total_tokens : false);
    if (bad) {
        if (threadIdx.x == 0) {
            report(v, kErrBadDescriptor);
        }
        return;
    }
    std::uint64_t const row = v.row;
    if (in == nullptr) {
        __half* dst = out + ((std::uint64_t(layer) * 2u + component) * total_tokens + begin) * row;
        std::uint64_t const n = std::uint64_t(d.valid_tokens) * row;
        for (std::uint64_t i = threadIdx.x * 8u; i < n; i += blockDim.x * 8u) {
            *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<uint4 const*>(page + i);
        }
        return;
    }
    std::uint32_t const lo = begin > first ? begin : first;
    std::uint32_t const hi = end < first + count ? end : first + count;
    if (lo >= hi) {
        return;
    }
    __half const* src = in + ((std::uint64_t(layer) * 2u + component) * count + (lo - first)) * row;
    __half* dst = page + std::uint64_t(lo - begin) * row;
    std::uint64_t const n = std::uint64_t(hi - lo) * row;
    for (std::uint64_t i = threadIdx.x * 8u; i < n; i += blockDim.x * 8u) {
        *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<uint4 const*>(src + i);
    }
}

// SplitMix64 finaliser: a well-mixed 64-bit hash of (seed, index).
__device__ __forceinline__ std::uint64_t mix64(std::uint64_t x)
{
    x += 0x9e3779b97f4a7c15ull;
    x = (x ^ (x >> 30)) * 0xbf58476d1ce4e5b9ull;
    x = (x ^ (x >> 27)) * 0x94d049bb133111ebull;
    return x ^ (x >> 31);
}

__global__ void fill_fp16_kernel(__half* data, std::uint64_t count, std::uint64_t seed, float scale)
{
    pdl_wait();
    for (std::uint64_t i = blockIdx.x * std::uint64_t(blockDim.x) + threadIdx.x; i < count;
         i += std::uint64_t(gridDim.x) * blockDim.x) {
        std::uint64_t const h = mix64(seed * 0x100000001b3ull + i);
        float const u = static_cast<float>(h >> 40) * (1.0f / 16777216.0f);  // [0, 1)
        data[i] = __float2half_rn((2.0f * u - 1.0f) * scale);
    }
}

bool poolsOk(kk_kv_pools const* p)
{
    return p != nullptr && p->layers != 0 && p->kv_heads != 0 && p->head_dim != 0
        && (p->kv_heads * p->head_dim) % 8 == 0 && microPageTokensValid(*p);
}

} // namespace
} // namespace kk

extern "C" {

int kk_kv_write(const kk_kv_pools* pools, uint32_t layer_begin, uint32_t layer_count,
    const kk_kv_slot* slots, uint32_t num_lanes, const uint16_t* key, const uint16_t* value,
    uint64_t lane_stride, uint64_t layer_stride, void* stream)
{
    return kk::kvWrite(pools, layer_begin, layer_count, slots, num_lanes, key, value, lane_stride,
        layer_stride, nullptr, static_cast<cudaStream_t>(stream));
}

int kk_kv_copy_tokens(const kk_kv_pools* pools, uint32_t layer_begin, uint32_t layer_count,
    const kk_kv_copy* copies, uint32_t num_copies, void* stream)
{
    return kk::kvCopy(pools, layer_begin, layer_count, copies, num_copies, nullptr,
        static_cast<cudaStream_t>(stream));
}

int kk_kv_append_rope(const kk_kv_append_desc* d, void* stream)
{
    using namespace kk;
    auto misaligned = [](void const* p, std::uint64_t stride, std::uint64_t row) {
        return p == nullptr || (reinterpret_cast<std::uintptr_t>(p) & 15u) != 0 || stride % 8 != 0 || stride < row;
    };
    if (d == nullptr || !poolsOk(&d->pools) || d->layer >= d->pools.layers || d->pools.head_dim % 8 != 0
        || (reinterpret_cast<std::uintptr_t>(d->pools.micro) & 15u) != 0
        || (reinterpret_cast<std::uintptr_t>(d->pools.extent) & 15u) != 0
        || d->rotary_dim % 16 != 0 || d->rotary_dim > d->pools.head_dim || d->rotary_dim > kMaxRotaryDim) {
        return KK_EINVAL;
    }
    // Heads and dims that cannot be counted in 32-bit steps are no model's.
    std::uint64_t const q_row = std::uint64_t(d->q_heads) * d->pools.head_dim;
    std::uint64_t const kv_row = std::uint64_t(d->pools.kv_heads) * d->pools.head_dim;
    if (q_row > (1u << 24) || kv_row > (1u << 24)) {
        return KK_EINVAL;
    }
    if (d->rows == 0) {
        return 0;
    }
    auto odd = [](void const* p) { return (reinterpret_cast<std::uintptr_t>(p) & 3u) != 0; };
    if (d->slots == nullptr || odd(d->slots) || misaligned(d->key, d->key_stride, kv_row)
        || misaligned(d->value, d->value_stride, kv_row)
        || (d->q_heads != 0
            && (misaligned(d->query, d->query_stride, q_row) || misaligned(d->query_out, d->query_out_stride, q_row)
                || (d->query == d->query_out && d->query_stride != d->query_out_stride)))) {
        return KK_EINVAL;
    }
    AppendArgs a{};
    if (d->rotary_dim != 0) {
        if (d->positions == nullptr || odd(d->positions) || (reinterpret_cast<std::uintptr_t>(d->cos_sin) & 7u) != 0
            || (d->cos_sin != nullptr && d->table_positions == 0)
            || (d->cos_sin == nullptr && !(d->theta >= 1.f && std::isfinite(d->theta)))) {
            return KK_EINVAL;
        }
        a.cos_sin = reinterpret_cast<float2 const*>(d->cos_sin);
        a.table_positions = d->table_positions;
        if (a.cos_sin == nullptr) {
            // theta^(-2i / rotary_dim) by repeated products of one power, with 64
            // bits of mantissa: after i of them, and with the power's own rounding, off by
            // less than 2i + 1 roundings of 2^-64 of a value below 2^-2.6. For 128 powers
            // that is 2^-58.6 turns per position and, with the cut to 2^-64, 2^-26.5 at the
            // farthest, 7e-8 rad. (With 53 bits it was 2.5e-5 rad for a theta near 1.)
            static_assert(std::numeric_limits<long double>::digits >= 64, "");
            long double const ratio = powl(d->theta, -2.0L / d->rotary_dim);
            long double turns = 0.159154943091895335768883763372514362L;  // 1 / (2 pi)
            for (std::uint32_t i = 0; i < d->rotary_dim / 2; ++i, turns *= ratio) {
                a.turns[i] = static_cast<std::uint64_t>(turns * 0x1p64L);
            }
        }
    }
    a.pools = view(d->pools);
    a.layer = d->layer;
    a.rows = d->rows;
    // One wave of CTAs where their tables hold the rows, each row's chain of loads
    // as short as that allows (a decode batch of 64 rows: 2.9 us, 3.7 with four rows
    // per CTA; 4,999 rows of 16 + 2 heads of 128, half rotated: 12.8 us, 14.6 with
    // four). More rows: many waves, of four rows per CTA (16,384 rows of 32 + 8
    // heads of 128: 72.5 us, 74.4 with five, 76.8 with seven, before loads went around L1).
    // On the two sides of the step, 5,920 and 5,921 rows: 29.3 and 27.9 us for 32 + 8
    // heads of 128, 16.1 and 17.4 for 32 + 4 of 64, 15.0 and 16.9 for 16 + 2 of 128 half rotated.
    a.rows_per_cta = d->rows <= kAppendWave * kAppendMaxRows ? (d->rows - 1u) / kAppendWave + 1u : 4u;
    a.q_heads = d->q_heads;
    a.kv_heads = d->pools.kv_heads;
    a.head_dim = d->pools.head_dim;
    a.rotary_half = d->rotary_dim / 2;
    a.slots = d->slots;
    a.positions = d->positions;
    a.query = reinterpret_cast<__half const*>(d->query);
    a.key = reinterpret_cast<__half const*>(d->key);
    a.value = reinterpret_cast<__half const*>(d->value);
    a.query_out = reinterpret_cast<__half*>(d->query_out);
    a.query_stride = d->query_stride;
    a.key_stride = d->key_stride;
    a.value_stride = d->value_stride;
    a.query_out_stride = d->query_out_stride;
    unsigned const grid = (d->rows - 1u) / a.rows_per_cta + 1u;
    return static_cast<int>(launch(
        d->rotary_dim == d->pools.head_dim ? kv_append_rope_kernel<true> : kv_append_rope_kernel<false>, dim3(grid), dim3(kAppendThreads), 0,
        static_cast<cudaStream_t>(stream), 1, a));
}

int kk_kv_promote(const kk_kv_pools* pools, const uint32_t* micro_slots, uint32_t extent_slot,
    void* stream)
{
    using namespace kk;
    if (!poolsOk(pools) || micro_slots == nullptr || pools->extent == nullptr
        || extent_slot >= pools->extent_capacity || microPageTokens(*pools) != 8u) {
        return KK_EINVAL;
    }
    PromoteSlots src{};
    for (int k = 0; k < 8; ++k) {
        if (micro_slots[k] >= pools->micro_capacity) {
            return KK_EINVAL;
        }
        src.micro[k] = micro_slots[k];
    }
    return static_cast<int>(launch(kv_promote_kernel, dim3(8, pools->layers, 2), dim3(128), 0,
        static_cast<cudaStream_t>(stream), 1, view(*pools), src, extent_slot));
}

int kk_kv_gather(const kk_kv_pools* pools, const kk_page_desc* descs, uint32_t num_descs,
    uint32_t total_tokens, uint16_t* out, void* stream)
{
    using namespace kk;
    if (!poolsOk(pools) || (num_descs != 0 && (descs == nullptr || out == nullptr))
        || (reinterpret_cast<std::uintptr_t>(out) & 15u) != 0) {
        return KK_EINVAL;
    }
    if (num_descs == 0) {
        return 0;
    }
    return static_cast<int>(launch(kv_gather_kernel, dim3(num_descs, pools->layers * 2u), dim3(256), 0,
        static_cast<cudaStream_t>(stream), 1, view(*pools), descs, total_tokens,
        reinterpret_cast<__half*>(out), static_cast<__half const*>(nullptr), 0u, 0u));
}

int kk_kv_scatter(const kk_kv_pools* pools, const kk_page_desc* descs, uint32_t num_descs,
    uint32_t first_token, uint32_t token_count, const uint16_t* in, void* stream)
{
    using namespace kk;
    if (!poolsOk(pools) || (num_descs != 0 && (descs == nullptr || in == nullptr))
        || (reinterpret_cast<std::uintptr_t>(in) & 15u) != 0) {
        return KK_EINVAL;
    }
    if (num_descs == 0 || token_count == 0) {
        return 0;
    }
    return static_cast<int>(launch(kv_gather_kernel, dim3(num_descs, pools->layers * 2u), dim3(256), 0,
        static_cast<cudaStream_t>(stream), 1, view(*pools), descs, 0u, static_cast<__half*>(nullptr),
        reinterpret_cast<__half const*>(in), first_token, token_count));
}

int kk_fill_fp16(uint16_t* data, uint64_t count, uint64_t seed, float scale, void* stream)
{
    using namespace kk;
    if (data == nullptr) {
        return KK_EINVAL;
    }
    if (count == 0) {
        return 0;
    }
    std::uint64_t blocks = (count + 255) / 256;
    blocks = blocks > 8192 ? 8192 : blocks;
    return static_cast<int>(launch(fill_fp16_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256),
        0, static_cast<cudaStream_t>(stream), 1, reinterpret_cast<__half*>(data), count, seed, scale));
}

} // extern "C"

namespace kk {
int pagesStatus(cudaStream_t stream) { return readStatus(&g_pages_status, stream); }

int kvCopyDevCount(kk_kv_pools const* pools, std::uint32_t layer_begin, std::uint32_t layer_count,
    kk_kv_copy const* copies, std::uint32_t const* num_copies, std::uint32_t max_copies,
    unsigned int* status, cudaStream_t stream)
{
    if (!poolsOk(pools) || layer_count == 0 || layer_begin + layer_count > pools->layers
        || copies == nullptr || num_copies == nullptr || max_copies == 0 || max_copies > 65535u) {
        return KK_EINVAL;
    }
    PoolView v = view(*pools);
    v.status = status;
    return static_cast<int>(launch(kv_copy_kernel, dim3(max_copies, layer_count, 2), dim3(128), 0,
        stream, 1, v, layer_begin, copies, num_copies));
}

int kvWrite(kk_kv_pools const* pools, std::uint32_t layer_begin, std::uint32_t layer_count,
    kk_kv_slot const* slots, std::uint32_t num_lanes, std::uint16_t const* key,
    std::uint16_t const* value, std::uint64_t lane_stride, std::uint64_t layer_stride,
    unsigned int* status, cudaStream_t stream)
{
    if (!poolsOk(pools) || layer_count == 0 || layer_begin + layer_count > pools->layers
        || slots == nullptr || key == nullptr || value == nullptr || lane_stride % 8 != 0
        || layer_stride % 8 != 0 || num_lanes > 65535u) {
        return KK_EINVAL;
    }
    if (num_lanes == 0) {
        return 0;
    }
    PoolView v = view(*pools);
    v.status = status;
    return static_cast<int>(launch(kv_write_kernel, dim3(num_lanes, layer_count, 2), dim3(64), 0,
        stream, 1, v, layer_begin, slots, reinterpret_cast<__half const*>(key),
        reinterpret_cast<__half const*>(value), lane_stride, layer_stride));
}

int kvCopy(kk_kv_pools const* pools, std::uint32_t layer_begin, std::uint32_t layer_count,
    kk_kv_copy const* copies, std::uint32_t num_copies, unsigned int* status, cudaStream_t stream)
{
    if (!poolsOk(pools) || layer_count == 0 || layer_begin + layer_count > pools->layers
        || copies == nullptr || num_copies > 65535u) {
        return KK_EINVAL;
    }
    if (num_copies == 0) {
        return 0;
    }
    PoolView v = view(*pools);
    v.status = status;
    return static_cast<int>(launch(kv_copy_kernel, dim3(num_copies, layer_count, 2), dim3(128), 0,
        stream, 1, v, layer_begin, copies, static_cast<std::uint32_t const*>(nullptr)));
}
} // namespace kk
