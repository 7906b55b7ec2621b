// K7 — penalties, biases and grammar masks on FP32 logits, and the greedy
// token, in one pass over the logits.
//
// One thread-block cluster takes one row; its CTAs own the vocabulary in turn,
// 256 tokens at a time (text names low ids far more often than high ones:
// with one contiguous slice per CTA the first one had half of the history). A CTA
//  1. counts, in shared memory, what of the row's history is its own (every CTA
//     reads the whole history) and lists each token at its first occurrence;
//  2. replaces the counts of the listed tokens by their penalised logits;
//  3. adds the biases to those, or to the plain logits;
//  4. streams its logits, 16 bytes a thread at a time (rows that start on odd
//     addresses included), takes the replaced ones from shared memory, applies
//     the mask and keeps the highest; the cluster's winners meet in its first
//     CTA.
// Few tokens of a vocabulary are ever penalised, but few warps of the stream
// meet none, so step 4 computes nothing for them. Counts are integers and a
// replaced logit has one writer, so the order of threads changes nothing.
//
// HBM bounds it: 4 bytes read and 4 written per logit. The CTA's logits are
// asked into L2 at the start, so that DRAM works while the history is counted.
// Measured on 256 rows of 128,000 logits with about 10,000 tokens of history
// each (262 MB, 40 us at the measured copy rate): @@LARGE@@; 132 us
// with the penalties inside the stream (82 instructions a logit); 150 us with
// contiguous slices and a second pass over the history in place of the list;
// 200 us with each history read once and counted through distributed shared
// memory.
#include "../../../include/kk_kernels.h"
#include "kernels_internal.h"
#include "launch.cuh"

#include <atomic>

namespace kk {

__device__ unsigned int g_logits_status;

namespace {

constexpr std::uint32_t kThreads = 384;
constexpr std::uint32_t kMaxCluster = 8;
constexpr std::uint32_t kBlock = 256;          // consecutive tokens of one CTA
constexpr std::uint32_t kVecs = 2;             // 16-byte loads in flight per thread
constexpr std::uint32_t kQuads = 4;            // 16-byte history loads in flight per thread
constexpr std::uint32_t kPrompt = 0x80000000u; // the prompt names the token; below: occurrences in the output
constexpr std::uint32_t kListed = 2048;        // tokens listed at most; with more, step 2 looks at every word
constexpr std::uint32_t kMaxSharedBytes = 222u * 1024u;

struct LogitsArgs {
    kk_logits_desc d;
    std::uint32_t cluster_log2;  // CTAs per row
    // Places in shared memory, in 32-bit words; a place of a token is its
    // number among the CTA's own (the first `capacity`), or capacity + token
    // for the up to three tokens before the row's first 16-byte step.
    std::uint32_t capacity;
    std::uint32_t touched_at;    // a bit per place, set: the word is the token's new logit
    std::uint32_t mask_at;       // a bit per place, set: allowed
    std::uint32_t list_at;       // 16-bit places
};

__device__ __forceinline__ void report(unsigned int code) { atomicCAS(&g_logits_status, kErrNone, code); }

__device__ __forceinline__ void cluster_arrive()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}

__device__ __forceinline__ void cluster_wait()
{
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void st_cluster_u64(std::uint32_t addr, std::uint64_t v)
{
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// A logit and its token as one key: a higher logit wins, then a lower id; 0 is
// below every candidate. NaN and -inf give 0.
__device__ __forceinline__ std::uint64_t candidate(float x, std::uint32_t id)
{
    if (!(x > -INFINITY)) {
        return 0;
    }
    std::uint32_t const u = __float_as_uint(x + 0.f);  // -0 and +0 are equal
    std::uint32_t const order = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return (std::uint64_t(order) << 32) | (0xffffffffu - id);
}

__global__ void __launch_bounds__(kThreads, 3) logits_process_kernel(const __grid_constant__ LogitsArgs a)
{
    extern __shared__ __align__(16) std::uint32_t s_words[];
    __shared__ std::uint64_t s_best[kThreads / 32];
    __shared__ std::uint64_t s_cluster[kMaxCluster];
    __shared__ std::uint32_t s_listed;
    pdl_launch_dependents();
    pdl_wait();
    kk_logits_desc const& d = a.d;
    std::uint32_t const tid = threadIdx.x;
    std::uint32_t const lc = a.cluster_log2;
    std::uint32_t const rank = blockIdx.x & ((1u << lc) - 1u);
    std::uint32_t const row = blockIdx.x >> lc;
    std::uint32_t const vocab = d.vocab;
    float const* const in = d.logits + row * d.logits_stride;
    float* const out = d.out != nullptr ? d.out + row * d.out_stride : nullptr;
    bool const same_phase = out == nullptr
        || ((reinterpret_cast<std::uintptr_t>(out) ^ reinterpret_cast<std::uintptr_t>(in)) & 15u) == 0;
    // Tokens before the first 16-byte step; the first CTA's.
    std::uint32_t head = (4u - static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>(in) >> 2)) & 3u;
    head = head < vocab ? head : vocab;
    std::uint32_t const body = vocab - head;
    std::uint32_t const all_blocks = (body + kBlock - 1u) / kBlock;
    std::uint32_t const blocks = all_blocks > rank ? ((all_blocks - 1u - rank) >> lc) + 1u : 0u;
    // Place <-> token, behind the head.
    auto token_of = [&](std::uint32_t at) {
        return head + ((((at / kBlock) << lc) + rank) * kBlock) + at % kBlock;
    };
    std::uint32_t const owner_mask = ((1u << lc) - 1u) * kBlock;
    std::uint32_t const owner = rank * kBlock;
    auto owned = [&](std::uint32_t v) { return v - head < body && ((v - head) & owner_mask) == owner; };
    auto place_of = [&](std::uint32_t v) {
        std::uint32_t const u = v - head;
        return ((u / kBlock) >> lc) * kBlock + u % kBlock;
    };
    auto in_head = [&](std::uint32_t v) { return v < head && rank == 0; };

    // ---- everything that can be asked for at once: logits, the row's lists
    for (std::uint32_t i = tid; i < blocks; i += kThreads) {
        std::uint32_t const v = token_of(i * kBlock);
        std::uint32_t const n = (vocab - v < kBlock ? vocab - v : kBlock) / 4u;
        if (n != 0) {
            l2_prefetch_bulk(in + v, n * 16u);
        }
    }
    std::uint32_t* const s_touched = s_words + a.touched_at;
    if (a.touched_at != 0) {  // the call has a history or biases
        if (d.history_offsets != nullptr) {
            for (std::uint32_t i = tid; i <= a.capacity / 4u; i += kThreads) {
                reinterpret_cast<uint4*>(s_words)[i] = make_uint4(0, 0, 0, 0);
            }
        }
        for (std::uint32_t i = tid; i <= a.capacity / 32u; i += kThreads) {
            s_touched[i] = 0;
        }
        if (tid == 0) {
            s_listed = 0;
        }
    }
    float rep = 1.f, pres = 0.f, freq = 0.f;
    std::uint32_t h0 = 0, h1 = 0, prompt = 0, b0 = 0, b1 = 0, mask_row = row;
    if (d.history_offsets != nullptr) {
        h0 = d.history_offsets[row];
        h1 = d.history_offsets[row + 1];
        rep = d.repetition != nullptr ? d.repetition[row] : 1.f;
        pres = d.presence != nullptr ? d.presence[row] : 0.f;
        freq = d.frequency != nullptr ? d.frequency[row] : 0.f;
        prompt = d.prompt_counts != nullptr ? d.prompt_counts[row] : 0u;
    }
    if (d.bias_offsets != nullptr) {
        b0 = d.bias_offsets[row];
        b1 = d.bias_offsets[row + 1];
    }
    if (d.mask != nullptr && d.mask_rows != nullptr) {
        mask_row = d.mask_rows[row];
    }
    bool bad = false;
    if (h1 < h0 || h1 > d.history_size) {
        bad = true;
        h0 = h1 = 0;
    }
    if (rep == 1.f && pres == 0.f && freq == 0.f) {
        h0 = h1 = 0;  // the history changes nothing
    }
    if (b1 < b0 || b1 > d.bias_size) {
        bad = true;
        b0 = b1 = 0;
    }
    std::uint32_t const* mask = nullptr;
    bool blocked = false;  // a mask row outside the masks: nothing is allowed
    if (d.mask != nullptr) {
        if (mask_row < d.num_masks) {
            mask = d.mask + std::uint64_t(mask_row) * d.mask_stride;
        } else if (mask_row != KK_NO_MASK || d.mask_rows == nullptr) {
            bad = blocked = true;
        }
    }
    if (bad && tid == 0) {
        report(kErrBadArgument);
    }
    bool const penal = h1 > h0;
    bool const use_words = penal || b1 > b0;
    // The first bias of each thread, and the logit that it changes.
    std::uint32_t bias_token = 0, bias_next = 0xffffffffu;
    float bias_value = 0.f, bias_logit = 0.f;
    auto load_bias = [&](std::uint32_t i) {
        bias_token = d.bias_tokens[i];
        bias_next = i + 1 < b1 ? d.bias_tokens[i + 1] : 0xffffffffu;
        bias_value = d.bias_values[i];
        bias_logit = owned(bias_token) || in_head(bias_token) ? in[bias_token] : 0.f;
    };
    if (b0 + tid < b1) {
        load_bias(b0 + tid);
    }
    // Before a CTA writes into another one's shared memory, all of the cluster
    // have started: they say so here and ask at the end.
    if (lc != 0 && d.tokens != nullptr) {
        cluster_arrive();
    }

    std::uint32_t* const s_mask = s_words + a.mask_at;
    std::uint16_t* const s_list = reinterpret_cast<std::uint16_t*>(s_words + a.list_at);
    if (mask != nullptr) {
        // Brought to the places' order; bits behind the vocabulary are never asked for.
        std::uint32_t const last = (vocab - 1u) / 32u;
        for (std::uint32_t i = tid; i < blocks * (kBlock / 32u); i += kThreads) {
            std::uint32_t const v = token_of(i * 32u);
            std::uint32_t const w = v / 32u < last ? v / 32u : last;
            s_mask[i] = __funnelshift_r(__ldg(mask + w), __ldg(mask + (w < last ? w + 1u : last)), v & 31u);
        }
    }
    __syncthreads();

    // ---- the history and the biases
    auto replace = [&](std::uint32_t at, float x) {
        s_words[at] = __float_as_uint(x);
        atomicOr(&s_touched[at / 32u], 1u << (at % 32u));
    };
    if (penal) {
        auto count = [&](std::uint32_t at, std::uint32_t i) {
            std::uint32_t const before = i < prompt ? atomicOr(&s_words[at], kPrompt) : atomicAdd(&s_words[at], 1u);
            if (before == 0) {
                std::uint32_t const n = atomicAdd(&s_listed, 1u);
                if (n < kListed) {
                    s_list[n] = static_cast<std::uint16_t>(at);
                }
            }
        };
        std::uint32_t const* const text = d.history + h0;
        std::uint32_t const len = h1 - h0;
        std::uint32_t const lead = (4u - static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>(text) >> 2)) & 3u;
        std::uint32_t const from = lead < len ? lead : len;
        std::uint32_t const quads = (len - from) / 4u;
        for (std::uint32_t q0 = tid; q0 < quads; q0 += kThreads * kQuads) {
            uint4 ahead[kQuads];
#pragma unroll
            for (std::uint32_t k = 0; k < kQuads; ++k) {
                std::uint32_t const q = q0 + k * kThreads;
                if (q < quads) {
                    ahead[k] = __ldg(reinterpret_cast<uint4 const*>(text + from) + q);
                }
            }
#pragma unroll
            for (std::uint32_t k = 0; k < kQuads; ++k) {
                std::uint32_t const q = q0 + k * kThreads;
                if (q >= quads) {
                    break;
                }
                uint4 const t = ahead[k];
                std::uint32_t mine = (owned(t.x) ? 1u : 0u) | (owned(t.y) ? 2u : 0u) | (owned(t.z) ? 4u : 0u)
                    | (owned(t.w) ? 8u : 0u);
                if (head != 0) {
                    std::uint32_t const v[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
                    for (std::uint32_t e = 0; e < 4u; ++e) {
                        if (in_head(v[e])) {
                            count(a.capacity + v[e], from + q * 4u + e);
                        }
                    }
                }
                // One token per thread and turn: about two turns a warp, not four.
                while (mine != 0) {
                    std::uint32_t const e = __ffs(mine) - 1u;
                    mine &= mine - 1u;
                    std::uint32_t const v = e < 2u ? (e == 0 ? t.x : t.y) : (e == 2u ? t.z : t.w);
                    count(place_of(v), from + q * 4u + e);
                }
            }
        }
        std::uint32_t const edge = tid < from ? tid : from + quads * 4u + (tid - from);
        if (edge < len && tid < from + 3u) {
            std::uint32_t const v = text[edge];
            if (owned(v)) {
                count(place_of(v), edge);
            } else if (in_head(v)) {
                count(a.capacity + v, edge);
            }
        }
        __syncthreads();
        auto logit_at = [&](std::uint32_t at) { return in[at < a.capacity ? token_of(at) : at - a.capacity]; };
        auto penalise = [&](std::uint32_t at, float x) {
            std::uint32_t const n = s_words[at] & ~kPrompt;
            x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
            if (n != 0) {
                x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(n)));
                x = __fsub_rn(x, pres);
            }
            replace(at, x);
        };
        std::uint32_t const listed = s_listed;
        if (listed <= kListed) {
            for (std::uint32_t i0 = tid; i0 < listed; i0 += kThreads * kQuads) {
                std::uint32_t at[kQuads];
                float x[kQuads];
#pragma unroll
                for (std::uint32_t k = 0; k < kQuads; ++k) {
                    std::uint32_t const i = i0 + k * kThreads;
                    at[k] = i < listed ? s_list[i] : 0u;
                    x[k] = i < listed ? logit_at(at[k]) : 0.f;
                }
#pragma unroll
                for (std::uint32_t k = 0; k < kQuads; ++k) {
                    if (i0 + k * kThreads < listed) {
                        penalise(at[k], x[k]);
                    }
                }
            }
        } else {
            for (std::uint32_t i = tid; i < blocks * kBlock + head; i += kThreads) {
                std::uint32_t const at = i < blocks * kBlock ? i : a.capacity + (i - blocks * kBlock);
                if (s_words[at] != 0) {
                    penalise(at, logit_at(at));
                }
            }
        }
        __syncthreads();
    }
    for (std::uint32_t i = b0 + tid; i < b1; i += kThreads) {
        if (i != b0 + tid) {
            load_bias(i);
        }
        std::uint32_t const v = bias_token;
        if (bias_next < v) {
            report(kErrBadArgument);
        }
        bool const low = in_head(v);
        if ((low || owned(v)) && bias_next != v) {
            std::uint32_t const at = low ? a.capacity + v : place_of(v);
            bool const replaced = (s_touched[at / 32u] >> (at % 32u) & 1u) != 0;
            replace(at, __fadd_rn(replaced ? __uint_as_float(s_words[at]) : bias_logit, bias_value));
        }
    }
    if (b1 > b0) {
        __syncthreads();
    }

    // ---- the logits
    // A thread meets its tokens in ascending order, so a strict comparison
    // keeps the lowest id of equal logits; NaN and -inf never pass it.
    float top = -INFINITY;
    std::uint32_t top_id = 0;
    auto offer = [&](float x, std::uint32_t v) {
        if (x > top) {
            top = x;
            top_id = v;
        }
    };
    auto bits_of = [&](std::uint32_t const* bits, std::uint32_t at) { return bits[at / 32u] >> (at % 32u); };
    auto one = [&](std::uint32_t at, std::uint32_t v, bool allowed) {
        float x = use_words && (bits_of(s_touched, at) & 1u) != 0 ? __uint_as_float(s_words[at]) : in[v];
        x = allowed && !blocked ? x : -INFINITY;
        if (out != nullptr) {
            out[v] = x;
        }
        offer(x, v);
    };
    if (rank == 0 && tid < head) {
        one(a.capacity + tid, tid, mask == nullptr || (mask[0] >> tid & 1u) != 0);
    }
    std::uint32_t const steps = blocks * (kBlock / 4u);
    for (std::uint32_t i0 = tid; i0 < steps; i0 += kThreads * kVecs) {
        float4 x[kVecs];
#pragma unroll
        for (std::uint32_t k = 0; k < kVecs; ++k) {
            std::uint32_t const i = i0 + k * kThreads;
            std::uint32_t const v = token_of(i * 4u);
            if (i < steps && v + 4u <= vocab) {
                x[k] = *reinterpret_cast<float4 const*>(in + v);
            }
        }
#pragma unroll
        for (std::uint32_t k = 0; k < kVecs; ++k) {
            std::uint32_t const i = i0 + k * kThreads;
            std::uint32_t const at = i * 4u;
            std::uint32_t const v = token_of(at);
            if (i >= steps || v >= vocab) {
                continue;
            }
            std::uint32_t allow = blocked ? 0u : 15u;
            if (mask != nullptr) {
                allow = bits_of(s_mask, at);
            }
            if (v + 4u > vocab) {  // the last, partial step
                for (std::uint32_t e = 0; v + e < vocab; ++e) {
                    one(at + e, v + e, (allow >> e & 1u) != 0);
                }
                continue;
            }
            if (use_words) {
                std::uint32_t const replaced = bits_of(s_touched, at) & 15u;
                if (replaced != 0) {
                    uint4 const w = *reinterpret_cast<uint4 const*>(&s_words[at]);
                    x[k].x = (replaced & 1u) != 0 ? __uint_as_float(w.x) : x[k].x;
                    x[k].y = (replaced & 2u) != 0 ? __uint_as_float(w.y) : x[k].y;
                    x[k].z = (replaced & 4u) != 0 ? __uint_as_float(w.z) : x[k].z;
                    x[k].w = (replaced & 8u) != 0 ? __uint_as_float(w.w) : x[k].w;
                }
            }
            x[k].x = (allow & 1u) != 0 ? x[k].x : -INFINITY;
            x[k].y = (allow & 2u) != 0 ? x[k].y : -INFINITY;
            x[k].z = (allow & 4u) != 0 ? x[k].z : -INFINITY;
            x[k].w = (allow & 8u) != 0 ? x[k].w : -INFINITY;
            if (d.tokens != nullptr) {
                offer(x[k].x, v);
                offer(x[k].y, v + 1u);
                offer(x[k].z, v + 2u);
                offer(x[k].w, v + 3u);
            }
            if (out != nullptr) {
                if (same_phase) {
                    *reinterpret_cast<float4*>(out + v) = x[k];
                } else {
                    out[v] = x[k].x;
                    out[v + 1u] = x[k].y;
                    out[v + 2u] = x[k].z;
                    out[v + 3u] = x[k].w;
                }
            }
        }
    }

    // ---- the greedy token
    if (d.tokens == nullptr) {
        return;
    }
    std::uint64_t best = candidate(top, top_id);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        std::uint64_t const other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if (tid % 32u == 0) {
        s_best[tid / 32u] = best;
    }
    __syncthreads();
    if (tid == 0) {
        for (std::uint32_t w = 1; w < kThreads / 32u; ++w) {
            best = s_best[w] > best ? s_best[w] : best;
        }
    }
    if (lc != 0) {
        cluster_wait();
        if (tid == 0 && rank != 0) {
            st_cluster_u64(cluster_map(&s_cluster[rank], 0), best);
        }
        // Only the first CTA waits; the others are done once they said so.
        __syncwarp();
        cluster_arrive();
        if (rank != 0) {
            return;
        }
        cluster_wait();
    }
    if (tid == 0) {
        for (std::uint32_t r = 1; r < 1u << lc; ++r) {
            best = s_cluster[r] > best ? s_cluster[r] : best;
        }
        d.tokens[row] = best != 0 ? 0xffffffffu - static_cast<std::uint32_t>(best) : KK_NO_TOKEN;
    }
}

// The kernel's shared-memory limit is raised once per device.
cudaError_t allowSharedMemory()
{
    static std::atomic<std::uint64_t> done{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && (done.load(std::memory_order_acquire) >> device & 1u) != 0)) {
        return e;
    }
    e = cudaFuncSetAttribute(logits_process_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
        static_cast<int>(kMaxSharedBytes));
    if (e == cudaSuccess && device < 64) {
        done.fetch_or(std::uint64_t(1) << device, std::memory_order_release);
    }
    return e;
}

} // namespace

int logitsStatus(cudaStream_t stream) { return readStatus(&g_logits_status, stream); }

} // namespace kk

extern "C" int kk_logits_process(const kk_logits_desc* d, void* stream)
{
    using namespace kk;
    auto odd = [](void const* p) { return (reinterpret_cast<std::uintptr_t>(p) & 3u) != 0; };
    if (d == nullptr || d->vocab == 0 || d->vocab > (1u << 30)) {
        return KK_EINVAL;
    }
    if (d->rows == 0) {
        return 0;
    }
    if (d->logits == nullptr || (d->out == nullptr && d->tokens == nullptr) || d->logits_stride < d->vocab
        || (d->out != nullptr && d->out_stride < d->vocab)
        || (d->out == d->logits && d->out_stride != d->logits_stride) || odd(d->logits) || odd(d->out)
        || odd(d->tokens)) {
        return KK_EINVAL;
    }
    LogitsArgs a{};
    a.d = *d;
    bool const penalties = d->repetition != nullptr || d->presence != nullptr || d->frequency != nullptr;
    if (!penalties) {
        a.d.history_offsets = nullptr;
    } else if (d->history_offsets == nullptr || (d->history == nullptr && d->history_size != 0)) {
        return KK_EINVAL;
    }
    if (d->bias_offsets != nullptr && d->bias_size != 0 && (d->bias_tokens == nullptr || d->bias_values == nullptr)) {
        return KK_EINVAL;
    }
    if (d->mask != nullptr && d->mask_stride < (d->vocab + 31u) / 32u) {
        return KK_EINVAL;
    }
    bool const words = a.d.history_offsets != nullptr || d->bias_offsets != nullptr;
    // CTAs per row: up to eight, none with fewer than 4,096 tokens.
    while ((1u << a.cluster_log2) < kMaxCluster && (d->vocab >> a.cluster_log2) > 4096u) {
        ++a.cluster_log2;
    }
    std::uint32_t const blocks = (d->vocab + kBlock - 1u) / kBlock;
    a.capacity = (((blocks - 1u) >> a.cluster_log2) + 1u) * kBlock;
    std::uint64_t bytes = 0;
    if (words) {
        a.touched_at = a.capacity + 4u;
        a.list_at = a.touched_at + a.capacity / 32u + 1u;
        bytes = (std::uint64_t(a.list_at) + kListed / 2u) * 4u;
    }
    if (d->mask != nullptr) {
        a.mask_at = static_cast<std::uint32_t>(bytes / 4u);
        bytes += a.capacity / 8u;
    }
    if (bytes > kMaxSharedBytes || (words && a.capacity + 4u > 65536u)
        || (std::uint64_t(d->rows) << a.cluster_log2) > 0x7fffffffu) {
        return KK_EINVAL;
    }
    cudaError_t const e = allowSharedMemory();
    if (e != cudaSuccess) {
        return static_cast<int>(e);
    }
    return static_cast<int>(launch(logits_process_kernel, dim3(d->rows << a.cluster_log2), dim3(kThreads), bytes,
        static_cast<cudaStream_t>(stream), 1u << a.cluster_log2, a));
}
