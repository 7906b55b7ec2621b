// K7 — penalties, biases and grammar masks on FP32 logits, and the greedy
// token, in one pass over the logits.
//
// One thread-block cluster takes one row; its CTAs own the vocabulary in turn,
// 256 tokens at a time (text names low ids far more often than high ones:
// with one contiguous slice per CTA the first one had half of the history). A CTA
//  1. counts, in shared memory, what of the row's history is its own (every CTA
//     reads the whole history) and marks the tokens, a bit each;
//  2. lists the marked tokens and replaces their counts by their penalised logits;
//  3. adds the biases to those, or to the plain logits;
//  4. streams its logits, 256 tokens a warp at a time (rows that start on odd
//     addresses included), takes the marked ones from shared memory, applies
//     the mask and keeps the highest; the cluster's winners meet in its first
//     CTA.
// Few tokens of a vocabulary are ever penalised, but few warps of the stream
// meet none, so step 4 computes nothing for them. Counts are integers and a
// replaced logit has one writer, so the order of threads changes nothing.
//
// HBM bounds it: 4 bytes read and 4 written per logit. The CTA's logits are
// asked into L2 at the start, so that DRAM works while the history is counted.
// Measured on 256 rows of 128,000 logits with about 10,000 tokens of history
// each (262 MB, 40 us at the measured copy rate): 130 us; 132 us
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

constexpr std::uint32_t kThreads = 256;
constexpr std::uint32_t kWarps = kThreads / 32;
constexpr std::uint32_t kMaxCluster = 8;
constexpr std::uint32_t kBlock = 256;          // consecutive tokens of one CTA
constexpr std::uint32_t kQuads = 2;            // 16-byte history loads in flight per thread
constexpr std::uint32_t kListed = 2048;        // marked tokens listed at most; others are taken bit by bit
constexpr std::uint32_t kGather = 2;           // listed tokens per thread at a time
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

// A read-only load issued where it stands in the program.
__device__ __forceinline__ std::uint32_t ldg_u32_now(void const* p)
{
    std::uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
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

__global__ void __launch_bounds__(kThreads, 4) logits_process_kernel(const __grid_constant__ LogitsArgs a)
{
    extern __shared__ __align__(16) std::uint32_t s_words[];
    __shared__ std::uint64_t s_best[kWarps];
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

    // ---- everything that can be asked for at once
    float rep = 1.f, pres = 0.f, freq = 0.f;
    std::uint32_t h0 = 0, h1 = 0, prompt = 0, b0 = 0, b1 = 0, mask_row = row;
    if (d.history_offsets != nullptr) {
        h0 = ldg_u32_now(d.history_offsets + row);
        h1 = ldg_u32_now(d.history_offsets + row + 1);
        rep = d.repetition != nullptr ? __uint_as_float(ldg_u32_now(d.repetition + row)) : 1.f;
        pres = d.presence != nullptr ? __uint_as_float(ldg_u32_now(d.presence + row)) : 0.f;
        freq = d.frequency != nullptr ? __uint_as_float(ldg_u32_now(d.frequency + row)) : 0.f;
        prompt = d.prompt_counts != nullptr ? ldg_u32_now(d.prompt_counts + row) : 0u;
    }
    if (d.bias_offsets != nullptr) {
        b0 = ldg_u32_now(d.bias_offsets + row);
        b1 = ldg_u32_now(d.bias_offsets + row + 1);
    }
    if (d.mask != nullptr && d.mask_rows != nullptr) {
        mask_row = ldg_u32_now(d.mask_rows + row);
    }
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
    // The thread's first 16-byte pieces of the history.
    std::uint32_t const* const text = d.history + h0;
    std::uint32_t const len = h1 - h0;
    std::uint32_t const lead = (4u - static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>(text) >> 2)) & 3u;
    std::uint32_t const from = lead < len ? lead : len;
    std::uint32_t const quads = (len - from) / 4u;
    uint4 ahead[kQuads];
    auto load_quads = [&](std::uint32_t q0) {
#pragma unroll
        for (std::uint32_t k = 0; k < kQuads; ++k) {
            std::uint32_t const q = q0 + k * kThreads;
            ahead[k] = make_uint4(0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu);  // no token
            if (q < quads) {
                ahead[k] = ldg_u4_now(text + from + q * 4u);
            }
        }
    };
    load_quads(tid);
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
    if (penal) {
        auto count = [&](std::uint32_t at, std::uint32_t i) {
            atomicOr(&s_touched[at / 32u], 1u << (at % 32u));
            if (i >= prompt) {
                atomicAdd(&s_words[at], 1u);
            }
        };
        for (std::uint32_t q0 = tid; q0 < quads; q0 += kThreads * kQuads) {
            uint4 now[kQuads];
#pragma unroll
            for (std::uint32_t k = 0; k < kQuads; ++k) {
                now[k] = ahead[k];
            }
            load_quads(q0 + kThreads * kQuads);
#pragma unroll
            for (std::uint32_t k = 0; k < kQuads; ++k) {
                std::uint32_t const i = from + (q0 + k * kThreads) * 4u;
                uint4 const t = now[k];
                std::uint32_t const v[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
                for (std::uint32_t e = 0; e < 4u; ++e) {
                    if (owned(v[e])) {
                        count(place_of(v[e]), i + e);
                    }
                }
                if (head != 0) {
#pragma unroll
                    for (std::uint32_t e = 0; e < 4u; ++e) {
                        if (in_head(v[e])) {
                            count(a.capacity + v[e], i + e);
                        }
                    }
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
            std::uint32_t const n = s_words[at];
            x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
            if (n != 0) {
                x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(n)));
                x = __fsub_rn(x, pres);
            }
            s_words[at] = __float_as_uint(x);
        };
        // Marked tokens lie in clumps: they are spread over the threads by a list.
        std::uint32_t const words = blocks * (kBlock / 32u);
        for (std::uint32_t i0 = 0; i0 <= words; i0 += kThreads) {
            std::uint32_t const i = i0 + tid;
            std::uint32_t const w = i < words ? i : a.capacity / 32u;  // the head's word stands behind all blocks
            std::uint32_t bits = i <= words ? s_touched[w] : 0u;
            std::uint32_t const own = __popc(bits);
            std::uint32_t upto = own;
#pragma unroll
            for (std::uint32_t o = 1; o < 32u; o *= 2u) {
                std::uint32_t const x = __shfl_up_sync(0xffffffffu, upto, o);
                upto += tid % 32u >= o ? x : 0u;
            }
            std::uint32_t base = 0;
            if (tid % 32u == 31u && upto != 0) {
                base = atomicAdd(&s_listed, upto);
            }
            std::uint32_t n = __shfl_sync(0xffffffffu, base, 31) + upto - own;
            auto list = [&](std::uint32_t at, std::uint32_t place) {
                if (place < kListed) {
                    s_list[place] = static_cast<std::uint16_t>(at);
                } else {
                    penalise(at, logit_at(at));
                }
            };
            // A word with many marks is taken by the whole warp, a lane a bit.
            for (std::uint32_t full = __ballot_sync(0xffffffffu, own > 4u); full != 0; full &= full - 1u) {
                std::uint32_t const from_lane = __ffs(full) - 1u;
                std::uint32_t const word = __shfl_sync(0xffffffffu, bits, from_lane);
                std::uint32_t const first = __shfl_sync(0xffffffffu, n, from_lane);
                std::uint32_t const at = __shfl_sync(0xffffffffu, w, from_lane) * 32u + tid % 32u;
                if ((word >> (tid % 32u) & 1u) != 0) {
                    list(at, first + __popc(word & ((1u << (tid % 32u)) - 1u)));
                }
            }
            // Straight-line, as above: loops of divergent length cost three times as much.
#pragma unroll
            for (std::uint32_t e = 0; e < 4u; ++e) {
                if (own <= 4u && bits != 0) {
                    list(w * 32u + __ffs(bits) - 1u, n++);
                    bits &= bits - 1u;
                }
            }
        }
        __syncthreads();
        std::uint32_t const listed = s_listed < kListed ? s_listed : kListed;
        for (std::uint32_t i0 = tid; i0 < listed; i0 += kThreads * kGather) {
            std::uint32_t at[kGather];
            float x[kGather];
#pragma unroll
            for (std::uint32_t k = 0; k < kGather; ++k) {
                std::uint32_t const i = i0 + k * kThreads;
                at[k] = i < listed ? s_list[i] : 0u;
                x[k] = i < listed ? logit_at(at[k]) : 0.f;
            }
#pragma unroll
            for (std::uint32_t k = 0; k < kGather; ++k) {
                if (i0 + k * kThreads < listed) {
                    penalise(at[k], x[k]);
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
            s_words[at] = __float_as_uint(
                __fadd_rn(replaced ? __uint_as_float(s_words[at]) : bias_logit, bias_value));
            atomicOr(&s_touched[at / 32u], 1u << (at % 32u));
        }
    }
    if (b1 > b0) {
        __syncthreads();
    }

    // ---- the logits
    // The highest logit so far and where: a thread meets its steps of four tokens in
    // ascending order, so a strict comparison keeps the lowest of equal ones; NaN
    // and -inf never pass it.
    float top = -INFINITY;
    std::uint32_t top_id = 0;
    auto bits_of = [&](std::uint32_t const* bits, std::uint32_t at) { return bits[at / 32u] >> (at % 32u); };
    bool const masked = mask != nullptr || blocked;
    std::uint64_t best = 0;  // of the tokens outside whole blocks
    auto one = [&](std::uint32_t at, std::uint32_t v) {
        bool const low = at >= a.capacity;
        bool const allowed = !blocked
            && (mask == nullptr || ((low ? mask[0] >> v : bits_of(s_mask, at)) & 1u) != 0);
        float x = use_words && (bits_of(s_touched, at) & 1u) != 0 ? __uint_as_float(s_words[at]) : in[v];
        x = allowed ? x : -INFINITY;
        std::uint64_t const c = candidate(x, v);
        best = c > best ? c : best;
        if (out != nullptr) {
            out[v] = x;
        }
    };
    if (rank == 0 && tid < head) {
        one(a.capacity + tid, tid);
    }
    // A warp takes a block of 256 tokens: two steps of four for every thread. The
    // places of consecutive blocks of a warp lie kWarps blocks apart, their
    // tokens that times the cluster's size.
    std::uint32_t const lane4 = (tid % 32u) * 4u;
    std::uint32_t const whole_blocks = blocks != 0 && token_of((blocks - 1u) * kBlock) + kBlock > vocab ? blocks - 1u : blocks;
    {
        std::uint32_t at = tid / 32u * kBlock + lane4;
        std::uint32_t v = head + ((tid / 32u << lc) + rank) * kBlock + lane4;
        std::uint32_t const stride = (kWarps * kBlock) << lc;
        bool const vector_out = out != nullptr && same_phase;
        for (std::uint32_t block = tid / 32u; block < whole_blocks; block += kWarps, at += kWarps * kBlock, v += stride) {
            float4 x[2] = {*reinterpret_cast<float4 const*>(in + v), *reinterpret_cast<float4 const*>(in + v + 128u)};
            if (use_words) {
#pragma unroll
                for (std::uint32_t k = 0; k < 2u; ++k) {
                    std::uint32_t const marked = bits_of(s_touched, at + k * 128u) & 15u;
                    if (marked != 0) {
                        uint4 const w = *reinterpret_cast<uint4 const*>(&s_words[at + k * 128u]);
                        x[k].x = (marked & 1u) != 0 ? __uint_as_float(w.x) : x[k].x;
                        x[k].y = (marked & 2u) != 0 ? __uint_as_float(w.y) : x[k].y;
                        x[k].z = (marked & 4u) != 0 ? __uint_as_float(w.z) : x[k].z;
                        x[k].w = (marked & 8u) != 0 ? __uint_as_float(w.w) : x[k].w;
                    }
                }
            }
            if (masked) {
#pragma unroll
                for (std::uint32_t k = 0; k < 2u; ++k) {
                    std::uint32_t const allow = blocked ? 0u : bits_of(s_mask, at + k * 128u);
                    x[k].x = (allow & 1u) != 0 ? x[k].x : -INFINITY;
                    x[k].y = (allow & 2u) != 0 ? x[k].y : -INFINITY;
                    x[k].z = (allow & 4u) != 0 ? x[k].z : -INFINITY;
                    x[k].w = (allow & 8u) != 0 ? x[k].w : -INFINITY;
                }
            }
#pragma unroll
            for (std::uint32_t k = 0; k < 2u; ++k) {
                float const high = fmaxf(fmaxf(fmaxf(x[k].x, x[k].y), x[k].z), x[k].w);  // passes NaN over
                if (high > top) {
                    top = high;
                    top_id = v + k * 128u + (x[k].x == high ? 0u : x[k].y == high ? 1u : x[k].z == high ? 2u : 3u);
                }
            }
            if (vector_out) {
                *reinterpret_cast<float4*>(out + v) = x[0];
                *reinterpret_cast<float4*>(out + v + 128u) = x[1];
            } else if (out != nullptr) {
#pragma unroll
                for (std::uint32_t k = 0; k < 2u; ++k) {
                    out[v + k * 128u] = x[k].x;
                    out[v + k * 128u + 1u] = x[k].y;
                    out[v + k * 128u + 2u] = x[k].z;
                    out[v + k * 128u + 3u] = x[k].w;
                }
            }
        }
    }
    if (whole_blocks < blocks) {  // the vocabulary's last, partial block
        std::uint32_t const at0 = whole_blocks * kBlock;
        for (std::uint32_t e = tid; token_of(at0) + e < vocab; e += kThreads) {
            one(at0 + e, token_of(at0) + e);
        }
    }

    // ---- the greedy token
    if (d.tokens == nullptr) {
        return;
    }
    std::uint64_t const whole = candidate(top, top_id);
    best = whole > best ? whole : best;
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
        for (std::uint32_t w = 1; w < kWarps; ++w) {
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
    for (void const* array : {static_cast<void const*>(d->history), static_cast<void const*>(d->history_offsets),
             static_cast<void const*>(d->prompt_counts), static_cast<void const*>(d->repetition),
             static_cast<void const*>(d->presence), static_cast<void const*>(d->frequency),
             static_cast<void const*>(d->bias_tokens), static_cast<void const*>(d->bias_values),
             static_cast<void const*>(d->bias_offsets), static_cast<void const*>(d->mask),
             static_cast<void const*>(d->mask_rows)}) {
        if (odd(array)) {
            return KK_EINVAL;
        }
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
