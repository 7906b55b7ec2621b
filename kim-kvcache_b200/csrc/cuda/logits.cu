// K7 — penalties, biases and grammar masks on FP32 logits, and the greedy
// token, in one pass over the logits.
//
// One thread-block cluster takes one row; its CTAs own the vocabulary in turn,
// 256 tokens at a time (text names low ids far more often than high ones:
// with one contiguous slice per CTA the first one had half of the history). A CTA
//  1. counts, in shared memory, what of the row's history is its own (every CTA
//     reads the whole history) and marks the tokens, a bit each;
//  2. lists the marked tokens, works out their penalised logits and replaces their
//     counts by their places in the list;
//  3. adds the biases to those, or lists the plain logits with their biases;
//  4. streams its logits, 256 tokens a warp at a time, takes the marked ones from
//     the list, applies the mask and keeps the highest; the cluster's winners meet
//     in its first CTA.
// Few tokens of a vocabulary are ever penalised, but few warps of the stream
// meet none, so step 4 computes nothing for them. Counts are integers and a logit
// has one owner, so the order of threads changes nothing. Counts have 16 bits,
// which lets four CTAs share an SM: what bounds the kernel is the chain of steps
// of a CTA. A row with more than 65,535 tokens of history is taken in two halves
// of the CTA's places, with 32 bits each; more marked tokens than the list holds
// are taken 2,048 places at a time.
//
// HBM is the floor: 4 bytes read and 4 written per logit. The CTA's logits are
// asked into L2 at the start, so that DRAM works while the history is counted.
// Measured on 256 rows of 128,000 logits with about 10,000 tokens of history
// each (262 MB, 40 us at the measured copy rate): 106 us. 130 us with a 32-bit
// word per place (three CTAs per SM); 132 us with the marked tokens of a warp's
// block spread over its lanes there, in place of steps 2 and 3 (twice the
// instructions); 150 us with contiguous slices and a second pass over the
// history; 157 us with clusters of 16; 200 us with each history read once and
// counted through distributed shared memory.
#include "../../../include/kk_kernels.h"
#include "kernels_internal.h"
#include "launch.cuh"

#include <atomic>
#include <type_traits>

namespace kk {

__device__ unsigned int g_logits_status;

namespace {

constexpr std::uint32_t kThreads = 256;
constexpr std::uint32_t kWarps = kThreads / 32;
constexpr std::uint32_t kMaxCluster = 8;
constexpr std::uint32_t kBlock = 256;          // consecutive tokens of one CTA
constexpr std::uint32_t kQuads = 2;            // 16-byte history loads in flight per thread
constexpr std::uint32_t kMaxCounted = 65535;   // history of a row that 16-bit counts hold
constexpr std::uint32_t kMaxWordsVocab = 400000;  // with a history or biases
constexpr std::uint32_t kMaxVocab = 10000000;     // with a mask
constexpr std::uint32_t kMaxSharedBytes = 222u * 1024u;
constexpr std::uint32_t kListed = 2048;        // listed tokens
constexpr std::uint32_t kGather = 2;           // of them per thread at a time
constexpr std::uint32_t kFewBlocks = kListed / kBlock;  // whose tokens the list holds in any case

struct LogitsArgs {
    kk_logits_desc d;
    std::uint32_t cluster_log2;  // CTAs per row
    std::uint32_t capacity;      // places (a token's number among the CTA's own) of a CTA, whole blocks, an even number
    // In shared memory, in 32-bit words; counts, 16 bits a place, come first.
    std::uint32_t touched_at;    // a bit per place, set: in the history or biased
    std::uint32_t value_at;      // logits of listed tokens
    std::uint32_t list_at;       // and their places, 16 bits each
    std::uint32_t mask_at;       // a bit per place, set: allowed
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

// A store into another CTA's shared memory that its barrier counts: neither side has
// to order it behind the stores of the logits (a cluster barrier would).
__device__ __forceinline__ void st_cluster_u64(std::uint32_t addr, std::uint64_t v, std::uint32_t bar)
{
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u64 [%0], %1, [%2];"
                 ::"r"(addr), "l"(v), "r"(bar)
                 : "memory");
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
    __shared__ std::uint32_t s_listed;
    __shared__ std::uint64_t s_best[kWarps];
    __shared__ std::uint64_t s_cluster[kMaxCluster];
    __shared__ std::uint64_t s_winners;  // barrier: the other CTAs' winners are here
    pdl_launch_dependents();
    pdl_wait();
    kk_logits_desc const& d = a.d;
    std::uint32_t const tid = threadIdx.x;
    std::uint32_t const lane = tid % 32u;
    std::uint32_t const warp = tid / 32u;
    std::uint32_t const lc = a.cluster_log2;
    std::uint32_t const rank = blockIdx.x & ((1u << lc) - 1u);
    std::uint32_t const row = blockIdx.x >> lc;
    std::uint32_t const vocab = d.vocab;
    // Blocks start on a 16-byte boundary: token v stands at u = v + shift of them.
    float const* in = d.logits + row * d.logits_stride;
    std::uint32_t const shift = static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>(in) >> 2) & 3u;
    in -= shift;
    float* const out = d.out != nullptr ? d.out + row * d.out_stride - shift : nullptr;
    bool const vector_out = (reinterpret_cast<std::uintptr_t>(out) & 15u) == 0;
    std::uint32_t const end = vocab + shift;
    std::uint32_t const all_blocks = (end + kBlock - 1u) / kBlock;
    std::uint32_t const blocks = all_blocks > rank ? ((all_blocks - 1u - rank) >> lc) + 1u : 0u;
    auto first_of = [&](std::uint32_t block) { return ((block << lc) + rank) * kBlock; };  // a block's first u
    std::uint32_t const owner_mask = ((1u << lc) - 1u) * kBlock;
    std::uint32_t const owner = rank * kBlock;
    auto owned = [&](std::uint32_t v) { return ((v + shift) & owner_mask) == owner && v < vocab; };
    auto place_of = [&](std::uint32_t v) {
        std::uint32_t const u = v + shift;
        return ((u / kBlock) >> lc) * kBlock + u % kBlock;
    };

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
        std::uint32_t u = first_of(i);
        std::uint32_t const stop = (u + kBlock < end ? u + kBlock : end) & ~3u;
        u = u < shift ? 4u : u;  // whole steps only: nothing before or behind the row is touched
        if (u < stop) {
            l2_prefetch_bulk(in + u, (stop - u) * 4u);
        }
    }
    std::uint32_t* const s_touched = s_words + a.touched_at;
    float* const s_value = reinterpret_cast<float*>(s_words + a.value_at);
    std::uint16_t* const s_list = reinterpret_cast<std::uint16_t*>(s_words + a.list_at);
    auto clear_counts = [&]() {
        for (std::uint32_t i = tid; i < a.capacity / 8u; i += kThreads) {
            reinterpret_cast<uint4*>(s_words)[i] = make_uint4(0, 0, 0, 0);
        }
    };
    if (d.history_offsets != nullptr) {
        clear_counts();
    }
    if (a.value_at != 0) {  // the call has a history or biases
        for (std::uint32_t i = tid; i < a.capacity / 32u; i += kThreads) {
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
    bool const biased = b1 > b0;
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
        bias_next = i + 1u < b1 ? d.bias_tokens[i + 1u] : 0xffffffffu;
        bias_value = d.bias_values[i];
        bias_logit = owned(bias_token) ? in[bias_token + shift] : 0.f;
    };
    if (b0 + tid < b1) {
        load_bias(b0 + tid);
    }
    std::uint32_t* const s_mask = s_words + a.mask_at;
    if (mask != nullptr) {
        // Brought to the places' order; words behind the vocabulary are never asked for.
        std::uint32_t const words = (vocab + 31u) / 32u;
        for (std::uint32_t i = tid; i < blocks * (kBlock / 32u); i += kThreads) {
            std::uint32_t const w = first_of(i / (kBlock / 32u)) / 32u + i % (kBlock / 32u);
            std::uint32_t const low = shift != 0 && w - 1u < words ? __ldg(mask + w - 1u) : 0u;
            s_mask[i] = __funnelshift_l(low, w < words ? __ldg(mask + w) : 0u, shift);
        }
    }
    // Before a CTA writes into another one's shared memory, all of the cluster
    // have started: they say so here and ask at the end.
    if (lc != 0 && d.tokens != nullptr) {
        if (rank == 0 && tid == 0) {
            mbar_init(&s_winners, 1);
            fence_barrier_init();
            mbar_arrive_expect_tx(&s_winners, ((1u << lc) - 1u) * 8u);
        }
        __syncwarp();
        cluster_arrive();
    }
    __syncthreads();

    // The highest logit so far and where: a thread meets its steps of four tokens in
    // ascending order, so a strict comparison keeps the lowest of equal ones; NaN
    // and -inf never pass it.
    float top = -INFINITY;
    std::uint32_t top_id = 0;
    auto bits_of = [&](std::uint32_t const* bits, std::uint32_t at) { return bits[at / 32u] >> (at % 32u); };
    bool const masked = mask != nullptr || blocked;
    bool const wide = len > kMaxCounted;
    std::uint32_t const span = wide ? a.capacity / 2u : a.capacity;  // places counted at a time
    for (std::uint32_t place0 = 0; place0 == 0 || (wide && place0 < a.capacity); place0 += span) {
        // ---- the history
        if (penal) {
            if (place0 != 0) {
                __syncthreads();
                clear_counts();
                if (tid == 0) {
                    s_listed = 0;
                }
                load_quads(tid);
                __syncthreads();
            }
            auto scan = [&](auto narrow) {
                auto count = [&](std::uint32_t v, std::uint32_t i) {
                    if (owned(v)) {
                        std::uint32_t const at = place_of(v);
                        atomicOr(&s_touched[at / 32u], 1u << (at % 32u));
                        if (i >= prompt) {
                            if (narrow) {
                                atomicAdd(&s_words[at / 2u], 1u << (at % 2u * 16u));
                            } else if (at - place0 < span) {
                                atomicAdd(&s_words[at - place0], 1u);
                            }
                        }
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
                        count(now[k].x, i);
                        count(now[k].y, i + 1u);
                        count(now[k].z, i + 2u);
                        count(now[k].w, i + 3u);
                    }
                }
                std::uint32_t const edge = tid < from ? tid : from + quads * 4u + (tid - from);
                if (edge < len && tid < from + 3u) {
                    count(text[edge], edge);
                }
            };
            if (wide) {
                scan(std::false_type{});
            } else {
                scan(std::true_type{});
            }
        }
        __syncthreads();
        // A place's word: its count, then its place in the list.
        auto* const s_half = reinterpret_cast<std::uint16_t*>(s_words);
        auto word_of = [&](std::uint32_t at) -> std::uint32_t { return wide ? s_words[at - place0] : s_half[at]; };
        auto set_word = [&](std::uint32_t at, std::uint32_t w) {
            if (wide) {
                s_words[at - place0] = w;
            } else {
                s_half[at] = static_cast<std::uint16_t>(w);
            }
        };
        std::uint32_t const stop = place0 / kBlock + span / kBlock < blocks ? place0 / kBlock + span / kBlock : blocks;
        std::uint32_t run = stop;  // blocks at a time
        for (std::uint32_t block0 = place0 / kBlock; block0 < stop;) {
            std::uint32_t const block1 = stop - block0 < run ? stop : block0 + run;
            // ---- the marked tokens' logits
            if (penal) {
                // They lie in clumps: a list spreads them over the threads.
                std::uint32_t const word1 = block1 * (kBlock / 32u);
                for (std::uint32_t i0 = block0 * (kBlock / 32u); i0 < word1; i0 += kThreads) {
                    std::uint32_t const w = i0 + tid;
                    std::uint32_t bits = w < word1 ? s_touched[w] : 0u;
                    std::uint32_t const own = __popc(bits);
                    std::uint32_t upto = own;
#pragma unroll
                    for (std::uint32_t o = 1; o < 32u; o *= 2u) {
                        std::uint32_t const x = __shfl_up_sync(0xffffffffu, upto, o);
                        upto += lane >= o ? x : 0u;
                    }
                    std::uint32_t base = 0;
                    if (lane == 31u && upto != 0) {
                        base = atomicAdd(&s_listed, upto);
                    }
                    std::uint32_t n = __shfl_sync(0xffffffffu, base, 31) + upto - own;
                    auto list = [&](std::uint32_t at, std::uint32_t place) {
                        if (place < kListed) {
                            s_list[place] = static_cast<std::uint16_t>(at);
                        }
                    };
                    // A word with many marks is taken by the whole warp, a lane a bit.
                    for (std::uint32_t full = __ballot_sync(0xffffffffu, own > 4u); full != 0; full &= full - 1u) {
                        std::uint32_t const from_lane = __ffs(full) - 1u;
                        std::uint32_t const word = __shfl_sync(0xffffffffu, bits, from_lane);
                        std::uint32_t const first = __shfl_sync(0xffffffffu, n, from_lane);
                        std::uint32_t const at = __shfl_sync(0xffffffffu, w, from_lane) * 32u + lane;
                        if ((word >> lane & 1u) != 0) {
                            list(at, first + __popc(word & ((1u << lane) - 1u)));
                        }
                    }
                    // Straight-line: loops of divergent length cost three times as much.
#pragma unroll
                    for (std::uint32_t e = 0; e < 4u; ++e) {
                        if (own <= 4u && bits != 0) {
                            list(w * 32u + __ffs(bits) - 1u, n++);
                            bits &= bits - 1u;
                        }
                    }
                }
                __syncthreads();
            }
            std::uint32_t const listed = penal ? s_listed : 0u;
            if ((listed > kListed || b1 - b0 > kListed - listed) && run > kFewBlocks) {
                run = kFewBlocks;
                __syncthreads();
                if (tid == 0) {
                    s_listed = 0;
                }
                __syncthreads();
                continue;
            }
            if (penal) {
                for (std::uint32_t i0 = tid; i0 < listed; i0 += kThreads * kGather) {
                    std::uint32_t at[kGather];
                    float x[kGather];
#pragma unroll
                    for (std::uint32_t k = 0; k < kGather; ++k) {
                        std::uint32_t const i = i0 + k * kThreads;
                        at[k] = i < listed ? s_list[i] : 0u;
                        x[k] = i < listed ? in[first_of(at[k] / kBlock) + at[k] % kBlock] : 0.f;
                    }
#pragma unroll
                    for (std::uint32_t k = 0; k < kGather; ++k) {
                        std::uint32_t const i = i0 + k * kThreads;
                        if (i < listed) {
                            std::uint32_t const n = word_of(at[k]);
                            float y = x[k] > 0.f ? __fdiv_rn(x[k], rep) : __fmul_rn(x[k], rep);
                            if (n != 0) {
                                y = __fsub_rn(y, __fmul_rn(freq, static_cast<float>(n)));
                                y = __fsub_rn(y, pres);
                            }
                            s_value[i] = y;
                            set_word(at[k], i);
                        }
                    }
                }
                __syncthreads();
            }
            if (biased) {
                for (std::uint32_t i = b0 + tid; i < b1; i += kThreads) {
                    if (i != b0 + tid || block0 != 0) {
                        load_bias(i);
                    }
                    std::uint32_t const v = bias_token;
                    if (bias_next < v) {
                        report(kErrBadArgument);
                    }
                    if (owned(v) && bias_next != v) {
                        std::uint32_t const at = place_of(v);
                        if (at / kBlock - block0 < block1 - block0) {
                            std::uint32_t const volatile& marks = s_touched[at / 32u];
                            if ((marks >> (at % 32u) & 1u) != 0) {
                                __threadfence_block();  // where ids descend, see below
                                float& y = s_value[word_of(at)];
                                y = __fadd_rn(y, bias_value);
                            } else {
                                std::uint32_t const place = atomicAdd(&s_listed, 1u);
                                if (place < kListed) {  // as ever, unless ids descend
                                    s_value[place] = __fadd_rn(bias_logit, bias_value);
                                    set_word(at, place);
                                    // Where ids descend, another thread may have the same
                                    // token: it sees the mark only with the place.
                                    __threadfence_block();
                                    atomicOr(&s_touched[at / 32u], 1u << (at % 32u));
                                }
                            }
                        }
                    }
                }
                __syncthreads();
            }
            // ---- the logits
            // A warp takes a block of 256 tokens: two steps of four for every thread.
            auto stream = [&](std::uint32_t block, auto inner) {
                std::uint32_t const u0 = first_of(block) + lane * 4u;
                std::uint32_t const at = block * kBlock + lane * 4u;
                bool const whole[2] = {inner || (u0 >= shift && u0 + 4u <= end), inner || u0 + 132u <= end};
                float x[8];
#pragma unroll
                for (std::uint32_t k = 0; k < 2u; ++k) {
                    float const* const src = in + u0 + k * 128u;
                    if (whole[k]) {
                        float4 const v = *reinterpret_cast<float4 const*>(src);
                        x[4u * k] = v.x;
                        x[4u * k + 1u] = v.y;
                        x[4u * k + 2u] = v.z;
                        x[4u * k + 3u] = v.w;
                    } else {
#pragma unroll
                        for (std::uint32_t e = 0; e < 4u; ++e) {
                            std::uint32_t const u = u0 + k * 128u + e;
                            x[4u * k + e] = u >= shift && u < end ? src[e] : -INFINITY;
                        }
                    }
                }
                if (penal || biased) {
#pragma unroll
                    for (std::uint32_t k = 0; k < 2u; ++k) {
                        std::uint32_t const marked = bits_of(s_touched, at + k * 128u) & 15u;
                        if (marked != 0) {
                            std::uint32_t w[4];
                            if (wide) {
                                uint4 const v = *reinterpret_cast<uint4 const*>(&s_words[at + k * 128u - place0]);
                                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                            } else {
                                uint2 const v = *reinterpret_cast<uint2 const*>(&s_half[at + k * 128u]);
                                w[0] = v.x & 0xffffu, w[1] = v.x >> 16, w[2] = v.y & 0xffffu, w[3] = v.y >> 16;
                            }
#pragma unroll
                            for (std::uint32_t e = 0; e < 4u; ++e) {
                                if ((marked >> e & 1u) != 0) {
                                    x[4u * k + e] = s_value[w[e]];
                                }
                            }
                        }
                    }
                }
                if (masked) {
#pragma unroll
                    for (std::uint32_t k = 0; k < 2u; ++k) {
                        std::uint32_t const allow = blocked ? 0u : bits_of(s_mask, at + k * 128u);
#pragma unroll
                        for (std::uint32_t e = 0; e < 4u; ++e) {
                            x[4u * k + e] = (allow >> e & 1u) != 0 ? x[4u * k + e] : -INFINITY;
                        }
                    }
                }
                float high[2];  // of each step; fmaxf passes NaN over
#pragma unroll
                for (std::uint32_t k = 0; k < 2u; ++k) {
                    high[k] = fmaxf(fmaxf(x[4u * k], x[4u * k + 1u]), fmaxf(x[4u * k + 2u], x[4u * k + 3u]));
                }
                if (fmaxf(high[0], high[1]) > top) {
                    top = fmaxf(high[0], high[1]);
                    std::uint32_t e = 7;
#pragma unroll
                    for (std::uint32_t i = 7; i-- > 0;) {
                        e = x[i] == top ? i : e;
                    }
                    top_id = u0 + e % 4u + e / 4u * 128u;
                }
                if (out != nullptr) {
#pragma unroll
                    for (std::uint32_t k = 0; k < 2u; ++k) {
                        float const* const y = x + 4u * k;
                        std::uint32_t const u = u0 + k * 128u;
                        if (vector_out && whole[k]) {
                            *reinterpret_cast<float4*>(out + u) = make_float4(y[0], y[1], y[2], y[3]);
                        } else {
#pragma unroll
                            for (std::uint32_t e = 0; e < 4u; ++e) {
                                if (u + e >= shift && u + e < end) {
                                    out[u + e] = y[e];
                                }
                            }
                        }
                    }
                }
            };
            for (std::uint32_t block = block0 + warp; block < block1; block += kWarps) {
                std::uint32_t const u = first_of(block);
                if (u >= shift && u + kBlock <= end) {
                    stream(block, std::true_type{});
                } else {  // the row's first and last
                    stream(block, std::false_type{});
                }
            }
            block0 = block1;
            if (block0 < stop) {
                __syncthreads();
                if (tid == 0) {
                    s_listed = 0;
                }
                __syncthreads();
            }
        }
    }

    // ---- the greedy token
    if (d.tokens == nullptr) {
        return;
    }
    std::uint64_t best = candidate(top, top_id - shift);
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
        if (tid == 0) {
            if (rank != 0) {
                st_cluster_u64(cluster_map(&s_cluster[rank], 0), best, cluster_map(&s_winners, 0));
            } else {
                mbar_wait(&s_winners, 0, &g_logits_status);
            }
        }
        if (rank != 0) {
            return;
        }
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
    // A 32-bit index passes the end of its list by a step of the block.
    constexpr std::uint64_t kMaxEntries = (std::uint64_t(1) << 32) - kThreads;
    if ((a.d.history_offsets != nullptr && d->history_size > kMaxEntries)
        || (d->bias_offsets != nullptr && d->bias_size > kMaxEntries)) {
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
    // A row that does not start on a 16-byte boundary reaches up to 3 places further.
    std::uint32_t const blocks = (d->vocab + 3u + kBlock - 1u) / kBlock;
    a.capacity = ((((blocks - 1u) >> a.cluster_log2) + 2u) & ~1u) * kBlock;
    std::uint64_t bytes = 0;
    auto reserve = [&](std::uint64_t n) {
        std::uint64_t const at = bytes / 4u;
        bytes += n;
        return static_cast<std::uint32_t>(at);
    };
    if (words) {
        reserve(a.capacity * 2u);
        a.touched_at = reserve(a.capacity / 8u);
        a.value_at = reserve(kListed * 4u);
        a.list_at = reserve(kListed * 2u);
    }
    if (d->mask != nullptr) {
        a.mask_at = reserve(a.capacity / 8u);
    }
    if (bytes > kMaxSharedBytes || (words && d->vocab > kMaxWordsVocab) || (d->mask != nullptr && d->vocab > kMaxVocab)
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
