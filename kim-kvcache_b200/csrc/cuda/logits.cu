// K7 — penalties, biases and grammar masks on FP32 logits, and the greedy
// token, in one pass over the logits.
//
// One thread-block cluster takes one row; each of its CTAs owns a contiguous
// slice of the vocabulary with one 32-bit word per token in shared memory:
// how often the row's output named the token (low 30 bits), whether the
// history names it at all, and whether a bias does. The history is read once
// for the whole row: every CTA reads its share of it and adds each token to
// the owner's word through distributed shared memory. Counts are integers, so
// the order in which they arrive changes nothing. Then every CTA streams its
// slice of the logits, 16 bytes a thread at a time (rows that start on odd
// addresses included), and keeps the highest allowed one; the cluster's
// winners meet in its first CTA.
//
// HBM bounds it: 4 bytes read and 4 written per logit. The slice is asked into
// L2 at the start, so that DRAM works while the history is counted.
#include "../../../include/kk_kernels.h"
#include "kernels_internal.h"
#include "launch.cuh"

#include <atomic>

namespace kk {

__device__ unsigned int g_logits_status;

namespace {

constexpr int kThreads = 512;
constexpr std::uint32_t kMaxCluster = 8;
constexpr std::uint32_t kSeen = 0x80000000u;    // the token is in the history
constexpr std::uint32_t kBiased = 0x40000000u;  // the token has a bias
constexpr std::uint32_t kCount = 0x3fffffffu;   // its occurrences in the output
constexpr std::uint32_t kVecs = 4;              // 16-byte loads in flight per thread
constexpr std::uint32_t kMaxSliceBytes = 200u * 1024u;

struct LogitsArgs {
    kk_logits_desc d;
    std::uint32_t cluster;  // CTAs per row
    std::uint32_t slice;    // tokens per CTA, a multiple of 32
};

__device__ __forceinline__ void report(unsigned int code) { atomicCAS(&g_logits_status, kErrNone, code); }

__device__ __forceinline__ void red_add_cluster(std::uint32_t addr, std::uint32_t v)
{
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__device__ __forceinline__ void red_or_cluster(std::uint32_t addr, std::uint32_t v)
{
    asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

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

__global__ void __launch_bounds__(kThreads) logits_process_kernel(const __grid_constant__ LogitsArgs a)
{
    extern __shared__ __align__(16) std::uint32_t s_words[];
    __shared__ std::uint64_t s_best[kThreads / 32];
    __shared__ std::uint64_t s_cluster[kMaxCluster];
    pdl_launch_dependents();
    pdl_wait();
    kk_logits_desc const& d = a.d;
    std::uint32_t const tid = threadIdx.x;
    std::uint32_t const rank = a.cluster > 1 ? cluster_rank() : 0u;
    std::uint32_t const row = blockIdx.x / a.cluster;
    std::uint32_t const begin = rank * a.slice < d.vocab ? rank * a.slice : d.vocab;
    std::uint32_t const end = d.vocab - begin < a.slice ? d.vocab : begin + a.slice;
    float const* in = d.logits + row * d.logits_stride;
    float* out = d.out != nullptr ? d.out + row * d.out_stride : nullptr;
    // 16-byte steps of logits start at body (slices start on whole 128-byte
    // steps from the row's start, so the row's misfit is every slice's).
    std::uint32_t const misfit = static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>(in) >> 2) & 3u;
    bool const same_phase = out == nullptr
        || ((reinterpret_cast<std::uintptr_t>(out) ^ reinterpret_cast<std::uintptr_t>(in)) & 15u) == 0;
    std::uint32_t head = (4u - misfit) & 3u;
    head = head < end - begin ? head : end - begin;
    std::uint32_t const vecs = (end - begin - head) / 4u;
    std::uint32_t const body = begin + head;
    // Words are shifted so that a 16-byte step of logits meets a 16-byte step
    // of words; the shift is the row's, the same in every CTA of the cluster.
    std::uint32_t const shift = misfit;
    std::uint32_t* const words = s_words + shift;  // word of token v: words[v - begin]

    if (tid == 0 && vecs != 0) {
        l2_prefetch_bulk(in + body, vecs * 16u);
    }

    // ---- the row's lists
    float rep = 1.f, pres = 0.f, freq = 0.f;
    std::uint32_t h0 = 0, h1 = 0, prompt = 0;
    if (d.history_offsets != nullptr) {
        rep = d.repetition != nullptr ? d.repetition[row] : 1.f;
        pres = d.presence != nullptr ? d.presence[row] : 0.f;
        freq = d.frequency != nullptr ? d.frequency[row] : 0.f;
        if (rep != 1.f || pres != 0.f || freq != 0.f) {
            h0 = d.history_offsets[row];
            h1 = d.history_offsets[row + 1];
            if (h1 < h0 || h1 > d.history_size) {
                if (tid == 0) {
                    report(kErrBadArgument);
                }
                h0 = h1 = 0;
            }
            prompt = d.prompt_counts != nullptr ? d.prompt_counts[row] : 0u;
        }
    }
    std::uint32_t b0 = 0, b1 = 0;
    if (d.bias_offsets != nullptr) {
        b0 = d.bias_offsets[row];
        b1 = d.bias_offsets[row + 1];
        if (b1 < b0 || b1 > d.bias_size) {
            if (tid == 0) {
                report(kErrBadArgument);
            }
            b0 = b1 = 0;
        }
    }
    bool const penal = h1 > h0;
    bool const biased = b1 > b0;
    std::uint32_t const* mask = nullptr;
    bool blocked = false;  // a mask row outside the masks: nothing is allowed
    if (d.mask != nullptr) {
        std::uint32_t const m = d.mask_rows != nullptr ? d.mask_rows[row] : row;
        if (m < d.num_masks) {
            mask = d.mask + std::uint64_t(m) * d.mask_stride;
        } else if (m != KK_NO_MASK || d.mask_rows == nullptr) {
            blocked = true;
            if (tid == 0) {
                report(kErrBadArgument);
            }
        }
    }

    // Before a CTA writes into another one's shared memory, all of the cluster
    // have started: with a history the barriers around its count see to
    // that, without one this pair does (its wait stands at the end).
    bool const greet = a.cluster > 1 && !penal && d.tokens != nullptr;
    if (greet) {
        cluster_arrive();
    }

    // ---- words
    if (penal || biased) {
        std::uint32_t const n = (end - begin + shift + 3u) / 4u;
        for (std::uint32_t i = tid; i < n; i += kThreads) {
            reinterpret_cast<uint4*>(s_words)[i] = make_uint4(0, 0, 0, 0);
        }
        if (penal && a.cluster > 1) {
            cluster_sync();
        } else {
            __syncthreads();
        }
        for (std::uint32_t i = b0 + tid; i < b1; i += kThreads) {
            std::uint32_t const v = d.bias_tokens[i];
            if (v >= begin && v < end) {
                atomicOr(&words[v - begin], kBiased);
            }
            if (i + 1 < b1 && d.bias_tokens[i + 1] < v) {
                report(kErrBadArgument);
            }
        }
        if (penal) {
            std::uint64_t const len = h1 - h0;
            std::uint32_t const lo = static_cast<std::uint32_t>(len * rank / a.cluster);
            std::uint32_t const hi = static_cast<std::uint32_t>(len * (rank + 1u) / a.cluster);
            for (std::uint32_t i = lo + tid; i < hi; i += kThreads) {
                std::uint32_t const v = d.history[std::uint64_t(h0) + i];
                if (v >= d.vocab) {
                    continue;
                }
                std::uint32_t const owner = v / a.slice;
                std::uint32_t* const word = &words[v - owner * a.slice];
                std::uint32_t const addr = a.cluster > 1 ? cluster_map(word, owner) : smem_u32(word);
                if (i < prompt) {
                    red_or_cluster(addr, kSeen);
                } else {
                    red_add_cluster(addr, 1u);
                }
            }
        }
        if (penal && a.cluster > 1) {
            cluster_sync();
        } else {
            __syncthreads();
        }
    }

    // ---- the slice
    auto penalised = [&](float x, std::uint32_t w) {
        if ((w & ~kBiased) != 0) {
            x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
            if ((w & kCount) != 0) {
                x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(w & kCount)));
                x = __fsub_rn(x, pres);
            }
        }
        return x;
    };
    auto allowed4 = [&](std::uint32_t v) -> std::uint32_t {  // bits of tokens v .. v + 3
        if (blocked) {
            return 0u;
        }
        if (mask == nullptr) {
            return 15u;
        }
        std::uint32_t const w0 = mask[v / 32u];
        std::uint32_t const last = v + 3u < d.vocab ? v + 3u : d.vocab - 1u;
        std::uint32_t const w1 = mask[last / 32u];
        return __funnelshift_r(w0, w1, v & 31u) & 15u;
    };
    bool const use_words = penal || biased;
    std::uint64_t best = 0;
    auto one = [&](std::uint32_t v) {
        std::uint32_t const w = use_words ? words[v - begin] : 0u;
        if (w & kBiased) {
            return;
        }
        float x = penalised(in[v], w);
        x = (allowed4(v) & 1u) != 0 ? x : -INFINITY;
        if (out != nullptr) {
            out[v] = x;
        }
        std::uint64_t const c = candidate(x, v);
        best = c > best ? c : best;
    };
    if (tid < head) {
        one(begin + tid);
    }
    {
        std::uint32_t const v = body + vecs * 4u + tid;  // at most 3 tokens
        if (v < end) {
            one(v);
        }
    }
    for (std::uint32_t i0 = tid; i0 < vecs; i0 += kThreads * kVecs) {
        float4 x[kVecs];
#pragma unroll
        for (std::uint32_t k = 0; k < kVecs; ++k) {
            std::uint32_t const i = i0 + k * kThreads;
            if (i < vecs) {
                x[k] = reinterpret_cast<float4 const*>(in + body)[i];
            }
        }
#pragma unroll
        for (std::uint32_t k = 0; k < kVecs; ++k) {
            std::uint32_t const i = i0 + k * kThreads;
            if (i >= vecs) {
                break;
            }
            std::uint32_t const v = body + i * 4u;
            std::uint32_t const allow = allowed4(v);
            float y[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
            std::uint32_t flagged = 0;
            if (use_words) {
                uint4 const w = *reinterpret_cast<uint4 const*>(&words[v - begin]);
                if ((w.x | w.y | w.z | w.w) != 0) {
                    y[0] = penalised(y[0], w.x);
                    y[1] = penalised(y[1], w.y);
                    y[2] = penalised(y[2], w.z);
                    y[3] = penalised(y[3], w.w);
                    flagged = (w.x | w.y | w.z | w.w) & kBiased;
                    if (flagged) {
                        // Biased tokens are left to the pass over the biases.
                        std::uint32_t const ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if ((ws[e] & kBiased) == 0) {
                                float const z = (allow >> e & 1u) != 0 ? y[e] : -INFINITY;
                                if (out != nullptr) {
                                    out[v + e] = z;
                                }
                                std::uint64_t const c = candidate(z, v + e);
                                best = c > best ? c : best;
                            }
                        }
                    }
                }
            }
            if (flagged) {
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = (allow >> e & 1u) != 0 ? y[e] : -INFINITY;
                std::uint64_t const c = candidate(y[e], v + e);
                best = c > best ? c : best;
            }
            if (out != nullptr) {
                if (same_phase) {
                    *reinterpret_cast<float4*>(out + v) = make_float4(y[0], y[1], y[2], y[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        out[v + e] = y[e];
                    }
                }
            }
        }
    }
    for (std::uint32_t i = b0 + tid; i < b1; i += kThreads) {
        std::uint32_t const v = d.bias_tokens[i];
        if (v < begin || v >= end || (i + 1 < b1 && d.bias_tokens[i + 1] == v)) {
            continue;
        }
        float x = __fadd_rn(penalised(in[v], words[v - begin]), d.bias_values[i]);
        x = (allowed4(v) & 1u) != 0 ? x : -INFINITY;
        if (out != nullptr) {
            out[v] = x;
        }
        std::uint64_t const c = candidate(x, v);
        best = c > best ? c : best;
    }

    // ---- the greedy token
    if (d.tokens == nullptr) {
        return;  // behind the last barrier of the count nothing reads another CTA's words
    }
    if (greet) {
        cluster_wait();
    }
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
        for (int w = 1; w < kThreads / 32; ++w) {
            best = s_best[w] > best ? s_best[w] : best;
        }
        if (a.cluster > 1) {
            st_cluster_u64(cluster_map(&s_cluster[rank], 0), best);
        }
    }
    if (a.cluster > 1) {
        cluster_sync();
    }
    if (rank == 0 && tid == 0) {
        for (std::uint32_t r = 1; r < a.cluster; ++r) {
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
        static_cast<int>(kMaxSliceBytes + 32u));
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
    std::uint32_t cluster = 1;
    while (cluster < kMaxCluster && d->vocab / cluster > 4096u) {
        cluster *= 2;
    }
    a.cluster = cluster;
    a.slice = ((d->vocab + cluster - 1u) / cluster + 31u) / 32u * 32u;
    std::uint64_t const bytes = words ? std::uint64_t(a.slice + 8u) * 4u : 0u;
    if (bytes > kMaxSliceBytes || std::uint64_t(d->rows) * cluster > 0x7fffffffu) {
        return KK_EINVAL;
    }
    cudaError_t const e = allowSharedMemory();
    if (e != cudaSuccess) {
        return static_cast<int>(e);
    }
    return static_cast<int>(launch(logits_process_kernel, dim3(d->rows * cluster), dim3(kThreads), bytes,
        static_cast<cudaStream_t>(stream), cluster, a));
}
