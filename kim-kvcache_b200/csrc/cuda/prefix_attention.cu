// K8 — decode attention of lanes that share a prefix, for sm_100a.
//
// Lanes of a group see the same leading pages. Their query rows of one KV head
// (lane_count x query heads per KV head) together are the M dimension of two
// matrix products per 128-token tile, S = Q K^T and O += P V, so the shared
// pages are read once per 256 rows instead of once per lane, and the products
// are large enough for tcgen05. What the lanes have of their own goes through
// the small-row path of the decode kernels. Both kinds of work run in one
// launch, one thread block per item; every item leaves unnormalised FP32 partials
// (O, row maximum, row sum) and a second, dependent launch joins each query
// row's partials and rounds once to FP16.
//
// Shared item (one block per SM), up to two tiles of 128 query rows:
//  * warp 8 walks the item's descriptors and fills a 6-stage ring with 128-token
//    tiles of one KV head, K then V, [token][64 dims] with the 128-byte
//    swizzle (TMA; an 8-token group is one swizzle atom, so pages of any size
//    meet in a tile; each lane issues the copies of one page). A tile that is
//    not full has the V rows of its invalid tokens zeroed in shared memory
//    (0 * NaN would be NaN);
//  * warp 9 issues the tcgen05.mma of both products: Q (shared memory, 128
//    rows) x K -> S (TMEM), P (TMEM) x V (shared memory, token rows = K
//    dimension, i.e. MN-major) -> O (TMEM). Three S tiles take turns: two are
//    in the hands of the softmax groups while the next scores are formed;
//  * warps 0-3 and 4-7 are two softmax groups, one thread per query row, each
//    with its own O. Two row tiles: one group each, every K/V tile for both. One
//    row tile: the groups take the token tiles in turn and join at the end.
// P goes into the second product as two FP16 values, what rounding leaves of it
// being the second, as in the per-lane kernels: 22 bits of a weight. With the first
// alone, a lane whose neighbours share its prefix would be less exact than one by
// itself (64 lanes over each of two prefixes of 32,749 tokens: 57 us in place of 68,
// results 1.4 times as far from 64 bits as FP16 rounding leaves them).
// The running maximum is only raised, and O only rescaled, when a row's maximum
// grows by more than 2^8 (P stays within FP16; the quotient is exact in either
// case).
// The exponentials, 16 per SM and clock, bound a K/V tile for 256 rows: 2,048
// clocks. Measured: 2,950 clocks (64 lanes over each of two prefixes of 32,749
// tokens: 68 us); 67.6 us with a quarter of them by a polynomial on the FMA pipes, which
// differ from the others by more than FP32 rounding. Without the second
// halves, of a group's turn of then 2,500 clocks 200 went by until it had seen its
// scores, 150 until it held them, 400 for the maximum, 1,450 for the weights, 300
// until it looked for the next. Steps on the way, per such tile: 2.6 us with two groups that
// waited for each product (or four of half rows), while the products were issued
// from a branch of one lane (see elect_lane); 1.9 us without that branch. Without the
// second halves: 1.6 us; 1.4 us with the third S tile. No faster there: four groups in
// turn over three S tiles (2.4 us, all three are then in use at once), 16 softmax
// warps with a quarter of two rows a thread (1.7 us), an issuer for each group.
//
// A lane's own pages: one warp per (lane, KV head, run of pages), 16-token
// slices through a private cp.async ring, scores transposed (tokens x heads) on
// m16n8k16 tiles: the products are at most 16 rows high, HBM bounds them.
#include "../../../include/kk_kernels.h"
#include "kernels_internal.h"
#include "launch.cuh"

#include <atomic>
#include <cmath>
#include <memory>
#include <new>

namespace kk {

__device__ unsigned int g_prefix_status;

namespace {

constexpr std::uint32_t kHeadDim = 64;
constexpr std::uint32_t kRowBytes = kHeadDim * 2;
constexpr std::uint32_t kSoftWarps = 8;
constexpr std::uint32_t kOwnWarps = 8;                // of a block that serves lanes' own pages
constexpr std::uint32_t kProducerWarp = 8;
constexpr std::uint32_t kIssuerWarp = 9;
constexpr std::uint32_t kThreads = 384;               // three warpgroups; warps 10 and 11 only fill the third
// A softmax thread holds a row of scores (128 values); the third warpgroup gives up
// registers for it. The block is launched with kLaunchRegs a thread, and the
// shares must fit into what was launched.
constexpr std::uint32_t kLaunchRegs = 168;
constexpr std::uint32_t kSoftRegs = 216;
constexpr std::uint32_t kFewRegs = 72;
static_assert(2 * kSoftRegs + kFewRegs <= 3 * kLaunchRegs, "a share beyond the launch's registers never comes");
constexpr std::uint32_t kStages = 6;
constexpr std::uint32_t kTile = 128;                  // tokens per tile, and query rows per row tile
constexpr std::uint32_t kSlots = kTile / 8;           // 8-token groups per tile
constexpr std::uint32_t kTileBytes = kTile * kRowBytes;  // K, V or Q
constexpr std::uint32_t kStageBytes = 2 * kTileBytes;
constexpr std::uint64_t kAllValid = 0x8888888888888888ull;  // 8 tokens in each of 16 groups

// TMEM columns.
constexpr std::uint32_t kTmemCols = 512;
constexpr std::uint32_t kSTiles = 3;
constexpr std::uint32_t kColS = 0;      // S tiles of 128 columns
constexpr std::uint32_t kColO = 384;    // two O tiles of 64
// P, two tokens to a column, replaces S from its start; its low halves follow.
constexpr std::uint32_t kColLow = kTile / 2;

// A lane's own pages.
constexpr std::uint32_t kSlice = 16;                       // tokens per step
constexpr std::uint32_t kSliceBytes = 2 * kSlice * kRowBytes;
constexpr std::uint32_t kSliceRing = kStages * kStageBytes / kOwnWarps / kSliceBytes;  // 6
static_assert(kSliceRing <= 9, "the validity queue below holds eight slices");

constexpr float kRescale = 8.f;  // log2 growth of a row maximum that rescales O
// Weights are 2^7 times as large as the maximum asks for: with that growth
// they still stay below FP16's 2^16, and what the two halves lose among its
// subnormals is below 2^-32 of the largest one.
constexpr float kWeightLog2 = 7.f;
// A score in log2 units from which on the rounding of kWeightLog2 less that score
// shows (2^-6 here; from 2^23 on weights leave FP16's range).
constexpr float kFarLog2 = 0x1p18f;

struct Args {
    __half const* micro;
    __half const* extent;
    std::uint64_t micro_page;   // elements
    std::uint64_t extent_page;
    std::uint32_t micro_slots;
    std::uint32_t extent_slots;
    std::uint32_t micro_cap;
    std::uint32_t layer;
    std::uint32_t kv_heads;
    std::uint32_t group;        // query heads per KV head
    kk_prefix_plan plan;
    kk_page_desc const* descs;
    kk_attn_lane const* lanes;
    kk_prefix_group const* groups;
    kk_prefix_item const* items;
    __half const* query;
    __half* output;
    std::uint64_t query_stride;
    std::uint64_t output_stride;
    float scale_log2;
    float far_score;            // scores of kFarLog2 and kRescale in log2 units
    float rescale_score;
    float* part_o;              // [part_rows][64]
    float2* part_ml;            // [part_rows] maximum (log2 units), sum
};

struct Maps {
    CUtensorMap micro;       // boxes of a whole page
    CUtensorMap micro8;      // boxes of 8 tokens
    CUtensorMap extent;
    CUtensorMap extent8;
};

struct Shared {  // behind the ring and the two Q tiles
    std::uint64_t full[kStages];    // K and V landed
    std::uint64_t fixed[kStages];   // V rows of invalid tokens are zero
    std::uint64_t empty[kStages];   // the products are done with the stage
    // Scores of turn q, in barrier q % 4: with three S tiles those of turn q + 2, for
    // the same group, can be there before its last warp has looked for q's. Those
    // of turn q + 4 cannot.
    std::uint64_t s_full[4];
    std::uint64_t p_full[kSTiles];  // weights in an S tile
    std::uint64_t o_done[2];        // the last product into an O tile
    std::uint64_t q_full;
    std::uint64_t o_full;
    std::uint64_t valid[kStages];   // valid tokens of each 8-token group, 4 bits each
    std::uint32_t tmem;
    int abort;
};

constexpr std::uint32_t kQBytes = 2 * kTileBytes;
constexpr std::size_t kSmemBytes = 1024 + kStages * kStageBytes + kQBytes + sizeof(Shared);

__device__ __forceinline__ void report(unsigned int code) { atomicCAS(&g_prefix_status, kErrNone, code); }

// Bounded wait that also ends when another warp gave up.
__device__ __forceinline__ bool wait_or_abort(std::uint64_t* bar, std::uint32_t phase, int volatile* abort)
{
    if (mbar_poll(bar, phase)) {
        return true;
    }
    std::uint64_t const t0 = global_ns();
    for (std::uint32_t i = 0; i < kMaxWaitPolls; ++i) {
        if (mbar_poll(bar, phase)) {
            return true;
        }
        if (*abort) {
            return false;
        }
        if (global_ns() - t0 > kWaitLimitNs) {
            break;
        }
    }
    *abort = 1;
    report(kErrWaitTimeout);
    return false;
}

__device__ __forceinline__ void tma_load_page(void* dst, CUtensorMap const* map, std::uint64_t* bar, int head,
    int token, int block, int page)
{
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<std::uint64_t>(map)), "r"(smem_u32(bar)),
        "r"(0), "r"(head), "r"(token), "r"(block), "r"(page)
        : "memory");
}

// The products are issued from code that the whole warp runs, each by its one
// elected lane: descriptors then stay in uniform registers. (Issued inside a
// branch of one lane, every descriptor is moved there first: 65 clocks per
// instruction measured, against 32 of work.)
__device__ __forceinline__ std::uint32_t elect_lane()
{
    std::uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}

// D(tmem) (+)= A(tmem) * B(smem desc).
__device__ __forceinline__ void mma_ts(std::uint32_t elected, std::uint32_t d, std::uint32_t a, std::uint64_t b,
    std::uint32_t idesc, std::uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %0, 0;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], %3, %4, p;\n\t}"
        ::"r"(elected), "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// D(tmem) (+)= A(smem desc) * B(smem desc)^T.
__device__ __forceinline__ void mma_ss(std::uint32_t elected, std::uint32_t d, std::uint64_t a, std::uint64_t b,
    std::uint32_t idesc, std::uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %0, 0;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%1], %2, %3, %4, p;\n\t}"
        ::"r"(elected), "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrives on the barrier once the elected lane's products are done.
__device__ __forceinline__ void commit(std::uint32_t elected, std::uint64_t* bar)
{
    if (elected) {
        tc_commit(bar);
    }
    __syncwarp();
}

// 32 lanes x 32 columns; the caller waits.
__device__ __forceinline__ void tmem_ld32(std::uint32_t addr, float* v)
{
    std::uint32_t* r = reinterpret_cast<std::uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32"
        " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21,"
        " %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(std::uint32_t addr, std::uint32_t const (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
        " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two FP32 values in one 64-bit register: one instruction for both.
__device__ __forceinline__ std::uint64_t pack_f32x2(float lo, float hi)
{
    std::uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ void unpack_f32x2(std::uint64_t v, float& lo, float& hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}

__device__ __forceinline__ std::uint64_t fma_f32x2(std::uint64_t a, std::uint64_t b, std::uint64_t c)
{
    std::uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ std::uint64_t add_f32x2(std::uint64_t a, std::uint64_t b)
{
    std::uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float max_nan(float a, float b, float c)  // NaN if one of them is
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ std::uint32_t pack_half2(float lo, float hi)
{
    __half2 const h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<std::uint32_t const*>(&h);
}

// The leading 11 bits of p: what FP16 holds of it exactly (above its subnormals).
__device__ __forceinline__ float leading(float p) { return __uint_as_float(__float_as_uint(p) & 0xffffe000u); }

// Partials are rows of 16 chunks of 16 bytes; a row's chunks are permuted by its
// number, so that a thread per row can write them to shared memory without bank
// conflicts. Place of chunk c:
__device__ __forceinline__ std::uint32_t part_chunk(std::uint64_t row, std::uint32_t c)
{
    return c ^ (static_cast<std::uint32_t>(row) & 15u);
}

// ---- shared items -------------------------------------------------------------

__device__ __forceinline__ void produce(Args const& a, Maps const& maps, kk_prefix_item const& item,
    std::uint8_t* ring, Shared* sh)
{
    std::uint32_t const lane = threadIdx.x % 32u;
    int volatile* abort = &sh->abort;
    int const block = static_cast<int>(a.layer * 2u);
    int const head = static_cast<int>(item.kv_head);
    // A window of 32 descriptors from e on, one per lane.
    std::uint32_t e = item.desc_begin;
    std::uint32_t slot = 0, tokens = 0, kind = 0;
    auto fetch = [&]() {
        std::uint32_t const i = e + lane;
        slot = tokens = kind = 0;
        if (i < item.desc_end) {
            std::uint32_t const* d = reinterpret_cast<std::uint32_t const*>(a.descs + i);
            std::uint32_t const word = __ldg(d + 2);
            slot = __ldg(d);
            tokens = word & 0xffffu;
            kind = (word >> 16) & 0xffu;
        }
    };
    fetch();
    bool ok = true;
    std::uint32_t tile = 0;
    for (; tile < item.token_tiles; ++tile) {
        std::uint32_t const s = tile % kStages;
        std::uint32_t const phase = (tile / kStages) & 1u;
        ok = tile < kStages || wait_or_abort(&sh->empty[s], phase ^ 1u, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
            break;
        }
        std::uint8_t* const k_dst = ring + s * kStageBytes;
        std::uint64_t valid = 0;
        std::uint32_t n = 0;  // groups of the tile filled
        for (bool more = true; more;) {
            // A page outside its pool or over its capacity counts nothing and is reported.
            std::uint32_t const cap = kind == 0 ? a.micro_cap : 64u;
            bool const good = kind <= 1u && slot < (kind == 0 ? a.micro_slots : a.extent_slots) && tokens <= cap;
            if (!good && e + lane < item.desc_end) {
                report(kErrBadDescriptor);
            }
            std::uint32_t const groups = good ? (tokens + 7u) / 8u : 0u;
            std::uint32_t last = groups;  // groups of the window up to this lane's
#pragma unroll
            for (std::uint32_t o = 1; o < 32u; o *= 2u) {
                std::uint32_t const x = __shfl_up_sync(0xffffffffu, last, o);
                last += lane >= o ? x : 0u;
            }
            bool const fits = n + last <= kSlots;  // a leading run of the lanes
            std::uint32_t const taken = __popc(__ballot_sync(0xffffffffu, fits));
            std::uint32_t const sum = __shfl_sync(0xffffffffu, last, taken == 0 ? 0 : taken - 1u);
            std::uint32_t const added = taken == 0 ? 0u : sum;
            // Counted before the copies: the phase cannot end before the arrival below.
            if (lane == 0 && added != 0) {
                asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;"
                             ::"r"(smem_u32(&sh->full[s])), "r"(2u * added * 8u * kRowBytes)
                             : "memory");
            }
            __syncwarp();
            std::uint64_t mine = 0;
            if (fits && groups != 0) {
                std::uint32_t const at = n + last - groups;
                bool const whole = groups * 8u == cap;
                CUtensorMap const* map = kind == 0 ? (whole ? &maps.micro : &maps.micro8)
                                                   : (whole ? &maps.extent : &maps.extent8);
                std::uint32_t const step = whole ? groups : 1u;  // groups per box
                for (std::uint32_t g = 0; g < groups; g += step) {
                    std::uint8_t* dst = k_dst + (at + g) * 8u * kRowBytes;
                    tma_load_page(dst, map, &sh->full[s], head, static_cast<int>(g * 8u), block,
                        static_cast<int>(slot));
                    tma_load_page(dst + kTileBytes, map, &sh->full[s], head, static_cast<int>(g * 8u), block + 1,
                        static_cast<int>(slot));
                }
                // 8 tokens in every group but the page's last.
                std::uint64_t const full = groups == 1u ? 0u : kAllValid >> (64u - 4u * (groups - 1u));
                std::uint64_t const rest = tokens - (groups - 1u) * 8u;
                mine = (full | (rest << (4u * (groups - 1u)))) << (4u * at);
            }
            std::uint32_t const lo = __reduce_or_sync(0xffffffffu, static_cast<std::uint32_t>(mine));
            std::uint32_t const hi = __reduce_or_sync(0xffffffffu, static_cast<std::uint32_t>(mine >> 32));
            valid |= (std::uint64_t(hi) << 32) | lo;
            n += added;
            e += taken;
            more = taken == 32u && e < item.desc_end;  // the tile may go on behind the window
            fetch();
        }
        e = e < item.desc_end ? e : item.desc_end;
        if (lane == 0) {
            sh->valid[s] = valid;
            mbar_arrive(&sh->full[s]);  // releases valid; the phase ends when the bytes land
        }
        if (valid != kAllValid) {
            ok = wait_or_abort(&sh->full[s], phase, abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                ++tile;
                break;
            }
            std::uint8_t* const v = k_dst + kTileBytes;
            for (std::uint32_t i = lane; i < kTile * 8u; i += 32u) {
                std::uint32_t const t = i / 8u;
                if (t % 8u >= ((valid >> (4u * (t / 8u))) & 15u)) {
                    *reinterpret_cast<uint4*>(v + i * 16u) = make_uint4(0, 0, 0, 0);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        }
        if (lane == 0) {
            mbar_arrive(&sh->fixed[s]);
        }
    }
    if (ok && lane == 0 && e < item.desc_end) {
        report(kErrBadArgument);  // more pages than the item's tiles
    }
    if (!ok) {
        // Nothing of this block may still be landing when it ends.
        if (lane == 0) {
            for (std::uint32_t j = tile > kStages ? tile - kStages : 0u; j < tile; ++j) {
                mbar_wait(&sh->full[j % kStages], (j / kStages) & 1u, nullptr);
            }
        }
        __syncwarp();
    }
}

// The tiles of an item in turn: turn q works on K/V tile q / 2 for row tile q % 2
// (two row tiles), or on K/V tile q (one). Its O tile is q % 2, its S tile q % 3.
__device__ __forceinline__ std::uint32_t turns_of(kk_prefix_item const& item) { return item.token_tiles * item.row_tiles; }

__device__ __forceinline__ void issue(kk_prefix_item const& item, std::uint8_t* ring, std::uint8_t* q_tiles,
    Shared* sh)
{
    int volatile* abort = &sh->abort;
    std::uint32_t const elected = elect_lane();
    std::uint32_t const tmem = sh->tmem;
    std::uint32_t const turns = turns_of(item);
    std::uint32_t const pair = item.row_tiles == 2u ? 1u : 0u;
    constexpr std::uint32_t kIdescQK = umma_idesc_f16_f32(128, 128);
    constexpr std::uint32_t kIdescPV = umma_idesc_f16_f32(128, 64) | (1u << 16);  // V is MN-major
    auto wait = [&](std::uint64_t* bar, std::uint32_t phase) {
        return __all_sync(0xffffffffu, wait_or_abort(bar, phase & 1u, abort)) != 0;
    };
    auto scores = [&](std::uint32_t q) {
        std::uint32_t const j = q >> pair;
        if (!wait(&sh->full[j % kStages], j / kStages)) {
            return false;
        }
        std::uint64_t const q_desc = umma_desc_k_sw128(q_tiles + (q & pair) * kTileBytes);
        std::uint64_t const k_desc = umma_desc_k_sw128(ring + (j % kStages) * kStageBytes);
#pragma unroll
        for (std::uint32_t k = 0; k < kHeadDim / 16u; ++k) {
            mma_ss(elected, tmem + kColS + (q % kSTiles) * kTile, q_desc + k * 2u, k_desc + k * 2u, kIdescQK, k != 0);
        }
        commit(elected, &sh->s_full[q % 4u]);
        return true;
    };
    bool ok = wait(&sh->q_full, 0);
    tc_fence_after();
    for (std::uint32_t q = 0; ok && q < kSTiles && q < turns; ++q) {
        ok = scores(q);
    }
    for (std::uint32_t q = 0; ok && q < turns; ++q) {
        std::uint32_t const j = q >> pair;
        ok = wait(&sh->fixed[j % kStages], j / kStages) && wait(&sh->p_full[q % kSTiles], q / kSTiles);
        if (!ok) {
            break;
        }
        tc_fence_after();
        std::uint64_t const v_desc = umma_desc_k_sw128(ring + (j % kStages) * kStageBytes + kTileBytes);
        std::uint32_t const o = tmem + kColO + (q % 2u) * kHeadDim;
#pragma unroll
        for (std::uint32_t i = 0; i < kTile / 16u; ++i) {
            std::uint32_t const p = tmem + kColS + (q % kSTiles) * kTile + i * 8u;
            std::uint64_t const b = v_desc + i * 16u * (kRowBytes / 16u);
            mma_ts(elected, o, p, b, kIdescPV, q >= 2u || i != 0);
            mma_ts(elected, o, p + kColLow, b, kIdescPV, 1u);
        }
        commit(elected, &sh->o_done[q % 2u]);
        if (!pair || q % 2u == 1u) {
            commit(elected, &sh->empty[j % kStages]);
        }
        // The scores that overwrite these weights are issued behind the
        // product that reads them; the tensor core runs the two in that order.
        if (q + kSTiles < turns) {
            ok = scores(q + kSTiles);
        }
    }
    commit(elected, &sh->o_full);
    if (!ok) {
        mbar_wait(&sh->o_full, 0, nullptr);  // no product outlives the TMEM
    }
}

// One thread per query row: warp % 4 selects the TMEM lanes, warp / 4 the group,
// which serves every second turn.
__device__ __forceinline__ void soften(Args const& a, kk_prefix_item const& item, std::uint8_t* ring,
    std::uint8_t* q_tiles, Shared* sh)
{
    int volatile* abort = &sh->abort;
    std::uint32_t const warp = threadIdx.x / 32u;
    std::uint32_t const lane = threadIdx.x % 32u;
    std::uint32_t const t = warp / 4u;  // group and O tile
    std::uint32_t const pair = item.row_tiles == 2u ? 1u : 0u;
    std::uint32_t const r = (warp % 4u) * 32u + lane;
    std::uint32_t const tile_row = (item.row_tile + (t & pair)) * kTile;
    std::uint32_t const rows = item.lane_count * a.group;
    bool const mine = tile_row + r < rows;
    bool const any = tile_row + (warp % 4u) * 32u < rows;  // some row of this warp exists
    std::uint32_t const tmem = sh->tmem + ((warp % 4u) * 32u << 16);
    std::uint32_t const o_col = tmem + kColO + t * kHeadDim;

    if (pair || t == 0) {
        uint4 q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            q[i] = make_uint4(0, 0, 0, 0);
        }
        if (mine) {
            std::uint32_t const row = tile_row + r;
            std::uint32_t const query_row = a.lanes[item.lane_begin + row / a.group].query_row;
            uint4 const* src = reinterpret_cast<uint4 const*>(a.query + query_row * a.query_stride
                + (item.kv_head * a.group + row % a.group) * kHeadDim);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[i] = src[i];
            }
        }
        std::uint8_t* const dst = q_tiles + t * kTileBytes + r * kRowBytes;
#pragma unroll
        for (std::uint32_t i = 0; i < 8u; ++i) {
            *reinterpret_cast<uint4*>(dst + ((i ^ (r & 7u)) << 4)) = q[i];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    if (lane == 0) {
        mbar_arrive(&sh->q_full);
    }

    auto wait = [&](std::uint64_t* bar, std::uint32_t phase) {
        return __all_sync(0xffffffffu, wait_or_abort(bar, phase & 1u, abort)) != 0;
    };
    std::uint32_t const turns = turns_of(item);
    float ref = -INFINITY;  // reference maximum of the row's scores
    float limit = -INFINITY;  // a score above this one moves the reference
    float shift = 0.f;      // weights are 2^(score * scale_log2 + shift)
    float l = 0.f;
    bool ok = true;
    for (std::uint32_t q = t; q < turns; q += 2u) {
        std::uint32_t const k = q / 2u;  // turn of this group
        std::uint32_t const j = q >> pair;
        std::uint32_t const buf = q % kSTiles;
        std::uint32_t const s_col = tmem + kColS + buf * kTile;
        // Both polls are under way at once: behind a queue of exponentials each takes long.
        bool const scored = mbar_poll(&sh->s_full[q % 4u], (q / 4u) & 1u);
        bool const landed = mbar_poll(&sh->full[j % kStages], (j / kStages) & 1u);
        if (!__all_sync(0xffffffffu, scored && landed)) {
            ok = wait(&sh->s_full[q % 4u], q / 4u) && wait(&sh->full[j % kStages], j / kStages);
            if (!ok) {
                break;
            }
        }
        tc_fence_after();
        if (any) {
            float x[kTile];
#pragma unroll
            for (std::uint32_t c = 0; c < 4u; ++c) {
                tmem_ld32(s_col + c * 32u, x + c * 32u);
            }
            std::uint64_t const valid = sh->valid[j % kStages];
            tmem_wait_ld();
            if (valid != kAllValid) {
#pragma unroll
                for (std::uint32_t i = 0; i < kTile; ++i) {
                    x[i] = (i % 8u) < (static_cast<std::uint32_t>(valid >> (4u * (i / 8u))) & 15u) ? x[i] : -INFINITY;
                }
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (std::uint32_t i = 0; i < kTile; i += 2u) {
                top[i / 2u % 4u] = max_nan(top[i / 2u % 4u], x[i], x[i + 1u]);
            }
            float const highest = max_nan(max_nan(top[0], top[1], top[2]), top[3], top[3]);
            if (__any_sync(0xffffffffu, highest > limit)) {
                bool const grow = (highest - ref) * a.scale_log2 > kRescale || ref == -INFINITY;
                float const now = grow ? highest : ref;
                float const alpha = ref == -INFINITY ? 1.f : exp2_approx((ref - now) * a.scale_log2);
                ref = now;
                l *= alpha;
                // So far out that kWeightLog2 less the reference would lose the weight: the
                // reference is taken off the scores, of every tile from here on.
                bool const far = fabsf(ref) > a.far_score && fabsf(ref) < INFINITY;
                limit = far ? -INFINITY : ref + a.rescale_score;
                shift = ref == -INFINITY ? 0.f : far ? kWeightLog2 : kWeightLog2 - ref * a.scale_log2;
                if (__any_sync(0xffffffffu, far)) {
                    float const less = far ? ref : 0.f;
#pragma unroll
                    for (std::uint32_t i = 0; i < kTile; ++i) {
                        x[i] -= less;
                    }
                }
                if (k != 0) {
                    // Once the last product into O is done.
                    ok = wait(&sh->o_done[t], k - 1u);
                    if (!ok) {
                        break;
                    }
                    tc_fence_after();
#pragma unroll 1
                    for (std::uint32_t c = 0; c < kHeadDim / 16u; ++c) {
                        float o[16];
                        tmem_ld16(o_col + c * 16u, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            o[i] *= alpha;
                        }
                        tmem_st16(o_col + c * 16u, reinterpret_cast<std::uint32_t const(&)[16]>(o));
                    }
                }
            }
            // A NaN or +inf among the scores makes the row NaN.
            float const use = highest < INFINITY ? shift : NAN;
            std::uint64_t const scale2 = pack_f32x2(a.scale_log2, a.scale_log2);
            std::uint64_t const shift2 = pack_f32x2(use, use);
            std::uint64_t sum2[2] = {0, 0};
#pragma unroll
            for (std::uint32_t c = 0; c < 4u; ++c) {
                std::uint32_t p[16], low[16];
#pragma unroll
                for (std::uint32_t i = 0; i < 16u; ++i) {
                    std::uint32_t const at = c * 32u + 2u * i;
                    std::uint64_t const y = fma_f32x2(pack_f32x2(x[at], x[at + 1u]), scale2, shift2);
                    float p0, p1;
                    unpack_f32x2(y, p0, p1);
                    p0 = exp2_approx(p0);
                    p1 = exp2_approx(p1);
                    sum2[i % 2u] = add_f32x2(sum2[i % 2u], pack_f32x2(p0, p1));
                    p[i] = pack_half2(p0, p1);
                    float l0, l1;  // what that leaves of the two: exact
                    asm("{\n\t.reg .b16 a, b, m;\n\tmov.b32 {a, b}, %2;\n\tmov.b16 m, 0xBC00;\n\t"
                        "fma.rn.f32.f16 %0, a, m, %3;\n\tfma.rn.f32.f16 %1, b, m, %4;\n\t}"
                        : "=f"(l0), "=f"(l1) : "r"(p[i]), "f"(p0), "f"(p1));
                    low[i] = pack_half2(l0, l1);
                }
                tmem_st16(s_col + c * 16u, p);
                tmem_st16(s_col + kColLow + c * 16u, low);
            }
            float s0, s1;
            unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
            l += s0 + s1;
            tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&sh->p_full[buf]);
        }
    }
    ok = ok && wait(&sh->o_full, 0);
    tc_fence_after();
    float m = ref * a.scale_log2;
    // One row tile: the second group's O joins the first's through the ring,
    // which nothing uses any more.
    constexpr std::uint32_t kStride = kHeadDim + 3;  // odd: rows fall into different banks
    static_assert(kTile * kStride * 4 <= 2 * kStageBytes, "room below the tiles that leave");
    float* const other = reinterpret_cast<float*>(ring) + r * kStride;
    if (!pair && t == 1u && ok) {
        bool const holds = any && turns > 1u;
#pragma unroll
        for (std::uint32_t c = 0; c < 4u; ++c) {
            float o[16];
            if (holds) {
                tmem_ld16(o_col + c * 16u, o);
            }
#pragma unroll
            for (std::uint32_t i = 0; i < 16u; ++i) {
                other[c * 16u + i] = holds ? o[i] : 0.f;
            }
        }
        other[kHeadDim] = m;
        other[kHeadDim + 1] = l;
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");  // the 8 softmax warps, all of which come here
    if (!pair && t == 1u) {
        return;
    }
    float f0 = 1.f, f1 = 0.f;
    if (!pair && ok) {
        float const m1 = other[kHeadDim];
        float const top = fmaxf(m, m1);
        float const use = top == -INFINITY ? 0.f : top;
        f0 = exp2_approx(m - use);
        f1 = exp2_approx(m1 - use);
        m = top;
        l = l * f0 + other[kHeadDim + 1] * f1;
    }
    // The rows leave through shared memory in one bulk copy (stores of a row per
    // thread took 3.4 us in place of 0.9 for two row tiles).
    std::uint64_t const first_row = std::uint64_t(item.part_row) + (t & pair) * kTile;
    float4* const tile = reinterpret_cast<float4*>(ring + (2u + t) * kStageBytes);
    if (ok && any) {
#pragma unroll
        for (std::uint32_t c = 0; c < 4u; ++c) {
            float o[16];
            tmem_ld16(o_col + c * 16u, o);  // the whole warp, also for rows that do not exist
            if (!pair) {
#pragma unroll
                for (std::uint32_t i = 0; i < 16u; ++i) {
                    o[i] = o[i] * f0 + other[c * 16u + i] * f1;
                }
            }
#pragma unroll
            for (std::uint32_t i = 0; i < 4u; ++i) {
                tile[r * 16u + part_chunk(first_row + r, c * 4u + i)] =
                    make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
        }
        if (mine) {
            a.part_ml[first_row + r] = make_float2(m - kWeightLog2, l);
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("bar.sync %0, 128;" ::"r"(2u + t) : "memory");  // the group's 4 warps, all of which come here
    if (r == 0 && !*abort) {
        std::uint32_t const left = rows - tile_row;
        std::uint32_t const bytes = (left < kTile ? left : kTile) * kHeadDim * 4u;
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                     ::"l"(a.part_o + first_row * kHeadDim), "r"(smem_u32(tile)), "r"(bytes)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    }
}

// ---- a lane's own pages -------------------------------------------------------

__device__ __forceinline__ void cp_async16(std::uint32_t dst, void const* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void ldsm_x4(std::uint32_t addr, std::uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void ldsm_x4_t(std::uint32_t addr, std::uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], std::uint32_t a0, std::uint32_t a1, std::uint32_t a2,
    std::uint32_t a3, std::uint32_t b0, std::uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ std::uint32_t transpose8x8(std::uint32_t x)
{
    std::uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// One (lane, KV head, run of pages) by one warp. NT: tiles of 8 query heads.
template <int NT>
__device__ __forceinline__ void own_task(Args const& a, kk_prefix_item const& item, std::uint8_t* warp_ring)
{
    std::uint32_t const lane = threadIdx.x % 32u;
    std::uint32_t const g = lane >> 2;
    std::uint32_t const c4 = lane & 3u;
    std::uint32_t const mi = lane >> 3;
    std::uint32_t const r8 = lane & 7u;
    std::uint32_t const G = a.group;
    std::uint64_t const row0 = item.part_row;
    // Queries as B fragments of S^T = K Q^T; heads past the group are zero.
    std::uint32_t qf[NT][4][2];
    {
        __half const* q = a.query + item.query_row * a.query_stride + item.kv_head * G * kHeadDim;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            std::uint32_t const h = nt * 8u + g;
#pragma unroll
            for (int k16 = 0; k16 < 4; ++k16) {
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                    qf[nt][k16][hi] = h < G ? *reinterpret_cast<std::uint32_t const*>(
                        q + h * kHeadDim + k16 * 16 + hi * 8 + c4 * 2u) : 0u;
                }
            }
        }
    }
    // Cursor over 8-token groups.
    std::uint32_t const row = a.kv_heads * kHeadDim;  // elements per token
    std::uint32_t win = item.desc_begin;
    std::uint32_t w_slot = 0, w_word = 0;
    auto fetch = [&]() {
        std::uint32_t const i = win + lane;
        w_slot = w_word = 0;
        if (i < item.desc_end) {
            std::uint32_t const* d = reinterpret_cast<std::uint32_t const*>(a.descs + i);
            w_slot = __ldg(d);
            w_word = __ldg(d + 2);
        }
    };
    fetch();
    std::uint32_t e = item.desc_begin, token = 0;
    __half const* src = nullptr;   // K of the next group's first token; V follows after v_off elements
    std::uint32_t v_off = 0;
    // Moves to the next group; its valid tokens, 0 at the end.
    auto next_group = [&](__half const*& at, std::uint32_t& off) -> std::uint32_t {
        for (; e < item.desc_end; ++e, token = 0) {
            if (e >= win + 32u) {
                win += 32u;
                fetch();
            }
            std::uint32_t const slot = __shfl_sync(0xffffffffu, w_slot, e - win);
            std::uint32_t const word = __shfl_sync(0xffffffffu, w_word, e - win);
            std::uint32_t const tokens = word & 0xffffu;
            std::uint32_t const kind = (word >> 16) & 0xffu;
            std::uint32_t const cap = kind == 0 ? a.micro_cap : 64u;
            if (kind > 1u || slot >= (kind == 0 ? a.micro_slots : a.extent_slots) || tokens > cap) {
                if (lane == 0) {
                    report(kErrBadDescriptor);
                }
                continue;
            }
            if (token >= tokens) {
                continue;
            }
            __half const* page = kind == 0 ? a.micro + slot * a.micro_page : a.extent + slot * a.extent_page;
            v_off = cap * row;
            src = page + std::uint64_t(a.layer) * 2u * v_off + token * row + item.kv_head * kHeadDim;
            std::uint32_t const left = tokens - token;
            token += 8u;
            at = src;
            off = v_off;
            return left < 8u ? left : 8u;
        }
        return 0u;
    };
    std::uint32_t const ring = smem_u32(warp_ring);
    std::uint64_t queue = 0;  // valid tokens of the slices in flight: 8 bits each, newest highest
    std::uint32_t head_slice = 0;  // slices requested
    auto request = [&]() {  // one slice (or nothing) into the ring, always one commit group
        __half const* at0 = nullptr;
        __half const* at1 = nullptr;
        std::uint32_t off0 = 0, off1 = 0;
        std::uint32_t const v0 = next_group(at0, off0);
        std::uint32_t const v1 = v0 != 0 ? next_group(at1, off1) : 0u;
        std::uint32_t const dst = ring + (head_slice % kSliceRing) * kSliceBytes;
        std::uint32_t const ch = lane & 7u;
#pragma unroll
        for (std::uint32_t i = 0; i < 4u; ++i) {
            std::uint32_t const t = (lane >> 3) + 4u * i;   // token of the slice
            std::uint32_t const in_group = t & 7u;
            if ((i < 2u ? v0 : v1) > in_group) {
                __half const* p = (i < 2u ? at0 : at1) + in_group * row + ch * 8u;
                std::uint32_t const o = t * kRowBytes + ((ch ^ in_group) << 4);
                cp_async16(dst + o, p);
                cp_async16(dst + kSlice * kRowBytes + o, p + (i < 2u ? off0 : off1));
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        queue = (queue >> 8) | (std::uint64_t(v0 | (v1 << 4)) << 56);
        ++head_slice;
    };
    float mrow[NT][2], lrow[NT][2], o[NT][4][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        mrow[nt][0] = mrow[nt][1] = -INFINITY;
        lrow[nt][0] = lrow[nt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
        }
    }
#pragma unroll 1
    for (std::uint32_t i = 0; i + 1u < kSliceRing; ++i) {
        request();
    }
    for (std::uint32_t slice = 0;; ++slice) {
        // The slice in turn is the oldest of the kSliceRing - 1 requested last.
        std::uint32_t const pairv = static_cast<std::uint32_t>(queue >> (64u - 8u * (kSliceRing - 1u))) & 0xffu;
        if (pairv == 0) {
            break;
        }
        request();
        asm volatile("cp.async.wait_group %0;" ::"n"(kSliceRing - 1u) : "memory");
        __syncwarp();
        std::uint32_t const v0 = pairv & 15u, v1 = pairv >> 4;
        std::uint32_t const kbase = ring + (slice % kSliceRing) * kSliceBytes;
        std::uint32_t const vbase = kbase + kSlice * kRowBytes;
        float st[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            st[nt][0] = st[nt][1] = st[nt][2] = st[nt][3] = 0.f;
        }
#pragma unroll
        for (std::uint32_t k16 = 0; k16 < 4; ++k16) {
            std::uint32_t const tr = (mi & 1u) * 8u + r8;
            std::uint32_t const ch = 2u * k16 + (mi >> 1);
            std::uint32_t ka[4];
            ldsm_x4(kbase + tr * kRowBytes + ((ch ^ r8) << 4), ka);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma16816(st[nt], ka[0], ka[1], ka[2], ka[3], qf[nt][k16][0], qf[nt][k16][1]);
            }
        }
        bool const tg = g < v0, tg8 = g < v1;
        // V of masked tokens is zeroed: bytes past the valid tokens are never trusted.
        std::uint32_t const mask0 = (2 * c4 < v0 ? 0x0000ffffu : 0u) | (2 * c4 + 1 < v0 ? 0xffff0000u : 0u);
        std::uint32_t const mask1 = (2 * c4 < v1 ? 0x0000ffffu : 0u) | (2 * c4 + 1 < v1 ? 0xffff0000u : 0u);
        std::uint32_t pb[NT][2], pl[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float x[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x[h] = tg ? st[nt][h] * a.scale_log2 : -INFINITY;
                x[2 + h] = tg8 ? st[nt][2 + h] * a.scale_log2 : -INFINITY;
            }
            // As in the shared items, the reference follows the maximum only when
            // that has grown by 2^8: a vote in place of two reductions a slice.
            float const top0 = fmaxf(x[0], x[2]), top1 = fmaxf(x[1], x[3]);
            if (__any_sync(0xffffffffu, top0 - mrow[nt][0] > kRescale || top1 - mrow[nt][1] > kRescale
                    || mrow[nt][0] == -INFINITY)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float mx = h == 0 ? top0 : top1;
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    float const m_new = fmaxf(mrow[nt][h], mx);
                    float const alpha = mrow[nt][h] == -INFINITY ? 0.f : exp2_approx(mrow[nt][h] - m_new);
                    lrow[nt][h] *= alpha;
                    mrow[nt][h] = m_new;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        o[nt][j][h] *= alpha;
                        o[nt][j][2 + h] *= alpha;
                    }
                }
            }
            float p[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float const use = mrow[nt][h] == -INFINITY ? 0.f : mrow[nt][h];
                p[h] = exp2_approx(x[h] - use + kWeightLog2);
                p[2 + h] = exp2_approx(x[2 + h] - use + kWeightLog2);
                lrow[nt][h] += p[h] + p[2 + h];
            }
            float hp[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                hp[i] = leading(p[i]);
            }
            pb[nt][0] = transpose8x8(pack_half2(hp[0], hp[1]));
            pb[nt][1] = transpose8x8(pack_half2(hp[2], hp[3]));
            pl[nt][0] = transpose8x8(pack_half2(p[0] - hp[0], p[1] - hp[1]));
            pl[nt][1] = transpose8x8(pack_half2(p[2] - hp[2], p[3] - hp[3]));
        }
#pragma unroll
        for (std::uint32_t j = 0; j < 4; ++j) {
            std::uint32_t const tr = (mi >> 1) * 8u + r8;
            std::uint32_t const ch = 2u * j + (mi & 1u);
            std::uint32_t va[4];
            ldsm_x4_t(vbase + tr * kRowBytes + ((ch ^ r8) << 4), va);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma16816(o[nt][j], va[0] & mask0, va[1] & mask0, va[2] & mask1, va[3] & mask1, pb[nt][0], pb[nt][1]);
                mma16816(o[nt][j], va[0] & mask0, va[1] & mask0, va[2] & mask1, va[3] & mask1, pl[nt][0], pl[nt][1]);
            }
        }
        __syncwarp();  // the slice's slot is requested again in the next step
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float l = lrow[nt][h];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            std::uint32_t const qh = nt * 8u + 2u * c4 + h;
            if (qh < G) {
                float* dst = a.part_o + (row0 + qh) * kHeadDim + g % 4u;
#pragma unroll
                for (std::uint32_t j = 0; j < 4u; ++j) {
                    dst[part_chunk(row0 + qh, 4u * j + g / 4u) * 4u] = o[nt][j][h];
                    dst[part_chunk(row0 + qh, 4u * j + 2u + g / 4u) * 4u] = o[nt][j][2 + h];
                }
                if (g == 0) {
                    a.part_ml[row0 + qh] = make_float2(mrow[nt][h] - kWeightLog2, l);
                }
            }
        }
    }
    __syncwarp();
}

template <int NT>
__global__ void __launch_bounds__(kThreads, 1) prefix_attention_kernel(const __grid_constant__ Maps maps,
    const __grid_constant__ Args a)
{
    extern __shared__ std::uint8_t smem_raw[];
    std::uint32_t const pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;  // swizzle atoms are 1 KB
    std::uint8_t* const ring = smem_raw + pad;
    std::uint8_t* const q_tiles = ring + kStages * kStageBytes;
    Shared* const sh = reinterpret_cast<Shared*>(q_tiles + kQBytes);
    std::uint32_t const warp = threadIdx.x / 32u;
    if (blockIdx.x >= a.plan.num_shared) {
        pdl_wait();
        pdl_launch_dependents();  // behind the wait: the joining launch reads the plan before its own
        if (warp >= kOwnWarps) {
            return;
        }
        std::uint32_t const own = a.plan.num_items - a.plan.num_shared;
        std::uint32_t const first = (blockIdx.x - a.plan.num_shared) * a.plan.tasks_per_cta;
        std::uint32_t const left = own - first;
        std::uint32_t const count = left < a.plan.tasks_per_cta ? left : a.plan.tasks_per_cta;
        for (std::uint32_t t = warp; t < count; t += kOwnWarps) {
            kk_prefix_item const item = a.items[a.plan.num_shared + first + t];
            if (item.row_tiles != 0 || item.owner >= a.plan.num_lanes || item.kv_head >= a.kv_heads
                || item.desc_begin > item.desc_end || item.desc_end > a.plan.num_descs
                || std::uint64_t(item.part_row) + a.group > a.plan.part_rows) {
                if (threadIdx.x % 32u == 0) {
                    report(kErrBadArgument);
                }
                continue;
            }
            own_task<NT>(a, item, ring + warp * kSliceRing * kSliceBytes);
        }
        return;
    }
    if (threadIdx.x == 0) {
        for (std::uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->fixed[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        for (std::uint32_t i = 0; i < kSTiles; ++i) {
            mbar_init(&sh->p_full[i], 4);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&sh->s_full[i], 1);
        }
        mbar_init(&sh->o_done[0], 1);
        mbar_init(&sh->o_done[1], 1);
        mbar_init(&sh->q_full, kSoftWarps);
        mbar_init(&sh->o_full, 1);
        sh->abort = 0;
        fence_barrier_init();
    }
    // All of TMEM, before the wait for what ran before: the block's shared memory
    // leaves room on the SM for none of the other kernels that use TMEM.
    if (warp == kIssuerWarp) {
        tmem_alloc(&sh->tmem, kTmemCols);
        tmem_relinquish();
        tc_fence_before();
    }
    if (warp == kProducerWarp && threadIdx.x % 32u < 4u) {
        CUtensorMap const* const all[4] = {&maps.micro, &maps.micro8, &maps.extent, &maps.extent8};
        prefetch_tensormap(all[threadIdx.x % 4u]);
    }
    pdl_wait();
    pdl_launch_dependents();
    kk_prefix_item const item = a.items[blockIdx.x];
    // The same for every thread.
    bool const fits = (item.row_tiles == 1u || item.row_tiles == 2u) && item.kv_head < a.kv_heads
        && item.desc_begin <= item.desc_end && item.desc_end <= a.plan.num_descs && item.token_tiles != 0
        && item.owner < a.plan.num_groups && item.lane_begin <= a.plan.num_lanes
        && item.lane_count <= a.plan.num_lanes - item.lane_begin
        && (item.row_tile + item.row_tiles - 1u) * kTile < std::uint64_t(item.lane_count) * a.group
        && std::uint64_t(item.part_row) + item.row_tiles * kTile <= a.plan.part_rows;
    if (!fits && threadIdx.x == 0) {
        report(kErrBadArgument);
    }
    __syncthreads();
    tc_fence_after();
    if (fits) {
        if (warp < kSoftWarps) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
            soften(a, item, ring, q_tiles, sh);
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
            if (warp == kProducerWarp) {
                produce(a, maps, item, ring, sh);
            } else if (warp == kIssuerWarp) {
                issue(item, ring, q_tiles, sh);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuerWarp) {
        tc_fence_after();
        tmem_dealloc(sh->tmem, kTmemCols);
    }
}

// ---- joining the partials -----------------------------------------------------

constexpr std::uint32_t kJoinThreads = 256;
constexpr std::uint32_t kJoinBatch = 10;  // partials that each half of the warp requests at once

// A warp per query row: out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over the
// row's partials. 16 lanes hold 4 dims each; the two halves of the warp take
// alternate partials, kJoinBatch of them at a time, and join in a fixed order.
__global__ void __launch_bounds__(kJoinThreads) prefix_join_kernel(const __grid_constant__ Args a)
{
    std::uint32_t const t = blockIdx.x * kJoinThreads + threadIdx.x;
    std::uint32_t const q_heads = a.plan.q_heads;
    std::uint32_t const lane = t / 32u / q_heads;
    if (lane >= a.plan.num_lanes) {
        return;
    }
    // The plan is older than the launch that writes the partials: it is read
    // before that one has ended. (That one began to let this one start behind its
    // own wait. Without items there is none, and what runs before may be the copy of
    // the plan.)
    if (a.plan.num_items == 0) {
        pdl_wait();
    }
    std::uint32_t const qh = t / 32u % q_heads;
    std::uint32_t const chunk = t % 16u;
    kk_attn_lane const ln = a.lanes[lane];
    std::uint64_t base = 0, step = 0;
    std::uint32_t shared = 0;
    if (ln.reserved - 1u < a.plan.num_groups) {
        kk_prefix_group const g = a.groups[ln.reserved - 1u];
        step = std::uint64_t(g.row_tiles) * kTile;
        shared = g.part_count;
        base = g.part_row + std::uint64_t(qh / a.group) * shared * step + (lane - g.lane_begin) * a.group + qh % a.group;
    }
    std::uint32_t const count = shared + ln.item_count;
    std::uint64_t const own = std::uint64_t(ln.item_offset) + qh;
    bool const fits = (shared == 0 || base + (shared - 1u) * step < a.plan.part_rows)
        && (ln.item_count == 0 || own + std::uint64_t(ln.item_count - 1u) * q_heads < a.plan.part_rows);
    if (!fits) {
        report(kErrBadArgument);
        pdl_wait();  // this launch must not end before the one that writes the partials
        return;
    }
    pdl_launch_dependents();
    pdl_wait();
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float m1, float l1, float4 const& o) {
        float const top = fmaxf(m, m1);
        float const use = top == -INFINITY ? 0.f : top;
        float const f = exp2_approx(m - use);
        float const f1 = exp2_approx(m1 - use);
        m = top;
        l = l * f + l1 * f1;
        acc.x = acc.x * f + o.x * f1;
        acc.y = acc.y * f + o.y * f1;
        acc.z = acc.z * f + o.z * f1;
        acc.w = acc.w * f + o.w * f1;
    };
    for (std::uint32_t first = 0; first < count; first += 2u * kJoinBatch) {
        float2 ml[kJoinBatch];
        float4 o[kJoinBatch];
        float top = m;
#pragma unroll
        for (std::uint32_t k = 0; k < kJoinBatch; ++k) {
            std::uint32_t const i = first + 2u * k + t % 32u / 16u;
            ml[k] = make_float2(-INFINITY, 0.f);
            o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i < count) {
                std::uint64_t const row = i < shared ? base + i * step : own + std::uint64_t(i - shared) * q_heads;
                ml[k] = __ldcg(a.part_ml + row);
                o[k] = __ldcg(reinterpret_cast<float4 const*>(a.part_o + row * kHeadDim) + part_chunk(row, chunk));
            }
        }
#pragma unroll
        for (std::uint32_t k = 0; k < kJoinBatch; ++k) {
            top = fmaxf(top, ml[k].x);
        }
        float const use = top == -INFINITY ? 0.f : top;
        float const f = exp2_approx(m - use);
        m = top;
        l *= f;
        acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
#pragma unroll
        for (std::uint32_t k = 0; k < kJoinBatch; ++k) {
            if (first + 2u * k < count) {  // the same for the whole warp
                float const f1 = exp2_approx(ml[k].x - use);
                l += ml[k].y * f1;
                acc.x += o[k].x * f1;
                acc.y += o[k].y * f1;
                acc.z += o[k].z * f1;
                acc.w += o[k].w * f1;
            }
        }
    }
    // The upper half's part joins the lower's.
    float const m1 = __shfl_down_sync(0xffffffffu, m, 16);
    float const l1 = __shfl_down_sync(0xffffffffu, l, 16);
    float4 o1;
    o1.x = __shfl_down_sync(0xffffffffu, acc.x, 16);
    o1.y = __shfl_down_sync(0xffffffffu, acc.y, 16);
    o1.z = __shfl_down_sync(0xffffffffu, acc.z, 16);
    o1.w = __shfl_down_sync(0xffffffffu, acc.w, 16);
    if (t % 32u >= 16u) {
        return;
    }
    add(m1, l1, o1);
    float const inv = l == 0.f ? 0.f : 1.f / l;  // no tokens at all: zeros
    uint2 out;
    out.x = pack_half2(acc.x * inv, acc.y * inv);
    out.y = pack_half2(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(a.output + ln.query_row * a.output_stride + qh * kHeadDim + chunk * 4u) = out;
}

// Kernel attributes are set once per device.
cudaError_t allowSharedMemory()
{
    static std::atomic<std::uint64_t> done{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && (done.load(std::memory_order_acquire) >> device & 1u) != 0)) {
        return e;
    }
    void const* const kernels[] = {reinterpret_cast<void const*>(prefix_attention_kernel<1>),
        reinterpret_cast<void const*>(prefix_attention_kernel<2>)};
    for (void const* kernel : kernels) {
        // The register shares wait for ever in a build that launches with fewer.
        cudaFuncAttributes attr{};
        e = e == cudaSuccess ? cudaFuncGetAttributes(&attr, kernel) : e;
        if (e == cudaSuccess && attr.numRegs < static_cast<int>(kLaunchRegs)) {
            e = cudaErrorInvalidKernelImage;
        }
        if (e == cudaSuccess) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes));
        }
    }
    if (e == cudaSuccess && device < 64) {
        done.fetch_or(std::uint64_t(1) << device, std::memory_order_release);
    }
    return e;
}

// ---- planning -------------------------------------------------------------------

// Times of a thread block, in nanoseconds, from which the plan deals the SMs out
// between the prefixes and the lanes' own pages. (Those of own items with the cost of
// joining their parts: shorter items than these give are no faster, 13.9 us in
// place of 13.0 for 32 lanes with up to 1,024 tokens.) Tiles measure 1,650 and 1,100
// where nothing else runs. With those two plans are no better, and worse where own
// pages, which then take longer than these say, get fewer SMs for it: 8 prefixes of
// 10,000 tokens, 8 KV heads, 8 lanes each with up to 1,000 of their own: 142 us in
// place of 119.
constexpr double kSharedNs = 5500.;     // a shared item without its tiles
constexpr double kTilePairNs = 1450.;   // a 128-token tile for two row tiles
constexpr double kTileSingleNs = 750.;  // for one
constexpr double kOwnNs = 1000.;        // a block of lanes' own items without them
constexpr double kTaskNs = 3000.;       // an own item without its tokens
constexpr double kTaskTokenNs = 40.;     // a token of an own item, by its warp
constexpr double kOwnTokenNs = 4.;      // the same by the block: 256 bytes at an SM's share of HBM
constexpr std::uint32_t kOwnMinTokens = 64;

std::uint32_t groupsOf(kk_page_desc const& d) { return d.valid_tokens > 64u ? 0u : (d.valid_tokens + 7u) / 8u; }

// 128-token tiles of a run of descriptors, filled as the kernel does; calls
// cut(tiles closed so far, first descriptor of the next tile) at every tile's end
// but the last.
template <typename Cut>
std::uint32_t walkTiles(kk_page_desc const* descs, std::uint32_t begin, std::uint32_t end, Cut&& cut)
{
    std::uint32_t closed = 0, n = 0;
    for (std::uint32_t e = begin; e < end; ++e) {
        std::uint32_t const g = groupsOf(descs[e]);
        if (n + g > kSlots) {
            cut(++closed, e);
            n = 0;
        }
        n += g;
    }
    return closed + (n != 0 ? 1u : 0u);
}

// ---- grouping

// A reader of pages costs its items' fixed part besides its tokens: as much as this
// many tokens of a lane's own (kSharedNs / kOwnTokenNs). One group of many lanes is so
// preferred to several that share a little more each.
constexpr std::uint64_t kReaderTokens = 1375;

struct Common {  // leading pages of two lanes that are the same
    std::uint32_t pages;
    std::uint64_t tokens;
};

struct Cut {  // between lanes at - 1 and at
    std::uint32_t at;
    std::uint32_t from;    // first lane of the group that ends here; at: none does
    std::uint64_t gain;    // of the groups in front
    std::uint32_t before;  // the cut where that choice begins,
    std::uint32_t next;    // and on the way back the next one
};

Common commonPages(kk_page_desc const* descs, kk_attn_lane const& x, kk_attn_lane const& y)
{
    kk_page_desc const* const p = descs + x.desc_offset;
    kk_page_desc const* const q = descs + y.desc_offset;
    std::uint32_t const most = x.desc_count < y.desc_count ? x.desc_count : y.desc_count;
    Common c{};
    while (c.pages < most && p[c.pages].slot == q[c.pages].slot && p[c.pages].kind == q[c.pages].kind
        && p[c.pages].valid_tokens == q[c.pages].valid_tokens) {
        c.tokens += p[c.pages].valid_tokens;
        ++c.pages;
    }
    return c;
}

bool headsServed(std::uint32_t q_heads, std::uint32_t kv_heads)
{
    return kv_heads != 0 && q_heads != 0 && q_heads % kv_heads == 0 && q_heads / kv_heads <= 16u && q_heads <= 4096u;
}

} // namespace

int prefixStatus(cudaStream_t stream) { return readStatus(&g_prefix_status, stream); }

} // namespace kk

extern "C" {

uint32_t kk_prefix_groups(const kk_page_desc* descs, kk_attn_lane* lanes, uint32_t num_lanes, uint32_t min_lanes,
    uint32_t min_tokens, kk_prefix_group* groups, uint32_t max_groups)
{
    using namespace kk;
    min_lanes = min_lanes < 2u ? 2u : min_lanes;
    if (descs == nullptr || lanes == nullptr || groups == nullptr || max_groups == 0 || num_lanes < min_lanes) {
        return 0;
    }
    // What lane b shares with lane b + 1. A run of lanes shares the least of its
    // neighbours' common pages.
    std::unique_ptr<Common[]> const common(new (std::nothrow) Common[num_lanes]);
    std::unique_ptr<Cut[]> const cuts(new (std::nothrow) Cut[std::size_t(num_lanes) + 1u]);
    if (common == nullptr || cuts == nullptr) {
        return 0;  // every lane by itself: the same results
    }
    for (std::uint32_t b = 0; b + 1u < num_lanes; ++b) {
        common[b] = commonPages(descs, lanes[b], lanes[b + 1u]);
        if (common[b].tokens < min_tokens) {
            common[b] = Common{};
        }
    }
    // The best sum of gains over the lanes in front of each cut. A group of two lanes
    // or more that could end or begin inside a run of equal neighbours gains no
    // less at one of the run's ends, so cuts inside are left out: 7 us for 32 lanes over
    // 2,048 tokens, 154 us for 2 x 64 over 32,749 (81,715 descriptors), on the host.
    std::uint32_t n = 0;
    cuts[n++] = Cut{0, 0, 0, 0, 0};
    for (std::uint32_t at = 1; at <= num_lanes; ++at) {
        bool const inside = min_lanes == 2u && at > 1u && at + 1u < num_lanes
            && common[at - 1u].pages == common[at - 2u].pages && common[at - 1u].pages == common[at].pages;
        if (inside) {
            continue;
        }
        Cut& cut = cuts[n];
        cut = Cut{at, at, cuts[n - 1u].gain, n - 1u, 0};  // no group ends here
        std::uint64_t least = ~std::uint64_t{0};  // tokens that the lanes from `from` on share
        for (std::uint32_t k = n; k-- > 0;) {
            std::uint32_t const from = cuts[k].at, to = cuts[k + 1u].at;
            if (to != at && common[to - 1u].tokens < least) {
                least = common[to - 1u].tokens;  // across the cut
            }
            if (to - from > 1u && common[from].tokens < least) {
                least = common[from].tokens;  // between the cuts: all equal
            }
            if (least == 0) {
                break;
            }
            // A group from here or further in front could end at `to` instead; no choice up to
            // there is worth more than that cut's gain, and the lanes behind it add no
            // more than this. Where that is too little the search is over. (2,048 lanes whose
            // neighbours all share different runs: 0.6 ms, 8.6 without this.)
            if (min_lanes == 2u && to != at && cuts[k + 1u].gain + (at - to) * (least + kReaderTokens) < cut.gain) {
                break;
            }
            if (at - from >= min_lanes) {
                std::uint64_t const gain = cuts[k].gain + (at - from - 1u) * (least + kReaderTokens);
                if (gain >= cut.gain) {
                    cut = Cut{at, from, gain, k, 0};
                }
            }
        }
        ++n;
    }
    // Back along the choices, then forward over the groups.
    std::uint32_t next = 0;
    for (std::uint32_t k = n - 1u; k != 0;) {
        std::uint32_t const before = cuts[k].before;
        cuts[k].next = next;
        next = k;
        k = before;
    }
    std::uint32_t found = 0;
    for (std::uint32_t k = next; k != 0 && found < max_groups; k = cuts[k].next) {
        std::uint32_t const from = cuts[k].from, end = cuts[k].at;
        if (from == end) {
            continue;
        }
        Common least = common[from];
        for (std::uint32_t b = from; b + 1u < end; ++b) {
            least = common[b].pages < least.pages ? common[b] : least;
        }
        std::uint32_t const count = static_cast<std::uint32_t>(least.tokens);
        groups[found++] = kk_prefix_group{lanes[from].desc_offset, least.pages, count, from, end - from, 0, 0, 0};
        for (std::uint32_t b = from; b < end; ++b) {
            lanes[b].desc_offset += least.pages;
            lanes[b].desc_count -= least.pages;
            lanes[b].token_count -= lanes[b].token_count < count ? lanes[b].token_count : count;
        }
    }
    return found;
}

int kk_prefix_attention_plan(const kk_page_desc* descs, uint32_t num_descs, kk_attn_lane* lanes, uint32_t num_lanes,
    kk_prefix_group* groups, uint32_t num_groups, uint32_t q_heads, uint32_t kv_heads, uint32_t num_sms,
    kk_prefix_item* items, uint32_t max_items, kk_prefix_plan* plan)
{
    using namespace kk;
    if (plan == nullptr || !headsServed(q_heads, kv_heads) || num_sms == 0 || (num_descs != 0 && descs == nullptr)
        || (num_lanes != 0 && lanes == nullptr) || (num_groups != 0 && groups == nullptr)
        || (max_items != 0 && items == nullptr)) {
        return KK_EINVAL;
    }
    *plan = kk_prefix_plan{0, 0, kOwnWarps, num_lanes, num_groups, num_descs, q_heads, kv_heads, 0};
    std::uint32_t const ratio = q_heads / kv_heads;
    auto outside = [&](std::uint32_t offset, std::uint32_t count) {
        return offset > num_descs || count > num_descs - offset;
    };
    // Tokens of a lane's own pages, in whole groups, stand in item_offset, and tiles
    // of a prefix in part_row, until the plan is made.
    std::uint64_t own_tokens = 0;
    for (std::uint32_t b = 0; b < num_lanes; ++b) {
        kk_attn_lane& ln = lanes[b];
        if (outside(ln.desc_offset, ln.desc_count)) {
            return KK_EINVAL;
        }
        ln.item_offset = ln.item_count = ln.reserved = 0;
        std::uint64_t tokens = 0;
        for (std::uint32_t e = ln.desc_offset; e < ln.desc_offset + ln.desc_count; ++e) {
            tokens += 8u * groupsOf(descs[e]);
        }
        if (tokens > 0xffffffffull) {
            return KK_EINVAL;
        }
        ln.item_offset = static_cast<std::uint32_t>(tokens);
        own_tokens += tokens;
    }
    auto tileNs = [](kk_prefix_group const& g) { return g.row_tiles > 1u ? kTilePairNs : kTileSingleNs; };
    double longest = 0.;
    for (std::uint32_t i = 0; i < num_groups; ++i) {
        kk_prefix_group& g = groups[i];
        if (outside(g.desc_offset, g.desc_count) || g.lane_begin > num_lanes
            || g.lane_count > num_lanes - g.lane_begin) {
            return KK_EINVAL;
        }
        std::uint64_t const row_tiles = (std::uint64_t(g.lane_count) * ratio + kTile - 1u) / kTile;
        if (row_tiles > 65535u) {
            return KK_EINVAL;
        }
        g.row_tiles = static_cast<std::uint32_t>(row_tiles);
        for (std::uint32_t b = g.lane_begin; b < g.lane_begin + g.lane_count; ++b) {
            if (lanes[b].reserved != 0) {
                return KK_EINVAL;
            }
            lanes[b].reserved = i + 1u;
        }
        g.part_row = walkTiles(descs, g.desc_offset, g.desc_offset + g.desc_count, [](std::uint32_t, std::uint32_t) {});
        longest = std::fmax(longest, kSharedNs + g.part_row * tileNs(g));
    }
    // The shortest time in which num_sms blocks, one to an SM, can do the work, or as
    // many rounds of them as take the least time in all.
    auto partsIn = [&](kk_prefix_group const& g, double ns) {
        double const most = std::fmax(1., std::floor((ns - kSharedNs) / tileNs(g)));
        return static_cast<std::uint32_t>(std::ceil(g.part_row / most));
    };
    auto taskTokensIn = [&](double ns) {
        return std::fmax(kOwnMinTokens, std::floor((ns - kOwnNs - kTaskNs) / kTaskTokenNs));
    };
    auto tasksOf = [&](double per_task) {
        double tasks = 0.;
        for (std::uint32_t b = 0; b < num_lanes; ++b) {
            tasks += std::ceil(lanes[b].item_offset / per_task) * kv_heads;
        }
        return tasks;
    };
    auto roundsIn = [&](double ns, double tasks) {  // items that a warp does one after the other
        double const tokens = static_cast<double>(own_tokens) * kv_heads;
        return std::fmax(1., std::floor((ns - kOwnNs) / (kTaskNs + kTaskTokenNs * tokens / tasks)));
    };
    auto ownBlocksIn = [&](double ns) {
        if (own_tokens == 0) {
            return 0.;
        }
        double const tasks = tasksOf(taskTokensIn(ns));
        double const tokens = static_cast<double>(own_tokens) * kv_heads;
        double const rounds = roundsIn(ns, tasks);
        return std::fmax(std::ceil(tasks / (rounds * kOwnWarps)),
            std::ceil(tokens * kOwnTokenNs / std::fmax(1., ns - kOwnNs - kTaskNs)));
    };
    auto sharedBlocksIn = [&](double ns) {
        double blocks = 0.;
        for (std::uint32_t i = 0; i < num_groups; ++i) {
            blocks += static_cast<double>(partsIn(groups[i], ns)) * kv_heads * ((groups[i].row_tiles + 1u) / 2u);
        }
        return blocks;
    };
    double const most_time = std::fmax(longest, kOwnNs + kTaskNs + kTaskTokenNs * 0x1p32);
    // One block per prefix, KV head and pair of row tiles, and one for the lanes' own
    // pages, are the fewest. Up to half of the SMs, the others are enough for own pages
    // (8 KV heads, 4 lanes with up to 1,000 tokens behind each prefix of 300, in one
    // round and in the best number: 10 prefixes 29.6 and 21.2 us, 16 prefixes 133 and 32).
    double const fewest = sharedBlocksIn(most_time) + (own_tokens != 0 ? 1. : 0.);
    double time = 0., waves = 0.;
    double const first_waves = std::fmax(1., std::ceil(fewest / num_sms));
    for (double w = first_waves; w < first_waves + 8.; ++w) {
        double lo = 0., hi = most_time;
        for (int i = 0; i < 48; ++i) {
            double const mid = 0.5 * (lo + hi);
            bool const done = mid >= kSharedNs && mid >= kOwnNs + kTaskNs
                && sharedBlocksIn(mid) + ownBlocksIn(mid) <= w * num_sms;
            (done ? hi : lo) = mid;
        }
        if (waves != 0. && w * hi >= waves * time) {
            break;
        }
        time = hi;
        waves = w;
        if (2. * fewest <= num_sms) {
            break;
        }
    }
    std::uint32_t count = 0;
    std::uint64_t part_rows = 0;
    auto put = [&](kk_prefix_item const& item) {
        if (count < max_items) {
            items[count] = item;
        }
        ++count;
    };
    for (std::uint32_t i = 0; i < num_groups; ++i) {
        kk_prefix_group& g = groups[i];
        std::uint32_t const tiles = g.part_row;
        std::uint32_t const parts = tiles != 0 ? partsIn(g, time) : 0u;
        g.part_row = g.part_count = 0;
        if (tiles == 0 || g.row_tiles == 0) {
            continue;
        }
        g.part_count = parts;
        std::uint64_t const rows = std::uint64_t(kv_heads) * parts * g.row_tiles * kTile;
        if (part_rows + rows > 0xffffffffull) {
            return KK_EINVAL;
        }
        g.part_row = static_cast<std::uint32_t>(part_rows);
        part_rows += rows;
        std::uint32_t part = 0, begin = g.desc_offset, before = 0;
        auto emit = [&](std::uint32_t end, std::uint32_t closed) {
            for (std::uint32_t h = 0; h < kv_heads; ++h) {
                for (std::uint32_t r = 0; r < g.row_tiles; r += 2u) {
                    put(kk_prefix_item{i, h, begin, end, part, static_cast<std::uint16_t>(r),
                        static_cast<std::uint16_t>(g.row_tiles - r > 1u ? 2u : 1u), closed - before,
                        g.part_row + ((h * parts + part) * g.row_tiles + r) * kTile, g.lane_begin, g.lane_count, 0, 0});
                }
            }
            ++part;
            begin = end;
            before = closed;
        };
        walkTiles(descs, g.desc_offset, g.desc_offset + g.desc_count, [&](std::uint32_t closed, std::uint32_t e) {
            if (closed == static_cast<std::uint32_t>(std::uint64_t(tiles) * (part + 1u) / parts)) {
                emit(e, closed);
            }
        });
        emit(g.desc_offset + g.desc_count, tiles);
    }
    plan->num_shared = count;
    if (own_tokens != 0) {
        // What the prefixes leave of the SMs, and no less than the plan set aside.
        std::uint32_t blocks = static_cast<std::uint32_t>(std::fmin(ownBlocksIn(time), 1e6));
        blocks = blocks < 1u ? 1u : blocks;
        double const left = std::fmin(waves * num_sms, 1e6) - count;
        blocks = blocks < left ? static_cast<std::uint32_t>(left) : blocks;
        // The shortest items that those blocks take in as many rounds.
        double const longest_task = taskTokensIn(time);
        double const room = std::floor(roundsIn(time, tasksOf(longest_task))) * blocks * kOwnWarps;
        double tokens = kOwnMinTokens;
        while (tokens < longest_task && tasksOf(tokens) > room) {
            tokens *= 1.125;
        }
        std::uint64_t const per_task = static_cast<std::uint64_t>(std::fmin(std::ceil(tokens), longest_task));
        for (std::uint32_t b = 0; b < num_lanes; ++b) {
            kk_attn_lane& ln = lanes[b];
            std::uint32_t const end = ln.desc_offset + ln.desc_count;
            std::uint64_t const len = ln.item_offset;
            ln.item_offset = 0;
            if (len == 0) {
                continue;
            }
            std::uint64_t const parts = (len + per_task - 1u) / per_task;
            ln.item_offset = static_cast<std::uint32_t>(part_rows);
            std::uint32_t begin = ln.desc_offset;
            std::uint64_t held = 0;
            // Cut i lies at the page boundary nearest to i / parts of the tokens.
            std::uint64_t seen = 0;
            auto goal = [&]() {
                return ln.item_count + 1u < parts ? len * (ln.item_count + 1u) / parts : ~std::uint64_t{0};
            };
            auto emit = [&](std::uint32_t to) {
                for (std::uint32_t h = 0; h < kv_heads; ++h) {
                    put(kk_prefix_item{b, h, begin, to, ln.item_count, 0, 0, 0,
                        static_cast<std::uint32_t>(part_rows) + h * ratio, 0, 0, ln.query_row, 0});
                }
                ++ln.item_count;
                part_rows += q_heads;
                begin = to;
                held = 0;
            };
            for (std::uint32_t e = ln.desc_offset; e < end; ++e) {
                std::uint64_t const more = 8u * groupsOf(descs[e]);
                if (held != 0 && seen + more > goal() && (seen >= goal() || seen + more - goal() > goal() - seen)) {
                    emit(e);
                }
                held += more;
                seen += more;
                if (seen >= goal()) {
                    emit(e + 1u);
                }
            }
            if (held != 0) {
                emit(end);
            } else {
                // Pages without tokens behind the last cut belong to the last items.
                for (std::uint32_t h = 0; begin != end && h < kv_heads; ++h) {
                    std::uint32_t const last = count - kv_heads + h;
                    if (last < max_items) {
                        items[last].desc_end = end;
                    }
                }
            }
            if (part_rows > 0xffffffffull) {
                return KK_EINVAL;
            }
        }
        std::uint32_t const tasks = count - plan->num_shared;
        std::uint32_t const per_cta = (tasks + blocks - 1u) / blocks;
        plan->tasks_per_cta = per_cta < kOwnWarps ? kOwnWarps : per_cta;
    }
    plan->num_items = count;
    plan->part_rows = part_rows;
    return 0;
}

uint64_t kk_prefix_attention_workspace_bytes(const kk_prefix_plan* plan)
{
    return plan == nullptr ? 0 : plan->part_rows * (kk::kHeadDim * 4u + 8u);
}

int kk_prefix_attention(const kk_prefix_attn_desc* d, void* stream)
{
    using namespace kk;
    auto misaligned = [](void const* p) { return p == nullptr || (reinterpret_cast<std::uintptr_t>(p) & 15u) != 0; };
    if (d == nullptr || d->pools.head_dim != kHeadDim || d->layer >= d->pools.layers
        || !headsServed(d->q_heads, d->pools.kv_heads) || !microPageTokensValid(d->pools)
        || d->pools.layers > (1u << 24) || d->plan.q_heads != d->q_heads || d->plan.kv_heads != d->pools.kv_heads
        || !(d->scale > 0.f) || !std::isfinite(d->scale) || d->plan.num_shared > d->plan.num_items
        || d->plan.tasks_per_cta == 0 || d->plan.part_rows > 0xffffffffull) {
        return KK_EINVAL;
    }
    if (d->plan.num_lanes == 0) {
        return 0;
    }
    std::uint64_t const q_row = std::uint64_t(d->q_heads) * kHeadDim;
    auto odd = [](void const* p) { return (reinterpret_cast<std::uintptr_t>(p) & 3u) != 0; };
    if (d->lanes == nullptr || odd(d->lanes) || odd(d->groups) || odd(d->items) || odd(d->descs) || misaligned(d->query) || misaligned(d->output) || d->query_stride % 8 != 0
        || d->output_stride % 8 != 0 || d->query_stride < q_row || d->output_stride < q_row
        || (d->plan.num_groups != 0 && d->groups == nullptr)
        || (d->plan.num_items != 0 && (d->items == nullptr || d->descs == nullptr))
        || (d->plan.part_rows != 0
            && (misaligned(d->workspace)
                || d->workspace_bytes < kk_prefix_attention_workspace_bytes(&d->plan)))) {
        return KK_EINVAL;
    }
    std::uint64_t const threads = std::uint64_t(d->plan.num_lanes) * d->q_heads * 32u;
    if (threads > 0xffffffffull) {
        return KK_EINVAL;
    }
    Args a{};
    a.micro_cap = microPageTokens(d->pools);
    a.micro = static_cast<__half const*>(d->pools.micro);
    a.extent = static_cast<__half const*>(d->pools.extent);
    std::uint64_t const row = std::uint64_t(d->pools.kv_heads) * kHeadDim;
    a.micro_page = std::uint64_t(d->pools.layers) * 2u * a.micro_cap * row;
    a.extent_page = std::uint64_t(d->pools.layers) * 2u * 64u * row;
    a.micro_slots = d->pools.micro == nullptr ? 0 : d->pools.micro_capacity;
    a.extent_slots = d->pools.extent == nullptr ? 0 : d->pools.extent_capacity;
    if ((a.micro_slots != 0 && misaligned(a.micro)) || (a.extent_slots != 0 && misaligned(a.extent))) {
        return KK_EINVAL;
    }
    a.layer = d->layer;
    a.kv_heads = d->pools.kv_heads;
    a.group = d->q_heads / d->pools.kv_heads;
    a.plan = d->plan;
    a.descs = d->descs;
    a.lanes = d->lanes;
    a.groups = d->groups;
    a.items = d->items;
    a.query = reinterpret_cast<__half const*>(d->query);
    a.output = reinterpret_cast<__half*>(d->output);
    a.query_stride = d->query_stride;
    a.output_stride = d->output_stride;
    a.scale_log2 = d->scale * 1.4426950408889634f;
    a.far_score = kFarLog2 / a.scale_log2;
    a.rescale_score = kRescale / a.scale_log2;
    a.part_o = static_cast<float*>(d->workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + d->plan.part_rows * kHeadDim);
    cudaStream_t const s = static_cast<cudaStream_t>(stream);
    if (d->plan.num_items != 0) {
        cudaError_t const e = allowSharedMemory();
        if (e != cudaSuccess) {
            return static_cast<int>(e);
        }
        Maps maps{};
        std::uint32_t const heads = d->pools.kv_heads;
        if (d->plan.num_shared != 0) {
            // A pool without pages keeps an empty map: no descriptor selects it.
            if ((a.micro_slots != 0
                    && (!encodePageHeadMap(&maps.micro8, a.micro, a.micro_slots, a.micro_cap, d->pools.layers, heads, 8)
                        || (a.micro_cap != 8u
                            && !encodePageHeadMap(&maps.micro, a.micro, a.micro_slots, a.micro_cap, d->pools.layers,
                                heads, a.micro_cap))))
                || (a.extent_slots != 0
                    && (!encodePageHeadMap(&maps.extent8, a.extent, a.extent_slots, 64, d->pools.layers, heads, 8)
                        || !encodePageHeadMap(&maps.extent, a.extent, a.extent_slots, 64, d->pools.layers, heads,
                            64)))) {
                return KK_EINVAL;
            }
            if (a.micro_cap == 8u) {
                maps.micro = maps.micro8;
            }
        }
        std::uint32_t const own = d->plan.num_items - d->plan.num_shared;
        std::uint64_t const grid = d->plan.num_shared
            + (std::uint64_t(own) + d->plan.tasks_per_cta - 1u) / d->plan.tasks_per_cta;
        if (grid > 0x7fffffffull) {
            return KK_EINVAL;
        }
        int const rc = static_cast<int>(launch(a.group <= 8u ? prefix_attention_kernel<1> : prefix_attention_kernel<2>,
            dim3(static_cast<unsigned>(grid)), dim3(kThreads), kSmemBytes, s, 1, maps, a));
        if (rc != 0) {
            return rc;
        }
    }
    // The joining launch is always a programmatic dependent of the first, if there is
    // one: its blocks are set up while the last items run, and wait for their end.
    bool const pdl = g_pdl_enabled;
    g_pdl_enabled = pdl || d->plan.num_items != 0;
    int const rc = static_cast<int>(launch(prefix_join_kernel,
        dim3(static_cast<unsigned>((threads + kJoinThreads - 1u) / kJoinThreads)), dim3(kJoinThreads), 0, s, 1, a));
    g_pdl_enabled = pdl;
    return rc;
}

} // extern "C"
