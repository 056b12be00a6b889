// Weight gradient of a projection whose input was kept in 8 bits: dW[n][k] = sum over tokens of dY[t][n] * X^[t][k], and the bias's, sum of dY[t][n].
//
// The product is D = X^^T dY on the tensor cores, M = inputs (features), N = outputs, summed over tokens; both operands lie in memory by tokens, which
// tcgen05 reads as they are. A pair of CTAs works on a tile of 256 features by 256 outputs, 64 tokens at a time: each CTA holds 128 features
// of X^ and 128 outputs of dY per step (32 KiB), the accumulators of its 128 features in tensor memory, twice, so that one tile is written while the
// next is summed. A pair halves what a tile reads: alone, a CTA with 128 x 256 would draw 80 bytes per cycle from L2 (32 KiB of dY
// and 8 KiB of codes every 512 cycles, which a step takes), the pair 48 per SM.
//
// Roles of a CTA's 16 warps: one thread copies dY and codes by TMA; one thread of the first CTA issues the products, and its counterpart in the second tells it that
// its dY has come; eight warps widen codes to 16-bit numbers, exactly (block8.cuh), straight into the swizzled operand (per 4 codes of bf16:
// two masks, two byte permutes and four two-wide products); four warps write finished tiles; two sum columns of dY
// for the bias out of shared memory, each tile of features for its own share of the steps, so that every step of dY is summed once; what the additions of
// steps round off is kept beside the sum (500,000 tokens of one sign, fp32: error 1.3e-5 -> 2e-7, in the same time).
//
// What bounds it is shared memory, and power: a step reads 32 KiB of operands, writes 16 KiB of dY, 8 KiB of codes and 16 KiB of widened X^, and reads the
// codes again; the products alone take three quarters of its time. So a long product has tiles of 256 x 512, for which a widened step of X^ serves twice
// (16384 x 4096 x 4096: 466 -> 395 us). They fill tensor memory, so that their epilogue stands alone: short products stay with 256 x 256.
//
// P pairs take P whole tiles at a time, as long as there are so many: they are at the same tokens then, and read them from L2 once one of them has.
// What is left is cut evenly, not by tiles: its steps stand in one row, and pair i takes steps [i S / P, (i+1) S / P). A tile that is
// cut is summed in pieces, in 32 bits in the workspace, and finish_kernel adds them in the order of tokens: the result does not depend on timing.
// (All tiles in one row: pairs are at different tokens, and 16384 x 4096 x 4096 draws 3.2 GB from HBM.) For the same reason, where there are fewer tiles than
// pairs, the pairs of all feature tiles go side by side through the outputs and tokens, as one group: dY is read once and not once for each.
//
// fp32: X^ is a bf16 number in any case, and dY is the exact sum of three (its 24 bits cut into eights; of a number below 2^-110 the last of them end
// under bf16's smallest), so three products of bf16 numbers with 32-bit accumulators give it in full. The tensor cores cut what an addition leaves below 24 bits, so the small parts are summed first, and the
// sums are added to those in memory, rounded, after every 1024 tokens: the error does not grow with the number of tokens as it would (8192 tokens:
// 7.5e-6 of the result's norm without either, 2.4e-6 with the leading part first).
//
// 16-bit types: an instruction cuts each of its 16 products at a quarter, and their sum with the accumulator at the whole, of the last of 24 bits (seen: products of
// 3/16 of it beside a 1 are lost, 16 of a quarter come through). Of a sum of one sign that takes 1.8e-4 in 65536 tokens and more than fp16's own rounding
// (4.9e-4) in 200,000. So their sums too are added to those in memory, rounded, but after every 16384 tokens: 7e-5 is lost, and at most
// 512 * 5 * 2^-23 = 3.1e-4, at any length. (65536 x 4096 x 4096 bf16: 1632 -> 1704 us; after every 8192 tokens 1786, and 16384 x 4096 x 4096 would go from 376 to 408.)
//
// dY that TMA cannot read (rows or address not at a multiple of 16 bytes) is copied first.
//
// 16384 x 4096 x 4096 bf16: 377 us and 17 for the pieces, 1.40 PFLOP/s, 0.85 of what a library product of 16-bit operands reaches in a burst; tensor pipe 0.78 busy.
// 8192 x 768 x 2304 fp32: 97 us, 0.44 busy (three products of every widened step, 27 us before them to lay dY out, 10 behind them). 1024 x 768 x 768: 12.5 + 6 us.
#include "kernels/sm100/weight_grad.h"

#include "core/check.h"
#include "kernels/sm100/block8.cuh"
#include "kernels/sm100/launch.h"
#include "kernels/sm100/tcgen05.cuh"
#include "mem/cu_driver.h"

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <mutex>
#include <stdexcept>
#include <type_traits>

namespace b200ccl::kernels {

using namespace b200ccl::dev;

namespace {

using u64 = unsigned long long;

constexpr unsigned kTile = 256;       // features and outputs of a pair's tile
constexpr unsigned kHalf = 128;       // of one CTA
constexpr unsigned kStep = 64;        // tokens
constexpr unsigned kDepth = 6;        // steps whose dY is in shared memory or on the way; half as many of wide tiles
constexpr unsigned kBlockBytes = kStep * 128;         // 64 elements of every token of a step
constexpr unsigned kOperandBytes = 2 * kBlockBytes;   // a CTA's half of an operand
constexpr unsigned kCodeBytes = kStep * kHalf;
constexpr unsigned kThreads = 512;
constexpr unsigned kFirstTransformWarp = 4, kFirstEpilogueWarp = 12;
// Transform warps: a group widens every fourth step, from codes at a place of its own into an operand of its own. (Its own, because a wait tells a phase
// from the one before it only: whoever waits on a barrier has to have seen every phase of it.)
constexpr unsigned kGroups = 4, kGroupWarps = 2;
constexpr unsigned kChunkSteps = 16;  // fp32: steps of each part between two additions to the sums in memory
constexpr unsigned kLongSteps = 256;  // 16-bit types: steps between two additions to the sums in memory, see above
constexpr unsigned kMaxPairs = 74;    // 148 SMs
constexpr unsigned kTurnBytes = 32 * 32 * 4;  // of an epilogue warp: 32 outputs of its 32 features
// Shared memory, from a multiple of 1024 bytes on: dY of the stages, X^ of the groups, their codes, what the epilogue turns, barriers.
constexpr unsigned kAtX = kDepth * kOperandBytes, kAtCodes = kAtX + kGroups * kOperandBytes, kAtTurn = kAtCodes + kGroups * kCodeBytes,
                   kAtBarriers = kAtTurn + 4 * kTurnBytes;
constexpr unsigned kShared = kAtBarriers + 512 + 1024;
static_assert(kShared <= 227 * 1024);

struct alignas(64) WeightGradArgs {
    CUtensorMap dy;     // [parts][tokens][outputs]
    CUtensorMap codes;  // [1][tokens][pitch]
    const unsigned char* scales;
    void* out;
    float* pieces;     // [2 * pairs][outputs of a tile][256 features]
    float* bias;       // [tiles + pairs][outputs of a tile], or null
    void* bias_out;    // or its gradient itself, where no tile is cut: the first tile of features sums all steps
    unsigned* status;  // host memory
    u64 wait_ns;       // limit of a wait
    u64 pitch;         // bytes of a token's codes
    bool wide;         // rows of `out` start at multiples of 16 bytes
    unsigned tokens, inputs, outputs;
    unsigned feature_tiles, parts, steps_of_part, steps_of_tile;
    unsigned pairs, waves;  // of whole tiles
    unsigned group;         // pairs side by side in the tiles that are left, each with a tile of its own
    unsigned groups;        // that share them
    unsigned steps;         // of one such row of tiles that are left
};

struct FinishArgs {
    void* out;
    void* bias_out;
    const float* pieces;
    const float* bias;
    unsigned inputs, outputs, width, feature_tiles, steps_of_tile, steps, group, groups;  // width: outputs of a tile
    unsigned whole_tiles;  // that come before those that are shared out
    unsigned piece_ctas;   // CTAs that add pieces; the others make the bias's gradient
};

// pair * steps / pairs, in 32 bits: pairs are few.
__host__ __device__ inline unsigned first_step(unsigned pair, unsigned steps, unsigned pairs) {
    const unsigned each = steps / pairs;
    return pair * each + pair * (steps - each * pairs) / pairs;
}

// Barriers of a CTA, in its shared memory.
struct Barriers {
    u64 dy[kDepth];       // this CTA's dY of a stage has come
    u64 dy_other[kDepth]; // first CTA: the other's has
    u64 empty[kDepth];    // it has been read
    u64 codes[kGroups];        // this CTA's codes of a group have come
    u64 codes_empty[kGroups];  // they have been read
    u64 x[kGroups];        // first CTA: both CTAs' X^ of a group is written
    u64 x_empty[kGroups];  // it has been read
    u64 sums[2];           // accumulators are complete
    u64 sums_free[2];      // first CTA: both CTAs have written theirs out
    u64 drained;           // all products are done
    unsigned tmem;
    unsigned failed;
};

__device__ __forceinline__ void store_shared16(unsigned at, unsigned a, unsigned b, unsigned c, unsigned d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 load_shared16(unsigned at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ unsigned load_shared4(unsigned at) {
    unsigned v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

// What a pair does, in order: `waves` whole tiles, then its steps of the tiles that are left.
struct Share {
    unsigned pair, group, begin, end;  // in the row of steps that are left
    unsigned whole, all;        // steps of its whole tiles, of everything
};
__device__ __forceinline__ Share share_of(const WeightGradArgs& a, unsigned pair) {
    Share s;
    s.pair = pair;
    s.group = pair / a.group;
    s.begin = first_step(min(s.group, a.groups), a.steps, a.groups);
    s.end = first_step(min(s.group + 1u, a.groups), a.steps, a.groups);
    s.whole = a.waves * a.steps_of_tile;
    s.all = s.whole + (s.end - s.begin);
    return s;
}
// Its n-th step.
struct Where {
    unsigned tile, k;
};
__device__ __forceinline__ Where where_is(const WeightGradArgs& a, const Share& s, unsigned n) {
    const bool whole = n < s.whole;
    const unsigned at = whole ? n : s.begin + (n - s.whole), row = at / a.steps_of_tile;
    return {whole ? row * a.pairs + s.pair : a.waves * a.pairs + row * a.group + (s.pair - s.group * a.group), at - row * a.steps_of_tile};
}
// A run of steps of one tile, from its n-th step on.
struct Piece {
    unsigned tile, from, to;  // steps of the tile
    bool whole;               // this pair sums all of the tile
    bool later;               // not the pair's first step of the tile
    unsigned slot;            // of the sums in memory: of a piece, or of a whole tile that is not done (a pair's last piece comes after its whole tiles)
};
__device__ __forceinline__ Piece piece_at(const WeightGradArgs& a, const Share& s, unsigned n) {
    const Where w = where_is(a, s, n);
    Piece p;
    p.tile = w.tile;
    p.from = w.k;
    p.to = min(a.steps_of_tile, w.k + (s.all - n));
    if (n < s.whole) {
        p.whole = true;
        p.later = w.k != 0;
        p.slot = 2u * s.pair + 1u;
    } else {
        const unsigned tile_at = s.begin + (n - s.whole) - w.k;  // in the row of steps
        p.whole = tile_at >= s.begin && tile_at + a.steps_of_tile <= s.end;
        p.later = w.k != 0 && n != s.whole;
        p.slot = 2u * s.pair + (tile_at <= s.begin ? 0u : 1u);
    }
    return p;
}
// The part of a piece that is summed on the tensor cores alone: 256 steps, fp32 sixteen of each part of dY.
__device__ __forceinline__ Piece segment_at(const WeightGradArgs& a, const Share& s, unsigned n) {
    Piece p = piece_at(a, s, n);
    const unsigned chunk = a.parts > 1 ? a.parts * kChunkSteps : kLongSteps;
    p.to = min(p.to, (p.from / chunk + 1u) * chunk);
    return p;
}
// Which part of dY, and which 64 tokens, step k of a tile takes: sixteen steps of the last part, whose sums are smallest, the same ones of the one before,
// then of the leading one.
struct Spot {
    unsigned part, step;
};
__device__ __forceinline__ Spot spot_of(const WeightGradArgs& a, unsigned k) {
    if (a.parts == 1) return {0u, k};
    const unsigned chunk = k / (a.parts * kChunkSteps), in_chunk = k - chunk * (a.parts * kChunkSteps);
    const unsigned length = min(kChunkSteps, a.steps_of_part - chunk * kChunkSteps), part = in_chunk / length;
    return {a.parts - 1u - part, chunk * kChunkSteps + in_chunk - part * length};
}

// sum + v, and to `low` what that rounds off (exactly, whichever is larger).
__device__ __forceinline__ void add_exactly(float& sum, float& low, float v) {
    const float s = sum + v, of_v = s - sum;
    low += (sum - (s - of_v)) + (v - of_v);
    sum = s;
}
// (What is rounded off an infinity is NaN.)
__device__ __forceinline__ float with_low(float sum, float low) { return (__float_as_uint(sum) & 0x7f800000u) != 0x7f800000u ? sum + low : sum; }

// Writes 32 outputs of a warp's 32 features, f[j] being output j of feature `lane`, to rows of `stride` elements at `to` (its feature 0): turned in
// shared memory so that every lane stores 16 bytes of a row (a row per store and lane made an epilogue of 8 us for a tile). Only the first `rows` rows and
// `columns` elements are there. later: added to what is there (32 bits).
template <typename T>
__device__ __forceinline__ void put(const float (&f)[32], unsigned turn, T* to, u64 stride, unsigned rows, unsigned columns, bool later) {
    constexpr unsigned kWide = 16 / sizeof(T), kLanes = 32 / kWide, kRows = 32 / kLanes;  // lanes of a row, rows of a store
    const unsigned lane = threadIdx.x & 31u, row = lane / kLanes, column = lane % kLanes * kWide;
    const bool mine = column < columns;  // (columns are whole 16 bytes)
    to += (u64)row * stride + column;
    float4 old[sizeof(T) == 4 ? 32 / kRows : 1];
    if constexpr (sizeof(T) == 4) {
        if (later) {
#pragma unroll
            for (unsigned i = 0; i < 32 / kRows; ++i)
                old[i] = mine && row + i * kRows < rows ? *reinterpret_cast<const float4*>(to + i * kRows * stride) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
#pragma unroll
    for (unsigned j = 0; j < 32; ++j) {
        if constexpr (sizeof(T) == 4) {
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(turn + j * 128u + lane * 4u), "r"(__float_as_uint(f[j])) : "memory");
        } else {
            const T v = Elem<T>::from_f(f[j]);
            asm volatile("st.shared.b16 [%0], %1;" ::"r"(turn + j * 64u + lane * 2u), "h"(*reinterpret_cast<const unsigned short*>(&v)) : "memory");
        }
    }
    __syncwarp();
#pragma unroll
    for (unsigned i = 0; i < 32 / kRows; ++i) {
        if (mine && row + i * kRows < rows) {
            uint4 v = load_shared16(turn + i * 512u + lane * 16u);
            if constexpr (sizeof(T) == 4) {
                if (later)
                    v = make_uint4(__float_as_uint(__uint_as_float(v.x) + old[i].x), __float_as_uint(__uint_as_float(v.y) + old[i].y),
                                   __float_as_uint(__uint_as_float(v.z) + old[i].z), __float_as_uint(__uint_as_float(v.w) + old[i].w));
            }
            *reinterpret_cast<uint4*>(to + i * kRows * stride) = v;
        }
    }
    __syncwarp();
}

// The same to the gradient: 32 outputs from `output` on, of which `there` are there, of the warp's features from `feature` on.
template <typename T>
__device__ __forceinline__ void put_out(const WeightGradArgs& a, float (&f)[32], unsigned turn, unsigned feature, unsigned output, unsigned there, bool later) {
    const unsigned lane = threadIdx.x & 31u;
    if (a.wide) {
        put<T>(f, turn, static_cast<T*>(a.out) + (u64)output * a.inputs + feature, a.inputs, there, a.inputs - feature, later);
    } else if (feature + lane < a.inputs) {
        T* out = static_cast<T*>(a.out) + (u64)output * a.inputs + feature + lane;
#pragma unroll
        for (unsigned j = 0; j < 32; ++j) {
            if (j < there) {
                if constexpr (sizeof(T) == 4) f[j] += later ? out[(u64)j * a.inputs] : 0.0f;
                out[(u64)j * a.inputs] = Elem<T>::from_f(f[j]);
            }
        }
    }
}

// 16-bit types: what was summed of a whole tile of a long sum, to the sums in memory, where each lane finds what it left (four outputs of its feature, beside
// those of the next), or with them to the gradient. (Apart, because in the loop below it costs a short call 0.3 us.)
template <typename T, unsigned kWidth>
__device__ __noinline__ void add_long_sum(const WeightGradArgs& a, const Piece& p, unsigned columns, unsigned turn, unsigned in_tile) {
    const unsigned feature = (p.tile % a.feature_tiles) * kTile + in_tile, output0 = (p.tile / a.feature_tiles) * kWidth;
    const unsigned outputs = feature < a.inputs ? min(kWidth, a.outputs - output0) : 0u;
    for (unsigned c = 0; c < outputs; c += 32u) {
        float f[32];
        __syncwarp();
        tmem_load32(columns + c, f);
        float4* sums = reinterpret_cast<float4*>(a.pieces + (u64)p.slot * (kWidth * kTile)) + c / 4u * kTile + in_tile + (threadIdx.x & 31u);
        if (p.later) {
            float4 old[8];
#pragma unroll
            for (unsigned j = 0; j < 8; ++j) old[j] = sums[j * kTile];
#pragma unroll
            for (unsigned j = 0; j < 8; ++j) { f[4 * j] += old[j].x; f[4 * j + 1] += old[j].y; f[4 * j + 2] += old[j].z; f[4 * j + 3] += old[j].w; }
        }
        if (p.to != a.steps_of_tile) {
#pragma unroll
            for (unsigned j = 0; j < 8; ++j) sums[j * kTile] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
        } else {
            put_out<T>(a, f, turn, feature, output0 + c, min(32u, outputs - c), false);
        }
    }
}

// After a wait that ran out: all that this CTA's pair was to write is NaN (its own half of the features and of the bias), so that whoever reads it sees it.
template <typename T, bool kBias, unsigned kWidth>
__device__ __noinline__ void spoil(const WeightGradArgs& a, const Share& share, unsigned rank) {
    const float nan = __uint_as_float(0x7fffffffu);
    const unsigned column = threadIdx.x % kHalf, row0 = threadIdx.x / kHalf;
    constexpr unsigned kRows = kThreads / kHalf;
    for (unsigned n = 0; n < share.all;) {
        const Piece p = piece_at(a, share, n);
        const unsigned feature = (p.tile % a.feature_tiles) * kTile + rank * kHalf + column, output0 = (p.tile / a.feature_tiles) * kWidth;
        for (unsigned r = row0; r < kWidth; r += kRows) {
            if (!p.whole) a.pieces[((u64)p.slot * kWidth + r) * kTile + rank * kHalf + column] = nan;
            else if (feature < a.inputs && output0 + r < a.outputs) static_cast<T*>(a.out)[(u64)(output0 + r) * a.inputs + feature] = Elem<T>::from_f(nan);
        }
        if constexpr (kBias) {
            for (unsigned b = row0; b < kWidth / kTile; b += kRows) {
                const unsigned output = b * kTile + rank * kHalf + column;
                if (a.bias_out == nullptr)
                    a.bias[(u64)(p.from == 0 ? p.tile : a.feature_tiles * ((a.outputs + kWidth - 1) / kWidth) + share.pair) * kWidth + output] = nan;
                else if (p.tile % a.feature_tiles == 0 && output0 + output < a.outputs) static_cast<T*>(a.bias_out)[output0 + output] = Elem<T>::from_f(nan);
            }
        }
        n += p.to - p.from;
    }
}

// T: type of dY and the gradients. kBias: also columns of dY. kWide: tiles of 512 outputs (16-bit types).
template <typename T, bool kBias, bool kWide>
__global__ void __launch_bounds__(kThreads, 1) weight_grad_kernel(const __grid_constant__ WeightGradArgs a) {
    constexpr unsigned kBlocks = kWide ? 2 : 1, kWidth = kBlocks * kTile;  // blocks of 256 outputs, outputs of a tile
    constexpr unsigned kStages = kWide ? kDepth / 2 : kDepth, kDyBytes = kBlocks * kOperandBytes;
    constexpr unsigned kBuffers = kWide ? 1 : 2;                           // sets of accumulators, in turn
    constexpr bool kBf16 = !std::is_same_v<T, __half>;
    using Operand = std::conditional_t<kBf16, __nv_bfloat16, __half>;
    extern __shared__ unsigned char raw[];
    // Swizzled operands start at multiples of 1024 bytes; the same place in both CTAs.
    unsigned char* shared = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    Barriers& bars = *reinterpret_cast<Barriers*>(shared + kAtBarriers);
    volatile unsigned* failed = &bars.failed;
    const unsigned base = smem_addr(shared);
    const unsigned warp = threadIdx.x / 32u, lane = threadIdx.x & 31u;
    const unsigned rank = cluster_rank();
    const Share share = share_of(a, blockIdx.x / 2u);

    if (warp == 0 && lane == 0) {
        for (unsigned s = 0; s < kStages; ++s) {
            mbar_init(&bars.dy[s], 1);
            mbar_init(&bars.dy_other[s], 1);
            mbar_init(&bars.empty[s], 1 + (kBias ? 2 : 0));
        }
        for (unsigned i = 0; i < kGroups; ++i) {
            mbar_init(&bars.codes[i], 1);
            mbar_init(&bars.codes_empty[i], kGroupWarps);
            mbar_init(&bars.x[i], 2 * kGroupWarps);
            mbar_init(&bars.x_empty[i], 1);
        }
        for (unsigned i = 0; i < kBuffers; ++i) {
            mbar_init(&bars.sums[i], 1);
            mbar_init(&bars.sums_free[i], 8);
        }
        mbar_init(&bars.drained, 1);
        bars.failed = 0;
        mbar_fence_init();
        tma_prefetch_map(&a.dy);
        tma_prefetch_map(&a.codes);
    }
    __syncwarp();
    if (warp == 1) tmem_alloc_pair(smem_addr(&bars.tmem), 2 * kTile);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tcgen05_fence_before();
    cluster_sync();
    tcgen05_fence_after();
    const unsigned tmem = bars.tmem;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const auto bar = [](u64& b) { return smem_addr(&b); };
    if (warp == 0) {
        if (lane == 0) {
            unsigned n = 0, asked = 0;  // steps whose dY, and whose codes, have been asked for
            bool ok = true;
            while (n < share.all && ok) {
                const Piece p = piece_at(a, share, n);
                const int output = (int)((p.tile / a.feature_tiles) * kWidth + rank * kHalf);
                const int feature = (int)((p.tile % a.feature_tiles) * kTile + rank * kHalf);
                for (unsigned k = p.from; k < p.to; ++k, ++n) {
                    const unsigned s = n % kStages, group = n % kGroups;
                    const Spot spot = spot_of(a, k);
                    ok = wait_phase(bar(bars.codes_empty[group]), ((n / kGroups) & 1u) ^ 1u, failed, a.wait_ns);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&bars.codes[group], kCodeBytes);
                    tma_load_box(base + kAtCodes + group * kCodeBytes, &a.codes, feature, (int)(spot.step * kStep), 0, bar(bars.codes[group]));
                    ++asked;
                    ok = wait_phase(bar(bars.empty[s]), ((n / kStages) & 1u) ^ 1u, failed, a.wait_ns);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&bars.dy[s], kDyBytes);
#pragma unroll
                    for (unsigned b = 0; b < 2 * kBlocks; ++b)  // 64 outputs each
                        tma_load_box(base + s * kDyBytes + b * kBlockBytes, &a.dy, output + (int)(b / 2 * kTile + b % 2 * 64), (int)(spot.step * kStep),
                                     (int)spot.part, bar(bars.dy[s]));
                }
            }
            // Stages have been given back, and after a failure copies have landed, before the CTA ends.
            for (unsigned i = n > kStages ? n - kStages : 0; i < n; ++i) {
                if (ok) wait_phase(bar(bars.empty[i % kStages]), (i / kStages) & 1u, failed, a.wait_ns);
                for (unsigned polls = 0; polls < 1000u && !phase_over<false>(bar(bars.dy[i % kStages]), (i / kStages) & 1u); ++polls) {}
            }
            for (unsigned i = asked > kGroups ? asked - kGroups : 0; i < asked; ++i)
                for (unsigned polls = 0; polls < 1000u && !phase_over<false>(bar(bars.codes[i % kGroups]), (i / kGroups) & 1u); ++polls) {}
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const unsigned shape = product_by_rows(kTile, kTile, kBf16);
            unsigned n = 0, pieces = 0;
            bool ok = true;
            for (; n < share.all && ok; ++pieces) {
                const Piece p = segment_at(a, share, n);
                const unsigned buffer = pieces % kBuffers;
                ok = wait_phase<true>(bar(bars.sums_free[buffer]), ((pieces / kBuffers) & 1u) ^ 1u, failed, a.wait_ns);
                if (!ok) break;
                tcgen05_fence_after();
                for (unsigned k = p.from; k < p.to; ++k, ++n) {
                    const unsigned s = n % kStages, parity = (n / kStages) & 1u, group = n % kGroups;
                    ok = wait_phase(bar(bars.dy[s]), parity, failed, a.wait_ns) && wait_phase<true>(bar(bars.dy_other[s]), parity, failed, a.wait_ns) &&
                         wait_phase<true>(bar(bars.x[group]), (n / kGroups) & 1u, failed, a.wait_ns);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const std::uint64_t x = operand_by_rows(base + kAtX + group * kOperandBytes, kBlockBytes);
#pragma unroll
                    for (unsigned b = 0; b < kBlocks; ++b) {
                        const std::uint64_t dy = operand_by_rows(base + s * kDyBytes + b * kOperandBytes, kBlockBytes);
#pragma unroll
                        for (unsigned i = 0; i < kStep / 16; ++i)  // 16 tokens are 2048 bytes
                            mma_pair(tmem + (buffer + b) * kTile, x + i * (2048 >> 4), dy + i * (2048 >> 4), shape, k > p.from || i > 0);
                    }
                    commit_pair(bar(bars.x_empty[group]));
                    commit_pair(bar(bars.empty[s]));
                }
                if (!ok) break;
                commit_pair(bar(bars.sums[buffer]));
            }
            // Products under way read shared memory and write tensor memory of both CTAs. Where a wait ran out, nobody else may be waiting for them.
            commit_pair(bar(bars.drained));
            for (unsigned polls = 0; polls < 1000u && !phase_over<false>(bar(bars.drained), 0); ++polls) {}
        } else if (lane == 0) {
            for (unsigned n = 0; n < share.all; ++n) {
                if (!wait_phase(bar(bars.dy[n % kStages]), (n / kStages) & 1u, failed, a.wait_ns)) break;
                mbar_arrive_at(bar(bars.dy_other[n % kStages]), 0);
            }
            if (!wait_phase(bar(bars.drained), 0, failed, a.wait_ns))
                for (unsigned polls = 0; polls < 1000u && !phase_over<false>(bar(bars.drained), 0); ++polls) {}
        }
    } else if (warp < kFirstTransformWarp) {
        if constexpr (kBias) {
            const unsigned column = (warp - 2u) * 64u + lane * 2u;  // of this CTA's 128 outputs
            unsigned n = 0;
            bool ok = true;
            while (n < share.all && ok) {
                const Piece p = piece_at(a, share, n);
                const unsigned turn = p.tile % a.feature_tiles;
                float2 sum[kBlocks], low[kBlocks];  // low: what the additions to sum rounded off
#pragma unroll
                for (unsigned b = 0; b < kBlocks; ++b) sum[b] = low[b] = make_float2(0.0f, 0.0f);
                for (unsigned k = p.from; k < p.to; ++k, ++n) {
                    const unsigned s = n % kStages;
                    ok = __all_sync(0xffffffffu, wait_phase(bar(bars.dy[s]), (n / kStages) & 1u, failed, a.wait_ns));
                    if (!ok) break;
                    if (a.bias_out != nullptr ? turn == 0u : k % a.feature_tiles == turn) {
#pragma unroll
                        for (unsigned b = 0; b < kBlocks; ++b) {
                            const unsigned from = base + s * kDyBytes + b * kOperandBytes + (warp - 2u) * kBlockBytes;
                            // Sixteen tokens, four times, then to the sum of all: an error of at most 20 roundings, however many tokens there are.
                            float2 step = make_float2(0.0f, 0.0f);
#pragma unroll
                            for (unsigned t0 = 0; t0 < kStep; t0 += 16) {
                                float2 some = make_float2(0.0f, 0.0f);
#pragma unroll
                                for (unsigned t = 0; t < 16; ++t) {
                                    const unsigned w = load_shared4(from + (t0 + t) * 128u + (((lane / 4u) ^ (t & 7u)) * 16u) + (lane & 3u) * 4u);
                                    const float2 f = kBf16 ? b2_to_f2(w) : h2_to_f2(w);
                                    some.x += f.x;
                                    some.y += f.y;
                                }
                                step.x += some.x;
                                step.y += some.y;
                            }
                            add_exactly(sum[b].x, low[b].x, step.x);
                            add_exactly(sum[b].y, low[b].y, step.y);
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(bars.empty[s]));
                }
                if (!ok) break;
#pragma unroll
                for (unsigned b = 0; b < kBlocks; ++b) sum[b] = make_float2(with_low(sum[b].x, low[b].x), with_low(sum[b].y, low[b].y));
                if (a.bias_out != nullptr) {
                    if (turn != 0u) continue;
                    const unsigned output = (p.tile / a.feature_tiles) * kWidth + rank * kHalf + column;
#pragma unroll
                    for (unsigned b = 0; b < kBlocks; ++b) {
                        T* out = static_cast<T*>(a.bias_out) + output + b * kTile;
                        if (output + b * kTile < a.outputs) out[0] = Elem<T>::from_f(sum[b].x);
                        if (output + b * kTile + 1u < a.outputs) out[1] = Elem<T>::from_f(sum[b].y);
                    }
                    continue;
                }
                float* to = a.bias + (u64)(p.from == 0 ? p.tile : a.feature_tiles * ((a.outputs + kWidth - 1) / kWidth) + share.pair) * kWidth;
#pragma unroll
                for (unsigned b = 0; b < kBlocks; ++b) *reinterpret_cast<float2*>(to + b * kTile + rank * kHalf + column) = sum[b];
            }
        }
    } else if (warp < kFirstEpilogueWarp) {
        const unsigned group = (warp - kFirstTransformWarp) / kGroupWarps;
        const unsigned tid = threadIdx.x & (kGroupWarps * 32u - 1u);
        const unsigned chunk = tid & 7u, row = tid >> 3;  // 16 features of the tokens row, row + 8, ... of a step
        // Scales are read a turn of the group ahead, straight from memory (a step's are 4 bytes of each of 64 tokens).
        unsigned scale[8];
        const auto load_scales = [&](unsigned n) {
            const Where w = where_is(a, share, n);
            const u64 token = (u64)spot_of(a, w.k).step * kStep + row;
            const unsigned feature = (w.tile % a.feature_tiles) * kTile + rank * kHalf + chunk * 16u;
            const unsigned char* from = a.scales + (token * a.pitch + feature) / kBlock8;
#pragma unroll
            for (unsigned u = 0; u < 8; ++u)
                scale[u] = token + 8u * u < a.tokens && feature < a.pitch ? from[8u * u * (a.pitch / kBlock8)] : 127u;
        };
        if (group < share.all) load_scales(group);
        // A chunk's two halves go to columns of 16 bytes, the odd one first for the second block of 64 features: eight lanes then write to eight
        // different columns of the shared memory's banks. (Eight tokens are 1024 bytes, so the swizzle is the same for all of a lane's.)
        const unsigned odd = chunk >> 2, column = (chunk & 3u) * 2u;
        const unsigned block = base + kAtX + group * kOperandBytes + odd * kBlockBytes + row * 128u;
        const unsigned first = block + (((column + odd) ^ row) * 16u), second = block + (((column + (odd ^ 1u)) ^ row) * 16u);
        const unsigned codes = base + kAtCodes + group * kCodeBytes + row * kHalf + chunk * 16u;
        unsigned n = group;
        for (; n < share.all; n += kGroups) {
            const unsigned parity = (n / kGroups) & 1u;
            if (!__all_sync(0xffffffffu, wait_phase(bar(bars.codes[group]), parity, failed, a.wait_ns) && wait_phase(bar(bars.x_empty[group]), parity ^ 1u, failed, a.wait_ns)))
                break;
#pragma unroll
            for (unsigned u = 0; u < 8; ++u) {
                const uint4 c = load_shared16(codes + u * (8u * kHalf));
                const unsigned s2 = step16<Operand>(scale[u]);
                const uint2 w0 = widen8x4<Operand>(odd ? c.z : c.x, s2), w1 = widen8x4<Operand>(odd ? c.w : c.y, s2);
                const uint2 w2 = widen8x4<Operand>(odd ? c.x : c.z, s2), w3 = widen8x4<Operand>(odd ? c.y : c.w, s2);
                store_shared16(first + u * 1024u, w0.x, w0.y, w1.x, w1.y);
                store_shared16(second + u * 1024u, w2.x, w2.y, w3.x, w3.y);
            }
            fence_shared_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_at(bar(bars.x[group]), 0);
                mbar_arrive(bar(bars.codes_empty[group]));
            }
            if (n + kGroups < share.all) load_scales(n + kGroups);  // (before the fence, the fence would wait for them)
        }
        // The arrival that gives the operand back comes before the CTA ends.
        if (n >= share.all && n != group) wait_phase(bar(bars.x_empty[group]), (n / kGroups - 1u) & 1u, failed, a.wait_ns);
    } else {
        const unsigned quarter = warp & 3u;  // lanes of tensor memory that this warp reaches
        const unsigned in_tile = rank * kHalf + quarter * 32u;
        const unsigned turn = base + kAtTurn + quarter * kTurnBytes;
        unsigned pieces = 0, n = 0;
        for (; n < share.all; ++pieces) {
            const Piece p = segment_at(a, share, n);
            const unsigned buffer = pieces % kBuffers;
            if (!__all_sync(0xffffffffu, wait_phase(bar(bars.sums[buffer]), (pieces / kBuffers) & 1u, failed, a.wait_ns))) break;
            tcgen05_fence_after();
            const unsigned feature = (p.tile % a.feature_tiles) * kTile + in_tile;
            const unsigned output0 = (p.tile / a.feature_tiles) * kWidth;
            float* piece = a.pieces + (u64)p.slot * (kWidth * kTile) + in_tile;
            const unsigned outputs = feature < a.inputs ? min(kWidth, a.outputs - output0) : 0u;  // of the tile, that this warp has to write
            if (sizeof(T) == 2 && p.whole && (p.later || p.to != a.steps_of_tile)) {
                add_long_sum<T, kWidth>(a, p, tmem + buffer * kTile + (quarter * 32u << 16), turn, in_tile);
            } else {
                for (unsigned c = 0; c < outputs; c += 32u) {
                    float f[32];
                    __syncwarp();
                    tmem_load32(tmem + buffer * kTile + c + (quarter * 32u << 16), f);
                    if (p.whole) put_out<T>(a, f, turn, feature, output0 + c, min(32u, outputs - c), p.later);
                    else put<float>(f, turn, piece + (u64)c * kTile, kTile, 32u, kTile, p.later);
                }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_at(bar(bars.sums_free[buffer]), 0);
            n += p.to - p.from;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && *failed != 0u) {
        *static_cast<volatile unsigned*>(a.status) = 1u;
        store_word_at(smem_addr(&bars.failed), rank ^ 1u, 1u);
    }
    __syncwarp();
    tcgen05_fence_before();
    cluster_sync();  // nothing of this CTA is read or arrived at by the other any more
    tcgen05_fence_after();
    __syncwarp();
    if (warp == 1) tmem_free_pair(tmem, 2 * kTile);
    if (*failed != 0u) {
        spoil<T, kBias, kWidth>(a, share, rank);
        if (rank == 1 && threadIdx.x == 0)  // (the last arrival from the first CTA)
            for (unsigned polls = 0; polls < 1000u && !phase_over<false>(bar(bars.drained), 0); ++polls) {}
    }
}

// Adds the pieces of cut tiles, and the bias's. kRows: rows of a thread, four outputs of a CTA for each. One where there are few tiles, whose
// pieces are many: eight loads of a thread are on the way at a time either way (two tiles of 37 pieces, 15126 x 320 x 61 fp32: 22 us less than one piece after another).
template <typename T, unsigned kRows>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ FinishArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x < a.piece_ctas) {
        const unsigned parts = a.width / (4u * kRows), index = blockIdx.x / parts, part = blockIdx.x % parts;
        const unsigned row = index / a.group, member = index % a.group, tile = a.whole_tiles + index;
        const unsigned from = row * a.steps_of_tile, to = from + a.steps_of_tile;
        // Its groups of pairs, in the order of tokens; a pair's last tile, if it began before it, is its second piece.
        const unsigned first = (unsigned)((u64)from * a.groups / a.steps);
        __shared__ unsigned slots[kMaxPairs + 8];
        unsigned count = 0;
        if (threadIdx.x < kMaxPairs + 8u) {
            const unsigned group = first + threadIdx.x;
            const unsigned begin = first_step(min(group, a.groups), a.steps, a.groups), end = first_step(min(group + 1u, a.groups), a.steps, a.groups);
            const bool has = begin < to && end > from && end != begin;
            const bool all = has && begin <= from && end >= to;
            slots[threadIdx.x] = has && !all ? 2u * (group * a.group + member) + (from <= begin ? 0u : 1u) : 0xffffffffu;
            count = has && !all ? threadIdx.x + 1u : 0u;
        }
        __shared__ unsigned counts[3];
        count = __reduce_max_sync(0xffffffffu, count);
        if (threadIdx.x < 96u && (threadIdx.x & 31u) == 0) counts[threadIdx.x / 32u] = count;
        __syncthreads();
        count = max(counts[0], max(counts[1], counts[2]));
        if (count == 0) return;
        constexpr unsigned kAtOnce = 8 / kRows;
        const unsigned column = (threadIdx.x & 63u) * 4u, row0 = (part * 4u + threadIdx.x / 64u) * kRows;
        const unsigned feature = (tile % a.feature_tiles) * kTile + column, output0 = (tile / a.feature_tiles) * a.width + row0;
        if (feature >= a.inputs || output0 >= a.outputs) return;
        float4 sum[kRows];
#pragma unroll
        for (unsigned r = 0; r < kRows; ++r) sum[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (unsigned i = 0; i < count; i += kAtOnce) {
            float4 v[kAtOnce][kRows];
#pragma unroll
            for (unsigned n = 0; n < kAtOnce; ++n) {
                const unsigned slot = slots[i + n];
                const float* piece = a.pieces + (u64)slot * (a.width * kTile) + row0 * kTile + column;
#pragma unroll
                for (unsigned r = 0; r < kRows; ++r)
                    v[n][r] = slot != 0xffffffffu && output0 + r < a.outputs ? *reinterpret_cast<const float4*>(piece + r * kTile) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (unsigned n = 0; n < kAtOnce; ++n) {
#pragma unroll
                for (unsigned r = 0; r < kRows; ++r) {
                    sum[r].x += v[n][r].x;
                    sum[r].y += v[n][r].y;
                    sum[r].z += v[n][r].z;
                    sum[r].w += v[n][r].w;
                }
            }
        }
#pragma unroll
        for (unsigned r = 0; r < kRows; ++r) {
            if (output0 + r >= a.outputs) continue;
            T* out = static_cast<T*>(a.out) + (u64)(output0 + r) * a.inputs + feature;
            const float f[4] = {sum[r].x, sum[r].y, sum[r].z, sum[r].w};
#pragma unroll
            for (unsigned i = 0; i < 4; ++i)
                if (feature + i < a.inputs) out[i] = Elem<T>::from_f(f[i]);
        }
        return;
    }
    // 32 outputs of a tile per CTA, eight threads for each.
    const unsigned index = blockIdx.x - a.piece_ctas, output_tile = index / (a.width / 32u), column = (index % (a.width / 32u)) * 32u + (threadIdx.x & 31u);
    const unsigned tiles = a.feature_tiles * ((a.outputs + a.width - 1) / a.width);
    // The pairs that began inside one of its tiles.
    constexpr unsigned kEach = (kMaxPairs + 7) / 8;
    __shared__ bool inside[kEach * 8];
    if (threadIdx.x < kEach * 8u) {
        const unsigned pair = threadIdx.x, group = pair / a.group;
        bool here = false;
        if (group < a.groups && a.steps != 0u) {
            const unsigned begin = first_step(group, a.steps, a.groups), end = first_step(group + 1u, a.steps, a.groups), row = begin / a.steps_of_tile;
            const unsigned tile = a.whole_tiles + row * a.group + (pair - group * a.group);
            here = begin != row * a.steps_of_tile && end != begin && tile / a.feature_tiles == output_tile;
        }
        inside[pair] = here;
    }
    __syncthreads();
    // (Their sums are all on the way at once: one after another, those of 62 pairs took 30 us.)
    const unsigned warp = threadIdx.x / 32u;
    float sum = 0.0f, more[kEach];
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) more[i] = inside[warp + 8u * i] ? a.bias[(u64)(tiles + warp + 8u * i) * a.width + column] : 0.0f;
#pragma unroll 4
    for (unsigned m = warp; m < a.feature_tiles; m += 8u) sum += a.bias[(u64)(output_tile * a.feature_tiles + m) * a.width + column];
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) sum += more[i];
    __shared__ float sums[8][32];
    sums[threadIdx.x / 32u][threadIdx.x & 31u] = sum;
    __syncthreads();
    if (threadIdx.x >= 32u) return;
    for (unsigned i = 1; i < 8; ++i) sum += sums[i][threadIdx.x];
    const unsigned output = output_tile * a.width + column;
    if (output < a.outputs) static_cast<T*>(a.bias_out)[output] = Elem<T>::from_f(sum);
}

// dY as TMA reads it: rows of `pitch` elements; fp32 in three parts.
struct LayOutArgs {
    const char* dy;
    long long stride;  // bytes
    char* out;
    unsigned tokens, outputs;
    Divisor eights;  // of a row
};

// A thread takes eight outputs of a token.
template <typename T>
__global__ void __launch_bounds__(256) lay_out_kernel(const __grid_constant__ LayOutArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned eights = a.eights.d, i = blockIdx.x * 256u + threadIdx.x, token = a.eights.divide(i), n = (i - token * eights) * 8u;
    if (token >= a.tokens) return;
    const T* from = reinterpret_cast<const T*>(a.dy + (long long)token * a.stride) + n;
    unsigned words[2 * sizeof(T)];
    load_any<T, 8>(reinterpret_cast<const char*>(from), n < a.outputs ? min(8u, a.outputs - n) : 0u, words);
    if constexpr (sizeof(T) == 2) {
        *(reinterpret_cast<uint4*>(a.out) + i) = make_uint4(words[0], words[1], words[2], words[3]);
    } else {
        unsigned part[3][4] = {};
#pragma unroll
        for (unsigned e = 0; e < 8; ++e) {
            float rest = __uint_as_float(words[e]);
            const bool finite = (words[e] & 0x7f800000u) != 0x7f800000u;
#pragma unroll
            for (int p = 0; p < 3; ++p) {  // the leading eight bits of what is left, cut off and not rounded: the rest is exact, and nothing overflows
                const unsigned cut = __float_as_uint(rest) >> 16;
                rest -= __uint_as_float(cut << 16);
                const unsigned put = finite ? cut : (p == 0 ? ((words[e] & 0x7fffffffu) > 0x7f800000u ? 0x7fc0u : cut) : 0u);
                part[p][e / 2u] |= put << (16u * (e & 1u));
            }
        }
        const u64 eight = (u64)a.tokens * eights;
#pragma unroll
        for (int p = 0; p < 3; ++p) *(reinterpret_cast<uint4*>(a.out) + p * eight + i) = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
    }
}

struct Plan {
    bool wide = false;
    unsigned parts = 1, width = kTile, pitch = 0, feature_tiles = 0, output_tiles = 0, steps_of_part = 0, steps_of_tile = 0, steps = 0, pairs = 0, waves = 0, group = 1, groups = 1;
    bool copied = false, cut = false;
    bool summed = false;  // sums in memory: pieces, or whole tiles of long sums
    bool direct = false;  // the bias's gradient comes from weight_grad_kernel itself
    std::size_t pieces_at = 0, bias_at = 0, bytes = 0;
};

// Pairs of CTAs that run at once: where GPCs have odd numbers of SMs, fewer than half the SMs.
unsigned pairs_of_device(int device) {
    static std::atomic<unsigned> known[64];
    if (device >= 0 && device < 64 && known[device].load() != 0) return known[device].load();
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(2 * kMaxPairs);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kShared;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    int clusters = 0;
    B2_CUDA(cudaOccupancyMaxActiveClusters(&clusters, weight_grad_kernel<__nv_bfloat16, true, false>, &config));
    const unsigned pairs = std::min(kMaxPairs, (unsigned)std::max(1, clusters));
    if (device >= 0 && device < 64) known[device].store(pairs);
    return pairs;
}

// Shared memory beyond 48 KiB is asked for once per kernel and device.
void prepare_device(int device) {
    static std::mutex mutex;
    static bool done[64] = {};
    std::lock_guard<std::mutex> lock(mutex);
    if (device >= 0 && device < 64 && done[device]) return;
    const void* kernels[] = {(const void*)weight_grad_kernel<float, false, false>,         (const void*)weight_grad_kernel<float, true, false>,
                             (const void*)weight_grad_kernel<__half, false, false>,        (const void*)weight_grad_kernel<__half, true, false>,
                             (const void*)weight_grad_kernel<__half, false, true>,         (const void*)weight_grad_kernel<__half, true, true>,
                             (const void*)weight_grad_kernel<__nv_bfloat16, false, false>, (const void*)weight_grad_kernel<__nv_bfloat16, true, false>,
                             (const void*)weight_grad_kernel<__nv_bfloat16, false, true>,  (const void*)weight_grad_kernel<__nv_bfloat16, true, true>};
    for (const void* k : kernels) B2_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kShared));
    if (device >= 0 && device < 64) done[device] = true;
}

int current_device() {
    int device = 0;
    B2_CUDA(cudaGetDevice(&device));
    return device;
}

// Whether tiles of 512 outputs are faster: with long sums, whose epilogue counts for little, and many steps for each pair. Steps of a tile squared, times tiles, tells
// them apart (us, 256 / 512 outputs; thousands): 8192 x 1024 x 1024 31 / 33 (131), 2048 x 4096 x 4096 84 / 87 (131), 8192 x 768 x 2304 47 / 60 (246),
// 4096 x 2048 x 4096 72 / 80 (262), 4096 x 4096 x 4096 163 / 131 (524), 8192 x 2048 x 2048 73 / 69 (524), 16384 x 2048 x 1000 75 / 73 (1049),
// 16384 x 4096 x 4096 466 / 395 (8389). Not where rounding the outputs up to 512 adds more than an eighth.
bool wide_tiles(const WeightGradCall& c, u64 steps) {
    const u64 tiles = (c.inputs + kTile - 1) / kTile * ((c.outputs + 2 * kTile - 1) / (2 * kTile));
    const u64 narrow = (c.outputs + kTile - 1) / kTile, wide = (c.outputs + 2 * kTile - 1) / (2 * kTile) * 2;
    return c.dtype != DType::Float && c.outputs > kTile && steps * steps * tiles >= 400000 && wide * 8 <= narrow * 9;
}

Plan plan_of(const WeightGradCall& c) {
    Plan p;
    const std::size_t bytes = c.dtype == DType::Float ? 4 : 2;
    p.parts = c.dtype == DType::Float ? 3 : 1;
    p.copied = c.dtype == DType::Float || (reinterpret_cast<std::uintptr_t>(c.dy) % 16) != 0 || (c.stride * (long long)bytes) % 16 != 0 ||
               c.stride < (long long)c.outputs;
    p.pitch = (unsigned)((c.outputs + 7) / 8 * 8);
    p.feature_tiles = (unsigned)((c.inputs + kTile - 1) / kTile);
    const u64 steps_of_part = (c.tokens + kStep - 1) / kStep;
    p.wide = wide_tiles(c, steps_of_part);
    p.width = p.wide ? 2 * kTile : kTile;
    p.output_tiles = (unsigned)((c.outputs + p.width - 1) / p.width);
    const u64 tiles = (u64)p.feature_tiles * p.output_tiles;
    B2_REQUIRE(steps_of_part * p.parts * tiles < (1ull << 31) && tiles < (1ull << 24) && c.tokens < (1ull << 31),
               "weight_grad8: too many tokens, inputs and outputs for one call");
    p.steps_of_part = (unsigned)steps_of_part;
    p.steps_of_tile = p.steps_of_part * p.parts;
    const int device = current_device();
    prepare_device(device);
    // A pair for each tile, or for every four steps: with less each, the pieces cost more than the sums (one is 256 KiB to write and read again).
    p.pairs = (unsigned)std::min<u64>(pairs_of_device(device), std::max(tiles, tiles * p.steps_of_tile / 4));
    if (tiles < p.pairs) {
        // All feature tiles side by side, unless that leaves more than a tenth of the pairs idle.
        const unsigned side = p.pairs / p.feature_tiles * p.feature_tiles;
        if (side * 10 >= p.pairs * 9) {
            p.group = p.feature_tiles;
            p.pairs = side;
        }
    }
    p.waves = (unsigned)tiles / p.pairs;
    const unsigned left = ((unsigned)tiles - p.waves * p.pairs) / p.group;
    p.steps = left * p.steps_of_tile;
    // The tiles that are left are cut where that saves every pair more than eight steps, which is what writing and adding pieces costs (bf16, cut / whole, us:
    // 512 x 4096 x 4096, a saving of 2 steps, 36.7 / 29.0; 1024 x 2048 x 2048, 2 steps, 23.6 / 16.8; 1024 x 768 x 768, 12 steps, 13.6 / 15.2).
    p.groups = std::max(1u, p.pairs / p.group);
    if (left != 0 && p.steps_of_tile < 8 + p.steps / p.groups) p.groups = left;
    if (p.waves == 0) p.pairs = p.groups * p.group;
    for (unsigned i = 1; i < p.groups; ++i) p.cut |= first_step(i, p.steps, p.groups) % p.steps_of_tile != 0;
    // (A warp sums a step's 64 columns about as fast as the step goes, but no faster: the first tile of features must not hold up a long sum.)
    p.direct = c.bias_grad != nullptr && !p.cut && (p.feature_tiles == 1 || p.steps_of_tile <= 32);
    const std::size_t copy = p.copied ? (std::size_t)p.parts * c.tokens * p.pitch * 2 : 0;
    p.pieces_at = (copy + 255) / 256 * 256;
    p.summed = p.cut || (p.parts == 1 && p.steps_of_tile > kLongSteps);
    p.bias_at = p.pieces_at + (p.summed ? (std::size_t)2 * p.pairs * p.width * kTile * sizeof(float) : 0);
    p.bytes = p.bias_at + (c.bias_grad != nullptr && !p.direct ? (tiles + p.pairs) * p.width * sizeof(float) : 0);
    return p;
}

// A word of host memory for each device, that a kernel whose wait ran out writes to.
constexpr int kDevices = 64;
std::atomic<unsigned*> status_words{nullptr};
unsigned* status_word(int device) {
    static unsigned* words = [] {
        // (Allocating is allowed beside a capture: nothing of it belongs to the graph.)
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        B2_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
        void* p = nullptr;
        const cudaError_t st = cudaHostAlloc(&p, kDevices * sizeof(unsigned), cudaHostAllocMapped | cudaHostAllocPortable);
        cudaThreadExchangeStreamCaptureMode(&mode);
        B2_CUDA(st);
        std::fill_n(static_cast<unsigned*>(p), kDevices, 0u);
        status_words.store(static_cast<unsigned*>(p));
        return static_cast<unsigned*>(p);
    }();
    return words + device % kDevices;
}

template <typename T>
void launch(const WeightGradCall& c, const Plan& p) {
    char* workspace = static_cast<char*>(c.workspace);
    const void* dy = c.dy;
    u64 row_bytes = (u64)c.stride * sizeof(T);
    if (p.copied) {
        LayOutArgs l;
        l.dy = static_cast<const char*>(c.dy);
        l.stride = c.stride * (long long)sizeof(T);
        l.out = workspace;
        l.tokens = (unsigned)c.tokens;
        l.outputs = (unsigned)c.outputs;
        l.eights = Divisor(p.pitch / 8);
        const u64 eights = (u64)c.tokens * (p.pitch / 8), ctas = (eights + 255) / 256;
        B2_REQUIRE(eights < (1ull << 31), "weight_grad8: dy is too large for one call");
        B2_CUDA(launch_dependent<LayOutArgs>(lay_out_kernel<T>, dim3((unsigned)ctas), 256, 0, c.stream, l));
        dy = workspace;
        row_bytes = (u64)p.pitch * 2;
    }
    WeightGradArgs a;
    const auto encode = cu::api().TensorMapEncodeTiled;
    if (encode == nullptr) throw std::runtime_error("weight_grad8: the driver does not export cuTensorMapEncodeTiled");
    const auto map = [&](CUtensorMap* m, CUtensorMapDataType type, const void* data, u64 columns, u64 rows, u64 planes, u64 bytes, cuuint32_t box_columns,
                         CUtensorMapSwizzle swizzle, const char* what) {
        const cuuint64_t extent[3] = {columns, rows, planes}, strides[2] = {bytes, bytes * rows};
        const cuuint32_t box[3] = {box_columns, kStep, 1}, element_strides[3] = {1, 1, 1};
        cu::check(encode(m, type, 3, const_cast<void*>(data), extent, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE), what);
    };
    map(&a.dy, std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dy, c.outputs, c.tokens, p.parts, row_bytes, 64,
        CU_TENSOR_MAP_SWIZZLE_128B, "weight_grad8: tensor map of dy");
    a.pitch = (c.inputs + kBlock8 - 1) / kBlock8 * kBlock8;
    map(&a.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.codes, a.pitch, c.tokens, 1, a.pitch, kHalf, CU_TENSOR_MAP_SWIZZLE_NONE, "weight_grad8: tensor map of the codes");
    a.scales = c.scales;
    a.out = c.weight_grad;
    a.pieces = reinterpret_cast<float*>(workspace + p.pieces_at);
    a.bias_out = p.direct ? c.bias_grad : nullptr;
    a.bias = c.bias_grad != nullptr && !p.direct ? reinterpret_cast<float*>(workspace + p.bias_at) : nullptr;
    a.status = status_word(current_device());
    a.wait_ns = c.wait_ns;
    a.tokens = (unsigned)c.tokens;
    a.inputs = (unsigned)c.inputs;
    a.outputs = (unsigned)c.outputs;
    a.wide = c.inputs * sizeof(T) % 16 == 0 && reinterpret_cast<std::uintptr_t>(c.weight_grad) % 16 == 0;
    a.feature_tiles = p.feature_tiles;
    a.parts = p.parts;
    a.steps_of_part = p.steps_of_part;
    a.steps_of_tile = p.steps_of_tile;
    a.steps = p.steps;
    a.pairs = p.pairs;
    a.waves = p.waves;
    a.group = p.group;
    a.groups = p.groups;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(2 * p.pairs);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kShared;
    config.stream = c.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 2;
    const bool bias = c.bias_grad != nullptr;
    void (*kernel)(WeightGradArgs) = bias ? weight_grad_kernel<T, true, false> : weight_grad_kernel<T, false, false>;
    if constexpr (sizeof(T) == 2)
        if (p.wide) kernel = bias ? weight_grad_kernel<T, true, true> : weight_grad_kernel<T, false, true>;
    B2_CUDA(cudaLaunchKernelEx(&config, kernel, a));
    if (!p.cut && (c.bias_grad == nullptr || p.direct)) return;
    FinishArgs f;
    f.out = c.weight_grad;
    f.bias_out = c.bias_grad;
    f.pieces = a.pieces;
    f.bias = a.bias;
    f.inputs = a.inputs;
    f.outputs = a.outputs;
    f.width = p.width;
    f.feature_tiles = p.feature_tiles;
    f.steps_of_tile = p.steps_of_tile;
    f.steps = p.steps;
    f.group = p.group;
    f.groups = p.groups;
    f.whole_tiles = p.waves * p.pairs;
    const unsigned shared_out = p.cut ? p.steps / p.steps_of_tile * p.group : 0, rows = shared_out * (p.width / 16) >= 4 * 2 * kMaxPairs ? 4 : 1;
    f.piece_ctas = shared_out * (p.width / (4 * rows));
    const unsigned grid = f.piece_ctas + (c.bias_grad != nullptr ? p.output_tiles * (p.width / 32) : 0);
    B2_CUDA(launch_dependent<FinishArgs>(rows == 4 ? finish_kernel<T, 4> : finish_kernel<T, 1>, dim3(grid), 256, 0, c.stream, f));
}

}  // namespace

std::size_t weight_grad_workspace(const WeightGradCall& call) {
    if (call.tokens == 0 || call.inputs == 0 || call.outputs == 0) return 0;
    return plan_of(call).bytes;
}

void launch_weight_grad(const WeightGradCall& c) {
    if (c.outputs == 0) return;
    const std::size_t bytes = dtype_size(c.dtype);
    if (c.tokens == 0 || c.inputs == 0) {
        if (c.inputs != 0) B2_CUDA(cudaMemsetAsync(c.weight_grad, 0, c.inputs * c.outputs * bytes, c.stream));
        B2_REQUIRE(c.inputs != 0 || c.bias_grad == nullptr, "weight_grad8: a bias gradient needs at least one input");
        if (c.bias_grad != nullptr) B2_CUDA(cudaMemsetAsync(c.bias_grad, 0, c.outputs * bytes, c.stream));
        return;
    }
    const Plan p = plan_of(c);
    B2_REQUIRE(p.bytes == 0 || c.workspace != nullptr, "the workspace must be non-null");
    switch (c.dtype) {
        case DType::Float: return launch<float>(c, p);
        case DType::Float16: return launch<__half>(c, p);
        case DType::BFloat16: return launch<__nv_bfloat16>(c, p);
    }
}

bool weight_grad_failed(int device) {
    B2_REQUIRE(device >= 0, "no such device");
    unsigned* words = status_words.load();  // (null before the first call of all)
    return words != nullptr && __atomic_exchange_n(words + device % kDevices, 0u, __ATOMIC_RELAXED) != 0u;
}

}  // namespace b200ccl::kernels
