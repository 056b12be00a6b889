// Weight gradient of a projection whose input was kept in 8 bits: dW[n][k] = sum over tokens of dY[t][n] * X^[t][k], and the bias's, sum of dY[t][n].
//
// The product is D = X^^T dY on the tensor cores, M = inputs (features), N = outputs, summed over tokens; both operands lie in memory by tokens, which
// tcgen05 reads as they are. A pair of CTAs works on a tile of 256 features by 256 outputs, 64 tokens at a time: each CTA holds 128 features
// of X^ and 128 outputs of dY per step (32 KiB), the accumulators of its 128 features in tensor memory, twice, so that one tile is written while the
// next is summed. A pair halves what a tile reads: alone, a CTA with 128 x 256 would draw 80 bytes per cycle from L2 (32 KiB of dY
// and 8 KiB of codes every 512 cycles, which a step takes), the pair 48 per SM.
//
// Roles of a CTA's 16 warps: one thread copies dY by TMA; one thread of the first CTA issues the products, and its counterpart in the second tells it that
// its dY has come; eight warps widen codes to 16-bit numbers, exactly (block8.cuh), straight into the swizzled operand (per 4 codes: 5 byte
// permutes and 4 two-wide operations, about a third of the issue slots of a step); four warps write finished tiles; two sum columns of dY
// for the bias out of shared memory, each tile of features for its own share of the steps, so that every step of dY is summed once.
//
// Work is cut evenly, not by tiles: the steps of all tiles stand in one row, and pair i of P takes steps [i S / P, (i+1) S / P). A tile that is
// cut is summed in pieces, in 32 bits in the workspace, and finish_kernel adds them in the order of tokens: the result does not depend on timing.
//
// fp32: X^ is a bf16 number in any case, and dY is the exact sum of three (its 24 bits cut into eights), so three products of bf16 numbers
// with 32-bit accumulators give it in full; the three parts follow one another along the summed axis.
//
// dY that TMA cannot read (rows or address not at a multiple of 16 bytes) is copied first.
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
constexpr unsigned kStages = 6;       // steps in shared memory
constexpr unsigned kBlockBytes = kStep * 128;         // 64 elements of every token of a step
constexpr unsigned kOperandBytes = 2 * kBlockBytes;   // a CTA's half of an operand
constexpr unsigned kStageBytes = 2 * kOperandBytes;
constexpr unsigned kThreads = 512;
constexpr unsigned kTransformWarps = 8, kFirstTransformWarp = 4, kFirstEpilogueWarp = 12;
constexpr unsigned kAhead = 3;        // steps whose codes are on the way
constexpr unsigned kMaxPairs = 74;    // 148 SMs
constexpr unsigned kFinishRows = 16;  // outputs of a tile that a CTA of finish_kernel adds up
constexpr unsigned kShared = kStages * kStageBytes + 1024 /* to the next multiple of 1024 */ + 512;

struct alignas(64) WeightGradArgs {
    CUtensorMap dy;  // [parts][tokens][outputs]
    const unsigned char* codes;
    const unsigned char* scales;
    void* out;
    float* pieces;     // [2 * pairs][256 outputs][256 features]
    float* bias;       // [tiles + pairs][256], or null
    unsigned* status;  // host memory
    u64 pitch;         // bytes of a token's codes
    unsigned tokens, inputs, outputs;
    unsigned feature_tiles, steps_of_part, steps_of_tile, steps, pairs;
};

struct FinishArgs {
    void* out;
    void* bias_out;
    const float* pieces;
    const float* bias;
    unsigned inputs, outputs, feature_tiles, steps_of_tile, steps, pairs;
    unsigned piece_ctas;  // CTAs that add pieces; the others make the bias's gradient
};

__host__ __device__ inline unsigned first_step(unsigned pair, unsigned steps, unsigned pairs) { return (unsigned)((u64)pair * steps / pairs); }

// Barriers of a CTA, in its shared memory.
struct Barriers {
    u64 dy[kStages];       // this CTA's dY of a stage has come
    u64 dy_other[kStages]; // first CTA: the other's has
    u64 x[kStages];        // first CTA: both CTAs' X^ is written
    u64 empty[kStages];    // the stage has been read
    u64 sums[2];           // accumulators are complete
    u64 sums_free[2];      // first CTA: both CTAs have written theirs out
    u64 drained;           // first CTA, after a failure
    unsigned tmem;
    unsigned failed;
};

// Four codes as two pairs of 16-bit numbers: 128 + m (bf16) or 1024 + m (fp16) by placing bytes, less 128 or 1024, times the step.
template <bool kBf16>
__device__ __forceinline__ uint2 widen4(unsigned word, unsigned step2) {
    const unsigned m = word & 0x7f7f7f7fu;
    const unsigned high = kBf16 ? 0x43434343u : 0x64646464u;
    unsigned a = __byte_perm(m, high, 0x4140), b = __byte_perm(m, high, 0x4342);
    const unsigned sa = __byte_perm(word, 0u, 0x1404), sb = __byte_perm(word, 0u, 0x3424);
    if constexpr (kBf16) {
        const __nv_bfloat162 off = __floats2bfloat162_rn(128.0f, 128.0f), s = *reinterpret_cast<const __nv_bfloat162*>(&step2);
        const __nv_bfloat162 va = __hmul2(__hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), off), s);
        const __nv_bfloat162 vb = __hmul2(__hsub2(*reinterpret_cast<__nv_bfloat162*>(&b), off), s);
        a = *reinterpret_cast<const unsigned*>(&va);
        b = *reinterpret_cast<const unsigned*>(&vb);
    } else {
        const __half2 off = __floats2half2_rn(1024.0f, 1024.0f), s = *reinterpret_cast<const __half2*>(&step2);
        const __half2 va = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&a), off), s);
        const __half2 vb = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&b), off), s);
        a = *reinterpret_cast<const unsigned*>(&va);
        b = *reinterpret_cast<const unsigned*>(&vb);
    }
    return make_uint2(a | (sa & 0x80008000u), b | (sb & 0x80008000u));
}
template <bool kBf16>
__device__ __forceinline__ unsigned step_pair(unsigned scale) {
    if constexpr (kBf16) return scale << 7 | scale << 23;
    const __half2 s = __float2half2_rn(step8(scale));
    return *reinterpret_cast<const unsigned*>(&s);
}
__device__ __forceinline__ void store_shared16(unsigned at, unsigned a, unsigned b, unsigned c, unsigned d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ unsigned load_shared4(unsigned at) {
    unsigned v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

// The pieces of a pair: steps of one tile each.
struct Piece {
    unsigned tile, from, to, at;  // steps of the tile; `at` in the row of all steps
};
__device__ __forceinline__ Piece piece_at(const WeightGradArgs& a, unsigned at, unsigned end) {
    Piece p;
    p.at = at;
    p.tile = at / a.steps_of_tile;
    p.from = at - p.tile * a.steps_of_tile;
    p.to = min(a.steps_of_tile, p.from + (end - at));
    return p;
}

// T: type of dY and the gradients. kBias: also columns of dY.
template <typename T, bool kBias>
__global__ void __launch_bounds__(kThreads, 1) weight_grad_kernel(const __grid_constant__ WeightGradArgs a) {
    constexpr bool kBf16 = !std::is_same_v<T, __half>;
    extern __shared__ unsigned char raw[];
    // Swizzled operands start at multiples of 1024 bytes; the same place in both CTAs.
    unsigned char* shared = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    Barriers& bars = *reinterpret_cast<Barriers*>(shared + kStages * kStageBytes);
    volatile unsigned* failed = &bars.failed;
    const unsigned base = smem_addr(shared);
    const unsigned warp = threadIdx.x / 32u, lane = threadIdx.x & 31u;
    const unsigned rank = cluster_rank(), pair = blockIdx.x / 2u;
    const unsigned begin = first_step(pair, a.steps, a.pairs), end = first_step(pair + 1, a.steps, a.pairs);

    if (warp == 0 && lane == 0) {
        for (unsigned s = 0; s < kStages; ++s) {
            mbar_init(&bars.dy[s], 1);
            mbar_init(&bars.dy_other[s], 1);
            mbar_init(&bars.x[s], 2 * kTransformWarps);
            mbar_init(&bars.empty[s], kBias ? 3 : 1);
        }
        for (unsigned i = 0; i < 2; ++i) {
            mbar_init(&bars.sums[i], 1);
            mbar_init(&bars.sums_free[i], 8);
        }
        mbar_init(&bars.drained, 1);
        bars.failed = 0;
        mbar_fence_init();
        tma_prefetch_map(&a.dy);
    }
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
            unsigned n = 0;  // steps so far
            bool ok = true;
            for (unsigned at = begin; at < end && ok;) {
                const Piece p = piece_at(a, at, end);
                const int output = (int)((p.tile / a.feature_tiles) * kTile + rank * kHalf);
                unsigned part = p.from / a.steps_of_part, step = p.from - part * a.steps_of_part;
                for (unsigned k = p.from; k < p.to; ++k, ++n) {
                    const unsigned s = n % kStages;
                    ok = wait_phase(bar(bars.empty[s]), ((n / kStages) & 1u) ^ 1u, failed);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&bars.dy[s], kOperandBytes);
                    const unsigned dst = base + s * kStageBytes + kOperandBytes;
                    tma_load_box(dst, &a.dy, output, (int)(step * kStep), (int)part, bar(bars.dy[s]));
                    tma_load_box(dst + kBlockBytes, &a.dy, output + 64, (int)(step * kStep), (int)part, bar(bars.dy[s]));
                    if (++step == a.steps_of_part) { step = 0; ++part; }
                }
                at += p.to - p.from;
            }
            // Copies have landed and stages been given back before the CTA ends, after a failure too.
            if (ok) {
                for (unsigned i = n > kStages ? n - kStages : 0; i < n; ++i) wait_phase(bar(bars.empty[i % kStages]), (i / kStages) & 1u, failed);
            } else {
                for (unsigned i = n > kStages ? n - kStages : 0; i < n; ++i)
                    for (unsigned polls = 0; polls < 1000u && !phase_over(bar(bars.dy[i % kStages]), (i / kStages) & 1u); ++polls) {}
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const unsigned shape = product_by_rows(kTile, kTile, kBf16);
            unsigned n = 0, pieces = 0;
            bool ok = true;
            for (unsigned at = begin; at < end && ok; ++pieces) {
                const Piece p = piece_at(a, at, end);
                const unsigned buffer = pieces & 1u;
                ok = wait_phase(bar(bars.sums_free[buffer]), ((pieces >> 1) & 1u) ^ 1u, failed);
                if (!ok) break;
                tcgen05_fence_after();
                for (unsigned k = p.from; k < p.to; ++k, ++n) {
                    const unsigned s = n % kStages, parity = (n / kStages) & 1u;
                    ok = wait_phase(bar(bars.dy[s]), parity, failed) && wait_phase(bar(bars.dy_other[s]), parity, failed) &&
                         wait_phase(bar(bars.x[s]), parity, failed);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const std::uint64_t x = operand_by_rows(base + s * kStageBytes, kBlockBytes);
                    const std::uint64_t dy = operand_by_rows(base + s * kStageBytes + kOperandBytes, kBlockBytes);
#pragma unroll
                    for (unsigned i = 0; i < kStep / 16; ++i)  // 16 tokens are 2048 bytes
                        mma_pair(tmem + buffer * kTile, x + i * (2048 >> 4), dy + i * (2048 >> 4), shape, k > p.from || i > 0);
                    commit_pair(bar(bars.empty[s]));
                }
                if (!ok) break;
                commit_pair(bar(bars.sums[buffer]));
                at += p.to - p.from;
            }
            if (!ok) {  // products under way read shared memory of both CTAs
                commit_pair(bar(bars.drained));
                for (unsigned polls = 0; polls < 1000u && !phase_over(bar(bars.drained), 0); ++polls) {}
            }
        } else if (lane == 0) {
            for (unsigned n = 0; n < end - begin; ++n) {
                if (!wait_phase(bar(bars.dy[n % kStages]), (n / kStages) & 1u, failed)) break;
                mbar_arrive_at(bar(bars.dy_other[n % kStages]), 0);
            }
        }
    } else if (warp < kFirstTransformWarp) {
        if constexpr (kBias) {
            const unsigned column = (warp - 2u) * 64u + lane * 2u;  // of this CTA's 128 outputs
            unsigned n = 0;
            bool ok = true;
            for (unsigned at = begin; at < end && ok;) {
                const Piece p = piece_at(a, at, end);
                const unsigned share = p.tile % a.feature_tiles;
                float x = 0.0f, y = 0.0f;
                for (unsigned k = p.from; k < p.to; ++k, ++n) {
                    const unsigned s = n % kStages;
                    ok = __all_sync(0xffffffffu, wait_phase(bar(bars.dy[s]), (n / kStages) & 1u, failed));
                    if (!ok) break;
                    if (k % a.feature_tiles == share) {
                        const unsigned from = base + s * kStageBytes + kOperandBytes + (warp - 2u) * kBlockBytes;
#pragma unroll 16
                        for (unsigned t = 0; t < kStep; ++t) {
                            const unsigned w = load_shared4(from + t * 128u + (((lane / 4u) ^ (t & 7u)) * 16u) + (lane & 3u) * 4u);
                            const float2 f = kBf16 ? b2_to_f2(w) : h2_to_f2(w);
                            x += f.x;
                            y += f.y;
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(bars.empty[s]));
                }
                if (!ok) break;
                float* to = a.bias + (u64)(p.from == 0 ? p.tile : a.feature_tiles * ((a.outputs + kTile - 1) / kTile) + pair) * kTile;
                *reinterpret_cast<float2*>(to + rank * kHalf + column) = make_float2(x, y);
                at += p.to - p.from;
            }
        }
    } else if (warp < kFirstEpilogueWarp) {
        const unsigned tid = threadIdx.x - kFirstTransformWarp * 32u;
        const unsigned chunk = tid & 7u, row = tid >> 3;  // 16 features of a token; the tokens row and row + 32 of a step
        uint4 code[kAhead][2];
        unsigned scale[kAhead][2];
        // Where the next codes are read.
        unsigned next = begin, tile = begin / a.steps_of_tile, k = begin - tile * a.steps_of_tile;
        unsigned step = k % a.steps_of_part;
        unsigned feature = (tile % a.feature_tiles) * kTile + rank * kHalf + chunk * 16u;
        const auto load = [&](uint4(&c)[2], unsigned(&sc)[2]) {
#pragma unroll
            for (unsigned u = 0; u < 2; ++u) {
                const u64 token = (u64)step * kStep + row + u * 32u;
                const bool there = token < a.tokens && feature < a.pitch;
                c[u] = there ? *reinterpret_cast<const uint4*>(a.codes + token * a.pitch + feature) : make_uint4(0u, 0u, 0u, 0u);
                sc[u] = there ? a.scales[(token * a.pitch + feature) / kBlock8] : 127u;
            }
            ++next;
            if (++step == a.steps_of_part) step = 0;
            if (++k == a.steps_of_tile) {
                k = 0;
                ++tile;
                feature = (tile % a.feature_tiles) * kTile + rank * kHalf + chunk * 16u;
            }
        };
#pragma unroll
        for (unsigned i = 0; i < kAhead; ++i)
            if (next < end) load(code[i], scale[i]);
        // The two halves of a chunk go out in turn, odd ones first for the second block of 64 features: eight lanes then write to eight
        // different 16-byte columns of the shared memory's banks.
        const unsigned block = base + (chunk >> 2) * kBlockBytes, odd = chunk >> 2;
        const unsigned column0 = ((chunk & 3u) * 2u + odd), column1 = ((chunk & 3u) * 2u + (odd ^ 1u));
        unsigned n = 0;
        bool ok = true;
        for (unsigned at = begin; at < end && ok; at += kAhead) {
#pragma unroll
            for (unsigned i = 0; i < kAhead; ++i) {
                if (at + i < end && ok) {
                    const unsigned s = n % kStages;
                    ok = __all_sync(0xffffffffu, wait_phase(bar(bars.empty[s]), ((n / kStages) & 1u) ^ 1u, failed));
                    if (!ok) break;
#pragma unroll
                    for (unsigned u = 0; u < 2; ++u) {
                        const unsigned t = row + u * 32u;
                        const unsigned s2 = step_pair<kBf16>(scale[i][u]);
                        const uint2 w0 = widen4<kBf16>(code[i][u].x, s2), w1 = widen4<kBf16>(code[i][u].y, s2);
                        const uint2 w2 = widen4<kBf16>(code[i][u].z, s2), w3 = widen4<kBf16>(code[i][u].w, s2);
                        const unsigned to = block + s * kStageBytes + t * 128u;
                        const unsigned c0 = to + ((column0 ^ (t & 7u)) * 16u), c1 = to + ((column1 ^ (t & 7u)) * 16u);
                        if (odd) {
                            store_shared16(c0, w2.x, w2.y, w3.x, w3.y);
                            store_shared16(c1, w0.x, w0.y, w1.x, w1.y);
                        } else {
                            store_shared16(c0, w0.x, w0.y, w1.x, w1.y);
                            store_shared16(c1, w2.x, w2.y, w3.x, w3.y);
                        }
                    }
                    fence_shared_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_at(bar(bars.x[s]), 0);
                    if (next < end) load(code[i], scale[i]);
                    ++n;
                }
            }
        }
    } else {
        const unsigned quarter = warp & 3u;  // lanes of tensor memory that this warp reaches
        const unsigned in_tile = rank * kHalf + quarter * 32u + lane;
        unsigned pieces = 0;
        for (unsigned at = begin; at < end; ++pieces) {
            const Piece p = piece_at(a, at, end);
            const unsigned buffer = pieces & 1u;
            if (!__all_sync(0xffffffffu, wait_phase(bar(bars.sums[buffer]), (pieces >> 1) & 1u, failed))) break;
            tcgen05_fence_after();
            const bool whole = p.from == 0 && p.to == a.steps_of_tile;
            const unsigned feature = (p.tile % a.feature_tiles) * kTile + in_tile;
            const unsigned output0 = (p.tile / a.feature_tiles) * kTile;
            float* piece = a.pieces + (u64)(2u * pair + (p.at == begin ? 0u : 1u)) * (kTile * kTile) + in_tile;
            for (unsigned c = 0; c < kTile; c += 32u) {
                float f[32];
                tmem_load32(tmem + buffer * kTile + c + (quarter * 32u << 16), f);
                if (whole) {
                    T* out = static_cast<T*>(a.out) + (u64)(output0 + c) * a.inputs + feature;
#pragma unroll
                    for (unsigned j = 0; j < 32; ++j)
                        if (feature < a.inputs && output0 + c + j < a.outputs) out[(u64)j * a.inputs] = Elem<T>::from_f(f[j]);
                } else {
#pragma unroll
                    for (unsigned j = 0; j < 32; ++j) piece[(u64)(c + j) * kTile] = f[j];
                }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_at(bar(bars.sums_free[buffer]), 0);
            at += p.to - p.from;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && *failed != 0u) *static_cast<volatile unsigned*>(a.status) = 1u;
    tcgen05_fence_before();
    cluster_sync();  // nothing of this CTA is read or arrived at by the other any more
    tcgen05_fence_after();
    if (warp == 1) tmem_free_pair(tmem, 2 * kTile);
}

// Adds the pieces of cut tiles, and the bias's.
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ FinishArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x < a.piece_ctas) {
        // One tile for each border between pairs that is the first inside its tile.
        constexpr unsigned kParts = kTile / kFinishRows;
        const unsigned border = blockIdx.x / kParts + 1u, part = blockIdx.x % kParts;
        const unsigned at = first_step(border, a.steps, a.pairs);
        const unsigned tile = at / a.steps_of_tile, from = tile * a.steps_of_tile;
        const unsigned before = first_step(border - 1u, a.steps, a.pairs);
        if (at == from || before > from) return;
        const unsigned output0 = (tile / a.feature_tiles) * kTile + part * kFinishRows, feature0 = (tile % a.feature_tiles) * kTile;
        const unsigned feature = feature0 + (threadIdx.x & 63u) * 4u;
        const unsigned to = from + a.steps_of_tile;
        for (unsigned r = threadIdx.x / 64u; r < kFinishRows; r += 4u) {
            const unsigned in_piece = (part * kFinishRows + r) * kTile + (threadIdx.x & 63u) * 4u;
            const auto read = [&](unsigned slot) { return *reinterpret_cast<const float4*>(a.pieces + (u64)slot * (kTile * kTile) + in_piece); };
            float4 sum = read(2u * (border - 1u) + (before == from ? 0u : 1u));
            for (unsigned p = border; p < a.pairs && first_step(p, a.steps, a.pairs) < to; ++p) {
                const float4 v = read(2u * p);
                sum.x += v.x;
                sum.y += v.y;
                sum.z += v.z;
                sum.w += v.w;
            }
            const unsigned output = output0 + r;
            if (output >= a.outputs) continue;
            T* out = static_cast<T*>(a.out) + (u64)output * a.inputs + feature;
            const float f[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (unsigned i = 0; i < 4; ++i)
                if (feature + i < a.inputs) out[i] = Elem<T>::from_f(f[i]);
        }
        return;
    }
    const unsigned output_tile = blockIdx.x - a.piece_ctas, output = output_tile * kTile + threadIdx.x;
    const unsigned tiles = a.feature_tiles * ((a.outputs + kTile - 1) / kTile);
    float sum = 0.0f;
    for (unsigned m = 0; m < a.feature_tiles; ++m) {
        const unsigned tile = output_tile * a.feature_tiles + m, from = tile * a.steps_of_tile, to = from + a.steps_of_tile;
        sum += a.bias[(u64)tile * kTile + threadIdx.x];
        unsigned p = (unsigned)((u64)from * a.pairs / a.steps);
        while (p < a.pairs && first_step(p, a.steps, a.pairs) <= from) ++p;
        for (; p < a.pairs && first_step(p, a.steps, a.pairs) < to; ++p) sum += a.bias[(u64)(tiles + p) * kTile + threadIdx.x];
    }
    if (output < a.outputs) static_cast<T*>(a.bias_out)[output] = Elem<T>::from_f(sum);
}

// dY as TMA reads it: rows of `pitch` elements; fp32 in three parts.
struct LayOutArgs {
    const char* dy;
    long long stride;  // bytes
    char* out;
    u64 tokens;
    unsigned outputs, pitch;
};

template <typename T>
__global__ void __launch_bounds__(256) lay_out_kernel(const __grid_constant__ LayOutArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const u64 i = (u64)blockIdx.x * 256u + threadIdx.x;
    const u64 token = i / a.pitch;
    const unsigned n = (unsigned)(i - token * a.pitch);
    if (token >= a.tokens) return;
    const bool there = n < a.outputs;
    const T* from = reinterpret_cast<const T*>(a.dy + (long long)token * a.stride) + n;
    if constexpr (sizeof(T) == 2) {
        reinterpret_cast<T*>(a.out)[i] = there ? *from : Elem<T>::from_f(0.0f);
    } else {
        const float x = there ? *from : 0.0f;
        unsigned part[3];
        float rest = x;
#pragma unroll
        for (int p = 0; p < 3; ++p) {  // the leading eight bits of what is left, cut off and not rounded: the rest is exact, and nothing overflows
            part[p] = __float_as_uint(rest) >> 16;
            rest -= __uint_as_float(part[p] << 16);
        }
        if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) {
            part[0] = x != x ? 0x7fc0u : part[0];
            part[1] = part[2] = 0u;
        }
        unsigned short* out = reinterpret_cast<unsigned short*>(a.out);
#pragma unroll
        for (int p = 0; p < 3; ++p) out[(u64)p * a.tokens * a.pitch + i] = (unsigned short)part[p];
    }
}

struct Plan {
    unsigned parts = 1, pitch = 0, feature_tiles = 0, output_tiles = 0, steps_of_part = 0, steps_of_tile = 0, steps = 0, pairs = 0;
    bool copied = false;
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
    B2_CUDA(cudaOccupancyMaxActiveClusters(&clusters, weight_grad_kernel<__nv_bfloat16, true>, &config));
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
    const void* kernels[] = {(const void*)weight_grad_kernel<float, false>, (const void*)weight_grad_kernel<float, true>,
                             (const void*)weight_grad_kernel<__half, false>, (const void*)weight_grad_kernel<__half, true>,
                             (const void*)weight_grad_kernel<__nv_bfloat16, false>, (const void*)weight_grad_kernel<__nv_bfloat16, true>};
    for (const void* k : kernels) B2_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kShared));
    if (device >= 0 && device < 64) done[device] = true;
}

int current_device() {
    int device = 0;
    B2_CUDA(cudaGetDevice(&device));
    return device;
}

Plan plan_of(const WeightGradCall& c) {
    Plan p;
    const std::size_t bytes = c.dtype == DType::Float ? 4 : 2;
    p.parts = c.dtype == DType::Float ? 3 : 1;
    p.copied = c.dtype == DType::Float || (reinterpret_cast<std::uintptr_t>(c.dy) % 16) != 0 || (c.stride * (long long)bytes) % 16 != 0 ||
               c.stride < (long long)c.outputs;
    p.pitch = (unsigned)((c.outputs + 7) / 8 * 8);
    p.feature_tiles = (unsigned)((c.inputs + kTile - 1) / kTile);
    p.output_tiles = (unsigned)((c.outputs + kTile - 1) / kTile);
    const u64 steps_of_part = (c.tokens + kStep - 1) / kStep, tiles = (u64)p.feature_tiles * p.output_tiles;
    B2_REQUIRE(steps_of_part * p.parts * tiles < (1ull << 31) && tiles < (1ull << 24) && c.tokens < (1ull << 31),
               "weight_grad8: too many tokens, inputs and outputs for one call");
    p.steps_of_part = (unsigned)steps_of_part;
    p.steps_of_tile = p.steps_of_part * p.parts;
    p.steps = p.steps_of_tile * (unsigned)tiles;
    const int device = current_device();
    prepare_device(device);
    // Four steps of a pair at least: less, and the pieces cost more than the sums (a piece is 256 KiB to write and read again).
    p.pairs = std::max(1u, std::min(pairs_of_device(device), p.steps / 4u));
    const std::size_t copy = p.copied ? (std::size_t)p.parts * c.tokens * p.pitch * 2 : 0;
    p.pieces_at = (copy + 255) / 256 * 256;
    p.bias_at = p.pieces_at + (std::size_t)2 * p.pairs * kTile * kTile * sizeof(float);
    p.bytes = p.bias_at + (c.bias_grad != nullptr ? (tiles + p.pairs) * kTile * sizeof(float) : 0);
    return p;
}

// A word of host memory that a kernel whose wait ran out writes to.
unsigned* status_word() {
    static unsigned* word = [] {
        // (Allocating is allowed beside a capture: nothing of it belongs to the graph.)
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        B2_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
        void* p = nullptr;
        const cudaError_t st = cudaHostAlloc(&p, sizeof(unsigned), cudaHostAllocMapped | cudaHostAllocPortable);
        cudaThreadExchangeStreamCaptureMode(&mode);
        B2_CUDA(st);
        *static_cast<unsigned*>(p) = 0;
        return static_cast<unsigned*>(p);
    }();
    return word;
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
        l.tokens = c.tokens;
        l.outputs = (unsigned)c.outputs;
        l.pitch = p.pitch;
        const u64 ctas = ((u64)c.tokens * p.pitch + 255) / 256;
        B2_REQUIRE(ctas < (1ull << 31), "weight_grad8: dy is too large for one call");
        B2_CUDA(launch_dependent<LayOutArgs>(lay_out_kernel<T>, dim3((unsigned)ctas), 256, 0, c.stream, l));
        dy = workspace;
        row_bytes = (u64)p.pitch * 2;
    }
    WeightGradArgs a;
    const auto encode = cu::api().TensorMapEncodeTiled;
    if (encode == nullptr) throw std::runtime_error("weight_grad8: the driver does not export cuTensorMapEncodeTiled");
    const cuuint64_t extent[3] = {c.outputs, c.tokens, p.parts};
    const cuuint64_t strides[2] = {row_bytes, row_bytes * c.tokens};
    const cuuint32_t box[3] = {64, kStep, 1}, element_strides[3] = {1, 1, 1};
    cu::check(encode(&a.dy, sizeof(T) == 2 && std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                     const_cast<void*>(dy), extent, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
              "weight_grad8: tensor map of dy");
    a.codes = c.codes;
    a.scales = c.scales;
    a.out = c.weight_grad;
    a.pieces = reinterpret_cast<float*>(workspace + p.pieces_at);
    a.bias = c.bias_grad != nullptr ? reinterpret_cast<float*>(workspace + p.bias_at) : nullptr;
    a.status = status_word();
    a.pitch = (c.inputs + kBlock8 - 1) / kBlock8 * kBlock8;
    a.tokens = (unsigned)c.tokens;
    a.inputs = (unsigned)c.inputs;
    a.outputs = (unsigned)c.outputs;
    a.feature_tiles = p.feature_tiles;
    a.steps_of_part = p.steps_of_part;
    a.steps_of_tile = p.steps_of_tile;
    a.steps = p.steps;
    a.pairs = p.pairs;
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
    B2_CUDA(cudaLaunchKernelEx(&config, c.bias_grad != nullptr ? weight_grad_kernel<T, true> : weight_grad_kernel<T, false>, a));
    bool cut = false;
    for (unsigned i = 1; i < p.pairs; ++i) cut |= first_step(i, p.steps, p.pairs) % p.steps_of_tile != 0;
    if (!cut && c.bias_grad == nullptr) return;
    FinishArgs f;
    f.out = c.weight_grad;
    f.bias_out = c.bias_grad;
    f.pieces = a.pieces;
    f.bias = a.bias;
    f.inputs = a.inputs;
    f.outputs = a.outputs;
    f.feature_tiles = p.feature_tiles;
    f.steps_of_tile = p.steps_of_tile;
    f.steps = p.steps;
    f.pairs = p.pairs;
    f.piece_ctas = cut ? (p.pairs - 1) * (kTile / kFinishRows) : 0;
    const unsigned grid = f.piece_ctas + (c.bias_grad != nullptr ? p.output_tiles : 0);
    B2_CUDA(launch_dependent<FinishArgs>(finish_kernel<T>, dim3(grid), 256, 0, c.stream, f));
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
    if (__atomic_exchange_n(status_word(), 0u, __ATOMIC_RELAXED) != 0u)
        throw std::runtime_error("weight_grad8: a wait inside an earlier call ran out; that call's gradients are not valid");
    const Plan p = plan_of(c);
    switch (c.dtype) {
        case DType::Float: return launch<float>(c, p);
        case DType::Float16: return launch<__half>(c, p);
        case DType::BFloat16: return launch<__nv_bfloat16>(c, p);
    }
}

}  // namespace b200ccl::kernels
