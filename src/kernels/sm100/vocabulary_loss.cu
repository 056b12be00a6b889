// Losses over a vocabulary, cross entropy and distillation from a teacher's top logits, without the logits in memory, and their gradients.
//
//   z = x w^T / tau,   q = softmax(z) over the vocabulary,   y: the target, or the teacher's distribution over its few entries
//   loss_t = sum_v y (log y - log q) tau^2,   dz = c_t (q - y),   c_t = tau * what comes back to loss_t (over the rows that count, for a mean)
//   dx = dz w,   dw = dz^T x
//
// Four products on the tensor cores, one kernel for all of them (product_kernel): a pair of CTAs works on a tile of 256 x 256 (a gradient of a narrow
// matrix: 256 x 128), 64 elements of the summed axis at a time, the accumulators in tensor memory, twice, so that one tile is worked off while the next is summed.
// Of a CTA's warps one copies by TMA, one issues products, eight work tiles off. The products bound it (8192 x 50257 x 768 bf16: tensor pipe 0.95 busy in the gradients, 1.6 PFLOP/s, 0.82 where
// exponentials are made), and in the long run power.
//   Stats   x w^T  -> the maximum of each row of a tile and the sum of e^(z - maximum) (cross entropy: of the words beside the target), joined by join_kernel; the logits that count by the way
//   Probs   x w^T  -> P = r_t (q - y) for a piece of the vocabulary, in 16 bits, to memory
//   WeightGrad  P^T x,   InputGrad  P w   of that piece
// So the backward pass makes the logits a second time, a third more than the products that it cannot do without; keeping them would take 2 to 4 bytes for every token
// and word of the vocabulary, from the forward pass on. Pieces of the vocabulary and not of the tokens, because a piece of dw is then
// complete; dx, which is small, is added up in 32 bits.
//
// bf16, one loss for all rows (both()): its gradient is known but for a factor when the loss is made, and bf16 has the exponents to do without a second product of
// logits. What is stored of a piece of the rows is E = 2^((z - r_t) log2(e) / tau), r_t being the target's logit (that of the entry which the teacher is surest of), which a small kernel makes first:
//   Exps  x w^T -> E in 16 bits, and its sums S_t over the words of a tile; close_kernel joins them and sets E of the targets to E - y S
//   WeightGrad  E^T (x / S),   InputGrad  (E w) / S      (few rows: x / S in two parts)      and the backward pass multiplies by what comes back, if that is not 1
// Where S_t passes 2^64 (a logit is 44 above the target's: E w and x / S have 2^64 to spare, whatever x and w are scaled by) a word in memory says so, and Stats, join_kernel and Probs, which look at it and end otherwise, make P instead.
// 8192 x 50257 x 768, loss and gradients: 2025 -> 1450 us; 4096 x 131072 x 4096: 13.2 -> 10.2 ms.
//
// P is the operand of two products and therefore of their type: its rounding (2^-8 of each
// element in bf16) is what the gradients lose beside their own. r_t = c_t / max |c| is 1 in a mean or a sum, so that the target's element
// stays -(1 - q); max |c| is multiplied in 32 bits at the end. fp16 has no exponents for a small q: P is 2^14 times as large there. Nor has it any for rows whose c is far below the largest: where
// rows have weights of their own, fp16 and fp32 leave the power of two of c out of P. The gradient of x takes it at the end, that of w with x, which is laid out once more (777 x 32003 x 1003 in fp16: 311 -> 318 us,
// 128 x 512 x 64 78 -> 81).
//
// fp32: x, w and P are sums of two fp16 matrices each, what fp16 makes of an element and what it makes of the rest, after a power of two that brings the largest
// element to 2^14: 22 bits, of elements down to 2^-28 of the largest (which stands for 2^-39 in those below). Three products of the four give theirs; the fourth is 2^-22 of
// it. For logits each row of x has a power of its own, so that no row's loss or gradient depends on how large another is; the gradient of w, which is a sum over rows, takes x
// with one power for all rows that count, laid out a second time (2048 x 768: 6 us).
// (Three bf16 matrices have 24 bits, of any element, and take six products: 2048 x 50257 x 768, loss and gradients, 3362 us, with these 1850.)
// The tensor cores cut what an addition leaves below 24 bits, so the small products come first, and their sums are added up in registers, rounded, after every 256 to 8192
// elements of the summed axis: a loss over columns of 4096 in bf16 is 1.8e-6 off otherwise, all of it in one direction.
//
// P pairs take P whole tiles of a gradient at a time, as long as there are so many. Those that are left are cut along the summed axis, all into the same number of pieces, which go over the pairs
// piece by piece and not tile by tile: pairs are at the same words, or tokens, then, and read them from L2 once one of them has. (Steps dealt out evenly, tile by
// tile: 4096 x 50257 x 768, the gradient of x, 300 us instead of 205, at the rate of HBM.) finish_kernel adds the pieces in order. Nothing depends on timing.
#include "kernels/sm100/vocabulary_loss.h"

#include "core/check.h"
#include "kernels/sm100/lay_out.cuh"
#include "kernels/sm100/pair32.cuh"
#include "kernels/sm100/tcgen05.cuh"
#include "kernels/sm100/vec.cuh"
#include "kernels/sm100/wait_status.h"
#include "mem/cu_driver.h"

#include <algorithm>
#include <cstdint>
#include <mutex>
#include <stdexcept>
#include <type_traits>

namespace b200ccl::kernels {

using namespace b200ccl::dev;

namespace {

using u64 = unsigned long long;

enum class Kind { Stats, Probs, Exps, WeightGrad, InputGrad };

constexpr unsigned kTile = 256;  // of both axes of a pair's tile
constexpr unsigned kHalf = 128;  // of one CTA
constexpr unsigned kStep = 64;   // elements of the summed axis
constexpr unsigned kStages = 6;
constexpr unsigned kBlockBytes = kStep * 128;
constexpr unsigned kOperandBytes = 2 * kBlockBytes;  // a CTA's half of an operand
constexpr unsigned kFirstEpilogueWarp = 4, kEpilogueWarps = 8, kThreads = (kFirstEpilogueWarp + kEpilogueWarps) * 32;
constexpr unsigned kMaxPairs = 74;     // 148 SMs
constexpr unsigned kStagingBytes = 32 * 128;  // of an epilogue warp: 128 bytes of each of its rows
constexpr unsigned kAtStaging = kStages * 2 * kOperandBytes, kAtBarriers = kAtStaging + kEpilogueWarps * kStagingBytes;
constexpr unsigned kShared = kAtBarriers + 256 + 1024;
static_assert(kShared <= 227 * 1024);
constexpr unsigned kTileFloats = kTile * kTile;
// Steps that are summed on the tensor cores alone, of each product: in fp32 and in small products; of logits; of gradients that are rounded to 16 bits. (fp32, 2048 x 50257 x 768, errors of dx and
// dw in the norm: 1.32e-6 and 1.23e-6 with sixteen, 4.0e-7 and 3.6e-7 with four.)
constexpr unsigned kShortChunkSteps = 4, kChunkSteps = 16, kLongChunkSteps = 128;
constexpr unsigned kEntryRounds = kMaxTeacherEntries / 32;  // of a warp through a row's entries
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kHalfScale = 16384.0f;  // of P in fp16

template <typename T>
using OperandOf = std::conditional_t<std::is_same_v<T, __nv_bfloat16>, __nv_bfloat16, __half>;

struct alignas(64) ProductArgs {
    CUtensorMap a, b;  // [parts][rows][columns]
    CUtensorMap out;   // P, or a gradient whose rows TMA can write
    unsigned m, n;     // extents of the result that are there
    unsigned m_tiles, n_tiles, n_tile;  // n_tile: extent of a tile along n, 256 or 128
    unsigned products, steps_of_part, steps_of_tile;  // products of parts of the operands
    unsigned chunk;  // steps that are summed on the tensor cores alone, of each of them
    unsigned b_offset;  // added to b's row
    bool b_in_parts;    // two products: b has two parts, and not a
    unsigned pairs, waves;  // whole tiles of a pair
    unsigned left, splits;  // tiles that are left, and the pieces of each
    bool n_first;       // neighbouring tiles lie along n
    float* slots;       // [splits][left][tile]: pieces
    float* sums;        // [tiles][tile]: sums of all pieces of the vocabulary, or null
    bool prior, last;   // there are sums of earlier pieces; this is the last one
    unsigned* status;   // host memory
    u64 wait_ns;
    const unsigned* condition;  // nothing is done while this word is 0, or null
    // Logits
    const unsigned* magnitudes;  // fp32: the largest of each row of x, see scale_of()
    const unsigned* w_magnitude; // fp32: that of w
    float factor, factor_rest;   // log2(e) / temperature, see exponentials()
    unsigned out_parts;          // matrices whose sum P is: fp32, and small products of 16 bits, two
    float2* stats; // [2 * tiles along n][m]
    float* exp_sums;  // the same, of Exps
    float* picked; // [m]
    const void* targets;  // cross entropy: [m]
    long long target_stride;
    bool targets64;
    const int* words;     // distillation: [entries][entry_stride] of each row, -1: none
    const float* probs;   // the teacher's
    float* entry_logits;  // made by Stats and Exps
    unsigned entries, entry_stride;
    const unsigned* hits;  // [words / 128][hit_rows][rounds]: entries whose word is of 128, in some of 32 rows
    unsigned hit_rows;
    const float* top;    // [m]: the largest logit, and the sum of e^(z - top): apart, because of a row that is sure of its target the logarithm of all
    const float* sum;    // would round off what it is not sure of
    const float* rest;   // cross entropy: 1 - q of the target, from the other words' sum
    const float* valid;  // whether the row counts: 1, 0, or NaN
    const float* loss_grad;  // [m], or null: the same for all rows
    long long loss_grad_stride;
    float temperature;
    // Gradients
    float* header;         // of the workspace: max |c|, NaN once a product went wrong, and fp16 and fp32: the power of two that brings x, as the gradient of w takes it, back
    void* gradient;        // rows of n elements
    const float* row_scale;  // [m], or null
    bool wide;             // TMA can write them
};

struct Barriers {
    u64 full[kStages];        // this CTA's operands of a stage have come
    u64 full_other[kStages];  // first CTA: the other's have
    u64 empty[kStages];       // they have been read
    u64 sums[2];              // accumulators are complete
    u64 sums_free[2];         // first CTA: both CTAs have worked theirs off
    u64 drained;              // all products are done
    unsigned tmem;
    unsigned failed;
};
static_assert(sizeof(Barriers) <= 256);

// Where piece i of n of a tile's steps begins.
__host__ __device__ inline unsigned piece_begin(unsigned i, unsigned steps, unsigned n) {
    const unsigned each = steps / n;
    return i * each + i * (steps - each * n) / n;
}

// What a pair does, in order: `waves` whole tiles, then pieces of those that are left. A run of steps of one tile:
struct Run {
    unsigned tile, from, to;
    bool whole;     // this pair sums all of the tile
    unsigned slot;  // of a piece
};
struct Share {
    unsigned pair, runs;
    __device__ __forceinline__ Share(const ProductArgs& a, unsigned p) : pair(p) {
        const unsigned pieces = a.left * a.splits;
        runs = a.waves + (pair < pieces ? (pieces - pair + a.pairs - 1u) / a.pairs : 0u);
    }
    __device__ __forceinline__ Run at(const ProductArgs& a, unsigned i) const {
        if (i < a.waves) return {i * a.pairs + pair, 0u, a.steps_of_tile, true, 0u};
        const unsigned piece = pair + (i - a.waves) * a.pairs, part = piece / a.left;
        Run r;
        r.tile = a.waves * a.pairs + (piece - part * a.left);
        r.from = piece_begin(part, a.steps_of_tile, a.splits);
        r.to = piece_begin(part + 1u, a.steps_of_tile, a.splits);
        r.whole = a.splits == 1u;
        r.slot = piece;
        return r;
    }
};
// The end of the part of a run, from step k on, that is summed on the tensor cores alone.
__device__ __forceinline__ unsigned segment_end(const ProductArgs& a, unsigned k, unsigned to) {
    const unsigned chunk = a.products * a.chunk;
    return min(to, (k / chunk + 1u) * chunk);
}
// Which parts of the operands, and which 64 elements, the steps of a tile take, one after another: of a chunk of steps the products with the smallest sums first. Three products:
// (1, 0), (0, 1), (0, 0); two, of a P of two parts with a matrix of one: (1, 0), (0, 0), or the other way round. (Divided out for each step, the copying thread would be slower than the products.)
struct Spot {
    unsigned product, step, from, to;  // of the chunk
    __device__ __forceinline__ Spot(const ProductArgs& a, unsigned k) {
        const unsigned chunk = k / (a.products * a.chunk), in_chunk = k - chunk * (a.products * a.chunk);
        from = chunk * a.chunk;
        to = min(from + a.chunk, a.steps_of_part);
        product = in_chunk / (to - from);
        step = from + in_chunk - product * (to - from);
    }
    __device__ __forceinline__ void next(const ProductArgs& a) {
        if (++step < to) return;
        step = from;
        if (++product < a.products) return;
        product = 0;
        step = from = to;
        to = min(from + a.chunk, a.steps_of_part);
    }
    __device__ __forceinline__ int part_a(const ProductArgs& a) const { return product == 0u && a.products > 1u && !a.b_in_parts ? 1 : 0; }
    __device__ __forceinline__ int part_b(const ProductArgs& a) const { return a.b_in_parts ? (product == 0u ? 1 : 0) : (product == 1u && a.products == 3u ? 1 : 0); }
};

struct Tile {
    unsigned m, n;  // first element
};
__device__ __forceinline__ Tile tile_at(const ProductArgs& a, unsigned tile) {
    const unsigned along = a.n_first ? a.n_tiles : a.m_tiles, row = tile / along, column = tile - row * along;
    return {(a.n_first ? row : column) * kTile, (a.n_first ? column : row) * a.n_tile};
}

__device__ __forceinline__ void store_shared16(unsigned at, unsigned a, unsigned b, unsigned c, unsigned d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float nan32() { return __uint_as_float(0x7fffffffu); }

// e^((z + off) / tau) of two logits, by powers of two: factor is log2(e) / tau, and factor_rest what rounding it left. fp32: what rounding the product left counts too (of a
// logit 20 below the largest, 1e-6 of the result).
template <typename T>
__device__ __forceinline__ float2 exponentials(float z0, float z1, float off, float factor, float factor_rest) {
    const Pair32 over = add2(pair32(z0, z1), both32(off)), by = both32(factor);
    const float2 p = apart(mul2(over, by));
    float2 e = make_float2(exp2_fast(p.x), exp2_fast(p.y));
    if constexpr (sizeof(T) == 4) {
        const float2 o = apart(over), rest = apart(fma2(over, by, pair32(-p.x, -p.y)));
        // (Nothing is left of infinities.)
        e.x = fabsf(p.x) < 200.0f ? e.x + e.x * (kLn2 * (rest.x + o.x * factor_rest)) : e.x;
        e.y = fabsf(p.y) < 200.0f ? e.y + e.y * (kLn2 * (rest.y + o.y * factor_rest)) : e.y;
    }
    return e;
}

// Element i of a few in registers.
template <unsigned kN>
__device__ __forceinline__ unsigned pick_of(const unsigned (&v)[kN], unsigned i) {
    unsigned r = 0;
#pragma unroll
    for (unsigned n = 0; n < kN; ++n) r = n == i ? v[n] : r;
    return r;
}

// Target `row` of a matrix; -1 where it is negative.
__device__ __forceinline__ long long target_at(const void* targets, bool wide, long long at) {
    const long long v = wide ? static_cast<const long long*>(targets)[at] : static_cast<const int*>(targets)[at];
    return v < 0 ? -1 : v;
}

// 32 columns of a warp's rows to columns 32 * part.. of its 128 bytes of each row (swizzled).
template <typename T>
__device__ __forceinline__ void stage(unsigned staging, unsigned part, const float (&f)[32]) {
    const unsigned lane = threadIdx.x & 31u, row = staging + lane * 128u, turn = lane & 7u;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (unsigned j = 0; j < 8; ++j)
            store_shared16(row + ((j ^ turn) << 4), __float_as_uint(f[4 * j]), __float_as_uint(f[4 * j + 1]), __float_as_uint(f[4 * j + 2]), __float_as_uint(f[4 * j + 3]));
    } else {
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) {
            unsigned w[4];
#pragma unroll
            for (unsigned i = 0; i < 4; ++i)
                w[i] = std::is_same_v<T, __half> ? f2_to_h2(f[8 * j + 2 * i], f[8 * j + 2 * i + 1]) : f2_to_b2(f[8 * j + 2 * i], f[8 * j + 2 * i + 1]);
            store_shared16(row + (((4u * part + j) ^ turn) << 4), w[0], w[1], w[2], w[3]);
        }
    }
}
// The staged rows have been read by the copy before.
__device__ __forceinline__ void staging_free() {
    if ((threadIdx.x & 31u) == 0) tma_wait_group_read<0>();
    __syncwarp();
}
// What was staged, to rows of a tensor map.
__device__ __forceinline__ void staging_out(const CUtensorMap* map, unsigned staging, unsigned column, unsigned row, unsigned part, unsigned rows) {
    fence_shared_async();
    __syncwarp();
    if ((threadIdx.x & 31u) == 0 && row < rows) {
        tma_store_box(map, staging, (int)column, (int)row, (int)part);
        tma_commit_group();
    }
}

// fp32: the power of two that brings a matrix whose largest magnitude has these bits to 2^14 and on, and back. (Below 2^-112 the largest stays smaller.)
__device__ __forceinline__ float scale_of(unsigned magnitude, bool back) {
    const int e = min(14 - ((int)(magnitude >> 23) - 127), 126);
    return __uint_as_float((unsigned)((back ? -e : e) + 127) << 23);
}

// max |c| and whether anything went wrong, in the first words of a gradient's workspace, and what P and the other operand were scaled with.
template <Kind kKind, typename T>
__device__ __forceinline__ float gradient_scale(const float* header, const unsigned* w_magnitude) {
    float scale = header[0] + header[1];
    if constexpr (!std::is_same_v<T, __nv_bfloat16>) scale *= 1.0f / kHalfScale * (kKind == Kind::WeightGrad ? header[2] : 1.0f);
    if constexpr (sizeof(T) == 4 && kKind != Kind::WeightGrad) scale *= scale_of(*w_magnitude, true);
    return scale;
}

// The power of two of a row's c, which fp16 and fp32 leave out of P: the largest that is not above it, 1 of an infinite c and NaN.
__device__ __forceinline__ float power_of(float c) {
    const unsigned exponent = __float_as_uint(c) & 0x7f800000u;
    return exponent == 0x7f800000u ? 1.0f : __uint_as_float(max(exponent, 0x00800000u));
}
// c_t over that power, in bf16 over max |c| of those that are numbers; 0 of rows that do not count. An infinite c, or NaN, stays what it is, in its own row.
template <bool kHalfType>
__device__ __forceinline__ float row_weight(float valid, const float* loss_grad, long long stride, float temperature, float largest, unsigned row) {
    if (loss_grad == nullptr || valid == 0.0f) return valid;
    const float c = loss_grad[(long long)row * stride] * temperature;
    if (!(fabsf(c) < __int_as_float(0x7f800000))) return c * valid;
    if (kHalfType) return c / power_of(c) * valid;
    return largest == 0.0f ? 0.0f * valid : c * valid / largest;
}

// After a wait that ran out: all that this CTA was to make is NaN.
template <Kind kKind, typename T>
__device__ __noinline__ void spoil(const ProductArgs& a, const Share& share, unsigned rank) {
    if (kKind == Kind::Probs && threadIdx.x == 0) a.header[1] = nan32();
    for (unsigned i = kKind == Kind::Probs ? share.runs : 0; i < share.runs; ++i) {
        const Run r = share.at(a, i);
        const Tile t = tile_at(a, r.tile);
        if constexpr (kKind == Kind::Stats || kKind == Kind::Exps) {
            const unsigned row = t.m + rank * kHalf + threadIdx.x % kHalf;
            if (threadIdx.x < kHalf && row < a.m) {
                for (unsigned group = 0; group < 2; ++group) {
                    const u64 at = (u64)(2u * (t.n / kTile) + group) * a.m + row;
                    if constexpr (kKind == Kind::Stats) a.stats[at] = make_float2(nan32(), nan32());
                    else a.exp_sums[at] = nan32();
                }
            }
        } else {
            float* sums = r.whole ? a.sums + (u64)r.tile * kTileFloats : a.slots + (u64)r.slot * kTileFloats;
            const bool gradient = r.whole && a.last;
            for (unsigned e = threadIdx.x; e < kHalf * a.n_tile; e += kThreads) {
                const unsigned row = rank * kHalf + e % kHalf, column = e / kHalf;
                if (!gradient) sums[((column / 4u) * kTile + row) * 4u + column % 4u] = nan32();
                else if (t.m + row < a.m && t.n + column < a.n) static_cast<T*>(a.gradient)[(u64)(t.m + row) * a.n + t.n + column] = Elem<T>::from_f(nan32());
            }
        }
    }
}

// T: type of x, w and their gradients. kLong: runs of several segments, whose sums are added up in registers: that unrolls what is made of them four times, which costs short runs a tenth.
// kTeacher: rows of logits have several words that count, and not one.
template <Kind kKind, typename T, bool kLong, bool kTeacher>
__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ ProductArgs a) {
    constexpr bool kLogits = kKind == Kind::Stats || kKind == Kind::Probs || kKind == Kind::Exps;
    constexpr bool kAByRows = kKind == Kind::WeightGrad, kBByRows = !kLogits;
    constexpr bool kHalfType = !std::is_same_v<T, __nv_bfloat16>;
    using Operand = OperandOf<T>;
    constexpr unsigned kUnit = !kLogits && sizeof(T) == 4 ? 1 : 2;  // 32 columns that are worked off at a time: 128 bytes of what is written
    extern __shared__ unsigned char raw[];
    // Swizzled operands start at multiples of 1024 bytes; the same place in both CTAs.
    unsigned char* shared = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    Barriers& bars = *reinterpret_cast<Barriers*>(shared + kAtBarriers);
    volatile unsigned* failed = &bars.failed;
    const unsigned base = smem_addr(shared);
    const unsigned warp = threadIdx.x / 32u, lane = threadIdx.x & 31u;
    const unsigned rank = cluster_rank();
    const Share share(a, blockIdx.x / 2u);
    const unsigned b_rows = a.n_tile / 2u;  // of a CTA

    if ((kKind == Kind::Stats || kKind == Kind::Probs) && a.condition != nullptr) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (*a.condition == 0u) return;  // (both CTAs of a pair read the same)
    }
    if (warp == 0 && lane == 0) {
        for (unsigned s = 0; s < kStages; ++s) {
            mbar_init(&bars.full[s], 1);
            mbar_init(&bars.full_other[s], 1);
            mbar_init(&bars.empty[s], 1);
        }
        for (unsigned i = 0; i < 2; ++i) {
            mbar_init(&bars.sums[i], 1);
            mbar_init(&bars.sums_free[i], 2 * kEpilogueWarps);
        }
        mbar_init(&bars.drained, 1);
        bars.failed = 0;
        mbar_fence_init();
        tma_prefetch_map(&a.a);
        tma_prefetch_map(&a.b);
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
    const auto operand_a = [&](unsigned stage) { return base + stage * (2u * kOperandBytes); };
    const auto operand_b = [&](unsigned stage) { return base + stage * (2u * kOperandBytes) + kOperandBytes; };
    if (warp == 0) {
        if (lane == 0) {
            const unsigned bytes = kOperandBytes + b_rows * 128u;
            unsigned n = 0;
            bool ok = true;
            for (unsigned i = 0; i < share.runs && ok; ++i) {
                const Run r = share.at(a, i);
                const Tile t = tile_at(a, r.tile);
                const int m = (int)(t.m + rank * kHalf), at = (int)(t.n + rank * b_rows);
                Spot spot(a, r.from);
                for (unsigned k = r.from; k < r.to; ++k, ++n, spot.next(a)) {
                    const unsigned s = n % kStages;
                    const int step = (int)(spot.step * kStep);
                    ok = wait_phase(bar(bars.empty[s]), ((n / kStages) & 1u) ^ 1u, failed, a.wait_ns);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&bars.full[s], bytes);
                    if constexpr (kAByRows) {
                        tma_load_box(operand_a(s), &a.a, m, step, spot.part_a(a), bar(bars.full[s]));
                        tma_load_box(operand_a(s) + kBlockBytes, &a.a, m + 64, step, spot.part_a(a), bar(bars.full[s]));
                    } else {
                        tma_load_box(operand_a(s), &a.a, step, m, spot.part_a(a), bar(bars.full[s]));
                    }
                    if constexpr (kBByRows) {
                        for (unsigned b = 0; b < b_rows / 64u; ++b)
                            tma_load_box(operand_b(s) + b * kBlockBytes, &a.b, at + (int)(b * 64u), step + (int)a.b_offset, spot.part_b(a), bar(bars.full[s]));
                    } else {
                        tma_load_box(operand_b(s), &a.b, step, at + (int)a.b_offset, spot.part_b(a), bar(bars.full[s]));
                    }
                }
            }
            // Stages have been given back, and after a failure copies have landed, before the CTA ends.
            for (unsigned i = n > kStages ? n - kStages : 0; i < n; ++i) {
                if (ok) wait_phase(bar(bars.empty[i % kStages]), (i / kStages) & 1u, failed, a.wait_ns);
                for (unsigned polls = 0; polls < 1000u && !phase_over<false>(bar(bars.full[i % kStages]), (i / kStages) & 1u); ++polls) {}
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const unsigned shape = product_shape(kTile, a.n_tile, !kHalfType, kAByRows, kBByRows);
            unsigned n = 0, segments = 0;
            bool ok = true;
            for (unsigned i = 0; i < share.runs && ok; ++i) {
                const Run r = share.at(a, i);
                for (unsigned k = r.from; k < r.to && ok; ++segments) {
                    const unsigned end = segment_end(a, k, r.to), buffer = segments & 1u;
                    ok = wait_phase<true>(bar(bars.sums_free[buffer]), ((segments >> 1) & 1u) ^ 1u, failed, a.wait_ns);
                    if (!ok) break;
                    tcgen05_fence_after();
                    for (bool add = false; k < end; ++k, ++n) {
                        const unsigned s = n % kStages, parity = (n / kStages) & 1u;
                        ok = wait_phase(bar(bars.full[s]), parity, failed, a.wait_ns) && wait_phase<true>(bar(bars.full_other[s]), parity, failed, a.wait_ns);
                        if (!ok) break;
                        tcgen05_fence_after();
                        // 16 elements of the summed axis: 2048 bytes of rows, 32 bytes of columns
                        const std::uint64_t x = kAByRows ? operand_by_rows(operand_a(s), kBlockBytes) : operand_by_columns(operand_a(s));
                        const std::uint64_t y = kBByRows ? operand_by_rows(operand_b(s), kBlockBytes) : operand_by_columns(operand_b(s));
#pragma unroll
                        for (unsigned j = 0; j < kStep / 16; ++j) {
                            mma_pair(tmem + buffer * kTile, x + j * (kAByRows ? 2048 >> 4 : 32 >> 4), y + j * (kBByRows ? 2048 >> 4 : 32 >> 4), shape, add);
                            add = true;
                        }
                        commit_pair(bar(bars.empty[s]));
                    }
                    if (!ok) break;
                    commit_pair(bar(bars.sums[buffer]));
                }
            }
            // Products under way read shared memory and write tensor memory of both CTAs. Where a wait ran out, nobody else may be waiting for them.
            commit_pair(bar(bars.drained));
            for (unsigned polls = 0; polls < 1000u && !phase_over<false>(bar(bars.drained), 0); ++polls) {}
        } else if (lane == 0) {
            unsigned steps = 0;
            for (unsigned i = 0; i < share.runs; ++i) {
                const Run r = share.at(a, i);
                steps += r.to - r.from;
            }
            for (unsigned n = 0; n < steps; ++n) {
                if (!wait_phase(bar(bars.full[n % kStages]), (n / kStages) & 1u, failed, a.wait_ns)) break;
                mbar_arrive_at(bar(bars.full_other[n % kStages]), 0);
            }
            if (!wait_phase(bar(bars.drained), 0, failed, a.wait_ns))
                for (unsigned polls = 0; polls < 1000u && !phase_over<false>(bar(bars.drained), 0); ++polls) {}
        }
    } else if (warp >= kFirstEpilogueWarp) {
        const unsigned quarter = warp & 3u, group = (warp - kFirstEpilogueWarp) / 4u;  // lanes of tensor memory that this warp reaches; its half of the columns
        const unsigned in_tile = rank * kHalf + quarter * 32u, column0 = group * b_rows;
        const unsigned staging = base + kAtStaging + (warp - kFirstEpilogueWarp) * kStagingBytes;
        float scale = 1.0f;
        if constexpr (!kLogits) scale = gradient_scale<kKind, T>(a.header, a.w_magnitude);
        Pair32 back_x = both32(1.0f), back_w = both32(1.0f);
        if constexpr (kLogits && sizeof(T) == 4) back_w = both32(scale_of(*a.w_magnitude, true));
        const float low = -__int_as_float(0x7f800000);
        unsigned segments = 0;
        for (unsigned i = 0; i < share.runs; ++i) {
            const Run r = share.at(a, i);
            const Tile t = tile_at(a, r.tile);
            const unsigned first = t.n + column0, row = t.m + in_tile + lane;
            const unsigned columns = first < a.n ? min(b_rows, a.n - first) : 0u;  // of this warp
            // What a row of logits needs beside them: the columns of this warp's that count in it.
            long long target = -1;
            constexpr unsigned kNear = kTeacher ? 6 : 1;
            unsigned hits[kTeacher ? kEntryRounds : 1] = {};  // kTeacher: entries that are here in some row of the warp,
            unsigned near_column[kNear] = {};                 // and the columns of the first few in this row
            const long long first_word = (long long)(first + a.b_offset);
            float weight = 0.0f, row_top = 0.0f, share_of_sum = 1.0f, of_target = 0.0f;
            if constexpr (kLogits) {
                if constexpr (kTeacher) {
                    const unsigned rounds = (a.entries + 31u) / 32u;
                    const unsigned* here = a.hits + ((u64)((unsigned)first_word / kHalf) * a.hit_rows + (t.m + in_tile) / 32u) * rounds;
                    const bool any = columns != 0u && t.m + in_tile < a.m;
#pragma unroll
                    for (unsigned b = 0; b < kEntryRounds; ++b) hits[b] = any && b < rounds ? here[b] : 0u;
                    // The words of the first few are read all at once, while the products are made.
                    unsigned round = 0, rest = hits[0];
#pragma unroll
                    for (unsigned i = 0; i < kNear; ++i) {
                        while (rest == 0u && round + 1u < rounds) rest = pick_of(hits, ++round);
                        const unsigned entry = rest != 0u ? 32u * round + (unsigned)__ffs((int)rest) - 1u : 0u;
                        near_column[i] = (unsigned)a.words[(u64)entry * a.entry_stride + min(row, a.m - 1u)];
                        rest &= rest - 1u;
                    }
#pragma unroll
                    for (unsigned i = 0; i < kNear; ++i) {
                        const long long column = (long long)(int)near_column[i] - first_word;
                        near_column[i] = row < a.m && column >= 0 && column < (long long)columns ? (unsigned)column : 0xffffffffu;
                    }
                }
                if (row < a.m) {
                    if constexpr (sizeof(T) == 4) back_x = both32(scale_of(a.magnitudes[row], true));
                    if constexpr (!kTeacher) target = target_at(a.targets, a.targets64, (long long)row * a.target_stride);
                    if constexpr (kKind == Kind::Probs) {
                        weight = row_weight<kHalfType>(a.valid[row], a.loss_grad, a.loss_grad_stride, a.temperature, a.header[0], row) * (kHalfType ? kHalfScale : 1.0f);
                        row_top = a.top[row];
                        share_of_sum = weight / a.sum[row];
                        if constexpr (!kTeacher) of_target = -weight * a.rest[row];
                    } else if constexpr (kKind == Kind::Exps) {
                        weight = a.valid[row];
                        row_top = a.top[row];
                    }
                }
                target = target < 0 ? -1 : target - first_word;
            }
            const unsigned own_target = target >= 0 && target < (long long)columns ? (unsigned)target : 0xffffffffu;  // its column of this warp's
            // What is made of `kUnit` times 32 columns of sums, from the warp's column c on.
            float top = low, sum = 0.0f, some[4] = {};
            float* sums = nullptr;
            float of_row = 1.0f;
            if constexpr (!kLogits) {
                sums = r.whole ? a.sums + (u64)r.tile * kTileFloats : a.slots + (u64)r.slot * kTileFloats;
                of_row = kKind == Kind::InputGrad && a.row_scale != nullptr && row < a.m ? scale * a.row_scale[row] : scale;
            }
            // f(column of the 32 from c on, entry, its place) for every entry that is there in some row; in the others the column is above 31.
            const auto each_entry = [&](unsigned c, auto&& f) {
                if constexpr (kTeacher) {
                    // (One body for all of them: unrolled, the code is more than the instruction cache holds beside the products' own.)
                    unsigned n = 0;
#pragma unroll 1
                    for (unsigned round = 0; 32u * round < a.entries; ++round) {
#pragma unroll 1
                        for (unsigned left = pick_of(hits, round); left != 0u; left &= left - 1u, ++n) {
                            const u64 place = (u64)(32u * round + (unsigned)__ffs((int)left) - 1u) * a.entry_stride + row;
                            unsigned column = 0xffffffffu;
                            if (n < kNear) {
                                column = pick_of(near_column, n);
                            } else if (row < a.m) {
                                const long long at = (long long)a.words[place] - first_word;
                                column = at >= 0 && at < (long long)columns ? (unsigned)at : 0xffffffffu;
                            }
                            column -= c;
                            if (__any_sync(0xffffffffu, column < 32u)) f(column, place);
                        }
                    }
                }
            };
            const auto work_off = [&](unsigned c, float (&f)[kUnit][32]) {
                if constexpr (kLogits && sizeof(T) == 4) {
#pragma unroll
                    for (unsigned h = 0; h < kUnit; ++h) {
#pragma unroll
                        for (unsigned j = 0; j < 32; j += 2) {
                            const float2 z = apart(mul2(mul2(pair32(f[h][j], f[h][j + 1]), back_x), back_w));
                            f[h][j] = z.x;
                            f[h][j + 1] = z.y;
                        }
                    }
                }
                if constexpr (kKind == Kind::Stats) {
#pragma unroll
                    for (unsigned h = 0; h < kUnit; ++h) {
                        if (c + 32u * h + 32u > columns) {
#pragma unroll
                            for (unsigned j = 0; j < 32; ++j) f[h][j] = c + 32u * h + j < columns ? f[h][j] : low;
                        }
                        const unsigned at = own_target - (c + 32u * h);
                        const auto pick = [&](unsigned column, float* to) {
                            float z = 0.0f;
#pragma unroll
                            for (unsigned j = 0; j < 32; ++j) z = j == column ? f[h][j] : z;
                            if (column < 32u) *to = z;
                        };
                        if (!kTeacher && __any_sync(0xffffffffu, at < 32u)) {
                            pick(at, a.picked + row);
                            // (Sums are of the other words: beside the target's 1, what they leave of a sure row would be lost.)
#pragma unroll
                            for (unsigned j = 0; j < 32; ++j) f[h][j] = j == at ? low : f[h][j];
                        }
                        each_entry(c + 32u * h, [&](unsigned column, u64 place) { pick(column, a.entry_logits + place); });
                        float most[4] = {f[h][0], f[h][1], f[h][2], f[h][3]};
#pragma unroll
                        for (unsigned j = 4; j < 32; ++j) most[j & 3u] = fmaxf(most[j & 3u], f[h][j]);
                        const float now = fmaxf(top, fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])));
                        const float off = now == low ? 0.0f : -now;
                        float parts[4] = {sum * exp2_fast((top + off) * a.factor), 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (unsigned j = 0; j < 32; j += 2) {
                            const float2 e = exponentials<T>(f[h][j], f[h][j + 1], off, a.factor, a.factor_rest);
                            parts[j & 2u] += e.x;
                            parts[(j & 2u) + 1u] += e.y;
                        }
                        sum = (parts[0] + parts[1]) + (parts[2] + parts[3]);
                        top = now;
                    }
                } else if constexpr (kLogits) {
#pragma unroll
                    for (unsigned h = 0; h < 2; ++h) {
                        const unsigned at = own_target - (c + 32u * h);
                        if constexpr (kKind == Kind::Exps) {
                            each_entry(c + 32u * h, [&](unsigned column, u64 place) {
                                float z = 0.0f;
#pragma unroll
                                for (unsigned j = 0; j < 32; ++j) z = j == column ? f[h][j] : z;
                                if (column < 32u) a.entry_logits[place] = z;
                            });
                        }
#pragma unroll
                        for (unsigned j = 0; j < 32; j += 2) {
                            const float2 e = exponentials<T>(f[h][j], f[h][j + 1], -row_top, a.factor, a.factor_rest);
                            f[h][j] = kKind == Kind::Probs ? share_of_sum * e.x : e.x;
                            f[h][j + 1] = kKind == Kind::Probs ? share_of_sum * e.y : e.y;
                        }
                        if constexpr (kKind == Kind::Probs) {
                            each_entry(c + 32u * h, [&](unsigned column, u64 place) {
                                const float off = column < 32u ? weight * a.probs[place] : 0.0f;
#pragma unroll
                                for (unsigned j = 0; j < 32; ++j) f[h][j] -= j == column ? off : 0.0f;
                            });
                        }
                        if (!kTeacher && __any_sync(0xffffffffu, at < 32u)) {
                            // (Exps: the target's is 1 by definition, its logit was made by another kernel, whose roundings differ. Sums are of the others alone, so that nothing is
                            // lost of a row that is sure of its target, and close_kernel makes the element itself.)
#pragma unroll
                            for (unsigned j = 0; j < 32; ++j) f[h][j] = j != at ? f[h][j] : (kKind == Kind::Probs ? of_target : 0.0f);
                        }
                        if (c + 32u * h + 32u > columns) {
#pragma unroll
                            for (unsigned j = 0; j < 32; ++j) f[h][j] = c + 32u * h + j < columns ? f[h][j] : 0.0f;
                        }
                        if (weight == 0.0f) {
#pragma unroll
                            for (unsigned j = 0; j < 32; ++j) f[h][j] = 0.0f;
                        }
                        if constexpr (kKind == Kind::Exps) {
#pragma unroll
                            for (unsigned j = 0; j < 32; ++j) some[j & 3u] += f[h][j];
                        }
                    }
                    for (unsigned part = 0; part < a.out_parts; ++part) {
                        staging_free();
#pragma unroll
                        for (unsigned h = 0; h < 2; ++h) {
                            stage<Operand>(staging, h, f[h]);
                            if (part + 1u == a.out_parts) continue;
#pragma unroll
                            for (unsigned j = 0; j < 32; ++j) f[h][j] -= Elem<Operand>::to_f(Elem<Operand>::from_f(f[h][j]));
                        }
                        staging_out(&a.out, staging, first + c, t.m + in_tile, part, a.m);
                    }
                } else {
                    // Sums of earlier pieces of the summed axis, and those that are not done: four columns of a row, beside those of the next.
                    float4* kept = reinterpret_cast<float4*>(sums) + ((column0 + c) / 4u) * kTile + in_tile + lane;
                    if (r.whole && a.prior) {
#pragma unroll
                        for (unsigned j = 0; j < 8 * kUnit; ++j) {
                            const float4 v = kept[j * kTile];
                            float* const to = &f[j / 8u][4u * (j & 7u)];
                            to[0] += v.x;
                            to[1] += v.y;
                            to[2] += v.z;
                            to[3] += v.w;
                        }
                    }
                    if (!r.whole || !a.last) {
#pragma unroll
                        for (unsigned j = 0; j < 8 * kUnit; ++j) {
                            const float* const from = &f[j / 8u][4u * (j & 7u)];
                            kept[j * kTile] = make_float4(from[0], from[1], from[2], from[3]);
                        }
                        return;
                    }
                    staging_free();
#pragma unroll
                    for (unsigned h = 0; h < kUnit; ++h) {
#pragma unroll
                        for (unsigned j = 0; j < 32; ++j) f[h][j] *= of_row;
                        stage<T>(staging, h, f[h]);
                    }
                    if (a.wide) {
                        staging_out(&a.out, staging, first + c, t.m + in_tile, 0, a.m);
                    } else {
                        __syncwarp();
                        const unsigned rows = t.m + in_tile < a.m ? min(32u, a.m - t.m - in_tile) : 0u;
                        T* to = static_cast<T*>(a.gradient) + (u64)(t.m + in_tile) * a.n + first + c;
#pragma unroll 8
                        for (unsigned s = 0; s < 32u; ++s) {
#pragma unroll
                            for (unsigned h = 0; h < kUnit; ++h) {
                                const unsigned j = lane + 32u * h, at = j * (unsigned)sizeof(T);
                                const T v = *reinterpret_cast<const T*>(shared + (staging - base) + s * 128u + (((at >> 4) ^ (s & 7u)) << 4) + (at & 15u));
                                if (s < rows && c + j < columns) to[(u64)s * a.n + j] = v;
                            }
                        }
                        __syncwarp();
                    }
                }
            };
            const auto wait_sums = [&] {
                const bool ok = __all_sync(0xffffffffu, wait_phase(bar(bars.sums[segments & 1u]), (segments >> 1) & 1u, failed, a.wait_ns));
                tcgen05_fence_after();
                return ok;
            };
            const auto free_sums = [&] {
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_at(bar(bars.sums_free[segments & 1u]), 0);
                ++segments;
            };
            if constexpr (!kLong) {
                if (!wait_sums()) break;
                const unsigned from = tmem + (segments & 1u) * kTile + column0 + (quarter * 32u << 16);
                for (unsigned c = 0; c < columns; c += 32u * kUnit) {
                    float f[kUnit][32];
#pragma unroll
                    for (unsigned h = 0; h < kUnit; ++h) {
                        __syncwarp();
                        tmem_load32(from + c + 32u * h, f[h]);
                    }
                    work_off(c, f);
                }
                free_sums();
            } else {
                // The sums of all segments, 128 columns of a row in registers.
                float f[4 / kUnit][kUnit][32];
                bool ok = true;
                for (unsigned k = r.from; k < r.to; k = segment_end(a, k, r.to)) {
                    ok = wait_sums();
                    if (!ok) break;
                    const unsigned from = tmem + (segments & 1u) * kTile + column0 + (quarter * 32u << 16);
#pragma unroll
                    for (unsigned c = 0; c < 4; ++c) {
                        if (32u * c >= b_rows) continue;
                        float more[32];
                        __syncwarp();
                        tmem_load32(from + 32u * c, more);
#pragma unroll
                        for (unsigned j = 0; j < 32; ++j) f[c / kUnit][c % kUnit][j] = k == r.from ? more[j] : f[c / kUnit][c % kUnit][j] + more[j];
                    }
                    free_sums();
                }
                if (!ok) break;
#pragma unroll
                for (unsigned c = 0; c < 4; c += kUnit)
                    if (32u * c < columns) work_off(32u * c, f[c / kUnit]);
            }
            if constexpr (kKind == Kind::Stats) {
                if (row < a.m) a.stats[(u64)(2u * (t.n / kTile) + group) * a.m + row] = make_float2(top, sum);
            } else if constexpr (kKind == Kind::Exps) {
                if (row < a.m) a.exp_sums[(u64)(2u * (t.n / kTile) + group) * a.m + row] = (some[0] + some[1]) + (some[2] + some[3]);
            }
        }
        if (lane == 0) tma_wait_group_all();
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
        spoil<kKind, T>(a, share, rank);
        if (rank == 1 && threadIdx.x == 0)  // (the last arrival from the first CTA)
            for (unsigned polls = 0; polls < 1000u && !phase_over<false>(bar(bars.drained), 0); ++polls) {}
    }
}

struct FinishArgs {
    void* out;           // rows of n elements
    const float* slots;
    float* sums;         // see ProductArgs
    bool prior, last;
    const float* header;
    const float* row_scale;
    const unsigned* w_magnitude;
    unsigned m, n, m_tiles, n_tiles, n_tile, whole_tiles, left, splits;
    bool n_first;
};

// Adds the pieces of cut tiles: 32 rows by 32 columns of a tile for a CTA (a tile that all pairs share has 74 pieces, and few CTAs took 51 us for two of them).
template <Kind kKind, typename T>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ FinishArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned columns = a.n_tile / 32u, blocks = 8u * columns, index = blockIdx.x / blocks, block = blockIdx.x % blocks;
    const unsigned tile = a.whole_tiles + index;
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x / 32u, row0 = block / columns * 32u, column0 = block % columns * 32u;
    const unsigned at = (column0 / 4u + warp) * kTile + row0 + lane;  // four columns of a row
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto add = [&sum](float4 v) {
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
    };
    if (a.prior) add(reinterpret_cast<const float4*>(a.sums + (u64)tile * kTileFloats)[at]);
    constexpr unsigned kAtOnce = 8;
    for (unsigned p = 0; p < a.splits; p += kAtOnce) {
        float4 v[kAtOnce];
#pragma unroll
        for (unsigned i = 0; i < kAtOnce; ++i) {
            const float4* piece = reinterpret_cast<const float4*>(a.slots + (u64)((p + i) * a.left + index) * kTileFloats);
            v[i] = p + i < a.splits ? piece[at] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (unsigned i = 0; i < kAtOnce; ++i) add(v[i]);
    }
    if (!a.last) {
        reinterpret_cast<float4*>(a.sums + (u64)tile * kTileFloats)[at] = sum;
        return;
    }
    const float scale = gradient_scale<kKind, T>(a.header, a.w_magnitude);
    __shared__ float turned[32][33];
    float* t = &turned[lane][warp * 4u];
    t[0] = sum.x * scale;
    t[1] = sum.y * scale;
    t[2] = sum.z * scale;
    t[3] = sum.w * scale;
    __syncthreads();
    const unsigned along = a.n_first ? a.n_tiles : a.m_tiles, tile_row = tile / along, tile_column = tile - tile_row * along;
    const unsigned m0 = (a.n_first ? tile_row : tile_column) * kTile + row0, n = (a.n_first ? tile_column : tile_row) * a.n_tile + column0 + lane;
#pragma unroll
    for (unsigned r = warp; r < 32u; r += 8u)
        if (m0 + r < a.m && n < a.n)
            static_cast<T*>(a.out)[(u64)(m0 + r) * a.n + n] = Elem<T>::from_f(a.row_scale != nullptr ? turned[r][lane] * a.row_scale[m0 + r] : turned[r][lane]);
}

// ---- what stands around the products -----------------------------------------------------------------------

struct JoinArgs {
    const float2* stats;
    unsigned rows, parts;
    const float* picked;  // cross entropy
    const void* targets;
    long long target_stride;
    bool targets64;
    unsigned long long vocabulary;
    const float* z;  // distillation: [entries][entry_stride]
    const float* p;
    unsigned entries, entry_stride;
    float temperature, factor;
    float* top;
    float* sum;
    float* rest;
    float* valid;
    float* loss;
    const unsigned* condition;  // see ProductArgs
    float* row_scale;           // 1 of rows that count, or null
};

// Each row's maximum and sum, those of the words beside the target brought together with it, and its loss. A CTA takes 32 rows, each of its warps every 32nd part of them (1024 rows of 394 parts: eight
// warps took 12 us).
__global__ void __launch_bounds__(1024) join_kernel(const __grid_constant__ JoinArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (a.condition != nullptr && *a.condition == 0u) return;
    constexpr unsigned kWarps = 32;
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x / 32u, row = blockIdx.x * 32u + lane;
    const float low = -__int_as_float(0x7f800000);
    const float factor = a.factor;
    const auto merge = [low, factor](float& top, float& sum, float2 v) {
        const float now = fmaxf(top, v.x), off = now == low ? 0.0f : now;
        sum = sum * exp2f((top - off) * factor) + v.y * exp2f((v.x - off) * factor);
        top = now;
    };
    float top = low, sum = 0.0f;
    if (row < a.rows) {
        for (unsigned p = warp; p < a.parts; p += 4u * kWarps) {
            float2 v[4];
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) v[i] = p + kWarps * i < a.parts ? a.stats[(u64)(p + kWarps * i) * a.rows + row] : make_float2(low, 0.0f);
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) merge(top, sum, v[i]);
        }
    }
    __shared__ float2 all[kWarps][33];
    __shared__ float2 of_row[32];
    all[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (warp == 0) {
        for (unsigned w = 1; w < kWarps; ++w) merge(top, sum, all[w][lane]);
        const float log_sum = log2f(sum);
        of_row[lane] = make_float2(top, log_sum);
        if (row < a.rows) {
            if (a.row_scale != nullptr) a.row_scale[row] = 1.0f;  // (P has the rows' weights in it)
            if (a.entries == 0) {
                const long long target = target_at(a.targets, a.targets64, (long long)row * a.target_stride);
                const bool bad = target >= (long long)a.vocabulary;
                float loss = 0.0f, rest = 0.0f;
                if (target >= 0 && !bad) {
                    // The other words' sum beside the target: the loss is log(1 + odds).
                    const float picked = a.picked[row], over = (top - picked) * factor, odds = sum * exp2f(over);
                    const bool odds_fit = over < 60.0f;
                    loss = odds_fit ? log1pf(odds) : kLn2 * (over + log_sum);
                    rest = odds_fit ? odds / (1.0f + odds) : 1.0f;
                    const float largest = fmaxf(top, picked);
                    sum = sum * exp2f((top - largest) * factor) + exp2f((picked - largest) * factor);
                    top = largest;
                    if (sum != sum) loss = rest = sum;  // (infinite logits, and NaN)
                }
                a.valid[row] = bad ? nan32() : (target < 0 ? 0.0f : 1.0f);
                a.loss[row] = bad ? nan32() : loss;
                a.rest[row] = rest;
            }
            a.top[row] = top;
            a.sum[row] = sum;
        }
    }
    if (a.entries == 0) return;
    __syncthreads();
    const u64 at = (u64)blockIdx.x * 32u + warp;  // a warp for each row
    if (at < a.rows) {
        float loss = 0.0f;
        for (unsigned k = lane; k < a.entries; k += 32u) {
            const float p = a.p[(u64)k * a.entry_stride + at];
            if (p != 0.0f) loss += p * (logf(p) + kLn2 * ((of_row[warp].x - a.z[(u64)k * a.entry_stride + at]) * factor + of_row[warp].y));
        }
#pragma unroll
        for (unsigned d = 16; d != 0; d /= 2) loss += __shfl_xor_sync(0xffffffffu, loss, d);
        const float valid = a.valid[at];
        if (lane == 0) a.loss[at] = valid == 0.0f ? 0.0f : loss * a.temperature * a.temperature * valid;
    }
}

struct SumArgs {
    const float* losses;
    const float* valid;
    unsigned rows;
    bool mean;
    float* out;
    float* count;
};

// The rows' losses in one, in an order that does not depend on timing.
__global__ void __launch_bounds__(1024) sum_kernel(const __grid_constant__ SumArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float sum = 0.0f;
    unsigned count = 0;
#pragma unroll 4
    for (unsigned i = threadIdx.x; i < a.rows; i += 1024u) {
        sum += a.losses[i];
        count += a.valid[i] == 0.0f ? 0u : 1u;
    }
    __shared__ float sums[32];
    __shared__ unsigned counts[32];
#pragma unroll
    for (unsigned d = 16; d != 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    count = __reduce_add_sync(0xffffffffu, count);
    if ((threadIdx.x & 31u) == 0) {
        sums[threadIdx.x / 32u] = sum;
        counts[threadIdx.x / 32u] = count;
    }
    __syncthreads();
    if (threadIdx.x >= 32u) return;
    sum = sums[threadIdx.x];
#pragma unroll
    for (unsigned d = 16; d != 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    count = __reduce_add_sync(0xffffffffu, counts[threadIdx.x]);
    if (threadIdx.x == 0) {
        *a.out = a.mean ? sum / fmaxf((float)count, 1.0f) : sum;
        *a.count = (float)count;
    }
}

struct EntriesArgs {
    const void* x;  // rows at multiples of 16 bytes
    long long x_stride;
    const void* weight;
    long long weight_stride;
    unsigned rows, width, entries;
    unsigned long long vocabulary;
    const void* targets;
    long long target_strides[2];
    bool targets64;
    const void* teacher;  // null: cross entropy, one entry
    int teacher_dtype;
    long long teacher_strides[2];
    float temperature;
    int* words;    // [entries][rows], or null
    float* probs;
    unsigned* hits;  // see ProductArgs; all zeros
    unsigned hit_rows;
    float* valid;
    float* top;    // the logit of the entry that the teacher is surest of, 0 of rows without entries; or null
};

__device__ __forceinline__ float load_as_float(const void* p, int dtype, long long at) {
    if (dtype == 0) return static_cast<const float*>(p)[at];
    return dtype == 1 ? __half2float(static_cast<const __half*>(p)[at]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}

// The teacher's distribution over its entries (cross entropy: the target), and near which logit a row's sum will be. A warp takes a row.
__global__ void __launch_bounds__(256) entries_kernel(const __grid_constant__ EntriesArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned lane = threadIdx.x & 31u, row = blockIdx.x * 8u + threadIdx.x / 32u;
    if (row >= a.rows) return;
    const float low = -__int_as_float(0x7f800000);
    long long token[kEntryRounds];
    float p[kEntryRounds], top = low;
    bool any = false, bad = false;
#pragma unroll
    for (unsigned i = 0; i < kEntryRounds; ++i) {
        const unsigned k = lane + 32u * i;
        token[i] = -1;
        p[i] = low;
        if (k < a.entries) {
            token[i] = target_at(a.targets, a.targets64, (long long)row * a.target_strides[0] + (long long)k * a.target_strides[1]);
            if (token[i] >= 0) p[i] = a.teacher == nullptr ? 0.0f : load_as_float(a.teacher, a.teacher_dtype, (long long)row * a.teacher_strides[0] + (long long)k * a.teacher_strides[1]);
            if (p[i] == low) token[i] = -1;
        }
        any |= token[i] >= 0;
        if (token[i] >= (long long)a.vocabulary) {
            bad = true;
            token[i] = -1;
        }
        top = fmaxf(top, p[i]);
    }
    any = __any_sync(0xffffffffu, any);
    bad = __any_sync(0xffffffffu, bad);
#pragma unroll
    for (unsigned d = 16; d != 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    // The place of the largest, if its word is one; the first of several.
    unsigned surest = 0xffffffffu;
#pragma unroll
    for (unsigned i = kEntryRounds; i-- > 0;) surest = token[i] >= 0 && p[i] == top ? lane + 32u * i : surest;
    surest = __reduce_min_sync(0xffffffffu, surest);
    float sum = 0.0f;
#pragma unroll
    for (unsigned i = 0; i < kEntryRounds; ++i) {
        p[i] = p[i] == low ? 0.0f : expf((p[i] - top) / a.temperature);
        sum += p[i];
    }
#pragma unroll
    for (unsigned d = 16; d != 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) a.valid[row] = bad ? nan32() : (any ? 1.0f : 0.0f);
    if (a.words != nullptr) {
#pragma unroll
        for (unsigned i = 0; i < kEntryRounds; ++i) {
            const unsigned k = lane + 32u * i;
            if (k >= a.entries) break;
            a.words[(u64)k * a.rows + row] = (int)token[i];
            if (token[i] >= 0) atomicOr(a.hits + ((u64)((unsigned)token[i] / kHalf) * a.hit_rows + row / 32u) * ((a.entries + 31u) / 32u) + i, 1u << lane);  // (in any order)
            a.probs[(u64)k * a.rows + row] = any ? p[i] / sum : 0.0f;
        }
    }
    if (a.top == nullptr) return;
    long long word = -1;
#pragma unroll
    for (unsigned i = 0; i < kEntryRounds; ++i) {
        const long long other = __shfl_sync(0xffffffffu, token[i], surest & 31u);
        word = surest / 32u == i ? other : word;
    }
    using T = __nv_bfloat16;
    float z = 0.0f;
    if (word >= 0) {
        const T *x = static_cast<const T*>(a.x) + (long long)row * a.x_stride, *w = static_cast<const T*>(a.weight) + word * a.weight_stride;
#pragma unroll 4
        for (unsigned h = lane * 8u; h < a.width; h += 256u) {
            const unsigned n = min(8u, a.width - h);  // (what lies behind a row may be anything)
            float v[8], u[8];
            Wide<T>::unpack(*reinterpret_cast<const uint4*>(x + h), v);
            Wide<T>::unpack(*reinterpret_cast<const uint4*>(w + h), u);
#pragma unroll
            for (unsigned q = 0; q < 8; ++q) z += q < n ? v[q] * u[q] : 0.0f;
        }
    }
#pragma unroll
    for (unsigned d = 16; d != 0; d /= 2) z += __shfl_xor_sync(0xffffffffu, z, d);
    if (lane == 0) a.top[row] = z;
}

struct HeaderArgs {
    const float* loss_grad;
    long long loss_grad_stride;
    const float* valid;
    const float* count;  // of a mean, or null
    unsigned rows;
    bool each;           // loss_grad has an element for each row
    float* powers;       // of each row's c, or null
    float temperature;
    float* header;
};

// The first three numbers of a gradient's header: max |c| of the rows, of those that are numbers, c itself where they share it, 1 where P has no powers of two of theirs; nothing went wrong; x as it is.
__device__ __forceinline__ void write_header(const HeaderArgs& a, unsigned most) {
    if (!a.each) a.header[0] = a.loss_grad[0] * a.temperature / (a.count != nullptr ? fmaxf(*a.count, 1.0f) : 1.0f);
    else a.header[0] = a.powers != nullptr ? 1.0f : __uint_as_float(most);
    a.header[1] = 0.0f;
    a.header[2] = 1.0f;
}

__global__ void __launch_bounds__(1024) header_kernel(const __grid_constant__ HeaderArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    unsigned most = 0;  // (of magnitudes as whole numbers: infinity and NaN are above all others)
    if (a.each) {
#pragma unroll 4
        for (unsigned i = threadIdx.x; i < a.rows; i += 1024u) {
            const float c = a.loss_grad[(long long)i * a.loss_grad_stride] * a.temperature;
            const unsigned bits = __float_as_uint(c) & 0x7fffffffu;
            most = max(most, a.valid[i] == 0.0f || bits >= 0x7f800000u ? 0u : bits);
            if (a.powers != nullptr) a.powers[i] = power_of(c);
        }
    }
    __shared__ unsigned all[32];
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31u) == 0) all[threadIdx.x / 32u] = most;
    __syncthreads();
    if (threadIdx.x >= 32u) return;
    most = __reduce_max_sync(0xffffffffu, all[threadIdx.x]);
    if (threadIdx.x == 0) write_header(a, most);
}

// Both at once: the rows' sums, their losses, what their gradients are divided by, and E of the targets.
struct CloseArgs {
    const float* exp_sums;  // [parts][rows]
    unsigned rows, parts;
    unsigned entries, entry_stride;  // 0: cross entropy
    long long vocabulary;
    const void* targets;
    long long target_stride;
    bool targets64;
    const int* words;  // [entries][entry_stride]
    const float* z;
    const float* p;
    const float* valid;
    const float* top;
    float temperature, factor;
    float* sum;
    float* rest;
    float* loss;
    float* row_scale;
    unsigned* condition;  // set where a sum is too large for E
    __nv_bfloat16* exps;  // [rows][pitch]
    u64 pitch;
};

constexpr float kLargestSum = 18446744073709551616.0f;  // 2^64

// A CTA takes 32 rows: each of its warps every 32nd part of them, then one row.
//
// Most of a row's gradient is that of its entries, and E of each is rounded on its own; but the row has a factor, in 32 bits, that may be a little off what it should be for all other
// words. Cross entropy: it is what makes the target's exact. Distillation: of 32 factors within 2^-9 the one that rounds the entries best. (8192 x 50257 x 768, errors in the
// norm of dx and dw: 2.35e-3 and 2.56e-3 otherwise, 1.67e-3 and 2.15e-3 so; with a teacher of 32 entries 1.89e-3 and 2.37e-3.)
__global__ void __launch_bounds__(1024) close_kernel(const __grid_constant__ CloseArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr unsigned kWarps = 32;
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x / 32u, first = blockIdx.x * 32u;
    const auto all_lanes = [](float v) {
#pragma unroll
        for (unsigned d = 16; d != 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
        return v;
    };
    float sum = 0.0f;
    if (first + lane < a.rows) {
        for (unsigned p = warp; p < a.parts; p += 4u * kWarps) {
            float v[4];
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) v[i] = p + kWarps * i < a.parts ? a.exp_sums[(u64)(p + kWarps * i) * a.rows + first + lane] : 0.0f;
            sum += (v[0] + v[1]) + (v[2] + v[3]);
        }
    }
    __shared__ float all[kWarps][33];
    all[warp][lane] = sum;
    __syncthreads();
    const unsigned row = first + warp;
    if (row >= a.rows) return;
    sum = all_lanes(all[lane][warp]);
    const float valid = a.valid[row];
    float loss = 0.0f, factor = 1.0f;
    if (a.entries == 0) {
        const long long target = target_at(a.targets, a.targets64, (long long)row * a.target_stride);
        if (target >= 0 && target < a.vocabulary) {
            const float others = sum;  // (E of the target less S is that of the others)
            const __nv_bfloat16 rounded = __float2bfloat16_rn(-others);
            if (lane == 0) a.exps[(u64)row * a.pitch + (u64)target] = rounded;
            if (others > 1e-30f) factor = -others / __bfloat162float(rounded);
            loss = log1pf(others);
            sum = 1.0f + others;
            if (lane == 0) a.rest[row] = others / sum;
        }
    } else {
        const float top = a.top[row], log_sum = log2f(sum);
        float value[kEntryRounds];
        int word[kEntryRounds];
#pragma unroll
        for (unsigned i = 0; i < kEntryRounds; ++i) {
            const unsigned k = lane + 32u * i;
            value[i] = 0.0f;
            word[i] = -1;
            if (32u * i >= a.entries) break;
            const u64 at = (u64)k * a.entry_stride + row;
            const float p = k < a.entries ? a.p[at] : 0.0f;
            word[i] = p != 0.0f ? a.words[at] : -1;
            const float over = word[i] >= 0 ? (a.z[at] - top) * a.factor : 0.0f;
            if (p != 0.0f) loss += p * (logf(p) + kLn2 * (log_sum - over));
            // Entries of the same word add up, and write the same.
            float together = p;
            if (a.entries > 32u) {
                together = 0.0f;
                for (unsigned e = 0; e < a.entries; ++e) {
                    const u64 other = (u64)e * a.entry_stride + row;
                    together += a.words[other] == word[i] ? a.p[other] : 0.0f;
                }
            } else {
                const unsigned same = __match_any_sync(0xffffffffu, word[i]);
                if (__any_sync(0xffffffffu, word[i] >= 0 && (same & (same - 1u)) != 0u)) {
                    together = 0.0f;
                    for (unsigned e = 0; e < 32u; ++e) {
                        const float q = __shfl_sync(0xffffffffu, p, e);
                        together += same >> e & 1u ? q : 0.0f;
                    }
                }
            }
            if (word[i] >= 0) value[i] = exp2_fast(over) - together * sum;
        }
        loss = all_lanes(loss);
        // A factor for each lane.
        const float by = 1.0f + (float)((int)lane - 16) * (1.0f / 8192.0f), over_by = 1.0f / by;
        float off = 0.0f;
#pragma unroll
        for (unsigned i = 0; i < kEntryRounds; ++i) {
            if (32u * i >= a.entries) break;
            for (unsigned e = 0; e < min(32u, a.entries - 32u * i); ++e) {
                const float v = __shfl_sync(0xffffffffu, value[i], e), d = v - by * __bfloat162float(__float2bfloat16_rn(v * over_by));
                off += d * d;
            }
        }
        // The best of them; of equal ones the first. (Squares are not negative: as whole numbers they are in the same order, and NaN is behind them.)
        const unsigned least = __reduce_min_sync(0xffffffffu, __float_as_uint(off) & 0x7fffffffu), best = __ballot_sync(0xffffffffu, (__float_as_uint(off) & 0x7fffffffu) == least);
        factor = __shfl_sync(0xffffffffu, by, __ffs((int)best) - 1);
        const float back = 1.0f / factor;
#pragma unroll
        for (unsigned i = 0; i < kEntryRounds; ++i)
            if (32u * i < a.entries && word[i] >= 0) a.exps[(u64)row * a.pitch + (u64)word[i]] = __float2bfloat16_rn(value[i] * back);
    }
    if (lane != 0) return;
    a.sum[row] = sum;
    a.loss[row] = valid == 0.0f ? 0.0f : loss * a.temperature * a.temperature * valid;
    a.row_scale[row] = valid == 0.0f ? 0.0f : valid / sum * factor;
    if (valid != 0.0f && !(sum <= kLargestSum)) *a.condition = 1u;
}

struct CountArgs {
    const float* valid;
    unsigned rows;
    bool mean;
    float temperature;
    float* count;
    float* header;
    unsigned* condition;
    unsigned conditions;
};

// What all rows' gradients are multiplied with, before the backward pass.
__global__ void __launch_bounds__(1024) count_kernel(const __grid_constant__ CountArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    unsigned count = 0;
#pragma unroll 4
    for (unsigned i = threadIdx.x; i < a.rows; i += 1024u) count += a.valid[i] == 0.0f ? 0u : 1u;
    for (unsigned i = threadIdx.x; i < a.conditions; i += 1024u) a.condition[i] = 0u;
    __shared__ unsigned counts[32];
    count = __reduce_add_sync(0xffffffffu, count);
    if ((threadIdx.x & 31u) == 0) counts[threadIdx.x / 32u] = count;
    __syncthreads();
    if (threadIdx.x >= 32u) return;
    count = __reduce_add_sync(0xffffffffu, counts[threadIdx.x]);
    if (threadIdx.x == 0) {
        *a.count = (float)count;
        a.header[0] = a.mean ? a.temperature / fmaxf((float)count, 1.0f) : a.temperature;
        a.header[1] = 0.0f;
    }
}

struct DivideArgs {
    const char* x;
    long long stride;  // bytes
    uint4* out;        // [parts][rows][pitch]
    unsigned rows, columns, parts;
    Divisor eights;  // of a row
    const float* row_scale;
};

// Rows of x over their sums, rounded, and what that leaves. A thread takes eight elements.
__global__ void __launch_bounds__(256) divide_kernel(const __grid_constant__ DivideArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    using T = __nv_bfloat16;
    const unsigned i = blockIdx.x * 256u + threadIdx.x, row = a.eights.divide(i), n = (i - row * a.eights.d) * 8u;
    if (row >= a.rows) return;
    unsigned w[4];
    load_any<T, 8>(a.x + (long long)row * a.stride + (u64)n * 2u, n < a.columns ? min(8u, a.columns - n) : 0u, w);
    const float scale = a.row_scale[row];
    float f[8];
    Wide<T>::unpack(make_uint4(w[0], w[1], w[2], w[3]), f);
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) f[e] = scale == 0.0f ? 0.0f : f[e] * scale;
    const uint4 v = Wide<T>::pack(f);
    a.out[i] = v;
    if (a.parts == 1) return;
    float rounded[8];
    Wide<T>::unpack(v, rounded);
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) f[e] = fabsf(rounded[e]) < __int_as_float(0x7f800000) ? f[e] - rounded[e] : 0.0f;  // (infinities and NaN have no rest)
    a.out[(u64)a.rows * a.eights.d + i] = Wide<T>::pack(f);
}

struct ScaleArgs {
    __nv_bfloat16* gradients[2];
    u64 elements[2];
    const float* loss_grad;
};

// Gradients times what comes back to the loss. Most often that is 1, and there is nothing to do.
__global__ void __launch_bounds__(512) times_kernel(const __grid_constant__ ScaleArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    using T = __nv_bfloat16;
    const float scale = *a.loss_grad;
    if (scale == 1.0f) return;
    for (unsigned which = 0; which < 2; ++which) {
        T* at = a.gradients[which];
        if (at == nullptr) continue;
        const u64 n = a.elements[which], step = (u64)gridDim.x * 512u, first = (u64)blockIdx.x * 512u + threadIdx.x;
        const bool wide = reinterpret_cast<std::uintptr_t>(at) % 16u == 0;
        const u64 eights = wide ? n / 8u : 0u;
#pragma unroll 4
        for (u64 i = first; i < eights; i += step) {
            float f[8];
            Wide<T>::unpack(reinterpret_cast<const uint4*>(at)[i], f);
#pragma unroll
            for (unsigned e = 0; e < 8; ++e) f[e] *= scale;
            reinterpret_cast<uint4*>(at)[i] = Wide<T>::pack(f);
        }
        for (u64 i = eights * 8u + first; i < n; i += step) at[i] = __float2bfloat16_rn(__bfloat162float(at[i]) * scale);
    }
}

// ---- fp32, and fp16 where rows have weights of their own ------------------------------------------------------

struct Matrix {
    const char* from;
    long long stride;  // bytes
    unsigned rows, columns;
    Divisor eights;  // of a row
};
// Eight elements; zeros behind the row.
template <typename T>
__device__ __forceinline__ void load_eight(const Matrix& m, unsigned row, unsigned n, float (&f)[8]) {
    unsigned w[2 * sizeof(T)];
    load_any<T, 8>(m.from + (long long)row * m.stride + (u64)n * sizeof(T), n < m.columns ? min(8u, m.columns - n) : 0u, w);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (unsigned e = 0; e < 8; ++e) f[e] = __uint_as_float(w[e]);
    } else {
        Wide<T>::unpack(make_uint4(w[0], w[1], w[2], w[3]), f);
    }
}
// The largest magnitude, as a whole number, without infinities and NaN.
__device__ __forceinline__ unsigned largest_of(const float (&f)[8]) {
    unsigned most = 0;
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) {
        const unsigned magnitude = __float_as_uint(f[e]) & 0x7fffffffu;
        most = max(most, magnitude < 0x7f800000u ? magnitude : 0u);
    }
    return most;
}
// Eight elements as fp16 numbers; fp32: as two times eight, `apart` sixteens of bytes from each other.
template <typename T>
__device__ __forceinline__ void store_split(char* out, u64 i, u64 apart, const float (&f)[8], float scale) {
    unsigned first[4], second[4];
#pragma unroll
    for (unsigned e = 0; e < 4; ++e) {
        const float x = f[2 * e] * scale, y = f[2 * e + 1] * scale;
        first[e] = f2_to_h2(x, y);
        const float2 rounded = h2_to_f2(first[e]);
        // (Infinities and NaN have no rest.)
        second[e] = f2_to_h2(fabsf(x) < 65536.0f ? x - rounded.x : 0.0f, fabsf(y) < 65536.0f ? y - rounded.y : 0.0f);
    }
    *(reinterpret_cast<uint4*>(out) + i) = make_uint4(first[0], first[1], first[2], first[3]);
    if constexpr (sizeof(T) == 4) *(reinterpret_cast<uint4*>(out) + apart + i) = make_uint4(second[0], second[1], second[2], second[3]);
}

constexpr unsigned kMagnitudeCtas = 256;  // for the matrix

struct MagnitudeArgs {
    Matrix x, w;
    unsigned* rows;     // of each row of x
    unsigned* partial;  // of each CTA's part of w
};

// The largest magnitudes. A warp takes a row of x; a thread eight elements of w at a time.
__global__ void __launch_bounds__(512) magnitude_kernel(const __grid_constant__ MagnitudeArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    unsigned most = 0;
    float f[8];
    if (blockIdx.x >= kMagnitudeCtas) {
        const unsigned row = (blockIdx.x - kMagnitudeCtas) * 16u + threadIdx.x / 32u;
        if (row >= a.x.rows) return;
#pragma unroll 4
        for (unsigned n = threadIdx.x % 32u * 8u; n < a.x.columns; n += 256u) {
            load_eight<float>(a.x, row, n, f);
            most = max(most, largest_of(f));
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (threadIdx.x % 32u == 0) a.rows[row] = most;
        return;
    }
    const unsigned eights = a.w.rows * a.w.eights.d;
#pragma unroll 4
    for (unsigned at = blockIdx.x * 512u + threadIdx.x; at < eights; at += kMagnitudeCtas * 512u) {
        const unsigned row = a.w.eights.divide(at);
        load_eight<float>(a.w, row, (at - row * a.w.eights.d) * 8u, f);
        most = max(most, largest_of(f));
    }
    most = __reduce_max_sync(0xffffffffu, most);
    __shared__ unsigned all[16];
    if ((threadIdx.x & 31u) == 0) all[threadIdx.x / 32u] = most;
    __syncthreads();
    if (threadIdx.x >= 32u) return;
    most = __reduce_max_sync(0xffffffffu, threadIdx.x < 16u ? all[threadIdx.x] : 0u);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = most;
}

struct SplitArgs {
    Matrix x, w;
    char *x_out, *w_out;      // two fp16 matrices [2][rows][pitch] each, scaled
    unsigned ctas_of_x;
    const unsigned* rows;     // of magnitude_kernel
    const unsigned* partial;  // the same; null: that of w is known
    unsigned* w_magnitude;
};

// fp32. A thread takes eight elements of a row.
__global__ void __launch_bounds__(256) split_kernel(const __grid_constant__ SplitArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    static_assert(kMagnitudeCtas == 256);
    const bool of_x = blockIdx.x < a.ctas_of_x;
    const Matrix& m = of_x ? a.x : a.w;
    const unsigned block = of_x ? blockIdx.x : blockIdx.x - a.ctas_of_x, i = block * 256u + threadIdx.x, row = m.eights.divide(i);
    const bool there = row < m.rows;
    float f[8] = {};
    unsigned magnitude = 0;
    if (there) load_eight<float>(m, row, (i - row * m.eights.d) * 8u, f);
    if (of_x) {
        if (there) magnitude = a.rows[row];
    } else if (a.partial != nullptr) {
        __shared__ unsigned all[8];
        magnitude = __reduce_max_sync(0xffffffffu, a.partial[threadIdx.x]);
        if ((threadIdx.x & 31u) == 0) all[threadIdx.x / 32u] = magnitude;
        __syncthreads();
#pragma unroll
        for (unsigned w = 0; w < 8; ++w) magnitude = max(magnitude, all[w]);
        if (block == 0 && threadIdx.x == 0) *a.w_magnitude = magnitude;
    } else {
        magnitude = *a.w_magnitude;
    }
    if (there) store_split<float>(of_x ? a.x_out : a.w_out, i, (u64)m.rows * m.eights.d, f, scale_of(magnitude, false));
}

constexpr unsigned kPowersCtas = 256;
constexpr int kNoExponent = -1000;

struct PowersArgs {
    HeaderArgs header;
    Matrix x;
    const unsigned* magnitudes;  // fp32: of each row of x
    int* partial;                // of each CTA
};

// header_kernel's work where the gradient of w takes x apart, and the exponent of the largest element of x times its row's power, of the rows that count. A warp takes a row.
template <typename T>
__global__ void __launch_bounds__(512) powers_kernel(const __grid_constant__ PowersArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const HeaderArgs& h = a.header;
    const unsigned lane = threadIdx.x % 32u;
    int exponent = kNoExponent;
    for (unsigned row = blockIdx.x * 16u + threadIdx.x / 32u; row < a.x.rows; row += gridDim.x * 16u) {
        unsigned most = 0;
        if constexpr (sizeof(T) == 4) {
            most = a.magnitudes[row];
        } else {
            float f[8];
#pragma unroll 4
            for (unsigned n = lane * 8u; n < a.x.columns; n += 256u) {
                load_eight<T>(a.x, row, n, f);
                most = max(most, largest_of(f));
            }
            most = __reduce_max_sync(0xffffffffu, most);
        }
        const float c = h.each ? h.loss_grad[(long long)row * h.loss_grad_stride] * h.temperature : 1.0f, power = h.powers != nullptr ? power_of(c) : 1.0f;
        if (h.powers != nullptr && lane == 0) h.powers[row] = power;
        const bool counts = h.valid[row] != 0.0f && c != 0.0f && fabsf(c) < __int_as_float(0x7f800000) && most != 0u;
        if (counts) exponent = max(exponent, (int)(most >> 23) + (int)(__float_as_uint(power) >> 23) - 254);
    }
    __shared__ int all[16];
    if (lane == 0) all[threadIdx.x / 32u] = exponent;
    __syncthreads();
    if (threadIdx.x >= 32u) return;
    exponent = __reduce_max_sync(0xffffffffu, all[lane % 16u]);
    if (lane != 0) return;
    a.partial[blockIdx.x] = exponent;
    if (blockIdx.x == 0) write_header(h, 0u);
}

struct WeighArgs {
    Matrix x;
    char* out;   // [parts][rows][pitch], from the first of x's rows on
    u64 apart;   // sixteens of bytes from part to part
    const float* valid;
    const float* powers;  // of each row, or null
    const int* partial;   // of powers_kernel
    unsigned partials;
    float* header;
};

// x as the gradient of w takes it: times the power of two of each row's c and one for all rows, zeros for rows that do not count. A thread takes eight elements.
template <typename T>
__global__ void __launch_bounds__(256) weigh_kernel(const __grid_constant__ WeighArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    static_assert(kPowersCtas == 256);
    const unsigned i = blockIdx.x * 256u + threadIdx.x, row = a.x.eights.divide(i);
    float f[8] = {};
    if (row < a.x.rows && a.valid[row] != 0.0f) load_eight<T>(a.x, row, (i - row * a.x.eights.d) * 8u, f);
    __shared__ int all[8];
    int exponent = __reduce_max_sync(0xffffffffu, threadIdx.x < a.partials ? a.partial[threadIdx.x] : kNoExponent);
    if ((threadIdx.x & 31u) == 0) all[threadIdx.x / 32u] = exponent;
    __syncthreads();
#pragma unroll
    for (unsigned w = 0; w < 8; ++w) exponent = max(exponent, all[w]);
    const int back = exponent == kNoExponent ? 0 : min(max(exponent - 14, -126), 127);
    if (i == 0) a.header[2] = ldexpf(1.0f, back);
    if (row >= a.x.rows) return;
    // (Powers may be further apart than floats reach: a row whose largest element is below 2^-112 stays smaller, and what is 2^-149 of another's is nothing beside it.)
    const int power = a.powers != nullptr ? (int)(__float_as_uint(a.powers[row]) >> 23) - 127 : 0;
    store_split<T>(a.out, i, a.apart, f, ldexpf(1.0f, min(power - back, 126)));
}

// ---- launches ------------------------------------------------------------------------------------------------

int current_device() {
    int device = 0;
    B2_CUDA(cudaGetDevice(&device));
    return device;
}

template <Kind kKind, bool kLong, bool kTeacher>
const void* kernel_of(DType dtype) {
    if constexpr (kKind == Kind::Exps) return (const void*)product_kernel<kKind, __nv_bfloat16, kLong, kTeacher>;
    else switch (dtype) {
        case DType::Float: return (const void*)product_kernel<kKind, float, kLong, kTeacher>;
        case DType::Float16: return (const void*)product_kernel<kKind, __half, kLong, kTeacher>;
        default: return (const void*)product_kernel<kKind, __nv_bfloat16, kLong, kTeacher>;
    }
}
template <Kind kKind>
const void* logits_kernel_of(DType dtype, bool longer, bool teacher) {
    return longer ? (teacher ? kernel_of<kKind, true, true>(dtype) : kernel_of<kKind, true, false>(dtype))
                  : (teacher ? kernel_of<kKind, false, true>(dtype) : kernel_of<kKind, false, false>(dtype));
}
const void* kernel_of(Kind kind, DType dtype, bool longer, bool teacher) {
    switch (kind) {
        case Kind::Stats: return logits_kernel_of<Kind::Stats>(dtype, longer, teacher);
        case Kind::Probs: return logits_kernel_of<Kind::Probs>(dtype, longer, teacher);
        case Kind::Exps: return logits_kernel_of<Kind::Exps>(dtype, longer, teacher);
        case Kind::WeightGrad: return longer ? kernel_of<Kind::WeightGrad, true, false>(dtype) : kernel_of<Kind::WeightGrad, false, false>(dtype);
        default: return longer ? kernel_of<Kind::InputGrad, true, false>(dtype) : kernel_of<Kind::InputGrad, false, false>(dtype);
    }
}

// Pairs of CTAs that run at once on `device` (where GPCs have odd numbers of SMs, fewer than half the SMs). The kernels' shared memory is asked for once.
unsigned pairs_of_device(int device) {
    static std::mutex mutex;
    static unsigned known[64] = {};
    std::lock_guard<std::mutex> lock(mutex);
    if (device >= 0 && device < 64 && known[device] != 0) return known[device];
    for (Kind kind : {Kind::Stats, Kind::Probs, Kind::Exps, Kind::WeightGrad, Kind::InputGrad})
        for (DType dtype : {DType::Float, DType::Float16, DType::BFloat16})
            for (int n = 0; n < 4; ++n) B2_CUDA(cudaFuncSetAttribute(kernel_of(kind, dtype, n / 2 != 0, n % 2 != 0), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kShared));
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
    B2_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kernel_of(Kind::Stats, DType::BFloat16, true, true), &config));
    const unsigned pairs = std::min(kMaxPairs, (unsigned)std::max(1, clusters));
    if (device >= 0 && device < 64) known[device] = pairs;
    return pairs;
}

// How the pairs share the tiles of one product.
struct Tiling {
    unsigned m_tiles = 0, n_tiles = 0, n_tile = kTile, products = 1, steps_of_part = 0, steps_of_tile = 0, pairs = 0, waves = 0, left = 0, splits = 1;
    std::size_t slots = 0;  // pieces in memory
};

Tiling tiling_of(u64 m, u64 n, u64 summed, unsigned products, unsigned n_tile, bool may_cut, unsigned device_pairs) {
    Tiling t;
    t.products = products;
    t.n_tile = n_tile;
    const u64 m_tiles = (m + kTile - 1) / kTile, n_tiles = (n + n_tile - 1) / n_tile, steps = (summed + kStep - 1) / kStep;
    const u64 tiles = m_tiles * n_tiles, steps_of_tile = steps * products;
    B2_REQUIRE(steps_of_tile < (1ull << 31) && tiles < (1ull << 31) && tiles * steps_of_tile < (1ull << 31), "too many tokens, words and columns for one call");
    t.m_tiles = (unsigned)m_tiles;
    t.n_tiles = (unsigned)n_tiles;
    t.steps_of_part = (unsigned)steps;
    t.steps_of_tile = (unsigned)steps_of_tile;
    t.pairs = device_pairs;
    t.waves = (unsigned)tiles / t.pairs;
    t.left = (unsigned)tiles - t.waves * t.pairs;
    // The tiles that are left are cut where that saves more steps than writing the pieces and adding them costs: about sixteen, and half a step for each piece of a tile.
    if (may_cut && t.left != 0) {
        u64 least = t.steps_of_tile;
        for (unsigned splits = 2; splits <= std::min(t.pairs, t.steps_of_tile / 8) && t.left * splits <= 4 * t.pairs; ++splits) {
            const u64 cost = (u64)((t.left * splits + t.pairs - 1) / t.pairs) * ((t.steps_of_tile + splits - 1) / splits) + 16 + splits / 2;
            if (cost >= least) continue;
            least = cost;
            t.splits = splits;
        }
    }
    if (t.waves == 0) t.pairs = std::min(t.pairs, t.left * t.splits);
    if (t.splits > 1) t.slots = (std::size_t)t.left * t.splits;
    return t;
}

// A piece of the vocabulary: so many bytes of P, unless that is fewer than kLeastPiece words, and of the matrix, which the gradient of x reads again for every few rows of tiles, out
// of L2 in part. (8192 x 50257 x 768, loss and gradients: 2073 us in two pieces of P, 2112 in four, 2195 in seven; 4096 x 131072 x 4096: 13.7 ms in two
// pieces, 13.2 in four of 256 MiB of the matrix, 13.3 in eight.)
constexpr std::size_t kProbsBytes = 512ull << 20, kMatrixBytes = 256ull << 20;
constexpr u64 kLeastPiece = 4096;

std::size_t padded(std::size_t bytes) { return (bytes + 255) / 256 * 256; }

// What a call needs of its workspace, and where.
struct Plan {
    unsigned parts = 1, products = 1;            // of x and the matrix, and of those of logits
    unsigned prob_parts = 1, grad_products = 1;  // of P, and of the gradients
    unsigned divided_parts = 1;                  // both at once: of x / S
    bool copy_x = false, copy_weight = false;
    std::size_t pitch = 0;  // elements of a row of the copies
    unsigned device_pairs = 0;
    u64 piece = 0, pieces = 1;  // words of the vocabulary
    u64 rows = 0;                // both at once: of a piece
    std::size_t exps_pitch = 0;
    unsigned n_tile = kTile;
    std::size_t scale_at = 0, divided_at = 0, weighed_at = 0, powers_at = 0, x_at = 0, weight_at = 0, stats_at = 0, picked_at = 0, losses_at = 0, partial_at = 0, header_at = 0, probs_at = 0, sums_at = 0, slots_at = 0, bytes = 0;
};

// Both at once: bytes of E in a piece of the rows, and of the sums of dw where there are several. (8192 x 50257 x 768, loss and gradients: 1459 us in one piece of 824 MB, 1565 in two,
// 1684 in four; 4096 x 131072 x 4096: 10.2 ms in one, two or four.)
constexpr std::size_t kExpsBytes = 1ull << 30, kSumsBytes = 1ull << 30;

bool readable(const void* p, long long stride, std::size_t columns, std::size_t rows, std::size_t element) {
    return reinterpret_cast<std::uintptr_t>(p) % 16 == 0 && (rows <= 1 || (stride * (long long)element % 16 == 0 && stride >= (long long)columns));
}

// 128 columns of a gradient to a tile instead of 256, where that leaves fewer of them empty.
unsigned n_tile_of(std::size_t width) { return (width + 127) / 128 * 128 < (width + 255) / 256 * 256 && width <= 640 ? 128u : 256u; }

enum class Pass { Loss, Gradient, Both };

// A product so small, up to a whole tile of rows, that launches count for more than it does: both() is not used, which has more of them (us, apart / at once; rows x words x columns in thousand
// millions: 512 x 512 x 64 90 / 93 (0.02), 512 x 5000 x 256 90 / 95 (0.7), 1024 x 5000 x 256 101 / 99 (1.3), 16 x 32000 x 768 91 / 96 (6.3), 16 x 50257 x 768 111 / 103 (9.9),
// 512 x 32000 x 768 132 / 126 (12.6), 1024 x 50257 x 768 277 / 230 (40)).
bool small(const VocabularyLossCall& c) { return std::max<std::size_t>(c.tokens, kTile) * c.vocabulary < (1ull << 33) / std::max<std::size_t>(c.width, 1); }
// Of those, and of any with few rows, P has two parts in 16-bit types too, which costs its gradients a second product and leaves them their own rounding alone; not where the rows are many, P itself
// large and its matrix narrow. (Few rows: what P's rounding makes of a row's entry with most of its weight is in all of the row's gradient, and few other rows make up for it: 12 x 23488 x 4072, a teacher
// of 12 entries in fp16, errors in the norm 3.6e-4 instead of 2.1e-4, which is the gradient's own rounding; 292 us instead of 262, 64 x 131072 x 4096 1265 instead of 1055;
// 64 x 262144 x 768 509 instead of 420, 64 x 1048576 x 16, the narrowest, 786 instead of 568.)
// x / S, of both(), has two parts for few rows, whose products' second step of 64 is mostly hidden behind what they write. (2 x 40065 x 2496: errors of dw in the
// norm 1.4e-3 -> 2.0e-4, most of it is of the targets; 64 x 131072 x 4096 644 -> 680 us, 16 x 50257 x 768 103 -> 101.)
constexpr u64 kFewRows = 64;
bool fine(const VocabularyLossCall& c) { return c.tokens <= kFewRows || (small(c) && std::max<std::size_t>(c.tokens, kTile) * c.vocabulary <= (1ull << 25)); }

// Whether P is without the powers of two of the rows' weights, and whether the gradient of w has its own x.
bool powers_apart(const VocabularyLossCall& c) { return c.dtype != DType::BFloat16 && c.reduction == LossReduction::None; }
bool weighed(const VocabularyLossCall& c) { return c.weight_grad != nullptr && (c.dtype == DType::Float || powers_apart(c)); }

Plan plan_of(const VocabularyLossCall& c, Pass pass) {
    Plan p;
    const std::size_t e = dtype_size(c.dtype), t = c.tokens, v = c.vocabulary;
    p.parts = c.dtype == DType::Float ? 2 : 1;
    p.products = c.dtype == DType::Float ? 3 : 1;
    p.prob_parts = c.dtype == DType::Float || (pass == Pass::Gradient && fine(c)) ? 2 : 1;
    p.grad_products = c.dtype == DType::Float ? 3 : p.prob_parts;
    p.device_pairs = pairs_of_device(current_device());
    p.pitch = (c.width + 7) / 8 * 8;
    p.copy_x = c.dtype == DType::Float || !readable(c.x, c.x_stride, c.width, t, e);
    p.copy_weight = c.dtype == DType::Float || !readable(c.weight, c.weight_stride, c.width, v, e);
    std::size_t at = 0;
    const auto take = [&](std::size_t bytes) {
        const std::size_t here = at;
        at += padded(bytes);
        return here;
    };
    p.x_at = take(p.copy_x ? p.parts * t * p.pitch * 2 : 0);
    p.weight_at = take(p.copy_weight ? p.parts * v * p.pitch * 2 : 0);
    std::size_t slots = 0;
    const auto look = [&](u64 m, u64 n, u64 k, unsigned products) { slots = std::max(slots, tiling_of(m, n, k, products, p.n_tile, true, p.device_pairs).slots); };
    if (pass == Pass::Loss) {
        p.stats_at = take((v + kTile - 1) / kTile * 2 * t * sizeof(float2));
        p.picked_at = take(t * std::max(c.entries, 1) * sizeof(float));
        p.losses_at = take(t * sizeof(float));
        p.partial_at = take(c.dtype == DType::Float ? kMagnitudeCtas * sizeof(unsigned) : 0);
    } else if (pass == Pass::Both) {
        p.n_tile = n_tile_of(c.width);
        p.exps_pitch = (v + kTile - 1) / kTile * kTile;
        const std::size_t most = kExpsBytes / (p.exps_pitch * 2) / kTile * kTile;
        p.rows = std::min<u64>(t, std::max<std::size_t>(most, kTile));
        p.pieces = (t + p.rows - 1) / p.rows;
        p.rows = std::min<u64>(t, ((t + p.pieces - 1) / p.pieces + kTile - 1) / kTile * kTile);
        p.pieces = (t + p.rows - 1) / p.rows;
        if (p.rows * p.exps_pitch * 2 > kExpsBytes) return Plan();  // (a tile's rows alone, over more than two million words)
        p.stats_at = take(p.exps_pitch / kTile * 2 * p.rows * sizeof(float2));
        p.picked_at = take(t * std::max(c.entries, 1) * sizeof(float));
        p.losses_at = take(t * sizeof(float));
        p.header_at = take((2 + p.pieces) * sizeof(float));
        p.scale_at = take(p.rows * sizeof(float));
        p.probs_at = take(p.rows * p.exps_pitch * 2);
        if (c.weight_grad != nullptr) {
            p.divided_parts = t <= kFewRows ? 2 : 1;
            p.divided_at = take(p.divided_parts * p.rows * p.pitch * 2);
            const std::size_t sums = p.exps_pitch / kTile * ((c.width + p.n_tile - 1) / p.n_tile) * kTileFloats * sizeof(float);
            if (p.pieces > 1 && sums > kSumsBytes) return Plan();
            if (p.pieces > 1) p.sums_at = take(sums);
        }
        for (const u64 rows : {p.rows, t - (p.pieces - 1) * p.rows}) {
            if (c.weight_grad != nullptr) look(v, c.width, rows, p.divided_parts);
            if (c.x_grad != nullptr) look(rows, c.width, v, 1);
        }
    } else {
        const u64 tiles = (v + kTile - 1) / kTile, bytes = (u64)p.prob_parts * t * 2;
        const u64 most = std::max<u64>(std::min<u64>(kProbsBytes / bytes, kMatrixBytes / (p.parts * c.width * 2)), kLeastPiece) / kTile;
        p.pieces = (tiles + most - 1) / most;
        p.piece = (tiles + p.pieces - 1) / p.pieces * kTile;
        p.pieces = (v + p.piece - 1) / p.piece;
        p.n_tile = n_tile_of(c.width);
        p.header_at = take(3 * sizeof(float));
        p.weighed_at = take(weighed(c) ? p.parts * t * p.pitch * 2 : 0);
        p.powers_at = take(powers_apart(c) ? t * sizeof(float) : 0);
        p.partial_at = take(weighed(c) ? kPowersCtas * sizeof(int) : 0);
        p.probs_at = take(bytes * p.piece);
        const u64 rest = v - (p.pieces - 1) * p.piece;
        if (c.x_grad != nullptr && p.pieces > 1)
            p.sums_at = take((t + kTile - 1) / kTile * ((c.width + p.n_tile - 1) / p.n_tile) * kTileFloats * sizeof(float));
        for (const u64 words : {p.piece, rest}) {
            if (c.weight_grad != nullptr) look(words, c.width, t, p.grad_products);
            if (c.x_grad != nullptr) look(t, c.width, words, p.grad_products);
        }
    }
    p.slots_at = take(slots * kTileFloats * sizeof(float));
    p.bytes = at;
    return p;
}

// A matrix as the tensor cores read it.
struct Operand {
    const void* data = nullptr;
    u64 columns = 0, rows = 0, row_bytes = 0;
};

CUtensorMap map_of(DType dtype, const Operand& o, unsigned parts, unsigned box_columns, unsigned box_rows) {
    CUtensorMap m;
    const auto encode = cu::api().TensorMapEncodeTiled;
    if (encode == nullptr) throw std::runtime_error("the driver does not export cuTensorMapEncodeTiled");
    const CUtensorMapDataType type = dtype == DType::Float     ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : dtype == DType::Float16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const cuuint64_t extent[3] = {o.columns, o.rows, parts}, strides[2] = {o.row_bytes, o.row_bytes * o.rows};
    const cuuint32_t box[3] = {box_columns, box_rows, 1}, element_strides[3] = {1, 1, 1};
    cu::check(encode(&m, type, 3, const_cast<void*>(o.data), extent, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
              "tensor map of an operand");
    return m;
}

void launch_product(Kind kind, const VocabularyLossCall& c, const Tiling& t, ProductArgs& a, u64 m, u64 n) {
    a.m = (unsigned)m;
    a.n = (unsigned)n;
    a.m_tiles = t.m_tiles;
    a.n_tiles = t.n_tiles;
    a.n_tile = t.n_tile;
    a.products = t.products;
    a.steps_of_part = t.steps_of_part;
    a.steps_of_tile = t.steps_of_tile;
    a.pairs = t.pairs;
    a.waves = t.waves;
    a.left = t.left;
    a.splits = t.splits;
    a.n_first = kind == Kind::WeightGrad || kind == Kind::InputGrad;
    a.chunk = c.dtype == DType::Float || (!a.n_first && small(c)) ? kShortChunkSteps : (a.n_first ? kLongChunkSteps : kChunkSteps);
    a.status = wait_status_word(WaitsOf::VocabularyLoss, current_device());
    a.wait_ns = c.wait_ns;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(2 * t.pairs);
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
    void* arguments[1] = {&a};
    B2_CUDA(cudaLaunchKernelExC(&config, kernel_of(kind, c.dtype, t.steps_of_tile > t.products * a.chunk, c.distillation), arguments));
}

// The pieces of a gradient's cut tiles.
template <Kind kKind, typename T>
void finish(const VocabularyLossCall& c, const Tiling& t, const ProductArgs& a) {
    if (t.splits == 1) return;
    FinishArgs f;
    f.out = a.gradient;
    f.slots = a.slots;
    f.sums = a.sums;
    f.prior = a.prior;
    f.last = a.last;
    f.header = a.header;
    f.row_scale = a.row_scale;
    f.w_magnitude = a.w_magnitude;
    f.m = a.m;
    f.n = a.n;
    f.m_tiles = t.m_tiles;
    f.n_tiles = t.n_tiles;
    f.n_tile = t.n_tile;
    f.whole_tiles = t.waves * t.pairs;
    f.left = t.left;
    f.splits = t.splits;
    f.n_first = a.n_first;
    B2_CUDA(launch_dependent<FinishArgs>(finish_kernel<kKind, T>, dim3(t.left * 8 * (t.n_tile / 32)), 256, 0, c.stream, f));
}

// Words of ProductArgs::hits.
std::size_t hit_words(const VocabularyLossCall& c) { return (c.vocabulary + kHalf - 1) / kHalf * ((c.tokens + 31) / 32) * (std::size_t)((c.entries + 31) / 32); }

struct Kept {
    float *top, *sum, *rest, *valid, *count, *probs;
    unsigned *w_magnitude, *magnitudes;  // fp32: of the matrix, of each row of x
    int* words;  // of the teacher's entries, and their probabilities: [entries][tokens]
    unsigned* hits;
};
Kept kept_of(const VocabularyLossCall& c) {
    Kept k;
    k.top = c.kept;
    k.sum = k.top + c.tokens;
    k.rest = k.sum + c.tokens;
    k.valid = k.rest + c.tokens;
    k.count = k.valid + c.tokens;
    k.w_magnitude = reinterpret_cast<unsigned*>(k.count + 1);
    k.probs = k.count + 2;
    k.words = reinterpret_cast<int*>(k.probs + c.tokens * (std::size_t)c.entries);
    k.hits = reinterpret_cast<unsigned*>(k.words + c.tokens * (std::size_t)c.entries);
    k.magnitudes = k.hits + hit_words(c);
    return k;
}

constexpr const char* kTooLarge = "an operand is too large for one call";

Matrix x_of(const VocabularyLossCall& c, const Plan& p) {
    return {static_cast<const char*>(c.x), c.x_stride * (long long)dtype_size(c.dtype), (unsigned)c.tokens, (unsigned)c.width, Divisor((unsigned)(p.pitch / 8))};
}

// x and the matrix as the tensor cores read them, copied where they have to be. known: fp32's magnitudes are, from the forward pass.
template <typename T>
void operands(const VocabularyLossCall& c, const Plan& p, bool known, Operand* x, Operand* w) {
    char* workspace = static_cast<char*>(c.workspace);
    // (The stride of a single row is not looked at, but must be a multiple of 16 bytes all the same.)
    *x = {c.x, c.width, c.tokens, (c.tokens > 1 ? (u64)c.x_stride : (u64)p.pitch) * sizeof(T)};
    *w = {c.weight, c.width, c.vocabulary, (c.vocabulary > 1 ? (u64)c.weight_stride : (u64)p.pitch) * sizeof(T)};
    if constexpr (sizeof(T) == 2) {
        const auto copy = [&](const void* from, long long stride, std::size_t rows, std::size_t at) -> Operand {
            lay_out<T>(from, stride, rows, c.width, p.pitch, workspace + at, c.stream, kTooLarge);
            return {workspace + at, c.width, rows, p.pitch * 2};
        };
        if (p.copy_x) *x = copy(c.x, c.x_stride, c.tokens, p.x_at);
        if (p.copy_weight) *w = copy(c.weight, c.weight_stride, c.vocabulary, p.weight_at);
    } else {
        const u64 x_eights = (u64)c.tokens * (p.pitch / 8), w_eights = (u64)c.vocabulary * (p.pitch / 8);
        B2_REQUIRE(x_eights < (1ull << 30) && w_eights < (1ull << 30), kTooLarge);
        const Kept kept = kept_of(c);
        SplitArgs s;
        s.x = x_of(c, p);
        s.w = {static_cast<const char*>(c.weight), c.weight_stride * 4, (unsigned)c.vocabulary, (unsigned)c.width, Divisor((unsigned)(p.pitch / 8))};
        s.x_out = workspace + p.x_at;
        s.w_out = workspace + p.weight_at;
        s.ctas_of_x = (unsigned)((x_eights + 255) / 256);
        s.rows = kept.magnitudes;
        s.partial = nullptr;
        s.w_magnitude = kept.w_magnitude;
        if (!known) {
            const MagnitudeArgs a = {s.x, s.w, kept.magnitudes, reinterpret_cast<unsigned*>(workspace + p.partial_at)};
            B2_CUDA(launch_dependent<MagnitudeArgs>(magnitude_kernel, dim3(kMagnitudeCtas + (unsigned)((c.tokens + 15) / 16)), 512, 0, c.stream, a));
            s.partial = a.partial;
        }
        B2_CUDA(launch_dependent<SplitArgs>(split_kernel, dim3(s.ctas_of_x + (unsigned)((w_eights + 255) / 256)), 256, 0, c.stream, s));
        *x = {s.x_out, c.width, c.tokens, p.pitch * 2};
        *w = {s.w_out, c.width, c.vocabulary, p.pitch * 2};
    }
}

template <typename T>
constexpr DType operand_type() { return std::is_same_v<T, __nv_bfloat16> ? DType::BFloat16 : DType::Float16; }

void logits_arguments(const VocabularyLossCall& c, ProductArgs& a) {
    a.magnitudes = kept_of(c).magnitudes;
    a.w_magnitude = kept_of(c).w_magnitude;
    const double factor = 1.4426950408889634 / (double)c.temperature;
    a.factor = (float)factor;
    a.factor_rest = (float)(factor - (double)a.factor);
    a.entries = (unsigned)c.entries;
    a.entry_stride = (unsigned)c.tokens;
    a.words = kept_of(c).words;
    a.probs = kept_of(c).probs;
    a.hits = kept_of(c).hits;
    a.hit_rows = (unsigned)((c.tokens + 31) / 32);
    a.targets = c.targets;
    a.target_stride = c.target_strides[0];
    a.targets64 = c.targets64;
    a.temperature = c.temperature;
}

// x and w: where top is wanted, in bf16.
void launch_entries(const VocabularyLossCall& c, const Operand& x, const Operand& w, float* top) {
    const Kept kept = kept_of(c);
    EntriesArgs e;
    e.x = x.data;
    e.x_stride = (long long)(x.row_bytes / 2);
    e.weight = w.data;
    e.weight_stride = (long long)(w.row_bytes / 2);
    e.rows = (unsigned)c.tokens;
    e.width = (unsigned)c.width;
    e.entries = c.distillation ? (unsigned)c.entries : 1u;
    e.vocabulary = c.vocabulary;
    e.targets = c.targets;
    e.targets64 = c.targets64;
    e.teacher = c.distillation ? c.teacher : nullptr;
    e.teacher_dtype = static_cast<int>(c.teacher_dtype);
    for (int i = 0; i < 2; ++i) {
        e.target_strides[i] = c.target_strides[i];
        e.teacher_strides[i] = c.teacher_strides[i];
    }
    e.temperature = c.temperature;
    e.words = c.distillation ? kept.words : nullptr;
    e.probs = kept.probs;
    e.hits = kept.hits;
    e.hit_rows = (unsigned)((c.tokens + 31) / 32);
    if (c.distillation) B2_CUDA(cudaMemsetAsync(kept.hits, 0, hit_words(c) * sizeof(unsigned), c.stream));
    e.valid = kept.valid;
    e.top = top;
    B2_CUDA(launch_dependent<EntriesArgs>(entries_kernel, dim3((unsigned)((c.tokens + 7) / 8)), 256, 0, c.stream, e));
}

template <typename T>
void loss(const VocabularyLossCall& c, const Plan& p) {
    char* workspace = static_cast<char*>(c.workspace);
    const Kept kept = kept_of(c);
    Operand x, w;
    operands<T>(c, p, false, &x, &w);
    if (c.distillation) launch_entries(c, x, w, nullptr);
    ProductArgs a = {};
    a.a = map_of(operand_type<T>(), x, p.parts, kStep, kHalf);
    a.b = map_of(operand_type<T>(), w, p.parts, kStep, kHalf);
    logits_arguments(c, a);
    a.stats = reinterpret_cast<float2*>(workspace + p.stats_at);
    a.picked = a.entry_logits = reinterpret_cast<float*>(workspace + p.picked_at);
    const Tiling t = tiling_of(c.tokens, c.vocabulary, c.width, p.products, kTile, false, p.device_pairs);
    launch_product(Kind::Stats, c, t, a, c.tokens, c.vocabulary);
    JoinArgs j;
    j.stats = a.stats;
    j.rows = (unsigned)c.tokens;
    j.parts = 2 * t.n_tiles;
    j.picked = a.picked;
    j.targets = c.targets;
    j.target_stride = c.target_strides[0];
    j.targets64 = c.targets64;
    j.vocabulary = c.vocabulary;
    j.z = a.entry_logits;
    j.p = kept.probs;
    j.entries = (unsigned)c.entries;
    j.entry_stride = a.entry_stride;
    j.temperature = c.temperature;
    j.factor = a.factor;
    j.top = kept.top;
    j.sum = kept.sum;
    j.rest = kept.rest;
    j.valid = kept.valid;
    j.condition = nullptr;
    j.row_scale = nullptr;
    j.loss = c.reduction == LossReduction::None ? c.loss : reinterpret_cast<float*>(workspace + p.losses_at);
    B2_CUDA(launch_dependent<JoinArgs>(join_kernel, dim3((unsigned)((c.tokens + 31) / 32)), 1024, 0, c.stream, j));
    if (c.reduction == LossReduction::None) return;
    SumArgs s;
    s.losses = j.loss;
    s.valid = kept.valid;
    s.rows = (unsigned)c.tokens;
    s.mean = c.reduction == LossReduction::Mean;
    s.out = c.loss;
    s.count = kept.count;
    B2_CUDA(launch_dependent<SumArgs>(sum_kernel, dim3(1), 1024, 0, c.stream, s));
}

template <typename T>
void gradient(const VocabularyLossCall& c, const Plan& p) {
    char* workspace = static_cast<char*>(c.workspace);
    const Kept kept = kept_of(c);
    const bool each = c.reduction == LossReduction::None, apart = !std::is_same_v<T, __nv_bfloat16> && weighed(c);
    float* header = reinterpret_cast<float*>(workspace + p.header_at);
    float* powers = powers_apart(c) ? reinterpret_cast<float*>(workspace + p.powers_at) : nullptr;
    HeaderArgs h;
    h.loss_grad = c.loss_grad;
    h.loss_grad_stride = c.loss_grad_stride;
    h.valid = kept.valid;
    h.count = c.reduction == LossReduction::Mean ? kept.count : nullptr;
    h.rows = (unsigned)c.tokens;
    h.each = each;
    h.powers = powers;
    h.temperature = c.temperature;
    h.header = header;
    int* partial = reinterpret_cast<int*>(workspace + p.partial_at);
    const unsigned partials = (unsigned)std::min<std::size_t>(kPowersCtas, (c.tokens + 15) / 16);
    if (!apart) B2_CUDA(launch_dependent<HeaderArgs>(header_kernel, dim3(1), 1024, 0, c.stream, h));
    if constexpr (!std::is_same_v<T, __nv_bfloat16>)
        if (apart) B2_CUDA(launch_dependent<PowersArgs>(powers_kernel<T>, dim3(partials), 512, 0, c.stream, PowersArgs{h, x_of(c, p), kept.magnitudes, partial}));
    Operand x, w;
    operands<T>(c, p, true, &x, &w);
    Operand weighed_x = x;
    if constexpr (!std::is_same_v<T, __nv_bfloat16>) {
        if (apart) {
            const u64 eights = p.pitch / 8, most = (1ull << 30) / eights;  // rows of a launch
            for (u64 first = 0; first < c.tokens; first += most) {
                WeighArgs e = {x_of(c, p), workspace + p.weighed_at + first * p.pitch * 2, c.tokens * eights, kept.valid + first, powers, partial, partials, header};
                e.x.from += (long long)first * e.x.stride;
                e.x.rows = (unsigned)std::min<u64>(most, c.tokens - first);
                if (powers != nullptr) e.powers += first;
                B2_CUDA(launch_dependent<WeighArgs>(weigh_kernel<T>, dim3((unsigned)((e.x.rows * eights + 255) / 256)), 256, 0, c.stream, e));
            }
            weighed_x = {workspace + p.weighed_at, c.width, c.tokens, p.pitch * 2};
        }
    }
    char* probs = workspace + p.probs_at;
    for (u64 piece = 0; piece < p.pieces; ++piece) {
        const u64 first = piece * p.piece, words = std::min<u64>(p.piece, c.vocabulary - first);
        const Operand probs_of = {probs, p.piece, c.tokens, p.piece * 2};
        ProductArgs a = {};
        a.a = map_of(operand_type<T>(), x, p.parts, kStep, kHalf);
        a.b = map_of(operand_type<T>(), w, p.parts, kStep, kHalf);
        a.out = map_of(operand_type<T>(), probs_of, p.prob_parts, 64, 32);
        a.out_parts = p.prob_parts;
        logits_arguments(c, a);
        a.b_offset = (unsigned)first;
        a.top = kept.top;
        a.sum = kept.sum;
        a.rest = kept.rest;
        a.valid = kept.valid;
        a.loss_grad = each ? c.loss_grad : nullptr;
        a.loss_grad_stride = c.loss_grad_stride;
        a.header = header;
        a.slots = reinterpret_cast<float*>(workspace + p.slots_at);
        launch_product(Kind::Probs, c, tiling_of(c.tokens, words, c.width, p.products, kTile, false, p.device_pairs), a, c.tokens, words);
        const unsigned columns = 128 / sizeof(T);
        const auto gradient_of = [&](void* out, u64 rows) {
            a.gradient = out;
            a.wide = c.width * sizeof(T) % 16 == 0 && reinterpret_cast<std::uintptr_t>(out) % 16 == 0;
            if (a.wide) a.out = map_of(c.dtype, {out, c.width, rows, c.width * sizeof(T)}, 1, columns, 32);
        };
        if (c.weight_grad != nullptr) {
            const Tiling t = tiling_of(words, c.width, c.tokens, p.grad_products, p.n_tile, true, p.device_pairs);
            a.a = map_of(operand_type<T>(), probs_of, p.prob_parts, 64, kStep);
            a.b = map_of(operand_type<T>(), weighed_x, p.parts, 64, kStep);
            a.b_offset = 0;
            a.sums = nullptr;
            a.prior = false;
            a.last = true;
            gradient_of(static_cast<T*>(c.weight_grad) + first * c.width, words);
            launch_product(Kind::WeightGrad, c, t, a, words, c.width);
            finish<Kind::WeightGrad, T>(c, t, a);
        }
        if (c.x_grad != nullptr) {
            const Tiling t = tiling_of(c.tokens, c.width, words, p.grad_products, p.n_tile, true, p.device_pairs);
            a.a = map_of(operand_type<T>(), probs_of, p.prob_parts, kStep, kHalf);
            a.b = map_of(operand_type<T>(), w, p.parts, 64, kStep);
            a.b_offset = (unsigned)first;
            a.sums = p.pieces > 1 ? reinterpret_cast<float*>(workspace + p.sums_at) : nullptr;
            a.prior = piece != 0;
            a.last = piece + 1 == p.pieces;
            a.row_scale = powers;
            gradient_of(c.x_grad, c.tokens);
            launch_product(Kind::InputGrad, c, t, a, c.tokens, c.width);
            finish<Kind::InputGrad, T>(c, t, a);
        }
    }
}

// bf16, one loss for all rows: the loss and, but for what comes back to it, its gradients.
void both(const VocabularyLossCall& c, const Plan& p) {
    using T = __nv_bfloat16;
    char* workspace = static_cast<char*>(c.workspace);
    const Kept kept = kept_of(c);
    float* header = reinterpret_cast<float*>(workspace + p.header_at);
    unsigned* conditions = reinterpret_cast<unsigned*>(header + 2);
    float* losses = reinterpret_cast<float*>(workspace + p.losses_at);
    float* row_scale = reinterpret_cast<float*>(workspace + p.scale_at);
    Operand all_x, w;
    operands<T>(c, p, false, &all_x, &w);
    launch_entries(c, all_x, w, kept.top);
    CountArgs n;
    n.valid = kept.valid;
    n.rows = (unsigned)c.tokens;
    n.mean = c.reduction == LossReduction::Mean;
    n.temperature = c.temperature;
    n.count = kept.count;
    n.header = header;
    n.condition = conditions;
    n.conditions = (unsigned)p.pieces;
    B2_CUDA(launch_dependent<CountArgs>(count_kernel, dim3(1), 1024, 0, c.stream, n));
    for (u64 piece = 0; piece < p.pieces; ++piece) {
        const u64 first = piece * p.rows, rows = std::min<u64>(p.rows, c.tokens - first);
        const long long element = c.targets64 ? 8 : 4;
        const void* targets = static_cast<const char*>(c.targets) + (long long)first * c.target_strides[0] * element;
        const Operand x = {static_cast<const char*>(all_x.data) + first * all_x.row_bytes, c.width, rows, all_x.row_bytes};
        const Operand exps = {workspace + p.probs_at, p.exps_pitch, rows, p.exps_pitch * 2};
        unsigned* condition = conditions + piece;
        ProductArgs a = {};
        a.a = map_of(DType::BFloat16, x, 1, kStep, kHalf);
        a.b = map_of(DType::BFloat16, w, 1, kStep, kHalf);
        a.out = map_of(DType::BFloat16, exps, 1, 64, 32);
        a.out_parts = 1;
        logits_arguments(c, a);
        a.targets = targets;
        a.exp_sums = reinterpret_cast<float*>(workspace + p.stats_at);
        a.stats = reinterpret_cast<float2*>(workspace + p.stats_at);
        a.picked = a.entry_logits = reinterpret_cast<float*>(workspace + p.picked_at);
        a.words = kept.words + first;
        a.probs = kept.probs + first;
        a.hits = kept.hits + first / 32 * (unsigned)((c.entries + 31) / 32);  // (pieces of the rows are whole tiles)
        a.top = kept.top + first;
        a.sum = kept.sum + first;
        a.rest = kept.rest + first;
        a.valid = kept.valid + first;
        a.header = header;
        a.slots = reinterpret_cast<float*>(workspace + p.slots_at);
        const Tiling logits = tiling_of(rows, c.vocabulary, c.width, 1, kTile, false, p.device_pairs);
        launch_product(Kind::Exps, c, logits, a, rows, c.vocabulary);
        CloseArgs s;
        s.exp_sums = a.exp_sums;
        s.rows = (unsigned)rows;
        s.parts = 2 * logits.n_tiles;
        s.entries = (unsigned)c.entries;
        s.entry_stride = a.entry_stride;
        s.vocabulary = (long long)c.vocabulary;
        s.targets = targets;
        s.target_stride = c.target_strides[0];
        s.targets64 = c.targets64;
        s.words = a.words;
        s.z = a.entry_logits;
        s.p = a.probs;
        s.valid = a.valid;
        s.top = a.top;
        s.temperature = c.temperature;
        s.factor = a.factor;
        s.sum = kept.sum + first;
        s.rest = kept.rest + first;
        s.loss = losses + first;
        s.row_scale = row_scale;
        s.condition = condition;
        s.exps = reinterpret_cast<T*>(workspace + p.probs_at);
        s.pitch = p.exps_pitch;
        const dim3 by_32((unsigned)((rows + 31) / 32));
        B2_CUDA(launch_dependent<CloseArgs>(close_kernel, by_32, 1024, 0, c.stream, s));
        // Where E has not the exponents: P, from the largest logits.
        a.condition = condition;
        launch_product(Kind::Stats, c, logits, a, rows, c.vocabulary);
        JoinArgs j;
        j.stats = a.stats;
        j.rows = (unsigned)rows;
        j.parts = 2 * logits.n_tiles;
        j.picked = a.picked;
        j.targets = targets;
        j.target_stride = c.target_strides[0];
        j.targets64 = c.targets64;
        j.vocabulary = c.vocabulary;
        j.z = s.z;
        j.p = s.p;
        j.entries = (unsigned)c.entries;
        j.entry_stride = a.entry_stride;
        j.temperature = c.temperature;
        j.factor = a.factor;
        j.top = kept.top + first;
        j.sum = kept.sum + first;
        j.rest = kept.rest + first;
        j.valid = kept.valid + first;
        j.loss = losses + first;
        j.condition = condition;
        j.row_scale = row_scale;
        B2_CUDA(launch_dependent<JoinArgs>(join_kernel, by_32, 1024, 0, c.stream, j));
        launch_product(Kind::Probs, c, logits, a, rows, c.vocabulary);
        a.condition = nullptr;
        const auto gradient_of = [&](void* out, u64 of_rows) {
            a.gradient = out;
            a.wide = c.width * sizeof(T) % 16 == 0 && reinterpret_cast<std::uintptr_t>(out) % 16 == 0;
            if (a.wide) a.out = map_of(DType::BFloat16, {out, c.width, of_rows, c.width * sizeof(T)}, 1, 64, 32);
        };
        if (c.weight_grad != nullptr) {
            DivideArgs d;
            d.x = static_cast<const char*>(x.data);
            d.stride = (long long)x.row_bytes;
            d.out = reinterpret_cast<uint4*>(workspace + p.divided_at);
            d.rows = (unsigned)rows;
            d.columns = (unsigned)c.width;
            d.parts = p.divided_parts;
            d.eights = Divisor((unsigned)(p.pitch / 8));
            d.row_scale = row_scale;
            const u64 eights = rows * (p.pitch / 8);
            B2_REQUIRE(eights < (1ull << 31), kTooLarge);
            B2_CUDA(launch_dependent<DivideArgs>(divide_kernel, dim3((unsigned)((eights + 255) / 256)), 256, 0, c.stream, d));
            const Tiling t = tiling_of(c.vocabulary, c.width, rows, p.divided_parts, p.n_tile, true, p.device_pairs);
            a.a = map_of(DType::BFloat16, exps, 1, 64, kStep);
            a.b = map_of(DType::BFloat16, {d.out, c.width, rows, p.pitch * 2}, p.divided_parts, 64, kStep);
            a.b_in_parts = p.divided_parts == 2;
            a.sums = p.pieces > 1 ? reinterpret_cast<float*>(workspace + p.sums_at) : nullptr;
            a.prior = piece != 0;
            a.last = piece + 1 == p.pieces;
            gradient_of(c.weight_grad, c.vocabulary);
            launch_product(Kind::WeightGrad, c, t, a, c.vocabulary, c.width);
            finish<Kind::WeightGrad, T>(c, t, a);
            a.b_in_parts = false;
        }
        if (c.x_grad != nullptr) {
            const Tiling t = tiling_of(rows, c.width, c.vocabulary, 1, p.n_tile, true, p.device_pairs);
            a.a = map_of(DType::BFloat16, exps, 1, kStep, kHalf);
            a.b = map_of(DType::BFloat16, w, 1, 64, kStep);
            a.sums = nullptr;
            a.prior = false;
            a.last = true;
            a.row_scale = row_scale;
            gradient_of(static_cast<T*>(c.x_grad) + first * c.width, rows);
            launch_product(Kind::InputGrad, c, t, a, rows, c.width);
            finish<Kind::InputGrad, T>(c, t, a);
        }
    }
    SumArgs s;
    s.losses = losses;
    s.valid = kept.valid;
    s.rows = (unsigned)c.tokens;
    s.mean = n.mean;
    s.out = c.loss;
    s.count = kept.count;
    B2_CUDA(launch_dependent<SumArgs>(sum_kernel, dim3(1), 1024, 0, c.stream, s));
}

// Whether both() makes a call's gradients.
bool at_once(const VocabularyLossCall& c) {
    return c.dtype == DType::BFloat16 && c.reduction != LossReduction::None && c.tokens != 0 && (c.x_grad != nullptr || c.weight_grad != nullptr) && !small(c);
}

}  // namespace

std::size_t vocabulary_loss_kept(const VocabularyLossCall& c) {
    return c.tokens * 4 + 2 + 2 * c.tokens * (std::size_t)c.entries + hit_words(c) + (c.dtype == DType::Float ? c.tokens : 0);
}

std::size_t vocabulary_loss_workspace(const VocabularyLossCall& call, bool gradient) {
    return call.tokens == 0 ? 0 : plan_of(call, gradient ? Pass::Gradient : Pass::Loss).bytes;
}

std::size_t vocabulary_loss_both_workspace(const VocabularyLossCall& call) { return at_once(call) ? plan_of(call, Pass::Both).bytes : 0; }

void launch_vocabulary_loss_both(const VocabularyLossCall& c) {
    const Plan p = at_once(c) ? plan_of(c, Pass::Both) : Plan();
    B2_REQUIRE(p.bytes != 0, "the loss and its gradient are not made at once of such a call");
    both(c, p);
}

void launch_vocabulary_loss_times(const VocabularyLossCall& c) {
    B2_REQUIRE(c.dtype == DType::BFloat16, "gradients of bf16 only are made with the loss");
    ScaleArgs a;
    a.gradients[0] = static_cast<__nv_bfloat16*>(c.x_grad);
    a.gradients[1] = static_cast<__nv_bfloat16*>(c.weight_grad);
    a.elements[0] = (u64)c.tokens * c.width;
    a.elements[1] = (u64)c.vocabulary * c.width;
    a.loss_grad = c.loss_grad;
    const u64 most = std::max(a.gradients[0] != nullptr ? a.elements[0] : 0, a.gradients[1] != nullptr ? a.elements[1] : 0);
    if (most == 0) return;
    B2_CUDA(launch_dependent<ScaleArgs>(times_kernel, dim3((unsigned)std::min<u64>(148 * 4, (most + 4095) / 4096)), 512, 0, c.stream, a));
}

void launch_vocabulary_loss(const VocabularyLossCall& c) {
    if (c.tokens == 0) {
        if (c.reduction != LossReduction::None) B2_CUDA(cudaMemsetAsync(c.loss, 0, sizeof(float), c.stream));
        return;
    }
    const Plan p = plan_of(c, Pass::Loss);
    switch (c.dtype) {
        case DType::Float: return loss<float>(c, p);
        case DType::Float16: return loss<__half>(c, p);
        case DType::BFloat16: return loss<__nv_bfloat16>(c, p);
    }
}

void launch_vocabulary_loss_gradient(const VocabularyLossCall& c) {
    if (c.x_grad == nullptr && c.weight_grad == nullptr) return;
    if (c.tokens == 0) {
        if (c.weight_grad != nullptr) B2_CUDA(cudaMemsetAsync(c.weight_grad, 0, c.vocabulary * c.width * dtype_size(c.dtype), c.stream));
        return;
    }
    const Plan p = plan_of(c, Pass::Gradient);
    switch (c.dtype) {
        case DType::Float: return gradient<float>(c, p);
        case DType::Float16: return gradient<__half>(c, p);
        case DType::BFloat16: return gradient<__nv_bfloat16>(c, p);
    }
}

}  // namespace b200ccl::kernels
