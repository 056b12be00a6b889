// Queries and keys turned by their positions, alone or in the same pass as the norm of each head, and the gradients.
//
// A head is `dim` numbers; of its first `rotated` ones every pair (u, v) becomes magnitude * (u cos - v sin, u sin + v cos), angle =
// position * frequency of the pair. With the norm, the pair is first n = x * rstd * w, rstd = (mean x^2 + eps)^-1/2 over the head. The
// gradient of a rotation is the rotation back: g = R^T dy; of the norm, dw = sum g x rstd, dx = rstd (g w - x rstd^2 mean(g w x)).
//
// Bound by HBM: every head is read once and written once. Angles are made where they are used: position * frequency as
// turns in 64 bits, less its whole turns, then one sincospi in 32 bits (error 2e-7, and beyond 2^26 turns 2^-49 radians for each of them;
// in 32 bits the product alone is off by 0.06 at a million). A warp makes them once for its tokens, in shared memory of its own, and all heads of a token, of queries and
// keys, share them. Warps meet nowhere but at the end of the backward pass.
//
// A group of lanes holds a head: each lane V pairs at V neighbouring places of either half (interleaved: 2V neighbouring elements), so
// both elements of a pair are in one lane and no exchange is needed but the sums over a head. Elements that do not turn are
// pairs with no angle. V = 8 (two 16-byte accesses of 16-bit types), 4, 2 or 1, as sizes and addresses allow. Halves that do not begin at a multiple of 4
// would leave V = 1 for most of them; there a lane holds 2V neighbouring elements (Layout::Apart) and finds their partners in shared memory (norm, forward and
// backward, of 27264 x (8 + 4) x 128 bf16: 102 elements turned 475 -> 174 us; all of them, in halves, 116).
//
// 32768 x (32 + 8) x 128 bf16 turn in 104 us (6.4 TB/s, 0.98 of a copy's rate); with the norm, 16384 x (32 + 8) x 128 take 85 us, and 108 backward, 0.75 and 0.6 of that
// rate. Forward, 380 instructions for 16 elements of a lane take 0.68 of the issue slots, and the 64 registers that 32 warps leave are too few: 48 to 56 bytes spill, 84 to 108
// where pairs are interleaved. Backward, 126 registers leave 16 warps, which take 0.57 of the slots: the rest of the time none of them has an instruction ready.
//
// The inputs of the norm are kept for the backward pass in 8 bits, a head being a block (block8.cuh): the largest magnitude comes from
// the same exchange as the sum of squares.
#include "kernels/sm100/head_rotation.h"

#include "kernels/sm100/block8.cuh"
#include "kernels/sm100/launch.h"
#include "kernels/sm100/pair32.cuh"

#include <algorithm>
#include <cstdint>
#include <type_traits>

namespace b200ccl::kernels {

using namespace b200ccl::dev;

namespace {

using u64 = unsigned long long;
using i64 = long long;

constexpr unsigned kThreads = 256;
constexpr unsigned kWarps = kThreads / 32;
constexpr unsigned kMaxTileTokens = 8;  // of a warp's table
constexpr unsigned kSms = 148;

// How the pairs of a head lie, and what a lane holds of them. Half: V first elements and the V second ones. Interleaved: V pairs, which are 2V neighbouring
// elements. Apart: 2V neighbouring elements whose partners other lanes hold.
enum class Layout { Half, Interleaved, Apart };

struct View {
    const char* data;
    i64 batch, token, head;  // bytes
};

// How tokens are dealt out: a tile of tokens to a warp, or to `split` warps, each for some of the heads.
struct Cut {
    unsigned tile, split;
    unsigned tiles;  // times split
    unsigned ctas;   // backward: CTAs that take them in turn
};

struct Side {
    View x, grad;
    char* out;
    const char* weight;
    unsigned char* codes;
    unsigned char* scales;
    char* weight_grad;
    float* partial;
    Divisor heads;  // d = 0: none
    Cut cut;        // backward: a CTA works on one side
};

struct RotationArgs {
    Side side[2];
    const char* positions;
    i64 position_batch, position_token;  // elements
    const double* frequencies;
    unsigned all;     // tokens of all sequences
    Divisor tokens;   // of one
    Divisor angles;   // of a token in a table
    unsigned dim, rotated, pitch;
    unsigned items;  // lanes' worth of pairs in a head
    unsigned group;  // lanes that hold a head, a power of two
    Cut cut;  // forward: a warp works on both sides of its tokens
    float magnitude, sine;  // what cosines and sines are multiplied with
    float eps, over_dim;
    bool positions64;
};

// Items of a lane: 16 elements (V = 1: 8), so that what a row costs besides them, its address and its sums, is spread over as many. (fp32 forward: 8
// elements, and two rows at a time.)
template <typename T, int V>
__host__ __device__ constexpr int items_of_lane(bool back) {
    return V == 1 ? 4 : (V == 4 && sizeof(T) == 4 && !back ? 1 : 8 / V);
}

// Numbers go by twos: V of them are (V + 1) / 2 pairs; a single one has a zero beside it.
template <int V>
constexpr int kPairs = (V + 1) / 2;

// V neighbouring elements of T, as they lie in memory.
template <typename T, int V>
struct Some {
    static constexpr int kBytes = V * sizeof(T);
    using Word = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<V == 2, unsigned, T>>>;
    static_assert(V == 1 || V == 2 || kBytes == 8 || kBytes == 16);
    Word w;
    __device__ __forceinline__ void clear() { w = Word(); }
    __device__ __forceinline__ void load(const char* p) {
        if constexpr (kBytes == 16) w = load16_once(p);
        else w = *reinterpret_cast<const Word*>(p);
    }
    __device__ __forceinline__ unsigned word(int i) const {
        if constexpr (kBytes == 16) return i == 0 ? w.x : (i == 1 ? w.y : (i == 2 ? w.z : w.w));
        else if constexpr (kBytes == 8) return i == 0 ? w.x : w.y;
        else return w;
    }
    static __device__ __forceinline__ float2 two(unsigned word) {
        if constexpr (std::is_same_v<T, __half>) return h2_to_f2(word);
        else return b2_to_f2(word);
    }
    __device__ __forceinline__ void widen(Pair32 (&f)[kPairs<V>]) const {
        if constexpr (V == 1) {
            f[0] = pair32(Elem<T>::to_f(w), 0.0f);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                if constexpr (sizeof(T) == 4) {
                    f[i] = pair32(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
                } else {
                    const float2 g = two(word(i));
                    f[i] = pair32(g.x, g.y);
                }
            }
        }
    }
    static __device__ __forceinline__ void store(char* p, const Pair32 (&f)[kPairs<V>]) {
        if constexpr (V == 1) {
            *reinterpret_cast<T*>(p) = Elem<T>::from_f(apart(f[0]).x);
        } else if constexpr (sizeof(T) == 4 && V == 2) {
            const float2 a = apart(f[0]);
            *reinterpret_cast<uint2*>(p) = make_uint2(__float_as_uint(a.x), __float_as_uint(a.y));
        } else if constexpr (sizeof(T) == 4) {
            const float2 a = apart(f[0]), b = apart(f[1]);
            store16_once(p, make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y)));
        } else {
            unsigned r[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 g = apart(f[i]);
                r[i] = std::is_same_v<T, __half> ? f2_to_h2(g.x, g.y) : f2_to_b2(g.x, g.y);
            }
            if constexpr (V == 8) store16_once(p, make_uint4(r[0], r[1], r[2], r[3]));
            else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(r[0], r[1]);
            else *reinterpret_cast<unsigned*>(p) = r[0];
        }
    }
    // The largest magnitude so far and of these: of 16-bit types as two halves, see larger_magnitudes<T>().
    __device__ __forceinline__ unsigned larger(unsigned so_far) const {
        if constexpr (V == 1) {
            return max(so_far, magnitude_bits(Elem<T>::to_f(w)));
        } else if constexpr (sizeof(T) == 4 && V == 2) {
            return max(so_far, max(w.x & 0x7fffffffu, w.y & 0x7fffffffu));
        } else if constexpr (sizeof(T) == 4) {
            return max(max(so_far, max(w.x & 0x7fffffffu, w.y & 0x7fffffffu)), max(w.z & 0x7fffffffu, w.w & 0x7fffffffu));
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) so_far = larger_magnitudes<T>(so_far, word(i));
            return so_far;
        }
    }
    static __device__ __forceinline__ unsigned magnitude(unsigned larger) { return V > 1 && sizeof(T) == 2 ? magnitude_of_pair<T>(larger) : larger; }
    // Its codes, to where they are kept.
    __device__ __forceinline__ void keep(unsigned char* p, unsigned scale) const {
        using Out = std::conditional_t<V == 8, uint2, std::conditional_t<V == 4, unsigned, std::conditional_t<V == 2, unsigned short, unsigned char>>>;
        if (scale == 255u) {
            *reinterpret_cast<Out*>(p) = Out();
        } else if constexpr (V == 1) {
            *p = (unsigned char)encode8(Elem<T>::to_f(w), inverse_step8(scale));
        } else if constexpr (V == 2) {
            const float inverse = inverse_step8(scale);
            const float2 f = sizeof(T) == 4 ? make_float2(__uint_as_float(word(0)), __uint_as_float(word(kBytes / 8))) : two(word(0));
            *reinterpret_cast<unsigned short*>(p) = (unsigned short)(encode8(f.x, inverse) | encode8(f.y, inverse) << 8);
        } else if constexpr (sizeof(T) == 4) {
            const float f[4] = {__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)};
            *reinterpret_cast<unsigned*>(p) = encode8x4(f, inverse_step8(scale));
        } else {
            const Inverse16<T> inverse(scale);
            const unsigned a = encode8x4(word(0), word(1), inverse);
            if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(a, encode8x4(word(2), word(3), inverse));
            else *reinterpret_cast<unsigned*>(p) = a;
        }
    }
};
// V neighbouring codes. What they stand for is a bf16 number too where T is fp32.
template <typename T, int V>
struct Codes {
    using Word = std::conditional_t<V == 8, uint2, std::conditional_t<V == 4, unsigned, std::conditional_t<V == 2, unsigned short, unsigned char>>>;
    using Narrow16 = std::conditional_t<std::is_same_v<T, __half>, __half, __nv_bfloat16>;
    Word w;
    __device__ __forceinline__ void clear() { w = Word(); }
    __device__ __forceinline__ void load(const unsigned char* p) { w = *reinterpret_cast<const Word*>(p); }
    static __device__ __forceinline__ void four(unsigned word, unsigned step, Pair32* f) {
        const uint2 v = widen8x4<Narrow16>(word, step);
        const float2 a = Some<Narrow16, 4>::two(v.x), b = Some<Narrow16, 4>::two(v.y);
        f[0] = pair32(a.x, a.y);
        f[1] = pair32(b.x, b.y);
    }
    __device__ __forceinline__ void widen(unsigned scale, Pair32 (&f)[kPairs<V>]) const {
        if constexpr (V == 1) {
            f[0] = pair32(decode8<0>(w, step8(scale)), 0.0f);
        } else if constexpr (V == 2) {
            f[0] = pair32(decode8<0>(w, step8(scale)), decode8<1>(w, step8(scale)));
        } else {
            const unsigned step = step16<Narrow16>(scale);
            if constexpr (V == 8) {
                four(w.x, step, f);
                four(w.y, step, f + 2);
            } else {
                four(w, step, f);
            }
        }
    }
};

// Where a lane's pairs lie in a head: first elements at `first`, second ones at `second` (interleaved or apart: 2V elements from `first` on).
struct Place {
    unsigned pair, first, second;
};
template <int V, Layout kLayout>
__device__ __forceinline__ Place place_of(const RotationArgs& a, unsigned item) {
    const unsigned p = item * V, turning = a.rotated / 2;
    if (kLayout != Layout::Half) return {p, 2 * p, 2 * p + V};
    if (p < turning) return {p, p, p + turning};
    const unsigned first = a.rotated + (p - turning);
    return {p, first, first + (a.dim - a.rotated) / 2};
}

// u, v: the first and second elements of the lane's pairs, in order. Interleaved ones arrive as u0 v0 u1 v1 ...
template <int V>
__device__ __forceinline__ void part(Pair32 (&u)[kPairs<V>], Pair32 (&v)[kPairs<V>]) {
    if constexpr (V > 1) {
        float2 f[V];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) { f[i] = apart(u[i]); f[V / 2 + i] = apart(v[i]); }
#pragma unroll
        for (int i = 0; i < V / 2; ++i) { u[i] = pair32(f[2 * i].x, f[2 * i + 1].x); v[i] = pair32(f[2 * i].y, f[2 * i + 1].y); }
    }
}
template <int V>
__device__ __forceinline__ void join(Pair32 (&u)[kPairs<V>], Pair32 (&v)[kPairs<V>]) {
    if constexpr (V > 1) {
        float2 f[V];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 a = apart(u[i]), b = apart(v[i]);
            f[2 * i] = make_float2(a.x, b.x);
            f[2 * i + 1] = make_float2(a.y, b.y);
        }
#pragma unroll
        for (int i = 0; i < V / 2; ++i) { u[i] = pair32(f[i].x, f[i].y); v[i] = pair32(f[V / 2 + i].x, f[V / 2 + i].y); }
    }
}
template <typename T, int V, Layout kLayout>
__device__ __forceinline__ void load_pairs(const char* head, const Place& at, Pair32 (&u)[kPairs<V>], Pair32 (&v)[kPairs<V>]) {
    Some<T, V> a, b;
    a.load(head + at.first * sizeof(T));
    b.load(head + at.second * sizeof(T));
    a.widen(u);
    b.widen(v);
    if constexpr (kLayout == Layout::Interleaved) part<V>(u, v);
}
template <typename T, int V, Layout kLayout>
__device__ __forceinline__ void store_pairs(char* head, const Place& at, Pair32 (&u)[kPairs<V>], Pair32 (&v)[kPairs<V>]) {
    if constexpr (kLayout == Layout::Interleaved) join<V>(u, v);
    Some<T, V>::store(head + at.first * sizeof(T), u);
    Some<T, V>::store(head + at.second * sizeof(T), v);
}

__device__ __forceinline__ float group_sum(float v, unsigned group) {
#pragma unroll
    for (unsigned o = 16; o > 0; o >>= 1)
        if (o < group) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ unsigned group_max(unsigned v, unsigned group) {
#pragma unroll
    for (unsigned o = 16; o > 0; o >>= 1)
        if (o < group) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// A warp's share of the work: some tokens, and of their heads one part in `split`.
struct Tile {
    unsigned token, tokens, part;
};
__device__ __forceinline__ Tile tile_at(const RotationArgs& a, const Cut& cut, unsigned index) {
    const unsigned t = cut.split == 1u ? index : index / cut.split;
    return {t * cut.tile, min(cut.tile, a.all - t * cut.tile), index - t * cut.split};
}
// Its rows (heads of tokens, in order) of one side.
struct Rows {
    unsigned from, to;
};
__device__ __forceinline__ Rows rows_of(const Cut& cut, const Side& s, const Tile& t) {
    const unsigned rows = t.tokens * s.heads.d;
    if (cut.split == 1u) return {0u, rows};
    const unsigned each = (rows + cut.split - 1u) / cut.split;
    return {min(rows, t.part * each), min(rows, (t.part + 1u) * each)};
}

// Cosines and sines of a tile's tokens, in a warp's own shared memory: (cos, cos, sin, sin) of two pairs (of one, with zeros: V = 1) of an item, those of
// neighbouring items beside one another, so that lanes read neighbouring 16 bytes. An interleaved item may hold pairs that do not turn behind others that do;
// the table has places for them. Apart: (cos, sin) of each pair, with a gap after every 2V, so that lanes read from different banks.
template <int V, Layout kLayout>
__host__ __device__ __forceinline__ unsigned table_items(const RotationArgs& a) {
    return kLayout == Layout::Interleaved ? (a.rotated / 2 + V - 1) / V : a.rotated / 2 / V;
}
template <int V, Layout kLayout>
__host__ __device__ __forceinline__ unsigned table_entries(const RotationArgs& a) {
    if (kLayout == Layout::Apart) return (a.rotated / 2 + a.rotated / 2 / (2 * V) + 2) / 2;
    return table_items<V, kLayout>(a) * kPairs<V>;
}
template <int V, Layout kLayout>
__device__ __forceinline__ void make_table(const RotationArgs& a, const Tile& tile, float4* table) {
    const unsigned pairs = a.rotated / 2, items = table_items<V, kLayout>(a), entries = table_entries<V, kLayout>(a);
    const unsigned all = pairs == 0 ? 0u : tile.tokens * a.angles.d;
    // Two angles of a lane at a time, so that their loads are on the way together.
    for (unsigned i0 = threadIdx.x & 31u; i0 < all; i0 += 64u) {
        double position[2], frequency[2];
        unsigned token[2], pair[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const unsigned i = min(i0 + 32u * j, all - 1u);
            token[j] = a.angles.divide(i);
            pair[j] = i - token[j] * a.angles.d;
            const unsigned n = tile.token + token[j], b = a.tokens.divide(n);
            const i64 at = (i64)b * a.position_batch + (i64)(n - b * a.tokens.d) * a.position_token;
            position[j] = a.positions64 ? (double)*(reinterpret_cast<const i64*>(a.positions) + at) : (double)*(reinterpret_cast<const int*>(a.positions) + at);
            frequency[j] = kLayout != Layout::Interleaved || pair[j] < pairs ? a.frequencies[pair[j]] : 0.0;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (j != 0 && i0 + 32u * j >= all) continue;
            const unsigned p = pair[j];
            double turns = position[j] * (frequency[j] * 0.15915494309189535);  // 1 / (2 pi)
            turns -= rint(turns);
            float sine, cosine;
            sincospif((float)(2.0 * turns), &sine, &cosine);
            sine *= a.sine;
            cosine *= a.magnitude;
            if constexpr (kLayout == Layout::Apart) {
                *(reinterpret_cast<float2*>(table + token[j] * entries) + p + p / (2 * V)) = make_float2(cosine, sine);
            } else {
                float* entry = reinterpret_cast<float*>(table + token[j] * entries + (p % V / 2) * items + p / V);
                entry[p % V % 2] = cosine;
                entry[2 + p % V % 2] = sine;
                if constexpr (V == 1) entry[1] = entry[3] = 0.0f;
            }
        }
    }
}

// Turns the K items of a lane, by their token's angles. All lanes of a warp call it; `row`: shared memory of the lane's head (apart).
template <int V, int K, Layout kLayout>
__device__ __forceinline__ void turn(const RotationArgs& a, const float4* angles, float* row, const Place (&at)[K], const bool (&mine)[K],
                                     Pair32 (&u)[K][kPairs<V>], Pair32 (&v)[K][kPairs<V>]) {
    if constexpr (kLayout != Layout::Apart) {
        const unsigned items = table_items<V, kLayout>(a), pairs = a.rotated / 2;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const unsigned item = at[k].pair / V;
            if (!mine[k] || item >= items) continue;
            if (kLayout == Layout::Interleaved && V > 1 && pairs % V != 0) {
                // The last item may hold pairs that do not turn. (The angle 0 would not do for them: infinity times its sine is not 0.)
#pragma unroll
                for (int i = 0; i < kPairs<V>; ++i) {
                    const float4 cs = angles[i * items + item];
                    const float2 x = apart(u[k][i]), y = apart(v[k][i]);
                    const bool first = at[k].pair + 2 * i < pairs, second = at[k].pair + 2 * i + 1 < pairs;
                    u[k][i] = pair32(first ? x.x * cs.x - y.x * cs.z : x.x, second ? x.y * cs.y - y.y * cs.w : x.y);
                    v[k][i] = pair32(first ? x.x * cs.z + y.x * cs.x : y.x, second ? x.y * cs.w + y.y * cs.y : y.y);
                }
                continue;
            }
#pragma unroll
            for (int i = 0; i < kPairs<V>; ++i) {
                const float4 cs = angles[i * items + item];
                const Pair32 c = pair32(cs.x, cs.y), s = pair32(cs.z, cs.w), x = u[k][i], y = v[k][i];
                u[k][i] = fma2(mul2(y, s), both32(-1.0f), mul2(x, c));
                v[k][i] = fma2(x, s, mul2(y, c));
            }
        }
    } else {
        // Element e lies at e + e / 2V: the lanes' elements j are at odd distances.
        const unsigned half = a.rotated / 2;
        float f[K][2 * V];
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 x = apart(u[k][j / 2]), y = apart(v[k][j / 2]);
                f[k][j] = j % 2 == 0 ? x.x : x.y;
                f[k][V + j] = j % 2 == 0 ? y.x : y.y;
            }
            if (mine[k]) {
#pragma unroll
                for (int j = 0; j < 2 * V; ++j) row[at[k].first + at[k].first / (2 * V) + j] = f[k][j];
            }
        }
        __syncwarp();
        const float2* table = reinterpret_cast<const float2*>(angles);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!mine[k] || at[k].first >= a.rotated) continue;
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
                // (No branch, so that all reads are on the way together; those behind the last pair are for nothing.)
                const unsigned e = at[k].first + j;
                const bool turns = e < a.rotated, low = e < half;
                const unsigned pair = turns ? (low ? e : e - half) : 0u, other = low ? e + half : pair;
                const float2 cs = table[pair + pair / (2 * V)];
                const float turned = fmaf(row[other + other / (2 * V)], low ? -cs.y : cs.y, f[k][j] * cs.x);
                f[k][j] = turns ? turned : f[k][j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (j % 2 == 0) {
                    u[k][j / 2] = pair32(f[k][j], V == 1 ? 0.0f : f[k][j + (V > 1)]);
                    v[k][j / 2] = pair32(f[k][V + j], V == 1 ? 0.0f : f[k][V + j + (V > 1)]);
                }
            }
        }
        __syncwarp();
    }
}
// Floats of a lane's share of a head in shared memory: an odd number, so that heads begin in different banks too.
template <int V, int K>
constexpr unsigned kLaneFloats = (K * (2 * V + 1)) | 1;
template <int V, int K, Layout kLayout>
constexpr unsigned kRowFloats = kLayout == Layout::Apart ? 32 * kLaneFloats<V, K> : 0;

// One row of one side: which token of the tile it belongs to, and where its head lies in a view.
struct Row {
    bool there;
    unsigned token;  // of the tile
    unsigned n, b, h;
};
__device__ __forceinline__ Row row_at(const RotationArgs& a, const Side& s, const Tile& tile, unsigned r, unsigned to) {
    Row w;
    w.there = r < to;
    w.token = w.there ? s.heads.divide(r) : 0u;
    w.h = w.there ? r - w.token * s.heads.d : 0u;
    w.n = tile.token + w.token;
    w.b = a.tokens.divide(w.n);
    return w;
}
__device__ __forceinline__ const char* head_in(const RotationArgs& a, const View& v, const Row& w) {
    return v.data + (i64)w.b * v.batch + (i64)(w.n - w.b * a.tokens.d) * v.token + (i64)w.h * v.head;
}

// K: items of a lane. U: rows of a group in flight. (Apart: 80 registers, because in 64 it spills 130 bytes; forward alone 66 -> 63 us.)
template <typename T, int V, int K, Layout kLayout, bool kNorm, int U>
__global__ void __launch_bounds__(kThreads, kLayout == Layout::Apart ? 3 : 4) rotate_kernel(const __grid_constant__ RotationArgs a) {
    constexpr int P = kPairs<V>;
    extern __shared__ __align__(16) unsigned char shared[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned warp = threadIdx.x / 32u, index = blockIdx.x * kWarps + warp;
    if (index >= a.cut.tiles) return;
    const Tile tile = tile_at(a, a.cut, index);
    const unsigned lane = threadIdx.x & (a.group - 1u), groups = 32u / a.group, group = (threadIdx.x & 31u) / a.group;
    const unsigned entries = table_entries<V, kLayout>(a);
    float4* table = reinterpret_cast<float4*>(shared) + warp * a.cut.tile * entries;
    float* heads = reinterpret_cast<float*>(reinterpret_cast<float4*>(shared) + kWarps * a.cut.tile * entries) + warp * kRowFloats<V, K, kLayout> + group * a.group * kLaneFloats<V, K>;
    Place at[K];
    bool mine[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned item = lane + k * a.group;
        mine[k] = item < a.items;
        at[k] = place_of<V, kLayout>(a, mine[k] ? item : 0u);
    }
    bool made = false;
    // (Each side in code of its own: which it is is then known to the compiler, and its arguments are operands instead of loads.)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const Side& s = a.side[i];
        if (s.heads.d == 0u) continue;
        const Rows rows = rows_of(a.cut, s, tile);
        Pair32 wu[kNorm ? K : 1][P], wv[kNorm ? K : 1][P];
        if constexpr (kNorm) {
#pragma unroll
            for (int k = 0; k < K; ++k) load_pairs<T, V, kLayout>(s.weight, at[k], wu[k], wv[k]);
        }
        // (All lanes of a warp stay to the end of a pass: they exchange sums.)
        for (unsigned r0 = rows.from; r0 < rows.to; r0 += groups * U) {
            Some<T, V> first[U][K], second[U][K];
            Row row[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                row[j] = row_at(a, s, tile, r0 + j * groups + group, rows.to);
                const char* head = head_in(a, s.x, row[j]);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (row[j].there && mine[k]) {
                        first[j][k].load(head + at[k].first * sizeof(T));
                        second[j][k].load(head + at[k].second * sizeof(T));
                    } else {
                        first[j][k].clear();
                        second[j][k].clear();
                    }
                }
            }
            if (!made) {  // while the first rows are on the way
                make_table<V, kLayout>(a, tile, table);
                __syncwarp();
                made = true;
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const u64 r = (u64)row[j].n * s.heads.d + row[j].h;
                if (kNorm && s.codes != nullptr) {
                    unsigned amax = 0;
#pragma unroll
                    for (int k = 0; k < K; ++k) amax = second[j][k].larger(first[j][k].larger(amax));
                    const unsigned scale = scale8<T>(group_max(Some<T, V>::magnitude(amax), a.group));
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        if (row[j].there && mine[k]) {
                            first[j][k].keep(s.codes + r * a.pitch + at[k].first, scale);
                            second[j][k].keep(s.codes + r * a.pitch + at[k].second, scale);
                        }
                    }
                    if (row[j].there && lane == 0) s.scales[r] = (unsigned char)scale;
                }
                Pair32 u[K][P], v[K][P];
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    first[j][k].widen(u[k]);
                    second[j][k].widen(v[k]);
                    if constexpr (kLayout == Layout::Interleaved) part<V>(u[k], v[k]);
                }
                if constexpr (kNorm) {
                    Pair32 sum = both32(0.0f);
#pragma unroll
                    for (int k = 0; k < K; ++k) {
#pragma unroll
                        for (int e = 0; e < P; ++e) sum = fma2(u[k][e], u[k][e], fma2(v[k][e], v[k][e], sum));
                    }
                    const float2 squares = apart(sum);
                    const Pair32 rstd = both32(rsqrtf(fmaf(group_sum(squares.x + squares.y, a.group), a.over_dim, a.eps)));
#pragma unroll
                    for (int k = 0; k < K; ++k) {
#pragma unroll
                        for (int e = 0; e < P; ++e) {
                            u[k][e] = mul2(mul2(u[k][e], rstd), wu[k][e]);
                            v[k][e] = mul2(mul2(v[k][e], rstd), wv[k][e]);
                        }
                    }
                }
                turn<V, K, kLayout>(a, table + row[j].token * entries, heads, at, mine, u, v);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (row[j].there && mine[k]) {
                        store_pairs<T, V, kLayout>(s.out + r * a.dim * sizeof(T), at[k], u[k], v[k]);
                    }
                }
            }
        }
    }
}

// Gradients of the norm and rotation. A CTA belongs to one side and its warps take tile after tile, so that a lane's share of the weight's gradient
// stays in registers; the CTA's share goes to `partial` and sum_kernel adds them in order, so that results do not depend on which CTA ends first.
template <typename T, int V, int K, Layout kLayout, bool kCodes, int U>
__device__ __forceinline__ void rotate_norm_backward(const RotationArgs& a, const Side& s, unsigned cta, unsigned char* shared) {
    constexpr int P = kPairs<V>;
    const unsigned warp = threadIdx.x / 32u, in_warp = threadIdx.x & 31u, lane = threadIdx.x & (a.group - 1u);
    const unsigned groups = 32u / a.group, group = in_warp / a.group, entries = table_entries<V, kLayout>(a);
    float4* table = reinterpret_cast<float4*>(shared) + warp * s.cut.tile * entries;
    float* heads = reinterpret_cast<float*>(reinterpret_cast<float4*>(shared) + kWarps * s.cut.tile * entries) + warp * kRowFloats<V, K, kLayout> + group * a.group * kLaneFloats<V, K>;
    Place at[K];
    bool mine[K];
    Pair32 wu[K][P], wv[K][P], du[K][P], dv[K][P];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned item = lane + k * a.group;
        mine[k] = item < a.items;
        at[k] = place_of<V, kLayout>(a, mine[k] ? item : 0u);
        load_pairs<T, V, kLayout>(s.weight, at[k], wu[k], wv[k]);
#pragma unroll
        for (int i = 0; i < P; ++i) du[k][i] = dv[k][i] = both32(0.0f);
    }
    for (unsigned index = cta * kWarps + warp; index < s.cut.tiles; index += s.cut.ctas * kWarps) {
        const Tile tile = tile_at(a, s.cut, index);
        const Rows rows = rows_of(s.cut, s, tile);
        for (unsigned r0 = rows.from; r0 < rows.to; r0 += groups * U) {
            Some<T, V> g1[U][K], g2[U][K];
            std::conditional_t<kCodes, Codes<T, V>, Some<T, V>> x1[U][K], x2[U][K];
            unsigned scale[U];
            Row row[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                row[j] = row_at(a, s, tile, r0 + j * groups + group, rows.to);
                const char* grad = head_in(a, s.grad, row[j]);
                const u64 r = (u64)row[j].n * s.heads.d + row[j].h;
                scale[j] = kCodes ? s.scales[r] : 0u;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (row[j].there && mine[k]) {
                        g1[j][k].load(grad + at[k].first * sizeof(T));
                        g2[j][k].load(grad + at[k].second * sizeof(T));
                        if constexpr (kCodes) {
                            x1[j][k].load(s.codes + r * a.pitch + at[k].first);
                            x2[j][k].load(s.codes + r * a.pitch + at[k].second);
                        } else {
                            const char* x = head_in(a, s.x, row[j]);
                            x1[j][k].load(x + at[k].first * sizeof(T));
                            x2[j][k].load(x + at[k].second * sizeof(T));
                        }
                    } else {
                        g1[j][k].clear();
                        g2[j][k].clear();
                        x1[j][k].clear();
                        x2[j][k].clear();
                    }
                }
            }
            if (r0 == rows.from) {  // while the first rows are on the way
                __syncwarp();       // the table of the tile before has been read
                make_table<V, kLayout>(a, tile, table);
                __syncwarp();
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                Pair32 gu[K][P], gv[K][P], u[K][P], v[K][P];
                Pair32 sum = both32(0.0f), product = both32(0.0f);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    g1[j][k].widen(gu[k]);
                    g2[j][k].widen(gv[k]);
                    if constexpr (kLayout == Layout::Interleaved) part<V>(gu[k], gv[k]);
                }
                turn<V, K, kLayout>(a, table + row[j].token * entries, heads, at, mine, gu, gv);
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if constexpr (kCodes) {
                        // (Zero times the step of a head that is not finite is not zero: lanes without elements take another step.)
                        const unsigned step = mine[k] ? scale[j] : 127u;
                        x1[j][k].widen(step, u[k]);
                        x2[j][k].widen(step, v[k]);
                    } else {
                        x1[j][k].widen(u[k]);
                        x2[j][k].widen(v[k]);
                    }
                    if constexpr (kLayout == Layout::Interleaved) part<V>(u[k], v[k]);
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        sum = fma2(u[k][e], u[k][e], fma2(v[k][e], v[k][e], sum));
                        product = fma2(mul2(gu[k][e], wu[k][e]), u[k][e], fma2(mul2(gv[k][e], wv[k][e]), v[k][e], product));
                    }
                }
                const float2 squares = apart(sum), products = apart(product);
                const float mean = group_sum(squares.x + squares.y, a.group) * a.over_dim, dot = group_sum(products.x + products.y, a.group) * a.over_dim;
                if (!row[j].there) continue;
                const float r1 = rsqrtf(mean + a.eps);
                const Pair32 rstd = both32(r1), back = both32(-dot * r1 * r1);
                const u64 r = (u64)row[j].n * s.heads.d + row[j].h;
#pragma unroll
                for (int k = 0; k < K; ++k) {
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        du[k][e] = fma2(mul2(gu[k][e], rstd), u[k][e], du[k][e]);
                        dv[k][e] = fma2(mul2(gv[k][e], rstd), v[k][e], dv[k][e]);
                        u[k][e] = mul2(rstd, fma2(u[k][e], back, mul2(gu[k][e], wu[k][e])));
                        v[k][e] = mul2(rstd, fma2(v[k][e], back, mul2(gv[k][e], wv[k][e])));
                    }
                    if (mine[k]) store_pairs<T, V, kLayout>(s.out + r * a.dim * sizeof(T), at[k], u[k], v[k]);
                }
            }
            __syncwarp();
        }
    }
    // The groups of a warp, then the warps.
    __syncthreads();
    float* sums = reinterpret_cast<float*>(shared);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float x = i % 2 == 0 ? apart(du[k][i / 2]).x : apart(du[k][i / 2]).y, y = i % 2 == 0 ? apart(dv[k][i / 2]).x : apart(dv[k][i / 2]).y;
            for (unsigned o = a.group; o < 32u; o <<= 1) {
                x += __shfl_xor_sync(0xffffffffu, x, o);
                y += __shfl_xor_sync(0xffffffffu, y, o);
            }
            if (in_warp < a.group && mine[k]) {
                sums[warp * a.dim + (kLayout == Layout::Interleaved ? at[k].first + 2 * i : at[k].first + i)] = x;
                sums[warp * a.dim + (kLayout == Layout::Interleaved ? at[k].first + 2 * i + 1 : at[k].second + i)] = y;
            }
        }
    }
    __syncthreads();
    for (unsigned d = threadIdx.x; d < a.dim; d += kThreads) {
        float sum = 0.0f;
        for (unsigned w = 0; w < kWarps; ++w) sum += sums[w * a.dim + d];
        s.partial[(u64)cta * a.dim + d] = sum;
    }
}

template <typename T, int V, int K, Layout kLayout, bool kCodes, int U>
__global__ void __launch_bounds__(kThreads, 2) rotate_norm_backward_kernel(const __grid_constant__ RotationArgs a) {
    extern __shared__ __align__(16) unsigned char shared[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned ctas = a.side[0].cut.ctas;
    if (blockIdx.x < ctas) rotate_norm_backward<T, V, K, kLayout, kCodes, U>(a, a.side[0], blockIdx.x, shared);
    else rotate_norm_backward<T, V, K, kLayout, kCodes, U>(a, a.side[1], blockIdx.x - ctas, shared);
}

// weight_grad[d] = sum of partial[cta][d]: 32 columns of one side per CTA.
template <typename T>
__global__ void __launch_bounds__(1024) sum_kernel(const __grid_constant__ RotationArgs a) {
    __shared__ float sums[32][33];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Side& s = a.side[blockIdx.y];
    const unsigned column = blockIdx.x * 32u + (threadIdx.x & 31u), part = threadIdx.x >> 5;
    if (s.weight_grad == nullptr) return;
    // (All loads at once: 295 x 128 sums, 5.6 us; one after another, 7.0.)
    constexpr unsigned kEach = (kHeadGradCtas + 31) / 32;
    float x[kEach], sum = 0.0f;
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) {
        const unsigned c = part + i * 32u;
        x[i] = column < a.dim && c < s.cut.ctas ? s.partial[(u64)c * a.dim + column] : 0.0f;
    }
#pragma unroll
    for (unsigned i = 0; i < kEach; ++i) sum += x[i];
    sums[part][threadIdx.x & 31u] = sum;
    __syncthreads();
    sum = sums[threadIdx.x & 31u][part];  // warp `part` adds column `part`
    for (unsigned o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const unsigned d = blockIdx.x * 32u + part;
    if ((threadIdx.x & 31u) == 0 && d < a.dim) reinterpret_cast<T*>(s.weight_grad)[d] = Elem<T>::from_f(sum);
}

struct Shape {
    unsigned vector, items, group;
    Layout layout;
};

View view_of(const HeadsView& v, long long bytes) {
    return {static_cast<const char*>(v.data), v.batch * bytes, v.token * bytes, v.head * bytes};
}

// Whether V elements of every head that is touched are one access.
bool fits(const RotationCall& c, Layout layout, unsigned v, unsigned bytes) {
    const unsigned turning = c.rotated / 2, rest = (c.dim - c.rotated) / 2;
    if (layout == Layout::Half ? turning % v != 0 || rest % v != 0 : c.dim / 2 % v != 0) return false;
    std::uintptr_t bits = 0;
    for (const HeadsSide& s : c.side) {
        if (s.heads == 0) continue;
        for (const HeadsView* w : {&s.x, &s.grad})
            if (w->data != nullptr) bits |= reinterpret_cast<std::uintptr_t>(w->data) | (std::uintptr_t)((w->batch | w->token | w->head) * (long long)bytes);
        bits |= reinterpret_cast<std::uintptr_t>(s.out) | reinterpret_cast<std::uintptr_t>(s.weight) | (std::uintptr_t)c.dim * bytes;
    }
    return bits % (v * bytes) == 0;
}

template <typename T>
Shape shape_of(const RotationCall& c, bool back) {
    constexpr unsigned kWidest = 16 / sizeof(T);
    Shape s;
    s.layout = c.interleaved ? Layout::Interleaved : Layout::Half;
    s.vector = kWidest;
    while (s.vector > 1 && !fits(c, s.layout, s.vector, sizeof(T))) s.vector /= 2;
    if (s.layout == Layout::Half && s.vector < 4) {
        s.layout = Layout::Apart;
        s.vector = kWidest;
        while (s.vector > 1 && !fits(c, s.layout, s.vector, sizeof(T))) s.vector /= 2;
    }
    s.items = (unsigned)c.dim / 2 / s.vector;
    const unsigned of_lane = s.vector == 8 ? items_of_lane<T, 8>(back) : (s.vector == 4 ? items_of_lane<T, 4>(back) : (s.vector == 2 ? items_of_lane<T, 2>(back) : items_of_lane<T, 1>(back)));
    s.group = 1;
    while (s.group * of_lane < s.items) s.group *= 2;
    return s;
}

RotationArgs args_of(const RotationCall& c, const Shape& shape, unsigned bytes) {
    RotationArgs a = {};
    a.positions = static_cast<const char*>(c.positions);
    a.position_batch = c.position_batch;
    a.position_token = c.position_token;
    a.positions64 = c.positions64;
    a.frequencies = c.frequencies;
    a.all = (unsigned)(c.batch * c.tokens);
    a.tokens = Divisor((unsigned)std::max(1ll, c.tokens));
    const unsigned pairs = (unsigned)c.rotated / 2;
    a.angles = Divisor(std::max(1u, shape.layout == Layout::Interleaved ? (pairs + shape.vector - 1) / shape.vector * shape.vector : pairs));
    a.dim = (unsigned)c.dim;
    a.rotated = (unsigned)c.rotated;
    a.pitch = (a.dim + 15u) / 16u * 16u;
    a.items = shape.items;
    a.group = shape.group;
    a.magnitude = c.magnitude;
    a.sine = c.inverse ? -c.magnitude : c.magnitude;
    a.eps = c.eps;
    a.over_dim = 1.0f / (float)c.dim;
    for (int i = 0; i < 2; ++i) {
        const HeadsSide& s = c.side[i];
        Side& t = a.side[i];
        t.x = view_of(s.x, bytes);
        t.grad = view_of(s.grad, bytes);
        t.out = static_cast<char*>(s.out);
        t.weight = static_cast<const char*>(s.weight);
        t.codes = s.codes;
        t.scales = s.scales;
        t.weight_grad = static_cast<char*>(s.weight_grad);
        t.partial = s.partial;
        if (s.heads != 0) t.heads = Divisor((unsigned)s.heads);
    }
    return a;
}

// A warp's tile: as many tokens as give it a round of rows of the side with fewer heads; fewer where that makes less than `few` warps (a round that is not full
// costs as much as a full one: 3712 tokens of one head, 6.4 us by fours and 10.1 by twos). Then several warps share a tile, down to one round of the side
// with more heads, until there are `enough` (384 tokens of 56 and 8 heads: 139 us without, 36 so), but not more than run at once.
struct Warps {
    unsigned few, enough, most;
};
Cut cut(const RotationArgs& a, unsigned rows, unsigned fewest, unsigned most, unsigned most_tokens, const Warps& warps) {
    Cut c = {};
    const unsigned round = 32 / a.group * rows;
    c.tile = std::min({kMaxTileTokens, std::max(1u, round / fewest), a.all, most_tokens});
    while (c.tile > 1 && (a.all + c.tile - 1) / c.tile < warps.few) c.tile = (c.tile + 1) / 2;
    const unsigned tiles = (a.all + c.tile - 1) / c.tile, rounds = (c.tile * most + round - 1) / round;
    c.split = std::max(1u, std::min(rounds, tiles < warps.enough ? std::min((warps.enough + tiles - 1) / tiles, warps.most / tiles) : 1u));
    c.tiles = tiles * c.split;
    return c;
}

// Tables and heads of a CTA's warps, in 48 KiB.
constexpr std::size_t kTableBytes = 32 * 1024;
template <int V, int K, Layout kLayout>
std::size_t shared_bytes(const RotationArgs& a, const Cut& c) {
    static_assert(kTableBytes / (kLayout == Layout::Apart ? 2 : 1) + kWarps * kRowFloats<V, K, kLayout> * sizeof(float) <= 48 * 1024);
    return kWarps * (c.tile * table_entries<V, kLayout>(a) * sizeof(float4) + kRowFloats<V, K, kLayout> * sizeof(float));
}
template <int V, Layout kLayout>
unsigned most_tokens(const RotationArgs& a) {
    const std::size_t of_token = kWarps * sizeof(float4) * std::max(1u, table_entries<V, kLayout>(a));
    return (unsigned)std::max<std::size_t>(1, kTableBytes / (kLayout == Layout::Apart ? 2 : 1) / of_token);
}

template <typename T, int V, Layout kLayout>
cudaError_t forward(const RotationCall& c, RotationArgs& a) {
    constexpr int K = items_of_lane<T, V>(false), U = V == 8 || K == 1 ? 2 : 1;
    const unsigned q = a.side[0].heads.d, k = a.side[1].heads.d;
    a.cut = cut(a, U, q == 0 || k == 0 ? q + k : std::min(q, k), std::max(q, k), most_tokens<V, kLayout>(a), {kSms * 4, kSms * 16, kSms * 32});
    return launch_dependent<RotationArgs>(c.norm ? rotate_kernel<T, V, K, kLayout, true, U> : rotate_kernel<T, V, K, kLayout, false, U>,
                                          (a.cut.tiles + kWarps - 1) / kWarps, kThreads, shared_bytes<V, K, kLayout>(a, a.cut), c.stream, a);
}

template <typename T, int V, Layout kLayout>
cudaError_t backward(const RotationCall& c, RotationArgs& a) {
    constexpr int K = items_of_lane<T, V>(true), U = V == 8 ? 2 : 1;
    const dim3 columns((a.dim + 31) / 32, 2);
    if (a.all == 0) return launch_dependent<RotationArgs>(sum_kernel<T>, columns, 1024, 0, c.stream, a);  // of nothing
    const unsigned heads = a.side[0].heads.d + a.side[1].heads.d;
    bool codes = false;
    std::size_t shared = kWarps * a.dim * sizeof(float);
    for (Side& s : a.side) {
        if (s.heads.d == 0) continue;
        codes |= s.codes != nullptr;
        const unsigned ctas = std::max(1u, kHeadGradCtas * s.heads.d / heads);  // all of them run at once
        s.cut = cut(a, U, s.heads.d, s.heads.d, most_tokens<V, kLayout>(a), {ctas * kWarps / 2, ctas * kWarps, ctas * kWarps});
        s.cut.ctas = std::min((s.cut.tiles + kWarps - 1) / kWarps, ctas);
        shared = std::max(shared, shared_bytes<V, K, kLayout>(a, s.cut));
    }
    const cudaError_t st = launch_dependent<RotationArgs>(
        codes ? rotate_norm_backward_kernel<T, V, K, kLayout, true, U> : rotate_norm_backward_kernel<T, V, K, kLayout, false, U>,
        a.side[0].cut.ctas + a.side[1].cut.ctas, kThreads, shared, c.stream, a);
    if (st != cudaSuccess) return st;
    return launch_dependent<RotationArgs>(sum_kernel<T>, columns, 1024, 0, c.stream, a);
}

template <typename T, int V, Layout kLayout>
cudaError_t start(const RotationCall& c, RotationArgs& a, bool back) {
    return back ? backward<T, V, kLayout>(c, a) : forward<T, V, kLayout>(c, a);
}

template <typename T, Layout kLayout>
cudaError_t start_laid_out(const RotationCall& c, RotationArgs& a, unsigned vector, bool back) {
    if constexpr (sizeof(T) == 2)
        if (vector == 8) return start<T, 8, kLayout>(c, a, back);
    if constexpr (kLayout != Layout::Half) {
        if (vector == 2) return start<T, 2, kLayout>(c, a, back);
        if (vector == 1) return start<T, 1, kLayout>(c, a, back);
    }
    return start<T, 4, kLayout>(c, a, back);
}

template <typename T>
cudaError_t start_typed(const RotationCall& c, bool back) {
    const Shape shape = shape_of<T>(c, back);
    RotationArgs a = args_of(c, shape, sizeof(T));
    switch (shape.layout) {
        case Layout::Half: return start_laid_out<T, Layout::Half>(c, a, shape.vector, back);
        case Layout::Interleaved: return start_laid_out<T, Layout::Interleaved>(c, a, shape.vector, back);
        case Layout::Apart: return start_laid_out<T, Layout::Apart>(c, a, shape.vector, back);
    }
    return cudaErrorInvalidValue;
}

cudaError_t start_any(const RotationCall& c, bool back) {
    switch (c.dtype) {
        case DType::Float: return start_typed<float>(c, back);
        case DType::Float16: return start_typed<__half>(c, back);
        case DType::BFloat16: return start_typed<__nv_bfloat16>(c, back);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_rotate_heads(const RotationCall& call) {
    if (call.batch == 0 || call.tokens == 0) return cudaSuccess;
    return start_any(call, false);
}

cudaError_t launch_rotate_heads_backward(const RotationCall& call) { return start_any(call, true); }

}  // namespace b200ccl::kernels
