// Queries and keys turned by their positions, alone or in the same pass as the norm of each head, and the gradients.
//
// A head is `dim` numbers; of its first `rotated` ones every pair (u, v) becomes magnitude * (u cos - v sin, u sin + v cos), angle =
// position * frequency of the pair. With the norm, the pair is first n = x * rstd * w, rstd = (mean x^2 + eps)^-1/2 over the head. The
// gradient of a rotation is the rotation back: g = R^T dy; of the norm, dw = sum g x rstd, dx = rstd (g w - x rstd^2 mean(g w x)).
//
// Bound by HBM: every head is read once and written once. Angles are made where they are used: position * frequency as
// turns in 64 bits, less its whole turns, then one sincospi in 32 bits (error 2e-7 at any position; in 32 bits the product alone is off by
// 0.06 at a million). A warp makes them once for its tokens, in shared memory of its own, and all heads of a token, of queries and
// keys, share them. Warps meet nowhere but at the end of the backward pass.
//
// A group of lanes holds a head: each lane V pairs at V neighbouring places of either half (interleaved: 2V neighbouring elements), so
// both elements of a pair are in one lane and no exchange is needed but the sums over a head. Elements that do not turn are
// pairs with no angle. V = 8 (two 16-byte accesses of 16-bit types), 4 or 1, as sizes and addresses allow.
//
// The inputs of the norm are kept for the backward pass in 8 bits, a head being a block (block8.cuh): the largest magnitude comes from
// the same exchange as the sum of squares.
#include "kernels/sm100/head_rotation.h"

#include "kernels/sm100/block8.cuh"
#include "kernels/sm100/launch.h"

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
constexpr u64 kSms = 148;

struct View {
    const char* data;
    i64 batch, token, head;  // bytes
};

// n / d for n below 2^31, as a product.
struct Divisor {
    unsigned d, factor, shift;
    __device__ __forceinline__ unsigned divide(unsigned n) const { return (unsigned)(((u64)n * factor) >> shift); }
};
Divisor divisor_of(unsigned d) {
    unsigned bits = 0;
    while ((1ull << bits) < d) ++bits;
    return {d, (unsigned)((1ull << (31 + bits)) / d + 1), 31 + bits};
}

struct Side {
    View x, grad;
    char* out;
    const char* weight;
    unsigned char* codes;
    unsigned char* scales;
    char* weight_grad;
    float* partial;
    Divisor heads;  // d = 0: none
};

struct RotationArgs {
    Side side[2];
    const char* positions;
    i64 position_batch, position_token;  // elements
    const double* frequencies;
    unsigned all;     // tokens of all sequences
    Divisor tokens;   // of one
    unsigned dim, rotated, pitch;
    unsigned items;  // lanes' worth of pairs in a head
    unsigned group;  // lanes that hold a head, a power of two
    unsigned tile;   // tokens of a warp's tile
    unsigned split;  // warps that share a tile, each for some of its heads
    unsigned tiles;  // times split
    unsigned ctas;
    float magnitude, sine;  // what cosines and sines are multiplied with
    float eps;
    bool positions64;
};

// V neighbouring elements of T, as they lie in memory.
template <typename T, int V>
struct Some {
    static constexpr int kBytes = V * sizeof(T);
    using Word = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, T>>;
    static_assert(kBytes == 16 || kBytes == 8 || V == 1);
    Word w;
    __device__ __forceinline__ void clear() { w = Word(); }
    __device__ __forceinline__ void load(const char* p) {
        if constexpr (kBytes == 16) w = ld16_stream(reinterpret_cast<const uint4*>(p));
        else w = *reinterpret_cast<const Word*>(p);
    }
    __device__ __forceinline__ void widen(float (&f)[V]) const {
        if constexpr (kBytes == 16) {
            Wide<T>::unpack(w, f);
        } else if constexpr (V > 1) {
            const float2 a = std::is_same_v<T, __half> ? h2_to_f2(w.x) : b2_to_f2(w.x), b = std::is_same_v<T, __half> ? h2_to_f2(w.y) : b2_to_f2(w.y);
            f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
        } else {
            f[0] = Elem<T>::to_f(w);
        }
    }
    static __device__ __forceinline__ void store(char* p, const float (&f)[V]) {
        if constexpr (kBytes == 16) {
            st16(reinterpret_cast<uint4*>(p), Wide<T>::pack(f));
        } else if constexpr (V > 1) {
            uint2 w;
            if constexpr (std::is_same_v<T, __half>) { w.x = f2_to_h2(f[0], f[1]); w.y = f2_to_h2(f[2], f[3]); }
            else { w.x = f2_to_b2(f[0], f[1]); w.y = f2_to_b2(f[2], f[3]); }
            *reinterpret_cast<uint2*>(p) = w;
        } else {
            *reinterpret_cast<T*>(p) = Elem<T>::from_f(f[0]);
        }
    }
};
// V neighbouring codes.
template <int V>
struct Codes {
    using Word = std::conditional_t<V == 8, uint2, std::conditional_t<V == 4, unsigned, unsigned char>>;
    Word w;
    __device__ __forceinline__ void clear() { w = Word(); }
    __device__ __forceinline__ void load(const unsigned char* p) { w = *reinterpret_cast<const Word*>(p); }
    __device__ __forceinline__ void widen(float step, float (&f)[V]) const {
        if constexpr (V == 8) {
            decode8x4(w.x, step, f);
            decode8x4(w.y, step, f + 4);
        } else if constexpr (V == 4) {
            decode8x4(w, step, f);
        } else {
            f[0] = decode8<0>(w, step);
        }
    }
};
template <int V>
__device__ __forceinline__ void store_codes(unsigned char* p, unsigned scale, const float (&f)[V]) {
    const float inverse = inverse_step8(scale);
    if constexpr (V == 8) {
        *reinterpret_cast<uint2*>(p) = make_uint2(finite8(encode8x4(f, inverse), scale), finite8(encode8x4(f + 4, inverse), scale));
    } else if constexpr (V == 4) {
        *reinterpret_cast<unsigned*>(p) = finite8(encode8x4(f, inverse), scale);
    } else {
        *p = (unsigned char)finite8(encode8(f[0], inverse), scale);
    }
}

// Where a lane's pairs lie in a head: first elements at `first`, second ones at `second` (interleaved: from `first` on, in turn).
struct Place {
    unsigned pair, first, second;
};
template <int V, bool kInterleaved>
__device__ __forceinline__ Place place_of(const RotationArgs& a, unsigned item) {
    const unsigned p = item * V, turning = a.rotated / 2;
    if (kInterleaved) return {p, 2 * p, 2 * p + V};
    if (p < turning) return {p, p, p + turning};
    const unsigned first = a.rotated + (p - turning);
    return {p, first, first + (a.dim - a.rotated) / 2};
}

// u[i], v[i]: the elements of pair i. Interleaved ones arrive as u0 v0 u1 v1 ...
template <int V>
__device__ __forceinline__ void part(float (&u)[V], float (&v)[V]) {
    float f[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) { f[i] = u[i]; f[V + i] = v[i]; }
#pragma unroll
    for (int i = 0; i < V; ++i) { u[i] = f[2 * i]; v[i] = f[2 * i + 1]; }
}
template <int V>
__device__ __forceinline__ void join(float (&u)[V], float (&v)[V]) {
    float f[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) { f[2 * i] = u[i]; f[2 * i + 1] = v[i]; }
#pragma unroll
    for (int i = 0; i < V; ++i) { u[i] = f[i]; v[i] = f[V + i]; }
}
template <typename T, int V, bool kInterleaved>
__device__ __forceinline__ void load_pairs(const char* head, const Place& at, float (&u)[V], float (&v)[V]) {
    Some<T, V> a, b;
    a.load(head + at.first * sizeof(T));
    b.load(head + at.second * sizeof(T));
    a.widen(u);
    b.widen(v);
    if constexpr (kInterleaved && V > 1) part(u, v);
}
template <typename T, int V, bool kInterleaved>
__device__ __forceinline__ void store_pairs(char* head, const Place& at, float (&u)[V], float (&v)[V]) {
    if constexpr (kInterleaved && V > 1) join(u, v);
    Some<T, V>::store(head + at.first * sizeof(T), u);
    Some<T, V>::store(head + at.second * sizeof(T), v);
}

__device__ __forceinline__ float group_sum(float v, unsigned group) {
    for (unsigned o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ unsigned group_max(unsigned v, unsigned group) {
    for (unsigned o = group >> 1; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// A warp's share of the work: some tokens, and of their heads one part in `split`.
struct Tile {
    unsigned token, tokens, part;
};
__device__ __forceinline__ Tile tile_at(const RotationArgs& a, unsigned index) {
    const unsigned t = a.split == 1u ? index : index / a.split;
    return {t * a.tile, min(a.tile, a.all - t * a.tile), index - t * a.split};
}
// Its rows (heads of tokens, in order) of one side.
struct Rows {
    unsigned from, to;
};
__device__ __forceinline__ Rows rows_of(const RotationArgs& a, const Side& s, const Tile& t) {
    const unsigned rows = t.tokens * s.heads.d;
    if (a.split == 1u) return {0u, rows};
    const unsigned each = (rows + a.split - 1u) / a.split;
    return {min(rows, t.part * each), min(rows, (t.part + 1u) * each)};
}

// Cosine and sine of every pair of a tile's tokens, in a warp's own shared memory: pair item * V + i of token t at (t * V + i) * turning items
// + item, so that neighbouring lanes read neighbouring words.
template <int V>
__device__ __forceinline__ void make_table(const RotationArgs& a, const Tile& tile, float2* table) {
    const unsigned pairs = a.rotated / 2, items = pairs / V, lane = threadIdx.x & 31u;
    for (unsigned t = 0; t < tile.tokens; ++t) {
        const unsigned n = tile.token + t, b = a.tokens.divide(n);
        const i64 at = (i64)b * a.position_batch + (i64)(n - b * a.tokens.d) * a.position_token;
        const double position = a.positions64 ? (double)*(reinterpret_cast<const i64*>(a.positions) + at)
                                              : (double)*(reinterpret_cast<const int*>(a.positions) + at);
        for (unsigned p = lane; p < pairs; p += 32u) {
            double turns = position * (a.frequencies[p] * 0.15915494309189535);  // 1 / (2 pi)
            turns -= rint(turns);
            float sine, cosine;
            sincospif((float)(2.0 * turns), &sine, &cosine);
            table[t * pairs + (p % V) * items + p / V] = make_float2(a.magnitude * cosine, a.sine * sine);
        }
    }
}

template <int V>
__device__ __forceinline__ void turn(const float2* angles, const Place& at, unsigned pairs, float (&u)[V], float (&v)[V]) {
    if (at.pair >= pairs) return;
    const unsigned items = pairs / V, item = at.pair / V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 cs = angles[i * items + item];
        const float x = u[i], y = v[i];
        u[i] = fmaf(x, cs.x, -y * cs.y);
        v[i] = fmaf(x, cs.y, y * cs.x);
    }
}

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

// K: items of a lane. U: rows of a group in flight.
template <typename T, int V, int K, bool kInterleaved, bool kNorm, int U>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const __grid_constant__ RotationArgs a) {
    extern __shared__ __align__(16) unsigned char shared[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned warp = threadIdx.x / 32u, index = blockIdx.x * kWarps + warp;
    if (index >= a.tiles) return;
    const Tile tile = tile_at(a, index);
    const unsigned pairs = a.rotated / 2, lane = threadIdx.x & (a.group - 1u), groups = 32u / a.group, group = (threadIdx.x & 31u) / a.group;
    float2* table = reinterpret_cast<float2*>(shared) + warp * a.tile * pairs;
    Place at[K];
    bool mine[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned item = lane + k * 32u;
        mine[k] = item < a.items;
        at[k] = place_of<V, kInterleaved>(a, mine[k] ? item : 0u);
    }
    bool made = false;
    for (int i = 0; i < 2; ++i) {
        const Side& s = a.side[i];
        if (s.heads.d == 0u) continue;
        const Rows rows = rows_of(a, s, tile);
        float wu[kNorm ? K : 1][V], wv[kNorm ? K : 1][V];
        if constexpr (kNorm) {
#pragma unroll
            for (int k = 0; k < K; ++k) load_pairs<T, V, kInterleaved>(s.weight, at[k], wu[k], wv[k]);
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
                make_table<V>(a, tile, table);
                __syncwarp();
                made = true;
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                float u[K][V], v[K][V];
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    first[j][k].widen(u[k]);
                    second[j][k].widen(v[k]);
                }
                const u64 r = (u64)row[j].n * s.heads.d + row[j].h;
                if constexpr (kNorm) {
                    float squares = 0.0f;
                    unsigned amax = 0;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            squares = fmaf(u[k][e], u[k][e], fmaf(v[k][e], v[k][e], squares));
                            amax = max(amax, max(magnitude_bits(u[k][e]), magnitude_bits(v[k][e])));
                        }
                    }
                    if (s.codes != nullptr) {
                        const unsigned scale = scale8<T>(group_max(amax, a.group));
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            if (row[j].there && mine[k]) {
                                store_codes<V>(s.codes + r * a.pitch + at[k].first, scale, u[k]);
                                store_codes<V>(s.codes + r * a.pitch + at[k].second, scale, v[k]);
                            }
                        }
                        if (row[j].there && lane == 0) s.scales[r] = (unsigned char)scale;
                    }
                    const float rstd = rsqrtf(group_sum(squares, a.group) / (float)a.dim + a.eps);
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        if constexpr (kInterleaved && V > 1) part(u[k], v[k]);
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            u[k][e] *= rstd * wu[k][e];
                            v[k][e] *= rstd * wv[k][e];
                        }
                    }
                } else if constexpr (kInterleaved && V > 1) {
#pragma unroll
                    for (int k = 0; k < K; ++k) part(u[k], v[k]);
                }
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (row[j].there && mine[k]) {
                        turn(table + row[j].token * pairs, at[k], pairs, u[k], v[k]);
                        store_pairs<T, V, kInterleaved>(s.out + r * a.dim * sizeof(T), at[k], u[k], v[k]);
                    }
                }
            }
        }
    }
}

// One side of a tile in the backward pass: gradients of the inputs, and this lane's share of the weight's.
template <typename T, int V, int K, bool kInterleaved, bool kCodes, int U>
__device__ __forceinline__ void backward_side(const RotationArgs& a, const Side& s, const Tile& tile, const Place (&at)[K], const bool (&mine)[K],
                                              float2* table, bool* made, float (&du)[K][V], float (&dv)[K][V]) {
    const unsigned pairs = a.rotated / 2, groups = 32u / a.group, group = (threadIdx.x & 31u) / a.group;
    const Rows rows = rows_of(a, s, tile);
    float wu[K][V], wv[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) load_pairs<T, V, kInterleaved>(s.weight, at[k], wu[k], wv[k]);
    for (unsigned r0 = rows.from; r0 < rows.to; r0 += groups * U) {
        Some<T, V> g1[U][K], g2[U][K];
        std::conditional_t<kCodes, Codes<V>, Some<T, V>> x1[U][K], x2[U][K];
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
        if (!*made) {
            __syncwarp();  // the table of the tile before has been read
            make_table<V>(a, tile, table);
            __syncwarp();
            *made = true;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float gu[K][V], gv[K][V], u[K][V], v[K][V];
            float squares = 0.0f, dot = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                g1[j][k].widen(gu[k]);
                g2[j][k].widen(gv[k]);
                if constexpr (kCodes) {
                    const float step = step8(scale[j]);
                    x1[j][k].widen(step, u[k]);
                    x2[j][k].widen(step, v[k]);
                } else {
                    x1[j][k].widen(u[k]);
                    x2[j][k].widen(v[k]);
                }
                if constexpr (kInterleaved && V > 1) {
                    part(gu[k], gv[k]);
                    part(u[k], v[k]);
                }
                if (!mine[k]) {  // (its codes are zeros, but zero times the step of a head that is not finite is not)
#pragma unroll
                    for (int e = 0; e < V; ++e) u[k][e] = v[k][e] = 0.0f;
                }
                turn(table + row[j].token * pairs, at[k], pairs, gu[k], gv[k]);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    squares = fmaf(u[k][e], u[k][e], fmaf(v[k][e], v[k][e], squares));
                    dot = fmaf(gu[k][e] * wu[k][e], u[k][e], fmaf(gv[k][e] * wv[k][e], v[k][e], dot));
                }
            }
            squares = group_sum(squares, a.group);
            dot = group_sum(dot, a.group);
            if (!row[j].there) continue;
            const float rstd = rsqrtf(squares / (float)a.dim + a.eps);
            const float back = dot / (float)a.dim * rstd * rstd;
            const u64 r = (u64)row[j].n * s.heads.d + row[j].h;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    du[k][e] = fmaf(gu[k][e] * rstd, u[k][e], du[k][e]);
                    dv[k][e] = fmaf(gv[k][e] * rstd, v[k][e], dv[k][e]);
                    u[k][e] = rstd * fmaf(-u[k][e], back, gu[k][e] * wu[k][e]);
                    v[k][e] = rstd * fmaf(-v[k][e], back, gv[k][e] * wv[k][e]);
                }
                if (mine[k]) store_pairs<T, V, kInterleaved>(s.out + r * a.dim * sizeof(T), at[k], u[k], v[k]);
            }
        }
        __syncwarp();
    }
}

// Gradients of the norm and rotation. A warp takes tile after tile, so that its share of the weights' gradients stays in registers; the shares
// of a CTA go to `partial` and sum_kernel adds them in order, so that results do not depend on which CTA ends first.
template <typename T, int V, int K, bool kInterleaved, bool kCodes, int U>
__global__ void __launch_bounds__(kThreads, 2) rotate_norm_backward_kernel(const __grid_constant__ RotationArgs a) {
    extern __shared__ __align__(16) unsigned char shared[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned warp = threadIdx.x / 32u, in_warp = threadIdx.x & 31u, lane = threadIdx.x & (a.group - 1u);
    float2* table = reinterpret_cast<float2*>(shared) + warp * a.tile * (a.rotated / 2);
    Place at[K];
    bool mine[K];
    float du[2][K][V], dv[2][K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned item = lane + k * 32u;
        mine[k] = item < a.items;
        at[k] = place_of<V, kInterleaved>(a, mine[k] ? item : 0u);
#pragma unroll
        for (int i = 0; i < V; ++i) du[0][k][i] = dv[0][k][i] = du[1][k][i] = dv[1][k][i] = 0.0f;
    }
    for (unsigned index = blockIdx.x * kWarps + warp; index < a.tiles; index += a.ctas * kWarps) {
        const Tile tile = tile_at(a, index);
        bool made = false;
        if (a.side[0].heads.d != 0u)
            backward_side<T, V, K, kInterleaved, kCodes, U>(a, a.side[0], tile, at, mine, table, &made, du[0], dv[0]);
        if (a.side[1].heads.d != 0u)
            backward_side<T, V, K, kInterleaved, kCodes, U>(a, a.side[1], tile, at, mine, table, &made, du[1], dv[1]);
    }
    // The groups of a warp, then the warps.
    __syncthreads();
    float* sums = reinterpret_cast<float*>(shared);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const Side& s = a.side[side];
        if (s.heads.d == 0u) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                for (unsigned o = a.group; o < 32u; o <<= 1) {
                    du[side][k][i] += __shfl_xor_sync(0xffffffffu, du[side][k][i], o);
                    dv[side][k][i] += __shfl_xor_sync(0xffffffffu, dv[side][k][i], o);
                }
                if (in_warp < a.group && mine[k]) {
                    sums[warp * a.dim + (kInterleaved ? at[k].first + 2 * i : at[k].first + i)] = du[side][k][i];
                    sums[warp * a.dim + (kInterleaved ? at[k].first + 2 * i + 1 : at[k].second + i)] = dv[side][k][i];
                }
            }
        }
        __syncthreads();
        for (unsigned d = threadIdx.x; d < a.dim; d += kThreads) {
            float sum = 0.0f;
            for (unsigned w = 0; w < kWarps; ++w) sum += sums[w * a.dim + d];
            s.partial[(u64)blockIdx.x * a.dim + d] = sum;
        }
        __syncthreads();
    }
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
    float sum = 0.0f;
    if (column < a.dim)
        for (unsigned c = part; c < a.ctas; c += 32u) sum += s.partial[(u64)c * a.dim + column];
    sums[part][threadIdx.x & 31u] = sum;
    __syncthreads();
    sum = sums[threadIdx.x & 31u][part];  // warp `part` adds column `part`
    for (unsigned o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const unsigned d = blockIdx.x * 32u + part;
    if ((threadIdx.x & 31u) == 0 && d < a.dim) reinterpret_cast<T*>(s.weight_grad)[d] = Elem<T>::from_f(sum);
}

struct Shape {
    unsigned vector, items, group;
};

View view_of(const HeadsView& v, long long bytes) {
    return {static_cast<const char*>(v.data), v.batch * bytes, v.token * bytes, v.head * bytes};
}

// Whether V elements of every head that is touched are one access.
bool fits(const RotationCall& c, unsigned v, unsigned bytes) {
    const unsigned turning = c.rotated / 2, rest = (c.dim - c.rotated) / 2;
    if (turning % v != 0 || rest % v != 0) return false;
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
Shape shape_of(const RotationCall& c) {
    const unsigned widest = 16 / sizeof(T);
    Shape s;
    s.vector = fits(c, widest, sizeof(T)) ? widest : (widest > 4 && fits(c, 4, sizeof(T)) ? 4 : 1);
    s.items = (unsigned)c.dim / 2 / s.vector;
    s.group = 1;
    while (s.group < s.items && s.group < 32) s.group *= 2;
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
    a.tokens = divisor_of((unsigned)std::max(1ll, c.tokens));
    a.dim = (unsigned)c.dim;
    a.rotated = (unsigned)c.rotated;
    a.pitch = (a.dim + 15u) / 16u * 16u;
    a.items = shape.items;
    a.group = shape.group;
    a.magnitude = c.magnitude;
    a.sine = c.inverse ? -c.magnitude : c.magnitude;
    a.eps = c.eps;
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
        if (s.heads != 0) t.heads = divisor_of((unsigned)s.heads);
    }
    return a;
}

// A warp's tile: as many tokens as give it `passes` rounds of rows of the side with fewer heads. Where that makes too few warps for the device, several
// share a tile, down to one round of the side with more heads.
void cut(RotationArgs& a, unsigned passes, u64 warps) {
    unsigned fewest = 0, most = 0;
    for (const Side& s : a.side) {
        if (s.heads.d == 0) continue;
        fewest = fewest == 0 ? s.heads.d : std::min(fewest, s.heads.d);
        most = std::max(most, s.heads.d);
    }
    const unsigned round = 32 / a.group * passes;
    a.tile = std::min({kMaxTileTokens, std::max(1u, round / fewest), a.all});
    while (a.tile > 1 && (a.all + a.tile - 1) / a.tile < warps) a.tile = (a.tile + 1) / 2;
    const unsigned tiles = (a.all + a.tile - 1) / a.tile, rounds = (a.tile * most + round - 1) / round;
    a.split = (unsigned)std::max<u64>(1, std::min<u64>(rounds, warps / tiles));
    a.tiles = tiles * a.split;
}

std::size_t table_bytes(const RotationArgs& a) { return (std::size_t)kWarps * a.tile * (a.rotated / 2) * sizeof(float2); }

template <typename T, int V, int K, bool kInterleaved>
cudaError_t forward(const RotationCall& c, RotationArgs& a) {
    constexpr int U = 2;
    cut(a, U, kSms * 4);
    return launch_dependent<RotationArgs>(c.norm ? rotate_kernel<T, V, K, kInterleaved, true, U> : rotate_kernel<T, V, K, kInterleaved, false, U>,
                                          (a.tiles + kWarps - 1) / kWarps, kThreads, table_bytes(a), c.stream, a);
}

template <typename T, int V, int K, bool kInterleaved>
cudaError_t backward(const RotationCall& c, RotationArgs& a) {
    constexpr int U = 1;
    const dim3 columns((a.dim + 31) / 32, 2);
    if (a.all == 0) return launch_dependent<RotationArgs>(sum_kernel<T>, columns, 1024, 0, c.stream, a);  // of nothing
    cut(a, U, kSms * 4);
    a.ctas = std::min(kHeadGradCtas, (a.tiles + kWarps - 1) / kWarps);
    bool codes = false;
    for (const Side& s : a.side) codes |= s.codes != nullptr;
    const std::size_t shared = std::max<std::size_t>(table_bytes(a), kWarps * a.dim * sizeof(float));
    const cudaError_t st = launch_dependent<RotationArgs>(
        codes ? rotate_norm_backward_kernel<T, V, K, kInterleaved, true, U> : rotate_norm_backward_kernel<T, V, K, kInterleaved, false, U>,
        a.ctas, kThreads, shared, c.stream, a);
    if (st != cudaSuccess) return st;
    return launch_dependent<RotationArgs>(sum_kernel<T>, columns, 1024, 0, c.stream, a);
}

template <typename T, int V, int K>
cudaError_t start(const RotationCall& c, RotationArgs& a, bool back) {
    if (back) return c.interleaved ? backward<T, V, K, true>(c, a) : backward<T, V, K, false>(c, a);
    return c.interleaved ? forward<T, V, K, true>(c, a) : forward<T, V, K, false>(c, a);
}

template <typename T>
cudaError_t start_typed(const RotationCall& c, bool back) {
    const Shape shape = shape_of<T>(c);
    RotationArgs a = args_of(c, shape, sizeof(T));
    if constexpr (sizeof(T) == 2)
        if (shape.vector == 8) return start<T, 8, 1>(c, a, back);
    if (shape.vector == 4) return start<T, 4, 1>(c, a, back);
    return shape.items > 32 ? start<T, 1, 4>(c, a, back) : start<T, 1, 1>(c, a, back);
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
