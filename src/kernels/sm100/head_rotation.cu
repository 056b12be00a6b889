// Queries and keys turned by their positions, alone or in the same pass as the norm of each head, and the gradients.
//
// A head is `dim` numbers; of its first `rotated` ones every pair (u, v) becomes magnitude * (u cos - v sin, u sin + v cos), angle =
// position * frequency of the pair. With the norm, the pair is first n = x * rstd * w, rstd = (mean x^2 + eps)^-1/2 over the head. The
// gradient of a rotation is the rotation back: g = R^T dy; of the norm, dw = sum g x rstd, dx = rstd (g w - x rstd^2 mean(g w x)).
//
// Bound by HBM: every head is read once and written once. Angles are made where they are used: position * frequency as
// turns in 64 bits, less its whole turns, then one sincospi in 32 bits (error 2e-7 at any position; in 32 bits the product alone is off by
// 0.06 at a million). A CTA makes them once for its tokens, in shared memory, and all heads of a token share them.
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

namespace b200ccl::kernels {

using namespace b200ccl::dev;

namespace {

using u64 = unsigned long long;
using i64 = long long;

constexpr unsigned kThreads = 256;
constexpr unsigned kWarps = kThreads / 32;

struct View {
    const char* data;
    i64 batch, token, head;  // bytes
};

struct Side {
    View x, grad;
    char* out;
    const char* weight;
    unsigned char* codes;
    unsigned char* scales;
    char* weight_grad;
    float* partial;
    unsigned heads;
    unsigned tile;   // tokens of a tile
    unsigned tiles;
    unsigned ctas;
};

struct RotationArgs {
    Side side[2];
    const char* positions;
    i64 position_batch, position_token;  // elements
    const double* frequencies;
    u64 all;  // tokens of all sequences
    u64 tokens;
    unsigned dim, rotated, pitch;
    unsigned items;  // lanes' worth of pairs in a head
    unsigned group;  // lanes that hold a head, a power of two
    float magnitude, sine;  // what cosines and sines are multiplied with
    float eps;
    bool positions64;
};

// V neighbouring elements of T.
template <typename T, int V>
__device__ __forceinline__ void load_some(const char* p, float (&f)[V]) {
    if constexpr (V * sizeof(T) == 16) {
        Wide<T>::unpack(ld16_stream(reinterpret_cast<const uint4*>(p)), f);
    } else if constexpr (V * sizeof(T) == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        float2 a, b;
        if constexpr (sizeof(T) == 2) {
            if constexpr (std::is_same_v<T, __half>) { a = h2_to_f2(w.x); b = h2_to_f2(w.y); }
            else { a = b2_to_f2(w.x); b = b2_to_f2(w.y); }
            f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
        }
    } else {
        static_assert(V == 1);
        f[0] = Elem<T>::to_f(*reinterpret_cast<const T*>(p));
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_some(char* p, const float (&f)[V]) {
    if constexpr (V * sizeof(T) == 16) {
        st16(reinterpret_cast<uint4*>(p), Wide<T>::pack(f));
    } else if constexpr (V * sizeof(T) == 8) {
        uint2 w;
        if constexpr (std::is_same_v<T, __half>) { w.x = f2_to_h2(f[0], f[1]); w.y = f2_to_h2(f[2], f[3]); }
        else { w.x = f2_to_b2(f[0], f[1]); w.y = f2_to_b2(f[2], f[3]); }
        *reinterpret_cast<uint2*>(p) = w;
    } else {
        static_assert(V == 1);
        *reinterpret_cast<T*>(p) = Elem<T>::from_f(f[0]);
    }
}
// V neighbouring codes.
template <int V>
__device__ __forceinline__ void load_codes(const unsigned char* p, float step, float (&f)[V]) {
    if constexpr (V == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        decode8x4(w.x, step, f);
        decode8x4(w.y, step, f + 4);
    } else if constexpr (V == 4) {
        decode8x4(*reinterpret_cast<const unsigned*>(p), step, f);
    } else {
        f[0] = decode8<0>(*p, step);
    }
}
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
    load_some<T, V>(head + at.first * sizeof(T), u);
    load_some<T, V>(head + at.second * sizeof(T), v);
    if constexpr (kInterleaved && V > 1) part(u, v);
}
template <typename T, int V, bool kInterleaved>
__device__ __forceinline__ void store_pairs(char* head, const Place& at, float (&u)[V], float (&v)[V]) {
    if constexpr (kInterleaved && V > 1) join(u, v);
    store_some<T, V>(head + at.first * sizeof(T), u);
    store_some<T, V>(head + at.second * sizeof(T), v);
}

__device__ __forceinline__ float group_sum(float v, unsigned group) {
    for (unsigned o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ unsigned group_max(unsigned v, unsigned group) {
    for (unsigned o = group >> 1; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Cosine and sine of every pair of a tile's tokens, and the place of each token's first head in x and grad (bytes).
__device__ __forceinline__ void make_table(const RotationArgs& a, const Side& s, u64 token0, unsigned tokens, float2* table, i64* x_at,
                                           i64* grad_at) {
    const unsigned pairs = a.rotated / 2;
    for (unsigned i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const unsigned t = i / pairs, p = i - t * pairs;
        const u64 n = token0 + t, b = n / a.tokens;
        const i64 at = (i64)b * a.position_batch + (i64)(n - b * a.tokens) * a.position_token;
        const double position = a.positions64 ? (double)*(reinterpret_cast<const i64*>(a.positions) + at)
                                              : (double)*(reinterpret_cast<const int*>(a.positions) + at);
        double turns = position * (a.frequencies[p] * 0.15915494309189535);  // 1 / (2 pi)
        turns -= rint(turns);
        float sine, cosine;
        sincospif((float)(2.0 * turns), &sine, &cosine);
        table[i] = make_float2(a.magnitude * cosine, a.sine * sine);
    }
    for (unsigned t = threadIdx.x; t < tokens; t += kThreads) {
        const u64 n = token0 + t, b = n / a.tokens;
        const i64 in = (i64)(n - b * a.tokens);
        x_at[t] = (i64)b * s.x.batch + in * s.x.token;
        grad_at[t] = (i64)b * s.grad.batch + in * s.grad.token;
    }
}

template <int V>
__device__ __forceinline__ void turn(const float2* angles, const Place& at, unsigned pairs, float (&u)[V], float (&v)[V]) {
    if (at.pair >= pairs) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 cs = angles[at.pair + i];
        const float x = u[i], y = v[i];
        u[i] = fmaf(x, cs.x, -y * cs.y);
        v[i] = fmaf(x, cs.y, y * cs.x);
    }
}

// K: items of a lane.
template <typename T, int V, int K, bool kInterleaved, bool kNorm, int U>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const __grid_constant__ RotationArgs a) {
    extern __shared__ __align__(16) unsigned char shared[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool second = blockIdx.x >= a.side[0].ctas;
    const Side& s = a.side[second ? 1 : 0];
    const unsigned tile = blockIdx.x - (second ? a.side[0].ctas : 0u);
    const u64 token0 = (u64)tile * s.tile;
    const unsigned tokens = (unsigned)min((u64)s.tile, a.all - token0);
    i64* x_at = reinterpret_cast<i64*>(shared);
    i64* grad_at = x_at + s.tile;
    float2* table = reinterpret_cast<float2*>(grad_at + s.tile);
    make_table(a, s, token0, tokens, table, x_at, grad_at);
    __syncthreads();
    const unsigned lane = threadIdx.x & (a.group - 1u), pairs = a.rotated / 2;
    Place at[K];
    bool mine[K];
    float wu[kNorm ? K : 1][V], wv[kNorm ? K : 1][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned item = lane + k * 32u;
        mine[k] = item < a.items;
        at[k] = place_of<V, kInterleaved>(a, mine[k] ? item : 0u);
        if constexpr (kNorm) load_pairs<T, V, kInterleaved>(s.weight, at[k], wu[k], wv[k]);
    }
    const unsigned rows = tokens * s.heads, step = kThreads / a.group;
    // (All lanes of a warp stay to the end of a pass: they exchange sums.)
    for (unsigned r0 = 0; r0 < rows; r0 += step * U) {
        float u[U][K][V], v[U][K][V];
        unsigned token[U];
        bool there[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const unsigned r = r0 + j * step + threadIdx.x / a.group;
            there[j] = r < rows;
            token[j] = there[j] ? r / s.heads : 0u;
            const char* head = s.x.data + x_at[token[j]] + (i64)(there[j] ? r - token[j] * s.heads : 0u) * s.x.head;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (there[j] && mine[k]) {
                    load_pairs<T, V, kInterleaved>(head, at[k], u[j][k], v[j][k]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) u[j][k][i] = v[j][k][i] = 0.0f;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const unsigned r = r0 + j * step + threadIdx.x / a.group;
            const u64 row = token0 * s.heads + r;
            if constexpr (kNorm) {
                float squares = 0.0f;
                unsigned amax = 0;
#pragma unroll
                for (int k = 0; k < K; ++k) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        squares = fmaf(u[j][k][i], u[j][k][i], fmaf(v[j][k][i], v[j][k][i], squares));
                        amax = max(amax, max(magnitude_bits(u[j][k][i]), magnitude_bits(v[j][k][i])));
                    }
                }
                if (s.codes != nullptr) {
                    const unsigned scale = scale8<T>(group_max(amax, a.group));
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        if (there[j] && mine[k]) {
                            float c[V], d[V];
#pragma unroll
                            for (int i = 0; i < V; ++i) { c[i] = u[j][k][i]; d[i] = v[j][k][i]; }
                            if constexpr (kInterleaved && V > 1) join(c, d);
                            store_codes<V>(s.codes + row * a.pitch + at[k].first, scale, c);
                            store_codes<V>(s.codes + row * a.pitch + at[k].second, scale, d);
                        }
                    }
                    if (there[j] && lane == 0) s.scales[row] = (unsigned char)scale;
                }
                const float rstd = rsqrtf(group_sum(squares, a.group) / (float)a.dim + a.eps);
#pragma unroll
                for (int k = 0; k < K; ++k) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        u[j][k][i] *= rstd * wu[k][i];
                        v[j][k][i] *= rstd * wv[k][i];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (there[j] && mine[k]) {
                    turn(table + token[j] * pairs, at[k], pairs, u[j][k], v[j][k]);
                    store_pairs<T, V, kInterleaved>(s.out + row * a.dim * sizeof(T), at[k], u[j][k], v[j][k]);
                }
            }
        }
    }
}

// Gradients of the norm and rotation. A CTA takes tile after tile, so that its share of the weight's gradient stays in registers; the shares go to
// `partial` and sum_kernel adds them in order, so that results do not depend on which CTA ends first.
template <typename T, int V, int K, bool kInterleaved, bool kCodes>
__global__ void __launch_bounds__(kThreads) rotate_norm_backward_kernel(const __grid_constant__ RotationArgs a) {
    extern __shared__ __align__(16) unsigned char shared[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool second = blockIdx.x >= a.side[0].ctas;
    const Side& s = a.side[second ? 1 : 0];
    const unsigned cta = blockIdx.x - (second ? a.side[0].ctas : 0u);
    i64* x_at = reinterpret_cast<i64*>(shared);
    i64* grad_at = x_at + s.tile;
    float2* table = reinterpret_cast<float2*>(grad_at + s.tile);
    const unsigned lane = threadIdx.x & (a.group - 1u), pairs = a.rotated / 2;
    const unsigned step = kThreads / a.group;
    Place at[K];
    bool mine[K];
    float wu[K][V], wv[K][V], du[K][V], dv[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const unsigned item = lane + k * 32u;
        mine[k] = item < a.items;
        at[k] = place_of<V, kInterleaved>(a, mine[k] ? item : 0u);
        load_pairs<T, V, kInterleaved>(s.weight, at[k], wu[k], wv[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) du[k][i] = dv[k][i] = 0.0f;
    }
    for (unsigned tile = cta; tile < s.tiles; tile += s.ctas) {
        const u64 token0 = (u64)tile * s.tile;
        const unsigned tokens = (unsigned)min((u64)s.tile, a.all - token0);
        __syncthreads();  // the table of the tile before has been read
        make_table(a, s, token0, tokens, table, x_at, grad_at);
        __syncthreads();
        const unsigned rows = tokens * s.heads;
        for (unsigned r0 = 0; r0 < rows; r0 += step) {
            const unsigned r = r0 + threadIdx.x / a.group;
            const bool there = r < rows;
            const unsigned token = there ? r / s.heads : 0u;
            const unsigned h = there ? r - token * s.heads : 0u;
            const u64 row = token0 * s.heads + (there ? r : 0u);
            const char* grad = s.grad.data + grad_at[token] + (i64)h * s.grad.head;
            float gu[K][V], gv[K][V], u[K][V], v[K][V];
            float step8_ = 0.0f;
            if constexpr (kCodes) step8_ = step8(s.scales[row]);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (there && mine[k]) {
                    load_pairs<T, V, kInterleaved>(grad, at[k], gu[k], gv[k]);
                    if constexpr (kCodes) {
                        load_codes<V>(s.codes + row * a.pitch + at[k].first, step8_, u[k]);
                        load_codes<V>(s.codes + row * a.pitch + at[k].second, step8_, v[k]);
                        if constexpr (kInterleaved && V > 1) part(u[k], v[k]);
                    } else {
                        load_pairs<T, V, kInterleaved>(s.x.data + x_at[token] + (i64)h * s.x.head, at[k], u[k], v[k]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) gu[k][i] = gv[k][i] = u[k][i] = v[k][i] = 0.0f;
                }
            }
            float squares = 0.0f, dot = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                turn(table + token * pairs, at[k], pairs, gu[k], gv[k]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    squares = fmaf(u[k][i], u[k][i], fmaf(v[k][i], v[k][i], squares));
                    dot = fmaf(gu[k][i] * wu[k][i], u[k][i], fmaf(gv[k][i] * wv[k][i], v[k][i], dot));
                }
            }
            squares = group_sum(squares, a.group);
            dot = group_sum(dot, a.group);
            const float rstd = there ? rsqrtf(squares / (float)a.dim + a.eps) : 0.0f;
            const float back = dot / (float)a.dim * rstd * rstd;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    du[k][i] = fmaf(gu[k][i] * rstd, u[k][i], du[k][i]);
                    dv[k][i] = fmaf(gv[k][i] * rstd, v[k][i], dv[k][i]);
                    u[k][i] = rstd * fmaf(-u[k][i], back, gu[k][i] * wu[k][i]);
                    v[k][i] = rstd * fmaf(-v[k][i], back, gv[k][i] * wv[k][i]);
                }
                if (there && mine[k]) store_pairs<T, V, kInterleaved>(s.out + row * a.dim * sizeof(T), at[k], u[k], v[k]);
            }
        }
    }
    // The groups of a warp, then the warps.
    __syncthreads();
    float* sums = reinterpret_cast<float*>(shared);
    const unsigned warp = threadIdx.x / 32u, in_warp = threadIdx.x & 31u;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            for (unsigned o = a.group; o < 32u; o <<= 1) {
                du[k][i] += __shfl_xor_sync(0xffffffffu, du[k][i], o);
                dv[k][i] += __shfl_xor_sync(0xffffffffu, dv[k][i], o);
            }
            if (in_warp < a.group && mine[k]) {
                sums[warp * a.dim + (kInterleaved ? at[k].first + 2 * i : at[k].first + i)] = du[k][i];
                sums[warp * a.dim + (kInterleaved ? at[k].first + 2 * i + 1 : at[k].second + i)] = dv[k][i];
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

// weight_grad[d] = sum of partial[cta][d]: 32 columns of one side per CTA.
template <typename T>
__global__ void __launch_bounds__(1024) sum_kernel(const __grid_constant__ RotationArgs a) {
    __shared__ float sums[32][33];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Side& s = a.side[blockIdx.y];
    const unsigned column = blockIdx.x * 32u + (threadIdx.x & 31u), part = threadIdx.x >> 5;
    float sum = 0.0f;
    if (column < a.dim)
        for (unsigned c = part; c < s.ctas; c += 32u) sum += s.partial[(u64)c * a.dim + column];
    sums[part][threadIdx.x & 31u] = sum;
    __syncthreads();
    sum = sums[threadIdx.x & 31u][part];  // warp `part` adds column `part`
    for (unsigned o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const unsigned d = blockIdx.x * 32u + part;
    if ((threadIdx.x & 31u) == 0 && d < a.dim && s.weight_grad != nullptr) reinterpret_cast<T*>(s.weight_grad)[d] = Elem<T>::from_f(sum);
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
    a.all = (u64)c.batch * (u64)c.tokens;
    a.tokens = (u64)c.tokens;
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
        t.heads = (unsigned)s.heads;
    }
    return a;
}

// Tokens of a tile: as many as give every group `passes` heads.
void cut(RotationArgs& a, unsigned passes) {
    for (Side& s : a.side) {
        if (s.heads == 0) continue;
        const unsigned want = passes * (kThreads / a.group);
        s.tile = (unsigned)std::min<u64>(std::max(1u, want / s.heads), a.all);
        s.tiles = (unsigned)((a.all + s.tile - 1) / s.tile);
    }
}

std::size_t table_bytes(const RotationArgs& a) {
    std::size_t most = 0;
    for (const Side& s : a.side) most = std::max<std::size_t>(most, s.tile * (16 + (std::size_t)a.rotated / 2 * 8));
    return most;
}

template <typename T, int V, int K, bool kInterleaved>
cudaError_t forward(const RotationCall& c, RotationArgs& a) {
    constexpr int U = 2;
    cut(a, U);
    for (Side& s : a.side) s.ctas = s.heads == 0 ? 0u : s.tiles;
    const unsigned grid = a.side[0].ctas + a.side[1].ctas;
    return launch_dependent<RotationArgs>(c.norm ? rotate_kernel<T, V, K, kInterleaved, true, U> : rotate_kernel<T, V, K, kInterleaved, false, U>,
                                          grid, kThreads, table_bytes(a), c.stream, a);
}

template <typename T, int V, int K, bool kInterleaved>
cudaError_t backward(const RotationCall& c, RotationArgs& a) {
    if (a.all == 0) return launch_dependent<RotationArgs>(sum_kernel<T>, dim3((a.dim + 31) / 32, 2), 1024, 0, c.stream, a);  // of nothing
    cut(a, 2);
    const unsigned heads = a.side[0].heads + a.side[1].heads;
    bool codes = false;
    for (Side& s : a.side) {
        if (s.heads == 0) continue;
        codes = s.codes != nullptr;
        s.ctas = std::min(s.tiles, std::max(1u, kHeadGradCtas * s.heads / heads));
    }
    const std::size_t shared = std::max<std::size_t>(table_bytes(a), kWarps * a.dim * sizeof(float));
    const cudaError_t st = launch_dependent<RotationArgs>(
        codes ? rotate_norm_backward_kernel<T, V, K, kInterleaved, true> : rotate_norm_backward_kernel<T, V, K, kInterleaved, false>,
        a.side[0].ctas + a.side[1].ctas, kThreads, shared, c.stream, a);
    if (st != cudaSuccess) return st;
    return launch_dependent<RotationArgs>(sum_kernel<T>, dim3((a.dim + 31) / 32, 2), 1024, 0, c.stream, a);
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
