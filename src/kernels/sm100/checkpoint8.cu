// Activations kept in 8 bits for the backward pass: the codec, alone and in the same pass as GELU and its derivative.
//
// Bound by HBM: a 16-bit element is read once and its 1 + 1/32 bytes are written once (and y beside them), or the other way round. bf16: 16384 x 4096 are kept in
// 28 us and read back in 30 (7.3 and 6.7 TB/s, some of it from L2); GELU of 8192 x 8192 takes 60 us, its gradient 64 (5.6 and 5.3 TB/s, 0.8 of a copy's rate, with
// 0.7 of the issue slots taken: codes two at a time and fp32 numbers by pairs took 95 and 87 to that).
// Formulas of the 8-bit form: block8.cuh. GELU keeps its INPUT: y = x Phi(x) is made from x itself, dx = dy * (Phi + x phi)(x^) from what
// was kept, so the forward result does not change and the backward needs neither x nor y.
//
// Phi comes from one exponential: for x >= 0, 1 - Phi(x) = exp(-x^2/2) R(t), t = 1/(1 + 0.28 x), where R(t) = t P(t) and P is a polynomial of
// degree 8 fitted to erfcx(x / sqrt 2) / 2 for least largest relative error on [0, 40] (9e-8; 4e-7 in fp32 arithmetic), so the far negative
// tail keeps its relative accuracy, and exp(-x^2/2) is also the derivative's density.
#include "kernels/sm100/checkpoint8.h"

#include "kernels/sm100/block8.cuh"
#include "kernels/sm100/launch.h"
#include "kernels/sm100/pair32.cuh"

#include <cstdint>
#include <type_traits>

namespace b200ccl::kernels {

using namespace b200ccl::dev;

namespace {

using u64 = unsigned long long;

constexpr unsigned kThreads = 256;

struct Kept8Args {
    const char* in;
    long long stride;  // bytes
    char* out;
    unsigned char* codes;
    unsigned char* scales;
    u64 elements;     // of all rows
    unsigned columns;
    Divisor halves;   // half blocks of a row
    unsigned items;   // half blocks of all rows
    Divisor by_columns;
};

// exp(-x^2/2) and 1 - Phi(|x|) of two numbers.
struct Tail {
    Pair32 density, tail;
};
__device__ __forceinline__ Tail normal_tail(float2 x) {
    const Pair32 d = fma2(pair32(fabsf(x.x), fabsf(x.y)), both32(0.28f), both32(1.0f));
    const float2 f = apart(d);
    const Pair32 t = pair32(reciprocal_fast(f.x), reciprocal_fast(f.y));
    Pair32 p = both32(0.02585814922f);
    p = fma2(p, t, both32(-0.09804277882f));
    p = fma2(p, t, both32(0.09953258518f));
    p = fma2(p, t, both32(-0.01241061024f));
    p = fma2(p, t, both32(0.07559080114f));
    p = fma2(p, t, both32(0.08288812189f));
    p = fma2(p, t, both32(0.1031858347f));
    p = fma2(p, t, both32(0.1116940188f));
    p = fma2(p, t, both32(0.1117039230f));
    const Pair32 v = pair32(x.x, x.y);
    const float2 e = apart(mul2(v, mul2(v, both32(-0.7213475204f))));  // -x^2 / 2 * log2(e)
    Tail r;
    r.density = pair32(exp2_fast(e.x), exp2_fast(e.y));
    r.tail = mul2(r.density, mul2(p, t));
    return r;
}

constexpr float kTanhSlope = 0.7978845608f, kTanhCube = 0.044715f;  // tanh(sqrt(2/pi) (x + 0.044715 x^3))

// e = exp(-2|u|) and s = 1 / (1 + e) of two numbers: (1 + tanh u) / 2 is s for u >= 0, e s below. u grows without bound, e ends at 0.
struct Logistic {
    float2 e, s;
    Pair32 square;
};
__device__ __forceinline__ Logistic logistic(float2 x) {
    Logistic r;
    const Pair32 v = pair32(x.x, x.y);
    r.square = mul2(v, v);
    const float2 u = apart(mul2(v, fma2(r.square, both32(kTanhCube), both32(1.0f))));
    constexpr float kSlope = -2.0f * kTanhSlope * 1.442695041f;
    r.e = make_float2(exp2_fast(kSlope * fabsf(u.x)), exp2_fast(kSlope * fabsf(u.y)));
    r.s = make_float2(reciprocal_fast(1.0f + r.e.x), reciprocal_fast(1.0f + r.e.y));
    return r;
}

template <Activation kAct>
__device__ __forceinline__ float2 activate(float2 x) {
    const Pair32 v = pair32(x.x, x.y);
    if constexpr (kAct == Activation::Gelu) {
        const Pair32 tail = normal_tail(x).tail;
        const float2 low = apart(tail), high = apart(fma2(tail, both32(-1.0f), both32(1.0f)));
        return apart(mul2(v, pair32(x.x >= 0.0f ? high.x : low.x, x.y >= 0.0f ? high.y : low.y)));
    } else if constexpr (kAct == Activation::GeluTanh) {
        const Logistic l = logistic(x);
        const float2 low = apart(mul2(pair32(l.e.x, l.e.y), pair32(l.s.x, l.s.y)));
        return apart(mul2(v, pair32(x.x >= 0.0f ? l.s.x : low.x, x.y >= 0.0f ? l.s.y : low.y)));
    } else {
        return x;
    }
}

// dy times the derivative at kept values: finite, or NaN (which min and max without .NaN would lose).
template <Activation kAct>
__device__ __forceinline__ float2 through(float2 x, float2 dy) {
    const Pair32 g = pair32(dy.x, dy.y);
    if constexpr (kAct == Activation::Gelu) {
        // Phi + x phi: for x >= 0, 1 - (tail - |x| phi)
        const Tail t = normal_tail(x);
        const Pair32 below = fma2(mul2(pair32(fabsf(x.x), fabsf(x.y)), both32(-0.3989422804f)), t.density, t.tail);
        const float2 low = apart(below), high = apart(fma2(below, both32(-1.0f), both32(1.0f)));
        return apart(mul2(g, pair32(x.x >= 0.0f ? high.x : low.x, x.y >= 0.0f ? high.y : low.y)));
    } else if constexpr (kAct == Activation::GeluTanh) {
        // Beyond 64 the slope is 1 or 0 in 32 bits, and x^2 would overflow further out.
        x = make_float2(OpMin::apply(OpMax::apply(x.x, -64.0f), 64.0f), OpMin::apply(OpMax::apply(x.y, -64.0f), 64.0f));
        const Logistic l = logistic(x);
        const Pair32 s = pair32(l.s.x, l.s.y), es = mul2(pair32(l.e.x, l.e.y), s);
        const float2 low = apart(es);
        // s(u) s(-u) = e s^2 for either sign: no difference of numbers near one
        const Pair32 du = mul2(mul2(pair32(x.x, x.y), both32(2.0f * kTanhSlope)), fma2(l.square, both32(3.0f * kTanhCube), both32(1.0f)));
        return apart(mul2(g, fma2(du, mul2(es, s), pair32(x.x >= 0.0f ? l.s.x : low.x, x.y >= 0.0f ? l.s.y : low.y))));
    } else {
        return x;
    }
}

// 16 elements of one row.
template <typename T>
struct Sixteen {
    static constexpr int kWords = 16 * sizeof(T) / 4;
    unsigned w[kWords];
    __device__ __forceinline__ void load(const char* p) {
#pragma unroll
        for (int i = 0; i < kWords / 8; ++i) put(i, ld32_stream(p + 32 * i));
    }
    __device__ __forceinline__ void put(int i, const Raw32& r) {
        w[8 * i] = r.lo.x; w[8 * i + 1] = r.lo.y; w[8 * i + 2] = r.lo.z; w[8 * i + 3] = r.lo.w;
        w[8 * i + 4] = r.hi.x; w[8 * i + 5] = r.hi.y; w[8 * i + 6] = r.hi.z; w[8 * i + 7] = r.hi.w;
    }
    __device__ __forceinline__ void store(char* p) const {
#pragma unroll
        for (int i = 0; i < kWords / 8; ++i) {
            Raw32 r;
            r.lo = make_uint4(w[8 * i], w[8 * i + 1], w[8 * i + 2], w[8 * i + 3]);
            r.hi = make_uint4(w[8 * i + 4], w[8 * i + 5], w[8 * i + 6], w[8 * i + 7]);
            st32(p + 32 * i, r);
        }
    }
    // Elements 2i and 2i + 1.
    __device__ __forceinline__ float2 pair(int i) const {
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else if constexpr (std::is_same_v<T, __half>) return h2_to_f2(w[i]);
        else return b2_to_f2(w[i]);
    }
    __device__ __forceinline__ void set(int i, float2 f) {
        if constexpr (sizeof(T) == 4) { w[2 * i] = __float_as_uint(f.x); w[2 * i + 1] = __float_as_uint(f.y); }
        else if constexpr (std::is_same_v<T, __half>) w[i] = f2_to_h2(f.x, f.y);
        else w[i] = f2_to_b2(f.x, f.y);
    }
    __device__ __forceinline__ unsigned amax() const {
        unsigned m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7fffffffu);
            return m;
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) m = larger_magnitudes<T>(m, w[i]);
            return magnitude_of_pair<T>(m);
        }
    }
    __device__ __forceinline__ uint4 codes(unsigned scale) const {
        unsigned c[4];
        if constexpr (sizeof(T) == 4) {
            const float inverse = inverse_step8(scale);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f[4] = {__uint_as_float(w[4 * i]), __uint_as_float(w[4 * i + 1]), __uint_as_float(w[4 * i + 2]), __uint_as_float(w[4 * i + 3])};
                c[i] = finite8(encode8x4(f, inverse), scale);
            }
        } else {
            const Inverse16<T> inverse(scale);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = finite8(encode8x4(w[2 * i], w[2 * i + 1], inverse), scale);
        }
        return make_uint4(c[0], c[1], c[2], c[3]);
    }
    __device__ __forceinline__ void widen(const uint4& codes, unsigned scale) {
        const unsigned c[4] = {codes.x, codes.y, codes.z, codes.w};
        if constexpr (sizeof(T) == 4) {
            const float step = step8(scale);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float f[4];
                decode8x4(c[i], step, f);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * i + e] = __float_as_uint(f[e]);
            }
        } else {
            const unsigned step = step16<T>(scale);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint2 v = widen8x4<T>(c[i], step);
                w[2 * i] = v.x;
                w[2 * i + 1] = v.y;
            }
        }
    }
};

// Half blocks in flight per thread: 64 bytes of input either way.
template <typename T>
constexpr int kInFlight = sizeof(T) == 4 ? 1 : 2;

// Whole blocks, rows at 32-byte boundaries: two neighbouring lanes hold a block, 16 elements each.
template <typename T, Activation kAct>
__global__ void __launch_bounds__(kThreads) keep8_kernel(const Kept8Args a) {
    constexpr int U = kInFlight<T>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned first = blockIdx.x * (kThreads * U) + threadIdx.x;
    Sixteen<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + u * kThreads;
        if (i < a.items) {
            const unsigned row = a.halves.divide(i), half = i - row * a.halves.d;
            x[u].load(a.in + (long long)row * a.stride + (u64)half * (16 * sizeof(T)));
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + u * kThreads;
        unsigned amax = i < a.items ? x[u].amax() : 0u;
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        if (i < a.items) {
            if (kAct == Activation::None || a.codes != nullptr) {
                const unsigned scale = scale8<T>(amax);
                st16(reinterpret_cast<uint4*>(a.codes) + i, x[u].codes(scale));
                if ((i & 1u) == 0) a.scales[i >> 1] = (unsigned char)scale;
            }
            if constexpr (kAct != Activation::None) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[u].set(e, activate<kAct>(x[u].pair(e)));
                x[u].store(a.out + (u64)i * (16 * sizeof(T)));
            }
        }
    }
}

template <typename T, Activation kAct>
__global__ void __launch_bounds__(kThreads) read8_kernel(const Kept8Args a) {
    constexpr int U = kInFlight<T>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned first = blockIdx.x * (kThreads * U) + threadIdx.x;
    uint4 c[U];
    unsigned scale[U];
    Sixteen<T> dy[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + u * kThreads;
        if (i < a.items) {
            c[u] = load16_once(reinterpret_cast<const uint4*>(a.codes) + i);
            scale[u] = a.scales[i >> 1];
            if constexpr (kAct != Activation::None) {
                const unsigned row = a.halves.divide(i), half = i - row * a.halves.d;
                dy[u].load(a.in + (long long)row * a.stride + (u64)half * (16 * sizeof(T)));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + u * kThreads;
        if (i < a.items) {
            Sixteen<T> x;
            x.widen(c[u], scale[u]);
            if constexpr (kAct != Activation::None) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x.set(e, through<kAct>(x.pair(e), dy[u].pair(e)));
            }
            x.store(a.out + (u64)i * (16 * sizeof(T)));
        }
    }
}

// ---- any columns, strides and alignment ------------------------------------------------------------------
// Inputs are read as the aligned 16 bytes that they lie in, and shifted; only those that hold a wanted element are touched. What is written to rows without
// gaps is cut where the memory is aligned, wherever rows and blocks begin: a thread makes 16 bytes of the output.

template <typename T>
constexpr int kGranule = 16 / sizeof(T);  // elements of 16 bytes

template <typename T>
__device__ __forceinline__ float2 pair_in(const unsigned* w, int i) {
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else if constexpr (std::is_same_v<T, __half>) return h2_to_f2(w[i]);
    else return b2_to_f2(w[i]);
}
template <typename T>
__device__ __forceinline__ void store_granule(char* p, const float2 (&f)[kGranule<T> / 2]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < kGranule<T> / 2; ++i) {
        if constexpr (sizeof(T) == 4) {
            w[2 * i] = __float_as_uint(f[i].x);
            w[2 * i + 1] = __float_as_uint(f[i].y);
        } else {
            w[i] = std::is_same_v<T, __half> ? f2_to_h2(f[i].x, f[i].y) : f2_to_b2(f[i].x, f[i].y);
        }
    }
    store16_once(p, make_uint4(w[0], w[1], w[2], w[3]));
}

// Where element `from + offset` of all lies, `from` being element (row, column): offsets are small.
struct Spot {
    unsigned row, column;
};
__device__ __forceinline__ Spot spot_at(const Kept8Args& a, const Spot& from, unsigned offset) {
    const unsigned in = from.column + offset, rows = a.by_columns.divide(in);
    return {from.row + rows, in - rows * a.columns};
}

// One element of the input, and of x^.
template <typename T>
__device__ __forceinline__ float input_at(const Kept8Args& a, const Spot& s) {
    return Elem<T>::to_f(*(reinterpret_cast<const T*>(a.in + (long long)s.row * a.stride) + s.column));
}
__device__ __forceinline__ float kept_at(const Kept8Args& a, const Spot& s) {
    const u64 half = (u64)s.row * a.halves.d;
    return decode8<0>(a.codes[half * 16u + s.column], step8(a.scales[half / 2u + s.column / kBlock8]));
}
// Two elements of the output.
template <typename T, Activation kAct, bool kRead>
__device__ __forceinline__ float2 two_at(const Kept8Args& a, const Spot& s, const Spot& t) {
    if constexpr (!kRead) return activate<kAct>(make_float2(input_at<T>(a, s), input_at<T>(a, t)));
    const float2 v = make_float2(kept_at(a, s), kept_at(a, t));
    if constexpr (kAct == Activation::None) return v;
    else return through<kAct>(v, make_float2(input_at<T>(a, s), input_at<T>(a, t)));
}
// A granule of the output that lies across rows, or not wholly in it: elements [begin, end) of the E from `origin` + `offset` on, `origin` being (row, column).
template <typename T, Activation kAct, bool kRead>
__device__ __forceinline__ void gather_granule(const Kept8Args& a, u64 begin, u64 end, const Spot& from, u64 origin) {
    constexpr unsigned E = kGranule<T>;
    if (end - begin == E) {
        float2 f[E / 2];
#pragma unroll
        for (unsigned i = 0; i < E / 2; ++i)
            f[i] = two_at<T, kAct, kRead>(a, spot_at(a, from, (unsigned)(begin - origin) + 2u * i), spot_at(a, from, (unsigned)(begin - origin) + 2u * i + 1u));
        store_granule<T>(a.out + begin * sizeof(T), f);
    } else {
        for (u64 e = begin; e < end; ++e) {
            const Spot s = spot_at(a, from, (unsigned)(e - origin));
            reinterpret_cast<T*>(a.out)[e] = Elem<T>::from_f(two_at<T, kAct, kRead>(a, s, s).x);
        }
    }
}

// Elements by which the output lies behind a multiple of 16 bytes.
template <typename T>
__device__ __forceinline__ unsigned behind(const Kept8Args& a) {
    return (unsigned)(reinterpret_cast<std::uintptr_t>(a.out) & 15u) / (unsigned)sizeof(T);
}
// Of the granules k0 to k1 those that lie across two rows, one at the end of a row: all of a CTA's side by side, because a warp that meets one
// among others goes the long way for it (GELU of 13760 x 185 bf16, there and back: 27.5 us with them among the others, 17.5 so).
template <typename T, Activation kAct, bool kRead>
__device__ __forceinline__ void across_rows(const Kept8Args& a, u64 k0, u64 k1, const Spot& from, u64 origin, unsigned m) {
    constexpr unsigned E = kGranule<T>;
    if (a.columns < E) return;
    for (u64 row = (u64)from.row + threadIdx.x;; row += kThreads) {
        const u64 end = (row + 1u) * a.columns, k = (end + m) / E;
        if (k >= k1) break;
        const u64 e = k * E - m;
        if ((end + m) % E != 0u && k >= k0 && k * E >= m && e + E <= a.elements) gather_granule<T, kAct, kRead>(a, e, e + E, from, origin);
    }
}

template <typename T, Activation kAct>
__global__ void __launch_bounds__(kThreads) keep8_any_kernel(const Kept8Args a) {
    constexpr int U = kInFlight<T>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned begin = blockIdx.x * (kThreads * U);
    if (kAct == Activation::None || a.codes != nullptr) {
        Sixteen<T> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned i = begin + threadIdx.x + u * kThreads;
            const unsigned row = a.halves.divide(i), column = (i - row * a.halves.d) * 16u;
            const unsigned count = i < a.items && column < a.columns ? min(16u, a.columns - column) : 0u;
            load_any<T, 16>(a.in + (count == 0u ? 0ll : (long long)row * a.stride + (long long)(column * (unsigned)sizeof(T))), count, x[u].w);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned i = begin + threadIdx.x + u * kThreads;
            unsigned amax = x[u].amax();
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            if (i < a.items) {
                const unsigned scale = scale8<T>(amax);
                store16_once(a.codes + (u64)i * 16u, x[u].codes(scale));
                if ((i & 1u) == 0) a.scales[i >> 1] = (unsigned char)scale;
            }
        }
    }
    if constexpr (kAct != Activation::None) {
        // The elements of the same half blocks, by granules of the output that begin among them; they are in L1.
        constexpr unsigned E = kGranule<T>;
        const unsigned end = min(a.items, begin + kThreads * U), m = behind<T>(a);
        const auto first_of = [&](unsigned i) {
            const unsigned row = a.halves.divide(i);
            return Spot{row, min(a.columns, (i - row * a.halves.d) * 16u)};
        };
        const Spot from = first_of(begin), to = first_of(end);
        const u64 origin = (u64)from.row * a.columns + from.column, stop = end == a.items ? a.elements : (u64)to.row * a.columns + to.column;
        const u64 k0 = origin == 0 ? 0 : (origin + m + E - 1) / E, k1 = (stop + m + E - 1) / E;
        for (u64 k = k0 + threadIdx.x; k < k1; k += kThreads) {
            const u64 e = k * E - m;  // before 0 for the first granule of an output that is not aligned
            const Spot s = spot_at(a, from, k * E < m ? 0u : (unsigned)(e - origin));
            if (k * E < m || e + E > a.elements || a.columns < E) {
                gather_granule<T, kAct, false>(a, k * E < m ? 0 : e, min(a.elements, e + E), from, origin);
            } else if (s.column + E <= a.columns) {
                unsigned w[4];
                load_any<T, E>(a.in + (long long)s.row * a.stride + (long long)(s.column * (unsigned)sizeof(T)), E, w);
                float2 f[E / 2];
#pragma unroll
                for (unsigned i = 0; i < E / 2; ++i) f[i] = activate<kAct>(pair_in<T>(w, i));
                store_granule<T>(a.out + e * sizeof(T), f);
            }
        }
        across_rows<T, kAct, false>(a, k0, k1, from, origin, m);
    }
}

constexpr unsigned kGranules = 2;  // of a thread

template <typename T, Activation kAct>
__global__ void __launch_bounds__(kThreads) read8_any_kernel(const Kept8Args a) {
    constexpr unsigned E = kGranule<T>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned m = behind<T>(a);
    const u64 k0 = (u64)blockIdx.x * (kThreads * kGranules);
    const u64 origin = k0 * E < m ? 0 : k0 * E - m;
    __shared__ Spot first;
    if (threadIdx.x == 0) {  // a division of 64 bits, once
        const u64 row = origin / a.columns;
        first = {(unsigned)row, (unsigned)(origin - row * a.columns)};
    }
    __syncthreads();
    const Spot from = first;
#pragma unroll
    for (unsigned u = 0; u < kGranules; ++u) {
        const u64 k = k0 + threadIdx.x + u * kThreads;
        const bool before = k * E < m;
        const u64 e = k * E - m;
        if (!before && e >= a.elements) continue;
        const Spot s = spot_at(a, from, before ? 0u : (unsigned)(e - origin));
        if (before || e + E > a.elements || a.columns < E) {
            gather_granule<T, kAct, true>(a, before ? 0 : e, min(a.elements, e + E), from, origin);
            continue;
        }
        if (s.column + E > a.columns) continue;
        // E codes, at any address, and the steps of the one or two blocks that they belong to.
        const u64 half = (u64)s.row * a.halves.d;
        const unsigned char* codes = a.codes + half * 16u + s.column;
        const unsigned shift = (unsigned)(reinterpret_cast<std::uintptr_t>(codes) & 3u) * 8u;
        const unsigned* words = reinterpret_cast<const unsigned*>(codes - shift / 8u);
        unsigned c[E / 4 + 1];
#pragma unroll
        for (unsigned i = 0; i < E / 4; ++i) c[i] = words[i];
        c[E / 4] = shift != 0u ? words[E / 4] : 0u;
        const unsigned char* scale = a.scales + half / 2u + s.column / kBlock8;
        const unsigned in_block = s.column % kBlock8;
        const float near = step8(scale[0]), far = in_block + E > kBlock8 ? step8(scale[1]) : near;
        unsigned dy[4];
        if constexpr (kAct != Activation::None)
            load_any<T, E>(a.in + (long long)s.row * a.stride + (long long)(s.column * (unsigned)sizeof(T)), E, dy);
        float2 f[E / 2];
#pragma unroll
        for (unsigned i = 0; i < E / 4; ++i) {
            const unsigned w = __funnelshift_r(c[i], c[i + 1], shift);
            f[2 * i] = make_float2(decode8<0>(w, in_block + 4u * i < kBlock8 ? near : far), decode8<1>(w, in_block + 4u * i + 1u < kBlock8 ? near : far));
            f[2 * i + 1] = make_float2(decode8<2>(w, in_block + 4u * i + 2u < kBlock8 ? near : far), decode8<3>(w, in_block + 4u * i + 3u < kBlock8 ? near : far));
        }
        if constexpr (kAct != Activation::None) {
#pragma unroll
            for (unsigned i = 0; i < E / 2; ++i) f[i] = through<kAct>(f[i], pair_in<T>(dy, i));
        }
        store_granule<T>(a.out + e * sizeof(T), f);
    }
    across_rows<T, kAct, true>(a, k0, k0 + kThreads * kGranules, from, origin, m);
}

template <typename T, Activation kAct>
cudaError_t start(const Kept8Call& c, bool keep) {
    if (c.rows == 0 || c.columns == 0) return cudaSuccess;
    Kept8Args a;
    a.in = static_cast<const char*>(c.in);
    a.stride = c.stride * (long long)sizeof(T);
    a.out = static_cast<char*>(c.out);
    a.codes = c.codes;
    a.scales = c.scales;
    const unsigned blocks = (unsigned)((c.columns + kBlock8 - 1) / kBlock8);
    a.columns = (unsigned)c.columns;
    a.by_columns = Divisor(a.columns);
    a.halves = Divisor(2u * blocks);
    a.items = (unsigned)(c.rows * blocks * 2);
    a.elements = (u64)c.rows * c.columns;
    const std::uintptr_t addresses = reinterpret_cast<std::uintptr_t>(c.in) | reinterpret_cast<std::uintptr_t>(c.out) |
                                     reinterpret_cast<std::uintptr_t>(c.codes) | (std::uintptr_t)(c.rows > 1 ? a.stride : 0);
    constexpr unsigned kPerCta = kThreads * kInFlight<T>;
    const unsigned ctas = (a.items + kPerCta - 1) / kPerCta;
    if (c.columns % kBlock8 == 0 && addresses % 32 == 0)
        return launch_dependent<Kept8Args>(keep ? keep8_kernel<T, kAct> : read8_kernel<T, kAct>, ctas, kThreads, 0, c.stream, a);
    if (keep) return launch_dependent<Kept8Args>(keep8_any_kernel<T, kAct>, ctas, kThreads, 0, c.stream, a);
    constexpr unsigned kElements = kThreads * kGranules * kGranule<T>;
    const u64 granules = (a.elements + kGranule<T> + kElements - 1) / kElements;  // one more for an output that is not aligned
    return launch_dependent<Kept8Args>(read8_any_kernel<T, kAct>, (unsigned)granules, kThreads, 0, c.stream, a);
}

template <typename T>
cudaError_t start_typed(const Kept8Call& c, bool keep) {
    switch (c.activation) {
        case Activation::None: return start<T, Activation::None>(c, keep);
        case Activation::Gelu: return start<T, Activation::Gelu>(c, keep);
        case Activation::GeluTanh: return start<T, Activation::GeluTanh>(c, keep);
    }
    return cudaErrorInvalidValue;
}

cudaError_t start_any(const Kept8Call& c, bool keep) {
    switch (c.dtype) {
        case DType::Float: return start_typed<float>(c, keep);
        case DType::Float16: return start_typed<__half>(c, keep);
        case DType::BFloat16: return start_typed<__nv_bfloat16>(c, keep);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_keep8(const Kept8Call& call) { return start_any(call, true); }
cudaError_t launch_read8(const Kept8Call& call) { return start_any(call, false); }

}  // namespace b200ccl::kernels
