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
#include "kernels/sm100/tma.cuh"

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
// A lane still has 16 elements of one row, or what is left of it. Inputs are read as the aligned 16 bytes that they lie in, and shifted. Outputs have no gaps
// between rows, so a warp's are one run of memory: it goes through shared memory, from where every lane writes aligned 16 bytes. (16384 x 2047 bf16, GELU there
// and back: 115 us when threads made 16 bytes of the output each from what they belong to, 88 so; 16384 x 2048: 62.)
template <typename T>
constexpr unsigned kStageBytes = (32 * 16 * sizeof(T) + 16) / 128 * 144 + 144;

// Byte p of a run, with a gap after every 128, so that lanes 32 bytes apart write to different banks.
__device__ __forceinline__ unsigned in_stage(unsigned stage, unsigned p) { return stage + p + (p >> 7 << 4); }
__device__ __forceinline__ void stage4(unsigned at, unsigned v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void stage2(unsigned at, unsigned v) { asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"((unsigned short)v) : "memory"); }

// Writes the warp's elements: `count` of a lane, from element `first` of all on, behind those of the lane before it. All lanes call it.
template <typename T>
__device__ __forceinline__ void store_run(char* out, unsigned stage, u64 first, unsigned count, const unsigned (&w)[4 * sizeof(T)]) {
    constexpr unsigned S = sizeof(T);
    const unsigned lane = threadIdx.x & 31u;
    const u64 begin = __shfl_sync(0xffffffffu, first, 0);
    const unsigned before = (unsigned)(first - begin), total = __shfl_sync(0xffffffffu, before + count, 31);
    char* to = out + begin * S;
    const unsigned off = (unsigned)(reinterpret_cast<std::uintptr_t>(to) & 15u), end = off + total * S, p = off + before * S;
    to -= off;
    if constexpr (S == 4) {
#pragma unroll
        for (unsigned i = 0; i < 16; ++i)
            if (i < count) stage4(in_stage(stage, p + 4u * i), w[i]);
    } else if (count < 16u) {
#pragma unroll
        for (unsigned i = 0; i < 16; ++i)
            if (i < count) stage2(in_stage(stage, p + 2u * i), w[i / 2] >> (i % 2 * 16));
    } else if ((p & 2u) == 0u) {
#pragma unroll
        for (unsigned i = 0; i < 8; ++i) stage4(in_stage(stage, p + 4u * i), w[i]);
    } else {
        stage2(in_stage(stage, p), w[0]);
#pragma unroll
        for (unsigned i = 1; i < 8; ++i) stage4(in_stage(stage, p + 4u * i - 2u), __funnelshift_r(w[i - 1], w[i], 16));
        stage2(in_stage(stage, p + 30u), w[7] >> 16);
    }
    __syncwarp();
    for (unsigned b = ((off + 15u) & ~15u) + lane * 16u; b + 16u <= end; b += 512u) {
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(in_stage(stage, b)) : "memory");
        store16_once(to + b, v);
    }
    // The ends: what stands before the first whole 16 bytes, and behind the last.
    const unsigned last = end & ~15u;
    const unsigned b = lane < 16u ? off + lane * S : last + (lane - 16u) * S;
    if (lane < 16u ? off != 0u && b < min(16u, end) : b < end && (last != 0u || off == 0u)) {
        const unsigned at = in_stage(stage, b);
        if constexpr (S == 4) {
            unsigned v;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
            *reinterpret_cast<unsigned*>(to + b) = v;
        } else {
            unsigned short v;
            asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
            *reinterpret_cast<unsigned short*>(to + b) = v;
        }
    }
    __syncwarp();
}

// Where the 16 elements of a half block lie.
struct Half {
    unsigned row, column, count;
};
__device__ __forceinline__ Half half_at(const Kept8Args& a, unsigned i) {
    const unsigned row = a.halves.divide(i), column = (i - row * a.halves.d) * 16u;
    return {row, column, i < a.items && column < a.columns ? min(16u, a.columns - column) : 0u};
}
// Its first element, of all; that of the next one if it has none.
__device__ __forceinline__ u64 first_of(const Kept8Args& a, const Half& h, unsigned i) {
    return i < a.items ? (u64)h.row * a.columns + min(h.column, a.columns) : a.elements;
}
template <typename T>
__device__ __forceinline__ void load_half(const Kept8Args& a, const Half& h, unsigned (&w)[4 * sizeof(T)]) {
    load_any<T, 16>(a.in + (h.count == 0u ? 0ll : (long long)h.row * a.stride + (long long)(h.column * (unsigned)sizeof(T))), h.count, w);
}

template <typename T, Activation kAct>
__global__ void __launch_bounds__(kThreads) keep8_any_kernel(const Kept8Args a) {
    __shared__ __align__(16) unsigned char stages[kAct == Activation::None ? 16 : kThreads / 32 * kStageBytes<T>];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned i = blockIdx.x * kThreads + threadIdx.x;
    const Half h = half_at(a, i);
    Sixteen<T> x;
    load_half<T>(a, h, x.w);
    if (kAct == Activation::None || a.codes != nullptr) {
        unsigned amax = x.amax();
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        if (i < a.items) {
            const unsigned scale = scale8<T>(amax);
            store16_once(a.codes + (u64)i * 16u, x.codes(scale));
            if ((i & 1u) == 0) a.scales[i >> 1] = (unsigned char)scale;
        }
    }
    if constexpr (kAct != Activation::None) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x.set(e, activate<kAct>(x.pair(e)));
        store_run<T>(a.out, smem_addr(stages) + threadIdx.x / 32u * kStageBytes<T>, first_of(a, h, i), h.count, x.w);
    }
}

template <typename T, Activation kAct>
__global__ void __launch_bounds__(kThreads) read8_any_kernel(const Kept8Args a) {
    __shared__ __align__(16) unsigned char stages[kThreads / 32 * kStageBytes<T>];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned i = blockIdx.x * kThreads + threadIdx.x;
    const Half h = half_at(a, i);
    uint4 c = make_uint4(0u, 0u, 0u, 0u);
    unsigned scale = 127u;
    if (i < a.items) {
        c = load16_once(reinterpret_cast<const uint4*>(a.codes) + i);
        scale = a.scales[i >> 1];
    }
    Sixteen<T> x, dy;
    if constexpr (kAct != Activation::None) load_half<T>(a, h, dy.w);
    x.widen(c, scale);
    if constexpr (kAct != Activation::None) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x.set(e, through<kAct>(x.pair(e), dy.pair(e)));
    }
    store_run<T>(a.out, smem_addr(stages) + threadIdx.x / 32u * kStageBytes<T>, first_of(a, h, i), h.count, x.w);
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
    a.halves = Divisor(2u * blocks);
    a.items = (unsigned)(c.rows * blocks * 2);
    a.elements = (u64)c.rows * c.columns;
    const std::uintptr_t addresses = reinterpret_cast<std::uintptr_t>(c.in) | reinterpret_cast<std::uintptr_t>(c.out) |
                                     reinterpret_cast<std::uintptr_t>(c.codes) | (std::uintptr_t)(c.rows > 1 ? a.stride : 0);
    constexpr unsigned kPerCta = kThreads * kInFlight<T>;
    if (c.columns % kBlock8 == 0 && addresses % 32 == 0)
        return launch_dependent<Kept8Args>(keep ? keep8_kernel<T, kAct> : read8_kernel<T, kAct>, (a.items + kPerCta - 1) / kPerCta, kThreads, 0, c.stream, a);
    return launch_dependent<Kept8Args>(keep ? keep8_any_kernel<T, kAct> : read8_any_kernel<T, kAct>, (a.items + kThreads - 1) / kThreads, kThreads, 0, c.stream, a);
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
