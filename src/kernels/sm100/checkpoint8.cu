// Activations kept in 8 bits for the backward pass: the codec, alone and in the same pass as GELU and its derivative.
//
// Bound by HBM: a 16-bit element is read once and its 1 + 1/32 bytes are written once (and y beside them), or the other way round.
// Formulas of the 8-bit form: block8.cuh. GELU keeps its INPUT: y = x Phi(x) is made from x itself, dx = dy * (Phi + x phi)(x^) from what
// was kept, so the forward result does not change and the backward needs neither x nor y.
//
// Phi comes from one exponential: for x >= 0, 1 - Phi(x) = exp(-x^2/2) R(t), t = 1/(1 + 0.28 x), where R(t) = t P(t) and P is a polynomial of
// degree 8 fitted to erfcx(x / sqrt 2) / 2 for least largest relative error on [0, 40] (9e-8; 4e-7 in fp32 arithmetic), so the far negative
// tail keeps its relative accuracy, and exp(-x^2/2) is also the derivative's density.
#include "kernels/sm100/checkpoint8.h"

#include "kernels/sm100/block8.cuh"
#include "kernels/sm100/launch.h"

#include <cstdint>

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
    unsigned columns, blocks;  // of a row
    unsigned items;            // half blocks (flat) or blocks (ragged) of all rows
};

// exp(-x^2/2) and 1 - Phi(|x|).
__device__ __forceinline__ void normal_tail(float x, float* density, float* tail) {
    const float t = __fdividef(1.0f, fmaf(fabsf(x), 0.28f, 1.0f));
    float p = 0.02585814922f;
    p = fmaf(p, t, -0.09804277882f);
    p = fmaf(p, t, 0.09953258518f);
    p = fmaf(p, t, -0.01241061024f);
    p = fmaf(p, t, 0.07559080114f);
    p = fmaf(p, t, 0.08288812189f);
    p = fmaf(p, t, 0.1031858347f);
    p = fmaf(p, t, 0.1116940188f);
    p = fmaf(p, t, 0.1117039230f);
    *density = __expf(-0.5f * x * x);
    *tail = *density * p * t;
}

constexpr float kTanhSlope = 0.7978845608f, kTanhCube = 0.044715f;  // tanh(sqrt(2/pi) (x + 0.044715 x^3))

template <Activation kAct>
__device__ __forceinline__ float activate(float x) {
    if constexpr (kAct == Activation::Gelu) {
        float density, tail;
        normal_tail(x, &density, &tail);
        return x * (x >= 0.0f ? 1.0f - tail : tail);
    } else if constexpr (kAct == Activation::GeluTanh) {
        // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
        const float u = kTanhSlope * fmaf(kTanhCube * x * x, x, x);
        const float e = __expf(-2.0f * fabsf(u)), s = __fdividef(1.0f, 1.0f + e);
        return x * (x >= 0.0f ? s : e * s);
    } else {
        return x;
    }
}

// The derivative at a kept value: finite, or NaN (which min and max without .NaN would lose).
template <Activation kAct>
__device__ __forceinline__ float slope(float x) {
    if constexpr (kAct == Activation::Gelu) {
        float density, tail;
        normal_tail(x, &density, &tail);
        return fmaf(x * 0.3989422804f, density, x >= 0.0f ? 1.0f - tail : tail);
    } else if constexpr (kAct == Activation::GeluTanh) {
        // Beyond 64 the slope is 1 or 0 in 32 bits, and x^2 would overflow further out.
        x = OpMin::apply(OpMax::apply(x, -64.0f), 64.0f);
        const float square = x * x;
        const float u = kTanhSlope * fmaf(kTanhCube * square, x, x);
        const float e = __expf(-2.0f * fabsf(u)), s = __fdividef(1.0f, 1.0f + e);
        // s(u) s(-u) = e s^2 for either sign: no difference of numbers near one
        return fmaf(x * (2.0f * kTanhSlope) * fmaf(3.0f * kTanhCube, square, 1.0f), e * s * s, x >= 0.0f ? s : e * s);
    } else {
        return 1.0f;
    }
}

// 16 elements of one row.
template <typename T>
struct Sixteen {
    static constexpr int kPacks = 16 * sizeof(T) / 32;
    Raw32 raw[kPacks];
    __device__ __forceinline__ void load(const char* p) {
#pragma unroll
        for (int i = 0; i < kPacks; ++i) raw[i] = ld32_stream(p + 32 * i);
    }
    __device__ __forceinline__ void widen(float (&f)[16]) const {
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
            float g[16 / kPacks];
            Wide32<T>::unpack(raw[i], g);
#pragma unroll
            for (int e = 0; e < 16 / kPacks; ++e) f[i * (16 / kPacks) + e] = g[e];
        }
    }
    static __device__ __forceinline__ void store(char* p, const float (&f)[16]) {
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
            float g[16 / kPacks];
#pragma unroll
            for (int e = 0; e < 16 / kPacks; ++e) g[e] = f[i * (16 / kPacks) + e];
            st32(p + 32 * i, Wide32<T>::pack(g));
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
            const unsigned row = i / (2u * a.blocks), half = i - row * (2u * a.blocks);
            x[u].load(a.in + (long long)row * a.stride + (u64)half * (16 * sizeof(T)));
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + u * kThreads;
        float f[16];
        unsigned amax = 0;
        if (i < a.items) {
            x[u].widen(f);
#pragma unroll
            for (int e = 0; e < 16; ++e) amax = max(amax, magnitude_bits(f[e]));
        }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        if (i < a.items) {
            if (kAct == Activation::None || a.codes != nullptr) {
                const unsigned scale = scale8<T>(amax);
                const float inverse = inverse_step8(scale);
                uint4 c;
                c.x = finite8(encode8x4(f, inverse), scale);
                c.y = finite8(encode8x4(f + 4, inverse), scale);
                c.z = finite8(encode8x4(f + 8, inverse), scale);
                c.w = finite8(encode8x4(f + 12, inverse), scale);
                st16(reinterpret_cast<uint4*>(a.codes) + i, c);
                if ((i & 1u) == 0) a.scales[i >> 1] = (unsigned char)scale;
            }
            if constexpr (kAct != Activation::None) {
#pragma unroll
                for (int e = 0; e < 16; ++e) f[e] = activate<kAct>(f[e]);
                Sixteen<T>::store(a.out + (u64)i * (16 * sizeof(T)), f);
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
            c[u] = ld16_stream(reinterpret_cast<const uint4*>(a.codes) + i);
            scale[u] = a.scales[i >> 1];
            if constexpr (kAct != Activation::None) {
                const unsigned row = i / (2u * a.blocks), half = i - row * (2u * a.blocks);
                dy[u].load(a.in + (long long)row * a.stride + (u64)half * (16 * sizeof(T)));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + u * kThreads;
        if (i < a.items) {
            const float step = step8(scale[u]);
            float f[16];
            decode8x4(c[u].x, step, f);
            decode8x4(c[u].y, step, f + 4);
            decode8x4(c[u].z, step, f + 8);
            decode8x4(c[u].w, step, f + 12);
            if constexpr (kAct != Activation::None) {
                float g[16];
                dy[u].widen(g);
#pragma unroll
                for (int e = 0; e < 16; ++e) f[e] = g[e] * slope<kAct>(f[e]);
            }
            Sixteen<T>::store(a.out + (u64)i * (16 * sizeof(T)), f);
        }
    }
}

// Any columns, strides and alignment: a warp takes a block, a lane an element, so that neighbouring lanes touch neighbouring bytes.
constexpr int kRaggedBlocks = 4;  // blocks in flight per warp

template <typename T, Activation kAct>
__global__ void __launch_bounds__(kThreads) keep8_ragged_kernel(const Kept8Args a) {
    constexpr int U = kRaggedBlocks;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned lane = threadIdx.x & 31u;
    const unsigned first = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * U;
    float f[U];
    u64 at[U];  // of the element among rows without gaps
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + u;
        const unsigned row = i / a.blocks, column = (i - row * a.blocks) * kBlock8 + lane;
        const bool there = i < a.items && column < a.columns;
        at[u] = there ? (u64)row * a.columns + column : ~0ull;
        f[u] = there ? Elem<T>::to_f(*(reinterpret_cast<const T*>(a.in + (long long)row * a.stride) + column)) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + u;
        if (i < a.items) {  // the same for the whole warp
            if (kAct == Activation::None || a.codes != nullptr) {
                const unsigned scale = scale8<T>(__reduce_max_sync(0xffffffffu, magnitude_bits(f[u])));
                a.codes[(u64)i * kBlock8 + lane] = (unsigned char)finite8(encode8(f[u], inverse_step8(scale)), scale);
                if (lane == 0) a.scales[i] = (unsigned char)scale;
            }
            if constexpr (kAct != Activation::None)
                if (at[u] != ~0ull) reinterpret_cast<T*>(a.out)[at[u]] = Elem<T>::from_f(activate<kAct>(f[u]));
        }
    }
}

template <typename T, Activation kAct>
__global__ void __launch_bounds__(kThreads) read8_ragged_kernel(const Kept8Args a) {
    constexpr int U = kRaggedBlocks;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned lane = threadIdx.x & 31u;
    const unsigned first = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * U;
    unsigned code[U], scale[U];
    float dy[U];
    u64 at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned i = first + u;
        const unsigned row = i / a.blocks, column = (i - row * a.blocks) * kBlock8 + lane;
        const bool there = i < a.items && column < a.columns;
        at[u] = there ? (u64)row * a.columns + column : ~0ull;
        code[u] = there ? a.codes[(u64)i * kBlock8 + lane] : 0u;
        scale[u] = there ? a.scales[i] : 1u;
        if constexpr (kAct != Activation::None)
            dy[u] = there ? Elem<T>::to_f(*(reinterpret_cast<const T*>(a.in + (long long)row * a.stride) + column)) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float f = decode8<0>(code[u], step8(scale[u]));
        if constexpr (kAct != Activation::None) f = dy[u] * slope<kAct>(f);
        if (at[u] != ~0ull) reinterpret_cast<T*>(a.out)[at[u]] = Elem<T>::from_f(f);
    }
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
    a.columns = (unsigned)c.columns;
    a.blocks = (unsigned)((c.columns + kBlock8 - 1) / kBlock8);
    const std::uintptr_t addresses = reinterpret_cast<std::uintptr_t>(c.in) | reinterpret_cast<std::uintptr_t>(c.out) |
                                     reinterpret_cast<std::uintptr_t>(c.codes) | (std::uintptr_t)(c.rows > 1 ? a.stride : 0);
    if (c.columns % kBlock8 == 0 && addresses % 32 == 0) {
        a.items = (unsigned)(c.rows * a.blocks * 2);
        const unsigned grid = (a.items + kThreads * kInFlight<T> - 1) / (kThreads * kInFlight<T>);
        return launch_dependent<Kept8Args>(keep ? keep8_kernel<T, kAct> : read8_kernel<T, kAct>, grid, kThreads, 0, c.stream, a);
    }
    a.items = (unsigned)(c.rows * a.blocks);
    constexpr unsigned kPerCta = kThreads / 32 * kRaggedBlocks;
    return launch_dependent<Kept8Args>(keep ? keep8_ragged_kernel<T, kAct> : read8_ragged_kernel<T, kAct>, (a.items + kPerCta - 1) / kPerCta,
                                       kThreads, 0, c.stream, a);
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
