// Lookup of tokens in an embedding, y[t] = scale * w[token[t]], and its gradient, dw[v] = scale * the sum of dy[t] over the t with token[t] = v, in the order of t.
//
// Both move memory and compute next to nothing. The gradient is a sum over places that only the tokens know: they are sorted, with their
// places, and each token's rows are then neighbours in the list. Sums are held in 32 bits and rounded once; they do not depend on timing, as those of
// atomic additions would.
//
// Sorting (sort_kernel) is a matter of latency: a cluster of eight CTAs sorts by eight bits at a time, counts and places of its 256 warps in shared memory and
// between the CTAs through distributed shared memory. Meanwhile the rest of the GPU fills the gradient with zeros (fill_kernel), which takes longer where the
// matrix is large beside the tokens, so that sorting is free (50257 x 768 in bf16: up to 32768 tokens; 131072 take 197 us, 1048576 1130, of which the sort is 600). (A CTA of few stores for each 64 KiB: 1.07 GB in 145 us, a loop in as many CTAs as run at once 170 us.)
// Adding (sum_kernel): the list is cut into chunks, and a group of threads goes through one, 16 bytes of a row for each thread. A token whose rows lie in one chunk is
// written at once. What crosses a chunk's ends is written as sums of 32 bits, and join_kernel adds them: a token may have any share of the rows.
#include "kernels/sm100/embedding.h"

#include "core/check.h"
#include "kernels/sm100/block8.cuh"
#include "kernels/sm100/launch.h"
#include "kernels/sm100/pair32.cuh"
#include "kernels/sm100/tcgen05.cuh"
#include "kernels/sm100/vec.cuh"

#include <algorithm>
#include <cstdint>

namespace b200ccl::kernels {

using namespace b200ccl::dev;

namespace {

using u64 = unsigned long long;

struct LookupArgs {
    const void* tokens;
    long long token_stride;
    const char* rows;
    long long stride;  // bytes
    char* out;
    u64 count, vocabulary;
    unsigned width, vectors;  // elements, 16 bytes of a row
    unsigned lanes;           // of a row: a power of two, at most 32
    bool tokens64, wide;      // every row starts at a multiple of 16 bytes
    float scale;
};

__device__ __forceinline__ long long token_at(const void* tokens, bool wide, long long at) {
    return wide ? static_cast<const long long*>(tokens)[at] : static_cast<const int*>(tokens)[at];
}

// Eight (fp32: four) elements from p on, of which n are there; p may be any element.
template <typename T>
__device__ __forceinline__ uint4 load_row16(const char* p, bool wide, unsigned n) {
    if (wide && n >= 16u / sizeof(T)) return load16_once(p);
    unsigned w[4];
    load_any<T, 16 / sizeof(T)>(p, n, w);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void store_row16(char* p, bool wide, unsigned n, uint4 v) {
    if (wide && n >= 16u / sizeof(T)) {
        store16_once(p, v);
        return;
    }
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (unsigned i = 0; i < 16u / sizeof(T); ++i) {
        if (i >= n) break;
        if constexpr (sizeof(T) == 4) reinterpret_cast<unsigned*>(p)[i] = w[i];
        else reinterpret_cast<unsigned short*>(p)[i] = (unsigned short)(w[i / 2] >> (16u * (i & 1u)));
    }
}

constexpr unsigned kLookupVectors = 4;  // of a thread, all on the way at once

template <typename T>
__global__ void __launch_bounds__(256) lookup_kernel(const __grid_constant__ LookupArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr unsigned kElems = 16 / sizeof(T);
    const u64 row = (u64)blockIdx.x * (256u / a.lanes) + threadIdx.x / a.lanes;
    if (row >= a.count) return;
    const long long token = token_at(a.tokens, a.tokens64, (long long)row * a.token_stride);
    const bool there = token >= 0 && (u64)token < a.vocabulary;
    const char* from = a.rows + token * a.stride;
    char* to = a.out + row * a.width * sizeof(T);
    const unsigned first = blockIdx.y * (a.lanes * kLookupVectors) + threadIdx.x % a.lanes;
    uint4 v[kLookupVectors];
#pragma unroll
    for (unsigned i = 0; i < kLookupVectors; ++i) {
        const unsigned at = first + i * a.lanes;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (there && at < a.vectors) v[i] = load_row16<T>(from + (u64)at * 16u, a.wide, a.width - at * kElems);
    }
    const float scale = token >= 0 && !there ? __uint_as_float(0x7fffffffu) : a.scale;
#pragma unroll
    for (unsigned i = 0; i < kLookupVectors; ++i) {
        const unsigned at = first + i * a.lanes;
        if (at >= a.vectors) break;
        if (scale != 1.0f && token >= 0) {
            float f[kElems];
            Wide<T>::unpack(v[i], f);
#pragma unroll
            for (unsigned e = 0; e < kElems; ++e) f[e] *= scale;
            v[i] = Wide<T>::pack(f);
        }
        store_row16<T>(to + (u64)at * 16u, a.wide, a.width - at * kElems, v[i]);
    }
}

// ---- gradient --------------------------------------------------------------------------------------------------

constexpr unsigned kSortCtas = 8, kSortThreads = 1024, kSortWarps = kSortThreads / 32, kBins = 256;

struct SortArgs {
    const void* tokens;
    long long token_stride;
    bool tokens64;
    unsigned count, vocabulary, passes;
    unsigned* keys[2];    // [count]: the last pass writes to the first
    unsigned* places[2];
};

// Tokens that are none are sorted behind all others.
__device__ __forceinline__ unsigned key_of(const SortArgs& a, unsigned i) {
    const long long token = token_at(a.tokens, a.tokens64, (long long)i * a.token_stride);
    return token < 0 || token >= (long long)a.vocabulary ? a.vocabulary : (unsigned)token;
}
__device__ __forceinline__ unsigned load_at_rank(const unsigned* p, unsigned rank) {
    unsigned v;
    asm volatile("{\n .reg .b32 remote;\n mapa.shared::cluster.u32 remote, %1, %2;\n ld.shared::cluster.u32 %0, [remote];\n}\n" : "=r"(v) : "r"(smem_addr(p)), "r"(rank) : "memory");
    return v;
}

__global__ void __launch_bounds__(kSortThreads) __cluster_dims__(kSortCtas, 1, 1) sort_kernel(const __grid_constant__ SortArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (after the wait: fill_kernel starts then, and what came before the sort is over)
    __shared__ unsigned counts[kSortWarps][kBins + 1];  // of each warp's part of the list, then where its next element of a bin goes in the CTA's
    __shared__ unsigned totals[kBins];                  // of this CTA
    __shared__ unsigned bases[kBins];                   // where its elements of a bin go
    __shared__ unsigned sums[kBins / 32];
    const unsigned rank = cluster_rank(), warp = threadIdx.x / 32u, lane = threadIdx.x & 31u;
    const unsigned each = ((a.count + kSortCtas * kSortWarps - 1) / (kSortCtas * kSortWarps) + 31u) / 32u * 32u;
    const u64 from = (u64)(rank * kSortWarps + warp) * each;
    const unsigned begin = (unsigned)min(from, (u64)a.count), end = (unsigned)min(from + each, (u64)a.count);
    for (unsigned pass = 0; pass < a.passes; ++pass) {
        const unsigned shift = 8u * pass, target = (a.passes - 1u - pass) & 1u;
        const unsigned *keys = a.keys[target ^ 1u], *places = a.places[target ^ 1u];
        for (unsigned b = lane; b < kBins; b += 32u) counts[warp][b] = 0;
        __syncwarp();
        for (unsigned i = begin + lane; i - lane < end; i += 32u) {
            const unsigned bin = i < end ? (pass == 0 ? key_of(a, i) : keys[i]) >> shift & (kBins - 1u) : kBins;
            const unsigned same = __match_any_sync(0xffffffffu, bin);
            if (bin < kBins && (int)lane == __ffs((int)same) - 1) counts[warp][bin] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        // Four threads for a bin, each with eight warps.
        const unsigned bin = threadIdx.x / 4u, part = threadIdx.x & 3u;
        unsigned total = 0;
#pragma unroll
        for (unsigned w = 0; w < kSortWarps / 4; ++w) {
            const unsigned n = counts[part * (kSortWarps / 4) + w][bin];
            counts[part * (kSortWarps / 4) + w][bin] = total;
            total += n;
        }
        unsigned scan = total;  // of this thread's and the parts before
#pragma unroll
        for (unsigned d = 1; d < 4u; d *= 2u) {
            const unsigned v = __shfl_up_sync(0xffffffffu, scan, d, 4);
            scan += part >= d ? v : 0u;
        }
#pragma unroll
        for (unsigned w = 0; w < kSortWarps / 4; ++w) counts[part * (kSortWarps / 4) + w][bin] += scan - total;
        if (part == 3u) totals[bin] = scan;
        cluster_sync();
        unsigned before = 0, all = 0;
        if (threadIdx.x < kBins) {
#pragma unroll
            for (unsigned r = 0; r < kSortCtas; ++r) {
                const unsigned n = load_at_rank(&totals[threadIdx.x], r);
                before += r < rank ? n : 0u;
                all += n;
            }
            scan = all;  // of the bins before, and this one
#pragma unroll
            for (unsigned d = 1; d < 32u; d *= 2u) {
                const unsigned v = __shfl_up_sync(0xffffffffu, scan, d);
                scan += lane >= d ? v : 0u;
            }
            if (lane == 31u) sums[warp] = scan;
        }
        __syncthreads();
        if (threadIdx.x < kBins) {
#pragma unroll
            for (unsigned w = 0; w < kBins / 32; ++w) before += w < warp ? sums[w] : 0u;
            bases[threadIdx.x] = before + scan - all;
        }
        __syncthreads();
        for (unsigned i = begin + lane; i - lane < end; i += 32u) {
            const bool there = i < end;
            const unsigned key = there ? (pass == 0 ? key_of(a, i) : keys[i]) : 0u, place = there && pass != 0 ? places[i] : i;
            const unsigned to = there ? key >> shift & (kBins - 1u) : kBins;
            const unsigned same = __match_any_sync(0xffffffffu, to);
            unsigned at = 0;
            if (there) at = bases[to] + counts[warp][to] + __popc(same & ((1u << lane) - 1u));
            __syncwarp();
            if (there && (int)lane == __ffs((int)same) - 1) counts[warp][to] += __popc(same);
            __syncwarp();
            if (there) {
                a.keys[target][at] = key;
                a.places[target][at] = place;
            }
        }
        cluster_sync();  // the list is whole, and the totals have been read
    }
}

struct FillArgs {
    char* gradient;
    u64 bytes;
};

constexpr unsigned kFillThreads = 512, kFillBytes = 65536;  // of a CTA

// Zeros. It runs beside the sort, on which it does not depend; the first CTA stays until that is done, so that both are over for what comes next.
__global__ void __launch_bounds__(kFillThreads) fill_kernel(const __grid_constant__ FillArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const u64 first = (u64)blockIdx.x * kFillBytes + threadIdx.x * 16u;
#pragma unroll
    for (unsigned i = 0; i < kFillBytes / (16u * kFillThreads); ++i) {
        const u64 at = first + i * (16u * kFillThreads);
        if (at + 16u <= a.bytes) store16_once(a.gradient + at, make_uint4(0u, 0u, 0u, 0u));
        else
            for (u64 b = at; b < a.bytes; ++b) a.gradient[b] = 0;
    }
    if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

struct SumArgs {
    const unsigned* keys;
    const unsigned* places;
    const char* dy;
    long long stride;  // bytes
    char* gradient;
    float* partial;    // [chunks][2][padded]: of the token that a chunk begins with, and of the one it ends with
    unsigned count, vocabulary, chunk, chunks, width, vectors, padded, lanes;
    bool wide, wide_out;
    float scale;
};

template <typename T>
__global__ void __launch_bounds__(128) sum_kernel(const __grid_constant__ SumArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr unsigned kElems = 16 / sizeof(T), kAtOnce = 8;
    const unsigned chunk = blockIdx.x * (128u / a.lanes) + threadIdx.x / a.lanes, vector = blockIdx.y * a.lanes + threadIdx.x % a.lanes;
    if (chunk >= a.chunks || vector >= a.vectors) return;
    const unsigned begin = chunk * a.chunk, end = min(begin + a.chunk, a.count), there = a.width - vector * kElems;
    const unsigned before = begin != 0 ? a.keys[begin - 1] : 0xffffffffu, after = end < a.count ? a.keys[end] : 0xffffffffu;
    unsigned current = a.keys[begin];
    bool first = true;  // the token that the chunk begins with
    float sum[kElems] = {};
    const auto write = [&](bool last) {
        if (current >= a.vocabulary) return;
        const bool from_before = first && current == before, goes_on = last && current == after;
        if (from_before || goes_on) {
            float* to = a.partial + ((u64)chunk * 2u + (from_before ? 0u : 1u)) * a.padded + vector * kElems;
#pragma unroll
            for (unsigned e = 0; e < kElems; e += 4) *reinterpret_cast<float4*>(to + e) = make_float4(sum[e], sum[e + 1], sum[e + 2], sum[e + 3]);
        } else {
            float f[kElems];
#pragma unroll
            for (unsigned e = 0; e < kElems; ++e) f[e] = sum[e] * a.scale;
            store_row16<T>(a.gradient + ((u64)current * a.width + vector * kElems) * sizeof(T), a.wide_out, there, Wide<T>::pack(f));
        }
    };
    for (unsigned i = begin; i < end; i += kAtOnce) {
        unsigned key[kAtOnce];
        uint4 v[kAtOnce];
#pragma unroll
        for (unsigned j = 0; j < kAtOnce; ++j) {
            key[j] = i + j < end ? a.keys[i + j] : 0xffffffffu;
            v[j] = make_uint4(0u, 0u, 0u, 0u);
            if (key[j] < a.vocabulary) v[j] = load_row16<T>(a.dy + (long long)a.places[i + j] * a.stride + (u64)vector * 16u, a.wide, there);
        }
#pragma unroll
        for (unsigned j = 0; j < kAtOnce; ++j) {
            if (i + j >= end) break;
            if (key[j] != current) {
                write(false);
                current = key[j];
                first = false;
#pragma unroll
                for (unsigned e = 0; e < kElems; ++e) sum[e] = 0.0f;
            }
            float f[kElems];
            Wide<T>::unpack(v[j], f);
#pragma unroll
            for (unsigned e = 0; e < kElems; ++e) sum[e] += f[e];
        }
    }
    write(true);
}

struct JoinArgs {
    const unsigned* keys;
    const float* partial;
    char* gradient;
    unsigned count, vocabulary, chunk, width, padded;
    float scale;
};

// The sums of a token whose rows lie in several chunks: the CTAs of the chunk that they begin in, 128 columns at a time, eight warps side by side. (Most CTAs
// find nothing to do: a CTA for every 128 columns of 4096 took 118 us to find that out.)
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ JoinArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned chunk = blockIdx.x, begin = chunk * a.chunk, next = begin + a.chunk;
    if (next >= a.count) return;
    const unsigned token = a.keys[next - 1], behind = a.keys[next], before = chunk != 0 ? a.keys[begin - 1] : 0xffffffffu;
    if (token != behind || token >= a.vocabulary || token == before) return;  // (before: it begins in another chunk)
    unsigned low = next, high = a.count;                   // the first of another token lies in [low, high]
    while (low < high) {
        const unsigned middle = low + (high - low) / 2u;
        if (a.keys[middle] == token) low = middle + 1u;
        else high = middle;
    }
    const unsigned last = (low - 1u) / a.chunk, more = last - chunk;  // chunks behind the first
    const unsigned warp = threadIdx.x / 32u, lane = threadIdx.x & 31u;
    const unsigned from = chunk + 1u + (unsigned)((u64)more * warp / 8u), to = chunk + 1u + (unsigned)((u64)more * (warp + 1u) / 8u);
    __shared__ float4 all[8][32];
    for (unsigned column = blockIdx.y * 128u + lane * 4u; column - lane * 4u < a.padded; column += gridDim.y * 128u) {
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const auto add = [&sum](float4 v) {
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        };
        if (column < a.padded) {
            const float* at = a.partial + column;
            if (warp == 0) add(*reinterpret_cast<const float4*>(at + ((u64)chunk * 2u + 1u) * a.padded));
#pragma unroll 8
            for (unsigned c = from; c < to; ++c) add(*reinterpret_cast<const float4*>(at + (u64)c * 2u * a.padded));
        }
        all[warp][lane] = sum;
        __syncthreads();
        if (warp == 0) {
            for (unsigned w = 1; w < 8; ++w) add(all[w][lane]);
            const float f[4] = {sum.x, sum.y, sum.z, sum.w};
            T* out = reinterpret_cast<T*>(a.gradient) + (u64)token * a.width + column;
#pragma unroll
            for (unsigned e = 0; e < 4; ++e)
                if (column + e < a.width) out[e] = Elem<T>::from_f(f[e] * a.scale);
        }
        __syncthreads();
    }
}

template <typename Args>
struct Kernels {
    void (*of[3])(Args);
    void (*at(DType d) const)(Args) { return of[static_cast<int>(d)]; }
};

unsigned power_of_two(unsigned n, unsigned most) {
    unsigned p = 1;
    while (p < n && p < most) p *= 2;
    return p;
}
bool on16(const void* p, long long bytes, std::size_t rows) { return reinterpret_cast<std::uintptr_t>(p) % 16 == 0 && (rows <= 1 || bytes % 16 == 0); }

// Chunks of the sorted list: enough of them for the whole GPU, and not so many that a token of all rows has more than a few thousand.
unsigned chunk_of(std::size_t count) { return (unsigned)std::max<std::size_t>(8, (count + 2047) / 2048); }

struct Workspace {
    std::size_t keys[2], places[2], partial, bytes;
    unsigned chunk, chunks, padded;
};
Workspace workspace_of(const EmbeddingCall& c) {
    Workspace w;
    std::size_t at = 0;
    const auto take = [&at](std::size_t bytes) {
        const std::size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    for (int i = 0; i < 2; ++i) {
        w.keys[i] = take(c.count * 4);
        w.places[i] = take(c.count * 4);
    }
    w.chunk = chunk_of(c.count);
    w.chunks = (unsigned)((c.count + w.chunk - 1) / w.chunk);
    w.padded = (unsigned)((c.width + 7) / 8 * 8);
    w.partial = take((std::size_t)w.chunks * 2 * w.padded * sizeof(float));
    w.bytes = at;
    return w;
}

}  // namespace

cudaError_t launch_embedding(const EmbeddingCall& c) {
    if (c.count == 0) return cudaSuccess;
    const std::size_t e = dtype_size(c.dtype);
    LookupArgs a;
    a.tokens = c.tokens;
    a.token_stride = c.token_stride;
    a.tokens64 = c.tokens64;
    a.rows = static_cast<const char*>(c.rows);
    a.stride = c.stride * (long long)e;
    a.out = static_cast<char*>(c.out);
    a.count = c.count;
    a.vocabulary = c.vocabulary;
    a.width = (unsigned)c.width;
    a.vectors = (unsigned)((c.width * e + 15) / 16);
    a.lanes = power_of_two((a.vectors + kLookupVectors - 1) / kLookupVectors, 32);
    a.wide = on16(c.rows, a.stride, c.vocabulary) && on16(c.out, (long long)(c.width * e), c.count);
    a.scale = c.scale;
    const std::size_t rows = 256 / a.lanes, ctas = (c.count + rows - 1) / rows, across = (a.vectors + a.lanes * kLookupVectors - 1) / (a.lanes * kLookupVectors);
    B2_REQUIRE(ctas < (1ull << 31) && across < 65536, "too many tokens or columns for one call");
    static constexpr Kernels<LookupArgs> kernels = {{lookup_kernel<float>, lookup_kernel<__half>, lookup_kernel<__nv_bfloat16>}};
    return launch_dependent<LookupArgs>(kernels.at(c.dtype), dim3((unsigned)ctas, (unsigned)across), 256, 0, c.stream, a);
}

std::size_t embedding_workspace(const EmbeddingCall& call) { return call.count == 0 ? 0 : workspace_of(call).bytes; }

cudaError_t launch_embedding_gradient(const EmbeddingCall& c) {
    const std::size_t e = dtype_size(c.dtype), bytes = c.vocabulary * c.width * e;
    if (c.count == 0) return cudaMemsetAsync(c.out, 0, bytes, c.stream);
    const Workspace w = workspace_of(c);
    char* workspace = static_cast<char*>(c.workspace);
    SortArgs s;
    s.tokens = c.tokens;
    s.token_stride = c.token_stride;
    s.tokens64 = c.tokens64;
    s.count = (unsigned)c.count;
    s.vocabulary = (unsigned)c.vocabulary;
    s.passes = 1;
    while (s.passes < 4 && (c.vocabulary >> (8 * s.passes)) != 0) ++s.passes;
    for (int i = 0; i < 2; ++i) {
        s.keys[i] = reinterpret_cast<unsigned*>(workspace + w.keys[i]);
        s.places[i] = reinterpret_cast<unsigned*>(workspace + w.places[i]);
    }
    cudaError_t st = launch_dependent<SortArgs>(sort_kernel, dim3(kSortCtas), kSortThreads, 0, c.stream, s);
    if (st != cudaSuccess) return st;
    FillArgs f;
    f.gradient = static_cast<char*>(c.out);
    f.bytes = bytes;
    const std::size_t ctas = (bytes + kFillBytes - 1) / kFillBytes;
    B2_REQUIRE(ctas < (1ull << 31), "the gradient is too large for one call");
    st = launch_dependent<FillArgs>(fill_kernel, dim3((unsigned)ctas), kFillThreads, 0, c.stream, f);
    if (st != cudaSuccess) return st;
    SumArgs a;
    a.keys = s.keys[0];
    a.places = s.places[0];
    a.dy = static_cast<const char*>(c.rows);
    a.stride = c.stride * (long long)e;
    a.gradient = f.gradient;
    a.partial = reinterpret_cast<float*>(workspace + w.partial);
    a.count = s.count;
    a.vocabulary = s.vocabulary;
    a.chunk = w.chunk;
    a.chunks = w.chunks;
    a.width = (unsigned)c.width;
    a.vectors = (unsigned)((c.width * e + 15) / 16);
    a.padded = w.padded;
    a.lanes = power_of_two(a.vectors, 128);
    a.wide = on16(c.rows, a.stride, c.count);
    a.wide_out = on16(c.out, (long long)(c.width * e), c.vocabulary);
    a.scale = c.scale;
    const unsigned each = 128 / a.lanes, across = (a.vectors + a.lanes - 1) / a.lanes;
    B2_REQUIRE(across < 65536, "too many columns for one call");
    static constexpr Kernels<SumArgs> sums = {{sum_kernel<float>, sum_kernel<__half>, sum_kernel<__nv_bfloat16>}};
    st = launch_dependent<SumArgs>(sums.at(c.dtype), dim3((w.chunks + each - 1) / each, across), 128, 0, c.stream, a);
    if (st != cudaSuccess || w.chunks < 2) return st;
    JoinArgs j;
    j.keys = a.keys;
    j.partial = a.partial;
    j.gradient = f.gradient;
    j.count = s.count;
    j.vocabulary = s.vocabulary;
    j.chunk = w.chunk;
    j.width = a.width;
    j.padded = w.padded;
    j.scale = c.scale;
    static constexpr Kernels<JoinArgs> joins = {{join_kernel<float>, join_kernel<__half>, join_kernel<__nv_bfloat16>}};
    return launch_dependent<JoinArgs>(joins.at(c.dtype), dim3(w.chunks - 1, std::min(4u, (w.padded + 127) / 128)), 256, 0, c.stream, j);
}

}  // namespace b200ccl::kernels
