// A matrix as TMA reads it: rows of a multiple of eight elements at a multiple of 16 bytes, the last of them padded with zeros. fp32 is cut into three bf16
// matrices whose sum it is, exactly (its 24 bits in eights; of a number below 2^-110 the last of them end under bf16's smallest).
#pragma once

#include "core/check.h"
#include "kernels/sm100/block8.cuh"
#include "kernels/sm100/launch.h"

namespace b200ccl::kernels {

namespace {

using namespace b200ccl::dev;

struct LayOutArgs {
    const char* from;
    long long stride;  // bytes
    char* out;
    unsigned rows, columns;
    Divisor eights;  // of a row
};

// A thread takes eight elements of a row.
template <typename T>
__global__ void __launch_bounds__(256) lay_out_kernel(const __grid_constant__ LayOutArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned eights = a.eights.d, i = blockIdx.x * 256u + threadIdx.x, row = a.eights.divide(i), n = (i - row * eights) * 8u;
    if (row >= a.rows) return;
    const T* at = reinterpret_cast<const T*>(a.from + (long long)row * a.stride) + n;
    unsigned words[2 * sizeof(T)];
    load_any<T, 8>(reinterpret_cast<const char*>(at), n < a.columns ? min(8u, a.columns - n) : 0u, words);
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
        const unsigned long long eight = (unsigned long long)a.rows * eights;
#pragma unroll
        for (int p = 0; p < 3; ++p) *(reinterpret_cast<uint4*>(a.out) + p * eight + i) = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
    }
}

// `stride`: elements from row to row. out: [parts][rows][pitch], pitch a multiple of 8.
template <typename T>
void lay_out(const void* from, long long stride, std::size_t rows, std::size_t columns, std::size_t pitch, void* out, cudaStream_t stream, const char* too_large) {
    LayOutArgs l;
    l.from = static_cast<const char*>(from);
    l.stride = stride * (long long)sizeof(T);
    l.out = static_cast<char*>(out);
    l.rows = (unsigned)rows;
    l.columns = (unsigned)columns;
    l.eights = Divisor((unsigned)(pitch / 8));
    const unsigned long long eights = (unsigned long long)rows * (pitch / 8), ctas = (eights + 255) / 256;
    B2_REQUIRE(eights < (1ull << 31), too_large);
    B2_CUDA(launch_dependent<LayOutArgs>(lay_out_kernel<T>, dim3((unsigned)ctas), 256, 0, stream, l));
}

}  // namespace

}  // namespace b200ccl::kernels
