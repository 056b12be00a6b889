// Two fp32 numbers in one 64-bit register: sm_100 multiplies and adds both with one instruction.
#pragma once

namespace b200ccl::dev {

struct Pair32 {
    unsigned long long v;
};
__device__ __forceinline__ Pair32 pair32(float a, float b) {
    Pair32 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ Pair32 both32(float a) { return pair32(a, a); }
__device__ __forceinline__ float2 apart(Pair32 p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
    return f;
}
__device__ __forceinline__ Pair32 fma2(Pair32 a, Pair32 b, Pair32 c) {
    Pair32 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Pair32 mul2(Pair32 a, Pair32 b) {
    Pair32 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

__device__ __forceinline__ Pair32 add2(Pair32 a, Pair32 b) {
    Pair32 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

// Wide accesses to what a kernel reads and writes once. They name no memory that they change, so that the compiler keeps a kernel's arguments in
// registers across them: nothing is read here that was written in the same kernel.
__device__ __forceinline__ uint4 load16_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void store16_once(void* p, uint4 v) {
    asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
}

// Hardware approximations: 2^x within 2 units in the last place, 1 / x within 1; subnormal results are zero.
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

}  // namespace b200ccl::dev
