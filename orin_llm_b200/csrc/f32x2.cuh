// Two-wide fp32 arithmetic.
#pragma once

#include <stdint.h>

namespace oattn {

// Pairs of fp32 in one 64-bit register: two-wide add, multiply and fma, each half rounded as the scalar instruction would.
struct F2 {
    unsigned long long v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float x, float y) { asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(x), "f"(y)); }
    __device__ __forceinline__ float x() const { return __uint_as_float((uint32_t)v); }
    __device__ __forceinline__ float y() const { return __uint_as_float((uint32_t)(v >> 32)); }
};
__device__ __forceinline__ F2 operator+(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }

} // namespace oattn
