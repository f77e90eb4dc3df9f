// dllm_pair.cuh -- two fp32 values in a register pair, for the instructions that work on both, and
// conversions to and from 64 bits.  Both keep subnormal numbers, which the compiler's own operators here
// flush to zero.
#pragma once

#include <cuda_runtime.h>

namespace dllm {

struct Pair {
    unsigned long long v;
    __device__ __forceinline__ Pair() {}
    __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void split(float &a, float &b) const {
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    }
    __device__ __forceinline__ float sum() const {
        float a, b;
        split(a, b);
        return a + b;
    }
};
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y.v) : "l"(a.v), "l"(b.v));
    return y;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y.v) : "l"(a.v), "l"(b.v));
    return y;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return y;
}

__device__ __forceinline__ double wide(float x) {
    double y;
    asm("cvt.f64.f32 %0, %1;" : "=d"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float narrow(double x) {
    float y;
    asm("cvt.rn.f32.f64 %0, %1;" : "=f"(y) : "d"(x));
    return y;
}
__device__ __forceinline__ float narrow_down(double x) {
    float y;
    asm("cvt.rm.f32.f64 %0, %1;" : "=f"(y) : "d"(x));
    return y;
}

}  // namespace dllm
