// ggq_attn_device.h -- device helpers that the attention kernels share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ggq {

// max of three, as one instruction (v_maximum3_f32); fmaxf would quiet each
// operand first.  A NaN wins here.
__device__ __forceinline__ float max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// The two values that lanes l and l ^ 32 (l ^ 16) hold, in both.
struct Two {
    float a, b;
};
__device__ __forceinline__ Two halves(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];  // (a bit_cast of r[1] itself takes r[0])
    return Two{__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ Two rows16(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];
    return Two{__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}

}  // namespace ggq
