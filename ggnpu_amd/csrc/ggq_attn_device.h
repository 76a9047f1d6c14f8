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

// ---- operands from the records of a quantized cache

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// A block's scale from its byte.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Under a block's scale, codes of this magnitude and above read back as infinite or NaN: with e the code's exponent bits, an e4m3
// one is 2^(e - 7) or more and below twice that, an e2m1 one (e > 0) 2^(e - 1), both times 2^(byte - 127); 2^128 is infinite.
template <int BITS> __device__ __forceinline__ uint32_t first_not_finite(uint32_t byte) {
    if (byte == 255u) return 0u;
    return BITS == 8 ? min(127u, 8u * (262u - byte)) : 2u * (256u - byte);
}

union Frag {
    uint32_t w[4];
    bf16x8 v;
};

__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float s, int b) {
    bf16x2 r;
    switch (b) {  // the byte is an immediate
    case 0: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0); break;
    case 1: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1); break;
    case 2: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2); break;
    default: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3); break;
    }
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, float s, int half) {
    const bf16x2 r = half ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true)
                          : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false);
    return __builtin_bit_cast(uint32_t, r);
}
// Values 2i and 2i + 1 of a run of codes.
template <int BITS> __device__ __forceinline__ uint32_t pair_of(const uint32_t* w, float s, int i) {
    if constexpr (BITS == 4) return fp4_pair(w[i / 4], s, i % 4);
    else return fp8_pair(w[i / 2], s, i % 2);
}

// Over the four groups of 16 lanes.
__device__ __forceinline__ float rows_max(float v) {
    const Two x = rows16(v), y = halves(max3(x.a, x.b, x.b));
    return max3(y.a, y.b, y.b);
}

__device__ __forceinline__ uint32_t bf16_pack(float a, float b) {  // upper halves
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}

}  // namespace ggq
