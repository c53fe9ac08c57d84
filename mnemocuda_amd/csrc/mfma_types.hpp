// mfma_types.hpp -- vectors that matrix instructions take, and int8 values as f16 ones.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mnemo {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// 8 int8 as f16: 0x64uu is 1024 + uu, so with the sign bit flipped and 1152 taken off it is the number.
__device__ __forceinline__ h4 cvt4(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const h2 a = __builtin_bit_cast(h2, lo) - off, b = __builtin_bit_cast(h2, hi) - off;
    return __builtin_shufflevector(a, b, 0, 1, 2, 3);
}
__device__ __forceinline__ h8 cvt8(uint32_t a, uint32_t b) {
    return __builtin_shufflevector(cvt4(a), cvt4(b), 0, 1, 2, 3, 4, 5, 6, 7);
}

// Three parts of 8 bits each that add up to v exactly (as long as the last is no subnormal of bf16): the upper halves of
// what is left.
__device__ __forceinline__ void bf16_parts(const float (&v)[8], b8 (&part)[3]) {
#pragma unroll
    for (int p = 0; p < 3; p++) {
        u4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float lo = v[2 * j], hi = v[2 * j + 1];
#pragma unroll
            for (int i = 0; i < p; i++) {
                lo -= __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, lo) & 0xffff0000u);
                hi -= __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, hi) & 0xffff0000u);
            }
            w[j] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
        }
        part[p] = __builtin_bit_cast(b8, w);
    }
}

}  // namespace mnemo
