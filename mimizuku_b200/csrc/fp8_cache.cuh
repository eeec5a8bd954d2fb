// The stored types of the 8-bit key/value cache: int8 and e4m3 codes, each the rounded quotient of a value and the
// fp32 scale of its block of tokens and head. Shared by kv8.cu and attn8.cu.
#pragma once
#include "common.cuh"

namespace mmz {

enum { KV8_INT8 = 0, KV8_E4M3 = 1 };

// blocks of tokens that share a scale: 16, 32, 64 or 128
__host__ __device__ constexpr bool kv8_block_ok(int block) {
    return block == 16 || block == 32 || block == 64 || block == 128;
}
// the largest code's magnitude: a block's scale is its largest value divided by this
template <int KIND>
__device__ __forceinline__ constexpr float kv8_top() {
    return KIND == KV8_INT8 ? 127.f : 448.f;
}

// two e4m3 values (the low byte first) as two fp16 numbers: every e4m3 number is one of fp16's
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t pair) {
    uint32_t r;
    asm("{\n .reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;\n}\n" : "=r"(r) : "r"(pair));
    return r;
}
// to even, saturating at +-448, NaN kept
__device__ __forceinline__ uint32_t f2_to_e4m3x2(float lo, float hi) {
    uint32_t r;
    asm("{\n .reg .b16 t;\n cvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n cvt.u32.u16 %0, t;\n}\n" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 h2_to_f2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// four codes of a 32-bit word as numbers
template <int KIND>
__device__ __forceinline__ void kv8_load4(uint32_t w, float (&x)[4]) {
    if constexpr (KIND == KV8_INT8) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (float)(int8_t)(w >> (8 * i));
    } else {
        const float2 a = h2_to_f2(e4m3x2_to_h2(w & 0xffff)), b = h2_to_f2(e4m3x2_to_h2(w >> 16));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
}
// The same of numbers known to be finite and within the codes' range. int8: adding 1.5 2^23 rounds to an integer that the
// low byte of the sum holds
template <int KIND>
__device__ __forceinline__ uint32_t kv8_store4_finite(float2 a, float2 b) {
    if constexpr (KIND == KV8_INT8) {
        const float2 magic = make_float2(12582912.f, 12582912.f);
        a = __fadd2_rn(a, magic);
        b = __fadd2_rn(b, magic);
        const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
        return __byte_perm(lo, hi, 0x5410);
    } else {
        return f2_to_e4m3x2(a.x, a.y) | (f2_to_e4m3x2(b.x, b.y) << 16);
    }
}
// four numbers rounded to codes (half to even; int8 clamped to +-127 with NaN as 0, e4m3 saturating with NaN kept)
template <int KIND>
__device__ __forceinline__ uint32_t kv8_store4(const float (&x)[4]) {
    if constexpr (KIND == KV8_INT8) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = max(-127, min(127, __float2int_rn(x[i])));
            w |= (uint32_t)(c & 255) << (8 * i);
        }
        return w;
    } else {
        return f2_to_e4m3x2(x[0], x[1]) | (f2_to_e4m3x2(x[2], x[3]) << 16);
    }
}

}  // namespace mmz
