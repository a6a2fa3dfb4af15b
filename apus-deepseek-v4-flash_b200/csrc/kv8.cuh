// The record of a cache row held in 8 bits (kv8.cu writes and reads it, attn_kv8.cu attends over it).
//
// A row is one latent vector of d channels, key and value at once, shared by all heads.  Its last rd channels (the
// rotated ones) stay BF16, the others are E4M3 codes with one power-of-two scale per 64 channels -- the grouping and the
// rounding of the reference's fp8_qat_sim (c/attn.h:290-369), which the model's rows have been through already, so that
// their values are held exactly:
//
//   [d - rd codes][rd BF16][(d - rd) / 64 UE8M0 bytes, zeros up to a multiple of 16]
//
// d and rd are multiples of 64, so every part starts on a 64-byte multiple and the scales lie in one 16-byte piece.
// Scale byte 255 marks a group that held an infinity or a NaN: all of it reads back as NaN.  Codes 0x7f and 0xff (E4M3's NaN), which
// the writer stores under no other scale, are not looked for and count as +-480: integer instructions bound the readers.
#pragma once
#include "common.cuh"

namespace apus {

constexpr int KV8_GROUP = 64, KV8_MAX_D = 512;

__host__ __device__ __forceinline__ int kv8_scale_off(int d, int rd) { return d + rd; }        // d - rd codes + 2 rd bytes
__host__ __device__ __forceinline__ int kv8_row_bytes(int d, int rd) { return d + rd + 16; }

// d a multiple of 64 up to 512, rd 0 or 64, at least one group of codes (0 = fine, else the message is set)
int kv8_check_row(const char *what, int d, int rd);

// f32 value of a UE8M0 byte, 255 = NaN
__device__ __forceinline__ float kv8_scale(uint32_t b) {
    return b == 255u ? __uint_as_float(0x7fffffffu) : ue8m0_f32(b);
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Four codes -> four BF16 values in the order 0 2 | 1 3, times 2^-120 and the factor in `f` (a BF16 value twice).  Exponent
// and significand move to their places in BF16 (whose bias is 120 larger; a subnormal code becomes a subnormal value) and
// the sign goes into the factor.  The order saves the byte permutations: integer instructions issue every other cycle, and
// they bound this.
__device__ __forceinline__ uint2 codes_bf16x4(uint32_t c, uint32_t f) {
    return make_uint2(mul_bf16x2(c << 4 & 0x07f007f0u, (c << 8 & 0x80008000u) | f), mul_bf16x2(c >> 4 & 0x07f007f0u, (c & 0x80008000u) | f));
}
// 2^120 times the scale of byte b <= 134, twice
__device__ __forceinline__ uint32_t code_factor(uint32_t b) { return b * 0x00800080u + 0x3c003c00u; }
// Two f32 -> two BF16, nearest even, lo in the low half; a NaN stays one whatever its payload is.
__device__ __forceinline__ uint32_t bf16x2_rn(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

}  // namespace apus
