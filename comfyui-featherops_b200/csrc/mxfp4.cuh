// MXFP4 (the OCP microscaling format: E2M1 elements in blocks of 32 along K, one E8M0 scale for each block) on the device:
// what the quantiser and the fused norm share, and the layout of the scales.
//
//   code  = max(0, exponent_bits(amax) - 2)           so that amax / 2^(code - 127) lies in [4, 8): the largest element lands in
//                                                      the top binade of E2M1 (4 and 6); what rounds above 6 saturates to 6
//   q     = round-to-nearest-even of x * 2^(127 - code) to {0, .5, 1, 1.5, 2, 3, 4, 6}
//   value = q * 2^(code - 127); code 255 stands for NaN (a block that held a NaN or an infinity)
//
// Scales are stored in tiles of 128 rows x 4 blocks (512 bytes): the byte of (row, block) is at
//   ((row / 128) * tiles_k + block / 4) * 512 + (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4
// which is the order in which tcgen05.cp puts one tile's scales on the tensor-memory lanes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace feather {

constexpr int kMxBlock = 32;
constexpr int kMxScaleTile = 512;

__host__ __device__ __forceinline__ long long mx_tiles_k(long long k) { return (k + 127) / 128; }
__host__ __device__ __forceinline__ long long mx_scale_bytes(long long rows, long long k) { return (rows + 127) / 128 * mx_tiles_k(k) * kMxScaleTile; }

// Offset of the four scale bytes of blocks 4 * tile_k .. 4 * tile_k + 3 of a row.
__device__ __forceinline__ long long mx_scale_word_offset(long long row, long long tile_k, long long tiles_k) {
    return ((row >> 7) * tiles_k + tile_k) * kMxScaleTile + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// 2^(code - 127); 2^-127 is an fp32 subnormal, code 255 a NaN.
__device__ __forceinline__ float mx_scale_value(uint32_t code) {
    return __uint_as_float(code == 0 ? 0x00400000u : code == 255u ? 0x7FC00000u : code << 23);
}

// Eight fp32 -> eight E2M1 codes, element i in nibble i.
__device__ __forceinline__ uint32_t mx_pack8(const float (&v)[8]) {
    uint32_t out;
    // cvt...x2 d, a, b: a -> upper nibble, b -> lower nibble
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
        "mov.b32 %0, {b0, b1, b2, b3};\n"
        "}\n"
        : "=r"(out)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return out;
}

// Two E2M1 codes of each byte of `w` -> four half2 (exact).
__device__ __forceinline__ void mx_unpack8(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "mov.b32 {b0, b1, b2, b3}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n"
        "}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// Scale code of a block whose largest |x| has these fp32 bits.  As unsigned integers the bits of |x| order like the values, with every
// NaN above infinity.
__device__ __forceinline__ uint32_t mx_code(uint32_t top) {
    const uint32_t exponent = top >> 23;
    return exponent == 255u ? 255u : exponent > 2u ? exponent - 2u : 0u;
}

// Eight values -> codes under a block's scale.
__device__ __forceinline__ uint32_t mx_scaled_pack8(const float (&x)[8], uint32_t code) {
    if (code == 255u) return 0u;
    const float inverse = __uint_as_float((254u - code) << 23);      // 2^(127 - code): a normal number, the product is exact
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i] * inverse;
    return mx_pack8(v);
}

// One block of 32 is held by four neighbouring lanes, eight elements each (lane % 4 = position); every lane of the warp calls
// this, a lane without elements with zeros.  Returns the lane's eight codes; `code` is the block's scale.
__device__ __forceinline__ uint32_t mx_quantize8(const float (&x)[8], uint32_t& code) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    code = mx_code(top);
    return mx_scaled_pack8(x, code);
}

// The scale bytes of the four blocks that 16 neighbouring lanes hold, as one word (the same on all 16).  Lanes beyond the row's
// last block pass 0, which fills the tile up.
__device__ __forceinline__ uint32_t mx_scale_word(uint32_t code, int lane) {
    uint32_t w = code << (8 * ((lane >> 2) & 3));
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
    w |= __shfl_xor_sync(0xffffffffu, w, 8);
    return w;
}

// Element type codes FEATHER_SRC_* at run time: one 16-bit word holds two bf16 or fp16 values.
__device__ __forceinline__ void unpack16x2(uint32_t w, bool bf16, float& lo, float& hi) {
    if (bf16) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xFFFF0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        lo = f.x;
        hi = f.y;
    }
}
__device__ __forceinline__ uint32_t pack16x2(float lo, float hi, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace feather
