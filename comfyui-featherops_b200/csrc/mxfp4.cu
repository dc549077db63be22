// MXFP4 weight and activation format: quantise rows of fp32 / bf16 / fp16 and the inverse.  The format is in mxfp4.cuh.
//
// All loads are ordinary ones, without __ldg or __restrict__: a kernel may be resident while the one before it still writes its source, and
// the read-only path asks for memory that nobody writes during the kernel's life.
//
// Both are byte movers.  A lane holds eight elements, four lanes a block of 32 (16 and two for aligned 16-bit sources), so the block's
// maximum is a shuffle or two and all loads and stores are whole vectors; nothing is staged and every byte is touched once.  Rows that do not
// begin on 16 bytes are loaded element by element: 4096 x 13824 bf16 40 us, 13824 x 5120 fp32 77 us (24 and 48 us aligned; bf16 rows on 16
// bytes only, eight elements a lane, 32 us).
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/feather_b200.h"
#include "host_util.h"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace feather {

constexpr int kMxThreads = 256;

// Rows of a thread of the eight-element forms where there are rows enough: loads under way against registers.  One, two, four and eight rows take
// 54, 49, 50, 71 us to quantise 13824 x 5120 fp32 (48 us now, 6.7 TB/s, a copy's rate) and 36, 31, 30, 33 us for 4096 x 13824 bf16 that is aligned to
// 16 bytes only; dequantising 4096 x 13824 to bf16 33, 26, 25, 25 us and 13824 x 5120 to fp32 70, 69, 72, 74 us.  What bounds the last is not the
// memory: a plain fill of its 283 MB takes 40 us, one of the 113 MB of the bf16 case 17 us; 82 % of the issue slots are used.
__host__ __device__ constexpr int mx_many_rows(int type) { return type == FEATHER_SRC_FP32 ? 2 : 4; }

// Eight elements as they lie in memory; 16-bit ones two to a word.  kVector: p is 16-byte aligned.
template <int kSrc>
struct MxRaw {
    uint32_t w[kSrc == FEATHER_SRC_FP32 ? 8 : 4];
};
template <int kSrc, bool kVector>
__device__ __forceinline__ void mx_load8(const void* p, MxRaw<kSrc>& r) {
    constexpr int kWords = kSrc == FEATHER_SRC_FP32 ? 8 : 4;
    if constexpr (kVector) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
            const uint4 a = static_cast<const uint4*>(p)[i];
            r.w[4 * i] = a.x; r.w[4 * i + 1] = a.y; r.w[4 * i + 2] = a.z; r.w[4 * i + 3] = a.w;
        }
    } else if constexpr (kSrc == FEATHER_SRC_FP32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = static_cast<const uint32_t*>(p)[i];
    } else {
        const uint16_t* const h = static_cast<const uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = static_cast<uint32_t>(h[2 * i]) | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
    }
}
template <int kSrc>
__device__ __forceinline__ void mx_values8(const MxRaw<kSrc>& r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kSrc == FEATHER_SRC_FP32) {
            x[2 * i] = __uint_as_float(r.w[2 * i]);
            x[2 * i + 1] = __uint_as_float(r.w[2 * i + 1]);
        } else {
            unpack16x2(r.w[i], kSrc == FEATHER_SRC_BF16, x[2 * i], x[2 * i + 1]);
        }
    }
}

// fp32 bits of the larger of two 16-bit |x|.
template <int kSrc>
__device__ __forceinline__ uint32_t mx_top16(uint32_t pair) {
    const uint32_t top = max(pair >> 16, pair & 0xFFFFu);
    return kSrc == FEATHER_SRC_BF16 ? top << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(top))));
}

// fp32 bits of the largest |x| of the block that four neighbouring lanes hold.  16-bit values are compared as they are, two a word: their
// bits order like the values too.
template <int kSrc>
__device__ __forceinline__ uint32_t mx_block_top(const MxRaw<kSrc>& r) {
    uint32_t top = 0;
    if constexpr (kSrc == FEATHER_SRC_FP32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, r.w[i] & 0x7FFFFFFFu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        return max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) top = __vmaxu2(top, r.w[i] & 0x7FFF7FFFu);
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
        return mx_top16<kSrc>(top);
    }
}

// Block (tx, ty): tx lanes along K (a multiple of 16, so that one scale word's four blocks sit in one half-warp), ty rows; a thread takes
// kRows rows, ty apart, and has all their loads under way at once.
template <int kSrc, int kRows, bool kVector>
__global__ void __launch_bounds__(kMxThreads)
mx_quantize_kernel(const void* src, long long rows, int k, long long ld, uint8_t* data, uint8_t* scales) {
    constexpr int kSize = kSrc == FEATHER_SRC_FP32 ? 4 : 2;
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();
    const long long row0 = static_cast<long long>(blockIdx.x) * (blockDim.y * kRows) + threadIdx.y;
    const int vec = blockIdx.y * blockDim.x + threadIdx.x;
    const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31;
    const bool in = vec * 8 < k;
    MxRaw<kSrc> raw[kRows] = {};
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const long long row = row0 + r * blockDim.y;
        if (in && row < rows) mx_load8<kSrc, kVector>(static_cast<const uint8_t*>(src) + (row * ld + vec * 8) * kSize, raw[r]);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const long long row = row0 + r * blockDim.y;
        const uint32_t code = mx_code(mx_block_top<kSrc>(raw[r]));
        float x[8];
        mx_values8<kSrc>(raw[r], x);
        const uint32_t q = mx_scaled_pack8(x, code);
        const uint32_t word = mx_scale_word(code, lane);
        if (in && row < rows) {
            reinterpret_cast<uint32_t*>(data)[row * (k / 8) + vec] = q;
            if ((vec & 15) == 0) *reinterpret_cast<uint32_t*>(scales + mx_scale_word_offset(row, vec >> 4, mx_tiles_k(k))) = word;
        }
    }
}

// 16-bit sources: a lane holds 16 elements, two lanes a block, so that what a block costs (shuffles, the scale, addresses) is shared by
// twice as many: the instructions bound this, not the bytes.  4096 x 13824 bf16 takes 23.5 us (143 MB, 6.1 TB/s) and 30.2 us with eight a
// lane, 1024 x 5120 3.9 and 4.9 us.  tx is a multiple of 8 (four blocks sit in a quarter-warp); src and its rows are 32-byte aligned.
template <int kSrc>
__global__ void __launch_bounds__(kMxThreads)
mx_quantize16_kernel(const uint16_t* src, long long rows, int k, long long ld, uint8_t* data, uint8_t* scales) {
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();
    const long long row = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    const int vec = blockIdx.y * blockDim.x + threadIdx.x;
    const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31;
    const bool in = vec * 16 < k;
    const uint16_t* const from = src + row * ld + vec * 16;
    uint32_t raw[8] = {};
    if (in && row < rows)
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3]), "=r"(raw[4]), "=r"(raw[5]), "=r"(raw[6]), "=r"(raw[7])
                     : "l"(from)
                     : "memory");
    uint2* const to = reinterpret_cast<uint2*>(data) + row * (k / 16) + vec;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __vmaxu2(top, raw[i] & 0x7FFF7FFFu);
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const uint32_t code = mx_code(mx_top16<kSrc>(top));
    uint32_t q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack16x2(raw[4 * h + i], kSrc == FEATHER_SRC_BF16, x[2 * i], x[2 * i + 1]);
        q[h] = mx_scaled_pack8(x, code);
    }
    uint32_t word = code << (8 * ((lane >> 1) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    if (in && row < rows) {
        *to = make_uint2(q[0], q[1]);
        if ((vec & 7) == 0) *reinterpret_cast<uint32_t*>(scales + mx_scale_word_offset(row, vec >> 3, mx_tiles_k(k))) = word;
    }
}

template <int kDst, int kRows>
__global__ void __launch_bounds__(kMxThreads)
mx_dequantize_kernel(const uint8_t* data, const uint8_t* scales, long long rows, int k, void* dst) {
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();
    const long long row0 = static_cast<long long>(blockIdx.x) * (blockDim.y * kRows) + threadIdx.y;
    const int vec = blockIdx.y * blockDim.x + threadIdx.x;
    if (vec * 8 >= k) return;
    const int block = vec >> 2;
    uint32_t q[kRows], code[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const long long row = row0 + r * blockDim.y;
        if (row < rows) {
            q[r] = reinterpret_cast<const uint32_t*>(data)[row * (k / 8) + vec];
            code[r] = scales[mx_scale_word_offset(row, block >> 2, mx_tiles_k(k)) + (block & 3)];
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const long long row = row0 + r * blockDim.y;
        if (row >= rows) continue;
        float v[8];
        mx_unpack8(q[r], v);
        const float s = mx_scale_value(code[r]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= s;
        const long long at = row * k + vec * 8;
        if constexpr (kDst == FEATHER_SRC_FP32) {
            float4* const o = reinterpret_cast<float4*>(static_cast<float*>(dst) + at);
            o[0] = make_float4(v[0], v[1], v[2], v[3]);
            o[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            constexpr bool kBf16 = kDst == FEATHER_SRC_BF16;
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst) + at) =
                make_uint4(pack16x2(v[0], v[1], kBf16), pack16x2(v[2], v[3], kBf16), pack16x2(v[4], v[5], kBf16), pack16x2(v[6], v[7], kBf16));
        }
    }
}

static int mx_check(int64_t rows, int64_t K) {
    if (rows < 0 || K <= 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "rows must not be negative and K must be positive");
    if (K % kMxBlock != 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "MXFP4 rows need K divisible by 32");
    if (rows > 0x7FFFFFFF || K > 0x40000000) return set_error(FEATHER_ERR_BAD_ARGUMENT, "rows must fit in 31 bits and K in 30");
    if (K > 65535LL * 8 * kMxThreads) return set_error(FEATHER_ERR_BAD_ARGUMENT, "K too large for one launch");
    return FEATHER_OK;
}

// (tx, ty) and grid: the narrowest power of two that covers a row's vectors, at most a whole block, and less where that leaves over a
// sixteenth of the lanes idle (8192 x 5120 bf16: 21.7 -> 17.2 us).  *many: rows enough for threads of many_rows rows, whose grid still
// fills the SMs twice over.
static void mx_grid(int64_t rows, int64_t K, int elements, int many_rows, bool vector, int sms, dim3* grid, dim3* block, bool* many) {
    const int64_t lanes = K / elements;
    unsigned tx = 128 / elements;
    while (tx < kMxThreads && tx < lanes) tx <<= 1;
    while (tx > 32 && ((lanes + tx - 1) / tx * tx - lanes) * 16 > lanes) tx >>= 1;
    const unsigned ty = kMxThreads / tx, along = static_cast<unsigned>((lanes + tx - 1) / tx);
    *many = vector && (rows + ty * many_rows - 1) / (ty * many_rows) * along >= 2 * sms * 8;
    const unsigned step = *many ? ty * many_rows : ty;
    *block = dim3(tx, ty, 1);
    *grid = dim3(static_cast<unsigned>((rows + step - 1) / step), along, 1);
}

template <typename... Params, typename... Args>
static int mx_launch(const char* what, void (*kernel)(Params...), dim3 grid, dim3 block, cudaStream_t stream, const Args&... args) {
    const cudaError_t e = launch_dependent(kernel, grid, block, 0, 0, stream, args...);
    if (e != cudaSuccess) return set_error(FEATHER_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    return FEATHER_OK;
}

template <int kSrc>
static int mx_launch_quantize(bool many, bool vector, dim3 grid, dim3 block, cudaStream_t stream, const void* src, long long rows, int k, long long ld, uint8_t* data, uint8_t* scales) {
    if (!vector) return mx_launch("mxfp4_quantize", mx_quantize_kernel<kSrc, 1, false>, grid, block, stream, src, rows, k, ld, data, scales);
    if (many) return mx_launch("mxfp4_quantize", mx_quantize_kernel<kSrc, mx_many_rows(kSrc), true>, grid, block, stream, src, rows, k, ld, data, scales);
    return mx_launch("mxfp4_quantize", mx_quantize_kernel<kSrc, 1, true>, grid, block, stream, src, rows, k, ld, data, scales);
}

static bool mx_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace feather

using namespace feather;

extern "C" size_t feather_mxfp4_scale_bytes(int64_t rows, int64_t K) {
    if (rows <= 0 || K <= 0) return 0;
    return static_cast<size_t>(mx_scale_bytes(rows, K));
}

extern "C" int feather_mxfp4_quantize(const void* src, int src_dtype, int64_t rows, int64_t K, int64_t ld, uint8_t* data, uint8_t* scales,
                                      feather_stream_t stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (int st = mx_check(rows, K)) return st;
    if (src_dtype != FEATHER_SRC_FP32 && src_dtype != FEATHER_SRC_BF16 && src_dtype != FEATHER_SRC_FP16)
        return set_error(FEATHER_ERR_BAD_ARGUMENT, "src_dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (rows == 0) return FEATHER_OK;
    if (src == nullptr || data == nullptr || scales == nullptr) return set_error(FEATHER_ERR_BAD_ARGUMENT, "src, data and scales must not be null");
    if (rows > 1 && ld < K) return set_error(FEATHER_ERR_BAD_ARGUMENT, "ld must be at least K");
    if (!mx_aligned16(data) || !mx_aligned16(scales)) return set_error(FEATHER_ERR_BAD_ARGUMENT, "data and scales must be 16-byte aligned");
    const int size = src_dtype == FEATHER_SRC_FP32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(src) % size != 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "src must be aligned to its element size");
    const bool vector = mx_aligned16(src) && (rows == 1 || ld * size % 16 == 0);
    const int sms = sm_count();
    if (sms < 1) return set_error(FEATHER_ERR_CUDA, "the number of SMs could not be read");
    dim3 grid, block;
    bool many;
    const int k = static_cast<int>(K);
    const long long r = rows, l = ld;
    if (size == 2 && reinterpret_cast<uintptr_t>(src) % 32 == 0 && (rows == 1 || ld % 16 == 0)) {
        mx_grid(rows, K, 16, 1, true, sms, &grid, &block, &many);
        const uint16_t* const s = static_cast<const uint16_t*>(src);
        return src_dtype == FEATHER_SRC_BF16 ? mx_launch("mxfp4_quantize", mx_quantize16_kernel<FEATHER_SRC_BF16>, grid, block, stream, s, r, k, l, data, scales)
                                             : mx_launch("mxfp4_quantize", mx_quantize16_kernel<FEATHER_SRC_FP16>, grid, block, stream, s, r, k, l, data, scales);
    }
    mx_grid(rows, K, 8, mx_many_rows(src_dtype), vector, sms, &grid, &block, &many);
    switch (src_dtype) {
        case FEATHER_SRC_FP32: return mx_launch_quantize<FEATHER_SRC_FP32>(many, vector, grid, block, stream, src, r, k, l, data, scales);
        case FEATHER_SRC_BF16: return mx_launch_quantize<FEATHER_SRC_BF16>(many, vector, grid, block, stream, src, r, k, l, data, scales);
        default: return mx_launch_quantize<FEATHER_SRC_FP16>(many, vector, grid, block, stream, src, r, k, l, data, scales);
    }
}

extern "C" int feather_mxfp4_dequantize(const uint8_t* data, const uint8_t* scales, int64_t rows, int64_t K, int dst_dtype, void* dst, feather_stream_t stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (int st = mx_check(rows, K)) return st;
    if (dst_dtype != FEATHER_SRC_FP32 && dst_dtype != FEATHER_SRC_BF16 && dst_dtype != FEATHER_SRC_FP16)
        return set_error(FEATHER_ERR_BAD_ARGUMENT, "dst_dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (rows == 0) return FEATHER_OK;
    if (dst == nullptr || data == nullptr || scales == nullptr) return set_error(FEATHER_ERR_BAD_ARGUMENT, "data, scales and dst must not be null");
    if (!mx_aligned16(data) || !mx_aligned16(scales) || !mx_aligned16(dst)) return set_error(FEATHER_ERR_BAD_ARGUMENT, "data, scales and dst must be 16-byte aligned");
    const int sms = sm_count();
    if (sms < 1) return set_error(FEATHER_ERR_CUDA, "the number of SMs could not be read");
    dim3 grid, block;
    bool many;
    mx_grid(rows, K, 8, mx_many_rows(dst_dtype), true, sms, &grid, &block, &many);
    const int k = static_cast<int>(K);
    const long long r = rows;
    switch (dst_dtype) {
        case FEATHER_SRC_FP32: return many ? mx_launch("mxfp4_dequantize", mx_dequantize_kernel<FEATHER_SRC_FP32, mx_many_rows(FEATHER_SRC_FP32)>, grid, block, stream, data, scales, r, k, dst)
                                            : mx_launch("mxfp4_dequantize", mx_dequantize_kernel<FEATHER_SRC_FP32, 1>, grid, block, stream, data, scales, r, k, dst);
        case FEATHER_SRC_BF16: return many ? mx_launch("mxfp4_dequantize", mx_dequantize_kernel<FEATHER_SRC_BF16, mx_many_rows(FEATHER_SRC_BF16)>, grid, block, stream, data, scales, r, k, dst)
                                            : mx_launch("mxfp4_dequantize", mx_dequantize_kernel<FEATHER_SRC_BF16, 1>, grid, block, stream, data, scales, r, k, dst);
        default: return many ? mx_launch("mxfp4_dequantize", mx_dequantize_kernel<FEATHER_SRC_FP16, mx_many_rows(FEATHER_SRC_FP16)>, grid, block, stream, data, scales, r, k, dst)
                                            : mx_launch("mxfp4_dequantize", mx_dequantize_kernel<FEATHER_SRC_FP16, 1>, grid, block, stream, data, scales, r, k, dst);
    }
}
