// MXFP4 weight and activation format: quantise rows of fp32 / bf16 / fp16 and the inverse.  The format is in mxfp4.cuh.
//
// Both are byte movers.  A lane holds eight elements, four lanes a block of 32, so the block's maximum is two shuffles and all
// loads and stores are whole 16-byte vectors; nothing is staged and every byte is touched once.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/feather_b200.h"
#include "host_util.h"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace feather {

constexpr int kMxThreads = 256;

// Eight elements at p; `vector`: p is 16-byte aligned.
template <int kSrc>
__device__ __forceinline__ void mx_load8(const void* p, bool vector, float (&x)[8]) {
    if constexpr (kSrc == FEATHER_SRC_FP32) {
        const float* f = static_cast<const float*>(p);
        if (vector) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(f)), b = __ldg(reinterpret_cast<const float4*>(f) + 1);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __ldg(f + i);
        }
    } else {
        uint32_t w[4];
        const uint16_t* h = static_cast<const uint16_t*>(p);
        if (vector) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(h));
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = static_cast<uint32_t>(__ldg(h + 2 * i)) | (static_cast<uint32_t>(__ldg(h + 2 * i + 1)) << 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack16x2(w[i], kSrc == FEATHER_SRC_BF16, x[2 * i], x[2 * i + 1]);
    }
}

// Block (tx, ty): tx lanes along K (a multiple of 16, so that one scale word's four blocks sit in one half-warp), ty rows.
template <int kSrc>
__global__ void __launch_bounds__(kMxThreads)
mx_quantize_kernel(const void* __restrict__ src, long long rows, int k, long long ld, bool vector, uint8_t* __restrict__ data, uint8_t* __restrict__ scales) {
    constexpr int kSize = kSrc == FEATHER_SRC_FP32 ? 4 : 2;
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();
    const long long row = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    const int vec = blockIdx.y * blockDim.x + threadIdx.x;
    const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31;
    const bool active = row < rows && vec * 8 < k;
    float x[8] = {};
    if (active) mx_load8<kSrc>(static_cast<const uint8_t*>(src) + (row * ld + vec * 8) * kSize, vector, x);
    uint32_t code;
    const uint32_t q = mx_quantize8(x, code);
    const uint32_t word = mx_scale_word(code, lane);
    if (active) {
        reinterpret_cast<uint32_t*>(data)[row * (k / 8) + vec] = q;
        if ((vec & 15) == 0) *reinterpret_cast<uint32_t*>(scales + mx_scale_word_offset(row, vec >> 4, mx_tiles_k(k))) = word;
    }
}

template <int kDst>
__global__ void __launch_bounds__(kMxThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scales, long long rows, int k, void* __restrict__ dst) {
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();
    const long long row = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    const int vec = blockIdx.y * blockDim.x + threadIdx.x;
    if (row >= rows || vec * 8 >= k) return;
    float v[8];
    mx_unpack8(__ldg(reinterpret_cast<const uint32_t*>(data) + row * (k / 8) + vec), v);
    const int block = vec >> 2;
    const float s = mx_scale_value(__ldg(scales + mx_scale_word_offset(row, block >> 2, mx_tiles_k(k)) + (block & 3)));
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

static int mx_check(int64_t rows, int64_t K) {
    if (rows < 0 || K <= 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "rows must not be negative and K must be positive");
    if (K % kMxBlock != 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "MXFP4 rows need K divisible by 32");
    if (rows > 0x7FFFFFFF || K > 0x40000000) return set_error(FEATHER_ERR_BAD_ARGUMENT, "rows must fit in 31 bits and K in 30");
    if (K > 65535LL * 8 * kMxThreads) return set_error(FEATHER_ERR_BAD_ARGUMENT, "K too large for one launch");
    return FEATHER_OK;
}

// (tx, ty) and grid: the narrowest power of two that covers a row's 8-element vectors, at most a whole block
static void mx_grid(int64_t rows, int64_t K, dim3* grid, dim3* block) {
    unsigned tx = 16;
    while (tx < kMxThreads && tx * 8 < K) tx <<= 1;
    const unsigned ty = kMxThreads / tx;
    *block = dim3(tx, ty, 1);
    *grid = dim3(static_cast<unsigned>((rows + ty - 1) / ty), static_cast<unsigned>((K / 8 + tx - 1) / tx), 1);
}

template <typename... Params, typename... Args>
static int mx_launch(const char* what, void (*kernel)(Params...), dim3 grid, dim3 block, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
    if (e != cudaSuccess) return set_error(FEATHER_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    return FEATHER_OK;
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
    dim3 grid, block;
    mx_grid(rows, K, &grid, &block);
    const int k = static_cast<int>(K);
    const long long r = rows, l = ld;
    switch (src_dtype) {
        case FEATHER_SRC_FP32: return mx_launch("mxfp4_quantize", mx_quantize_kernel<FEATHER_SRC_FP32>, grid, block, stream, src, r, k, l, vector, data, scales);
        case FEATHER_SRC_BF16: return mx_launch("mxfp4_quantize", mx_quantize_kernel<FEATHER_SRC_BF16>, grid, block, stream, src, r, k, l, vector, data, scales);
        default: return mx_launch("mxfp4_quantize", mx_quantize_kernel<FEATHER_SRC_FP16>, grid, block, stream, src, r, k, l, vector, data, scales);
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
    dim3 grid, block;
    mx_grid(rows, K, &grid, &block);
    const int k = static_cast<int>(K);
    const long long r = rows;
    switch (dst_dtype) {
        case FEATHER_SRC_FP32: return mx_launch("mxfp4_dequantize", mx_dequantize_kernel<FEATHER_SRC_FP32>, grid, block, stream, data, scales, r, k, dst);
        case FEATHER_SRC_BF16: return mx_launch("mxfp4_dequantize", mx_dequantize_kernel<FEATHER_SRC_BF16>, grid, block, stream, data, scales, r, k, dst);
        default: return mx_launch("mxfp4_dequantize", mx_dequantize_kernel<FEATHER_SRC_FP16>, grid, block, stream, data, scales, r, k, dst);
    }
}
