// The norms before and after a block, its gate and its residual, in one pass over the rows:
//
//   z = y                      or  norm(y) * post_weight
//   r = x + residual_scale * gate * z
//   h = (norm(r) * weight + bias) * (1 + scale) + shift
//   norm(v) = v / sqrt(mean(v^2) + eps)      or  (v - mean(v)) / sqrt(var(v) + eps)
//
// A row lives in the registers of one warp or one block from its only read to its only write; sums are fp32, over the values as
// they are before r is rounded to x's type.  The variance is taken about the mean in a second pass over the registers.  h leaves in
// 16 or 32 bits or, rounded to 16 bits first, as the MXFP4 operand of the product that follows (mxfp4.cuh).
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/feather_b200.h"
#include "host_util.h"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace feather {

// V consecutive elements as they lie in memory: 16-bit elements two to a word.
template <int V, bool F32>
struct Raw {
    uint32_t w[F32 ? V : (V + 1) / 2];
};

template <int V, bool F32>
__device__ __forceinline__ Raw<V, F32> raw_load(const void* base, long long at) {
    Raw<V, F32> r;
    if constexpr (V == 8) {
        if constexpr (F32) {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + at);
            const uint4 a = __ldg(p), b = __ldg(p + 1);
            r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
            r.w[4] = b.x; r.w[5] = b.y; r.w[6] = b.z; r.w[7] = b.w;
        } else {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at));
            r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
        }
    } else {
        static_assert(V == 1, "eight elements or one");
        if constexpr (F32) r.w[0] = __ldg(static_cast<const uint32_t*>(base) + at);
        else r.w[0] = __ldg(static_cast<const uint16_t*>(base) + at);
    }
    return r;
}

template <int V, bool F32>
__device__ __forceinline__ void raw_values(const Raw<V, F32>& r, bool bf16, float (&v)[V]) {
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = __uint_as_float(r.w[i]);
    } else if constexpr (V == 1) {
        float unused;
        unpack16x2(r.w[0], bf16, v[0], unused);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) unpack16x2(r.w[i], bf16, v[2 * i], v[2 * i + 1]);
    }
}

template <int V>
__device__ __forceinline__ void load_values(const void* base, int dtype, long long at, float (&v)[V]) {
    if (dtype == FEATHER_SRC_FP32) raw_values<V, true>(raw_load<V, true>(base, at), false, v);
    else raw_values<V, false>(raw_load<V, false>(base, at), dtype == FEATHER_SRC_BF16, v);
}

template <int V>
__device__ __forceinline__ void store_values(void* base, int dtype, long long at, const float (&v)[V]) {
    if (dtype == FEATHER_SRC_FP32) {
        float* const o = static_cast<float*>(base) + at;
        if constexpr (V == 8) {
            reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *o = v[0];
        }
    } else {
        const bool bf16 = dtype == FEATHER_SRC_BF16;
        uint16_t* const o = static_cast<uint16_t*>(base) + at;
        if constexpr (V == 8)
            *reinterpret_cast<uint4*>(o) = make_uint4(pack16x2(v[0], v[1], bf16), pack16x2(v[2], v[3], bf16), pack16x2(v[4], v[5], bf16), pack16x2(v[6], v[7], bf16));
        else
            *o = static_cast<uint16_t>(pack16x2(v[0], 0.0f, bf16) & 0xFFFFu);
    }
}

struct NormParams {
    feather_norm_args a;
    int vecs;             // vectors of a row
    float inv_cols;
};

// Sum over the row's threads: one warp (WARP_ROW), or the whole block through `part` (a buffer of its own for each call, so that one
// barrier is enough).
template <bool WARP_ROW>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (!WARP_ROW) {
        const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        if (lane == 0) part[threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < warps ? part[lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// Scales the row's values in place to norm(v); `part`: 2 x 32 floats.
template <int V, int NV, bool WARP_ROW>
__device__ __forceinline__ void normalise(float (&v)[NV][V], const NormParams& p, int first, int step, float* part) {
    if (p.a.kind == FEATHER_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[i][j];                         // vectors past the row hold zeros
        const float mean = row_sum<WARP_ROW>(s, part) * p.inv_cols;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (first + i * step < p.vecs) {
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] -= mean;
            }
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) s += v[i][j] * v[i][j];
    const float inv = 1.0f / sqrtf(row_sum<WARP_ROW>(s, part + 32) * p.inv_cols + p.a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] *= inv;
}

template <int V, int NV, bool WARP_ROW, bool XF32, bool YF32>
__global__ void __launch_bounds__(WARP_ROW ? 256 : (NV == 1 ? 1024 : (V == 1 ? 1024 : 512))) gated_norm_kernel(const NormParams p) {
    __shared__ float part[4][32];
    const feather_norm_args& a = p.a;
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();
    const long long row = WARP_ROW ? blockIdx.x * 8LL + (threadIdx.x >> 5) : static_cast<long long>(blockIdx.x);
    const int lane = threadIdx.x & 31;
    const int first = WARP_ROW ? lane : static_cast<int>(threadIdx.x);
    const int step = WARP_ROW ? 32 : static_cast<int>(blockDim.x);
    if (row >= a.rows) return;                                                // a whole warp or a whole block
    const bool xbf = a.x_dtype == FEATHER_SRC_BF16, ybf = a.y_dtype == FEATHER_SRC_BF16;

    Raw<V, XF32> xr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (first + i * step < p.vecs) xr[i] = raw_load<V, XF32>(a.x, row * a.ldx + (first + i * step) * V);
    float v[NV][V];
    if (a.y != nullptr) {
        Raw<V, YF32> yr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (first + i * step < p.vecs) yr[i] = raw_load<V, YF32>(a.y, row * a.ldy + (first + i * step) * V);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (first + i * step < p.vecs) {
                raw_values<V, YF32>(yr[i], ybf, v[i]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] = 0.0f;
            }
        }
        if (a.post_norm) normalise<V, NV, WARP_ROW>(v, p, first, step, part[0]);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (first + i * step) * V;
            if (first + i * step >= p.vecs) continue;
            float m[V];
            if (a.post_weight != nullptr) {
                load_values<V>(a.post_weight, a.post_weight_dtype, at, m);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] *= m[j];
            }
            if (a.gate != nullptr) {
                load_values<V>(a.gate, a.gate_dtype, row / a.gate_rows * a.gate_ld + at, m);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] *= m[j];
            }
            raw_values<V, XF32>(xr[i], xbf, m);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] = m[j] + a.residual_scale * v[i][j];
            if (a.r != nullptr) store_values<V>(a.r, a.x_dtype, row * a.ldr + at, v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (first + i * step < p.vecs) {
                raw_values<V, XF32>(xr[i], xbf, v[i]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] = 0.0f;
            }
        }
    }
    if (a.h == nullptr) return;
    normalise<V, NV, WARP_ROW>(v, p, first, step, part[2]);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int vec = first + i * step;
        const int at = vec * V;
        if (vec < p.vecs) {
            float m[V];
            if (a.weight != nullptr) {
                load_values<V>(a.weight, a.weight_dtype, at, m);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] *= m[j];
            }
            if (a.bias != nullptr) {
                load_values<V>(a.bias, a.bias_dtype, at, m);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] += m[j];
            }
            if (a.scale != nullptr) {
                load_values<V>(a.scale, a.scale_dtype, row / a.scale_rows * a.scale_ld + at, m);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] *= 1.0f + m[j];
            }
            if (a.shift != nullptr) {
                load_values<V>(a.shift, a.shift_dtype, row / a.shift_rows * a.shift_ld + at, m);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] += m[j];
            }
        }
        if constexpr (V == 8) {
            if (a.h_scales != nullptr) {
                // the 16-bit value first, so that the bits are those of quantising the h this call would store
                const bool bf16 = a.h_dtype == FEATHER_SRC_BF16;
#pragma unroll
                for (int j = 0; j < V; j += 2) unpack16x2(pack16x2(v[i][j], v[i][j + 1], bf16), bf16, v[i][j], v[i][j + 1]);
                uint32_t code;
                const uint32_t q = mx_quantize8(v[i], code);
                const uint32_t word = mx_scale_word(code, lane);
                if (vec < p.vecs) {
                    static_cast<uint32_t*>(a.h)[row * a.ldh + vec] = q;
                    if ((vec & 15) == 0) *reinterpret_cast<uint32_t*>(a.h_scales + mx_scale_word_offset(row, vec >> 4, mx_tiles_k(a.cols))) = word;
                }
                continue;
            }
        }
        if (vec < p.vecs) store_values<V>(a.h, a.h_dtype, row * a.ldh + at, v[i]);
    }
}

template <int V, int NV, bool WARP_ROW>
static cudaError_t norm_launch(const NormParams& p, int threads, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(WARP_ROW ? (p.a.rows + 7) / 8 : p.a.rows), 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(WARP_ROW ? 256 : threads), 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool xf = p.a.x_dtype == FEATHER_SRC_FP32, yf = p.a.y != nullptr && p.a.y_dtype == FEATHER_SRC_FP32;
    if (xf) return yf ? cudaLaunchKernelEx(&cfg, gated_norm_kernel<V, NV, WARP_ROW, true, true>, p) : cudaLaunchKernelEx(&cfg, gated_norm_kernel<V, NV, WARP_ROW, true, false>, p);
    return yf ? cudaLaunchKernelEx(&cfg, gated_norm_kernel<V, NV, WARP_ROW, false, true>, p) : cudaLaunchKernelEx(&cfg, gated_norm_kernel<V, NV, WARP_ROW, false, false>, p);
}

static bool norm_dtype_ok(int d) { return d == FEATHER_SRC_FP32 || d == FEATHER_SRC_BF16 || d == FEATHER_SRC_FP16; }
static int norm_size(int d) { return d == FEATHER_SRC_FP32 ? 4 : 2; }

// A [rows, cols] operand: type, alignment to its elements, row pitch; clears `vector` when its rows are not 16-byte aligned.
static bool norm_operand(const void* p, int dtype, int64_t ld, int64_t rows, int64_t cols, bool* vector) {
    if (p == nullptr) return true;
    if (!norm_dtype_ok(dtype) || reinterpret_cast<uintptr_t>(p) % norm_size(dtype) != 0 || (rows > 1 && ld < cols)) return false;
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0 || (rows > 1 && ld * norm_size(dtype) % 16 != 0)) *vector = false;
    return true;
}

constexpr int64_t kNormMaxCols = 16384;

}  // namespace feather

using namespace feather;

extern "C" int feather_gated_norm(const feather_norm_args* args_host, feather_stream_t stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (args_host == nullptr) return set_error(FEATHER_ERR_BAD_ARGUMENT, "args_host must not be null");
    NormParams p{};
    p.a = *args_host;
    feather_norm_args& a = p.a;
    if (a.rows < 0 || a.cols <= 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "rows must not be negative and cols must be positive");
    if (a.cols > kNormMaxCols) return set_error(FEATHER_ERR_UNSUPPORTED, "the fused norm takes rows of at most 16384 elements");
    if (a.rows > 0x7FFFFFFF) return set_error(FEATHER_ERR_BAD_ARGUMENT, "rows must fit in 31 bits");
    if (a.kind != FEATHER_NORM_RMS && a.kind != FEATHER_NORM_LAYER) return set_error(FEATHER_ERR_BAD_ARGUMENT, "kind must be 0 (rms) or 1 (layer)");
    if (a.rows == 0) return FEATHER_OK;
    if (a.x == nullptr || (a.r == nullptr && a.h == nullptr)) return set_error(FEATHER_ERR_BAD_ARGUMENT, "x and at least one of r and h must not be null");
    if (a.y == nullptr && (a.r != nullptr || a.gate != nullptr || a.post_norm != 0 || a.post_weight != nullptr))
        return set_error(FEATHER_ERR_BAD_ARGUMENT, "r, gate and the norm after the block need y");
    if (a.post_weight != nullptr && a.post_norm == 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "post_weight needs post_norm");
    const bool packed = a.h != nullptr && a.h_scales != nullptr;
    if ((a.gate != nullptr && a.gate_rows <= 0) || (a.scale != nullptr && a.scale_rows <= 0) || (a.shift != nullptr && a.shift_rows <= 0))
        return set_error(FEATHER_ERR_BAD_ARGUMENT, "gate_rows, scale_rows and shift_rows must be positive");
    bool vector = a.cols % 8 == 0;
    bool ok = norm_operand(a.x, a.x_dtype, a.ldx, a.rows, a.cols, &vector) && norm_operand(a.y, a.y_dtype, a.ldy, a.rows, a.cols, &vector) &&
              norm_operand(a.r, a.x_dtype, a.ldr, a.rows, a.cols, &vector) && norm_operand(a.weight, a.weight_dtype, 0, 1, a.cols, &vector) &&
              norm_operand(a.bias, a.bias_dtype, 0, 1, a.cols, &vector) && norm_operand(a.post_weight, a.post_weight_dtype, 0, 1, a.cols, &vector);
    ok = ok && norm_operand(a.gate, a.gate_dtype, a.gate_ld, a.gate ? (a.rows - 1) / a.gate_rows + 1 : 1, a.cols, &vector) &&
         norm_operand(a.scale, a.scale_dtype, a.scale_ld, a.scale ? (a.rows - 1) / a.scale_rows + 1 : 1, a.cols, &vector) &&
         norm_operand(a.shift, a.shift_dtype, a.shift_ld, a.shift ? (a.rows - 1) / a.shift_rows + 1 : 1, a.cols, &vector);
    if (!packed) ok = ok && norm_operand(a.h, a.h_dtype, a.ldh, a.rows, a.cols, &vector);
    if (!ok) return set_error(FEATHER_ERR_BAD_ARGUMENT, "an operand has an unknown type, a misaligned pointer or a row pitch below cols");
    if (packed) {
        if (a.cols % kMxBlock != 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "MXFP4 rows need cols divisible by 32");
        if (a.h_dtype != FEATHER_SRC_BF16 && a.h_dtype != FEATHER_SRC_FP16)
            return set_error(FEATHER_ERR_BAD_ARGUMENT, "an MXFP4 h is rounded to h_dtype first: 1 (bf16) or 2 (fp16)");
        if ((reinterpret_cast<uintptr_t>(a.h) & 15u) != 0 || (reinterpret_cast<uintptr_t>(a.h_scales) & 15u) != 0)
            return set_error(FEATHER_ERR_BAD_ARGUMENT, "an MXFP4 h and its scales must be 16-byte aligned");
        if (!vector) return set_error(FEATHER_ERR_BAD_ARGUMENT, "an MXFP4 h needs every operand's rows 16-byte aligned");
        a.ldh = a.cols / 8;                                                    // 32-bit words of a packed row
    }
    p.inv_cols = 1.0f / static_cast<float>(a.cols);
    p.vecs = static_cast<int>(vector ? a.cols / 8 : a.cols);
    cudaError_t e;
    const auto threads = [&](int nv) { return (p.vecs + 32 * nv - 1) / (32 * nv) * 32; };
    if (vector) {
        if (p.vecs <= 32) e = norm_launch<8, 1, true>(p, 0, stream);
        else if (p.vecs <= 128) e = norm_launch<8, 4, true>(p, 0, stream);
        else if (p.vecs <= 1024 && a.rows <= 296) e = norm_launch<8, 1, false>(p, threads(1), stream);
        else e = norm_launch<8, 4, false>(p, threads(4), stream);
    } else {
        if (p.vecs <= 128) e = norm_launch<1, 4, true>(p, 0, stream);
        else if (p.vecs <= 4096) e = norm_launch<1, 4, false>(p, threads(4), stream);
        else e = norm_launch<1, 16, false>(p, threads(16), stream);
    }
    if (e != cudaSuccess) return set_error(FEATHER_ERR_CUDA, "gated_norm launch failed: %s", cudaGetErrorString(e));
    return FEATHER_OK;
}
