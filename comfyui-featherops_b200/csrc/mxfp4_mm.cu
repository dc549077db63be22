// MXFP4 activations @ MXFP4 weights -> fp16 / bf16, fp32 accumulate, for sm_100a:
//
//   c[m, n] = round( sum_k a[m, k] b[n, k] + bias[n] )      a, b: E2M1 elements times the E8M0 scale of their block of 32
//
// The tensor core multiplies the 4-bit operands as they are (tcgen05.mma kind::mxf4, block_scale): both operands sit in shared
// memory as packed bytes (128-byte rows = 256 elements, 128-byte swizzle), their scales in tensor memory, the accumulator in
// tensor memory.
//
//   out^T tile [128 weight columns n  x  TN tokens]  +=  B[128 n x 64 k] * A^T[64 k x TN tokens]
//
//   producer warp   TMA: 128 weight rows and TN token rows of 256 k each; bulk copies: their scale tiles (512 bytes for 128 rows x 128 k)
//   MMA warp        tcgen05.cp puts a stage's scales on the lanes, four tcgen05.mma (64 k each) consume the stage
//   epilogue warps  tcgen05.ld -> + bias -> one rounding -> store
//
// A cluster splits K: rank r of S takes every stage of its share, parks its fp32 tile in its own shared memory, and sums TN / S of
// the tile's token columns over all ranks in rank order (distributed shared memory).  No workspace, no atomics, the same bits on every run.
//
// Every wait is bounded (ptx.cuh); on expiry the CTA records a code in *status, drains and returns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <mutex>

#include "../../include/feather_b200.h"
#include "host_util.h"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace feather {

constexpr int kMxStageK = 256;                      // k per stage: one 128-byte row of packed elements
constexpr int kMxRowBytes = kMxStageK / 2;
constexpr int kMxTilesPerStage = kMxStageK / 128;   // scale tiles along K

enum { kMxRoleProducer = 1, kMxRoleMma = 2, kMxRoleEpilogue = 4 };   // bits 8..15 of the status word, as scaled_mm_kernel's

__device__ __forceinline__ void mx_give_up(int* status, volatile int* abort_flag, int role, int detail) {
    *abort_flag = 1;
    if (status != nullptr) atomicCAS(status, 0, FEATHER_ERR_DEVICE_TIMEOUT | (role << 8) | ((detail & 0xFFFF) << 16));
}

// ------------------------------------------------------------------------------------------------ PTX of the block-scaled path
// Contiguous bytes global -> shared (both 16-byte aligned, size a multiple of 16), completion on an mbarrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// 32 rows x 16 bytes of shared memory -> 32 lanes x 4 columns of tensor memory, repeated in all four lane quarters.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D[tmem] (+)= A[smem] * B[smem], E2M1 operands with an E8M0 scale for every 32 elements (two for the 64 k of one instruction).
__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n"
        "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
        : "memory");
}

// Shared-memory descriptor without a swizzle: 8 rows x 16 bytes contiguous, 8-row groups 128 bytes apart (a scale tile).
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>(128 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    return d;
}

// Instruction descriptor of kind::mxf4: E2M1 x E2M1, E8M0 scales, both operands K-major.  sf: which two of a scale word's four bytes
// (0 or 2) belong to the instruction's 64 k, the same for A and B.
__host__ __device__ constexpr uint32_t umma_idesc_mxf4(uint32_t m, uint32_t n, uint32_t sf) {
    return (sf << 4)             // scale data ID of B
           | (1u << 7)           // A: E2M1
           | (1u << 10)          // B: E2M1
           | ((n >> 3) << 17)    // N
           | (1u << 23)          // scales: E8M0
           | ((m >> 4) << 24)    // M (bits 27..28 hold m / 128)
           | (sf << 29);         // scale data ID of A
}

struct MxMmParams {
    const uint8_t* a_scales;
    const uint8_t* b_scales;
    const uint16_t* bias;
    uint16_t* c;
    int* status;
    long long ldc;
    int M, N, K;
    int out_bf16;
    int tiles_n;
    int stages_total;     // ceil(K / 256)
    int tiles_k;          // ceil(K / 128): scale tiles along K
};

__device__ __forceinline__ float load16(const uint16_t* p, bool bf16) {
    const uint16_t v = __ldg(p);
    return bf16 ? __uint_as_float(static_cast<uint32_t>(v) << 16) : __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ uint16_t round16(float v, bool bf16) { return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v)); }

constexpr int kMxRows = 128;                        // weight rows of a tile: the lanes
constexpr int kMxMmThreads = 192;                   // producer warp, MMA warp, four epilogue warps

template <int TN>
struct MxCfg {
    static_assert(TN == 16 || TN == 32 || TN == 64 || TN == 128, "tokens of a tile");
    static constexpr int kWBytes = kMxRows * kMxRowBytes;
    static constexpr int kTBytes = TN * kMxRowBytes;
    static constexpr int kSfBytes = kMxTilesPerStage * kMxScaleTile;       // scales of up to 128 rows
    static constexpr int kStageBytes = kWBytes + kTBytes + 2 * kSfBytes;
    static constexpr int kStages = TN == 128 ? 5 : 4;
    static constexpr int kSfCols = 2 * kMxTilesPerStage * 4;               // tensor-memory columns of a stage's scales
    static constexpr int kAccCols = TN < 32 ? 32 : TN;
    static constexpr int kTmemCols = kAccCols + kStages * kSfCols <= 128 ? 128 : 256;
    static constexpr int kPartialBytes = TN * kMxRows * 4;                 // the fp32 tile of a K split, in the stages' place
    static_assert(kPartialBytes <= kStages * kStageBytes, "partial tile");
    static constexpr int kBarBytes = 256;
    static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kBarBytes;
};

template <int TN>
__global__ void __launch_bounds__(kMxMmThreads) mx_mm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_t, const MxMmParams p,
                                                             const int splits) {
    using C = MxCfg<TN>;
    constexpr int kStages = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const base_gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bar_base = base + kStages * C::kStageBytes;
    const uint32_t bar_full = bar_base, bar_empty = bar_base + 8 * kStages, bar_acc = bar_base + 16 * kStages;
    uint8_t* const words = base_gen + kStages * C::kStageBytes + 16 * kStages + 8;
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(words);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(words + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % splits;                                   // position in the cluster
    const int tile = blockIdx.x / splits;
    const int n0 = (tile % p.tiles_n) * kMxRows;
    const int t0 = (tile / p.tiles_n) * TN;
    const int per = p.stages_total / splits, extra = p.stages_total % splits;
    const int begin = rank * per + (rank < extra ? rank : extra);
    const int count = per + (rank < extra ? 1 : 0);                          // at least 1: the host takes no more splits than stages

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        mbar_init(bar_acc, 1);
        *abort_flag = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_t);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_slot)), C::kTmemCols);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();

    if (warp == 0) {
        if (lane == 0) {
            int issued = 0;
            bool ok = true;
            for (int i = 0; i < count; ++i) {
                const int s = i % kStages;
                if (!mbar_wait(bar_empty + 8 * s, ((i / kStages) & 1) ^ 1, abort_flag)) {
                    mx_give_up(p.status, abort_flag, kMxRoleProducer, s);
                    ok = false;
                    break;
                }
                const int kt = (begin + i) * kMxTilesPerStage;
                const uint32_t sf_bytes = min(kMxTilesPerStage, p.tiles_k - kt) * kMxScaleTile;
                const uint32_t w = base + s * C::kStageBytes, t = w + C::kWBytes, sfw = t + C::kTBytes, sft = sfw + C::kSfBytes;
                mbar_arrive_expect_tx(bar_full + 8 * s, C::kWBytes + C::kTBytes + 2 * sf_bytes);
                tma_load_2d(w, &tmap_w, bar_full + 8 * s, (begin + i) * kMxRowBytes, n0);
                tma_load_2d(t, &tmap_t, bar_full + 8 * s, (begin + i) * kMxRowBytes, t0);
                bulk_load(sfw, p.b_scales + (static_cast<long long>(n0 / 128) * p.tiles_k + kt) * kMxScaleTile, sf_bytes, bar_full + 8 * s);
                bulk_load(sft, p.a_scales + (static_cast<long long>(t0 / 128) * p.tiles_k + kt) * kMxScaleTile, sf_bytes, bar_full + 8 * s);
                ++issued;
            }
            if (!ok) {
                // the copies in flight land before the CTA's shared memory is given back
                const uint64_t begin_ns = globaltimer_ns();
                for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
                    while (!mbar_try_wait(bar_full + 8 * (i % kStages), (i / kStages) & 1) && globaltimer_ns() - begin_ns < kWaitLimitNs) {
                    }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            for (int i = 0; i < count; ++i) {
                const int s = i % kStages;
                if (!mbar_wait(bar_full + 8 * s, (i / kStages) & 1, abort_flag)) {
                    mx_give_up(p.status, abort_flag, kMxRoleMma, s);
                    break;
                }
                tc_fence_after();
                const uint32_t w = base + s * C::kStageBytes, t = w + C::kWBytes, sfw = t + C::kTBytes, sft = sfw + C::kSfBytes;
                const uint32_t sf_col = tmem + C::kAccCols + s * C::kSfCols;
                const int k_left = p.K - (begin + i) * kMxStageK;
                const int tiles = k_left > 128 ? 2 : 1;
                for (int j = 0; j < tiles; ++j) {
                    tmem_cp_scales(sf_col + 4 * j, smem_desc_scales(sfw + j * kMxScaleTile));
                    tmem_cp_scales(sf_col + 4 * (kMxTilesPerStage + j), smem_desc_scales(sft + j * kMxScaleTile));
                }
                const uint64_t wd = umma_desc_kmajor_sw128(w), td = umma_desc_kmajor_sw128(t);
                const int steps = k_left >= kMxStageK ? 4 : (k_left + 63) / 64;
                for (int j = 0; j < steps; ++j)
                    umma_mxf4(tmem, wd + 2 * j, td + 2 * j, umma_idesc_mxf4(kMxRows, TN, (j & 1) * 2), sf_col + 4 * (j >> 1), sf_col + 4 * (kMxTilesPerStage + (j >> 1)),
                              (i | j) != 0);
                umma_commit_1cta(bar_empty + 8 * s);
            }
            umma_commit_1cta(bar_acc);
        }
        __syncwarp();
    }
    // everybody: the tile is complete (or given up) before it is read and before shared or tensor memory is given back
    const bool ok = mbar_wait(bar_acc, 0, abort_flag);
    if (!ok && lane == 0) mx_give_up(p.status, abort_flag, kMxRoleEpilogue, warp);
    __syncthreads();
    tc_fence_after();
    const bool bf16 = p.out_bf16 != 0;
    const int q = warp & 3;                                                  // lane quarter of tensor memory this warp may read
    const int row = q * 32 + lane;
    const int n = n0 + row;
    const float bias = (warp >= 2 && n < p.N && p.bias != nullptr) ? load16(p.bias + n, bf16) : 0.0f;
    constexpr int kCols = 16;
    if (splits == 1) {
        if (warp >= 2) {
#pragma unroll 1
            for (int c = 0; c < TN; c += kCols) {
                uint32_t v[kCols];
                tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(q * 32) << 16) + c, v);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < kCols; ++j)
                    if (t0 + c + j < p.M && n < p.N) p.c[(t0 + c + j) * p.ldc + n] = round16(__uint_as_float(v[j]) + bias, bf16);
            }
        }
    } else {
        float* const partial = reinterpret_cast<float*>(base_gen);
        if (warp >= 2) {
#pragma unroll 1
            for (int c = 0; c < TN; c += kCols) {
                uint32_t v[kCols];
                tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(q * 32) << 16) + c, v);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < kCols; ++j) partial[(c + j) * kMxRows + row] = __uint_as_float(v[j]);
            }
        }
        cluster_arrive_release();
        cluster_wait_acquire();
        if (warp >= 2) {
            const int cols = TN / splits, c0 = rank * cols;                  // TN is a multiple of the splits
            for (int j = 0; j < cols; ++j) {
                float sum = 0.0f;
                for (int r = 0; r < splits; ++r) {
                    float x;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(mapa_u32(base + static_cast<uint32_t>(((c0 + j) * kMxRows + row) * 4), r)) : "memory");
                    sum += x;
                }
                if (t0 + c0 + j < p.M && n < p.N) p.c[(t0 + c0 + j) * p.ldc + n] = round16(sum + bias, bf16);
            }
        }
        cluster_arrive_release();                                            // no rank leaves while another still reads its tile
        cluster_wait_acquire();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem, C::kTmemCols);
    }
}

// ================================================================================================
// Host side
// ================================================================================================
typedef CUresult (*MxEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                               CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static MxEncodeFn mx_encode_fn() {
    static MxEncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<MxEncodeFn>(f);
    }();
    return fn;
}

// [rows, row_bytes] bytes, box of 128 bytes x box_rows, 128-byte swizzle; what lies outside reads as zero.
static CUresult mx_operand_map(MxEncodeFn encode, CUtensorMap* out, const void* ptr, int64_t rows, int64_t row_bytes, int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
    const cuuint32_t box[2] = {kMxRowBytes, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t step[2] = {1, 1};
    return encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

template <int TN>
static cudaError_t mx_launch_mm(const CUtensorMap& tw, const CUtensorMap& tt, const MxMmParams& p, int splits, long long ctas, cudaStream_t stream) {
    using C = MxCfg<TN>;
    static std::mutex mu;
    static bool configured[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!configured[dev]) {
            e = cudaFuncSetAttribute(mx_mm_kernel<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
            if (e != cudaSuccess) return e;
            configured[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
    cfg.blockDim = dim3(kMxMmThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, mx_mm_kernel<TN>, tw, tt, p, splits);
}

}  // namespace feather

using namespace feather;

extern "C" int feather_mxfp4_mm(const uint8_t* a, const uint8_t* a_scales, const uint8_t* b, const uint8_t* b_scales, const void* bias, void* c, int64_t M, int64_t N,
                                int64_t K, int64_t ldc, int output_dtype, int* status_dev, feather_stream_t stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (M < 0 || N <= 0 || K <= 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "M must not be negative, N and K must be positive");
    if (K % kMxBlock != 0) return set_error(FEATHER_ERR_BAD_ARGUMENT, "MXFP4 rows need K divisible by 32");
    if (M > 0x3FFFFFFF || N > 0x3FFFFFFF || K > 0x3FFFFFFF) return set_error(FEATHER_ERR_BAD_ARGUMENT, "M, N and K must fit in 30 bits");
    if (output_dtype != FEATHER_OUT_FP16 && output_dtype != FEATHER_OUT_BF16) return set_error(FEATHER_ERR_BAD_ARGUMENT, "output_dtype must be 0 (fp16) or 1 (bf16)");
    if (ldc < N) return set_error(FEATHER_ERR_BAD_ARGUMENT, "ldc must be at least N");
    if (M == 0) return FEATHER_OK;
    if (a == nullptr || a_scales == nullptr || b == nullptr || b_scales == nullptr || c == nullptr) return set_error(FEATHER_ERR_BAD_ARGUMENT, "a, b, their scales and c must not be null");
    if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(b_scales)) & 15u)
        return set_error(FEATHER_ERR_BAD_ARGUMENT, "a, b and their scales must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(bias)) & 1u) return set_error(FEATHER_ERR_BAD_ARGUMENT, "c and bias must be aligned to their element size");
    MxEncodeFn encode = mx_encode_fn();
    if (encode == nullptr) return set_error(FEATHER_ERR_NO_DEVICE, "cuTensorMapEncodeTiled is not available from the driver");

    const int tn = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    MxMmParams p{};
    p.a_scales = a_scales;
    p.b_scales = b_scales;
    p.bias = static_cast<const uint16_t*>(bias);
    p.c = static_cast<uint16_t*>(c);
    p.status = status_dev;
    p.ldc = ldc;
    p.M = static_cast<int>(M);
    p.N = static_cast<int>(N);
    p.K = static_cast<int>(K);
    p.out_bf16 = output_dtype == FEATHER_OUT_BF16 ? 1 : 0;
    p.tiles_n = static_cast<int>((N + kMxRows - 1) / kMxRows);
    p.stages_total = static_cast<int>((K + kMxStageK - 1) / kMxStageK);
    p.tiles_k = static_cast<int>(mx_tiles_k(K));
    const long long tiles = static_cast<long long>(p.tiles_n) * ((M + tn - 1) / tn);
    int splits = 1;
    while (splits < 8 && splits * 2 <= p.stages_total && tiles * splits < 148) splits *= 2;
    if (tiles * splits > 0x7FFFFFFF) return set_error(FEATHER_ERR_BAD_ARGUMENT, "too many tiles for one launch");

    CUtensorMap tw, tt;
    CUresult r = mx_operand_map(encode, &tw, b, N, K / 2, kMxRows);
    if (r != CUDA_SUCCESS) return set_error(FEATHER_ERR_CUDA, "cuTensorMapEncodeTiled(b) failed with CUresult %d", static_cast<int>(r));
    r = mx_operand_map(encode, &tt, a, M, K / 2, tn);
    if (r != CUDA_SUCCESS) return set_error(FEATHER_ERR_CUDA, "cuTensorMapEncodeTiled(a) failed with CUresult %d", static_cast<int>(r));
    cudaError_t e;
    switch (tn) {
        case 16: e = mx_launch_mm<16>(tw, tt, p, splits, tiles * splits, stream); break;
        case 32: e = mx_launch_mm<32>(tw, tt, p, splits, tiles * splits, stream); break;
        case 64: e = mx_launch_mm<64>(tw, tt, p, splits, tiles * splits, stream); break;
        default: e = mx_launch_mm<128>(tw, tt, p, splits, tiles * splits, stream); break;
    }
    if (e != cudaSuccess) return set_error(FEATHER_ERR_CUDA, "mxfp4_mm launch failed: %s", cudaGetErrorString(e));
    return FEATHER_OK;
}
