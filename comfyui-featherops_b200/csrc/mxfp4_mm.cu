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
// A cluster splits K: every rank pushes its fp32 tile, a slice of the token columns to each rank (distributed shared memory), and a rank
// sums its slice over all ranks in rank order.  No workspace, no atomics, the same bits on every run.
//
// Every wait is bounded (ptx.cuh); on expiry the CTA records a code in *status, drains and returns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

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
// One lane of a converged warp.  The TMA and MMA loops are run by one thread chosen this way and not by `lane == 0`: what the compiler
// makes of it issues a stage of the 192-feature pair kernel in half the time (8192 x 13824 x 5120: 380 us -> 231 us).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(p));
    return p != 0;
}

// 32 rows x 16 bytes of shared memory -> 32 lanes x 4 columns of tensor memory, repeated in all four lane quarters.  The pair form
// does so in both CTAs, each from its own shared memory.
template <int kCtaGroup>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
    if constexpr (kCtaGroup == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D[tmem] (+)= A[smem] * B[smem], E2M1 operands with an E8M0 scale for every 32 elements (two for the 64 k of one instruction).
template <int kCtaGroup>
__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
    if constexpr (kCtaGroup == 1)
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n"
            "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n"
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
    int stages_total;     // ceil(K / 256)
    int tiles_k;          // ceil(K / 128): scale tiles along K
};

__device__ __forceinline__ float load16(const uint16_t* p, bool bf16) {
    const uint16_t v = *p;                              // not __ldg: the kernel before this one may have written it
    return bf16 ? __uint_as_float(static_cast<uint32_t>(v) << 16) : __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ uint16_t round16(float v, bool bf16) { return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v)); }

// Up to this many tokens the weights are on the lanes and K is split over a cluster: 64 x 13824 x 5120 takes 11.9 us this way and 13.9 us
// on CTA pairs, 128 x 13824 x 5120 15.8 us (with 128-token tiles) and 13.9 us.  17 and 64 x 5120 x 13824: 11.2 and 12.7 us against 23.0 and 16.9;
// 17 and 64 x 5120 x 5120: 8.0 and 8.8 against 11.1 and 9.2.  Where K is short the border lies lower: 32 and 64 x 1024 x 1024 4.0 and 5.8 against 4.7
// and 4.8, 32 and 64 x 2811 x 1056 5.2 and 6.5 against 6.3 and 6.4.
constexpr int kMxSmallTokens = 64;
constexpr int kMxRows = 128;                        // weight rows of a tile: the lanes
constexpr int kMxMmThreads = 192;                   // producer warp, MMA warp, four epilogue warps
constexpr int kMxMaxSplits = 6;                     // K splits are 1, 2, 3, 4 or 6 (a cluster has at most 8 CTAs)

// Token columns of a tile that one rank of a K split sums: a multiple of 4 (16-byte pieces); the last ranks may have none.
__host__ __device__ constexpr int mx_slice_cols(int tn, int splits) { return ((tn + splits - 1) / splits + 3) / 4 * 4; }

template <int TN>
struct MxCfg {
    static_assert(TN == 16 || TN == 32 || TN == 64, "tokens of a tile");
    static constexpr int kWBytes = kMxRows * kMxRowBytes;
    static constexpr int kTBytes = TN * kMxRowBytes;
    static constexpr int kSfBytes = kMxTilesPerStage * kMxScaleTile;       // scales of up to 128 rows
    static constexpr int kStageBytes = kWBytes + kTBytes + 2 * kSfBytes;
    // Up to 32 tokens two CTAs share an SM; a 64-token tile's CTA has one to itself.
    static constexpr int kPerSm = TN <= 32 ? 2 : 1;
    static constexpr int kStages = TN == 16 ? 5 : TN == 32 ? 4 : 7;
    static constexpr int kSfCols = 2 * kMxTilesPerStage * 4;               // tensor-memory columns of a stage's scales
    static constexpr int kAccCols = TN < 32 ? 32 : TN;
    static constexpr int kTmemCols = kAccCols + kStages * kSfCols <= 128 ? 128 : 256;
    // K split: this rank's columns of every rank's tile, for the worst of the splits
    static constexpr int kSliceCols = TN == 16 ? 24 : TN == 32 ? 48 : 72;
    static_assert(2 * mx_slice_cols(TN, 2) <= kSliceCols && 3 * mx_slice_cols(TN, 3) <= kSliceCols && 4 * mx_slice_cols(TN, 4) <= kSliceCols && 6 * mx_slice_cols(TN, 6) <= kSliceCols, "slices");
    static constexpr int kSliceBytes = kSliceCols * kMxRows * 4;
    static constexpr int kBarBytes = 256;
    static constexpr int kSmemBytes = kStages * kStageBytes + kSliceBytes + kBarBytes;
    static_assert(kStageBytes % 1024 == 0 && kPerSm * (kSmemBytes + 1024) <= 228 * 1024, "shared memory");
};

// L2 prefetch of a box; reads nothing into the SM, so it may run ahead of the kernel that wrote the tensor.
__device__ __forceinline__ void tma_prefetch_2d(const void* tmap, int32_t c0, int32_t c1) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1) : "memory");
}

// 16 bytes to a cluster CTA's shared memory, counted on a barrier there.
__device__ __forceinline__ void st_async_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar) : "memory");
}

template <int TN>
__global__ void __launch_bounds__(kMxMmThreads) mx_mm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_t, const MxMmParams p,
                                                             const int splits) {
    using C = MxCfg<TN>;
    constexpr int kStages = C::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];                        // no static shared memory: the block's memory begins on a 1024-byte boundary
    const uint32_t base = smem_u32(smem);
    const uint32_t slice_base = base + kStages * C::kStageBytes;
    const uint32_t bar_full = slice_base + C::kSliceBytes, bar_empty = bar_full + 8 * kStages, bar_acc = bar_empty + 8 * kStages, bar_slice = bar_acc + 8;
    uint8_t* const words = smem + kStages * C::kStageBytes + C::kSliceBytes + 16 * kStages + 16;
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(words);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(words + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = splits == 1 ? 0 : static_cast<int>(cluster_ctarank());  // position in the cluster
    const int n0 = static_cast<int>(blockIdx.x) / splits * kMxRows;
    const int per = p.stages_total / splits, extra = p.stages_total % splits;
    const int begin = rank * per + (rank < extra ? rank : extra);
    const int count = per + (rank < extra ? 1 : 0);                          // at least 1: the host takes no more splits than stages
    const int cols = mx_slice_cols(TN, splits);
    const int my_cols = max(0, min(cols, TN - rank * cols));

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        mbar_init(bar_acc, 1);
        mbar_init(bar_slice, 1);
        *abort_flag = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
        mbar_arrive_expect_tx(bar_slice, static_cast<uint32_t>((splits - 1) * my_cols * kMxRows * 4));
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_slot)), C::kTmemCols);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (splits > 1) cluster_arrive_release();                                // this CTA's barriers are up; waited for before the first push
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    if (warp == 0 && elect_one()) {
        // the weights' way from memory does not depend on the kernel in front of this one
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_t);
        for (int i = begin; i < begin + min(count, kStages); ++i) tma_prefetch_2d(&tmap_w, i * kMxRowBytes, n0);
    }
    __syncwarp();
    pdl_wait_for_previous_kernel();

    if (warp == 0) {
        if (elect_one()) {
            uint32_t s = 0, ph = 0;
            int issued = 0;
            bool ok = true;
            const uint8_t* const w_sf = p.b_scales + static_cast<long long>(n0 / 128) * p.tiles_k * kMxScaleTile;
            for (int i = begin; i < begin + count; ++i) {
                if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, abort_flag)) {
                    mx_give_up(p.status, abort_flag, kMxRoleProducer, s);
                    ok = false;
                    break;
                }
                const int kt = i * kMxTilesPerStage;
                const uint32_t sf_bytes = min(kMxTilesPerStage, p.tiles_k - kt) * kMxScaleTile;
                const uint32_t w = base + s * C::kStageBytes, t = w + C::kWBytes, sfw = t + C::kTBytes, sft = sfw + C::kSfBytes;
                const uint32_t bar = bar_full + 8 * s;
                mbar_arrive_expect_tx(bar, C::kWBytes + C::kTBytes + 2 * sf_bytes);
                tma_load_2d(w, &tmap_w, bar, i * kMxRowBytes, n0);
                tma_load_2d(t, &tmap_t, bar, i * kMxRowBytes, 0);
                bulk_load(sfw, w_sf + static_cast<long long>(kt) * kMxScaleTile, sf_bytes, bar);
                bulk_load(sft, p.a_scales + static_cast<long long>(kt) * kMxScaleTile, sf_bytes, bar);
                ++issued;
                if (++s == kStages) {
                    s = 0;
                    ph ^= 1u;
                }
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
        if (elect_one()) {
            uint32_t s = 0, ph = 0;
            int k_left = p.K - begin * kMxStageK;
            for (int i = 0; i < count; ++i, k_left -= kMxStageK) {
                if (!mbar_wait(bar_full + 8 * s, ph, abort_flag)) {
                    mx_give_up(p.status, abort_flag, kMxRoleMma, s);
                    break;
                }
                tc_fence_after();
                const uint32_t w = base + s * C::kStageBytes, sfw = w + C::kWBytes + C::kTBytes;
                const uint32_t cw = tmem + C::kAccCols + s * C::kSfCols, ct = cw + kMxTilesPerStage * 4;
                const uint64_t fw = smem_desc_scales(sfw), ft = smem_desc_scales(sfw + C::kSfBytes);
                // a last stage of one scale tile copies whatever the other half holds; no MMA reads it
#pragma unroll
                for (int j = 0; j < kMxTilesPerStage; ++j) {
                    tmem_cp_scales<1>(cw + 4 * j, fw + j * (kMxScaleTile >> 4));
                    tmem_cp_scales<1>(ct + 4 * j, ft + j * (kMxScaleTile >> 4));
                }
                const uint64_t wd = umma_desc_kmajor_sw128(w), td = umma_desc_kmajor_sw128(w + C::kWBytes);
                const auto mma = [&](int j, uint32_t accumulate) {
                    umma_mxf4<1>(tmem, wd + 2 * j, td + 2 * j, umma_idesc_mxf4(kMxRows, TN, (j & 1) * 2), cw + 4 * (j >> 1), ct + 4 * (j >> 1), accumulate);
                };
                mma(0, i == 0 ? 0u : 1u);
                if (k_left > 192) {
                    mma(1, 1u);
                    mma(2, 1u);
                    mma(3, 1u);
                } else {
                    if (k_left > 64) mma(1, 1u);
                    if (k_left > 128) mma(2, 1u);
                }
                umma_commit_1cta(bar_empty + 8 * s);
                if (++s == kStages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
            umma_commit_1cta(bar_acc);
            const uint64_t t0_ns = globaltimer_ns();                          // no MMA reads shared memory any more when this warp leaves
            while (!mbar_try_wait(bar_acc, 0) && globaltimer_ns() - t0_ns < kWaitLimitNs) {
            }
        }
        __syncwarp();
    } else {
        const bool bf16 = p.out_bf16 != 0;
        const int q = warp & 3;                                              // lane quarter of tensor memory this warp may read
        const int row = q * 32 + lane;
        const int n = n0 + row;
        const bool in = n < p.N;
        const float bias = (in && p.bias != nullptr) ? load16(p.bias + n, bf16) : 0.0f;
        const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16);
        uint16_t* const out = p.c + n;
        const int tokens = min(TN, p.M);
        bool ok = mbar_wait_warp(bar_acc, 0, abort_flag, lane);
        if (!ok && lane == 0) mx_give_up(p.status, abort_flag, kMxRoleEpilogue, warp);
        tc_fence_after();
        if (splits == 1) {
#pragma unroll 1
            for (int c = 0; c < tokens && ok; c += 16) {
                uint32_t v[16];
                tmem_ld_32x32b_x16(acc + c, v);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (in && c + j < tokens) out[(c + j) * p.ldc] = round16(__uint_as_float(v[j]) + bias, bf16);
            }
        } else {
            cluster_wait_acquire();                                          // every rank's barriers are up
            // Push: [source rank][row][cols] on the rank that sums the columns.  The source is registers, so a rank may leave while its
            // pushes are still on their way; the owner counts their bytes.  A rank that gave up pushes what it has: the owner must not wait.
#pragma unroll 1
            for (int c = 0; c < TN; c += 16) {
                uint32_t v[16];
                tmem_ld_32x32b_x16(acc + c, v);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const int owner = (c + j) / cols;
                    const uint32_t at = slice_base + static_cast<uint32_t>(((rank * kMxRows + row) * cols + (c + j - owner * cols)) * 4);
                    if (owner == rank)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[j]), "r"(v[j + 1]), "r"(v[j + 2]), "r"(v[j + 3]) : "memory");
                    else
                        st_async_v4(mapa_u32(at, owner), v[j], v[j + 1], v[j + 2], v[j + 3], mapa_u32(bar_slice, owner));
                }
            }
            __syncwarp();
            cluster_arrive_release();                                        // nothing more is pushed from here
            if (my_cols > 0) {
                if (!mbar_wait_warp(bar_slice, 0, abort_flag, lane)) {
                    if (lane == 0) mx_give_up(p.status, abort_flag, kMxRoleEpilogue, 0x100 | warp);
                    ok = false;
                }
                // a thread sums its own row, in rank order
                const int first = rank * cols;
                for (int c = 0; c < my_cols; c += 4) {
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int r = 0; r < kMxMaxSplits; ++r) {
                        if (r < splits) {
                            float x[4];
                            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                                         : "r"(slice_base + static_cast<uint32_t>(((r * kMxRows + row) * cols + c) * 4))
                                         : "memory");
#pragma unroll
                            for (int e = 0; e < 4; ++e) sum[e] += x[e];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (ok && in && first + c + e < tokens) out[(first + c + e) * p.ldc] = round16(sum[e] + bias, bf16);
                }
            }
        }
    }
    if (splits > 1) {
        // A rank's shared memory outlives every push into it, also those of columns it gave up on.
        if (warp < 2) {
            cluster_wait_acquire();
            cluster_arrive_release();
        }
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
// Many tokens: a persistent kernel of CTA pairs
// ================================================================================================
//   out tile [256 tokens x TF features]  +=  A[256 x 64 k] * B^T[64 k x TF]        (tcgen05 cta_group::2)
//
// A thread's lane is a token here, so an epilogue thread holds consecutive features of one row: it packs them into 16-byte pieces
// of a swizzled staging tile that one TMA store writes.  Each CTA of the pair loads its own 128 token rows, half of the TF weight
// rows, its tokens' scales and all of the weights' scales (the pair's tensor cores share the operands, not the scales).
constexpr int kMxPairTokens = 256;
constexpr int kMxPairEpilogueWarps = 8;
constexpr int kMxPairThreads = 32 * (2 + kMxPairEpilogueWarps);
constexpr int kMxChunk = 32;                        // features of one staged store: a 64-byte row

template <int TF>
struct MxPairCfg {
    static_assert(TF == 128 || TF == 192 || TF == 256, "features of a tile");
    static constexpr int kABytes = 128 * kMxRowBytes;
    static constexpr int kBBytes = TF / 2 * kMxRowBytes;
    static constexpr int kSfaBytes = kMxTilesPerStage * kMxScaleTile;
    static constexpr int kSfbBlocks = TF == 128 ? 1 : 2;                    // 128-row scale tiles that a tile's weight rows touch
    static constexpr int kSfbBytes = kSfbBlocks * kSfaBytes;
    static constexpr int kStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes;
    static constexpr int kAccs = TF <= 192 ? 2 : 1;
    static constexpr int kSfCols = kMxTilesPerStage * 4 * (1 + kSfbBlocks);
    static constexpr int kOutBufs = 2;
    static constexpr int kOutBufBytes = 32 * kMxChunk * 2;                  // a warp's 32 rows of one chunk
    static constexpr int kOutBytes = kMxPairEpilogueWarps * kOutBufs * kOutBufBytes;
    static constexpr int kBarBytes = 256;
    static constexpr int kStagesSmem = (227 * 1024 - kOutBytes - kBarBytes) / kStageBytes;
    static constexpr int kStagesTmem = (512 - kAccs * TF) / kSfCols;
    static constexpr int kStages = kStagesSmem < kStagesTmem ? kStagesSmem : kStagesTmem;
    static_assert(kStages >= 3 && kStages <= 8 && kStageBytes % 1024 == 0, "ring");
    static constexpr int kSmemBytes = kStages * kStageBytes + kOutBytes + kBarBytes;
};

struct MxPairMaps {
    CUtensorMap a, b, sfa, sfb, c;
};

struct MxPairParams {
    const uint16_t* bias;
    uint16_t* c;
    int* status;
    long long ldc;
    int M, N, K;
    int out_bf16;
    int tma_store;
    int tiles_m, tiles_n;
    int stages_total;
};

__device__ __forceinline__ void mx_pair_give_up(int* status, volatile int* abort_flag, int role, int detail) {
    mx_give_up(status, abort_flag, role, detail);
    const uint32_t peer = mapa_u32(smem_u32(const_cast<int*>(abort_flag)), cluster_ctarank() ^ 1u);
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer), "r"(1) : "memory");
}

// Tiles in bands of eight token tiles, token tile fastest: the pairs that run together share a few tiles of either operand.
__device__ __forceinline__ void mx_pair_tile(const MxPairParams& p, int tile, int tf, int& m0, int& n0) {
    constexpr int kBand = 8;
    const int band = tile / (kBand * p.tiles_n), in_band = tile - band * kBand * p.tiles_n;
    const int rows = min(kBand, p.tiles_m - band * kBand);
    n0 = in_band / rows * tf;
    m0 = (band * kBand + in_band % rows) * kMxPairTokens;
}

// Offset of 16-byte piece j of a staged row under the store's 64-byte swizzle.
__device__ __forceinline__ uint32_t mx_staged(int row, int j) { return row * 64 + ((j ^ ((row >> 1) & 3)) << 4); }

template <int TF>
__global__ void __launch_bounds__(kMxPairThreads, 1) mx_mm_pair_kernel(const __grid_constant__ MxPairMaps maps, const MxPairParams p) {
    using C = MxPairCfg<TF>;
    constexpr int kStages = C::kStages;
    constexpr int kAccs = C::kAccs;
    extern __shared__ __align__(1024) uint8_t smem_pair[];                  // no static shared memory: the block's memory begins on a 1024-byte boundary
    const uint32_t base = smem_u32(smem_pair);
    uint8_t* const base_gen = smem_pair;
    const uint32_t out_base = base + kStages * C::kStageBytes;
    const uint32_t bar_base = out_base + C::kOutBytes;
    const uint32_t bar_full = bar_base, bar_empty = bar_full + 8 * kStages, bar_accfull = bar_empty + 8 * kStages, bar_accempty = bar_accfull + 16, bar_drain = bar_accempty + 16;
    uint8_t* const words = base_gen + kStages * C::kStageBytes + C::kOutBytes + 16 * kStages + 40;
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(words);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(words + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
    const int tiles = p.tiles_m * p.tiles_n;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_full + 8 * s, 2);                                 // both producers
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_accfull + 8 * a, 1);
            mbar_init(bar_accempty + 8 * a, 2 * kMxPairEpilogueWarps);
        }
        mbar_init(bar_drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&maps.a);
        prefetch_tmap(&maps.b);
        prefetch_tmap(&maps.sfa);
        prefetch_tmap(&maps.sfb);
        if (p.tma_store) prefetch_tmap(&maps.c);
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish<2>();
    }
    tc_fence_before();
    cluster_arrive_release();
    cluster_wait_acquire();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();

    if (warp == 0) {
        if (elect_one()) {
            uint32_t s = 0, ph = 0;
            int issued = 0;
            bool ok = true;
            const uint32_t full0 = mapa_u32(bar_full, 0);                   // the leader CTA's barriers
            for (int tile = cluster; ok && tile < tiles; tile += clusters) {
                int m0, n0;
                mx_pair_tile(p, tile, TF, m0, n0);
                for (int i = 0; i < p.stages_total; ++i) {
                    if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, abort_flag)) {
                        mx_pair_give_up(p.status, abort_flag, kMxRoleProducer, s);
                        ok = false;
                        break;
                    }
                    const uint32_t a = base + s * C::kStageBytes, b = a + C::kABytes, sfa = b + C::kBBytes, sfb = sfa + C::kSfaBytes;
                    const uint32_t bar = full0 + 8 * s;
                    mbar_arrive_expect_tx_cluster(bar, C::kStageBytes);
                    tma_load_2d_pair(a, &maps.a, bar, i * kMxRowBytes, m0 + static_cast<int>(rank) * 128);
                    tma_load_2d_pair(b, &maps.b, bar, i * kMxRowBytes, n0 + static_cast<int>(rank) * (TF / 2));
                    tma_load_2d_pair(sfa, &maps.sfa, bar, i * (kMxTilesPerStage * kMxScaleTile / 8), m0 / 128 + static_cast<int>(rank));
                    tma_load_2d_pair(sfb, &maps.sfb, bar, i * (kMxTilesPerStage * kMxScaleTile / 8), n0 / 128);
                    ++issued;
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            if (!ok && rank == 0) {
                // the copies in flight (both CTAs' count on this barrier) land before shared memory is given back
                const uint64_t begin_ns = globaltimer_ns();
                for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
                    while (!mbar_try_wait(bar_full + 8 * (i % kStages), (i / kStages) & 1) && globaltimer_ns() - begin_ns < kWaitLimitNs) {
                    }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const auto issue_stage = [&](uint32_t s, uint32_t d, uint32_t sfb_shift, int k_left, bool first) {      // by one thread
                const uint32_t a = base + s * C::kStageBytes, sfa = a + C::kABytes + C::kBBytes;
                const uint32_t ca = tmem + kAccs * TF + s * C::kSfCols, cb = ca + kMxTilesPerStage * 4;
                const uint64_t ad = umma_desc_kmajor_sw128(a), bd = umma_desc_kmajor_sw128(a + C::kABytes);
                const uint64_t fa = smem_desc_scales(sfa), fb = smem_desc_scales(sfa + C::kSfaBytes);
#pragma unroll
                for (int j = 0; j < kMxTilesPerStage; ++j) {
                    tmem_cp_scales<2>(ca + 4 * j, fa + j * (kMxScaleTile >> 4));
#pragma unroll
                    for (int blk = 0; blk < C::kSfbBlocks; ++blk)
                        tmem_cp_scales<2>(cb + (j * C::kSfbBlocks + blk) * 4, fb + ((blk * C::kSfaBytes + j * kMxScaleTile) >> 4));
                }
                const auto mma = [&](int j, uint32_t accumulate) {
                    umma_mxf4<2>(d, ad + 2 * j, bd + 2 * j, umma_idesc_mxf4(kMxPairTokens, TF, (j & 1) * 2), ca + 4 * (j >> 1),
                                 cb + (j >> 1) * C::kSfbBlocks * 4 + sfb_shift, accumulate);
                };
                mma(0, first ? 0u : 1u);
                if (k_left > 192) {
                    mma(1, 1u);
                    mma(2, 1u);
                    mma(3, 1u);
                } else {
                    if (k_left > 64) mma(1, 1u);
                    if (k_left > 128) mma(2, 1u);
                }
            };
            uint32_t s = 0, ph = 0;
            int done = 0;
            bool ok = true;
            if (elect_one()) {
                for (int tile = cluster; ok && tile < tiles; tile += clusters, ++done) {
                    int m0, n0;
                    mx_pair_tile(p, tile, TF, m0, n0);
                    const int acc = kAccs == 2 ? done & 1 : 0;
                    const uint32_t acc_ph = kAccs == 2 ? (done >> 1) & 1 : done & 1;
                    if (!mbar_wait(bar_accempty + 8 * acc, acc_ph ^ 1u, abort_flag)) {
                        mx_pair_give_up(p.status, abort_flag, kMxRoleMma, 0x100 | acc);
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem + acc * TF;
                    const uint32_t sfb_shift = (n0 & 127) >> 5;
                    int k_left = p.K;
                    for (int i = 0; i < p.stages_total; ++i, k_left -= kMxStageK) {
                        if (!mbar_wait(bar_full + 8 * s, ph, abort_flag)) {
                            mx_pair_give_up(p.status, abort_flag, kMxRoleMma, s);
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        issue_stage(s, d, sfb_shift, k_left, i == 0);
                        umma_commit_pair(bar_empty + 8 * s, 0x3);
                        if (++s == kStages) {
                            s = 0;
                            ph ^= 1u;
                        }
                    }
                    if (ok) umma_commit_pair(bar_accfull + 8 * acc, 0x3);
                }
            }
            __syncwarp();
            // nothing of the pair is torn down while an MMA still reads it
            if (elect_one()) {
                umma_commit_2cta_local(bar_drain);
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(bar_drain, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
                }
            }
        }
        __syncwarp();
    } else {
        // epilogue: warp w reads the tensor-memory lanes of quarter w % 4; the two groups of four warps take alternate chunks
        const int q = warp & 3, grp = (warp - 2) >> 2;
        const bool bf16 = p.out_bf16 != 0;
        const uint32_t stage0 = out_base + (warp - 2) * (C::kOutBufs * C::kOutBufBytes);
        int done = 0;
        uint32_t flip = 0;
        bool alive = true;                                                  // a warp whose wait ran out keeps to the barriers and touches nothing
        for (int tile = cluster; tile < tiles; tile += clusters, ++done) {
            int m0, n0;
            mx_pair_tile(p, tile, TF, m0, n0);
            m0 += static_cast<int>(rank) * 128;
            const int acc = kAccs == 2 ? done & 1 : 0;
            const uint32_t acc_ph = kAccs == 2 ? (done >> 1) & 1 : done & 1;
            // the bias of this warp's chunks, one feature a lane, on its way while the tile is being multiplied
            constexpr int kChunks = TF / kMxChunk / 2;                      // of each group
            float b[kChunks];
#pragma unroll
            for (int h = 0; h < kChunks; ++h) {
                const int f = n0 + (grp + 2 * h) * kMxChunk + lane;
                b[h] = (p.bias != nullptr && f < p.N) ? load16(p.bias + f, bf16) : 0.0f;
            }
            if (alive && !mbar_wait_warp(bar_accfull + 8 * acc, acc_ph, abort_flag, lane)) {
                if (lane == 0) mx_pair_give_up(p.status, abort_flag, kMxRoleEpilogue, acc);
                alive = false;
            }
            tc_fence_after();
            // One accumulator (256 features): a warp takes its four chunks into registers at once and gives the accumulator back before it
            // packs them.  Two accumulators: chunk by chunk, the other one is being filled meanwhile.
            constexpr int kHold = kAccs == 1 ? kChunks : 1;
            uint32_t v[kHold][kMxChunk / 16][16];
            const auto read_chunk = [&](int c, uint32_t(&x)[kMxChunk / 16][16]) {
#pragma unroll
                for (int j = 0; j < kMxChunk / 16; ++j) tmem_ld_32x32b_x16(tmem + acc * TF + (static_cast<uint32_t>(q * 32) << 16) + c + 16 * j, x[j]);
            };
            const auto release = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(mapa_u32(bar_accempty + 8 * acc, 0));
            };
            if constexpr (kAccs == 1) {
                if (alive) {
#pragma unroll
                    for (int h = 0; h < kHold; ++h) read_chunk((grp + 2 * h) * kMxChunk, v[h]);
                    tc_wait_ld();
                }
                release();
            }
            const auto emit = [&](int c, const uint32_t(&x)[kMxChunk / 16][16], float bias) {
                const int n = n0 + c;
                // the store that last used this staging buffer has read it
                if (lane == 0) tma_store_wait_read<C::kOutBufs - 1>();
                __syncwarp();
                const uint32_t buf = stage0 + flip * C::kOutBufBytes;
                if (alive) {
#pragma unroll
                    for (int j = 0; j < kMxChunk / 8; ++j) {                // 16-byte pieces of the lane's row
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int e = 8 * j + 2 * i;
                            float lo = __uint_as_float(x[e / 16][e % 16]), hi = __uint_as_float(x[e / 16][e % 16 + 1]);
                            if (p.bias != nullptr) {
                                lo += __shfl_sync(0xffffffffu, bias, e);
                                hi += __shfl_sync(0xffffffffu, bias, e + 1);
                            }
                            w[i] = pack16x2(lo, hi, bf16);
                        }
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(buf + mx_staged(lane, j)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                    }
                }
                if (p.tma_store) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (alive && n < p.N && m0 + q * 32 < p.M) tma_store_2d(&maps.c, buf, n, m0 + q * 32);
                        tma_store_commit();
                    }
                    __syncwarp();
                } else {
                    // rows that TMA cannot store: two bytes a lane
                    __syncwarp();
                    const int rows = alive ? min(32, p.M - m0 - q * 32) : 0;
                    if (n + lane < p.N) {
                        uint16_t* const out = p.c + (m0 + q * 32) * p.ldc + n + lane;
#pragma unroll 8
                        for (int r = 0; r < rows; ++r) {
                            uint16_t y;
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(buf + mx_staged(r, lane >> 3) + (lane & 7) * 2) : "memory");
                            out[r * p.ldc] = y;
                        }
                    }
                    __syncwarp();
                }
                flip ^= 1u;
            };
            if constexpr (kAccs == 1) {
#pragma unroll
                for (int h = 0; h < kHold; ++h) emit((grp + 2 * h) * kMxChunk, v[h], b[h]);
            } else {
#pragma unroll
                for (int h = 0; h < kChunks; ++h) {
                    const int c = (grp + 2 * h) * kMxChunk;
                    if (alive) {
                        read_chunk(c, v[0]);
                        tc_wait_ld();
                    }
                    if (h + 1 == kChunks) release();                        // this warp's last read of the accumulator
                    emit(c, v[0], b[h]);
                }
            }
        }
        if (lane == 0) tma_store_wait_all<0>();
        __syncwarp();
    }
    tc_fence_before();
    cluster_arrive_release();
    cluster_wait_acquire();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<2>(tmem, 512);
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

// The scale tiles of an operand as 8-byte elements: 64 of them are a tile, a row holds the tiles of 128 rows along K.
static CUresult mx_scale_map(MxEncodeFn encode, CUtensorMap* out, const void* ptr, int64_t rows, int64_t tiles_k, int box_blocks) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(tiles_k) * (kMxScaleTile / 8), static_cast<cuuint64_t>((rows + 127) / 128)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(tiles_k) * kMxScaleTile};
    const cuuint32_t box[2] = {kMxTilesPerStage * kMxScaleTile / 8, static_cast<cuuint32_t>(box_blocks)};
    const cuuint32_t step[2] = {1, 1};
    return encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT64, 2, const_cast<void*>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

static CUresult mx_output_map(MxEncodeFn encode, CUtensorMap* out, void* c, int64_t M, int64_t N, int64_t ldc) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(M)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ldc) * 2};
    const cuuint32_t box[2] = {kMxChunk, 32};
    const cuuint32_t step[2] = {1, 1};
    return encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, c, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Features of a pair tile, by the time that its waves take.  Nanoseconds of a stage (256 k) and of a tile around its stages, fitted to
// 8192 x 13824 x 5120 and 8192 x 5120 x 13824: 128 features 261 / 252 us, 192: 221 / 216, 256: 215 / 200 (the widest tile loads the least
// and has the one accumulator that is read out between tiles).  Where few tiles leave pairs idle the narrower ones win:
// 520 x 2811 x 1056 takes 7.6 / 8.9 / 11.7 us, 1024 x 5120 x 5120 18.8 / 17.3 / 20.0 us.
static int mx_pair_features(int64_t M, int64_t N, int stages, int pairs) {
    constexpr struct { int tf, stage_ns, tile_ns; } kTiles[] = {{128, 250, 500}, {192, 328, 330}, {256, 390, 1130}};
    int best = 0;
    double least = 0.0;
    for (const auto& t : kTiles) {
        const int64_t tiles = (M + kMxPairTokens - 1) / kMxPairTokens * ((N + t.tf - 1) / t.tf);
        const double ns = static_cast<double>((tiles + pairs - 1) / pairs) * (static_cast<double>(stages) * t.stage_ns + t.tile_ns);
        if (best == 0 || ns < least) {
            best = t.tf;
            least = ns;
        }
    }
    return best;
}

template <int TF>
static cudaError_t mx_launch_pair(const MxPairMaps& maps, const MxPairParams& p, int sms, cudaStream_t stream) {
    using C = MxPairCfg<TF>;
    static SmemOptIn opt_in;
    cudaError_t e = opt_in(mx_mm_pair_kernel<TF>, C::kSmemBytes);
    if (e != cudaSuccess) return e;
    const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
    const long long clusters = tiles < sms / 2 ? tiles : sms / 2;
    return launch_dependent(mx_mm_pair_kernel<TF>, dim3(static_cast<unsigned>(clusters * 2)), dim3(kMxPairThreads), 2, C::kSmemBytes, stream, maps, p);
}

// K splits of a small product: the largest of 1, 2, 3, 4, 6 with which all CTAs are resident at once (two to an SM up to 32 tokens).
// One more wave costs more than the split gives: 64 x 13824 x 5120 takes 11.9 us unsplit (108 CTAs) and 21.1 us split in two;
// 1 x 5120 x 5120 takes 7.8 us on 40 CTAs, 5.8 us on 160.
template <int TN>
static cudaError_t mx_launch_mm(const CUtensorMap& tw, const CUtensorMap& tt, const MxMmParams& p, int sms, cudaStream_t stream) {
    using C = MxCfg<TN>;
    static SmemOptIn opt_in;
    cudaError_t e = opt_in(mx_mm_kernel<TN>, C::kSmemBytes);
    if (e != cudaSuccess) return e;
    const long long tiles = (p.N + kMxRows - 1) / kMxRows;
    int splits = 1;
    for (int s : {2, 3, 4, kMxMaxSplits})
        if (s <= p.stages_total && tiles * s <= static_cast<long long>(sms) * C::kPerSm) splits = s;
    const long long ctas = tiles * splits;
    return launch_dependent(mx_mm_kernel<TN>, dim3(static_cast<unsigned>(ctas)), dim3(kMxMmThreads), splits, C::kSmemBytes, stream, tw, tt, p, splits);
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

    const int sms = sm_count();
    if (sms < 2) return set_error(FEATHER_ERR_CUDA, "the number of SMs could not be read");
    const int stages = static_cast<int>((K + kMxStageK - 1) / kMxStageK);
    cudaError_t e;
    if (M > kMxSmallTokens) {
        const int tf = mx_pair_features(M, N, stages, sms / 2);
        MxPairMaps maps;
        memset(&maps, 0, sizeof(maps));
        MxPairParams p{};
        p.bias = static_cast<const uint16_t*>(bias);
        p.c = static_cast<uint16_t*>(c);
        p.status = status_dev;
        p.ldc = ldc;
        p.M = static_cast<int>(M);
        p.N = static_cast<int>(N);
        p.K = static_cast<int>(K);
        p.out_bf16 = output_dtype == FEATHER_OUT_BF16 ? 1 : 0;
        // TMA stores need 16-byte aligned output rows
        p.tma_store = ldc % 8 == 0 && (reinterpret_cast<uintptr_t>(c) & 15u) == 0 ? 1 : 0;
        p.tiles_m = static_cast<int>((M + kMxPairTokens - 1) / kMxPairTokens);
        p.tiles_n = static_cast<int>((N + tf - 1) / tf);
        p.stages_total = stages;
        if (static_cast<long long>(p.tiles_m) * p.tiles_n > 0x3FFFFFFF) return set_error(FEATHER_ERR_BAD_ARGUMENT, "too many tiles for one launch");
        CUresult r = mx_operand_map(encode, &maps.a, a, M, K / 2, 128);
        if (r == CUDA_SUCCESS) r = mx_operand_map(encode, &maps.b, b, N, K / 2, tf / 2);
        if (r == CUDA_SUCCESS) r = mx_scale_map(encode, &maps.sfa, a_scales, M, mx_tiles_k(K), 1);
        if (r == CUDA_SUCCESS) r = mx_scale_map(encode, &maps.sfb, b_scales, N, mx_tiles_k(K), tf == 128 ? 1 : 2);
        if (r == CUDA_SUCCESS && p.tma_store) r = mx_output_map(encode, &maps.c, c, M, N, ldc);
        if (r != CUDA_SUCCESS) return set_error(FEATHER_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
        e = tf == 128 ? mx_launch_pair<128>(maps, p, sms, stream) : tf == 192 ? mx_launch_pair<192>(maps, p, sms, stream) : mx_launch_pair<256>(maps, p, sms, stream);
    } else {
        const int tn = M <= 16 ? 16 : M <= 32 ? 32 : 64;
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
        p.stages_total = stages;
        p.tiles_k = static_cast<int>(mx_tiles_k(K));
        CUtensorMap tw, tt;
        CUresult r = mx_operand_map(encode, &tw, b, N, K / 2, kMxRows);
        if (r == CUDA_SUCCESS) r = mx_operand_map(encode, &tt, a, M, K / 2, tn);
        if (r != CUDA_SUCCESS) return set_error(FEATHER_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
        e = tn == 16 ? mx_launch_mm<16>(tw, tt, p, sms, stream) : tn == 32 ? mx_launch_mm<32>(tw, tt, p, sms, stream) : mx_launch_mm<64>(tw, tt, p, sms, stream);
    }
    if (e != cudaSuccess) return set_error(FEATHER_ERR_CUDA, "mxfp4_mm launch failed: %s", cudaGetErrorString(e));
    return FEATHER_OK;
}
