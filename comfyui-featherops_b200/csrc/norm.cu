// The norms before and after a block, its gate and its residual, in one pass over the rows:
//
//   z = y                      or  norm(y) * post_weight
//   r = x + residual_scale * gate * z
//   h = (norm(r) * weight + bias) * (1 + scale) + shift
//   norm(v) = v / sqrt(mean(v^2) + eps)      or  (v - mean(v)) / sqrt(var(v) + eps)
//
// A row lives in the registers of a block, or of one group of a block's threads, from its only read to its only write; sums are fp32, over the values as
// they are before r is rounded to x's type.  h leaves in 16 or 32 bits or, rounded to 16 bits first, as the MXFP4 operand of the
// product that follows (mxfp4.cuh).
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdlib.h>

#include <type_traits>

#include "../../include/feather_b200.h"
#include "host_util.h"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace feather {

// Two fp32 values an instruction.
struct F2 {
    unsigned long long u;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.u) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void f2_split(F2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v.u)); }
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
    return r;
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
    return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(a.u), "l"(b.u), "l"(c.u));
    return r;
}

// ------------------------------------------------------------------------------------------------ memory <-> registers
// Every load here is an ordinary one: the kernels may be resident while the kernel before them still writes their operands, so the
// read-only path (__ldg), which asks for memory that nobody writes during the kernel's life, is not theirs to take.
//
// Eight consecutive elements as they lie in memory (16-byte aligned).
template <int T>
struct alignas(16) Raw8 {
    uint32_t w[T == FEATHER_SRC_FP32 ? 8 : 4];
};
template <int T>
__device__ __forceinline__ Raw8<T> load8(const void* base, long long at) {
    Raw8<T> r;
    if constexpr (T == FEATHER_SRC_FP32) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + at);
        const uint4 a = p[0], b = p[1];
        r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
        r.w[4] = b.x; r.w[5] = b.y; r.w[6] = b.z; r.w[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
        r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
    }
    return r;
}
template <int T>
__device__ __forceinline__ void values8(const Raw8<T>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (T == FEATHER_SRC_FP32) {
            v[2 * i] = __uint_as_float(r.w[2 * i]);
            v[2 * i + 1] = __uint_as_float(r.w[2 * i + 1]);
        } else {
            unpack16x2(r.w[i], T == FEATHER_SRC_BF16, v[2 * i], v[2 * i + 1]);
        }
    }
}
template <int T>
__device__ __forceinline__ void store8(void* base, long long at, const float (&f)[8]) {
    if constexpr (T == FEATHER_SRC_FP32) {
        float4* const o = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
        o[0] = make_float4(f[0], f[1], f[2], f[3]);
        o[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        constexpr bool kBf16 = T == FEATHER_SRC_BF16;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) =
            make_uint4(pack16x2(f[0], f[1], kBf16), pack16x2(f[2], f[3], kBf16), pack16x2(f[4], f[5], kBf16), pack16x2(f[6], f[7], kBf16));
    }
}

// A vector of any of the three types, its type known at run time.  Nothing is converted here, so that several loads are under way at once.
struct RawAny {
    uint32_t w[8];
};
__device__ __forceinline__ void load_any(RawAny& r, const void* base, int type, long long at) {
    if (base == nullptr) return;
    if (type == FEATHER_SRC_FP32) {
        const Raw8<FEATHER_SRC_FP32> v = load8<FEATHER_SRC_FP32>(base, at);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = v.w[i];
    } else {
        const Raw8<FEATHER_SRC_BF16> v = load8<FEATHER_SRC_BF16>(base, at);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = v.w[i];
    }
}
__device__ __forceinline__ void values_any(const RawAny& r, int type, float (&v)[8]) {
    if (type == FEATHER_SRC_FP32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack16x2(r.w[i], type == FEATHER_SRC_BF16, v[2 * i], v[2 * i + 1]);
    }
}

struct NormParams {
    feather_norm_args a;
    int vecs;             // vectors (or elements) of a row
    int chunk;            // consecutive rows of a block
    int groups, stages;   // of the kernel for many rows
    float inv_cols;
    uint64_t wait_ns;     // limit of its waits for a row
};

// ------------------------------------------------------------------------------------------------ sums over a row
// Sum over a row, which is the whole block's, through `part`.  A buffer is used again two sums later, past the other buffer's barrier, so one
// barrier for each sum is enough.  Entries past the block's warps are zero (clear_parts).
constexpr int kNormMaxWarps = 32;
__device__ __forceinline__ void clear_parts(float (*part)[kNormMaxWarps]) {
    for (int i = threadIdx.x; i < 2 * kNormMaxWarps; i += blockDim.x) (&part[0][0])[i] = 0.0f;
    __syncthreads();
}
__device__ __forceinline__ float row_sum(float v, float (*part)[kNormMaxWarps], int& flip) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) part[flip][threadIdx.x >> 5] = v;
    __syncthreads();
    const float4* const q = reinterpret_cast<const float4*>(part[flip]);
    const int quads = (blockDim.x + 127) >> 7;
    v = 0.0f;
    for (int i = 0; i < quads; ++i) {                                         // the same order in every thread
        const float4 x = q[i];
        v += (x.x + x.y) + (x.z + x.w);
    }
    flip ^= 1;
    return v;
}

// ------------------------------------------------------------------------------------------------ whole vectors
// What multiplies and adds to a row's values, folded into three vectors:
//   r = x + G z      G = residual_scale * gate * post_weight
//   h = A n + B      A = weight * (1 + scale),  B = bias * (1 + scale) + shift
// They change only where a row belongs to another row of gate, scale or shift, so a thread keeps those of its own columns in shared
// memory (no other thread reads them: no barrier).
constexpr int kNormG = 1, kNormA = 2, kNormB = 4;

__host__ __device__ __forceinline__ int norm_present(const feather_norm_args& a) {
    return ((a.gate != nullptr || a.post_weight != nullptr) ? kNormG : 0) | ((a.weight != nullptr || a.scale != nullptr) ? kNormA : 0) |
           ((a.bias != nullptr || a.shift != nullptr) ? kNormB : 0);
}

// Where a row's gate, scale and shift begin.
struct ModulationAt {
    long long gate, scale, shift;
};
__device__ __forceinline__ long long share_of(long long row, int64_t rows) { return static_cast<uint32_t>(row) / static_cast<uint32_t>(rows); }   // both fit (host)
__device__ __forceinline__ ModulationAt modulation_at(const feather_norm_args& a, long long row) {
    return {a.gate != nullptr ? share_of(row, a.gate_rows) * a.gate_ld : 0, a.scale != nullptr ? share_of(row, a.scale_rows) * a.scale_ld : 0,
            a.shift != nullptr ? share_of(row, a.shift_rows) * a.shift_ld : 0};
}

__device__ __forceinline__ void fold_g(const feather_norm_args& a, const RawAny& gate, const RawAny& post_weight, float (&u)[8]) {
    float m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = a.residual_scale;
    if (a.gate != nullptr) {
        values_any(gate, a.gate_dtype, m);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] *= m[j];
    }
    if (a.post_weight != nullptr) {
        values_any(post_weight, a.post_weight_dtype, m);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] *= m[j];
    }
}
// A in s, B in u, in two steps of two vectors each.
__device__ __forceinline__ void start_ab(const feather_norm_args& a, const RawAny& scale, const RawAny& bias, float (&s)[8], float (&u)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = 1.0f, u[j] = 0.0f;
    if (a.scale != nullptr) {
        values_any(scale, a.scale_dtype, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += u[j], u[j] = 0.0f;
    }
    if (a.bias != nullptr) {
        values_any(bias, a.bias_dtype, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] *= s[j];
    }
}
__device__ __forceinline__ void finish_ab(const feather_norm_args& a, const RawAny& weight, const RawAny& shift, float (&s)[8], float (&u)[8]) {
    float m[8];
    if (a.shift != nullptr) {
        values_any(shift, a.shift_dtype, m);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] += m[j];
    }
    if (a.weight != nullptr) {
        values_any(weight, a.weight_dtype, m);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] *= m[j];
    }
}

// First row after `row` that belongs to another row of gate, scale or shift.
__device__ __forceinline__ long long next_change(const feather_norm_args& a, long long row) {
    long long change = a.rows;
    if (a.gate != nullptr) change = min(change, (share_of(row, a.gate_rows) + 1) * a.gate_rows);
    if (a.scale != nullptr) change = min(change, (share_of(row, a.scale_rows) + 1) * a.scale_rows);
    if (a.shift != nullptr) change = min(change, (share_of(row, a.shift_rows) + 1) * a.shift_rows);
    return change;
}

// Takes a thread's vector of the row to v - mean (layer) and returns 1 / sqrt(mean square + eps); in: the vector exists, it holds zeros otherwise.
// The variance is taken about the mean in a second pass over the registers: sums of squares of unshifted values lose a small variance beside a
// large mean.
__device__ __forceinline__ float normalise(float (&v)[8], const NormParams& p, bool in, float (*part)[kNormMaxWarps], int& flip) {
    if (p.a.kind == FEATHER_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
        const float mean = row_sum(s, part, flip) * p.inv_cols;
        if (in) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] -= mean;
        }
    }
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += v[j] * v[j];
    return 1.0f / sqrtf(row_sum(s, part, flip) * p.inv_cols + p.a.eps);
}

// One vector of h, given n.  All lanes of a warp call this together (the MXFP4 form exchanges between lanes); `in`: the vector exists.
__device__ __forceinline__ void store_h(const NormParams& p, long long row, int vec, bool in, const float (&h)[8]) {
    const feather_norm_args& a = p.a;
    if (a.h_scales != nullptr) {
        // the 16-bit value first, so that the bits are those of quantising the h this call would store
        const bool bf16 = a.h_dtype == FEATHER_SRC_BF16;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j += 2) unpack16x2(pack16x2(h[j], h[j + 1], bf16), bf16, f[j], f[j + 1]);
        uint32_t code;
        const uint32_t q = mx_quantize8(f, code);
        const uint32_t word = mx_scale_word(in ? code : 0u, threadIdx.x & 31);
        if (in) {
            static_cast<uint32_t*>(a.h)[row * a.ldh + vec] = q;
            if ((vec & 15) == 0) *reinterpret_cast<uint32_t*>(a.h_scales + mx_scale_word_offset(row, vec >> 4, mx_tiles_k(a.cols))) = word;
        }
    } else if (in) {
        if (a.h_dtype == FEATHER_SRC_BF16) store8<FEATHER_SRC_BF16>(a.h, row * a.ldh + vec * 8, h);
        else if (a.h_dtype == FEATHER_SRC_FP16) store8<FEATHER_SRC_FP16>(a.h, row * a.ldh + vec * 8, h);
        else store8<FEATHER_SRC_FP32>(a.h, row * a.ldh + vec * 8, h);
    }
}

template <int T>
__device__ __forceinline__ void values8(const Raw8<T>& r, F2 (&v)[4]) {
    float f[8];
    values8<T>(r, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f2(f[2 * j], f[2 * j + 1]);
}
__device__ __forceinline__ void split8(const F2 (&v)[4], float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f2_split(v[j], f[2 * j], f[2 * j + 1]);
}
__device__ __forceinline__ void join8(const float (&f)[8], F2 (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f2(f[2 * j], f[2 * j + 1]);
}

// ------------------------------------------------------------------------------------------------ many rows
// A block is `groups` groups of threads that each have a row of their own under way, so that one group's sums (shuffles, a barrier) lie
// under the others' arithmetic; it takes `chunk` consecutive rows, a wave of one row a group at a time.  The rows come through a ring in
// shared memory, `stages` rows for each group, that bulk copies fill ahead: what is in flight does not depend on the registers.  G, A and B
// lie in shared memory, once for the block, and are folded anew where a wave begins that belongs to other rows of gate, scale or shift
// (a wave ends there).
// Bound by the instructions around the arithmetic rather than by memory: 2 x 8192 x 5120 bf16 with fp32 gate, scale and shift of each
// sample takes 128 us as layer norm (5.2 TB/s of 671 MB), 156 us as a packed result, 185 us with a norm of y before it; a block for each
// row that reads its vectors from the cache takes 213 us for the first.  Leaving the loop when a wait runs out costs the first 1 us and the
// packed one 3 us (the vote after the wait); a flag that the rows test instead cost up to 10 us, and 20 us at 256 columns.
constexpr int kNormMaxStages = 4, kNormMaxGroups = 32, kNormMaxBarriers = 15;    // a group of one warp needs no barrier
// Registers of a thread.  POST: y may go through a norm first, and x has to wait for it in registers.  Without that norm r is formed as x
// and y are read, 96 registers are enough, and rows of 5120 have four groups instead of three (127 us where 128 registers take 141).
__host__ __device__ constexpr int norm_regs(int nv, bool post) { return nv == 4 && post ? 128 : nv == 1 ? 64 : 96; }

struct GroupBarrier {
    int id, threads;
    __device__ __forceinline__ void sync() const {
        if (threads == 32) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
    }
};

// A group's place for its warps' partial sums: two buffers in turn, so that one barrier for each sum is enough.
struct GroupSums {
    float2* part;                                                             // the second buffer kNormMaxWarps further on
    const float* elements;                                                    // of the row in each warp
    int warps, warp, flip;
};

// 1 / sqrt(mean square + eps) of the group's row; layer: v - mean first.  A warp takes its own mean and the squares about it, and the warps'
// results are joined about the row's mean: sums of squares of unshifted values lose a small variance beside a large mean.
template <int NV, bool FULL>
__device__ __forceinline__ float normalise_group(F2 (&v)[NV][4], const NormParams& p, int first, int step, const GroupBarrier& barrier, GroupSums& sums) {
    const auto total = [](float x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        return x;
    };
    const auto shift_by = [&](float by) {
        const F2 d = f2(by, by);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (FULL || first + i * step < p.vecs) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = f2_add(v[i][j], d);
            }
    };
    const bool layer = p.a.kind == FEATHER_NORM_LAYER;
    float mean = 0.0f, lo, hi;
    if (layer) {
        F2 t = v[0][0];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j != 0) t = f2_add(t, v[i][j]);                       // vectors past the row hold zeros
        f2_split(t, lo, hi);
        mean = total(lo + hi) / fmaxf(sums.elements[sums.warp], 1.0f);
        shift_by(-mean);
    }
    F2 q = f2_mul(v[0][0], v[0][0]);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j != 0) q = f2_fma(v[i][j], v[i][j], q);
    f2_split(q, lo, hi);
    float squares = total(lo + hi);
    if (sums.warps > 1) {
        float2* const part = sums.part + sums.flip * kNormMaxWarps;
        sums.flip ^= 1;
        if ((threadIdx.x & 31) == 0) part[sums.warp] = make_float2(mean, squares);
        barrier.sync();
        if (layer) {
            float all = 0.0f;
            for (int w = 0; w < sums.warps; ++w) all += part[w].x * sums.elements[w];
            all *= p.inv_cols;
            squares = 0.0f;
            for (int w = 0; w < sums.warps; ++w) {
                const float d = part[w].x - all;
                squares += part[w].y + d * d * sums.elements[w];
            }
            shift_by(mean - all);
        } else {
            squares = 0.0f;
            for (int w = 0; w < sums.warps; ++w) squares += part[w].y;
        }
    }
    return 1.0f / sqrtf(squares * p.inv_cols + p.a.eps);
}

template <int XT, int YT, int NV, bool KEEP, bool FULL, bool POST>
__global__ void __maxnreg__(norm_regs(NV, POST)) gated_norm_groups_kernel(const __grid_constant__ NormParams p) {
    __shared__ float2 part[2][kNormMaxWarps];                                 // by the block's warps
    __shared__ float elements[kNormMaxWarps];
    __shared__ __align__(8) uint64_t bars[kNormMaxGroups][kNormMaxStages];
    __shared__ int abort_flag;
    extern __shared__ __align__(128) float4 dynamic[];
    const feather_norm_args& a = p.a;
    constexpr int kXSize = XT == FEATHER_SRC_FP32 ? 4 : 2, kYSize = YT == FEATHER_SRC_FP32 ? 4 : 2;
    const int step = blockDim.x / p.groups;                                   // threads of a group
    const int group = threadIdx.x / step, t = threadIdx.x - group * step;
    const bool has_y = a.y != nullptr;
    const int present = norm_present(a);
    const uint32_t x_bytes = static_cast<uint32_t>(a.cols) * kXSize, y_bytes = has_y ? static_cast<uint32_t>(a.cols) * kYSize : 0u, row_bytes = x_bytes + y_bytes;
    // coefficients: [G | A | B][two 16-byte halves][vectors]
    const float4* const kept = dynamic;
    const int kept_step = 2 * p.vecs;
    uint8_t* const ring = reinterpret_cast<uint8_t*>(dynamic + (KEEP && present != 0 ? 3 * kept_step : 0)) + group * p.stages * row_bytes;
    const uint32_t bar0 = smem_u32(bars[group]);
    if (t == 0) {
        for (int s = 0; s < p.stages; ++s) mbar_init(bar0 + 8 * s, 1);
        if (group == 0) abort_flag = 0;
        fence_mbar_init();
    }
    if (threadIdx.x < step / 32) {
        int n = 0;
        for (int i = 0; i < NV; ++i) n += max(0, min(32, p.vecs - i * step - 32 * static_cast<int>(threadIdx.x)));
        elements[threadIdx.x] = static_cast<float>(8 * n);
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();
    const GroupBarrier barrier{1 + group, step};
    GroupSums sums{part[0] + group * (step / 32), elements, step / 32, t / 32, 0};
    const long long begin = static_cast<long long>(blockIdx.x) * p.chunk, end = begin + p.chunk < a.rows ? begin + p.chunk : a.rows;
    // A wave: rows wave .. wave + groups - 1, one a group, short of the next change of coefficients.
    long long fetch_wave = begin, fetch_change = begin;
    int fetch_slot = 0;
    const auto fetch = [&]() {                                                // by the group's first thread: its next row, if it has one
        while (fetch_wave < end) {
            if (fetch_wave >= fetch_change) fetch_change = KEEP ? min(end, next_change(a, fetch_wave)) : end;
            const long long row = fetch_wave + group;
            fetch_wave = min(fetch_wave + p.groups, fetch_change);
            if (row >= fetch_change) continue;
            const uint32_t bar = bar0 + 8 * fetch_slot, to = smem_u32(ring) + fetch_slot * row_bytes;
            mbar_arrive_expect_tx(bar, row_bytes);
            bulk_load(to, static_cast<const uint8_t*>(a.x) + row * a.ldx * kXSize, x_bytes, bar);
            if (has_y) bulk_load(to + x_bytes, static_cast<const uint8_t*>(a.y) + row * a.ldy * kYSize, y_bytes, bar);
            if (++fetch_slot == p.stages) fetch_slot = 0;
            return;
        }
    };
    if (t == 0)
        for (int s = 0; s < p.stages; ++s) fetch();
    const auto fold = [&](long long first) {                                  // the coefficients of the rows from `first` on, by the whole block
        __syncthreads();                                                      // nobody reads the old ones any more
        const ModulationAt m = modulation_at(a, first);
        for (int vec = threadIdx.x; vec < p.vecs; vec += blockDim.x) {
            RawAny q, w;
            float f[8], h[8];
            if (present & kNormG) {
                load_any(q, a.gate, a.gate_dtype, m.gate + vec * 8);
                load_any(w, a.post_weight, a.post_weight_dtype, vec * 8);
                fold_g(a, q, w, f);
                dynamic[vec] = make_float4(f[0], f[1], f[2], f[3]);
                dynamic[p.vecs + vec] = make_float4(f[4], f[5], f[6], f[7]);
            }
            if (present & (kNormA | kNormB)) {
                load_any(q, a.scale, a.scale_dtype, m.scale + vec * 8);
                load_any(w, a.bias, a.bias_dtype, vec * 8);
                start_ab(a, q, w, f, h);
                load_any(q, a.weight, a.weight_dtype, vec * 8);
                load_any(w, a.shift, a.shift_dtype, m.shift + vec * 8);
                finish_ab(a, q, w, f, h);
                dynamic[kept_step + vec] = make_float4(f[0], f[1], f[2], f[3]);
                dynamic[kept_step + p.vecs + vec] = make_float4(f[4], f[5], f[6], f[7]);
                dynamic[2 * kept_step + vec] = make_float4(h[0], h[1], h[2], h[3]);
                dynamic[2 * kept_step + p.vecs + vec] = make_float4(h[4], h[5], h[6], h[7]);
            }
        }
        __syncthreads();
    };
    long long wave = begin, change = begin;
    int slot = 0;
    uint32_t parity = 0;
    for (; wave < end; wave = min(wave + p.groups, change)) {
        if (wave >= change) {
            change = KEEP ? min(end, next_change(a, wave)) : end;
            if (KEEP && present != 0) fold(wave);
        }
        const long long row = wave + group;
        if (row >= change) continue;                                          // a whole group
        if (!__all_sync(0xffffffffu, mbar_wait_within(bar0 + 8 * slot, parity, &abort_flag, p.wait_ns))) break;     // the warp is lost
        const uint8_t* const from = ring + slot * row_bytes;
        if (++slot == p.stages) {
            slot = 0;
            parity ^= 1u;
        }
        ModulationAt m{};
        if constexpr (!KEEP) m = modulation_at(a, row);
        const auto coefficient = [&](int c, int vec, F2(&v)[4]) {
            const float4 x = kept[c * kept_step + vec], y = kept[c * kept_step + p.vecs + vec];
            v[0] = f2(x.x, x.y);
            v[1] = f2(x.z, x.w);
            v[2] = f2(y.x, y.y);
            v[3] = f2(y.z, y.w);
        };
        const auto residual = [&](int i, const Raw8<XT>& x_raw, F2(&y)[4], F2 by) {  // r of one vector, in y's place
            const int vec = t + i * step;
            F2 g[4], x[4];
            float f[8];
            if (!(present & kNormG)) {
#pragma unroll
                for (int j = 0; j < 4; ++j) g[j] = f2(a.residual_scale, a.residual_scale);
            } else if constexpr (KEEP) {
                coefficient(0, vec, g);
            } else {
                RawAny q, w;
                load_any(q, a.gate, a.gate_dtype, m.gate + vec * 8);
                load_any(w, a.post_weight, a.post_weight_dtype, vec * 8);
                fold_g(a, q, w, f);
                join8(f, g);
            }
            values8<XT>(x_raw, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = f2_fma(g[j], POST ? f2_mul(y[j], by) : y[j], x[j]);
            if (a.r != nullptr) {
                split8(y, f);
                store8<XT>(a.r, row * a.ldr + vec * 8, f);
            }
        };
        Raw8<XT> xr[POST ? NV : 1];
        F2 v[NV][4];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int vec = t + i * step;
            if (FULL || vec < p.vecs) {
                Raw8<XT>& x = xr[POST ? i : 0];
                x = reinterpret_cast<const Raw8<XT>*>(from)[vec];
                if (has_y) values8<YT>(reinterpret_cast<const Raw8<YT>*>(from + x_bytes)[vec], v[i]);
                else values8<XT>(x, v[i]);
                if (!POST && has_y) residual(i, x, v[i], F2{});
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = f2(0.0f, 0.0f);
            }
        }
        barrier.sync();                                                       // every thread has its part in registers
        if (t == 0) fetch();
        if constexpr (POST) {
            if (has_y) {
                const float inv = a.post_norm ? normalise_group<NV, FULL>(v, p, t, step, barrier, sums) : 1.0f;
                const F2 by = f2(inv, inv);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (FULL || t + i * step < p.vecs) residual(i, xr[i], v[i], by);
            }
        }
        if (a.h == nullptr) continue;
        const float inv = normalise_group<NV, FULL>(v, p, t, step, barrier, sums);
        const F2 by = f2(inv, inv);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int vec = t + i * step;
            [[maybe_unused]] float f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = f2_mul(v[i][j], by);
            if ((present & (kNormA | kNormB)) && (FULL || vec < p.vecs)) {
                F2 s[4], u[4];
                if constexpr (KEEP) {
                    coefficient(1, vec, s);
                    coefficient(2, vec, u);
                } else {
                    RawAny q, w;
                    float h[8];
                    load_any(q, a.scale, a.scale_dtype, m.scale + vec * 8);
                    load_any(w, a.bias, a.bias_dtype, vec * 8);
                    start_ab(a, q, w, f, h);
                    load_any(q, a.weight, a.weight_dtype, vec * 8);
                    load_any(w, a.shift, a.shift_dtype, m.shift + vec * 8);
                    finish_ab(a, q, w, f, h);
                    join8(f, s);
                    join8(h, u);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = f2_fma(v[i][j], s[j], u[j]);
            }
        }
        const long long h_at = row * a.ldh + t * 8;
        const auto store_all = [&](auto type) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float f[8];
                split8(v[i], f);
                if (FULL || t + i * step < p.vecs) store8<decltype(type)::value>(a.h, h_at + i * step * 8, f);
            }
        };
        if (a.h_scales != nullptr) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float f[8];
                split8(v[i], f);
                store_h(p, row, t + i * step, FULL || t + i * step < p.vecs, f);
            }
        } else if (a.h_dtype == FEATHER_SRC_BF16) {
            store_all(std::integral_constant<int, FEATHER_SRC_BF16>{});
        } else if (a.h_dtype == FEATHER_SRC_FP16) {
            store_all(std::integral_constant<int, FEATHER_SRC_FP16>{});
        } else {
            store_all(std::integral_constant<int, FEATHER_SRC_FP32>{});
        }
    }
    if (wave >= end) return;
    // A warp whose wait ran out reads and stores nothing from there on and keeps to the barriers; its part of a sum is NaN, and so is every h
    // that would be made of it. The warp that fetches starts no further copy (its group's other warps are lost where a row was never fetched)
    // and lets those in flight land, before the block gives its memory back.
    abort_flag = 1;
    if (a.status_dev != nullptr) atomicCAS(a.status_dev, 0, FEATHER_ERR_DEVICE_TIMEOUT | (1 << 8));
    if (t == 0) {
        const uint64_t begin_ns = globaltimer_ns();
        long long until = change;
        for (long long w = wave; w < fetch_wave; w = min(w + p.groups, until)) {             // as `fetch` went
            if (w >= until) until = KEEP ? min(end, next_change(a, w)) : end;
            if (w + group >= until) continue;
            while (!mbar_try_wait(bar0 + 8 * slot, parity) && globaltimer_ns() - begin_ns < kWaitLimitNs) {
            }
            if (++slot == p.stages) {
                slot = 0;
                parity ^= 1u;
            }
        }
    }
    __syncwarp();
    const int rounds = 1 + (sums.warps > 1 ? (POST && has_y && a.post_norm ? 1 : 0) + (a.h != nullptr ? 1 : 0) : 0);      // barriers of a row
#pragma unroll 1
    for (; wave < end; wave = min(wave + p.groups, change)) {
        if (wave >= change) {
            change = KEEP ? min(end, next_change(a, wave)) : end;
            if (KEEP && present != 0) fold(wave);
        }
        if (wave + group >= change) continue;
        barrier.sync();
#pragma unroll 1
        for (int i = 1; i < rounds; ++i) {
            if ((threadIdx.x & 31) == 0) sums.part[sums.flip * kNormMaxWarps + sums.warp] = make_float2(__int_as_float(0x7FC00000), __int_as_float(0x7FC00000));
            sums.flip ^= 1;
            barrier.sync();
        }
    }
}

// Few rows, or a modulation for each row: a block takes one row.  DENSE: 48 registers instead of 64, with spills, so that two blocks of a
// wide row fit an SM (4096 x 5120 bf16 with fp32 modulation of each row: 129 -> 101 us); one row alone takes 4.6 us that way, 4.1 us otherwise.
template <int XT, int YT, bool DENSE>
__global__ void __maxnreg__(DENSE ? 48 : 64) gated_norm_row_kernel(const __grid_constant__ NormParams p) {
    __shared__ __align__(16) float part[2][kNormMaxWarps];
    const feather_norm_args& a = p.a;
    clear_parts(part);
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();
    const long long row = blockIdx.x;
    const int vec = threadIdx.x, at = vec * 8;
    const bool in = vec < p.vecs;
    const int present = norm_present(a);
    const ModulationAt m = modulation_at(a, row);
    Raw8<XT> xr;
    Raw8<YT> yr;
    RawAny gate, post_weight;
    if (in) {
        if (a.y != nullptr) {
            yr = load8<YT>(a.y, row * a.ldy + at);
            load_any(gate, a.gate, a.gate_dtype, m.gate + at);
            load_any(post_weight, a.post_weight, a.post_weight_dtype, at);
        }
        xr = load8<XT>(a.x, row * a.ldx + at);
    }
    int flip = 0;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    if (a.y != nullptr) {
        if (in) values8<YT>(yr, v);
        const float inv = a.post_norm ? normalise(v, p, in, part, flip) : 1.0f;
        if (in) {
            float g[8], x[8];
            fold_g(a, gate, post_weight, g);
            values8<XT>(xr, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = x[j] + g[j] * (v[j] * inv);
            if (a.r != nullptr) store8<XT>(a.r, row * a.ldr + at, v);
        }
    } else if (in) {
        values8<XT>(xr, v);
    }
    if (a.h == nullptr) return;
    RawAny weight, bias, scale, shift;                                        // on their way during the sums
    if (in) {
        load_any(scale, a.scale, a.scale_dtype, m.scale + at);
        load_any(shift, a.shift, a.shift_dtype, m.shift + at);
        load_any(weight, a.weight, a.weight_dtype, at);
        load_any(bias, a.bias, a.bias_dtype, at);
    }
    const float inv = normalise(v, p, in, part, flip);
    if (in) {
        float s[8], u[8];
        start_ab(a, scale, bias, s, u);
        finish_ab(a, weight, shift, s, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float n = v[j] * inv;
            if (present & kNormA) n *= s[j];
            if (present & kNormB) n += u[j];
            v[j] = n;
        }
    }
    store_h(p, row, vec, in, v);
}

// ------------------------------------------------------------------------------------------------ single elements
// Rows that are not 16-byte aligned or not a multiple of eight long: a block takes a row, a warp NE * 32 elements of it, a lane every 32nd of
// those, so that a thread's addresses are one pointer and constants.  Element i exists if 32 i < left.
// Bound by instructions (79 % of the issue slots where the row's threads took every blockDim-th element: 36 us for 4000 x 1027 fp16 with a
// norm of y and a modulation, 21 us this way); a second copy of the code for warps whose part is whole, without the checks, takes 28 us.
template <int NE>
__device__ __forceinline__ void load_elements(uint32_t (&r)[NE], const void* base, int type, long long at, int left) {
    if (base == nullptr) return;
    if (type == FEATHER_SRC_FP32) {
        const uint32_t* const q = static_cast<const uint32_t*>(base) + at;
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (32 * i < left) r[i] = q[32 * i];
    } else {
        const uint16_t* const q = static_cast<const uint16_t*>(base) + at;
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (32 * i < left) r[i] = q[32 * i];
    }
}
// The type is looked at once for a thread's elements, not for each.
template <int NE, typename Op>
__device__ __forceinline__ void each_element(const uint32_t (&r)[NE], int type, Op op) {
    if (type == FEATHER_SRC_FP32) {
#pragma unroll
        for (int i = 0; i < NE; ++i) op(i, __uint_as_float(r[i]));
    } else if (type == FEATHER_SRC_BF16) {
#pragma unroll
        for (int i = 0; i < NE; ++i) op(i, __uint_as_float(r[i] << 16));
    } else {
#pragma unroll
        for (int i = 0; i < NE; ++i) op(i, __half2float(__ushort_as_half(static_cast<uint16_t>(r[i]))));
    }
}
template <int NE>
__device__ __forceinline__ void store_elements(void* base, int type, long long at, int left, const float (&v)[NE]) {
    const auto store = [&](auto* o, auto convert) {
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (32 * i < left) o[32 * i] = convert(v[i]);
    };
    if (type == FEATHER_SRC_FP32) store(static_cast<float*>(base) + at, [](float f) { return f; });
    else if (type == FEATHER_SRC_BF16) store(static_cast<__nv_bfloat16*>(base) + at, [](float f) { return __float2bfloat16_rn(f); });
    else store(static_cast<__half*>(base) + at, [](float f) { return __float2half_rn(f); });
}

template <int NE>
__device__ __forceinline__ float normalise_elements(float (&v)[NE], const NormParams& p, int left, float (*part)[kNormMaxWarps], int& flip) {
    if (p.a.kind == FEATHER_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NE; ++i) s += v[i];
        const float mean = row_sum(s, part, flip) * p.inv_cols;
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (32 * i < left) v[i] -= mean;
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) s += v[i] * v[i];
    return 1.0f / sqrtf(row_sum(s, part, flip) * p.inv_cols + p.a.eps);
}

// EARLY: what makes r is loaded together, what makes h of it before the second norm's sums; otherwise each where it is used.  48 registers there
// (62 without the bound) let all of 999 rows of 1027 be resident at once: 7.9 us and 9.1 us with a modulation of each row, and 8.9 us with 40.
template <int NE, bool EARLY>
__global__ void __launch_bounds__(EARLY ? 256 : 1024, EARLY ? 5 : 1) gated_norm_elements_kernel(const __grid_constant__ NormParams p) {
    __shared__ __align__(16) float part[2][kNormMaxWarps];
    const feather_norm_args& a = p.a;
    clear_parts(part);
    pdl_launch_dependents();
    pdl_wait_for_previous_kernel();
    const long long row = blockIdx.x;
    const int at = (threadIdx.x >> 5) * (32 * NE) + (threadIdx.x & 31), left = p.vecs - at;
    int flip = 0;
    const ModulationAt m = modulation_at(a, row);
    uint32_t x[NE] = {}, y[NE] = {}, gate[NE], post_weight[NE], weight[NE], bias[NE], scale[NE], shift[NE];
    load_elements<NE>(x, a.x, a.x_dtype, row * a.ldx + at, left);
    load_elements<NE>(y, a.y, a.y_dtype, row * a.ldy + at, left);
    const auto load_before = [&]() {
        load_elements<NE>(gate, a.gate, a.gate_dtype, m.gate + at, left);
        load_elements<NE>(post_weight, a.post_weight, a.post_weight_dtype, at, left);
    };
    if (EARLY) load_before();
    float v[NE];                                                              // elements past the row are zero until the sums are done
    if (a.y != nullptr) {
        each_element<NE>(y, a.y_dtype, [&](int i, float e) { v[i] = e; });
        const float inv = a.post_norm ? normalise_elements<NE>(v, p, left, part, flip) : 1.0f;
        if (!EARLY) load_before();
#pragma unroll
        for (int i = 0; i < NE; ++i) v[i] *= inv * a.residual_scale;
        if (a.gate != nullptr) each_element<NE>(gate, a.gate_dtype, [&](int i, float e) { v[i] *= e; });
        if (a.post_weight != nullptr) each_element<NE>(post_weight, a.post_weight_dtype, [&](int i, float e) { v[i] *= e; });
        each_element<NE>(x, a.x_dtype, [&](int i, float e) { v[i] = 32 * i < left ? v[i] + e : 0.0f; });
        if (a.r != nullptr) store_elements<NE>(a.r, a.x_dtype, row * a.ldr + at, left, v);
    } else {
        each_element<NE>(x, a.x_dtype, [&](int i, float e) { v[i] = e; });
    }
    if (a.h == nullptr) return;
    if (EARLY) {
        load_elements<NE>(weight, a.weight, a.weight_dtype, at, left);
        load_elements<NE>(bias, a.bias, a.bias_dtype, at, left);
        load_elements<NE>(scale, a.scale, a.scale_dtype, m.scale + at, left);
        load_elements<NE>(shift, a.shift, a.shift_dtype, m.shift + at, left);
    }
    const float inv = normalise_elements<NE>(v, p, left, part, flip);
#pragma unroll
    for (int i = 0; i < NE; ++i) v[i] *= inv;
    const auto apply = [&](uint32_t(&r)[NE], const void* base, int type, long long from, auto op) {
        if (base == nullptr) return;
        if (!EARLY) load_elements<NE>(r, base, type, from, left);
        each_element<NE>(r, type, op);
    };
    apply(weight, a.weight, a.weight_dtype, at, [&](int i, float e) { v[i] *= e; });
    apply(bias, a.bias, a.bias_dtype, at, [&](int i, float e) { v[i] += e; });
    apply(scale, a.scale, a.scale_dtype, m.scale + at, [&](int i, float e) { v[i] *= 1.0f + e; });
    apply(shift, a.shift, a.shift_dtype, m.shift + at, [&](int i, float e) { v[i] += e; });
    store_elements<NE>(a.h, a.h_dtype, row * a.ldh + at, left, v);
}

// ------------------------------------------------------------------------------------------------ launches
// Limit of a wait for a row of the ring: two seconds, or what FEATHER_NORM_WAIT_NS says if that is less (0: a row that is not there at the
// first look counts as lost, which is how giving up is tested).
static uint64_t norm_wait_ns() {
    static const uint64_t ns = [] {
        const char* const text = getenv("FEATHER_NORM_WAIT_NS");
        char* rest = nullptr;
        const unsigned long long asked = text != nullptr ? strtoull(text, &rest, 10) : 0;
        if (text == nullptr || rest == text || *rest != '\0') return kWaitLimitNs;             // unset, or not a number
        return asked < kWaitLimitNs ? static_cast<uint64_t>(asked) : kWaitLimitNs;
    }();
    return ns;
}

constexpr int kNormMaxSmem = 225 * 1024;      // dynamic, beside the sums and barriers

// One block an SM: its groups take the registers, its ring the shared memory. A block has consecutive rows.
template <int XT, int YT, int NV, bool KEEP, bool FULL, bool POST>
static cudaError_t norm_launch_groups_kernel(NormParams p, int threads, int smem, int sms, cudaStream_t stream) {
    static SmemOptIn opt_in;
    const cudaError_t e = opt_in(gated_norm_groups_kernel<XT, YT, NV, KEEP, FULL, POST>, kNormMaxSmem);
    if (e != cudaSuccess) return e;
    p.chunk = static_cast<int>((p.a.rows + sms - 1) / sms);
    return launch_dependent(gated_norm_groups_kernel<XT, YT, NV, KEEP, FULL, POST>, dim3(static_cast<unsigned>((p.a.rows + p.chunk - 1) / p.chunk)),
                            dim3(static_cast<unsigned>(threads * p.groups)), 0, smem, stream, p);
}

template <int XT, int YT>
static int norm_row_bytes(const feather_norm_args& a) {
    return static_cast<int>(a.cols) * ((XT == FEATHER_SRC_FP32 ? 4 : 2) + (a.y == nullptr ? 0 : YT == FEATHER_SRC_FP32 ? 4 : 2));
}

template <int XT, int YT, int NV, bool POST>
static cudaError_t norm_launch_groups(NormParams p, int sms, bool shared, cudaStream_t stream) {
    const int threads = (p.vecs + 32 * NV - 1) / (32 * NV) * 32;
    const int row_bytes = norm_row_bytes<XT, YT>(p.a);
    const int kept = norm_present(p.a) != 0 ? 3 * 32 * p.vecs : 0;
    // As many groups as its registers hold, each with two rows of ring at least; the coefficients stay in shared memory
    // if one group's row fits beside them.
    const bool keep = shared && kept + row_bytes <= kNormMaxSmem;
    const int room = kNormMaxSmem - (keep ? kept : 0);
    p.groups = 65536 / norm_regs(NV, POST) / 128 * 128 / threads;             // registers go to four warps at a time
    if (threads > 32 && p.groups > kNormMaxBarriers) p.groups = kNormMaxBarriers;
    if (p.groups * threads > 1024) p.groups = 1024 / threads;
    while (p.groups > 1 && p.groups * 2 * row_bytes > room) --p.groups;
    if (p.groups < 1) return cudaErrorInvalidConfiguration;
    p.stages = room / (p.groups * row_bytes);
    if (p.stages > kNormMaxStages) p.stages = kNormMaxStages;
    if (p.stages < 1) return cudaErrorInvalidConfiguration;
    const int smem = (keep ? kept : 0) + p.groups * p.stages * row_bytes;
    if (!keep && !(NV == 4 && POST)) return cudaErrorInvalidConfiguration;
    if constexpr (NV == 4 && POST)
        if (!keep) return norm_launch_groups_kernel<XT, YT, NV, false, false, POST>(p, threads, smem, sms, stream);
    return p.vecs == threads * NV ? norm_launch_groups_kernel<XT, YT, NV, true, true, POST>(p, threads, smem, sms, stream)
                                  : norm_launch_groups_kernel<XT, YT, NV, true, false, POST>(p, threads, smem, sms, stream);
}

template <int XT, int YT>
static cudaError_t norm_launch_typed(const NormParams& p, int sms, cudaStream_t stream) {
    const feather_norm_args& a = p.a;
    // rows that share a row of each modulation
    int64_t shared = a.rows;
    if (a.gate != nullptr && a.gate_rows < shared) shared = a.gate_rows;
    if (a.scale != nullptr && a.scale_rows < shared) shared = a.scale_rows;
    if (a.shift != nullptr && a.shift_rows < shared) shared = a.shift_rows;
    // A block for each row up to two waves of them (16 of narrow rows: 2080 x 1024 fp32 7.8 us against 8.6 us, 1000 x 5120 27 us against 17 us),
    // and where every row has a modulation of its own.  bf16 with a norm of y, a block a row against groups: 600 x 256 3.2 and 6.5 us, 2368 x 512 5.8
    // and 6.5, 4800 x 512 10.7 and 9.0; 600 x 1024 4.7 and 6.1, but 1200 x 1024 7.1 and 6.4; 300 x 2048 4.8 and 6.6, 600 x 2048 7.3 and 7.0; 150 x 5120
    // 7.8 and 7.8, 300 x 5120 10.2 and 8.8.
    if (p.vecs <= 1024 && (shared < 4 || a.rows <= (p.vecs <= 128 ? 16 : 2) * sms)) {
        const dim3 grid(static_cast<unsigned>(a.rows)), block((p.vecs + 31) / 32 * 32);
        return a.rows > 2 * sms && p.vecs > 512
                   ? launch_dependent(gated_norm_row_kernel<XT, YT, true>, grid, block, 0, 0, stream, p)
                   : launch_dependent(gated_norm_row_kernel<XT, YT, false>, grid, block, 0, 0, stream, p);
    }
    if (p.vecs <= 32) return norm_launch_groups<XT, YT, 1, true>(p, sms, shared >= 4, stream);
    if (p.vecs <= 64) return norm_launch_groups<XT, YT, 2, true>(p, sms, shared >= 4, stream);
    // The form without a norm of y, for the pairs of types that models have; it has its coefficients in shared memory always, and above 1536
    // vectors 96 registers give no further group (16384 rows of 6144: 95 -> 79 us, 8192: 153 -> 113 us; fp32 2 x 2048 x 5120 127 -> 96 us;
    // an rms norm with a weight alone, which is nearest to the memory's rate, loses 123 -> 128 us).
    if constexpr (XT == YT || XT == FEATHER_SRC_FP32)
        if (!a.post_norm && shared >= 4 && p.vecs <= 1536 && 96 * p.vecs + norm_row_bytes<XT, YT>(a) <= kNormMaxSmem)
            return norm_launch_groups<XT, YT, 4, false>(p, sms, true, stream);
    return norm_launch_groups<XT, YT, 4, true>(p, sms, shared >= 4, stream);
}

static cudaError_t norm_launch(const NormParams& p, int sms, cudaStream_t stream) {
    constexpr int F = FEATHER_SRC_FP32, B = FEATHER_SRC_BF16, H = FEATHER_SRC_FP16;
    const int y = p.a.y != nullptr ? p.a.y_dtype : p.a.x_dtype;
    switch (p.a.x_dtype * 3 + y) {
        case F * 3 + F: return norm_launch_typed<F, F>(p, sms, stream);
        case F * 3 + B: return norm_launch_typed<F, B>(p, sms, stream);
        case F * 3 + H: return norm_launch_typed<F, H>(p, sms, stream);
        case B * 3 + F: return norm_launch_typed<B, F>(p, sms, stream);
        case B * 3 + B: return norm_launch_typed<B, B>(p, sms, stream);
        case B * 3 + H: return norm_launch_typed<B, H>(p, sms, stream);
        case H * 3 + F: return norm_launch_typed<H, F>(p, sms, stream);
        case H * 3 + B: return norm_launch_typed<H, B>(p, sms, stream);
        default: return norm_launch_typed<H, H>(p, sms, stream);
    }
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
    a.gate_rows = a.gate_rows < a.rows ? a.gate_rows : a.rows;                 // 31 bits
    a.scale_rows = a.scale_rows < a.rows ? a.scale_rows : a.rows;
    a.shift_rows = a.shift_rows < a.rows ? a.shift_rows : a.rows;
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
    p.wait_ns = norm_wait_ns();
    p.vecs = static_cast<int>(vector ? a.cols / 8 : a.cols);
    const int sms = sm_count();
    if (sms < 1) return set_error(FEATHER_ERR_CUDA, "the number of SMs could not be read");
    cudaError_t e;
    const dim3 grid(static_cast<unsigned>(a.rows));
    const auto block = [&](int n) { return dim3((p.vecs + 32 * n - 1) / (32 * n) * 32); };
    if (vector) e = norm_launch(p, sms, stream);
    else if (p.vecs <= 2048) e = launch_dependent(gated_norm_elements_kernel<8, true>, grid, block(8), 0, 0, stream, p);
    else e = launch_dependent(gated_norm_elements_kernel<16, false>, grid, block(16), 0, 0, stream, p);
    if (e != cudaSuccess) return set_error(FEATHER_ERR_CUDA, "gated_norm launch failed: %s", cudaGetErrorString(e));
    return FEATHER_OK;
}
