// linear.cuh -- shared parts of the dense, grouped and routed products.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>

#include "common.cuh"

namespace spmm {

constexpr float kSlopeUnit = 1.f / 16384.f;   // of the 16-bit fixed-point act'(z)

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// 8 16-bit values (16 bytes) as floats and back.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &v, float (&f)[8]) {
    T t[8];
    memcpy(t, &v, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32(t[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(f[i]);
    uint4 v;
    memcpy(&v, t, 16);
    return v;
}

// Whether every pointer (null too) lies on a boundary of `bytes`, a power of two.
inline bool on_boundary(size_t bytes, std::initializer_list<const void *> pointers) {
    uintptr_t all = 0;
    for (const void *p : pointers) all |= (uintptr_t)p;
    return (all & (bytes - 1)) == 0;
}

// First row of group g (offsets clamped into [0, total], so a wrong table reads and writes nothing outside; the
// first group starts at 0 whatever the table says, so that no row before it stays unwritten).
__device__ __forceinline__ int64_t group_first(const int32_t *offsets, int64_t g, int64_t total) {
    if (g == 0) return 0;
    const int64_t o = __ldg(offsets + g);
    return o < 0 ? 0 : o > total ? total : o;
}

// Chained launches.  Every kernel of these operators starts with chained_start():
// its blocks may be launched as soon as the blocks of the kernel before it on
// the stream have ended, set themselves up, and wait there until that kernel's
// writes are visible; nothing in global memory is read or written before.  Every
// thread waits, so that a kernel never ends before the one it follows.  Forward
// and backward of 512 x 1536 x 2304, call after call: 66 -> 56 us.  (Letting the
// next kernel in at the start of this one instead: 61 us; its blocks then sit on
// the SMs that this one's last blocks want.)
__device__ __forceinline__ void chained_start() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
int launch_chained(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t shared, cudaStream_t s, int cluster,
                   Args &&...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kernel, Params(args)...) != cudaSuccess) {
        (void)cudaGetLastError();
        return SPMM_ECUDA;
    }
    note_product_launch();
    return SPMM_OK;
}

// A tile of up to `size` consecutive rows of one group; group == groups is the
// tail of rows behind the last group, group > groups no tile.
struct RowTile {
    int64_t group, first;
    int rows;
};

// The t-th tile when every group's rows (and then the tail's) are cut into
// tiles of `size` rows.  Called by a whole warp; a prefix sum over 32 groups
// at a time.
__device__ __forceinline__ RowTile find_row_tile(const int32_t *offsets, int64_t groups, int64_t total, int size,
                                                 int64_t t) {
    RowTile r{groups + 1, 0, 0};
    if (offsets == nullptr) {
        if (t * size < total) {
            const int64_t left = total - t * size;
            r = RowTile{0, t * size, (int)(left < size ? left : size)};
        }
        return r;
    }
    const int lane = threadIdx.x & 31;
    int64_t before = 0;
    for (int64_t g0 = 0; g0 <= groups; g0 += 32) {
        const int64_t g = g0 + lane;
        int64_t a = 0, b = 0;
        if (g <= groups) {
            a = group_first(offsets, g, total);
            b = g < groups ? group_first(offsets, g + 1, total) : total;
            if (b < a) b = a;
        }
        const int64_t tiles = (b - a + size - 1) / size;
        int64_t incl = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(kFullMask, incl, o);
            if (lane >= o) incl += v;
        }
        const unsigned past = __ballot_sync(kFullMask, before + incl > t);
        if (past) {
            const int l = __ffs(past) - 1;
            const int64_t first = a + (t - before - (incl - tiles)) * size;
            const int64_t left = b - first;
            r.group = g0 + l;
            r.first = __shfl_sync(kFullMask, first, l);
            r.rows = (int)__shfl_sync(kFullMask, left < size ? left : (int64_t)size, l);
            return r;
        }
        before += __shfl_sync(kFullMask, incl, 31);
    }
    return r;
}

// The activation and its derivative at z.  Exponentials and reciprocals are the
// hardware's (about 2^-21 relative near 0, growing with |z|; far below a 16-bit
// rounding): with expf and full divisions the epilogue of an 8192 x 16384 x 4096
// product took longer than the product.  Far out each function is at its limit,
// which also keeps 0 * inf away.
__device__ __forceinline__ float exp2_fast(float x) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
    return e;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float sigmoid_fast(float z) {
    return reciprocal_fast(1.f + exp2_fast(z * -1.4426950408889634f));
}

// The normal distribution function at -v, v >= 0, for bell = exp(-v^2 / 2): bell
// times 0.5 exp(v^2 / 2) erfc(v / sqrt 2), which falls smoothly from 0.5 and is a
// polynomial in t = 1 / (1 + 0.3 v) to 4e-7 of its value up to v = 14 (a minimax fit
// of degree 8 to 64-bit values; degree 7: 9e-7).  A difference 0.5 - 0.5 erf(v /
// sqrt 2) was 4 % off at v = 5, and with CUDA's erfcf a gelu of 8192 x 512 x 8192 took
// 215 us (with its erff 145, so 115).
__device__ __forceinline__ float normal_tail(float v, float bell) {
    const float t = reciprocal_fast(fmaf(0.3f, v, 1.f));
    float m = 0.0383915901184082f;
    m = fmaf(m, t, -0.16923069953918457f);
    m = fmaf(m, t, 0.22879335284233093f);
    m = fmaf(m, t, -0.076658695936203f);
    m = fmaf(m, t, 0.14264048635959625f);
    m = fmaf(m, t, 0.0946388989686966f);
    m = fmaf(m, t, 0.12193173170089722f);
    m = fmaf(m, t, 0.11948609352111816f);
    m = fmaf(m, t, 7.26198595657479e-06f);
    return bell * m;
}

template <int ACT, bool SLOPE>
__device__ __forceinline__ float activate(float z, float &d) {
    if constexpr (ACT == SPMM_ACT_RELU) {
        if constexpr (SLOPE) d = z > 0.f ? 1.f : 0.f;
        return z < 0.f ? 0.f : z;                     // NaN stays
    } else if constexpr (ACT == SPMM_ACT_SILU) {
        const float s = sigmoid_fast(z), y = z < -100.f ? 0.f : z * s;
        if constexpr (SLOPE) d = z > 80.f ? 1.f : fmaf(y, 1.f - s, s);
        return y;
    } else if constexpr (ACT == SPMM_ACT_GELU) {
        const float bell = exp2_fast(z * z * -0.72134752044448170f), tail = normal_tail(fabsf(z), bell);
        const float cdf = z > 0.f ? 1.f - tail : tail;
        if constexpr (SLOPE)
            d = fabsf(z) > 12.f ? (z > 0.f ? 1.f : 0.f) : fmaf(z * 0.3989422804014327f, bell, cdf);
        return z < -14.f ? 0.f : z * cdf;                // below 2^-126
    } else if constexpr (ACT == SPMM_ACT_GELU_TANH) {
        // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), 2 u = 2 sqrt(2 / pi) (z + 0.044715 z^3)
        const float z2 = z * z;
        const float s = sigmoid_fast(1.5957691216057308f * z * fmaf(0.044715f, z2, 1.f));
        const float y = z < -12.f ? 0.f : z * s;
        if constexpr (SLOPE)
            d = fabsf(z) > 12.f ? (z > 0.f ? 1.f : 0.f)
                                : fmaf(y * (1.f - s), fmaf(0.21406445f, z2, 1.5957691216057308f), s);
        return y;
    } else {
        d = 1.f;
        return z;
    }
}

// act'(z) in 16 bits.  It lies within (-2, 2), so fixed point in units of 2^-14
// (off by at most 2^-15) keeps 4 to 30 times more of it than a 16-bit float
// would near 1; a derivative below 2^-15 counts as 0, which moves dz by at most
// 2^-15 of dy, less than its own rounding where the derivative is 2^-7 (bf16) or
// 2^-4 (float16) or more.  -32768 stands for NaN.  Adding 1.5 * 2^23 rounds to an integer in the
// low bits.
__device__ __forceinline__ uint16_t slope_code(float s) {
    const uint32_t c = __float_as_uint(fmaf(s, 16384.f, 12582912.f));
    return s != s ? (uint16_t)0x8000 : (uint16_t)c;
}
__device__ __forceinline__ float slope_value(int16_t c) {
    return c == -32768 ? __int_as_float(0x7fc00000) : (float)c * kSlopeUnit;
}

// One product D[p][q] = sum_r A[p][r] * B[q][r], stored as C[q * c_q + p].
//   ragged rows (red == 0): q runs over the rows of all groups, group g's rows
//     use A + g * a_g; epilogue bias, activation, slope, residual.
//   ragged sums (red == 1): r runs over the rows of group g, for every group.
struct Product {
    int64_t P, Q, R;             // Q (red == 0) or R (red == 1) counts the rows of all groups
    int64_t groups;
    const int32_t *offsets;      // null: one group
    int32_t red, act, f16, out_f32;
    const void *A, *B;
    int64_t a_p, a_r, a_g, b_q, b_r;   // one of (a_p, a_r) and of (b_q, b_r) is 1
    void *C;
    int64_t c_q, c_g;
    const void *bias;
    int64_t bias_g;
    const void *residual;
    int64_t residual_ld;
    int16_t *slope;              // [Q][P]
    // A handful of rows: row q of B is row gather[q] of the operand, zeros where that lies outside [0, gather_rows).
    const int32_t *gather;
    int64_t gather_rows;
    int32_t *status;
    int64_t wait_cycles;
};

// How a product runs, decided before anything is launched; scratch comes from `arena`.
struct ProductPlan {
    bool launches, skinny;
    int cg, bq, splits;      // tensor-core kernel: CTAs of a tile, its q, parts of the sum over r
    float *parts;
    int dev, sms;
};
int plan_product(const Product &p, bool probe, Arena &arena, ProductPlan &plan);
// `clear`: the kernel sets *status to 0 first (the first product of a call); `probe`: SPMM_CFG_EXPIRE_FIRST_WAIT.
int run_product(const Product &p, const ProductPlan &plan, bool clear, bool probe, cudaStream_t s);

// The same for about one row per group (operands aligned, see skinny_fits).
bool skinny_fits(const Product &p);
int launch_skinny(const Product &p, bool clear, cudaStream_t s);

}  // namespace spmm
