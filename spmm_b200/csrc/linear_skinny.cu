// linear_skinny.cu -- products of a handful of rows: y[q][p] = sum_r A[p][r] B[q][r]
// for about one q per group, the single tokens of a decoding step.
//
// Every value of A (the weights) is used once per row, so the time is that of
// reading A; what counts is many independent 16-byte loads from the first
// microsecond on.  Plain loads and FMAs do that with less start-up than a ring
// of bulk copies, barriers and tensor memory: 1 x 4096 x 4096 takes 9.2 us with
// the weights in HBM where the tensor-core kernel needs 12.5 (and 8 against 12
// with them in L2); its floor is 5.1 us.
//
// r contiguous: KS of a CTA's 8 warps share 4 p and take 256 r each in turn, a
// lane 8 of them (KS = 1 where there are warps enough without: sharing costs a
// barrier and leaves a warp little to stream).  p contiguous: a CTA owns WP = 64
// p (32 where that leaves SMs without work); WP / 8 lanes cover them, so a warp
// reads 4 (8) rows r of 128 (64) bytes at once and 16 warps take the next ones.
// Sums over lanes by shuffles, over warps in shared memory, in a fixed order.
#include "linear.cuh"

namespace spmm {
namespace {

struct Rows {
    int64_t q0, q1;
    bool zero;
};

__device__ __forceinline__ Rows group_rows(const Product &p, int64_t g) {
    if (!p.offsets) return {0, p.Q, false};
    const int64_t a = group_first(p.offsets, g, p.Q), b = g < p.groups ? group_first(p.offsets, g + 1, p.Q) : p.Q;
    return {a, b, g == p.groups};
}

// Row q of B (null: zeros).
template <typename T>
__device__ __forceinline__ const T *row_of(const Product &p, int64_t q) {
    if (p.gather) {
        q = __ldg(p.gather + q);
        if (q < 0 || q >= p.gather_rows) return nullptr;
    }
    return (const T *)p.B + q * p.b_q;
}

template <typename T, typename O, int ACT>
__device__ __forceinline__ void put_act(const Product &p, int64_t q, int64_t pp, float z) {
    float d, y = activate<ACT, true>(z, d);
    if (p.residual) y += to_f32(((const T *)p.residual)[q * p.residual_ld + pp]);
    ((O *)p.C)[q * p.c_q + pp] = from_f32<O>(y);
    if (p.slope) p.slope[q * p.P + pp] = (int16_t)slope_code(d);
}

template <typename T, typename O>
__device__ __forceinline__ void put(const Product &p, int64_t g, int64_t q, int64_t pp, float z) {
    if (p.bias) z += to_f32(((const T *)p.bias)[g * p.bias_g + pp]);
    switch (p.act) {
        case SPMM_ACT_NONE: put_act<T, O, SPMM_ACT_NONE>(p, q, pp, z); break;
        case SPMM_ACT_RELU: put_act<T, O, SPMM_ACT_RELU>(p, q, pp, z); break;
        case SPMM_ACT_GELU: put_act<T, O, SPMM_ACT_GELU>(p, q, pp, z); break;
        case SPMM_ACT_GELU_TANH: put_act<T, O, SPMM_ACT_GELU_TANH>(p, q, pp, z); break;
        default: put_act<T, O, SPMM_ACT_SILU>(p, q, pp, z); break;
    }
}

// Rows behind the last group: zeros at this CTA's p.
template <typename O>
__device__ __forceinline__ void put_zeros(const Product &p, Rows w, int64_t p0, int np) {
    for (int64_t i = threadIdx.x; i < (w.q1 - w.q0) * np; i += blockDim.x) {
        const int64_t q = w.q0 + i / np, pp = p0 + i % np;
        if (pp < p.P) {
            ((O *)p.C)[q * p.c_q + pp] = from_f32<O>(0.f);
            if (p.slope) p.slope[q * p.P + pp] = 0;
        }
    }
}

constexpr int kNP = 4;      // p of a CTA, r contiguous

template <typename T, typename O, int R, int KS>
__device__ __forceinline__ void rows_rmajor(const Product &p, int64_t g, int64_t q, int64_t p0, float *sm) {
    const int lane = threadIdx.x & 31, part = (threadIdx.x >> 5) % KS;
    const T *A = (const T *)p.A + g * p.a_g, *b[R];
#pragma unroll
    for (int j = 0; j < R; ++j) b[j] = row_of<T>(p, q + j);
    const T *a[kNP];
#pragma unroll
    for (int i = 0; i < kNP; ++i) a[i] = A + (p0 + i < p.P ? p0 + i : p.P - 1) * p.a_p;
    float acc[kNP][R] = {};
#pragma unroll (KS == 1 && R <= 2 ? 4 : 2)
    for (int64_t r = part * 256 + lane * 8; r < p.R; r += KS * 256) {
        uint4 w[kNP], x[R];
#pragma unroll
        for (int i = 0; i < kNP; ++i) w[i] = __ldg((const uint4 *)(a[i] + r));
#pragma unroll
        for (int j = 0; j < R; ++j) x[j] = b[j] ? __ldg((const uint4 *)(b[j] + r)) : uint4{0, 0, 0, 0};
        float xf[R][8];
#pragma unroll
        for (int j = 0; j < R; ++j) unpack8<T>(x[j], xf[j]);
#pragma unroll
        for (int i = 0; i < kNP; ++i) {
            float wf[8];
            unpack8<T>(w[i], wf);
#pragma unroll
            for (int j = 0; j < R; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[i][j] = fmaf(wf[e], xf[j][e], acc[i][j]);
        }
    }
    float z = 0.f;           // lane i * R + j: sum (i, j)
#pragma unroll
    for (int i = 0; i < kNP; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float v = acc[i][j];
#pragma unroll
            for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
            if (lane == i * R + j) z = v;
        }
    const int64_t pp = p0 + lane / R;
    if constexpr (KS > 1) {
        const int warp = threadIdx.x >> 5;
        if (lane < kNP * R) sm[warp * (kNP * R) + lane] = z;
        __syncthreads();
        if (part == 0 && lane < kNP * R) {
            z = 0.f;
#pragma unroll
            for (int w = 0; w < KS; ++w) z += sm[(warp + w) * (kNP * R) + lane];
        }
    }
    if (part == 0 && lane < kNP * R && pp < p.P) put<T, O>(p, g, q + lane % R, pp, z);
    if constexpr (KS > 1) __syncthreads();
}

template <typename T, typename O, int KS>
__global__ void __launch_bounds__(256) skinny_rmajor_kernel(const __grid_constant__ Product p, int clear) {
    chained_start();
    __shared__ float sm[8 * kNP * 4];
    if (clear && p.status && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.status = 0;
    const int64_t g = blockIdx.y;
    const Rows w = group_rows(p, g);
    if (w.zero) return put_zeros<O>(p, w, (int64_t)blockIdx.x * (kNP * 8 / KS), kNP * 8 / KS);
    int64_t p0 = ((int64_t)blockIdx.x * (8 / KS) + (threadIdx.x >> 5) / KS) * kNP;
    if (p0 >= p.P) {
        if constexpr (KS == 1) return;
        p0 = (p.P - 1) / kNP * kNP;          // walks along for the barriers, computing the last p once more
    }
    for (int64_t q = w.q0; q < w.q1;) {
        const int64_t n = w.q1 - q;
        if (n >= 4) rows_rmajor<T, O, 4, KS>(p, g, q, p0, sm), q += 4;
        else if (n == 3) rows_rmajor<T, O, 3, KS>(p, g, q, p0, sm), q += 3;
        else if (n == 2) rows_rmajor<T, O, 2, KS>(p, g, q, p0, sm), q += 2;
        else rows_rmajor<T, O, 1, KS>(p, g, q, p0, sm), q += 1;
    }
}

constexpr int kWarps = 16;  // of a CTA, p contiguous

template <typename T, typename O, int R, int WP>
__device__ __forceinline__ void rows_pmajor(const Product &p, int64_t g, int64_t q, int64_t p0, float *sm) {
    constexpr int kLanes = WP / 8, kRows = 32 / kLanes;       // lanes a row of A, rows a warp
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t pl = p0 + (lane % kLanes) * 8;
    const T *A = (const T *)p.A + g * p.a_g + (pl + 8 <= p.P ? pl : 0), *b[R];
#pragma unroll
    for (int j = 0; j < R; ++j) b[j] = row_of<T>(p, q + j);
    float acc[R][8] = {};
#pragma unroll 8
    for (int64_t r = warp * kRows + lane / kLanes; r < p.R; r += kWarps * kRows) {
        const uint4 w = __ldg((const uint4 *)(A + r * p.a_r));
        float x[R], wf[8];
#pragma unroll
        for (int j = 0; j < R; ++j) x[j] = b[j] ? to_f32(b[j][r]) : 0.f;
        unpack8<T>(w, wf);
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[j][e] = fmaf(wf[e], x[j], acc[j][e]);
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = acc[j][e];
#pragma unroll
            for (int o = kLanes; o < 32; o <<= 1) v += __shfl_xor_sync(kFullMask, v, o);
            if (lane < kLanes) sm[(warp * R + j) * WP + lane * 8 + e] = v;
        }
    __syncthreads();
    if (threadIdx.x < WP * R) {
        float z = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) z += sm[w * R * WP + threadIdx.x];
        const int64_t pp = p0 + threadIdx.x % WP;
        if (pp < p.P) put<T, O>(p, g, q + threadIdx.x / WP, pp, z);
    }
    __syncthreads();
}

template <typename T, typename O, int WP>
__global__ void __launch_bounds__(kWarps * 32) skinny_pmajor_kernel(const __grid_constant__ Product p, int clear) {
    chained_start();
    __shared__ float sm[kWarps * 4 * WP];
    if (clear && p.status && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.status = 0;
    const int64_t g = blockIdx.y, p0 = (int64_t)blockIdx.x * WP;
    const Rows w = group_rows(p, g);
    if (w.zero) return put_zeros<O>(p, w, p0, WP);
    for (int64_t q = w.q0; q < w.q1;) {
        const int64_t n = w.q1 - q;
        if (n >= 4) rows_pmajor<T, O, 4, WP>(p, g, q, p0, sm), q += 4;
        else if (n == 3) rows_pmajor<T, O, 3, WP>(p, g, q, p0, sm), q += 3;
        else if (n == 2) rows_pmajor<T, O, 2, WP>(p, g, q, p0, sm), q += 2;
        else rows_pmajor<T, O, 1, WP>(p, g, q, p0, sm), q += 1;
    }
}

template <typename T, typename O>
int run(const Product &p, bool clear, cudaStream_t s) {
    const unsigned gy = (unsigned)(p.offsets ? p.groups + 1 : 1);
    const int64_t busy = p.Q < p.groups ? p.Q : p.groups;      // groups with rows, at most
    if (p.a_r == 1) {
        // warps of the whole call without sharing: 148 SMs hold about 4,700 at once
        const int64_t quads = ceil_div(p.P, kNP), warps = quads * busy;
        if (warps >= 4096 || p.R <= 256)
            return launch_chained(skinny_rmajor_kernel<T, O, 1>, dim3((unsigned)ceil_div(quads, 8), gy), 256, 0, s, 1, p,
                                  clear);
        if (warps >= 2048 || p.R <= 512)
            return launch_chained(skinny_rmajor_kernel<T, O, 2>, dim3((unsigned)ceil_div(quads, 4), gy), 256, 0, s, 1, p,
                                  clear);
        return launch_chained(skinny_rmajor_kernel<T, O, 8>, dim3((unsigned)quads, gy), 256, 0, s, 1, p, clear);
    }
    if (ceil_div(p.P, 64) * busy >= 148 * 2)
        return launch_chained(skinny_pmajor_kernel<T, O, 64>, dim3((unsigned)ceil_div(p.P, 64), gy), kWarps * 32, 0, s, 1,
                              p, clear);
    return launch_chained(skinny_pmajor_kernel<T, O, 32>, dim3((unsigned)ceil_div(p.P, 32), gy), kWarps * 32, 0, s, 1, p,
                          clear);
}

}  // namespace

// Where this kernel is the faster one.  One group of 4096 x 4096, us here / on
// the tensor cores: 1 row 9.2 / 12.5 (p contiguous) and 10.9 / 13.3 (r
// contiguous), 2 rows 9.9 / 12.7 and 12.3 / 13.0, 3 rows 11.4 / 12.6 and 14.0 /
// 13.4.  64 groups of 2048 x 1408: 64 rows 45 / 49 (and it gathers rows itself,
// which saves a copy), 128 rows 65 / 60.  It takes four rows at a time, so many
// rows in one group cost far more than on the tensor cores; hence at most 64.
bool skinny_fits(const Product &p) {
    const int64_t most = !p.offsets ? (p.a_r == 1 ? 2 : 3) : p.groups < 64 ? p.groups : 64;
    if (p.red || p.Q > most || p.b_r != 1) return false;
    return p.a_r == 1 ? p.R % 8 == 0 : p.P % 8 == 0;
}

int launch_skinny(const Product &p, bool clear, cudaStream_t s) {
    if (p.f16) return p.out_f32 ? run<__half, float>(p, clear, s) : run<__half, __half>(p, clear, s);
    return p.out_f32 ? run<__nv_bfloat16, float>(p, clear, s) : run<__nv_bfloat16, __nv_bfloat16>(p, clear, s);
}

}  // namespace spmm
