// linear.cu -- dense and grouped products of 16-bit operands: the C entries,
// operand copies and the gradient of the activation.
//
//   forward   y[r] = act(x[r] w[g] + bias[g]) + residual[r]
//   backward  dz = dy * act'(z), dx = dz w^T, dw = x^T dz, dbias = sum dz
//
// All three products are one form, D[p][q] = sum_r A[p][r] B[q][r] (linear.cuh),
// with groups that are ragged in q (forward, dx) or in r (dw).
#include <type_traits>

#include "linear.cuh"

namespace spmm {
namespace {

// ---- operand copies -----------------------------------------------------------

// dst[i][c] = src[map ? map[i] : i][c], rows of `cols` 16-bit values in pieces of
// 8 (16 bytes, aligned in dst, whose rows are padded), read `width` values at a
// time; a map value outside [0, src_rows) gives zeros.  `copies` blocks of rows,
// src_gs / dst_gs apart.
struct CopyJob {
    const uint16_t *src;
    int64_t src_ld, src_gs, src_rows;
    const int32_t *map;
    uint16_t *dst;
    int64_t dst_ld, dst_gs, rows, cols, copies;
    int32_t width;
};
struct Copies {          // the operands of a call that are copied, in one launch
    CopyJob job[3];
    int count;
};

template <int W>
__device__ __forceinline__ void copy_piece(const uint16_t *row, int64_t c, int64_t cols, uint16_t (&v)[8]) {
    using V = typename std::conditional<W == 8, uint4, typename std::conditional<W == 4, uint2,
              typename std::conditional<W == 2, uint32_t, uint16_t>::type>::type>::type;
#pragma unroll
    for (int u = 0; u < 8 / W; ++u) {
        V x{};
        if (c + u * W < cols) x = __ldg(reinterpret_cast<const V *>(row + c + u * W));
        memcpy(v + u * W, &x, sizeof(V));
    }
}

// I: 32-bit piece numbers where they suffice; two 64-bit divisions a piece took longer than moving it.
template <typename I>
__global__ void __launch_bounds__(256) copy_rows_kernel(const __grid_constant__ Copies all) {
    chained_start();
    const CopyJob &j = all.job[blockIdx.y];
    const I per = (I)(j.dst_ld / 8), block = (I)j.rows * per, items = block * (I)j.copies;
    for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < items; i += (I)gridDim.x * 256) {
        const I g = i / block, k = i - g * block, row_in = k / per;
        const int64_t r = row_in, c = (int64_t)(k - row_in * per) * 8;
        const int64_t from = j.map ? __ldg(j.map + r) : r;
        uint16_t v[8] = {};
        if (from >= 0 && from < j.src_rows) {
            const uint16_t *row = j.src + g * j.src_gs + from * j.src_ld;
            if (j.width == 8) copy_piece<8>(row, c, j.cols, v);
            else if (j.width == 4) copy_piece<4>(row, c, j.cols, v);
            else if (j.width == 2) copy_piece<2>(row, c, j.cols, v);
            else copy_piece<1>(row, c, j.cols, v);
        }
        uint4 o;
        memcpy(&o, v, 16);
        *reinterpret_cast<uint4 *>(j.dst + g * j.dst_gs + r * j.dst_ld + c) = o;
    }
}

int run_copies(const Copies &all, cudaStream_t s) {
    if (all.count == 0) return SPMM_OK;
    int64_t most = 1, pieces = 0;
    for (int i = 0; i < all.count; ++i) {
        const CopyJob &j = all.job[i];
        const int64_t blocks = ceil_div(j.copies * j.rows * (j.dst_ld / 8), 256);
        most = blocks > most ? blocks : most;
        pieces = j.copies * j.rows * (j.dst_ld / 8) > pieces ? j.copies * j.rows * (j.dst_ld / 8) : pieces;
    }
    const dim3 grid((unsigned)(most < 148 * 32 ? most : 148 * 32), (unsigned)all.count);
    return launch_chained(pieces < INT32_MAX ? copy_rows_kernel<uint32_t> : copy_rows_kernel<int64_t>, grid, 256, 0, s,
                          1, all);
}

// ---- gradient of the activation and of the bias -------------------------------

constexpr int kDzRows = 64;    // rows of a tile
constexpr int kDzCols = 256;   // columns of a CTA: 32 lanes of 8

// Where the sums of the tile that starts at row `first` of group g stand.  Group
// [a, b) takes places from a / 64 + g on, the last at most b / 64 + g, which lies
// before the next group's first; every place is below ceil(rows / 64) + groups
// whatever the table holds, where a count of the tiles before would not be.
__device__ __forceinline__ int64_t part_place(int64_t first, int64_t g) { return first / kDzRows + g; }

// dz = dy * act'(z) and the tile's column sums of the unrounded products.  dz is
// rounded to the operands' type, as the two products take 16-bit operands: dx and
// dw are then up to sqrt 2 times as far from the exact gradient as a rounding of
// it (bf16 4096 x 2048 x 8192: 0.0023 against 0.0017 relative), and float16 loses
// a dz below 2^-25, which scaling the loss avoids.  A warp takes a row at a time,
// a lane 16 bytes of it; bound by reading dy and the slopes and writing dz once.
// Where dz is written, dy and the slopes are not read again: they are loaded as a
// stream, so that the cache keeps dz for the products (4096 x 8192: 47.5 -> 43.3
// us; tiles of 32 rows, before the streamed loads, took 50 us against 47.5).
// Strips of columns and tiles share one grid dimension, which sizes past 2^24
// columns need (and 32 registers instead of 48: 40 -> 34.5 us, as the difference
// of two backward passes).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dz_kernel(const T *dy, int64_t dy_ld, const int16_t *slope, T *dz,
                                                 int64_t dz_ld, float *part, T *dbias, const int32_t *offsets,
                                                 int64_t groups, int64_t rows, int64_t n, uint32_t tiles) {
    chained_start();
    __shared__ float sums[8][kDzCols];
    const int64_t strip = (int64_t)(blockIdx.x / tiles) * kDzCols;     // its first column
    const RowTile t = find_row_tile(offsets, groups, rows, kDzRows, blockIdx.x % tiles);
    if (t.group > groups || (offsets && t.group == groups)) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c0 = strip + lane * 8;
    const int cols = c0 >= n ? 0 : n - c0 < 8 ? (int)(n - c0) : 8;
    float acc[8] = {};
    if (cols) {
#pragma unroll 4
        for (int i = warp; i < t.rows; i += 8) {
            const int64_t r = t.first + i;
            float d[8];
            if constexpr (VEC) {
                const uint4 *from = (const uint4 *)(dy + r * dy_ld + c0);
                unpack8<T>(slope ? __ldcs(from) : __ldg(from), d);
                if (slope) {
                    const uint4 v = __ldcs((const uint4 *)(slope + r * n + c0));
                    int16_t c[8];
                    memcpy(c, &v, 16);
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] *= slope_value(c[e]);
                    if (dz) *(uint4 *)(dz + r * dz_ld + c0) = pack8<T>(d);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    d[e] = 0.f;
                    if (e < cols) {
                        d[e] = to_f32(dy[r * dy_ld + c0 + e]);
                        if (slope) {
                            d[e] *= slope_value(slope[r * n + c0 + e]);
                            if (dz) dz[r * dz_ld + c0 + e] = from_f32<T>(d[e]);
                        }
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += d[e];
        }
    }
    if (part == nullptr && dbias == nullptr) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[warp][lane * 8 + e] = acc[e];
    __syncthreads();
    const int64_t c = strip + threadIdx.x;
    if (c < n) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += sums[w][threadIdx.x];
        if (dbias) dbias[c] = from_f32<T>(v);       // the only tile of the only group
        else part[part_place(t.first, t.group) * n + c] = v;
    }
}

// dbias[g] = sum of group g's tiles: 32 columns a CTA, each of its 8 warps every
// eighth tile, the warps' sums added in order.
template <typename T>
__global__ void __launch_bounds__(256) dbias_kernel(const float *part, const int32_t *offsets, int64_t rows, int64_t n,
                                                    T *out, int64_t out_g) {
    chained_start();
    __shared__ float sums[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t g = blockIdx.y, c = (int64_t)blockIdx.x * 32 + lane;
    int64_t first = 0, count = (rows + kDzRows - 1) / kDzRows;
    if (offsets) {
        const int64_t a = group_first(offsets, g, rows), b = group_first(offsets, g + 1, rows);
        first = part_place(a, g);
        count = b > a ? (b - a + kDzRows - 1) / kDzRows : 0;
    }
    float v = 0.f;
    if (c < n) {
#pragma unroll 8
        for (int64_t t = warp; t < count; t += 8) v += part[(first + t) * n + c];
    }
    sums[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && c < n) {
        v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += sums[w][lane];
        out[g * out_g + c] = from_f32<T>(v);
    }
}

// out[t] = sum_j src[slots[t][j]], in order of j: V values a thread, the rows of
// four choices in flight.
template <typename T, int V>
__global__ void __launch_bounds__(256) gather_sum_kernel(const float *src, int64_t rows, const int32_t *slots,
                                                         int64_t tokens, int64_t top, int64_t n, T *out,
                                                         int64_t out_ld) {
    chained_start();
    const int64_t per = n / V, items = tokens * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / per, c = (i - t * per) * V;
        float acc[V] = {};
        for (int64_t j0 = 0; j0 < top; j0 += 4) {
            float f[4][V];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t s = j0 + u < top ? __ldg(slots + t * top + j0 + u) : -1;
                const bool in = s >= 0 && s < rows;
                if constexpr (V == 4) {
                    const float4 v = in ? __ldg((const float4 *)(src + s * n + c)) : float4{0.f, 0.f, 0.f, 0.f};
                    f[u][0] = v.x, f[u][1] = v.y, f[u][2] = v.z, f[u][3] = v.w;
                } else {
                    f[u][0] = in ? __ldg(src + s * n + c) : 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += f[u][e];
        }
        if constexpr (V == 4) {
            T o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(acc[e]);
            memcpy(__builtin_assume_aligned(out + t * out_ld + c, 8), o, 8);
        } else {
            out[t * out_ld + c] = from_f32<T>(acc[0]);
        }
    }
}

template <typename T>
int gather_sum(const float *src, int64_t rows, const int32_t *slots, int64_t tokens, int64_t top, int64_t n, T *out,
               int64_t out_ld, cudaStream_t s) {
    const bool vec = n % 4 == 0 && out_ld % 4 == 0 && (uintptr_t)out % 8 == 0;
    const int64_t blocks = ceil_div(tokens * (vec ? n / 4 : n), 256);
    const unsigned grid = (unsigned)(blocks < 148 * 64 ? blocks : 148 * 64);
    return launch_chained(vec ? gather_sum_kernel<T, 4> : gather_sum_kernel<T, 1>, dim3(grid), 256, 0, s, 1, src, rows,
                          slots, tokens, top, n, out, out_ld);
}

// ---- host side ------------------------------------------------------------------

int check_sizes(const spmm_linear *p) {
    if (!p || p->version != 1) return SPMM_EINVAL;
    if (p->dtype != SPMM_DENSE_BF16 && p->dtype != SPMM_DENSE_F16) return SPMM_EUNSUPPORTED;
    if (p->rows < 0 || p->k < 0 || p->n < 0 || p->groups < 1 || p->x_rows < 0) return SPMM_EINVAL;
    if (p->groups > SPMM_MAX_GROUPS) return SPMM_EUNSUPPORTED;
    if (p->rows > INT32_MAX || p->k > INT32_MAX || p->n > INT32_MAX || p->x_rows > INT32_MAX)
        return SPMM_EUNSUPPORTED;
    if (!p->offsets && p->groups != 1) return SPMM_EINVAL;
    if (!p->gather && p->x_rows != p->rows) return SPMM_EINVAL;
    if ((p->wait_us != 0 && p->wait_us < 1000) || (p->flags & ~(SPMM_CFG_EXPIRE_FIRST_WAIT | SPMM_LINEAR_KEEP_STATUS)))
        return SPMM_EINVAL;
    if (p->w_k != 1 && p->w_n != 1) return SPMM_EUNSUPPORTED;
    if (!on_boundary(2, {p->x, p->w, p->bias, p->residual, p->y, p->slope, p->dy, p->dx, p->dw, p->dbias}) ||
        !on_boundary(4, {p->offsets, p->gather, p->slots, p->status}) || !on_boundary(256, {p->workspace}))
        return SPMM_EALIGN;
    return SPMM_OK;
}

// An operand as the product reads it: in place, or a copy with aligned rows.
struct Operand {
    const void *ptr;
    int64_t ld, gs;   // row stride, group stride
};

// Tensor copies need 16-byte aligned rows.
bool in_place(const void *p, int64_t ld, int64_t gs, int64_t cols) {
    return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && gs % 8 == 0 && ld >= cols;
}

// `rows` x `cols` values (per group): in place, or a copy (gathered by `map`) that run_copies makes.
Operand carve(const Operand src, int64_t src_rows, const int32_t *map, int64_t groups, int64_t rows, int64_t cols,
              Arena &a, Copies &copies) {
    Operand out = src;
    if (rows == 0 || cols == 0) return out;
    const int64_t ld = ceil_div(cols, 8) * 8;
    if (rows == 1) out.ld = ld;         // one row: its stride is never used
    if (groups == 1) out.gs = 0;
    if (!map && in_place(src.ptr, out.ld, out.gs, cols)) return out;
    const int64_t blocks = groups > 1 && src.gs == 0 ? 1 : groups;   // one block shared by all groups
    out.ld = ld;
    out.gs = blocks > 1 ? rows * ld : 0;
    uint16_t *buf = a.take<uint16_t>(blocks * rows * ld);
    out.ptr = buf;
    const int64_t all = (int64_t)((uintptr_t)src.ptr / 2) | src.ld | (blocks > 1 ? src.gs : 0) | cols;
    const int32_t width = all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
    copies.job[copies.count++] = CopyJob{(const uint16_t *)src.ptr, src.ld, src.gs, src_rows, map, buf,
                                         ld, out.gs, rows, cols, blocks, width};
    return out;
}

Operand carve_x(const spmm_linear *p, Arena &a, Copies &copies) {
    return carve({p->x, p->x_ld, 0}, p->x_rows, p->gather, 1, p->rows, p->k, a, copies);
}

// w's strides along n, k and the groups, in place or of the copy.
struct Weight {
    const void *ptr;
    int64_t n, k, g;
};

Weight carve_w(const spmm_linear *p, Arena &a, Copies &copies) {
    const bool n_unit = p->w_n == 1;
    const int64_t rows = n_unit ? p->k : p->n, cols = n_unit ? p->n : p->k;
    const Operand o = carve({p->w, n_unit ? p->w_k : p->w_n, p->w_g}, rows, nullptr, p->groups, rows, cols, a, copies);
    return n_unit ? Weight{o.ptr, 1, o.ld, o.gs} : Weight{o.ptr, o.ld, 1, o.gs};
}

int64_t wait_cycles(int32_t wait_us) { return wait_us > 0 ? (int64_t)wait_us * 2000 : 1ll << 32; }

Product base(const spmm_linear *p) {
    Product g{};
    g.groups = p->groups;
    g.offsets = p->offsets;
    g.f16 = p->dtype == SPMM_DENSE_F16;
    g.status = p->status;
    g.wait_cycles = wait_cycles(p->wait_us);
    return g;
}

// A call lays out its scratch and decides on its kernels first; only then, and
// if the workspace suffices, it launches anything.  need: the scratch in bytes
// (all that a sizing call wants).
int settle(const Arena &a, bool sizing, size_t &need) {
    need = (a.used + 255) & ~(size_t)255;
    return !sizing && a.used > a.cap ? SPMM_EWORKSPACE : SPMM_OK;
}

int forward(const spmm_linear *p, Arena &a, bool sizing, size_t &need, cudaStream_t s) {
    const bool probe = p->flags & SPMM_CFG_EXPIRE_FIRST_WAIT, clear = !(p->flags & SPMM_LINEAR_KEEP_STATUS);
    Copies copies{};
    const Weight w = carve_w(p, a, copies);
    Product g = base(p);
    g.P = p->n;
    g.Q = p->rows;
    g.R = p->k;
    g.act = p->activation;
    g.A = w.ptr;
    g.a_p = w.n;
    g.a_r = w.k;
    g.a_g = w.g;
    g.b_r = 1;
    Operand x{p->x, p->x_ld, 0};
    if (p->gather && skinny_fits(g) && in_place(p->x, p->x_ld, 0, p->k)) {   // reads the gathered rows itself
        g.gather = p->gather;
        g.gather_rows = p->x_rows;
    } else {
        x = carve_x(p, a, copies);
    }
    g.B = x.ptr;
    g.b_q = x.ld;
    g.C = p->y;
    g.c_q = p->y_ld;
    g.bias = p->bias;
    g.bias_g = p->bias_g;
    g.residual = p->residual;
    g.residual_ld = p->residual_ld;
    g.slope = p->slope;
    ProductPlan plan;
    SPMM_TRY(plan_product(g, probe, a, plan));
    SPMM_TRY(settle(a, sizing, need));
    if (sizing) return SPMM_OK;
    if (p->status && clear && !plan.launches) SPMM_CUDA_TRY(cudaMemsetAsync(p->status, 0, sizeof(int32_t), s));
    SPMM_TRY(run_copies(copies, s));
    return run_product(g, plan, clear, probe, s);
}

template <typename T>
int gradients(const spmm_linear *p, Arena &a, bool sizing, size_t &need, cudaStream_t s) {
    const bool any = p->rows > 0 && p->n > 0, probe = p->flags & SPMM_CFG_EXPIRE_FIRST_WAIT;
    const bool clear = !(p->flags & SPMM_LINEAR_KEEP_STATUS);
    const int64_t tiles = ceil_div(p->rows, kDzRows) + (p->offsets ? p->groups + 1 : 0);
    const bool make_dz = p->slope && any && (p->dx || p->dw);
    const bool one_tile = p->dbias && any && tiles == 1 && !p->offsets;
    const bool parts = p->dbias && any && !one_tile, sums = p->dx && p->gather;
    const int64_t dz_blocks = tiles * ceil_div(p->n, kDzCols);
    if ((make_dz || parts || one_tile) && dz_blocks > INT32_MAX) return SPMM_EUNSUPPORTED;
    Copies copies{};
    Operand x{}, dz{p->dy, p->dy_ld, 0};
    Weight w{};
    if (p->dw) x = carve_x(p, a, copies);
    if (p->dx) w = carve_w(p, a, copies);
    T *dzp = nullptr;
    float *part = nullptr, *dxs = nullptr;
    if (make_dz) {
        const int64_t ld = ceil_div(p->n, 8) * 8;
        dzp = a.take<T>(p->rows * ld);
        dz = Operand{dzp, ld, 0};
    } else if (any && (p->dx || p->dw)) {
        dz = carve(dz, p->rows, nullptr, 1, p->rows, p->n, a, copies);
    }
    if (parts) part = a.take<float>(tiles * p->n);
    if (sums) dxs = a.take<float>(p->rows * p->k);
    Product gx = base(p), gw = base(p);
    ProductPlan px{}, pw{};
    if (p->dx) {
        gx.P = p->k;
        gx.Q = p->rows;
        gx.R = p->n;
        gx.A = w.ptr;
        gx.a_p = w.k;
        gx.a_r = w.n;
        gx.a_g = w.g;
        gx.B = dz.ptr;
        gx.b_q = dz.ld;
        gx.b_r = 1;
        gx.C = sums ? (void *)dxs : p->dx;
        gx.c_q = sums ? p->k : p->dx_ld;
        gx.out_f32 = sums;
        SPMM_TRY(plan_product(gx, probe, a, px));
    }
    if (p->dw) {
        const bool n_unit = p->dw_n == 1;
        gw.red = 1;
        gw.R = p->rows;
        gw.P = n_unit ? p->n : p->k;
        gw.Q = n_unit ? p->k : p->n;
        gw.A = n_unit ? dz.ptr : x.ptr;
        gw.a_p = 1;
        gw.a_r = n_unit ? dz.ld : x.ld;
        gw.B = n_unit ? x.ptr : dz.ptr;
        gw.b_q = 1;
        gw.b_r = n_unit ? x.ld : dz.ld;
        gw.C = p->dw;
        gw.c_q = n_unit ? p->dw_k : p->dw_n;
        gw.c_g = p->dw_g;
        SPMM_TRY(plan_product(gw, probe, a, pw));
    }
    SPMM_TRY(settle(a, sizing, need));
    if (sizing) return SPMM_OK;
    if (p->status && clear && !px.launches && !pw.launches)
        SPMM_CUDA_TRY(cudaMemsetAsync(p->status, 0, sizeof(int32_t), s));
    SPMM_TRY(run_copies(copies, s));
    if (make_dz || parts || one_tile) {
        const bool vec = p->n % 8 == 0 && in_place(p->dy, p->dy_ld, 0, p->n) && (uintptr_t)p->slope % 16 == 0;
        T *direct = one_tile ? (T *)p->dbias : nullptr;
        SPMM_TRY(launch_chained(vec ? dz_kernel<T, true> : dz_kernel<T, false>, dim3((unsigned)dz_blocks), 256, 0, s, 1,
                                (const T *)p->dy, p->dy_ld, p->slope, dzp, dz.ld, part, direct, p->offsets, p->groups,
                                p->rows, p->n, (uint32_t)tiles));
    }
    if (p->dbias && p->n && !one_tile) {
        const dim3 grid((unsigned)ceil_div(p->n, 32), (unsigned)p->groups);
        SPMM_TRY(launch_chained(dbias_kernel<T>, grid, 256, 0, s, 1, part, p->offsets, any ? p->rows : 0, p->n,
                                (T *)p->dbias, p->dbias_g));
    }
    SPMM_TRY(run_product(gx, px, clear, probe, s));
    if (sums && p->x_rows && p->k)
        SPMM_TRY(gather_sum(dxs, p->rows, p->slots, p->x_rows, p->top, p->k, (T *)p->dx, p->dx_ld, s));
    return run_product(gw, pw, clear && !px.launches, probe, s);
}

int backward(const spmm_linear *p, Arena &a, bool sizing, size_t &need, cudaStream_t s) {
    return p->dtype == SPMM_DENSE_F16 ? gradients<__half>(p, a, sizing, need, s)
                                      : gradients<__nv_bfloat16>(p, a, sizing, need, s);
}

size_t sized(const spmm_linear *p, int (*run)(const spmm_linear *, Arena &, bool, size_t &, cudaStream_t)) {
    if (check_sizes(p) != SPMM_OK) return 0;
    Arena a(nullptr, 0);
    size_t need = 0;
    return run(p, a, true, need, nullptr) == SPMM_OK ? need : 0;
}

}  // namespace

}  // namespace spmm

extern "C" size_t spmm_linear_forward_workspace_size(const spmm_linear *p) {
    return spmm::sized(p, spmm::forward);
}

extern "C" size_t spmm_linear_backward_workspace_size(const spmm_linear *p) {
    return spmm::sized(p, spmm::backward);
}

extern "C" int spmm_linear_forward(const spmm_linear *p, spmm_stream_t stream) {
    SPMM_TRY(spmm::check_sizes(p));
    if (p->activation < SPMM_ACT_NONE || p->activation > SPMM_ACT_SILU) return SPMM_EINVAL;
    const int64_t out = p->rows * p->n;
    if (out && !p->y) return SPMM_EINVAL;
    if (out && p->k && (!p->x || !p->w)) return SPMM_EINVAL;
    if (p->rows > 1 && p->y_ld < p->n) return SPMM_EINVAL;
    spmm::Arena a(p->workspace, p->workspace ? p->workspace_bytes : 0);
    size_t need;
    return spmm::forward(p, a, false, need, (cudaStream_t)stream);
}

extern "C" int spmm_linear_backward(const spmm_linear *p, spmm_stream_t stream) {
    SPMM_TRY(spmm::check_sizes(p));
    if (p->rows * p->n && !p->dy) return SPMM_EINVAL;
    if (p->dx && ((p->k * p->n && !p->w) || (p->gather && (!p->slots || p->top < 1)))) return SPMM_EINVAL;
    if (p->dw && ((p->rows * p->k && !p->x) || (p->dw_k != 1 && p->dw_n != 1))) return SPMM_EINVAL;
    if (p->dx && p->x_rows > 1 && p->dx_ld < p->k) return SPMM_EINVAL;
    spmm::Arena a(p->workspace, p->workspace ? p->workspace_bytes : 0);
    size_t need;
    return spmm::backward(p, a, false, need, (cudaStream_t)stream);
}
