// linear.cu -- dense and grouped products of 16-bit operands: the C entries,
// operand copies, the gradient of the activation, and a plain product kernel.
//
//   forward   y[r] = act(x[r] w[g] + bias[g]) + residual[r]
//   backward  dz = dy * act'(z), dx = dz w^T, dw = x^T dz, dbias = sum dz
//
// All three products are one form, D[p][q] = sum_r A[p][r] B[q][r] (linear.cuh),
// with groups that are ragged in q (forward, dx) or in r (dw).
#include "linear.cuh"

namespace spmm {
namespace {

// ---- plain product ----------------------------------------------------------

// Any strides, any sizes: a 64 x 64 tile per CTA of 256 threads, 4 x 4 sums
// each, operands through shared memory 16 at a time.
template <typename T, typename O, int ACT>
__global__ void __launch_bounds__(256) product_kernel(Product p) {
    __shared__ float As[16][65], Bs[16][65];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t p0 = (int64_t)blockIdx.x * 64;
    RowTile t;
    int64_t r0 = 0, r1 = p.R, q0, g;
    int nq;
    if (p.red) {
        const int64_t qt = (p.Q + 63) / 64;
        g = blockIdx.y / qt;
        q0 = (blockIdx.y % qt) * 64;
        nq = (int)(p.Q - q0 < 64 ? p.Q - q0 : 64);
        if (p.offsets) {
            r0 = group_first(p.offsets, g, p.R);
            r1 = group_first(p.offsets, g + 1, p.R);
        }
    } else {
        t = find_row_tile(p.offsets, p.groups, p.Q, 64, blockIdx.y);
        if (t.group > p.groups) return;
        g = t.group;
        q0 = t.first;
        nq = t.rows;
    }
    const bool tail = !p.red && p.offsets && g == p.groups;
    if (tail) r1 = 0;
    const int64_t gi = tail ? 0 : g;
    const T *A = (const T *)p.A + (p.red ? 0 : gi * p.a_g), *B = (const T *)p.B;
    float acc[4][4] = {};
    for (int64_t r = r0; r < r1; r += 16) {
        for (int i = tid; i < 64 * 16; i += 256) {
            const int pr = p.a_r == 1 ? i & 15 : i >> 6, pp = p.a_r == 1 ? i >> 4 : i & 63;
            As[pr][pp] = r + pr < r1 && p0 + pp < p.P ? to_f32(A[(p0 + pp) * p.a_p + (r + pr) * p.a_r]) : 0.f;
            const int qr = p.b_r == 1 ? i & 15 : i >> 6, qq = p.b_r == 1 ? i >> 4 : i & 63;
            Bs[qr][qq] = r + qr < r1 && qq < nq ? to_f32(B[(q0 + qq) * p.b_q + (r + qr) * p.b_r]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[k][tx + 16 * i], Bs[k][ty + 16 * j], acc[i][j]);
        __syncthreads();
    }
    O *C = (O *)p.C + (p.red ? g * p.c_g : 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int qq = ty + 16 * j;
        if (qq >= nq) continue;
        const int64_t q = q0 + qq;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t pp = p0 + tx + 16 * i;
            if (pp >= p.P) continue;
            float z = acc[i][j];
            ActValue a{0.f, 0.f};
            if (!tail) {
                if (p.bias) z += to_f32(((const T *)p.bias)[gi * p.bias_g + pp]);
                a = activate<ACT>(z);
                if (p.residual) a.y += to_f32(((const T *)p.residual)[q * p.residual_ld + pp]);
            }
            C[q * p.c_q + pp] = from_f32<O>(a.y);
            if (p.slope) p.slope[q * p.P + pp] = slope_code(a.slope);
        }
    }
}

template <typename T, typename O>
int launch_act(const Product &p, dim3 grid, cudaStream_t s) {
    switch (p.act) {
        case SPMM_ACT_NONE: product_kernel<T, O, SPMM_ACT_NONE><<<grid, 256, 0, s>>>(p); break;
        case SPMM_ACT_RELU: product_kernel<T, O, SPMM_ACT_RELU><<<grid, 256, 0, s>>>(p); break;
        case SPMM_ACT_GELU: product_kernel<T, O, SPMM_ACT_GELU><<<grid, 256, 0, s>>>(p); break;
        case SPMM_ACT_GELU_TANH: product_kernel<T, O, SPMM_ACT_GELU_TANH><<<grid, 256, 0, s>>>(p); break;
        default: product_kernel<T, O, SPMM_ACT_SILU><<<grid, 256, 0, s>>>(p); break;
    }
    SPMM_PRODUCT_LAUNCHED();
    return SPMM_OK;
}

// ---- operand copies -----------------------------------------------------------

// dst[i][c] = src[map ? map[i] : i][c], rows of `cols` 16-bit values, destination rows `dst_ld` apart; a map
// value outside [0, src_rows) gives zeros.  Blocks of src_gs / dst_gs (groups) in blockIdx.z.
__global__ void copy_rows_kernel(const uint16_t *src, int64_t src_ld, int64_t src_gs, int64_t src_rows,
                                 const int32_t *map, uint16_t *dst, int64_t dst_ld, int64_t dst_gs, int64_t rows,
                                 int64_t cols, int vec) {
    src += blockIdx.z * src_gs;
    dst += blockIdx.z * dst_gs;
    const int64_t per = vec ? cols / 8 : cols;
    for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
        const int64_t from = map ? __ldg(map + i) : i;
        const bool in = from >= 0 && from < src_rows;
        for (int64_t c = threadIdx.x; c < per; c += blockDim.x) {
            if (vec) {
                uint4 v{0, 0, 0, 0};
                if (in) v = __ldg(reinterpret_cast<const uint4 *>(src + from * src_ld) + c);
                reinterpret_cast<uint4 *>(dst + i * dst_ld)[c] = v;
            } else {
                dst[i * dst_ld + c] = in ? __ldg(src + from * src_ld + c) : (uint16_t)0;
            }
        }
    }
}

// ---- gradient of the activation and of the bias -------------------------------

constexpr int kDzRows = 128;   // rows of a tile
constexpr int kDzCols = 64;    // columns of a CTA

// dz = dy * act'(z) (rounded to the operands' type) and the tile's column sums
// of the unrounded products.
template <typename T>
__global__ void __launch_bounds__(256) dz_kernel(const T *dy, int64_t dy_ld, const int16_t *slope, T *dz,
                                                 int64_t dz_ld, float *part, const int32_t *offsets, int64_t groups,
                                                 int64_t rows, int64_t n) {
    __shared__ float sums[8][kDzCols];
    const RowTile t = find_row_tile(offsets, groups, rows, kDzRows, blockIdx.y);
    if (t.group > groups) return;
    const bool tail = offsets && t.group == groups;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c0 = (int64_t)blockIdx.x * kDzCols;
    float acc[2] = {0.f, 0.f};
    if (!tail) {
        for (int i = warp; i < t.rows; i += 8) {
            const int64_t r = t.first + i;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int64_t c = c0 + u * 32 + lane;
                if (c < n) {
                    float d = to_f32(dy[r * dy_ld + c]);
                    if (slope) {
                        d *= slope_value(slope[r * n + c]);
                        if (dz) dz[r * dz_ld + c] = from_f32<T>(d);
                    }
                    acc[u] += d;
                }
            }
        }
    }
    if (part == nullptr) return;
    sums[warp][lane] = acc[0];
    sums[warp][lane + 32] = acc[1];
    __syncthreads();
    if (threadIdx.x < kDzCols && c0 + threadIdx.x < n) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += sums[w][threadIdx.x];
        part[(int64_t)blockIdx.y * n + c0 + threadIdx.x] = v;
    }
}

// dbias[g] = sum of group g's tiles, in order.
template <typename T>
__global__ void dbias_kernel(const float *part, const int32_t *offsets, int64_t rows, int64_t n, T *out,
                             int64_t out_g) {
    const int64_t g = blockIdx.y, c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    int64_t first = 0, last;
    if (offsets) {
        for (int64_t e = 0; e <= g; ++e) {
            const int64_t a = group_first(offsets, e, rows), b = group_first(offsets, e + 1, rows);
            const int64_t tiles = b > a ? (b - a + kDzRows - 1) / kDzRows : 0;
            if (e < g) first += tiles; else last = first + tiles;
        }
    } else {
        last = (rows + kDzRows - 1) / kDzRows;
    }
    if (c >= n) return;
    float v = 0.f;
    for (int64_t t = first; t < last; ++t) v += part[t * n + c];
    out[g * out_g + c] = from_f32<T>(v);
}

// out[t] = sum_j src[slots[t][j]], in order of j.
template <typename T>
__global__ void gather_sum_kernel(const float *src, int64_t rows, const int32_t *slots, int64_t tokens, int64_t top,
                                  int64_t n, T *out, int64_t out_ld) {
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x)
        for (int64_t c = threadIdx.x; c < n; c += blockDim.x) {
            float v = 0.f;
            for (int64_t j = 0; j < top; ++j) {
                const int64_t s = __ldg(slots + t * top + j);
                if (s >= 0 && s < rows) v += __ldg(src + s * n + c);
            }
            out[t * out_ld + c] = from_f32<T>(v);
        }
}

__global__ void clear_status_kernel(int32_t *status) { *status = 0; }

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
    if (p->wait_us != 0 && p->wait_us < 1000) return SPMM_EINVAL;
    if (p->w_k != 1 && p->w_n != 1) return SPMM_EUNSUPPORTED;
    return SPMM_OK;
}

// x as the product reads it: in place, or a copy (gathered).
struct Operand {
    const void *ptr;
    int64_t ld;
};

int carve_x(const spmm_linear *p, Arena &a, bool sizing, Operand &x, cudaStream_t s) {
    x = Operand{p->x, p->x_ld};
    if (!p->gather || p->rows == 0 || p->k == 0) return SPMM_OK;
    const int64_t ld = ceil_div(p->k, 8) * 8;
    uint16_t *buf = a.take<uint16_t>(p->rows * ld);
    if (sizing) return SPMM_OK;
    if (!buf) return SPMM_EWORKSPACE;
    const int vec = p->k % 8 == 0 && p->x_ld % 8 == 0 && (uintptr_t)p->x % 16 == 0;
    const int64_t per = vec ? p->k / 8 : p->k;
    const int threads = per >= 256 ? 256 : (int)ceil_div(per, 32) * 32;
    copy_rows_kernel<<<(unsigned)(p->rows < 65536 ? p->rows : 65536), threads, 0, s>>>(
        (const uint16_t *)p->x, p->x_ld, 0, p->x_rows, p->gather, buf, ld, 0, p->rows, p->k, vec);
    SPMM_PRODUCT_LAUNCHED();
    x = Operand{buf, ld};
    return SPMM_OK;
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

int forward(const spmm_linear *p, Arena &a, bool sizing, cudaStream_t s) {
    Operand x;
    SPMM_TRY(carve_x(p, a, sizing, x, s));
    if (sizing) return SPMM_OK;
    Product g = base(p);
    g.P = p->n;
    g.Q = p->rows;
    g.R = p->k;
    g.act = p->activation;
    g.A = p->w;
    g.a_p = p->w_n;
    g.a_r = p->w_k;
    g.a_g = p->w_g;
    g.B = x.ptr;
    g.b_q = x.ld;
    g.b_r = 1;
    g.C = p->y;
    g.c_q = p->y_ld;
    g.bias = p->bias;
    g.bias_g = p->bias_g;
    g.residual = p->residual;
    g.residual_ld = p->residual_ld;
    g.slope = p->slope;
    return launch_product(g, s);
}

template <typename T>
int gradients(const spmm_linear *p, Arena &a, bool sizing, cudaStream_t s) {
    Operand x{p->x, p->x_ld};
    if (p->dw) SPMM_TRY(carve_x(p, a, sizing, x, s));
    Operand dz{p->dy, p->dy_ld};
    const int64_t tiles = ceil_div(p->rows, kDzRows) + (p->offsets ? p->groups + 1 : 0);
    if (tiles > 65535) return SPMM_EUNSUPPORTED;
    T *dzp = nullptr;
    float *part = nullptr, *dxs = nullptr;
    const bool any = p->rows > 0 && p->n > 0;
    if (p->slope && any && (p->dx || p->dw)) {
        const int64_t ld = ceil_div(p->n, 8) * 8;
        dzp = a.take<T>(p->rows * ld);
        dz = Operand{dzp, ld};
    }
    if (p->dbias && any) part = a.take<float>(tiles * p->n);
    if (p->dx && p->gather) dxs = a.take<float>(p->rows * p->k);
    if (sizing) return SPMM_OK;
    if ((p->slope && any && (p->dx || p->dw) && !dzp) || (p->dbias && any && !part) || (p->dx && p->gather && !dxs))
        return SPMM_EWORKSPACE;
    if (dzp || part) {
        dz_kernel<T><<<dim3((unsigned)ceil_div(p->n, kDzCols), (unsigned)tiles), 256, 0, s>>>(
            (const T *)p->dy, p->dy_ld, p->slope, dzp, dz.ld, part, p->offsets, p->groups, p->rows, p->n);
        SPMM_PRODUCT_LAUNCHED();
    }
    if (p->dbias && p->n) {
        dbias_kernel<T><<<dim3((unsigned)ceil_div(p->n, 128), (unsigned)p->groups), 128, 0, s>>>(
            part, p->offsets, any ? p->rows : 0, p->n, (T *)p->dbias, p->dbias_g);
        SPMM_PRODUCT_LAUNCHED();
    }
    if (p->dx) {
        Product g = base(p);
        g.P = p->k;
        g.Q = p->rows;
        g.R = p->n;
        g.A = p->w;
        g.a_p = p->w_k;
        g.a_r = p->w_n;
        g.a_g = p->w_g;
        g.B = dz.ptr;
        g.b_q = dz.ld;
        g.b_r = 1;
        g.C = dxs ? (void *)dxs : p->dx;
        g.c_q = dxs ? p->k : p->dx_ld;
        g.out_f32 = dxs != nullptr;
        SPMM_TRY(launch_product(g, s));
        if (dxs)
            SPMM_TRY(launch_gather_sum(dxs, p->rows, p->slots, p->x_rows, p->top, p->k, p->dx, p->dx_ld, g.f16, s));
    }
    if (p->dw) {
        Product g = base(p);
        const bool n_unit = p->dw_n == 1;
        g.red = 1;
        g.R = p->rows;
        g.P = n_unit ? p->n : p->k;
        g.Q = n_unit ? p->k : p->n;
        g.A = n_unit ? dz.ptr : x.ptr;
        g.a_p = 1;
        g.a_r = n_unit ? dz.ld : x.ld;
        g.B = n_unit ? x.ptr : dz.ptr;
        g.b_q = 1;
        g.b_r = n_unit ? x.ld : dz.ld;
        g.C = p->dw;
        g.c_q = n_unit ? p->dw_k : p->dw_n;
        g.c_g = p->dw_g;
        SPMM_TRY(launch_product(g, s));
    }
    return SPMM_OK;
}

int backward(const spmm_linear *p, Arena &a, bool sizing, cudaStream_t s) {
    return p->dtype == SPMM_DENSE_F16 ? gradients<__half>(p, a, sizing, s)
                                      : gradients<__nv_bfloat16>(p, a, sizing, s);
}

size_t sized(const spmm_linear *p, int (*run)(const spmm_linear *, Arena &, bool, cudaStream_t)) {
    if (check_sizes(p) != SPMM_OK) return 0;
    Arena a(nullptr, 0);
    (void)run(p, a, true, nullptr);
    return (a.used + 255) & ~(size_t)255;
}

int clear_status(const spmm_linear *p, cudaStream_t s) {
    if (!p->status) return SPMM_OK;
    clear_status_kernel<<<1, 1, 0, s>>>(p->status);
    SPMM_LAUNCH_CHECK();
    return SPMM_OK;
}

}  // namespace

int launch_product(const Product &p, cudaStream_t s) {
    if (p.P == 0 || p.Q == 0) return SPMM_OK;
    const int64_t gy = p.red ? p.groups * ceil_div(p.Q, 64) : ceil_div(p.Q, 64) + (p.offsets ? p.groups + 1 : 0);
    if (gy > 65535) return SPMM_EUNSUPPORTED;
    const dim3 grid((unsigned)ceil_div(p.P, 64), (unsigned)gy);
    if (p.f16) return p.out_f32 ? launch_act<__half, float>(p, grid, s) : launch_act<__half, __half>(p, grid, s);
    return p.out_f32 ? launch_act<__nv_bfloat16, float>(p, grid, s)
                     : launch_act<__nv_bfloat16, __nv_bfloat16>(p, grid, s);
}

int launch_gather_sum(const float *src, int64_t rows, const int32_t *slots, int64_t tokens, int64_t top, int64_t n,
                      void *out, int64_t out_ld, int f16, cudaStream_t s) {
    if (tokens == 0 || n == 0) return SPMM_OK;
    const unsigned grid = (unsigned)(tokens < 65536 ? tokens : 65536);
    if (f16)
        gather_sum_kernel<<<grid, 256, 0, s>>>(src, rows, slots, tokens, top, n, (__half *)out, out_ld);
    else
        gather_sum_kernel<<<grid, 256, 0, s>>>(src, rows, slots, tokens, top, n, (__nv_bfloat16 *)out, out_ld);
    SPMM_PRODUCT_LAUNCHED();
    return SPMM_OK;
}

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
    SPMM_TRY(spmm::clear_status(p, (cudaStream_t)stream));
    spmm::Arena a(p->workspace, p->workspace_bytes);
    return spmm::forward(p, a, false, (cudaStream_t)stream);
}

extern "C" int spmm_linear_backward(const spmm_linear *p, spmm_stream_t stream) {
    SPMM_TRY(spmm::check_sizes(p));
    if (p->rows * p->n && !p->dy) return SPMM_EINVAL;
    if (p->dx && ((p->k * p->n && !p->w) || (p->gather && (!p->slots || p->top < 1)))) return SPMM_EINVAL;
    if (p->dw && ((p->rows * p->k && !p->x) || (p->dw_k != 1 && p->dw_n != 1))) return SPMM_EINVAL;
    SPMM_TRY(spmm::clear_status(p, (cudaStream_t)stream));
    spmm::Arena a(p->workspace, p->workspace_bytes);
    return spmm::backward(p, a, false, (cudaStream_t)stream);
}
