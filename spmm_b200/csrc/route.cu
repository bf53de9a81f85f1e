// route.cu -- expert choice, the grouping of the chosen rows, and the weighted
// sums back in token order.
//
// Choice.  A warp per token holds the token's logits in registers (expert e in
// lane e % 32); top rounds of a warp-wide maximum over order-preserving 32-bit
// keys, ties resolved to the lowest expert by a second reduction.  The choice
// depends on float32(logit) + bias alone, so it is exact; weights come from
// float32 exponentials relative to the row's maximum.
//
// Grouping.  A stable counting sort by expert: tokens are cut into one chunk per
// SM, a CTA counts its chunk's choices per expert, and a second kernel's CTA per
// chunk sums the counts of the chunks before its own and places its choices in
// order (ranks within a warp by match, warps by a prefix over their counts).
// Integer sums only: the result does not depend on the order of the atomics.  A
// third kernel that scanned the counts of 512 chunks cost 5 us and a launch.
#include <type_traits>

#include "linear.cuh"

namespace spmm {
namespace {

constexpr int kWarps = 8;                  // warps of a CTA that differentiates
constexpr int kMaxExperts = SPMM_MAX_GROUPS;
constexpr uint32_t kNone = 0x007FFFFFu;    // key of -inf: not selectable, like every smaller key

// Order-preserving key: a < b as floats <=> key(a) < key(b); -0 counts as +0, NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) return kNone;
    const uint32_t u = __float_as_uint(v + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The same in 16 bits for a 16-bit value, and the key of its -inf.
template <typename T>
__device__ __forceinline__ uint32_t half_key(float v) {
    if (v != v) v = -INFINITY;
    const T h = from_f32<T>(v + 0.f);
    uint16_t u;
    memcpy(&u, &h, 2);
    return u & 0x8000u ? (uint16_t)~u : u | 0x8000u;
}
template <typename T>
__host__ __device__ constexpr uint32_t half_floor() {
    return sizeof(T) == 2 ? (std::is_same<T, __half>::value ? 0x03FFu : 0x007Fu) : 0u;
}

// A logit as the weights use it: +inf as the largest float, NaN as -inf.
__device__ __forceinline__ float clean_logit(float v) {
    return v != v ? -INFINITY : fminf(v, 3.402823466e38f);
}

struct Row {
    float peak;    // softmax: largest logit (0 when there is none)
    float total;   // softmax: sum of exp(logit - peak)
};

template <int V>
__device__ __forceinline__ Row softmax_row(const float (&l)[V]) {
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) m = fmaxf(m, l[v]);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, o));
    if (m == -INFINITY) m = 0.f;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) s += expf(l[v] - m);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
    return {m, s};
}

template <typename T, int V>
__device__ __forceinline__ void load_row(const T *row, int experts, int lane, float (&l)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = v * 32 + lane;
        l[v] = e < experts ? to_f32(row[e]) : -INFINITY;
    }
}

// sigmoid(v); 1 - sigmoid(v) is sigmoid(-v).  The exponential is of -|v|, so that neither end loses its bits: 1 - s
// is 0 in float32 from a logit of 17 on, and 1 / (1 + exp(-v)) is 0 below -88.
__device__ __forceinline__ float sigmoid(float v) {
    const float e = expf(-fabsf(v));
    return (v > 0.f ? 1.f : e) / (1.f + e);
}

// A renormalised sigmoid counts as 0 below this logit, where 64 bits cannot hold 1 + exp(-v) either: what masks by
// the type's lowest value leave.
constexpr float kSigmoidZero = -709.78f;

// sigmoid(mine) over the sum of the chosen lanes' sigmoids, in a whole warp.  Sigmoids are taken relative to
// exp(min(largest logit, 0)), so that the sum is at least 1 / 2 and small ones keep their ratios.
__device__ __forceinline__ float sigmoid_share(float mine, bool chosen) {
    const bool live = chosen && mine > kSigmoidZero;
    const uint32_t m = __reduce_max_sync(kFullMask, live ? order_key(mine) : 0u);
    const float largest = __uint_as_float(m & 0x80000000u ? m & 0x7FFFFFFFu : ~m);
    const float e = expf(-fabsf(mine));
    const float s = !live ? 0.f : (mine > 0.f ? 1.f : expf(mine - fminf(largest, 0.f))) / (1.f + e);
    float sum = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
    return sum > 0.f ? s / sum : 0.f;
}

// Descending, by Batcher's odd-even merge network.
template <int V>
__device__ __forceinline__ void sort_descending(uint32_t (&k)[V]) {
#pragma unroll
    for (int p = 1; p < V; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < V; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t a = k[i + j], b = k[i + j + q];
                        k[i + j] = a > b ? a : b;
                        k[i + j + q] = a > b ? b : a;
                    }
}

// One token: lane j < top ends with choice j in (expert, weight).
//
// PACKED (16-bit logits without bias): a 16-bit key with the expert below it
// makes one 32-bit word; each lane sorts its words once, and a round is one
// reduction of the lanes' first ones and a shift in the lane that won.
// Otherwise the key needs all 32 bits and the expert a second reduction.
template <typename T, int V, bool PACKED>
__device__ __forceinline__ void choose(const spmm_route_args &p, int64_t t, int lane, int &expert, float &weight) {
    const int experts = (int)p.experts, top = (int)p.top;
    float l[V];
    load_row<T, V>((const T *)p.logits + t * p.logits_ld, experts, lane, l);
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = v * 32 + lane;
        if constexpr (PACKED) {
            key[v] = e >= experts ? 0u : half_key<T>(l[v]) << 16 | (0xFFFFu - e);
        } else {
            key[v] = e >= experts ? 0u : order_key(p.bias ? l[v] + __ldg(p.bias + e) : l[v]);
        }
        l[v] = clean_logit(l[v]);
    }
    if constexpr (PACKED) sort_descending(key);
    expert = -1;
    float mine = -INFINITY;   // the logit of this lane's choice
    for (int j = 0; j < top; ++j) {
        int e;
        if constexpr (PACKED) {
            const uint32_t m = __reduce_max_sync(kFullMask, key[0]);
            if (m >> 16 <= half_floor<T>()) break;
            e = (int)(0xFFFFu - (m & 0xFFFFu));
            const bool won = key[0] == m;
#pragma unroll
            for (int v = 0; v < V; ++v) key[v] = won ? (v + 1 < V ? key[v + 1] : 0u) : key[v];
        } else {
            uint32_t best = 0u;
            int at = 0;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (key[v] > best) {
                    best = key[v];
                    at = v;
                }
            const uint32_t m = __reduce_max_sync(kFullMask, best);
            if (m <= kNone) break;
            e = (int)__reduce_min_sync(kFullMask, best == m ? (unsigned)(at * 32 + lane) : ~0u);
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v * 32 + lane == e) key[v] = 0u;
        }
        if (lane == j) expert = e;
    }
    // each choice's logit, from the row just read
    if (expert >= 0) mine = clean_logit(to_f32(((const T *)p.logits)[t * p.logits_ld + expert]));
    __syncwarp();
    // weights
    if (p.scoring == SPMM_SCORE_SOFTMAX) {
        Row r;
        if (p.renormalize) {   // relative to the chosen ones alone
            float c[1] = {mine};
            r = softmax_row<1>(c);
        } else {
            r = softmax_row<V>(l);
        }
        weight = expert >= 0 && r.total > 0.f ? expf(mine - r.peak) / r.total : 0.f;
    } else if (p.renormalize) {
        weight = sigmoid_share(mine, expert >= 0);
    } else {
        weight = expert >= 0 ? sigmoid(mine) : 0.f;
    }
    weight *= p.scale;
}

// Choices of the tokens [t0, t1) of this CTA, and their counts per expert in `count`.
template <typename T, int V, bool PACKED>
__device__ __forceinline__ void choose_chunk(const spmm_route_args &p, int64_t t0, int64_t t1, int *count) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (int64_t t = t0 + warp; t < t1; t += warps) {
        int e;
        float w;
        choose<T, V, PACKED>(p, t, lane, e, w);
        if (lane < p.top) {
            p.weights[t * p.top + lane] = w;
            p.experts_out[t * p.top + lane] = e;
            if (e >= 0) atomicAdd(count + e, 1);
        }
    }
}

// Exclusive prefix sums of v[0, n) in place, the total returned; the whole CTA.
__device__ __forceinline__ int cta_exclusive(int *v, int n, int *tmp /* 33 */) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int carry = 0;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        const int x = i < n ? v[i] : 0;
        int s = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(kFullMask, s, o);
            if (lane >= o) s += y;
        }
        if (lane == 31) tmp[warp] = s;
        __syncthreads();
        if (warp == 0) {
            const int own = lane < warps ? tmp[lane] : 0;
            int b = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(kFullMask, b, o);
                if (lane >= o) b += y;
            }
            tmp[lane] = b - own;
            if (lane == 31) tmp[32] = b;
        }
        __syncthreads();
        if (i < n) v[i] = carry + tmp[warp] + s - x;
        carry += tmp[32];
        __syncthreads();
    }
    return carry;
}

// Places the choices [i0, i1) (flat, in order) of this CTA: base[e] is the position of the chunk's first choice
// of expert e.  `wcount`: [warps][experts].  Each warp owns a contiguous part.
__device__ __forceinline__ void place(const spmm_route_args &p, int64_t i0, int64_t i1, const int *base,
                                      int *wcount) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int experts = (int)p.experts;
    const int64_t part = ((i1 - i0 + warps - 1) / warps + 31) / 32 * 32;
    const int64_t a = i0 + warp * part, b = a + part < i1 ? a + part : i1;
    int *mine = wcount + warp * experts;
    for (int e = lane; e < experts; e += 32) mine[e] = 0;
    __syncwarp();
    for (int64_t i = a + lane; i < b; i += 32) {
        const int e = p.experts_out[i];
        if (e >= 0) atomicAdd(mine + e, 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {
        int run = base[e];
        for (int w = 0; w < warps; ++w) {
            const int c = wcount[w * experts + e];
            wcount[w * experts + e] = run;
            run += c;
        }
    }
    __syncthreads();
    for (int64_t i = a; i < b; i += 32) {   // a and the loop bound are the same for the whole warp
        const bool in = i + lane < b;
        const int e = in ? p.experts_out[i + lane] : -1;
        const unsigned same = __match_any_sync(kFullMask, e);
        const int rank = __popc(same & lanemask_lt());
        int pos = -1;
        if (e >= 0) pos = mine[e] + rank;
        __syncwarp();
        if (e >= 0 && rank == 0) mine[e] += __popc(same);
        __syncwarp();
        if (in) {
            p.slots[i + lane] = pos;
            if (pos >= 0) p.rows[pos] = (int32_t)((i + lane) / p.top);
        }
    }
}

// Everything in one CTA: for few tokens, where launches are what it costs.
template <typename T, int V, bool PACKED>
__global__ void __launch_bounds__(V <= 8 ? 1024 : 512) route_small_kernel(spmm_route_args p) {
    chained_start();
    extern __shared__ int sm[];
    __shared__ int tmp[33];
    const int experts = (int)p.experts;
    int *count = sm, *wcount = sm + experts;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) count[e] = 0;
    __syncthreads();
    choose_chunk<T, V, PACKED>(p, 0, p.tokens, count);
    __syncthreads();
    const int total = cta_exclusive(count, experts, tmp);
    for (int e = threadIdx.x; e < experts; e += blockDim.x) p.offsets[e] = count[e];
    if (threadIdx.x == 0) p.offsets[experts] = total;
    const int64_t all = p.tokens * p.top;
    for (int64_t i = total + threadIdx.x; i < all; i += blockDim.x) p.rows[i] = -1;
    place(p, 0, all, count, wcount);
}

template <typename T, int V, bool PACKED>
__global__ void __launch_bounds__(V <= 8 ? 1024 : 512) route_choose_kernel(spmm_route_args p, int64_t chunk, int *counts) {
    chained_start();
    extern __shared__ int sm[];
    const int experts = (int)p.experts;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) sm[e] = 0;
    __syncthreads();
    const int64_t t0 = blockIdx.x * chunk, t1 = t0 + chunk < p.tokens ? t0 + chunk : p.tokens;
    choose_chunk<T, V, PACKED>(p, t0, t1, sm);
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[(int64_t)blockIdx.x * experts + e] = sm[e];
}

__global__ void __launch_bounds__(1024) route_place_kernel(spmm_route_args p, int64_t chunk, const int *counts,
                                                           int chunks) {
    chained_start();
    extern __shared__ int sm[];
    __shared__ int tmp[33];
    const int experts = (int)p.experts;
    int *base = sm, *wcount = sm + experts;
    int *before = wcount;              // choices of an expert in earlier chunks, until place() needs the room
    for (int e = threadIdx.x; e < experts; e += blockDim.x) base[e] = before[e] = 0;
    __syncthreads();
    // Four experts a thread where their number allows, several threads an expert, each every parts-th chunk: what
    // this costs is the loads' latency.
    const int each = experts % 4 == 0 ? 4 : 1, columns = experts / each;
    const int parts = (int)blockDim.x > columns ? blockDim.x / columns : 1;
    for (int i = threadIdx.x; i < parts * columns; i += blockDim.x) {
        const int e = i % columns * each;
        int sum[4] = {}, earlier[4] = {};
#pragma unroll 8
        for (int c = i / columns; c < chunks; c += parts) {
            int v[4] = {};
            const int *row = counts + (int64_t)c * experts + e;
            if (each == 4) {
                const int4 w = __ldg((const int4 *)row);
                v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
            } else {
                v[0] = __ldg(row);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                earlier[u] += c < (int)blockIdx.x ? v[u] : 0;
                sum[u] += v[u];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (u < each) {
                atomicAdd(base + e + u, sum[u]);
                atomicAdd(before + e + u, earlier[u]);
            }
    }
    __syncthreads();
    const int total = cta_exclusive(base, experts, tmp);
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e < experts; e += blockDim.x) p.offsets[e] = base[e];
        if (threadIdx.x == 0) p.offsets[experts] = total;
        __syncthreads();
    }
    const int64_t all = p.tokens * p.top;
    const int64_t i0 = blockIdx.x * chunk * p.top, i1 = i0 + chunk * p.top < all ? i0 + chunk * p.top : all;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += blockDim.x)
        if (i >= total) p.rows[i] = -1;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) base[e] += before[e];
    __syncthreads();
    place(p, i0, i1, base, wcount);
}

// dlogits, a warp per token.  With g = scale * dweights at the chosen experts and 0 elsewhere:
//   renormalised, w = s / sum s:  ds = (g - <g, w>) / sum s at the chosen ones
//   softmax over all:             dl = p (ds - <ds, p>);  renormalised, s = exp(l) of the chosen ones: w (g - <g, w>)
//   sigmoid:                      dl = ds s (1 - s);  renormalised w (g - <g, w>) (1 - s)
template <typename T, int V>
__global__ void __launch_bounds__(kWarps * 32) route_backward_kernel(spmm_route_args p) {
    chained_start();
    const int lane = threadIdx.x & 31;
    const int experts = (int)p.experts, top = (int)p.top;
    const int64_t step = (int64_t)gridDim.x * kWarps;
    for (int64_t t = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); t < p.tokens; t += step) {
        const T *row = (const T *)p.logits + t * p.logits_ld;
        T *out = (T *)p.dlogits + t * experts;
        int e = -1;
        float g = 0.f, l = -INFINITY;
        if (lane < top) {
            e = p.experts_out[t * top + lane];
            if (e >= experts) e = -1;
            if (e >= 0) {
                g = p.scale * p.dweights[t * top + lane];
                l = clean_logit(to_f32(row[e]));
            }
        }
        float d;               // gradient at this lane's choice
        float all = 0.f;       // softmax over all: <g, p>
        Row r{0.f, 1.f};
        float s = 0.f;
        if (p.scoring == SPMM_SCORE_SOFTMAX) {
            if (p.renormalize) {
                float c[1] = {l};
                r = softmax_row<1>(c);
            } else {
                float x[V];
                load_row<T, V>(row, experts, lane, x);
#pragma unroll
                for (int v = 0; v < V; ++v) x[v] = clean_logit(x[v]);
                r = softmax_row<V>(x);
            }
            s = e >= 0 && r.total > 0.f ? expf(l - r.peak) / r.total : 0.f;
        } else {               // the weight
            s = p.renormalize ? sigmoid_share(l, e >= 0) : e >= 0 ? sigmoid(l) : 0.f;
        }
        float dot = g * s;
#pragma unroll
        for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(kFullMask, dot, o);
        if (p.scoring == SPMM_SCORE_SOFTMAX) {
            d = s * (g - dot);
            all = p.renormalize ? 0.f : dot;
        } else {
            d = s * (p.renormalize ? g - dot : g) * sigmoid(-l);
        }
        if (all != 0.f) {      // softmax over all: experts that were not chosen have -p <g, p>
            float x[V];
            load_row<T, V>(row, experts, lane, x);
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v * 32 + lane < experts)
                    out[v * 32 + lane] = from_f32<T>(-all * (expf(clean_logit(x[v]) - r.peak) / r.total));
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v * 32 + lane < experts) out[v * 32 + lane] = from_f32<T>(0.f);
        }
        __syncwarp();
        if (e >= 0) out[e] = from_f32<T>(d);
    }
}

// ---- combine --------------------------------------------------------------------

// VEC values as they lie in memory: loads are issued together and converted
// afterwards, or each would be waited for in turn.
template <typename T, int VEC>
struct Raw {
    typename std::conditional<VEC * sizeof(T) == 16, uint4, T>::type v;
    static_assert(VEC * sizeof(T) == 16 || VEC == 1, "one value or 16 bytes");

    __device__ __forceinline__ void clear() { memset(&v, 0, sizeof(v)); }
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (VEC * sizeof(T) == 16) v = __ldg(reinterpret_cast<const uint4 *>(p));
        else v = p[0];
    }
    __device__ __forceinline__ void get(float (&f)[VEC]) const {
        T t[VEC];
        memcpy(t, &v, sizeof(t));
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = to_f32(t[i]);
    }
};
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float (&f)[VEC]) {
    T t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = from_f32<T>(f[i]);
    if constexpr (VEC * sizeof(T) == 16) {
        uint4 u;
        memcpy(&u, t, 16);
        *reinterpret_cast<uint4 *>(p) = u;
    } else {
        p[0] = t[0];
    }
}

// A warp per token, or per part of its columns where tokens are few: lane j
// holds choice j's slot and weight, and the chosen rows' loads are issued eight
// at a time.  Bound by reading each chosen row once.  A warp per 32 VEC columns
// whatever the tokens, each fetching the slots anew, took twice as long
// (16384 tokens x 8 rows of 4 KB: 229 us).
template <typename T, int VEC>
__global__ void __launch_bounds__(256, 3) combine_kernel(const __grid_constant__ spmm_combine_args p, int parts,
                                                         int part_cols) {
    chained_start();
    const int lane = threadIdx.x & 31, top = (int)p.top;
    const int64_t items = p.tokens * parts, step = (int64_t)gridDim.x * 8;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < items; i += step) {
        const int64_t t = i / parts, c0 = (i - t * parts) * part_cols;
        const int64_t end = c0 + part_cols < p.n ? c0 + part_cols : p.n;
        int slot = -1;
        float weight = 0.f;
        if (lane < top) {
            slot = __ldg(p.slots + t * top + lane);
            weight = __ldg(p.weights + t * top + lane);
            if (slot >= p.rows) slot = -1;
        }
        int s[8];
        float w[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            s[u] = __shfl_sync(kFullMask, slot, u);
            w[u] = __shfl_sync(kFullMask, weight, u);
        }
        for (int64_t cb = c0; cb < end; cb += 32 * VEC) {      // the whole warp
            const int64_t c = cb + lane * VEC;
            const bool in = c < end;
            Raw<T, VEC> residual, y[8];
            if (p.residual && in) residual.load((const T *)p.residual + t * p.residual_ld + c);
            float acc[VEC] = {};
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                y[u].clear();
                if (s[u] >= 0 && in) y[u].load((const T *)p.y + s[u] * p.y_ld + c);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (s[u] >= 0) {
                    float f[VEC];
                    y[u].get(f);
#pragma unroll
                    for (int x = 0; x < VEC; ++x) acc[x] = fmaf(w[u], f[x], acc[x]);
                }
            for (int j = 8; j < top; j += 4) {                 // more than eight choices
                Raw<T, VEC> z[4];
                int sj[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    sj[u] = j + u < top ? __ldg(p.slots + t * top + j + u) : -1;
                    z[u].clear();
                    if (sj[u] >= 0 && sj[u] < p.rows && in) z[u].load((const T *)p.y + sj[u] * p.y_ld + c);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (sj[u] >= 0 && sj[u] < p.rows) {
                        const float wj = __ldg(p.weights + t * top + j + u);
                        float f[VEC];
                        z[u].get(f);
#pragma unroll
                        for (int x = 0; x < VEC; ++x) acc[x] = fmaf(wj, f[x], acc[x]);
                    }
            }
            if (!in) continue;
            if (p.residual) {
                float f[VEC];
                residual.get(f);
#pragma unroll
                for (int x = 0; x < VEC; ++x) acc[x] += f[x];
            }
            store_vec<T, VEC>((T *)p.out + t * p.out_ld + c, acc);
        }
    }
}

// A warp per token: dout's row, read once per eight choices, against their rows
// of y, with eight sums in registers.
template <typename T, int VEC>
__global__ void __launch_bounds__(256, 3) combine_backward_kernel(const __grid_constant__ spmm_combine_args p,
                                                                  const int32_t *tokens_of) {
    chained_start();
    const int lane = threadIdx.x & 31, top = (int)p.top;
    const int64_t step = (int64_t)gridDim.x * 8;
    const int64_t w0 = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    for (int64_t t = w0; t < p.tokens; t += step) {
        for (int j0 = 0; j0 < top; j0 += 8) {
            int slot = -1;
            float weight = 0.f;
            if (lane < 8 && j0 + lane < top) {
                slot = __ldg(p.slots + t * top + j0 + lane);
                weight = __ldg(p.weights + t * top + j0 + lane);
                if (slot >= p.rows) slot = -1;
            }
            int s[8];
            float w[8], dot[8] = {};
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                s[u] = __shfl_sync(kFullMask, slot, u);
                w[u] = __shfl_sync(kFullMask, weight, u);
            }
            for (int64_t c = lane * VEC; c < p.n; c += 32 * VEC) {
                Raw<T, VEC> dr, y[8];
                dr.load((const T *)p.dout + t * p.dout_ld + c);
                if (p.dweights) {
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        y[u].clear();
                        if (s[u] >= 0) y[u].load((const T *)p.y + s[u] * p.y_ld + c);
                    }
                }
                float d[VEC];
                dr.get(d);
                if (p.dweights) {
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (s[u] >= 0) {
                            float f[VEC];
                            y[u].get(f);
#pragma unroll
                            for (int x = 0; x < VEC; ++x) dot[u] = fmaf(d[x], f[x], dot[u]);
                        }
                }
                if (p.dy) {
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (s[u] >= 0) {
                            float o[VEC];
#pragma unroll
                            for (int x = 0; x < VEC; ++x) o[x] = w[u] * d[x];
                            store_vec<T, VEC>((T *)p.dy + s[u] * p.dy_ld + c, o);
                        }
                }
            }
            if (p.dweights) {
                float mine = 0.f;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    float v = dot[u];
#pragma unroll
                    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
                    if (lane == u) mine = v;
                }
                if (lane < 8 && j0 + lane < top) p.dweights[t * top + j0 + lane] = mine;
            }
        }
    }
    if (p.dy == nullptr) return;
    auto clear = [&](int64_t r) {
        for (int64_t c = lane; c < p.n; c += 32) ((T *)p.dy)[r * p.dy_ld + c] = from_f32<T>(0.f);
    };
    const int64_t end = group_first(p.offsets, p.experts, p.rows);
    for (int64_t r = end + w0; r < p.rows; r += step) clear(r);      // behind the last group
    if (tokens_of == nullptr) return;
    for (int64_t r0 = w0 * 32; r0 < end; r0 += step * 32) {          // rows that no choice has, a lane each
        const int64_t r = r0 + lane, t = r < end ? __ldg(tokens_of + r) : -1;
        bool named = r >= end;
        if (t >= 0 && t < p.tokens)
            for (int j = 0; j < top; ++j) named |= __ldg(p.slots + t * top + j) == r;
        for (unsigned left = __ballot_sync(kFullMask, !named); left; left &= left - 1) clear(r0 + __ffs(left) - 1);
    }
}

// ---- host side --------------------------------------------------------------------

constexpr int64_t kChunks = 148;   // chunks of the grouping, at most

// Warps of a CTA that keeps an int per expert and warp in shared memory (below 48 KB with the static part).
int warps_for(int64_t experts, int most) {
    const int64_t fit = 40 * 1024 / (experts * 4) - 1;
    return (int)(fit < 1 ? 1 : fit < most ? fit : most);
}

int check_route(const spmm_route_args *p) {
    if (!p || p->version != 1) return SPMM_EINVAL;
    if (p->dtype != SPMM_DENSE_F32 && p->dtype != SPMM_DENSE_BF16 && p->dtype != SPMM_DENSE_F16)
        return SPMM_EUNSUPPORTED;
    if (p->tokens < 0 || p->experts < 1 || p->top < 1 || p->top > p->experts) return SPMM_EINVAL;
    if (p->experts > kMaxExperts || p->top > SPMM_MAX_TOP || p->tokens > INT32_MAX / p->top)
        return SPMM_EUNSUPPORTED;
    if (p->scoring != SPMM_SCORE_SOFTMAX && p->scoring != SPMM_SCORE_SIGMOID) return SPMM_EINVAL;
    if (!on_boundary(p->dtype == SPMM_DENSE_F32 ? 4 : 2, {p->logits, p->dlogits}) ||
        !on_boundary(4, {p->bias, p->weights, p->experts_out, p->slots, p->rows, p->offsets, p->dweights}) ||
        !on_boundary(16, {p->workspace}))
        return SPMM_EALIGN;
    return SPMM_OK;
}

bool small_route(const spmm_route_args *p) { return p->tokens <= 128; }

int64_t chunk_tokens(const spmm_route_args *p) {
    const int64_t c = ceil_div(p->tokens, kChunks);
    return c < 32 ? 32 : c;
}

template <typename T, int V, bool PACKED>
int run_route(const spmm_route_args &p, cudaStream_t s) {
    const int e4 = (int)p.experts * 4, most = V <= 8 ? 32 : 16;   // registers: V logits and keys a thread
    if (small_route(&p)) {
        const int fit = warps_for(p.experts, most);
        const int warps = (int)(p.tokens < 1 ? 1 : p.tokens < fit ? p.tokens : fit);
        return launch_chained(route_small_kernel<T, V, PACKED>, dim3(1), warps * 32, (warps + 1) * e4, s, 1, p);
    }
    const int64_t chunk = chunk_tokens(&p), chunks = ceil_div(p.tokens, chunk);
    int *counts = (int *)p.workspace;
    const int choose = (int)(chunk < most ? chunk : most), place = warps_for(p.experts, 32);
    SPMM_TRY(launch_chained(route_choose_kernel<T, V, PACKED>, dim3((unsigned)chunks), choose * 32, e4, s, 1, p, chunk,
                            counts));
    return launch_chained(route_place_kernel, dim3((unsigned)chunks), place * 32, (place + 1) * e4, s, 1, p, chunk, counts,
                          (int)chunks);
}

template <typename T, int V>
int run_route_backward(const spmm_route_args &p, cudaStream_t s) {
    int64_t grid = ceil_div(p.tokens, kWarps);
    if (grid > 148 * 8) grid = 148 * 8;
    return launch_chained(route_backward_kernel<T, V>, dim3((unsigned)grid), kWarps * 32, 0, s, 1, p);
}

template <typename T>
int by_width(const spmm_route_args &p, bool backward, cudaStream_t s) {
#define SPMM_ROUTE_V(V)                                         \
    do {                                                        \
        if (backward) return run_route_backward<T, V>(p, s);    \
        if constexpr (sizeof(T) == 2)                           \
            if (!p.bias) return run_route<T, V, true>(p, s);    \
        return run_route<T, V, false>(p, s);                    \
    } while (0)
    if (p.experts <= 32) SPMM_ROUTE_V(1);
    if (p.experts <= 64) SPMM_ROUTE_V(2);
    if (p.experts <= 128) SPMM_ROUTE_V(4);
    if (p.experts <= 256) SPMM_ROUTE_V(8);
    if (p.experts <= 512) SPMM_ROUTE_V(16);
    SPMM_ROUTE_V(32);
#undef SPMM_ROUTE_V
}

int by_type(const spmm_route_args &p, bool backward, cudaStream_t s) {
    if (p.dtype == SPMM_DENSE_F32) return by_width<float>(p, backward, s);
    if (p.dtype == SPMM_DENSE_F16) return by_width<__half>(p, backward, s);
    return by_width<__nv_bfloat16>(p, backward, s);
}

int check_combine(const spmm_combine_args *p) {
    if (!p || p->version != 1) return SPMM_EINVAL;
    if (p->dtype != SPMM_DENSE_F32 && p->dtype != SPMM_DENSE_BF16 && p->dtype != SPMM_DENSE_F16)
        return SPMM_EUNSUPPORTED;
    if (p->tokens < 0 || p->top < 1 || p->rows < 0 || p->n < 0) return SPMM_EINVAL;
    if (p->rows > INT32_MAX || p->top > INT32_MAX) return SPMM_EUNSUPPORTED;
    if (!on_boundary(p->dtype == SPMM_DENSE_F32 ? 4 : 2, {p->y, p->residual, p->out, p->dout, p->dy}) ||
        !on_boundary(4, {p->slots, p->offsets, p->weights, p->dweights}))
        return SPMM_EALIGN;
    return SPMM_OK;
}

bool aligned16(const void *p, int64_t ld, int64_t per) { return (uintptr_t)p % 16 == 0 && ld % per == 0; }

template <typename T>
int run_combine(const spmm_combine_args &p, bool backward, const int32_t *tokens_of, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    bool vec = p.n % W == 0 && aligned16(p.y, p.y_ld, W);
    if (backward)
        vec = vec && aligned16(p.dout, p.dout_ld, W) && aligned16(p.dy, p.dy_ld, W);
    else
        vec = vec && aligned16(p.out, p.out_ld, W) && aligned16(p.residual, p.residual_ld, W);
    if (backward) {
        int64_t grid = ceil_div(p.tokens > 0 ? p.tokens : 1, 8);
        if (grid > 148 * 8) grid = 148 * 8;
        return launch_chained(vec ? combine_backward_kernel<T, W> : combine_backward_kernel<T, 1>, dim3((unsigned)grid),
                              256, 0, s, 1, p, tokens_of);
    }
    {
        const int64_t wide = vec ? 32 * W : 32, chunks = ceil_div(p.n, wide);
        if (p.n > INT32_MAX - 1024) return SPMM_EUNSUPPORTED;
        int64_t parts = ceil_div(148 * 24, p.tokens);          // 24 warps an SM are resident
        if (parts > chunks) parts = chunks;
        const int64_t cols = ceil_div(chunks, parts) * wide;
        parts = ceil_div(p.n, cols);
        int64_t grid = ceil_div(p.tokens * parts, 8);
        if (grid > 148 * 12) grid = 148 * 12;
        return launch_chained(vec ? combine_kernel<T, W> : combine_kernel<T, 1>, dim3((unsigned)grid), 256, 0, s, 1, p,
                              (int)parts, (int)cols);
    }
}

}  // namespace
}  // namespace spmm

using namespace spmm;

extern "C" size_t spmm_route_workspace_size(const spmm_route_args *p) {
    if (check_route(p) != SPMM_OK || small_route(p)) return 0;
    return (size_t)ceil_div(p->tokens, chunk_tokens(p)) * p->experts * 4;
}

extern "C" int spmm_route(const spmm_route_args *p, spmm_stream_t stream) {
    SPMM_TRY(check_route(p));
    if (!p->offsets || (p->tokens && (!p->logits || !p->weights || !p->experts_out || !p->slots || !p->rows)))
        return SPMM_EINVAL;
    const size_t need = spmm_route_workspace_size(p);
    if (need && (!p->workspace || p->workspace_bytes < need)) return SPMM_EWORKSPACE;
    return by_type(*p, false, (cudaStream_t)stream);
}

extern "C" int spmm_route_backward(const spmm_route_args *p, spmm_stream_t stream) {
    SPMM_TRY(check_route(p));
    if (p->tokens == 0) return SPMM_OK;
    if (!p->logits || !p->experts_out || !p->dweights || !p->dlogits) return SPMM_EINVAL;
    return by_type(*p, true, (cudaStream_t)stream);
}

static int combine_by_type(const spmm_combine_args *p, bool backward, const int32_t *tokens_of, cudaStream_t s) {
    if (p->dtype == SPMM_DENSE_F32) return run_combine<float>(*p, backward, tokens_of, s);
    if (p->dtype == SPMM_DENSE_F16) return run_combine<__half>(*p, backward, tokens_of, s);
    return run_combine<__nv_bfloat16>(*p, backward, tokens_of, s);
}

extern "C" int spmm_combine(const spmm_combine_args *p, spmm_stream_t stream) {
    SPMM_TRY(check_combine(p));
    if (p->tokens == 0 || p->n == 0) return SPMM_OK;
    if (!p->slots || !p->weights || !p->out || (p->rows && !p->y)) return SPMM_EINVAL;
    return combine_by_type(p, false, nullptr, (cudaStream_t)stream);
}

extern "C" int spmm_combine_backward_rows(const spmm_combine_args *p, const int32_t *tokens_of, spmm_stream_t stream) {
    SPMM_TRY(check_combine(p));
    if (!on_boundary(4, {tokens_of})) return SPMM_EALIGN;
    if (!p->dy && !p->dweights) return SPMM_OK;
    if (p->tokens && (!p->slots || !p->weights || (p->n && (!p->dout || (p->rows && !p->y))))) return SPMM_EINVAL;
    if (p->dy && (!p->offsets || p->experts < 0)) return SPMM_EINVAL;
    return combine_by_type(p, true, tokens_of, (cudaStream_t)stream);
}

extern "C" int spmm_combine_backward(const spmm_combine_args *p, spmm_stream_t stream) {
    return spmm_combine_backward_rows(p, nullptr, stream);
}
