// linear_tc.cu -- D[p][q] = sum_r A[p][r] B[q][r] for 16-bit operands on the
// 5th-generation tensor cores: the kernel behind the dense and grouped products
// (linear.cuh).
//
// A tile is 128 p (tensor-memory lanes) x up to BQ q (tensor-memory columns).
// p is the dimension that is contiguous in the result (features), q the other
// one (rows of x, or the second weight dimension for dw): a group of 37 rows
// costs an MMA of N = 48, not a padded tile of 128.  With CG = 2 two CTAs
// share a tile of 256 p x BQ q (cta_group::2): each loads its 128 rows of A
// and half of B's rows, so a CTA reads 32 KB instead of 48 KB for the same
// 128 x 256 x 64 products.
//
// Persistent CTAs (or pairs); warp 0 loads 64-wide steps of r by TMA into a
// ring of 128-byte-swizzled stages, warp 1 issues the MMAs, warps 4-7 bring
// the finished accumulator out of tensor memory while the next tile is summed
// into the other one.  Either operand may be contiguous along r (K-major) or
// along p / q (MN-major): only the TMA box and the descriptors differ, so
// forward, dx and dw read their operands where they lie.
//
// Ragged groups: q tiles never span groups (a prefix table in shared memory
// maps tiles to groups); for dw a group's rows are the summed dimension, and
// rows of the next group that a box brings along are zeroed in shared memory
// before the MMA reads them (0 * NaN would not do).
//
// Every wait is bounded; on expiry the CTA raises its abort flag and the
// call's status word, drains its copies and MMAs, frees tensor memory and
// returns.
#include <cuda.h>

#include "linear.cuh"
#include "ptx.cuh"

namespace spmm {
namespace {

constexpr int kR = 64;              // r per stage: 128 bytes
constexpr int kP = 128;             // p per CTA
constexpr int kChunk = kR * 128;    // bytes of 64 rows of 128 bytes
constexpr int kThreads = 256;
constexpr int kBand = 8;            // q tiles that one sweep over p covers

struct Maps {
    CUtensorMap a, b;
};

struct TcArgs {
    Product p;
    int32_t a_kmajor, b_kmajor, a_grouped;   // a_grouped: the group is A's third coordinate
    int32_t bf16, clear_status, expire_probe;
};

template <int CG, int BQ>
struct Shape {
    static constexpr int kBRows = BQ / CG;                    // B rows of one CTA
    static constexpr int kStageBytes = kP * 128 + kBRows * 128;
    static constexpr int kStages = CG == 2 ? 6 : BQ == 256 ? 4 : BQ == 128 ? 6 : 8;
    static constexpr int kBoxQ = kBRows < 64 ? kBRows : 64;   // rows of a K-major B box
    static constexpr int kTmem = 2 * BQ;
    static constexpr int kTable = 2 * (SPMM_MAX_GROUPS + 2) * 4;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kTable + 512;
    static_assert(BQ % 64 == 0 && kTmem >= 32 && kTmem <= 512, "accumulators");
    static_assert(kSmem <= 227 * 1024, "shared memory per CTA");
};

struct Tile {
    int64_t group, p0, q0, r0;
    int nq, steps;       // columns; steps of kR
    int last;            // rows of r in the last step when it is ragged, else 0
    bool zero;           // rows behind the last group: written as zeros
};

struct Bars {
    uint64_t full[8], empty[8], acc_full[2], acc_empty[2], drain, never;
    uint32_t tmem;
    volatile int abort;
};

// ---- PTX ------------------------------------------------------------------------

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t map_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z,
                                         uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
            "[%1, {%2, %3, %4}], [%5];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
            "[%1, {%2, %3, %4}], [%5];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
}
// The same on this CTA's barrier alone.
template <int CG>
__device__ __forceinline__ void commit_local(uint64_t *bar) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                         smem_u32(bar))
                     : "memory");
    else
        mma_commit(bar);
}
// Arrives on `bar` (of both CTAs of a pair) when the MMAs issued before are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t *bar) {
    if constexpr (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
    else
        mma_commit(bar);
}
template <int CG>
__device__ __forceinline__ void alloc_tmem(uint32_t *dst, uint32_t cols) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)),
                     "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tmem_alloc(dst, cols);
    }
}
template <int CG>
__device__ __forceinline__ void free_tmem(uint32_t addr, uint32_t cols) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
    else
        tmem_dealloc(addr, cols);
}
// 32 consecutive tensor-memory columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(t));
}

// Bounded wait for the phase of `bar` with the given parity; false on abort or expiry.
__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, Bars &s, const TcArgs &a) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (s.abort) return false;
        if (clock64() - t0 > a.p.wait_cycles) {
            s.abort = 1;
            if (a.p.status) atomicCAS(a.p.status, 0, (int)SPMM_ETIMEOUT);
            return false;
        }
    }
}
// The same without the abort flag: for copies and MMAs already in flight.
__device__ __forceinline__ bool drain_bar(uint64_t *bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (clock64() - t0 > (1ll << 32)) return false;
    return true;
}

// Shared-memory matrix descriptor, 128-byte swizzle.  K-major: 8-row atoms of 1024 bytes, stride byte offset
// 1024.  MN-major: 64 values of p / q a row; 8 rows of r are 1024 bytes (stride), 64 more p / q a chunk (leading).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, bool kmajor) {
    const uint64_t lead = kmajor ? 1 : kChunk >> 4;
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (lead << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}

// ---- tiles ------------------------------------------------------------------------

// first[g]: first row of group g (g <= groups + 1: the tail, the end); qtiles[g]: q tiles before group g.
struct Table {
    int32_t *first, *qtiles;
};

template <int BQ>
__device__ __forceinline__ void fill_table(const Product &p, Table t) {
    if (!p.offsets) return;
    const int64_t total = p.red ? p.R : p.Q;
    const int G = (int)p.groups;
    for (int g = threadIdx.x; g <= G; g += blockDim.x) t.first[g] = (int32_t)group_first(p.offsets, g, total);
    if (threadIdx.x == 0) t.first[G + 1] = (int32_t)total;
    __syncthreads();
    if (p.red || threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    int before = 0;
    for (int g0 = 0; g0 <= G; g0 += 32) {
        const int g = g0 + lane;
        int tiles = 0;
        if (g <= G) {
            const int64_t n = (int64_t)t.first[g + 1] - t.first[g];
            tiles = n > 0 ? (int)((n + BQ - 1) / BQ) : 0;
        }
        const int incl = [&] {
            int v = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(kFullMask, v, o);
                if (lane >= o) v += y;
            }
            return v;
        }();
        if (g <= G) t.qtiles[g] = before + incl - tiles;
        before += __shfl_sync(kFullMask, incl, 31);
    }
    if (lane == 0) t.qtiles[G + 1] = before;
}

// (p tile, q tile) number i of np x nq: bands of kBand q tiles, within a band every p in turn, q fastest.
__device__ __forceinline__ void raster(int64_t i, int64_t np, int64_t nq, int64_t &pt, int64_t &qt) {
    const int64_t band = i / (np * kBand), rest = i - band * np * kBand;
    const int64_t width = nq - band * kBand < kBand ? nq - band * kBand : kBand;
    pt = rest / width;
    qt = band * kBand + rest - pt * width;
}

// Tile number i; false behind the last one.
template <int CG, int BQ>
__device__ __forceinline__ bool get_tile(const Product &p, Table t, int64_t i, Tile &o) {
    const int64_t np = (p.P + kP * CG - 1) / (kP * CG);
    int64_t pt, qt;
    o.zero = false;
    o.r0 = 0;
    o.last = 0;
    int64_t len = p.R;
    if (p.red) {
        const int64_t nq = (p.Q + BQ - 1) / BQ, per = np * nq;
        o.group = i / per;
        if (o.group >= p.groups) return false;
        raster(i - o.group * per, np, nq, pt, qt);
        o.q0 = qt * BQ;
        o.nq = (int)(p.Q - o.q0 < BQ ? p.Q - o.q0 : BQ);
        if (p.offsets) {
            o.r0 = t.first[o.group];
            len = t.first[o.group + 1] - o.r0;
            if (len < 0) len = 0;
            o.last = (int)(len & (kR - 1));
        }
    } else if (p.offsets) {
        const int G = (int)p.groups;
        const int64_t nq = t.qtiles[G + 1];
        if (i >= np * nq) return false;
        raster(i, np, nq, pt, qt);
        int lo = 0, hi = G;          // the last group with qtiles[g] <= qt
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (t.qtiles[mid] <= qt) lo = mid; else hi = mid - 1;
        }
        o.group = lo;
        o.q0 = t.first[lo] + (qt - t.qtiles[lo]) * BQ;
        const int64_t left = t.first[lo + 1] - o.q0;
        o.nq = (int)(left < BQ ? left : BQ);
        if (lo == G) {
            o.zero = true;
            len = 0;
        }
    } else {
        const int64_t nq = (p.Q + BQ - 1) / BQ;
        if (i >= np * nq) return false;
        raster(i, np, nq, pt, qt);
        o.group = 0;
        o.q0 = qt * BQ;
        o.nq = (int)(p.Q - o.q0 < BQ ? p.Q - o.q0 : BQ);
    }
    o.p0 = pt * kP * CG;
    o.steps = (int)((len + kR - 1) / kR);
    return true;
}

// MMA columns of a tile: a multiple of 16 (of 32 for a pair, half from each CTA).
template <int CG>
__device__ __forceinline__ int mma_cols(int nq) {
    return CG == 2 ? (nq + 31) & ~31 : (nq + 15) & ~15;
}

// ---- epilogue -----------------------------------------------------------------------

template <typename T, typename O, int ACT>
__device__ __forceinline__ void store_columns(const Product &p, const Tile &t, int64_t pp, float bias,
                                              const uint32_t (&v)[32], int c0) {
    const int n = t.nq - c0 < 32 ? t.nq - c0 : 32;
    const int64_t q = t.q0 + c0;
    O *out = (O *)p.C + (p.red ? t.group * p.c_g : 0) + q * p.c_q + pp;
    const T *res = p.residual ? (const T *)p.residual + q * p.residual_ld + pp : nullptr;
    int16_t *slope = p.slope ? p.slope + q * p.P + pp : nullptr;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        if (j >= n) break;
        ActValue a = activate<ACT>(__uint_as_float(v[j]) + bias);
        if (res) a.y += to_f32(res[j * p.residual_ld]);
        if (t.zero) a.y = a.slope = 0.f;
        out[j * p.c_q] = from_f32<O>(a.y);
        if (slope) slope[j * p.P] = slope_code(a.slope);
    }
}

template <typename T, typename O>
__device__ __forceinline__ void epilogue(const Product &p, const Tile &t, int64_t pp, uint32_t tmem, bool have) {
    float bias = 0.f;
    const bool in = pp < p.P;
    if (in && p.bias && !t.zero) bias = to_f32(((const T *)p.bias)[t.group * p.bias_g + pp]);
    for (int c0 = 0; c0 < t.nq; c0 += 32) {
        uint32_t v[32];
        if (have) {
            __syncwarp();
            tmem_ld32(tmem + c0, v);
            tmem_wait_ld();
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0u;
        }
        if (in) switch (p.act) {
            case SPMM_ACT_NONE: store_columns<T, O, SPMM_ACT_NONE>(p, t, pp, bias, v, c0); break;
            case SPMM_ACT_RELU: store_columns<T, O, SPMM_ACT_RELU>(p, t, pp, bias, v, c0); break;
            case SPMM_ACT_GELU: store_columns<T, O, SPMM_ACT_GELU>(p, t, pp, bias, v, c0); break;
            case SPMM_ACT_GELU_TANH: store_columns<T, O, SPMM_ACT_GELU_TANH>(p, t, pp, bias, v, c0); break;
            default: store_columns<T, O, SPMM_ACT_SILU>(p, t, pp, bias, v, c0); break;
        }
    }
}

// ---- the kernel -----------------------------------------------------------------------

template <int CG, int BQ, typename T, typename O>
__global__ void __launch_bounds__(kThreads, 1) tc_kernel(const __grid_constant__ Maps maps,
                                                         const __grid_constant__ TcArgs a) {
    using Sh = Shape<CG, BQ>;
    extern __shared__ uint8_t raw[];
    uint8_t *ring = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    Table table;
    table.first = (int32_t *)(ring + Sh::kStages * Sh::kStageBytes);
    table.qtiles = table.first + SPMM_MAX_GROUPS + 2;
    Bars &s = *(Bars *)((uint8_t *)table.first + Sh::kTable);
    const Product &p = a.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const int64_t first_tile = blockIdx.x / CG, tile_step = gridDim.x / CG;

    if (threadIdx.x == 0) {
        for (int i = 0; i < Sh::kStages; ++i) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.acc_full[i], 1);
            mbar_init(&s.acc_empty[i], 4 * CG);
        }
        mbar_init(&s.drain, 1);
        mbar_init(&s.never, 1);
        s.abort = 0;
        fence_mbar_init();
        if (a.clear_status && blockIdx.x == 0 && p.status) *p.status = 0;
    }
    if (warp == 2) alloc_tmem<CG>(&s.tmem, Sh::kTmem);
    fill_table<BQ>(p, table);
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    Tile t;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t n = 0;      // steps issued
            bool ok = true;
            if (a.expire_probe) ok = wait_bar(&s.never, 0u, s, a);
            for (int64_t i = first_tile; ok && get_tile<CG, BQ>(p, table, i, t); i += tile_step) {
                const int cols = mma_cols<CG>(t.nq), mine = cols / CG;    // B rows of this CTA
                const int boxes = (mine + (a.b_kmajor ? Sh::kBoxQ : 64) - 1) / (a.b_kmajor ? Sh::kBoxQ : 64);
                const uint32_t bytes = kP * 128 + boxes * (a.b_kmajor ? Sh::kBoxQ * 128 : kChunk);
                const int32_t pa = (int32_t)(t.p0 + rank * kP), qb = (int32_t)(t.q0 + rank * mine);
                const int32_t g = a.a_grouped ? (int32_t)t.group : 0;
                for (int k = 0; k < t.steps; ++k, ++n) {
                    const uint32_t st = n % Sh::kStages, ph = (n / Sh::kStages) & 1;
                    if (!wait_bar(&s.empty[st], ph ^ 1, s, a)) {
                        ok = false;
                        break;
                    }
                    uint32_t bar = smem_u32(&s.full[st]);
                    if (rank == 0) mbar_arrive_expect_tx(&s.full[st], bytes * CG);
                    if constexpr (CG == 2) bar = map_cta(bar, 0);
                    const uint32_t dst = smem_u32(ring + st * Sh::kStageBytes);
                    const int32_t r = (int32_t)(t.r0 + (int64_t)k * kR);
                    if (a.a_kmajor) {
                        tma_load<CG>(dst, &maps.a, r, pa, g, bar);
                    } else {
                        tma_load<CG>(dst, &maps.a, pa, r, g, bar);
                        tma_load<CG>(dst + kChunk, &maps.a, pa + 64, r, g, bar);
                    }
                    for (int b = 0; b < boxes; ++b) {
                        const uint32_t d = dst + kP * 128;
                        if (a.b_kmajor) tma_load<CG>(d + b * Sh::kBoxQ * 128, &maps.b, r, qb + b * Sh::kBoxQ, 0, bar);
                        else tma_load<CG>(d + b * kChunk, &maps.b, qb + b * 64, r, 0, bar);
                    }
                }
            }
            if (ok) {               // every stage has been read: nothing arrives here after the CTA has left
                for (uint32_t m = n > Sh::kStages ? n - Sh::kStages : 0; m < n; ++m)
                    if (!wait_bar(&s.empty[m % Sh::kStages], (m / Sh::kStages) & 1, s, a)) {
                        ok = false;
                        break;
                    }
            }
            if (!ok && rank == 0)   // copies in flight land before the CTA leaves
                for (uint32_t m = n > Sh::kStages ? n - Sh::kStages : 0; m < n; ++m)
                    if (!drain_bar(&s.full[m % Sh::kStages], (m / Sh::kStages) & 1)) break;
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        uint32_t n = 0, acc = 0;   // steps, accumulators used
        bool ok = true, issued = false;
        const uint32_t idesc0 = (1u << 4) | ((uint32_t)a.bf16 << 7) | ((uint32_t)a.bf16 << 10) |
                                ((a.a_kmajor ? 0u : 1u) << 15) | ((a.b_kmajor ? 0u : 1u) << 16) |
                                ((uint32_t)(kP * CG >> 4) << 24);
        const uint32_t a_adv = (a.a_kmajor ? 32 : 2048) >> 4, b_adv = (a.b_kmajor ? 32 : 2048) >> 4;
        for (int64_t i = first_tile; ok && get_tile<CG, BQ>(p, table, i, t); i += tile_step) {
            if (t.steps == 0) continue;
            const uint32_t as = acc & 1, ap = (acc >> 1) & 1;
            ++acc;
            if (lane == 0) ok = wait_bar(&s.acc_empty[as], ap ^ 1, s, a);
            ok = __shfl_sync(kFullMask, ok, 0);
            if (!ok) break;
            tc_fence_after();
            const uint32_t idesc = idesc0 | ((uint32_t)(mma_cols<CG>(t.nq) >> 3) << 17);
            for (int k = 0; k < t.steps; ++k, ++n) {
                const uint32_t st = n % Sh::kStages, ph = (n / Sh::kStages) & 1;
                if (lane == 0) ok = wait_bar(&s.full[st], ph, s, a);
                ok = __shfl_sync(kFullMask, ok, 0);
                if (!ok) break;
                uint8_t *sa = ring + st * Sh::kStageBytes;
                int chunks = kR / 16;
                if (t.last && k == t.steps - 1) {   // rows behind the group: zeros up to the MMA's 16
                    chunks = (t.last + 15) / 16;
                    const int rows = chunks * 16 - t.last;
                    for (int c = 0; c < Sh::kStageBytes / kChunk; ++c)
                        for (int x = lane; x < rows * 8; x += 32)
                            *(uint4 *)(sa + c * kChunk + t.last * 128 + x * 16) = uint4{0, 0, 0, 0};
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                if (lane == 0) {
                    tc_fence_after();
                    const uint64_t da = smem_desc(smem_u32(sa), a.a_kmajor);
                    const uint64_t db = smem_desc(smem_u32(sa + kP * 128), a.b_kmajor);
                    for (int c = 0; c < chunks; ++c)
                        mma_f16<CG>(tmem + as * BQ, da + (uint64_t)(c * a_adv), db + (uint64_t)(c * b_adv), idesc,
                                    k > 0 || c > 0);
                    commit<CG>(&s.empty[st]);
                    if (k == t.steps - 1) commit<CG>(&s.acc_full[as]);
                }
                issued = true;
                __syncwarp();
            }
        }
        if (!ok && issued && lane == 0) {   // MMAs in flight end before tensor memory is freed
            commit_local<CG>(&s.drain);
            drain_bar(&s.drain, 0);
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int quad = warp & 3;
        uint32_t acc = 0;
        for (int64_t i = first_tile; get_tile<CG, BQ>(p, table, i, t); i += tile_step) {
            const bool have = t.steps > 0;
            uint32_t at = tmem + ((uint32_t)(quad * 32) << 16);
            uint32_t as = 0;
            if (have) {
                as = acc & 1;
                const uint32_t ap = (acc >> 1) & 1;
                ++acc;
                at += as * BQ;
                int ok = 1;
                if (lane == 0) ok = wait_bar(&s.acc_full[as], ap, s, a);
                if (!__shfl_sync(kFullMask, ok, 0)) break;
                tc_fence_after();
            }
            epilogue<T, O>(p, t, t.p0 + rank * kP + quad * 32 + lane, at, have);
            if (have) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CG == 2) arrive_cluster(map_cta(smem_u32(&s.acc_empty[as]), 0));
                    else mbar_arrive(&s.acc_empty[as]);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tc_fence_after();
    if (warp == 2) free_tmem<CG>(tmem, Sh::kTmem);
}

// ---- host ---------------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
    static EncodeFn fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) !=
                cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (EncodeFn)f;
    }();
    return fn;
}

// inner x outer x depth 16-bit values, `outer_ld` and `depth_ld` values apart; boxes of 64 x rows.
int encode(CUtensorMap *m, const void *ptr, bool bf16, int64_t inner, int64_t outer, int64_t depth, int64_t outer_ld,
           int64_t depth_ld, int rows) {
    const EncodeFn fn = encoder();
    if (!fn) return SPMM_ECUDA;
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)depth};
    const cuuint64_t strides[2] = {(cuuint64_t)outer_ld * 2, (cuuint64_t)depth_ld * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)rows, 1}, es[3] = {1, 1, 1};
    const CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                          const_cast<void *>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? SPMM_OK : SPMM_EALIGN;
}

template <int CG, int BQ, typename T, typename O>
int launch(const Product &p, bool clear, bool probe, cudaStream_t s) {
    using Sh = Shape<CG, BQ>;
    Maps maps{};
    TcArgs a{};
    a.p = p;
    a.a_kmajor = p.a_r == 1;
    a.b_kmajor = p.b_r == 1;
    a.bf16 = !p.f16;
    a.clear_status = clear;
    a.expire_probe = probe;
    if (p.R > 0) {
        const bool grouped = !p.red && p.groups > 1 && p.a_g != 0;
        a.a_grouped = grouped;
        const int64_t depth = grouped ? p.groups : 1, a_ld = a.a_kmajor ? p.a_p : p.a_r;
        const int64_t b_ld = a.b_kmajor ? p.b_q : p.b_r;
        SPMM_TRY(encode(&maps.a, p.A, a.bf16, a.a_kmajor ? p.R : p.P, a.a_kmajor ? p.P : p.R, depth, a_ld,
                        grouped ? p.a_g : a_ld, a.a_kmajor ? kP : 64));
        SPMM_TRY(encode(&maps.b, p.B, a.bf16, a.b_kmajor ? p.R : p.Q, a.b_kmajor ? p.Q : p.R, 1, b_ld, b_ld,
                        a.b_kmajor ? Sh::kBoxQ : 64));
    }
    const int64_t np = ceil_div(p.P, kP * CG);
    int64_t tiles = np * (p.red ? p.groups * ceil_div(p.Q, BQ) : ceil_div(p.Q, BQ) + (p.offsets ? p.groups : 0));
    int dev = 0, sms = 0;
    SPMM_CUDA_TRY(cudaGetDevice(&dev));
    SPMM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    if (tiles > sms / CG) tiles = sms / CG;
    auto kernel = tc_kernel<CG, BQ, T, O>;
    SPMM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(tiles * CG));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Sh::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CG;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CG == 2 ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kernel, maps, a) != cudaSuccess) {
        (void)cudaGetLastError();
        return SPMM_ECUDA;
    }
    note_product_launch();
    return SPMM_OK;
}

template <typename T, typename O>
int by_shape(const Product &p, bool clear, bool probe, cudaStream_t s) {
    const int64_t per = p.red ? p.Q : ceil_div(p.Q, p.groups);
    if (per <= 64) return launch<1, 64, T, O>(p, clear, probe, s);
    if (p.red) return launch<1, 256, T, O>(p, clear, probe, s);
    return launch<2, 256, T, O>(p, clear, probe, s);
}

}  // namespace

int launch_product(const Product &p, bool clear, bool probe, cudaStream_t s) {
    if (p.P == 0 || p.Q == 0 || (p.red && p.groups == 0)) return SPMM_OK;
    if (p.f16) return p.out_f32 ? by_shape<__half, float>(p, clear, probe, s)
                                : by_shape<__half, __half>(p, clear, probe, s);
    return p.out_f32 ? by_shape<__nv_bfloat16, float>(p, clear, probe, s)
                     : by_shape<__nv_bfloat16, __nv_bfloat16>(p, clear, probe, s);
}

}  // namespace spmm
