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
// ring of 128-byte-swizzled stages, warp 1 issues the MMAs, warps 4-11 bring
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
// What bounds it: the MMAs (the tensor pipe is active 80 % of the time at 4096 x
// 8192 x 2048 with silu), and over seconds the card's power limit: 8192 x 16384
// x 4096 bf16 811 us alone and 814 us sustained (1,350 TFLOP/s, 96 % of the
// library product measured beside it), 4096 x 8192 x 2048 111 us (1,236).
//
// Every wait is bounded; on expiry the CTA raises its abort flag and the
// call's status word, drains its copies and MMAs, frees tensor memory and
// returns.
#include <cuda.h>

#include <atomic>

#include "linear.cuh"
#include "ptx.cuh"

namespace spmm {
namespace {

constexpr int kR = 64;              // r per stage: 128 bytes
constexpr int kP = 128;             // p per CTA
constexpr int kChunk = kR * 128;    // bytes of 64 rows of 128 bytes
constexpr int kThreads = 384;       // 4 warps of roles, 8 of the epilogue
constexpr int kEpiWarps = 8;
// q tiles that one sweep over p covers: sixteen of one group's rows (8192 x 16384 x 4096: 811 us, with 8 833 us, as
// the weights pass through L2 half as often), eight of ragged groups, whose weights change every few q tiles anyway
// (4096 x 4096 x 4096 in 8 groups: 303 us, with 16 308 us).
constexpr int kBandOne = 16, kBandGroups = 8;

struct Maps {
    CUtensorMap a, b;
};

struct TcArgs {
    Product p;
    int32_t a_kmajor, b_kmajor, a_grouped;   // a_grouped: the group is A's third coordinate
    int32_t bf16, clear_status, expire_probe, splits;
    int32_t vec_out, vec_slope, vec_residual;   // 16-byte aligned rows
    int64_t part_stride;                        // between the partial results of one group's split sum
};

template <int CG, int BQ>
struct Shape {
    static constexpr int kBRows = BQ / CG;                    // B rows of one CTA
    static constexpr int kStageBytes = kP * 128 + kBRows * 128;
    static constexpr int kStages = CG == 2 || BQ == 128 ? 6 : 8;
    // Rows of a K-major B box.  Few rows come in boxes of 16: one token then costs 2 KB a stage, not 8.
    static constexpr int kBoxQ = BQ == 64 ? 16 : CG == 2 ? 128 : 64;
    static constexpr int kTmem = 2 * BQ;
    static constexpr int kTable = 2 * (SPMM_MAX_GROUPS + 2) * 4;
    static constexpr int kRing = kStages * kStageBytes, kOut = kEpiWarps * 2048;
    static constexpr int kSmem = 1024 + kRing + kOut + kTable + 512;
    static_assert(BQ % 64 == 0 && kTmem <= 512, "accumulators");
    static_assert(kSmem <= 227 * 1024, "shared memory per CTA");
};

struct Tile {
    int64_t group, p0, q0, r0;
    int nq, steps;       // columns; steps of kR
    int part;            // of the sum over r (TcArgs::splits)
    int last;            // rows of r in the last step when it is ragged, else 0
    bool zero;           // rows behind the last group: written as zeros
};

struct Bars {
    uint64_t full[8], empty[8], acc_full[2], acc_empty[2], drain, never;
    // Pairs, for a ragged last step in a stage: this CTA's copies have landed; the second CTA has zeroed its
    // rows.  One per stage, as several short groups' last steps can be in the ring at once.
    uint64_t tail[8], peer[8];
    uint32_t tmem;
    volatile int abort;
};

// ---- PTX ------------------------------------------------------------------------

// One lane of a converged warp.  The compiler keeps operands of the issuing
// instructions in uniform registers only behind an election: with `lane == 0`
// four MMAs and a commit took 680 cycles to issue instead of under 100.
__device__ __forceinline__ bool elect() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
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
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive_local(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
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
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                     : "memory");
}
// Arrives on `bar` (of both CTAs of a pair) when the MMAs issued before are done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar, uint16_t mask) {
    if constexpr (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"(mask)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                     : "memory");
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

__device__ __forceinline__ bool poll(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// One poll during which the thread may sleep in the hardware until the phase completes (2 us at most): eight
// epilogue warps wait for most of a tile's time, and polling costs power that the tensor cores could use.
__device__ __forceinline__ bool poll_asleep(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(2000u)
        : "memory");
    return ok != 0;
}
// The rest of a wait that did not end at once; false on abort or expiry.
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int *abort, int32_t *status,
                                     long long cycles) {
    const long long t0 = clock64();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 16; ++i)
            if (poll_asleep(bar, parity)) return true;
        if (*abort) return false;
        if (clock64() - t0 > cycles) {
            *abort = 1;
            if (status) atomicCAS(status, 0, (int)SPMM_ETIMEOUT);
            return false;
        }
    }
}
// Bounded wait of a converged warp for the phase of `bar` (shared address) with the given parity: one answer for
// all lanes, so that they stay converged; false on abort or expiry.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, Bars &s, const TcArgs &a) {
    if (__all_sync(kFullMask, poll(bar, parity))) return true;
    return __all_sync(kFullMask, wait_on(bar, parity, &s.abort, a.p.status, a.p.wait_cycles));
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

// Where the offsets decrease, their running maximum stands in for them: groups that overlapped could have more
// tiles together than 32 bits hold, and two of them would write the same rows.
template <int BQ>
__device__ __forceinline__ void fill_table(const Product &p, Table t) {
    if (!p.offsets) return;
    const int64_t total = p.red ? p.R : p.Q;
    const int G = (int)p.groups;
    bool falls = false;
    for (int g = threadIdx.x; g <= G; g += blockDim.x) {
        const int64_t a = group_first(p.offsets, g, total);
        falls |= g < G && group_first(p.offsets, g + 1, total) < a;
        t.first[g] = (int32_t)a;
    }
    if (threadIdx.x == 0) t.first[G + 1] = (int32_t)total;
    if (__syncthreads_or(falls)) {
        if (threadIdx.x == 0)
            for (int g = 1; g <= G; ++g) t.first[g] = t.first[g] > t.first[g - 1] ? t.first[g] : t.first[g - 1];
        __syncthreads();
    }
    if (p.red || threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    int before = 0;
    for (int g0 = 0; g0 <= G; g0 += 32) {
        const int g = g0 + lane;
        int tiles = 0;
        if (g <= G) {
            const int64_t n = (int64_t)t.first[g + 1] - t.first[g];
            tiles = (int)((n + BQ - 1) / BQ);
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

// (p tile, q tile) number i of np x nq: bands of `wide` q tiles, within a band every p in turn, q fastest.
__device__ __forceinline__ void raster(uint32_t i, uint32_t np, uint32_t nq, uint32_t wide, uint32_t &pt,
                                       uint32_t &qt) {
    const uint32_t band = i / (np * wide), rest = i - band * np * wide;
    const uint32_t left = nq - band * wide, width = left < wide ? left : wide;
    pt = rest / width;
    qt = band * wide + rest - pt * width;
}

// Tile number i; false behind the last one.  32-bit numbers (the host checks): every role asks for every tile,
// and three 64-bit divisions each time showed between tiles.
template <int CG, int BQ>
__device__ __forceinline__ bool get_tile(const TcArgs &a, Table t, uint32_t i, Tile &o) {
    const Product &p = a.p;
    const uint32_t P = (uint32_t)p.P, Q = (uint32_t)p.Q;
    const uint32_t np = (P + kP * CG - 1) / (kP * CG);
    uint32_t pt, qt;
    o.zero = false;
    o.r0 = 0;
    o.last = 0;
    o.part = 0;
    int32_t len = (int32_t)p.R;
    if (p.red && p.offsets) {
        const uint32_t nq = (Q + BQ - 1) / BQ, per = np * nq, g = i / per;
        if (g >= (uint32_t)p.groups) return false;
        o.group = g;
        raster(i - g * per, np, nq, kBandGroups, pt, qt);
        o.q0 = qt * BQ;
        o.nq = (int)(Q - qt * BQ < BQ ? Q - qt * BQ : BQ);
        o.r0 = t.first[g];
        len = t.first[g + 1] - t.first[g];
        o.last = len & (kR - 1);
    } else if (p.offsets) {
        const int G = (int)p.groups;
        const uint32_t nq = (uint32_t)t.qtiles[G + 1];
        if (i >= np * nq) return false;
        raster(i, np, nq, kBandGroups, pt, qt);
        int lo = 0, hi = G;          // the last group with qtiles[g] <= qt
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if ((uint32_t)t.qtiles[mid] <= qt) lo = mid; else hi = mid - 1;
        }
        o.group = lo;
        const int32_t q0 = t.first[lo] + (int32_t)(qt - t.qtiles[lo]) * BQ, left = t.first[lo + 1] - q0;
        o.q0 = q0;
        o.nq = left < BQ ? left : BQ;
        if (lo == G) {
            o.zero = true;
            len = 0;
        }
    } else {
        const uint32_t nq = (Q + BQ - 1) / BQ, all = np * nq;
        if (i >= all * a.splits) return false;
        o.part = a.splits > 1 ? (int)(i / all) : 0;
        raster(i - o.part * all, np, nq, kBandOne, pt, qt);
        o.group = 0;
        o.q0 = qt * BQ;
        o.nq = (int)(Q - qt * BQ < BQ ? Q - qt * BQ : BQ);
    }
    o.p0 = (int64_t)pt * (kP * CG);
    o.steps = (int)(((uint32_t)len + kR - 1) / kR);
    if (a.splits > 1) {
        const int lo = (int)((int64_t)o.steps * o.part / a.splits);
        o.steps = (int)((int64_t)o.steps * (o.part + 1) / a.splits) - lo;
        o.r0 = (int64_t)lo * kR;
    }
    return true;
}

// MMA columns of a tile: a multiple of 16 (of 32 for a pair, half from each CTA).
template <int CG>
__device__ __forceinline__ int mma_cols(int nq) {
    return CG == 2 ? (nq + 31) & ~31 : (nq + 15) & ~15;
}

// ---- epilogue -----------------------------------------------------------------------

// A warp's 32 x 32 piece of the result goes through 2 KB of shared memory, so
// that it leaves as runs of 64 contiguous bytes a row: 2-byte stores straight
// from the accumulator's layout (lane = p) cost 15 cycles each, 15,500 a 128 x
// 256 tile, as much as summing it over 2048.  16-bit values travel as words of
// two neighbouring columns, which halves the shared-memory accesses: the MMAs'
// operands and the copies already take nearly all of its bandwidth.
//
// put(j) gives this lane's value of column j; the values of columns [0, n) are
// stored at base + j * ld (lane 0's first).  `cols`: valid p from lane 0's on.
template <typename O, typename F>
__device__ __forceinline__ void store_piece(uint8_t *stage, O *base, int64_t ld, bool vec, int cols, int n, F put) {
    const int lane = threadIdx.x & 31, row = lane >> 3, at = (lane & 7) * 4;   // a lane moves 4 p
    if constexpr (sizeof(O) == 2) {
        uint32_t *word = (uint32_t *)stage;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 16; ++j) word[j * 32 + lane] = put(2 * j);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = i * 4 + row;
            const uint4 w = *(const uint4 *)(word + j * 32 + at);
            const uint2 even{__byte_perm(w.x, w.y, 0x5410), __byte_perm(w.z, w.w, 0x5410)};
            const uint2 odd{__byte_perm(w.x, w.y, 0x7632), __byte_perm(w.z, w.w, 0x7632)};
            O *out = base + (int64_t)(2 * j) * ld + at;
            if (vec && at + 4 <= cols) {
                if (2 * j < n) *(uint2 *)out = even;
                if (2 * j + 1 < n) *(uint2 *)(out + ld) = odd;
            } else {             // unaligned results and the last, partial run
                O e[4], o[4];
                memcpy(e, &even, 8);
                memcpy(o, &odd, 8);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (2 * j < n && at + x < cols) out[x] = e[x];
                    if (2 * j + 1 < n && at + x < cols) out[ld + x] = o[x];
                }
            }
        }
    } else {
#pragma unroll
        for (int j0 = 0; j0 < 32; j0 += 16) {
            float *value = (float *)stage;
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) value[j * 32 + lane] = put(j0 + j);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = i * 4 + row;
                const float4 v = *(const float4 *)(value + j * 32 + at);
                O *out = base + (int64_t)(j0 + j) * ld + at;
                if (j0 + j >= n) continue;
                if (vec && at + 4 <= cols) {
                    *(float4 *)out = v;
                } else {
                    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if (at + x < cols) out[x] = e[x];
                }
            }
        }
    }
}

// The other way: r[j] = column j's value at this lane, from base + j * ld.
template <typename T>
__device__ __forceinline__ void load_piece(uint8_t *stage, const T *base, int64_t ld, bool vec, int cols, int n,
                                           float (&r)[32]) {
    const int lane = threadIdx.x & 31, row = lane >> 3, at = (lane & 7) * 4;
    uint32_t *word = (uint32_t *)stage;
    uint2 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int j = (i >> 1) * 8 + row * 2 + (i & 1);
        const T *src = base + (int64_t)j * ld + at;
        v[i] = uint2{0, 0};
        if (vec && at + 4 <= cols) {
            if (j < n) v[i] = __ldg((const uint2 *)src);
        } else {
            T e[4] = {};
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (j < n && at + x < cols) e[x] = src[x];
            memcpy(&v[i], e, 8);
        }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint2 a = v[2 * i], b = v[2 * i + 1];
        *(uint4 *)(word + (i * 4 + row) * 32 + at) =
            uint4{__byte_perm(a.x, b.x, 0x5410), __byte_perm(a.x, b.x, 0x7632), __byte_perm(a.y, b.y, 0x5410),
                  __byte_perm(a.y, b.y, 0x7632)};
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const uint32_t w = word[j * 32 + lane];
        T e[2];
        memcpy(e, &w, 4);
        r[2 * j] = to_f32(e[0]);
        r[2 * j + 1] = to_f32(e[1]);
    }
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    uint32_t w;
    memcpy(&w, &v, 4);
    return w;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    uint32_t w;
    memcpy(&w, &v, 4);
    return w;
}

// Columns [c0, c0 + n) of a tile, n <= 32, for the warp whose first p is p0: v[j] is column c0 + j at this lane.
template <typename T, typename O, int ACT, bool SLOPE>
__device__ __forceinline__ void store_columns(const TcArgs &a, const Tile &t, uint8_t *stage, int64_t p0, float bias,
                                              const float (&v)[32], int c0, int n) {
    const Product &p = a.p;
    const int64_t q = t.q0 + c0;
    const int cols = p.P - p0 < 32 ? (int)(p.P - p0) : 32;
    float y[32], d[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = activate<ACT, SLOPE>(v[j] + bias, d[j]);
    if (p.residual) {
        float r[32];
        load_piece<T>(stage, (const T *)p.residual + q * p.residual_ld + p0, p.residual_ld, a.vec_residual, cols, n, r);
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j] += r[j];
    }
    store_piece<O>(stage, (O *)p.C + (p.red ? t.group * p.c_g : 0) + t.part * a.part_stride + q * p.c_q + p0, p.c_q, a.vec_out, cols, n,
                   [&](int j) {
                       if constexpr (sizeof(O) == 2) return pack2<O>(y[j], y[j + 1]);
                       else return y[j];
                   });
    if constexpr (SLOPE)
        store_piece<uint16_t>(stage, (uint16_t *)p.slope + q * p.P + p0, p.P, a.vec_slope, cols, n,
                              [&](int j) { return (uint32_t)slope_code(d[j]) | (uint32_t)slope_code(d[j + 1]) << 16; });
}

template <typename T, typename O, int ACT>
__device__ __forceinline__ void store_act(const TcArgs &a, const Tile &t, uint8_t *stage, int64_t p0, float bias,
                                          const float (&v)[32], int c0, int n) {
    if (a.p.slope) store_columns<T, O, ACT, true>(a, t, stage, p0, bias, v, c0, n);
    else store_columns<T, O, ACT, false>(a, t, stage, p0, bias, v, c0, n);
}

template <typename T, typename O>
__device__ __forceinline__ void finish_columns(const TcArgs &a, const Tile &t, uint8_t *stage, int64_t p0, float bias,
                                               const float (&v)[32], int c0, int end) {
    const Product &p = a.p;
    if (p0 >= p.P) return;
    const int n = end - c0 < 32 ? end - c0 : 32;
    if (t.zero) {
        const int64_t q = t.q0 + c0, pp = p0 + (threadIdx.x & 31);
        if (pp < p.P)
            for (int j = 0; j < n; ++j) {
                ((O *)p.C)[(q + j) * p.c_q + pp] = from_f32<O>(0.f);
                if (p.slope) p.slope[(q + j) * p.P + pp] = 0;
            }
        return;
    }
    if constexpr (sizeof(O) == 4) {     // the float32 result is a plain product
        store_columns<T, O, SPMM_ACT_NONE, false>(a, t, stage, p0, bias, v, c0, n);
    } else {
        switch (p.act) {
            case SPMM_ACT_NONE: store_act<T, O, SPMM_ACT_NONE>(a, t, stage, p0, bias, v, c0, n); break;
            case SPMM_ACT_RELU: store_act<T, O, SPMM_ACT_RELU>(a, t, stage, p0, bias, v, c0, n); break;
            case SPMM_ACT_GELU: store_act<T, O, SPMM_ACT_GELU>(a, t, stage, p0, bias, v, c0, n); break;
            case SPMM_ACT_GELU_TANH: store_act<T, O, SPMM_ACT_GELU_TANH>(a, t, stage, p0, bias, v, c0, n); break;
            default: store_act<T, O, SPMM_ACT_SILU>(a, t, stage, p0, bias, v, c0, n); break;
        }
    }
}

// 32 columns from c0 of the accumulator at `tmem` (zeros where nothing was summed).  The whole warp.
__device__ __forceinline__ void read_columns(uint32_t tmem, bool have, float (&v)[32]) {
    __syncwarp();
    uint32_t u[32];
    if (have) {
        tmem_ld32(tmem, u);
        tmem_wait_ld();
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) u[j] = 0u;
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(u[j]);
}

template <typename T>
__device__ __forceinline__ float load_bias(const Product &p, const Tile &t, int64_t pp) {
    return p.bias && !t.zero && pp < p.P ? to_f32(((const T *)p.bias)[t.group * p.bias_g + pp]) : 0.f;
}

// ---- the kernel -----------------------------------------------------------------------

// Zeros in rows [last, next multiple of 16) of a stage of 64-row chunks, visible to the MMAs.  A whole warp.
__device__ __forceinline__ void zero_rows(uint8_t *stage, int bytes, int last) {
    const int rows = ((last + 15) & ~15) - last;
    for (int c = 0; c < bytes; c += kChunk)
        for (int x = threadIdx.x & 31; x < rows * 8; x += 32)
            *(uint4 *)(stage + c + last * 128 + x * 16) = uint4{0, 0, 0, 0};
    fence_proxy_async_smem();
    __syncwarp();
}

// The producer: a step's boxes into the next stage of the ring.  Called by the
// whole warp, an elected lane issues.  What a tile fixes is worked out once a
// tile: with everything inside the step, issuing three copies took 350 cycles
// of the 512 that the MMAs of a pair's step take.
template <int CG, int BQ>
struct Loader {
    using Sh = Shape<CG, BQ>;
    const Maps &maps;
    const TcArgs &a;
    uint32_t full, full_lead, tail, ring;    // shared addresses; the barriers of the pair's first CTA
    uint32_t rank;
    uint32_t n, st, ph;      // steps issued; the next stage and its phase
    uint32_t tails, odd;     // pairs: bit st, whether stage st has held a ragged last step; an odd number of them
    int32_t pa, qb, g, r;    // the tile's coordinates
    uint32_t bytes;
    int boxes;

    __device__ __forceinline__ void open(const Tile &t) {
        const int mine = mma_cols<CG>(t.nq) / CG, box_rows = a.b_kmajor ? Sh::kBoxQ : 64;   // B rows of this CTA
        boxes = (mine + box_rows - 1) / box_rows;
        bytes = kP * 128 + boxes * box_rows * 128;
        pa = (int32_t)t.p0 + rank * kP;
        qb = (int32_t)t.q0 + rank * mine;
        g = a.a_grouped ? (int32_t)t.group : 0;
        r = (int32_t)t.r0;
    }
    // `ragged`: the last step of a tile whose group ends within it.
    __device__ __forceinline__ void step(bool ragged) {
        if (elect()) {
            uint32_t bar = full_lead + st * 8;
            if (CG == 2 && ragged) {         // each CTA has rows to zero first
                bar = tail + st * 8;
                expect(bar, bytes);
                if (rank == 0) arrive_local(full + st * 8);
            } else if (rank == 0) {
                expect(full + st * 8, bytes * CG);
            }
            const uint32_t dst = ring + st * Sh::kStageBytes, db = dst + kP * 128;
            if (a.a_kmajor) {
                tma_load<CG>(dst, &maps.a, r, pa, g, bar);
            } else {
                tma_load<CG>(dst, &maps.a, pa, r, g, bar);
                tma_load<CG>(dst + kChunk, &maps.a, pa + 64, r, g, bar);
            }
            if (a.b_kmajor) {
#pragma unroll
                for (int b = 0; b < Sh::kBRows / Sh::kBoxQ; ++b)
                    if (b < boxes) tma_load<CG>(db + b * Sh::kBoxQ * 128, &maps.b, r, qb + b * Sh::kBoxQ, 0, bar);
            } else {
#pragma unroll
                for (int b = 0; b < Sh::kBRows / 64; ++b)
                    if (b < boxes) tma_load<CG>(db + b * kChunk, &maps.b, qb + b * 64, r, 0, bar);
            }
        }
        __syncwarp();
        if (CG == 2 && ragged) {
            tails |= 1u << st;
            odd ^= 1u << st;
        }
        r += kR;
        ++n;
        if (++st == Sh::kStages) {
            st = 0;
            ph ^= 1;
        }
    }
};

template <int CG, int BQ, typename T, typename O>
__global__ void __launch_bounds__(kThreads, 1) tc_kernel(const __grid_constant__ Maps maps,
                                                         const __grid_constant__ TcArgs a) {
    using Sh = Shape<CG, BQ>;
    extern __shared__ uint8_t raw[];
    uint8_t *ring = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    Table table;
    uint8_t *stages = ring + Sh::kRing;      // the epilogue warps' 2 KB each
    table.first = (int32_t *)(stages + Sh::kOut);
    table.qtiles = table.first + SPMM_MAX_GROUPS + 2;
    Bars &s = *(Bars *)((uint8_t *)table.first + Sh::kTable);
    const Product &p = a.p;
    const int warp = __shfl_sync(kFullMask, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t crank = CG == 2 ? cluster_rank() : 0;
    const uint32_t rank = crank % CG, lead = crank - rank;     // within the pair; the pair's first CTA
    const uint32_t first_tile = blockIdx.x / CG, tile_step = gridDim.x / CG;

    if (threadIdx.x == 0) {
        if (p.R > 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.b) : "memory");
        }
        for (int i = 0; i < Sh::kStages; ++i) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
            mbar_init(&s.tail[i], 1);
            mbar_init(&s.peer[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.acc_full[i], 1);
            mbar_init(&s.acc_empty[i], kEpiWarps * CG);
        }
        mbar_init(&s.drain, 1);
        mbar_init(&s.never, 1);
        s.abort = 0;
        fence_mbar_init();
    }
    if (warp == 2) alloc_tmem<CG>(&s.tmem, Sh::kTmem);
    __syncwarp();
    chained_start();
    if (a.clear_status && threadIdx.x == 0 && blockIdx.x == 0 && p.status) *p.status = 0;
    const uint32_t full = smem_u32(s.full), empty = smem_u32(s.empty), tail = smem_u32(s.tail), peer = smem_u32(s.peer);
    const uint32_t acc_full = smem_u32(s.acc_full), acc_empty = smem_u32(s.acc_empty);
    Loader<CG, BQ> load{maps, a, full, CG == 2 ? map_cta(full, lead) : full, tail, smem_u32(ring), rank};
    Tile t;
    if (CG == 1 && warp == 0 && !p.offsets && !a.expire_probe) {   // fill the ring before anything else is ready
        __syncwarp();
        if (get_tile<CG, BQ>(a, table, first_tile, t)) {
            load.open(t);
            for (int k = 0; k < t.steps && k < Sh::kStages; ++k) load.step(false);
        }
    }
    fill_table<BQ>(p, table);
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s.tmem;

    if (warp == 0) {
        bool ok = true;
        if (a.expire_probe) ok = wait_warp(smem_u32(&s.never), 0u, s, a);
        int k = (int)load.n;
        for (uint32_t i = first_tile; ok && get_tile<CG, BQ>(a, table, i, t); i += tile_step, k = 0) {
            if (k == 0) load.open(t);
            for (; k < t.steps; ++k) {
                ok = wait_warp(empty + load.st * 8, load.ph ^ 1, s, a);
                if (!ok) break;
                load.step(t.last && k == t.steps - 1);
            }
        }
        const uint32_t n = load.n;
        if (ok) {               // every stage has been read: nothing arrives here after the CTA has left
            for (uint32_t m = n > Sh::kStages ? n - Sh::kStages : 0; m < n; ++m)
                if (!wait_warp(empty + m % Sh::kStages * 8, (m / Sh::kStages) & 1, s, a)) {
                    ok = false;
                    break;
                }
        }
        for (int i = 0; !ok && i < Sh::kStages; ++i)
            if (load.tails >> i & 1) drain_bar(&s.tail[i], load.odd >> i & 1 ^ 1);
        if (!ok && rank == 0)   // copies in flight land before the CTA leaves
            for (uint32_t m = n > Sh::kStages ? n - Sh::kStages : 0; m < n; ++m)
                if (!drain_bar(&s.full[m % Sh::kStages], (m / Sh::kStages) & 1)) break;
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        const uint16_t both = (uint16_t)(3u << lead);
        uint32_t acc = 0, st = 0, ph = 0, odd = 0;   // accumulators used; stage and its phase; see Loader
        bool ok = true;
        const uint32_t idesc0 = (1u << 4) | ((uint32_t)a.bf16 << 7) | ((uint32_t)a.bf16 << 10) |
                                ((a.a_kmajor ? 0u : 1u) << 15) | ((a.b_kmajor ? 0u : 1u) << 16) |
                                ((uint32_t)(kP * CG >> 4) << 24);
        const uint32_t a_adv = (a.a_kmajor ? 32 : 2048) >> 4, b_adv = (a.b_kmajor ? 32 : 2048) >> 4;
        // descriptors of the first stage; only their low words depend on the stage and on r
        const uint64_t da0 = smem_desc(smem_u32(ring), a.a_kmajor);
        const uint64_t db0 = smem_desc(smem_u32(ring) + kP * 128, a.b_kmajor);
        const uint32_t da_hi = (uint32_t)(da0 >> 32), db_hi = (uint32_t)(db0 >> 32);
        uint32_t da = (uint32_t)da0, db = (uint32_t)db0;
        auto mma = [&](uint32_t d, uint32_t idesc, int c, uint32_t accumulate) {
            mma_f16<CG>(d, (uint64_t)da_hi << 32 | (da + c * a_adv), (uint64_t)db_hi << 32 | (db + c * b_adv), idesc,
                        accumulate);
        };
        for (uint32_t i = first_tile; ok && get_tile<CG, BQ>(a, table, i, t); i += tile_step) {
            if (t.steps == 0) continue;
            const uint32_t as = acc & 1, ap = (acc >> 1) & 1;
            ++acc;
            ok = wait_warp(acc_empty + as * 8, ap ^ 1, s, a);
            if (!ok) break;
            tc_fence_after();
            const uint32_t idesc = idesc0 | ((uint32_t)(mma_cols<CG>(t.nq) >> 3) << 17), d = tmem + as * BQ;
            for (int k = 0; k < t.steps; ++k) {
                ok = wait_warp(full + st * 8, ph, s, a);
                if (!ok) break;
                const bool last = k == t.steps - 1;
                if (t.last && last) {           // rows behind the group: zeros up to the MMA's 16
                    if constexpr (CG == 2) ok = wait_warp(tail + st * 8, odd >> st & 1, s, a);
                    if (!ok) break;
                    zero_rows(ring + st * Sh::kStageBytes, Sh::kStageBytes, t.last);
                    if constexpr (CG == 2) {
                        ok = wait_warp(peer + st * 8, odd >> st & 1, s, a);
                        asm volatile("fence.acq_rel.cluster;" ::: "memory");
                    }
                    if (!ok) break;
                    odd ^= 1u << st;
                    tc_fence_after();
                    if (elect())
                        for (int c = 0; c < (t.last + 15) / 16; ++c) mma(d, idesc, c, k > 0 || c > 0);
                } else {
                    tc_fence_after();
                    if (elect()) {
                        mma(d, idesc, 0, k > 0);
#pragma unroll
                        for (int c = 1; c < kR / 16; ++c) mma(d, idesc, c, 1);
                    }
                }
                __syncwarp();
                if (elect()) {
                    commit<CG>(empty + st * 8, both);
                    if (last) commit<CG>(acc_full + as * 8, both);
                }
                __syncwarp();
                da += Sh::kStageBytes >> 4;
                db += Sh::kStageBytes >> 4;
                if (++st == Sh::kStages) {
                    st = 0;
                    ph ^= 1;
                    da = (uint32_t)da0;
                    db = (uint32_t)db0;
                }
            }
        }
        if (!ok && acc) {      // MMAs in flight end before tensor memory is freed
            if (elect()) commit_local<CG>(&s.drain);
            __syncwarp();
            drain_bar(&s.drain, 0);
        }
        __syncwarp();
    } else if (CG == 2 && warp == 1) {      // the pair's second CTA zeroes its rows of ragged last steps
        uint32_t n = 0, odd = 0;
        for (uint32_t i = first_tile; p.red && p.offsets && get_tile<CG, BQ>(a, table, i, t); i += tile_step) {
            n += t.steps;
            if (t.steps == 0 || t.last == 0) continue;
            const uint32_t st = (n - 1) % Sh::kStages;
            if (!wait_warp(tail + st * 8, odd >> st & 1, s, a)) break;
            odd ^= 1u << st;
            zero_rows(ring + st * Sh::kStageBytes, Sh::kStageBytes, t.last);
            if (lane == 0) arrive_cluster(map_cta(peer + st * 8, lead));
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int quad = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        uint8_t *stage = stages + (warp - 4) * 2048;
        uint32_t acc = 0;
        for (uint32_t i = first_tile; get_tile<CG, BQ>(a, table, i, t); i += tile_step) {
            const int64_t p0 = t.p0 + rank * kP + quad * 32;
            const bool have = t.steps > 0;
            const uint32_t as = acc & 1, at = lanes + as * BQ;
            const float bias = load_bias<T>(p, t, p0 + lane);
            if (have) {
                const uint32_t ap = (acc >> 1) & 1;
                ++acc;
                if (!wait_warp(acc_full + as * 8, ap, s, a)) break;
                tc_fence_after();
            }
            float v[32];
            for (int c0 = half * 32; c0 < t.nq; c0 += 64) {
                read_columns(at + c0, have, v);
                finish_columns<T, O>(a, t, stage, p0, bias, v, c0, t.nq);
            }
            if (have) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CG == 2) arrive_cluster(map_cta(smem_u32(&s.acc_empty[as]), lead));
                    else mbar_arrive(&s.acc_empty[as]);
                }
            }
        }
    }
    __syncwarp();
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

// Tile shape and splits by an estimate of the time in cycles: rounds of tiles
// over the SMs, each its steps at the shape's measured rate plus what a tile
// costs once; a split adds a second kernel that reads every part.
struct Choice {
    int cg, bq, splits;
};

Choice choose(const Product &p, int sms) {
    struct Cost {
        int cg, bq;
        int64_t step, tile;
    };
    // measured at 4096 x 4096 weights with 16 to 1024 rows: a step of a narrow tile costs nearly what a wide one
    // does (its weights come through the same 64 bytes a cycle from L2), but there are more tiles to share out
    static const Cost costs[] = {{2, 256, 540, 6000}, {1, 128, 500, 3500}, {1, 64, 460, 2500}};
    const int64_t steps = ceil_div(p.red && p.offsets ? ceil_div(p.R, p.groups) : p.R, kR);
    Choice best{2, 256, 1};
    int64_t least = INT64_MAX;
    for (const Cost &c : costs) {
        const int64_t np = ceil_div(p.P, kP * c.cg), slots = sms / c.cg;
        int64_t nq = ceil_div(p.Q, c.bq);
        if (p.red) {
            nq *= p.groups;
        } else if (p.offsets) {      // every group ends within a tile, half a tile early on average
            const int64_t per = p.Q / p.groups;
            nq = per < 1 ? p.Q : p.groups * ceil_div(per, c.bq) + (per > c.bq / 2 ? p.groups / 2 : 0);
        }
        const int64_t tiles = np * nq;
        for (int s = 1; s <= 16; s += s < 4 ? 1 : 4) {
            if (s > 1 && (p.offsets || p.out_f32 || steps < 4 * s || tiles * s > slots)) break;
            int64_t t = ceil_div(tiles * s, slots) * (ceil_div(steps, s) * c.step + c.tile);
            if (s > 1) t += 9000 + p.P * p.Q * s / 1000;    // a second launch, every part once more
            if (t < least) {
                least = t;
                best = Choice{c.cg, c.bq, s};
            }
        }
    }
    return best;
}

// Partial results of a split sum: C = finish(sum over parts, in order).  Eight p a thread.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Product p, const float *parts, int splits) {
    chained_start();
    constexpr int V = VEC ? 8 : 1;
    const int64_t per = p.P / V, items = p.Q * per;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const int64_t q = i / per, pp = (i - q * per) * V;
    float z[V] = {}, d[V];
    const float *src = parts + q * p.P + pp;
#pragma unroll 4
    for (int x = 0; x < splits; ++x, src += p.P * p.Q) {
        if constexpr (VEC) {
            const float4 a = __ldcg((const float4 *)src), b = __ldcg((const float4 *)src + 1);
            z[0] += a.x, z[1] += a.y, z[2] += a.z, z[3] += a.w, z[4] += b.x, z[5] += b.y, z[6] += b.z, z[7] += b.w;
        } else {
            z[0] += __ldcg(src);
        }
    }
    if (p.bias) {
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] += to_f32(((const T *)p.bias)[pp + e]);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = activate<ACT, true>(z[e], d[e]);
    if (p.residual) {
        const T *r = (const T *)p.residual + q * p.residual_ld + pp;
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] += to_f32(r[e]);
    }
    T *out = (T *)p.C + q * p.c_q + pp;
    if constexpr (VEC) *(uint4 *)out = pack8<T>(z);
    else out[0] = from_f32<T>(z[0]);
    if (p.slope) {
        uint16_t c[V];
#pragma unroll
        for (int e = 0; e < V; ++e) c[e] = slope_code(d[e]);
        if constexpr (VEC) memcpy(__builtin_assume_aligned(p.slope + q * p.P + pp, 16), c, 16);
        else p.slope[q * p.P + pp] = (int16_t)c[0];
    }
}

template <typename T>
int join(const Product &p, const float *parts, int splits, cudaStream_t s) {
    const bool vec = p.P % 8 == 0 && (uintptr_t)p.C % 16 == 0 && p.c_q % 8 == 0 && (uintptr_t)p.slope % 16 == 0;
    const unsigned grid = (unsigned)ceil_div(p.Q * (vec ? p.P / 8 : p.P), 256);
#define SPMM_JOIN(ACT)                                                                       \
    do {                                                                                     \
        SPMM_TRY(launch_chained(vec ? join_kernel<T, ACT, true> : join_kernel<T, ACT, false>, dim3(grid), 256, 0, s, \
                                1, p, parts, splits));                                       \
    } while (0)
    switch (p.act) {
        case SPMM_ACT_NONE: SPMM_JOIN(SPMM_ACT_NONE); break;
        case SPMM_ACT_RELU: SPMM_JOIN(SPMM_ACT_RELU); break;
        case SPMM_ACT_GELU: SPMM_JOIN(SPMM_ACT_GELU); break;
        case SPMM_ACT_GELU_TANH: SPMM_JOIN(SPMM_ACT_GELU_TANH); break;
        default: SPMM_JOIN(SPMM_ACT_SILU); break;
    }
#undef SPMM_JOIN
    return SPMM_OK;
}

struct How {
    bool clear, probe;
    int splits, dev, sms;
};

template <int CG, int BQ, typename T, typename O>
int launch(const Product &p, const How &how, cudaStream_t s) {
    using Sh = Shape<CG, BQ>;
    Maps maps{};
    TcArgs a{};
    a.p = p;
    a.a_kmajor = p.a_r == 1;
    a.b_kmajor = p.b_r == 1;
    a.bf16 = !p.f16;
    a.clear_status = how.clear;
    a.expire_probe = how.probe;
    a.splits = how.splits;
    a.part_stride = p.P * p.Q;
    const int64_t per16 = 16 / sizeof(O);
    a.vec_out = (uintptr_t)p.C % 16 == 0 && p.c_q % per16 == 0 && p.c_g % per16 == 0 &&
                (how.splits == 1 || a.part_stride % per16 == 0);
    a.vec_slope = (uintptr_t)p.slope % 16 == 0 && p.P % 8 == 0;
    a.vec_residual = (uintptr_t)p.residual % 16 == 0 && p.residual_ld % 8 == 0;
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
    tiles *= how.splits;
    if (tiles > INT32_MAX / 2) return SPMM_EUNSUPPORTED;
    if (tiles > how.sms / CG) tiles = how.sms / CG;
    auto kernel = tc_kernel<CG, BQ, T, O>;
    static std::atomic<uint64_t> ready{0};        // devices (below 64) on which the kernel may use its shared memory
    const uint64_t bit = how.dev < 64 ? 1ull << how.dev : 0;
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        SPMM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem));
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    return launch_chained(kernel, dim3((unsigned)(tiles * CG)), kThreads, Sh::kSmem, s, CG, maps, a);
}

template <typename T, typename O>
int by_shape(const Product &p, const Choice &c, const How &how, cudaStream_t s) {
    if (c.cg == 2) return launch<2, 256, T, O>(p, how, s);
    if (c.bq == 128) return launch<1, 128, T, O>(p, how, s);
    return launch<1, 64, T, O>(p, how, s);
}

template <typename T>
int run(const Product &p, const ProductPlan &plan, How how, cudaStream_t s) {
    const Choice c{plan.cg, plan.bq, plan.splits};
    if (c.splits == 1) return p.out_f32 ? by_shape<T, float>(p, c, how, s) : by_shape<T, T>(p, c, how, s);
    Product raw = p;          // plain float32 sums of each part
    raw.C = plan.parts;
    raw.c_q = p.P;
    raw.c_g = 0;
    raw.out_f32 = 1;
    raw.act = SPMM_ACT_NONE;
    raw.bias = raw.residual = nullptr;
    raw.slope = nullptr;
    SPMM_TRY((by_shape<T, float>(raw, c, how, s)));
    return join<T>(p, plan.parts, c.splits, s);
}

}  // namespace

int plan_product(const Product &p, bool probe, Arena &arena, ProductPlan &plan) {
    plan = ProductPlan{};
    if (p.P == 0 || p.Q == 0) return SPMM_OK;
    plan.launches = true;
    plan.skinny = !probe && skinny_fits(p);
    if (plan.skinny) return SPMM_OK;
    static std::atomic<int> known[64];        // SMs of a device
    SPMM_CUDA_TRY(cudaGetDevice(&plan.dev));
    plan.sms = plan.dev < 64 ? known[plan.dev].load(std::memory_order_relaxed) : 0;
    if (plan.sms == 0) {
        SPMM_CUDA_TRY(cudaDeviceGetAttribute(&plan.sms, cudaDevAttrMultiProcessorCount, plan.dev));
        if (plan.dev < 64) known[plan.dev].store(plan.sms, std::memory_order_relaxed);
    }
    const Choice c = choose(p, plan.sms);
    plan.cg = c.cg;
    plan.bq = c.bq;
    plan.splits = c.splits;
    if (c.splits > 1) plan.parts = arena.take<float>(p.P * p.Q * c.splits);
    return SPMM_OK;
}

int run_product(const Product &p, const ProductPlan &plan, bool clear, bool probe, cudaStream_t s) {
    if (!plan.launches) return SPMM_OK;
    if (plan.skinny) return launch_skinny(p, clear, s);
    const How how{clear, probe, plan.splits, plan.dev, plan.sms};
    return p.f16 ? run<__half>(p, plan, how, s) : run<__nv_bfloat16>(p, plan, how, s);
}

}  // namespace spmm
