// Tensor-core kernels of cross attention on packed clouds (tcgen05, sm_100a).
//
// Operands are bf16 tiles of `rows x 64 features` in shared memory (128-byte swizzle, one block per 64 features), brought in
// by TMA.  32-bit features come as three bf16 planes, x = h + m + l with h = bf16(x), m = bf16(x - h), l = bf16(x - h - m):
// 24 bits, and a product is the six plane products h h + h m + m h + m m + h l + l h in one fp32 accumulator (the dropped
// ones are below 2^-24 of it).  An infinity among a cloud's own 32-bit features becomes NaN this way.
//
// A streamed tile in which the cloud ends gets zeros behind the cloud's last row: the rows that follow belong to another cloud
// and may hold infinities, which would reach this one as 0 * inf.
//
// Roles of the eleven warps of a CTA: two groups of four warps do the element-wise work (one row of a 128-row tile per thread,
// which is one lane of tensor memory), warp 8 loads, and elected lanes of warps 9 and 10 issue the products, the logits and
// the weighted sums: each of the two waits for barriers of its own, and a wait costs as much as issuing a product (measured with one
// warp for both, 64-row units: 460 of the 1120 cycles of a unit).  The element-wise groups work on different units in turn, so
// one of them computes while the tensor cores run the products of the other.
// Every wait is bounded: a role whose wait runs out sets a flag that ends the other roles' waits, the CTA waits for its
// copies and products in flight, frees its tensor memory and records the failure in the pinned status word.
#pragma once

#include <cuda_bf16.h>

#include "attention.cuh"
#include "common.cuh"
#include "features.cuh"
#include "tc_ptx.cuh"

namespace pccnn {

constexpr int kTcThreads = 352;
constexpr int kTcRows = 128;  // rows of the tile whose products have them as the M dimension
constexpr int kTcMaxStages = 8;
constexpr int kTcRoundRows = 65536;  // streamed rows that a bf16 accumulator takes before it is emptied: 4096 sums of 16 rows, each truncated by at most 2^-23

// bf16 rows [planes][rows, heads, size] for the loads that TMA does not do.
struct TcRows {
    const __nv_bfloat16* data;
    int64_t row, head, plane;
};

struct TcControl {
    uint32_t poll_limit;
    int withhold_from;  // test hook: the loader stops in front of this streamed tile (-1: off)
    int* sticky;        // pinned status word
    int status;         // value to record: origin in the upper bits
};

struct TcShared {
    uint64_t fixed_full, full[kTcMaxStages], empty[kTcMaxStages], s_full[2], s_free[2], e_ready[2],
        e_done[2], all_done, drained[2], round_done, acc_free;
    uint32_t tmem;
    int failed;
};

// Bounded wait of a converged warp, with one answer for all its lanes; it also ends when another role of the CTA has failed.
// The phase has usually completed already, so the first poll is all that costs (a loop of single lanes took 350 cycles).
__device__ __forceinline__ bool tc_poll(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return __all_sync(kFullMask, done != 0);
}
__device__ __forceinline__ bool tc_wait_warp(uint64_t* bar, uint32_t parity, uint32_t limit, volatile int* failed) {
    const uint32_t addr = smem_u32(bar);
    if (tc_poll(addr, parity)) return true;
#pragma unroll 1
    for (uint32_t n = 1; n < limit; ++n) {
        if (tc_poll(addr, parity)) return true;
        if ((n & 255) == 0 && __any_sync(kFullMask, *failed)) return false;
    }
    return false;
}

// One arrival for a warp, behind the tensor-memory accesses of all its lanes.
__device__ __forceinline__ void tc_arrive_warp(uint64_t* bar) {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// What block `slot` of a grid with rows / ROWS + clouds + 1 blocks works on: rows [row0, row_end) of a cloud (its end, not the
// block's) and the cloud's streamed rows [begin, end).  Cloud b's blocks start at begin(b) / ROWS + b, which leaves room for
// all of them without a prefix sum.  Cloud `clouds` is the rest of the rows; it streams nothing.  All lanes of a warp work
// together.  Returns false for a block without rows.
template <int ROWS>
__device__ __forceinline__ bool tc_block_rows(const int32_t* __restrict__ row_ends, const int32_t* __restrict__ stream_ends, int clouds,
                                              int64_t num_rows, int64_t num_stream, int64_t slot, int64_t& row0, int64_t& row_end,
                                              int64_t& begin, int64_t& end) {
    const int lane = threadIdx.x & 31;
    int64_t first;
    int cloud;
    if (clouds <= 30) {  // lane b has the first rows of cloud b: one round of loads
        const int64_t rows_at = lane <= clouds ? cloud_begin(row_ends, lane, num_rows) : num_rows;
        const int64_t stream_at = lane <= clouds ? cloud_begin(stream_ends, lane, num_stream) : num_stream;
        const int count = __popc(__ballot_sync(kFullMask, lane <= clouds && rows_at / ROWS + lane <= slot));
        cloud = count > 0 ? count - 1 : 0;
        first = __shfl_sync(kFullMask, rows_at, cloud);
        row_end = max(first, __shfl_sync(kFullMask, rows_at, cloud + 1));
        begin = __shfl_sync(kFullMask, stream_at, cloud);
        end = max(begin, __shfl_sync(kFullMask, stream_at, cloud + 1));
    } else {
        int lo = 0, hi = clouds + 1;  // the answer lies in [lo, hi)
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) / 32, b = lo + lane * step;
            const bool before = b < hi && cloud_begin(row_ends, b, num_rows) / ROWS + b <= slot;
            const int count = __popc(__ballot_sync(kFullMask, before));  // lane 0's is always true for a valid range
            const int at = lo + (count > 0 ? count - 1 : 0) * step;
            hi = min(hi, at + step);
            lo = at;
        }
        cloud = lo;
        first = cloud_begin(row_ends, cloud, num_rows);
        row_end = cloud_end(row_ends, cloud, clouds, num_rows);
        begin = cloud_begin(stream_ends, cloud, num_stream);
        end = cloud_end(stream_ends, cloud, clouds, num_stream);
    }
    if (cloud >= clouds) begin = end = 0;
    row0 = first + (slot - (first / ROWS + cloud)) * ROWS;
    return row0 >= first && row0 < row_end;
}

constexpr int kTcSplitRows = 512;  // rows that a split has at least while there are more
constexpr int kTcGradRows = 64;    // rows of the gradients' largest streamed tiles

// Tiles of a split: an equal share, but at least that of `least` rows while there are more, so that small clouds make few
// splits and the splits of large ones are not longer than need be.
template <int BN>
__device__ __forceinline__ int64_t tc_tiles_of_split(int64_t tiles, int splits, int least) {
    const int64_t share = (tiles + splits - 1) / splits, floor = (least + BN - 1) / BN;
    return splits > 1 && share < floor ? floor : share;
}

__device__ __forceinline__ void tc_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ---- loads ------------------------------------------------------------------------------------------------------
// R rows from row0 of `head` into the tile at dst ([plane][64 features][R rows]), by one thread; `bar` has been told the bytes.
template <int R, int NP, int GR>
__device__ __forceinline__ void tc_load_whole(uint8_t* dst, const CUtensorMap* map, int64_t plane_rows, int head, int64_t row0, uint64_t* bar) {
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int g = 0; g < GR; ++g) tma_load_3d(dst + (p * GR + g) * R * 128, map, bar, g * 64, head, (int)(p * plane_rows + row0));
}

// The same for a streamed tile of which only the first `valid` rows belong to the cloud, with zeros behind them.  Called by a
// whole warp; completes one phase of `bar`.  A tile that ends inside the cloud takes boxes of eight rows (map8) as far as they
// go and at most seven rows through registers.
template <int R, int NP, int GR>
__device__ __forceinline__ void tc_load_tile(uint8_t* dst, const CUtensorMap* map, const CUtensorMap* map8, const TcRows& src,
                                             int64_t plane_rows, int head, int64_t row0, int valid, int size, uint64_t* bar) {
    const int lane = threadIdx.x & 31;
    if (valid >= R) {
        if (lane == 0) {
            mbar_expect_tx(bar, NP * GR * R * 128);
            tc_load_whole<R, NP, GR>(dst, map, plane_rows, head, row0, bar);
        }
    } else {
        const int chunks = size >> 3, boxed = valid & ~7;
#pragma unroll 1
        for (int pg = 0; pg < NP * GR; ++pg) {
            const int p = pg / GR, g = pg % GR;
            const __nv_bfloat16* from = src.data + p * src.plane + row0 * src.row + head * src.head + g * 64;
#pragma unroll 4
            for (int i = boxed * 8 + lane; i < R * 8; i += 32) {
                const int r = i >> 3, c = i & 7;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r < valid && g * 8 + c < chunks) v = *reinterpret_cast<const uint4*>(from + r * src.row + c * 8);
                *reinterpret_cast<uint4*>(dst + pg * R * 128 + sw128_offset(r, c)) = v;
            }
        }
        fence_smem_to_async_proxy();
        __syncwarp();
        if (lane == 0) {
            mbar_expect_tx(bar, NP * GR * boxed * 128);
            for (int pg = 0; pg < NP * GR; ++pg)
                for (int r = 0; r < boxed; r += 8)
                    tma_load_3d(dst + pg * R * 128 + r * 128, map8, bar, (pg % GR) * 64, head, (int)((pg / GR) * plane_rows + row0 + r));
        }
    }
    __syncwarp();
}

// One lane of a converged warp, always the same one.
__device__ __forceinline__ bool tc_elect() {
    uint32_t yes;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
    return yes != 0;
}

// ---- products (one elected thread of a converged warp) ----------------------------------------------------------
// The plane pairs of a product, smallest first; one pair (0, 0) for bf16 features.
template <int NP> struct TcPairs;
template <> struct TcPairs<1> {
    static constexpr int kCount = 1;
    __device__ static constexpr int a(int) { return 0; }
    __device__ static constexpr int b(int) { return 0; }
};
template <> struct TcPairs<3> {
    static constexpr int kCount = 6;
    __device__ static constexpr int a(int i) { return i == 0 ? 1 : i == 1 ? 2 : i == 2 ? 0 : i == 3 ? 1 : 0; }
    __device__ static constexpr int b(int i) { return i == 0 ? 1 : i == 1 ? 0 : i == 2 ? 2 : i == 3 ? 0 : i == 4 ? 1 : 0; }
};

// fp32 accumulate, bf16 x bf16, M = 128, N = n; b_mn: B's rows in memory are the K dimension.
__device__ __forceinline__ uint32_t tc_idesc(int n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTcRows >> 4) << 24);
}

// One thread issues all products, and until it has issued those of a unit the rows of that unit wait: the loops are unrolled
// and a descriptor is its tile's first one plus a constant (measured with descriptors built in the loop: 3500 of the 5700
// cycles of a unit were spent waiting for the next logits).
// D[128, RB] = A[128, features] B[RB, features]^T, both tiles in shared memory; `steps` blocks of 16 features.
template <int NP, int GR, int RB>
__device__ __forceinline__ void tc_rows_by_rows(uint32_t d, uint32_t a, uint32_t b, int steps) {
    const uint32_t idesc = tc_idesc(RB, false);
    const uint64_t da = umma_desc_k_sw128(a), db = umma_desc_k_sw128(b);
#pragma unroll
    for (int i = 0; i < TcPairs<NP>::kCount; ++i) {
#pragma unroll
        for (int k = 0; k < GR * 4; ++k) {  // 16 features = 32 bytes further inside the swizzled row; addresses in 16-byte units
            const int at_a = (TcPairs<NP>::a(i) * GR + (k >> 2)) * kTcRows * 8 + 2 * (k & 3);
            const int at_b = (TcPairs<NP>::b(i) * GR + (k >> 2)) * RB * 8 + 2 * (k & 3);
            if (k < steps) tc_mma_bf16(d, da + at_a, db + at_b, idesc, (i > 0 || k > 0) ? 1u : 0u);
        }
    }
}

// The same with A in tensor memory (planes of GR x 32 columns): the products of tiles of few rows are bound by reading A from
// shared memory otherwise (128 rows x 16 features are 4 KB, 32 cycles; with 32 rows of B the product itself takes 16).
template <int NP, int GR, int RB>
__device__ __forceinline__ void tc_kept_by_rows(uint32_t d, uint32_t a, uint32_t b, int steps) {
    const uint32_t idesc = tc_idesc(RB, false);
    const uint64_t db = umma_desc_k_sw128(b);
#pragma unroll
    for (int i = 0; i < TcPairs<NP>::kCount; ++i) {
#pragma unroll
        for (int k = 0; k < GR * 4; ++k) {
            const int at_b = (TcPairs<NP>::b(i) * GR + (k >> 2)) * RB * 8 + 2 * (k & 3);
            if (k < steps) tc_mma_bf16_ts(d, a + TcPairs<NP>::a(i) * GR * 32 + k * 8, db + at_b, idesc, (i > 0 || k > 0) ? 1u : 0u);
        }
    }
}

// D[128, n] (+)= E[128, RB] B[RB, n]: E in tensor memory (planes of RB / 2 columns), B's tile in shared memory; `steps` blocks
// of 16 rows of B.
template <int NP, int GR, int RB>
__device__ __forceinline__ void tc_weights_by_rows(uint32_t d, uint32_t e, uint32_t b, int n, int steps, bool accumulate) {
    const uint32_t idesc = tc_idesc(n, true);
    const uint64_t db = umma_desc_mn_sw128(b, RB * 128);
#pragma unroll
    for (int i = 0; i < TcPairs<NP>::kCount; ++i) {
#pragma unroll
        for (int k = 0; k < RB / 16; ++k)
            if (k < steps)
                tc_mma_bf16_ts(d, e + TcPairs<NP>::a(i) * (RB / 2) + k * 8, db + TcPairs<NP>::b(i) * GR * RB * 8 + k * 128, idesc,
                               (accumulate || i > 0 || k > 0) ? 1u : 0u);
    }
}

// ---- element-wise ------------------------------------------------------------------------------------------------
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float r;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// N values of this thread's row as bf16 planes into tensor memory, N / 2 columns of each plane.
template <int N>
__device__ __forceinline__ void tc_store_columns(uint32_t dst, const uint32_t (&w)[N / 2]) {
    if constexpr (N == 32) tc_st_32x16(dst, w);
    else tc_st_32x8(dst, w);
}
template <int NP, int PLANE_COLS, int N>
__device__ __forceinline__ void tc_store_weights(uint32_t dst, const float (&p)[N]) {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pack_bf16(p[2 * i], p[2 * i + 1]);
    tc_store_columns<N>(dst, w);
    if constexpr (NP == 3) {
        float r[N];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            r[2 * i] = p[2 * i] - __uint_as_float(w[i] << 16);
            r[2 * i + 1] = p[2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u);
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = pack_bf16(r[2 * i], r[2 * i + 1]);
        tc_store_columns<N>(dst + PLANE_COLS, w);
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
            w[i] = pack_bf16(r[2 * i] - __uint_as_float(w[i] << 16), r[2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u));
        tc_store_columns<N>(dst + 2 * PLANE_COLS, w);
    }
}

// sum[c] += column c of this thread's row, for the first n of N columns (n is a multiple of 16).
template <int N>
__device__ __forceinline__ void tc_add_columns(uint32_t from, int n, float (&sum)[N]) {
#pragma unroll
    for (int c = 0; c < N; c += 16) {
        if (c < n) {
            uint32_t r[16];
            tc_ld_32x16(from + c, r);
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[c + i] += __uint_as_float(r[i]);
        }
    }
}

// sum[c] = sum[c] fade + column c, or the column alone where the sums start.  For sums of rounds of many units: they lie in local
// memory (the loop keeps them out of the registers), which only calls with long clouds reach.
template <int N>
__device__ __forceinline__ void tc_empty_columns(uint32_t from, int n, bool start, float fade, float (&sum)[N]) {
#pragma unroll 1
    for (int c = 0; c < n; c += 16) {
        uint32_t r[16];
        tc_ld_32x16(from + c, r);
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[c + i] = start ? __uint_as_float(r[i]) : fmaf(sum[c + i], fade, __uint_as_float(r[i]));
    }
}

template <class T>
__device__ __forceinline__ void tc_write16(T* __restrict__ dst, int c, int size, const float (&x)[16]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (c + 8 * h >= size) break;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = x[8 * h + i];
        store_vec<T, 8>(dst + c + 8 * h, v);
    }
}

// ---- set-up and teardown -----------------------------------------------------------------------------------------
template <int COLUMNS>
__device__ __forceinline__ uint32_t tc_begin(TcShared* sh, int stages, int tiles_of_a_stage, int fixed_arrivals) {
    if (threadIdx.x == 0) {
        mbar_init(&sh->fixed_full, fixed_arrivals);
        for (int i = 0; i < stages; ++i) {
            mbar_init(&sh->full[i], tiles_of_a_stage);
            mbar_init(&sh->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh->s_full[i], 1);
            mbar_init(&sh->s_free[i], 4);  // the four warps of a group
            mbar_init(&sh->e_ready[i], 4);
            mbar_init(&sh->e_done[i], 1);
        }
        mbar_init(&sh->all_done, 1);
        mbar_init(&sh->drained[0], 1);
        mbar_init(&sh->drained[1], 1);
        mbar_init(&sh->round_done, 1);
        mbar_init(&sh->acc_free, 8);
        sh->failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem)), "r"(COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    return sh->tmem;
}
template <int COLUMNS>
__device__ __forceinline__ void tc_end(uint32_t tmem) {
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x < 32)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLUMNS) : "memory");
}
__device__ __forceinline__ void tc_fail(TcShared* sh, const TcControl& ctl, int code) {
    *(volatile int*)&sh->failed = 1;
    atomicCAS_system(ctl.sticky, 0, ctl.status | code);
}
// The end of a warp that issues products.  Every logit is waited for by the rows, and all sums have finished when all_done
// completes; after a failure the warp waits for its products in flight, since tensor memory may only be released after them.
__device__ __forceinline__ void tc_finish_products(TcShared* sh, const TcControl& ctl, bool ok, bool leader, bool sums) {
    if (leader) {
        if (!ok) {
            tc_fail(sh, ctl, 2);
            tc_commit(&sh->drained[sums]);
            mbar_wait(&sh->drained[sums], 0, ctl.poll_limit);
        } else if (sums) {
            tc_commit(&sh->all_done);
        }
    }
    __syncwarp();
}
// After a failure: copies that nobody has waited for must land before the CTA retires.
__device__ __forceinline__ void tc_drain_loads(TcShared* sh, int issued, int stages, uint32_t limit) {
    mbar_wait(&sh->fixed_full, 0, limit);
    for (int i = issued > stages ? issued - stages : 0; i < issued; ++i) mbar_wait(&sh->full[i % stages], (i / stages) & 1, limit);
}

// ---- forward ------------------------------------------------------------------------------------------------------
// Block = up to QT x 128 queries of one cloud and head x one split of the keys.  Units: with two query tiles unit u is
// (keys u / 2, tile u % 2); with one, unit u is key tile u, and the two element-wise groups take every other one, each with an
// accumulator, running maximum and sum of its own that are joined at the end.
// The tensor cores truncate when they add to an accumulator (measured on 32-bit heads of 64, 1000 keys: 3.7e-6 of the output with
// one accumulator for all keys).  For 32-bit features every unit starts its accumulator anew and the thread of a row adds the
// units up in registers, rounding to nearest.  bf16 weights hide the truncation of some 10^4 keys but not of any number (3 million
// keys: 1.6% of the output), so there an accumulator is emptied every kTcRoundRows rows, which bounds it by 2^-11, an eighth of the
// bf16 output's half step.
// Measured: 40001 queries, 20003 keys, 16 clouds, 8 heads on 2 of 128, bf16: 371 us, 727 TFLOP/s (44% of a cuBLAS product), tensor
// pipe 38% active: bound by the chain logits, probabilities, sums with two units in flight, and by products of 64 keys, which
// read their 128 rows from shared memory longer (48 cycles) than they compute (32).  Heads of 64, 30011 queries and
// keys, 8 clouds, 8 heads: 477 us, 637 TFLOP/s: the element-wise groups have a unit in hand 92% of the time, with the exponential unit
// 65% and the issue slots 44% busy, so they wait on the latency of their own chain (two warps per scheduler).
// 32-bit heads of 64, 16001 x 8003, 8 heads on 4: 319 us, the tensor pipe 41%.
// The accumulator is scaled only when the maximum has grown by more than 2^8 since it was last scaled: the probabilities
// stay below 2^8, and the final division is by a sum relative to the same reference.
// The logits and the probabilities have columns of their own: once the rows have been read into registers the logits of the
// group's next unit can be computed, while this unit's probabilities are still being made.  (Heads of 128 features: tiles of 128
// keys whose probabilities take the logits' place are slower, 415 us against 370 us for 40001 x 20003 points, 8 heads on 2.)
template <int GR, int BN, int NP, int QT>
struct TcForward {
    static constexpr int kQ = QT * NP * GR * kTcRows * 128;
    static constexpr int kSlot = NP * GR * BN * 128;
    static constexpr int kFit = (200 * 1024 - kQ) / kSlot;
    static constexpr int kStages = kFit > kTcMaxStages ? kTcMaxStages : kFit;
    static constexpr int kWeights = 2 * BN;             // columns of the probabilities, behind the logits of both groups
    static constexpr int kWeightCols = NP * (BN / 2);   // of one group
    static constexpr int kAcc = kWeights + 2 * kWeightCols;
    static constexpr int kRound = kTcRoundRows / BN;    // units of a group between two emptyings (bf16)
    static constexpr int kBytes = kQ + kStages * kSlot + 1024 + 512;
    static_assert(QT == 1 || NP == 1, "two query tiles are loaded as one plane");
    static_assert(kStages >= 4 && kStages % 2 == 0 && kAcc + 2 * GR * 64 <= 512, "does not fit");
    static_assert(kTcRows * GR * 64 * 4 + 2 * kTcRows * 4 <= kQ + kStages * kSlot, "no room to join the two groups");
};

template <int GR, int BN, int NP, int QT, class T>
__global__ void __launch_bounds__(kTcThreads, 1)
attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k8,
                    const __grid_constant__ CUtensorMap map_v8, AttentionCall a, TcRows rows_k, TcRows rows_v, int splits, int split_rows,
                    T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part_out, float2* __restrict__ part_stat,
                    TcControl ctl) {
    using Cfg = TcForward<GR, BN, NP, QT>;
    constexpr int kStages = Cfg::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = smem + Cfg::kQ;
    TcShared* sh = (TcShared*)(ring + kStages * Cfg::kSlot);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y, kv = h / (a.heads / a.kv_heads), split = blockIdx.z;
    if (threadIdx.x == 0) {
        tc_prefetch_map(&map_q);
        tc_prefetch_map(&map_k);
        tc_prefetch_map(&map_v);
    }
    int64_t row0, row_end, begin, end;
    if (!tc_block_rows<QT * kTcRows>(a.query_ends, a.key_ends, a.clouds, a.num_queries, a.num_keys, blockIdx.x, row0, row_end, begin, end)) return;
    const int rows_here = (int)min((int64_t)(QT * kTcRows), row_end - row0);
    {  // this split's keys, in whole tiles
        const int64_t tiles = (end - begin + BN - 1) / BN, per = tc_tiles_of_split<BN>(tiles, splits, split_rows);
        const int64_t lo = begin + split * per * BN;
        end = min(end, lo + per * BN);
        begin = min(lo, end);
    }
    const int64_t stat0 = ((int64_t)split * a.num_queries + row0) * a.heads + h;
    if (begin == end) {  // the same for the whole block
        for (int r = threadIdx.x; r < rows_here; r += kTcThreads) {
            if (splits > 1) {
                part_stat[stat0 + (int64_t)r * a.heads] = make_float2(-INFINITY, 0.f);
            } else {
                lse[(int64_t)h * a.num_queries + row0 + r] = -INFINITY;
                const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (int c = 0; c < a.size; c += 8) store_vec<T, 8>(out + ((row0 + r) * a.heads + h) * a.size + c, zero);
            }
        }
        return;
    }
    const uint32_t tmem = tc_begin<512>(sh, kStages, 1, 1);
    const int tiles = (int)((end - begin + BN - 1) / BN), q_tiles = rows_here > kTcRows ? 2 : 1, units = tiles * q_tiles;
    const int last_valid = (int)(end - begin) - (tiles - 1) * BN;
    const int steps = (a.size + 15) >> 4, n_out = steps * 16;
    const uint32_t acc = tmem + Cfg::kAcc;  // accumulator of group w: acc + w * GR * 64
    volatile int* failed = &sh->failed;
    const uint32_t limit = ctl.poll_limit;

    int issued = 0;  // streamed tiles that the loader has started
    const int ahead = min(tiles, q_tiles == 2 ? 1 : 2);  // key tiles in front of the first value tile
    if (warp == 8) {
        // ---- loader: the tiles in the order in which the products use them
        bool ok = true;
        // rows behind the cloud's last query are other clouds' (or zeros): each of them only reaches its own row of the products
        if (lane == 0) {
            mbar_expect_tx(&sh->fixed_full, q_tiles * NP * GR * kTcRows * 128);
            for (int t = 0; t < q_tiles; ++t)
                tc_load_whole<kTcRows, NP, GR>(smem + t * NP * GR * kTcRows * 128, &map_q, a.num_queries, h, row0 + t * kTcRows, &sh->fixed_full);
        }
        __syncwarp();
        // the logits run ahead by two units: K0 K1 V0 K2 V1 ... for two query tiles, K0 K1 K2 V0 K3 V1 ... for one
        const int loads = 2 * tiles;
        for (; issued < loads; ++issued) {
            const int it = issued;
            if (ctl.withhold_from >= 0 && it >= ctl.withhold_from) ok = false;
            const int s = it % kStages;
            if (ok && it >= kStages) ok = tc_wait_warp(&sh->empty[s], (it / kStages - 1) & 1, limit, failed);
            if (!ok) break;
            const int pair = (it - ahead) >> 1;
            const bool rest = it >= ahead && pair >= tiles - ahead, is_value = rest || (it >= ahead && ((it - ahead) & 1));
            const int j = it < ahead ? it : rest ? it - tiles : is_value ? pair : ahead + pair;
            const int valid = j == tiles - 1 ? last_valid : BN;
            if (is_value) tc_load_tile<BN, NP, GR>(ring + s * Cfg::kSlot, &map_v, &map_v8, rows_v, a.num_keys, kv, begin + (int64_t)j * BN, valid, a.size, &sh->full[s]);
            else tc_load_tile<BN, NP, GR>(ring + s * Cfg::kSlot, &map_k, &map_k8, rows_k, a.num_keys, kv, begin + (int64_t)j * BN, valid, a.size, &sh->full[s]);
        }
        if (!ok && lane == 0) tc_fail(sh, ctl, 1);
    } else if (warp == 9) {
        // ---- logits
        const bool leader = tc_elect();
        bool ok = tc_wait_warp(&sh->fixed_full, 0, limit, failed);
        int slot = 0;
        for (int u = 0; u < units && ok; ++u) {
            const bool first = q_tiles == 1 || !(u & 1), last = q_tiles == 1 || (u & 1);
            if (first) {  // key tile j is load j, or from `ahead` on every other one (an even ring: no value tile was in its slot)
                const int j = q_tiles == 2 ? u >> 1 : u, it = j < ahead ? j : 2 * j - ahead;
                slot = it % kStages;
                ok = tc_wait_warp(&sh->full[slot], (it / kStages) & 1, limit, failed);
            }
            if (u >= 2) ok = ok && tc_wait_warp(&sh->s_free[u & 1], ((u >> 1) - 1) & 1, limit, failed);  // unit u - 2 has been read
            if (!ok) break;
            tc_fence_after();
            if (leader) {
                tc_rows_by_rows<NP, GR, BN>(tmem + (u & 1) * BN, smem_u32(smem + (q_tiles == 2 ? u & 1 : 0) * NP * GR * kTcRows * 128),
                                            smem_u32(ring + slot * Cfg::kSlot), steps);
                if (last) tc_commit(&sh->empty[slot]);
                tc_commit(&sh->s_full[u & 1]);
            }
            __syncwarp();
        }
        tc_finish_products(sh, ctl, ok, leader, false);
    } else if (warp == 10) {
        // ---- sums of the values
        const bool leader = tc_elect();
        bool ok = true;
        int slot = 0;
        for (int u = 0; u < units && ok; ++u) {
            const bool first = q_tiles == 1 || !(u & 1), last = q_tiles == 1 || (u & 1);
            const int j = q_tiles == 2 ? u >> 1 : u, valid = j == tiles - 1 ? last_valid : BN;
            // First the probabilities: they exist only after the logits of this unit, hence after every key tile that can have been
            // in this value tile's slot before it (the ring has at least four slots), so the slot's barrier is not a phase behind.
            ok = tc_wait_warp(&sh->e_ready[u & 1], (u >> 1) & 1, limit, failed);
            if (first) {
                const int it = j < tiles - ahead ? ahead + 2 * j + 1 : tiles + j;
                slot = it % kStages;
                ok = ok && tc_wait_warp(&sh->full[slot], (it / kStages) & 1, limit, failed);
            }
            if (!ok) break;
            tc_fence_after();
            if (leader) {
                tc_weights_by_rows<NP, GR, BN>(acc + (u & 1) * GR * 64, tmem + Cfg::kWeights + (u & 1) * Cfg::kWeightCols,
                                               smem_u32(ring + slot * Cfg::kSlot), n_out, (valid + 15) >> 4, NP == 1 && (u >> 1) % Cfg::kRound != 0);
                if (last) tc_commit(&sh->empty[slot]);
                tc_commit(&sh->e_done[u & 1]);
            }
            __syncwarp();
        }
        tc_finish_products(sh, ctl, ok, leader, true);
    }

    const int group = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of tensor memory, in the address's upper half
    const float c2 = a.scale * kLog2e;
    float base = -INFINITY, total = 0.f;  // reference of the exponents (log2 units) and sum of the probabilities
    float kept[GR * 64];  // the output of all units but the last, for 32-bit features; of the emptied rounds in bf16, relative to kept_base
    if constexpr (NP == 3) {
#pragma unroll
        for (int c = 0; c < GR * 64; ++c) kept[c] = 0.f;
    }
    bool emptied = false;
    float kept_base = -INFINITY, kept_fade = 0.f;
    bool ok = true;
    if (warp < 8) {
        // ---- element-wise: logits to probabilities
        const uint32_t buf = tmem + lanes + group * BN, my_acc = acc + lanes + group * GR * 64;
        const uint32_t weights = tmem + lanes + Cfg::kWeights + group * Cfg::kWeightCols;
        const bool live = (q_tiles == 2 ? group * kTcRows : 0) + row < rows_here;  // a row behind the cloud may hold anything
        for (int u = group; u < units; u += 2) {
            if (!(ok = tc_wait_warp(&sh->s_full[group], (u >> 1) & 1, limit, failed))) break;
            tc_fence_after();
            const int j = q_tiles == 2 ? u >> 1 : u, valid = j == tiles - 1 ? last_valid : BN;
            uint32_t s[BN / 32][32];
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) tc_ld_32x32(buf + 32 * i, s[i]);
            tc_arrive_warp(&sh->s_free[group]);
            if (valid < BN) {  // columns behind the cloud repeat the first one, which changes no maximum
#pragma unroll
                for (int i = 0; i < BN; ++i)
                    if (i >= valid) s[i / 32][i % 32] = s[0][0];
            }
            float m[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = __uint_as_float(s[0][i]);
            if (c2 >= 0.f) {
#pragma unroll
                for (int i = 4; i < BN; i += 2) m[(i >> 1) & 3] = max3(m[(i >> 1) & 3], __uint_as_float(s[i / 32][i % 32]), __uint_as_float(s[i / 32][i % 32 + 1]));
                m[0] = fmaxf(max3(m[0], m[1], m[2]), m[3]);
            } else {
#pragma unroll
                for (int i = 4; i < BN; i += 2) m[(i >> 1) & 3] = min3(m[(i >> 1) & 3], __uint_as_float(s[i / 32][i % 32]), __uint_as_float(s[i / 32][i % 32 + 1]));
                m[0] = fminf(min3(m[0], m[1], m[2]), m[3]);
            }
            const float top = m[0] * c2;
            if (u >= 2) {  // the group's last unit has been added: its accumulator and its columns of probabilities are free
                if (!(ok = tc_wait_warp(&sh->e_done[group], ((u >> 1) - 1) & 1, limit, failed))) break;
                tc_fence_after();
            }
            const bool fresh = (u >> 1) % Cfg::kRound == 0;
            if constexpr (NP == 3) {
                if (u >= 2) tc_add_columns<GR * 64>(my_acc, n_out, kept);
            } else if (u >= 2 && fresh) {
                tc_empty_columns<GR * 64>(my_acc, n_out, !emptied, exp2_fast(kept_base - (base == -INFINITY ? 0.f : base)), kept);
                kept_base = base;
                emptied = true;
            }
            if (__any_sync(kFullMask, live && !(top <= base + 8.f))) {
                const float now = fmaxf(base, top), fade = exp2_fast(base - (now == -INFINITY ? 0.f : now));
                base = now;
                total *= fade;
                if constexpr (NP == 3) {
#pragma unroll
                    for (int c = 0; c < GR * 64; ++c) kept[c] *= fade;
                } else if (u >= 2 && !fresh) {
#pragma unroll 1
                    for (int c = 0; c < n_out; c += 16) {
                        uint32_t r[16];
                        tc_ld_32x16(my_acc + c, r);
#pragma unroll
                        for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * fade);
                        tc_st_32x16(my_acc + c, r);
                    }
                }
            }
            const float from = base == -INFINITY ? 0.f : base;
            const unsigned long long scale2 = pack_f32x2(c2, c2), from2 = pack_f32x2(-from, -from);
            unsigned long long sum[2] = {0ull, 0ull};
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) {
                float p[32];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[i][e]), __uint_as_float(s[i][e + 1])), scale2, from2), p[e], p[e + 1]);
                    p[e] = exp2_fast(p[e]);
                    p[e + 1] = exp2_fast(p[e + 1]);
                }
                if (valid < BN) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (i * 32 + e >= valid) p[e] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 2) sum[(e >> 1) & 1] = add_f32x2(sum[(e >> 1) & 1], pack_f32x2(p[e], p[e + 1]));
                // rounded to bf16 (NP = 1) only as the weights of the values; their sum is taken before
                tc_store_weights<NP, BN / 2>(weights + 16 * i, p);
            }
            float sum0, sum1;
            unpack_f32x2(add_f32x2(sum[0], sum[1]), sum0, sum1);
            total += sum0 + sum1;
            tc_wait_st();
            tc_arrive_warp(&sh->e_ready[group]);
        }
        if (ok && group < units) {
            ok = tc_wait_warp(&sh->all_done, 0, limit, failed);
            tc_fence_after();
        }
        if (!ok && lane == 0) tc_fail(sh, ctl, 3);
        if constexpr (NP == 3) {
            if (ok && group < units) tc_add_columns<GR * 64>(my_acc, n_out, kept);
        }
        kept_fade = exp2_fast(kept_base - (base == -INFINITY ? 0.f : base));
    }
    __syncthreads();
    const bool good = !*failed;
    if (!good && warp == 8) tc_drain_loads(sh, issued, kStages, limit);
    // 16 columns of this thread's accumulator from column c
    auto result = [&](int c, float (&x)[16]) {
        if constexpr (NP == 3) {
#pragma unroll
            for (int k = 0; k < GR * 64; k += 16)
                if (c == k) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = kept[k + i];
                }
        } else {
            uint32_t r[16];
            tc_ld_32x16(acc + lanes + group * GR * 64 + c, r);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(r[i]);
            if (emptied) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = fmaf(kept[c + i], kept_fade, x[i]);
            }
        }
    };
    // ---- joining the two groups of a single query tile, through the shared memory of the tiles
    float* swap_acc = (float*)smem;                    // [features][128 rows]
    float* swap_stat = swap_acc + kTcRows * GR * 64;   // [2][128]
    if (good && warp >= 4 && warp < 8 && q_tiles == 1) {
        if (units > 1) {
#pragma unroll 1
            for (int c = 0; c < n_out; c += 16) {
                float x[16];
                result(c, x);
#pragma unroll
                for (int i = 0; i < 16; ++i) swap_acc[(c + i) * kTcRows + row] = x[i];
            }
        }
        swap_stat[row] = base;
        swap_stat[kTcRows + row] = total;
    }
    __syncthreads();
    if (good && warp < 4 * q_tiles) {
        const int64_t m = row0 + group * kTcRows + row;
        const bool live = m < row_end;
        float own = 1.f, other = 0.f;
        if (q_tiles == 1 && units > 1) {
            const float b1 = swap_stat[row], now = fmaxf(base, b1), from = now == -INFINITY ? 0.f : now;
            own = exp2_fast(base - from);
            other = exp2_fast(b1 - from);
            total = total * own + swap_stat[kTcRows + row] * other;
            base = now;
        }
        const float inv = splits > 1 ? 1.f : total == 0.f ? 0.f : 1.f / total;
        const int64_t at = m * a.heads + h;
        if (live) {
            if (splits > 1) part_stat[stat0 + ((int64_t)group * kTcRows + row) * a.heads] = make_float2(base, total);
            else lse[(int64_t)h * a.num_queries + m] = total == 0.f ? -INFINITY : (base + log2f(total)) * kLn2;
        }
        const int64_t slot = (int64_t)split * a.num_queries * a.heads + at;
#pragma unroll 1
        for (int c = 0; c < n_out; c += 16) {
            float x[16];
            result(c, x);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (q_tiles == 1 && units > 1) x[i] = x[i] * own + swap_acc[(c + i) * kTcRows + row] * other;
                x[i] *= inv;
            }
            if (live) {
                if (splits > 1) tc_write16<float>(part_out + slot * a.size, c, a.size, x);
                else tc_write16<T>(out + at * a.size, c, a.size, x);
            }
        }
    }
    tc_end<512>(tmem);
}


// ---- backward -----------------------------------------------------------------------------------------------------
// KEYS = false: block = 128 queries of one cloud and head; it keeps Q and dO and streams K and V:
//   s = Q K^T, t = dO V^T, e = exp(scale s - lse) (t - delta),  dQ += e K.
// KEYS = true: block = 128 keys of one cloud and key head; it keeps K and V and streams Q and dO of every head that shares them:
//   s = K Q^T, t = V dO^T, p = exp(scale s - lse), e = p (t - delta),  dK += e Q,  dV += p dO.
// The accumulators are emptied every kRound units, for 32-bit features into registers (see the forward kernel on truncation).
// Measured on the calls of the forward kernel: bf16 647 us (queries) and 798 us (keys), tensor pipe 34 and 36% active; the queries'
// kernel waits for logits 40% of the time, the keys' is bound by its products, which take 82 cycles each where 32 to 48
// would do (two warps issue them in turn; with one warp they take 45 to 58, but it waits as long in between).  32 bits:
// 369 us and 549 us, tensor pipe 55%, products of 32 rows.  (622 us for the queries' gradient in bf16 before the accumulators were
// emptied and delta was decided cloud by cloud.)
// Two kernels, each recomputing the logits, instead of one that adds dQ with atomics: every sum is taken in a fixed order.
// 32-bit features: the two tiles that stay are kept as planes in tensor memory (kKeepInTmem), which leaves the keys' kernel no
// columns of their own for the weights: there they take the place of the logits (kInPlace), and the logits of a group's
// next unit wait until this one has been added.  Measured on 16001 x 8003 points, 8 heads on 4 of 64, with the tiles in shared
// memory and columns of their own: queries' gradient 534 us, keys' 598 us.
template <bool KEYS, int GR, int NP>
struct TcBackward {
    static constexpr bool kKeepInTmem = NP == 3 || (!KEYS && GR == 1), kInPlace = NP == 3 && KEYS;
    // streamed rows of a unit: as many as leave columns for s, t, the weights and the accumulators, and three slots of the ring (a
    // slot is held until its unit has been added, and the logits run ahead by two units)
    static constexpr int kBN = NP == 3 || (KEYS && GR == 2) ? 32 : 64;
    static constexpr int kFixed = kKeepInTmem ? 0 : NP * GR * kTcRows * 128;  // one of the two tiles that stay
    static constexpr int kTile = NP * GR * kBN * 128;                        // one of the two tiles of a slot
    static constexpr int kFit = (200 * 1024 - 2 * kFixed) / (2 * kTile);
    static constexpr int kStages = kFit > kTcMaxStages ? kTcMaxStages : kFit;
    static constexpr int kPlane = kBN / 2;
    static constexpr int kWeightCols = (KEYS ? 2 : 1) * NP * kPlane;          // weights of one group: e, then p
    static constexpr int kBuffer = kInPlace ? (kWeightCols > 2 * kBN ? kWeightCols : 2 * kBN) : 2 * kBN;  // s and t of one group
    static constexpr int kWeights = kInPlace ? 0 : 2 * kBuffer;               // columns of the weights
    static constexpr int kWeightStride = kInPlace ? kBuffer : kWeightCols;
    static constexpr int kAccStart = 2 * kBuffer + (kInPlace ? 0 : 2 * kWeightCols);
    static constexpr int kAcc = GR * 64;
    static constexpr int kKeep = kAccStart + (KEYS ? 2 : 1) * kAcc;           // the tiles that stay: planes of GR x 32 columns
    static constexpr int kKeepCols = NP * GR * 32;
    static constexpr int kRound = NP == 3 ? 4 : kTcRoundRows / kBN;           // even: both groups have units in a round
    static constexpr int kKept = KEYS ? kAcc : kAcc / 2;                      // columns of which a thread adds the rounds up
    static constexpr int kBytes = 2 * kFixed + kStages * (2 * kTile + 2 * kBN * 4) + 1024 + 512;
    static_assert(kStages >= 3 && kKeep + (kKeepInTmem ? 2 * kKeepCols : 0) <= 512 && kBytes <= 227 * 1024, "does not fit");
    static_assert(kTcGradRows % kBN == 0, "a split has whole tiles");
};

template <bool KEYS, int GR, int NP, class T>
__global__ void __launch_bounds__(kTcThreads, 1)
attention_tc_grads_kernel(const __grid_constant__ CUtensorMap map_f1, const __grid_constant__ CUtensorMap map_f2,
                          const __grid_constant__ CUtensorMap map_y1, const __grid_constant__ CUtensorMap map_y2,
                          const __grid_constant__ CUtensorMap map_y18, const __grid_constant__ CUtensorMap map_y28, AttentionCall a,
                          TcRows rows_f1, TcRows rows_f2, TcRows rows_y1, TcRows rows_y2, int splits, int split_rows, const float* __restrict__ lse,
                          float* __restrict__ delta, T* __restrict__ out1, T* __restrict__ out2, float* __restrict__ part1,
                          float* __restrict__ part2, TcControl ctl) {
    using Cfg = TcBackward<KEYS, GR, NP>;
    constexpr int kStages = Cfg::kStages, BN = Cfg::kBN;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = smem + 2 * Cfg::kFixed;
    float* column_stats = (float*)(ring + kStages * 2 * Cfg::kTile);  // [stages][lse in log2 units, delta][BN]
    TcShared* sh = (TcShared*)(column_stats + kStages * 2 * BN);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.y, split = blockIdx.z, share = a.heads / a.kv_heads;
    const int64_t num_rows = KEYS ? a.num_keys : a.num_queries, num_stream = KEYS ? a.num_queries : a.num_keys;
    const int32_t* row_ends = KEYS ? a.key_ends : a.query_ends;
    const int32_t* stream_ends = KEYS ? a.query_ends : a.key_ends;
    const int out_heads = KEYS ? a.kv_heads : a.heads;
    if (threadIdx.x == 0) {
        if (!Cfg::kKeepInTmem) {
            tc_prefetch_map(&map_f1);
            tc_prefetch_map(&map_f2);
        }
        tc_prefetch_map(&map_y1);
        tc_prefetch_map(&map_y2);
    }
    int64_t row0, row_end, begin, end;
    if (!tc_block_rows<kTcRows>(row_ends, stream_ends, a.clouds, num_rows, num_stream, blockIdx.x, row0, row_end, begin, end)) return;
    const int rows_here = (int)min((int64_t)kTcRows, row_end - row0);
    bool all_streamed;  // this split has all rows of the cloud (the cloud's other splits have none)
    {
        const int64_t tiles = (end - begin + BN - 1) / BN, per = tc_tiles_of_split<BN>(tiles, splits, split_rows);
        const int64_t lo = begin + split * per * BN;
        all_streamed = per >= tiles;
        end = min(end, lo + per * BN);
        begin = min(lo, end);
    }
    const int64_t out0 = (row0 * out_heads + head) * a.size, shift = (int64_t)split * num_rows * out_heads * a.size;
    if (begin == end) {
        const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int r = threadIdx.x; r < rows_here; r += kTcThreads)
            for (int c = 0; c < a.size; c += 8) {
                const int64_t at = out0 + (int64_t)r * out_heads * a.size + c;
                if (splits > 1) {
                    store_vec<float, 8>(part1 + shift + at, zero);
                    if (KEYS) store_vec<float, 8>(part2 + shift + at, zero);
                } else {
                    store_vec<T, 8>(out1 + at, zero);
                    if (KEYS) store_vec<T, 8>(out2 + at, zero);
                }
            }
        return;
    }
    const uint32_t tmem = tc_begin<512>(sh, kStages, 2, Cfg::kKeepInTmem ? 8 : 1);
    const int tiles = (int)((end - begin + BN - 1) / BN), units = tiles * (KEYS ? share : 1);
    const int last_valid = (int)(end - begin) - (tiles - 1) * BN;
    const int steps = (a.size + 15) >> 4, n_out = steps * 16;
    const uint32_t acc = tmem + Cfg::kAccStart;
    volatile int* failed = &sh->failed;
    const uint32_t limit = ctl.poll_limit;
    const float c2 = a.scale * kLog2e;

    int issued = 0;
    if (warp == 8) {
        // ---- loader: the two tiles of a slot share a barrier
        bool ok = true;
        if (!Cfg::kKeepInTmem && lane == 0) {  // rows behind the cloud's last one: see the forward kernel
            mbar_expect_tx(&sh->fixed_full, 2 * Cfg::kFixed);
            tc_load_whole<kTcRows, NP, GR>(smem, &map_f1, num_rows, head, row0, &sh->fixed_full);
            tc_load_whole<kTcRows, NP, GR>(smem + Cfg::kFixed, &map_f2, num_rows, head, row0, &sh->fixed_full);
        }
        __syncwarp();
        // KEYS: the columns' statistics of the next unit are on their way while the loader waits for its slot
        float next_lse[BN / 32], next_delta[BN / 32];
        auto fetch = [&](int u) {
            const int64_t at = (int64_t)(head * share + u / tiles) * num_stream + begin + (int64_t)(u % tiles) * BN;
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) {
                const bool in = u < units && (u % tiles < tiles - 1 || i * 32 + lane < last_valid);
                next_lse[i] = in ? lse[at + i * 32 + lane] : -INFINITY;
                next_delta[i] = in ? delta[at + i * 32 + lane] : 0.f;
            }
        };
        if (KEYS) fetch(0);
        for (; issued < units; ++issued) {
            if (ctl.withhold_from >= 0 && issued >= ctl.withhold_from) ok = false;
            const int s = issued % kStages;
            if (ok && issued >= kStages) ok = tc_wait_warp(&sh->empty[s], (issued / kStages - 1) & 1, limit, failed);
            if (!ok) break;
            const int j = issued % tiles, h = KEYS ? head * share + issued / tiles : head / share;
            const int valid = j == tiles - 1 ? last_valid : BN;
            const int64_t from = begin + (int64_t)j * BN;
            uint8_t* slot = ring + s * 2 * Cfg::kTile;
            if (KEYS) {  // an absent query has probability 2^-inf
                float* stats = column_stats + s * 2 * BN;
#pragma unroll
                for (int i = 0; i < BN / 32; ++i) {
                    stats[i * 32 + lane] = next_lse[i] == -INFINITY ? INFINITY : next_lse[i] * kLog2e;
                    stats[BN + i * 32 + lane] = next_delta[i];
                }
                __syncwarp();
                fetch(issued + 1);
            }
            tc_load_tile<BN, NP, GR>(slot, &map_y1, &map_y18, rows_y1, num_stream, h, from, valid, a.size, &sh->full[s]);
            tc_load_tile<BN, NP, GR>(slot + Cfg::kTile, &map_y2, &map_y28, rows_y2, num_stream, h, from, valid, a.size, &sh->full[s]);
        }
        if (!ok && lane == 0) tc_fail(sh, ctl, 1);
    } else if (warp == 9) {
        // ---- logits
        const bool leader = tc_elect();
        bool ok = tc_wait_warp(&sh->fixed_full, 0, limit, failed);
        for (int u = 0; u < units && ok; ++u) {
            const int s = u % kStages;
            ok = tc_wait_warp(&sh->full[s], (u / kStages) & 1, limit, failed);
            if (u >= 2)  // unit u - 2 has been read (or, where its weights are in its place, added)
                ok = ok && tc_wait_warp(Cfg::kInPlace ? &sh->e_done[u & 1] : &sh->s_free[u & 1], ((u >> 1) - 1) & 1, limit, failed);
            if (!ok) break;
            tc_fence_after();
            const uint32_t buf = tmem + (u & 1) * Cfg::kBuffer, slot = smem_u32(ring + s * 2 * Cfg::kTile);
            if (leader) {
                if constexpr (Cfg::kKeepInTmem) {
                    tc_kept_by_rows<NP, GR, BN>(buf, tmem + Cfg::kKeep, slot, steps);
                    tc_kept_by_rows<NP, GR, BN>(buf + BN, tmem + Cfg::kKeep + Cfg::kKeepCols, slot + Cfg::kTile, steps);
                } else {
                    tc_rows_by_rows<NP, GR, BN>(buf, smem_u32(smem), slot, steps);
                    tc_rows_by_rows<NP, GR, BN>(buf + BN, smem_u32(smem + Cfg::kFixed), slot + Cfg::kTile, steps);
                }
                tc_commit(&sh->s_full[u & 1]);
            }
            __syncwarp();
        }
        tc_finish_products(sh, ctl, ok, leader, false);
    } else if (warp == 10) {
        // ---- sums
        const bool leader = tc_elect();
        bool ok = true;
        for (int u = 0; u < units && ok; ++u) {
            ok = tc_wait_warp(&sh->e_ready[u & 1], (u >> 1) & 1, limit, failed);
            const bool fresh = u % Cfg::kRound == 0;
            if (u > 0 && fresh) ok = ok && tc_wait_warp(&sh->acc_free, (u / Cfg::kRound - 1) & 1, limit, failed);
            if (!ok) break;
            tc_fence_after();
            const int s = u % kStages, valid = u % tiles == tiles - 1 ? last_valid : BN;
            const uint32_t weights = tmem + Cfg::kWeights + (u & 1) * Cfg::kWeightStride, slot = smem_u32(ring + s * 2 * Cfg::kTile);
            if (leader) {
                tc_weights_by_rows<NP, GR, BN>(acc, weights, slot, n_out, (valid + 15) >> 4, !fresh);
                if (KEYS)
                    tc_weights_by_rows<NP, GR, BN>(acc + Cfg::kAcc, weights + NP * Cfg::kPlane, slot + Cfg::kTile, n_out, (valid + 15) >> 4,
                                                   !fresh);
                tc_commit(&sh->empty[s]);
                tc_commit(&sh->e_done[u & 1]);
                if ((u + 1) % Cfg::kRound == 0 && u + 1 < units) tc_commit(&sh->round_done);
            }
            __syncwarp();
        }
        tc_finish_products(sh, ctl, ok, leader, true);
    }

    const int group = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    float kept[Cfg::kKept];
    if constexpr (NP == 3) {
#pragma unroll
        for (int c = 0; c < Cfg::kKept; ++c) kept[c] = 0.f;
    }
    int emptied = 0;  // rounds
    // KEYS: the first group holds dK, the second dV.  Otherwise each group holds half the columns of dQ.
    const uint32_t my_acc = acc + lanes + group * (KEYS ? Cfg::kAcc : Cfg::kAcc / 2);
    // KEYS = false: of this thread's query (an absent one: probability 0).  delta comes from the forward pass' output, in bf16 rounded to
    // 8 bits; with few keys dp - delta is a small difference of the two (two keys: 0.4% of the gradients).  The sum of p dp over
    // the row, which delta is, comes out here: a cloud of one unit uses it at once, and the keys' kernel, which runs after this one,
    // finds it in delta's place wherever the cloud's keys are in one split (any number of keys below kTcSplitRows, whatever the
    // call's other clouds are: a small cloud's gradients do not depend on what it is batched with).
    float row_base = INFINITY, row_delta = 0.f, weighted_sum = 0.f;
    const int my_columns = KEYS ? n_out : min(max(n_out - group * (Cfg::kAcc / 2), 0), Cfg::kAcc / 2);
    if (warp < 8) {
        // ---- element-wise
        bool ok = true;
        const uint32_t buf = tmem + lanes + group * Cfg::kBuffer, weights = tmem + lanes + Cfg::kWeights + group * Cfg::kWeightStride;
        if constexpr (Cfg::kKeepInTmem) {
            // the first group brings the first tile that stays into tensor memory, the second the second: a row per thread
            const TcRows& from = group == 0 ? rows_f1 : rows_f2;
            const int chunks = row < rows_here ? a.size >> 3 : 0;
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const __nv_bfloat16* src = from.data + p * from.plane + (row0 + row) * from.row + head * from.head;
#pragma unroll
                for (int c = 0; c < GR * 8; c += 4) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (c + i < chunks) v = *reinterpret_cast<const uint4*>(src + (c + i) * 8);
                        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
                    }
                    tc_st_32x16(tmem + lanes + Cfg::kKeep + group * Cfg::kKeepCols + p * GR * 32 + c * 4, w);
                }
            }
            tc_wait_st();
            tc_arrive_warp(&sh->fixed_full);
        }
        auto empty_until = [&](int round) {  // adds up the accumulators of the rounds before `round`
            for (; emptied < round && ok; ++emptied) {
                if (!(ok = tc_wait_warp(&sh->round_done, emptied & 1, limit, failed))) break;
                tc_fence_after();
                if constexpr (NP == 3) tc_add_columns<Cfg::kKept>(my_acc, my_columns, kept);
                else tc_empty_columns<Cfg::kKept>(my_acc, my_columns, emptied == 0, 1.f, kept);
                tc_arrive_warp(&sh->acc_free);
            }
        };
        const bool whole = all_streamed && units == 1;  // this unit has all keys of the cloud
        if (!KEYS && row < rows_here) {
            const float l = lse[(int64_t)head * num_rows + row0 + row];
            row_base = l == -INFINITY ? INFINITY : l * kLog2e;
            row_delta = delta[(int64_t)head * num_rows + row0 + row];
        }
        for (int u = group; u < units; u += 2) {
            empty_until(u / Cfg::kRound);
            ok = ok && tc_wait_warp(&sh->s_full[group], (u >> 1) & 1, limit, failed);
            if (KEYS && ok) ok = tc_wait_warp(&sh->full[u % kStages], (u / kStages) & 1, limit, failed);  // the statistics are visible
            if (!ok) break;
            tc_fence_after();
            const int valid = u % tiles == tiles - 1 ? last_valid : BN;
            const float* stats = column_stats + (u % kStages) * 2 * BN;
            if constexpr (KEYS) {
                // 16 columns at a time, their statistics read ahead of the tensor memory: the products' operands keep the
                // shared memory busy
                constexpr int kParts = BN / 16;
                float4 base[4], d[4];
                auto read_stats = [&](int i) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        base[c] = *reinterpret_cast<const float4*>(stats + i * 16 + 4 * c);
                        d[c] = *reinterpret_cast<const float4*>(stats + BN + i * 16 + 4 * c);
                    }
                };
                read_stats(0);
                uint32_t s[Cfg::kInPlace ? kParts : 1][16], t[Cfg::kInPlace ? kParts : 1][16];
                if constexpr (Cfg::kInPlace) {  // all of them before the first weight is stored
#pragma unroll
                    for (int i = 0; i < kParts; ++i) {
                        tc_ld_32x16(buf + 16 * i, s[i]);
                        tc_ld_32x16(buf + BN + 16 * i, t[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < kParts; ++i) {
                    const int at = Cfg::kInPlace ? i : 0;
                    if constexpr (!Cfg::kInPlace) {
                        tc_ld_32x16(buf + 16 * i, s[0]);
                        tc_ld_32x16(buf + BN + 16 * i, t[0]);
                        if (i == kParts - 1) tc_arrive_warp(&sh->s_free[group]);
                    }
                    float p[16], e[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        p[c] = exp2_fast(fmaf(__uint_as_float(s[at][c]), c2, -(&base[c / 4].x)[c % 4]));
                        e[c] = p[c] * (__uint_as_float(t[at][c]) - (&d[c / 4].x)[c % 4]);
                    }
                    if (i + 1 < kParts) read_stats(i + 1);
                    if (!Cfg::kInPlace && i == 0 && u >= 2) {  // the group's last unit has been added: its columns of weights are free
                        if (!(ok = tc_wait_warp(&sh->e_done[group], ((u >> 1) - 1) & 1, limit, failed))) break;
                        tc_fence_after();
                    }
                    // rounded to bf16 (NP = 1) as the weights of the last two products, as the probabilities of the forward pass
                    tc_store_weights<NP, Cfg::kPlane>(weights + 8 * i, e);
                    tc_store_weights<NP, Cfg::kPlane>(weights + NP * Cfg::kPlane + 8 * i, p);
                }
            } else {
                uint32_t s[BN / 32][32], t[BN / 32][32];
#pragma unroll
                for (int i = 0; i < BN / 32; ++i) {
                    tc_ld_32x32(buf + 32 * i, s[i]);
                    tc_ld_32x32(buf + BN + 32 * i, t[i]);
                }
                tc_arrive_warp(&sh->s_free[group]);
                float p[BN / 32][32], weighted = 0.f;
#pragma unroll
                for (int i = 0; i < BN / 32; ++i) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        p[i][c] = exp2_fast(fmaf(__uint_as_float(s[i][c]), c2, -row_base));
                        if (valid < BN && i * 32 + c >= valid) p[i][c] = 0.f;  // a key behind the cloud: its probability may overflow
                        if (NP == 1) weighted = fmaf(p[i][c], __uint_as_float(t[i][c]), weighted);
                    }
                }
                if (NP == 1 && whole) row_delta = weighted;
                if (NP == 1) weighted_sum += weighted;
#pragma unroll
                for (int i = 0; i < BN / 32; ++i) {
                    float e[32];
#pragma unroll
                    for (int c = 0; c < 32; ++c) e[c] = p[i][c] * (__uint_as_float(t[i][c]) - row_delta);
                    if (i == 0 && u >= 2) {
                        if (!(ok = tc_wait_warp(&sh->e_done[group], ((u >> 1) - 1) & 1, limit, failed))) break;
                        tc_fence_after();
                    }
                    tc_store_weights<NP, Cfg::kPlane>(weights + 16 * i, e);
                }
            }
            if (!ok) break;
            tc_wait_st();
            tc_arrive_warp(&sh->e_ready[group]);
        }
        empty_until((units - 1) / Cfg::kRound);
        if (ok) {
            ok = tc_wait_warp(&sh->all_done, 0, limit, failed);
            tc_fence_after();
        }
        if constexpr (NP == 3) {
            if (ok) tc_add_columns<Cfg::kKept>(my_acc, my_columns, kept);
        }
        if (!ok && lane == 0) tc_fail(sh, ctl, 3);
    }
    __syncthreads();
    const bool good = !*failed;
    if (!good && warp == 8) tc_drain_loads(sh, issued, kStages, limit);
    if (!KEYS && NP == 1 && all_streamed) {  // the same for the block; no other block reads or writes these rows' delta
        float* swap = (float*)smem;  // all products have finished
        if (good && warp >= 4 && warp < 8) swap[row] = weighted_sum;
        __syncthreads();
        if (good && warp < 4 && row < rows_here) delta[(int64_t)head * num_rows + row0 + row] = weighted_sum + swap[row];
    }
    if (good && warp < 8) {
        const float factor = KEYS && group == 1 ? 1.f : a.scale;
        const int64_t at = out0 + (int64_t)row * out_heads * a.size;
        T* out = KEYS && group == 1 ? out2 : out1;
        float* part = KEYS && group == 1 ? part2 : part1;
        const int column0 = KEYS ? 0 : group * (Cfg::kAcc / 2);
#pragma unroll
        for (int c = 0; c < (KEYS ? Cfg::kAcc : Cfg::kAcc / 2); c += 16) {
            if (c >= my_columns) break;
            float x[16];
            if constexpr (NP == 3) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = kept[c + i] * factor;
            } else {
                uint32_t r[16];
                tc_ld_32x16(my_acc + c, r);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(r[i]);
                if (emptied > 0) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] += kept[c + i];
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] *= factor;
            }
            if (row < rows_here) {
                if (splits > 1) tc_write16<float>(part + shift + at, column0 + c, a.size, x);
                else tc_write16<T>(out + at, column0 + c, a.size, x);
            }
        }
    }
    tc_end<512>(tmem);
}

}  // namespace pccnn
