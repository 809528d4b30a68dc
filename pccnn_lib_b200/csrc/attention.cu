// Cross attention between packed clouds: every query of cloud b attends to the keys of cloud b.
//
//   out = softmax(scale q k^T) v,  lse = log sum exp(scale q k^T)      per head; heads / kv_heads heads share keys and values
//   p = exp(scale q k^T - lse), dp = g v^T, ds = p (dp - sum(g out)):  dq = scale ds k,  dk = scale ds^T q,  dv = p^T g
//
// The kernels of this file work on rows: a block owns one query (or, for the keys' gradients, one key) and streams the other
// side of its cloud.  They serve any head size up to 256, any stride and alignment, and are the ones for few queries: with
// one query per cloud the call is bound by reading keys and values once, and a query's keys are then split over several
// blocks whose results are joined by a second kernel.  Sums, maxima and probabilities are 32-bit floats.
#include <cuda_bf16.h>

#include <type_traits>

#include "attention.cuh"
#include "common.cuh"
#include "features.cuh"
#include "status.cuh"

namespace pccnn {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kMaxHeadSize = 256;

// ---- layout of a block: LPK lanes of a warp share a streamed row (V elements each, NC times), 32 / LPK rows per warp ----
template <class T, int V, int NC>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int lane_in_row, int lanes_per_row, int size, float (&x)[NC][V]) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = (c * lanes_per_row + lane_in_row) * V;
        if (d < size) {
            load_vec<T, V>(p + d, x[c]);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[c][e] = 0.f;
        }
    }
}
template <int V, int NC>
__device__ __forceinline__ float dot(const float (&a)[NC][V], const float (&b)[NC][V]) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) s = fmaf(a[c][e], b[c][e], s);
    return s;
}
__device__ __forceinline__ float sum_lanes(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    return v;
}

// Adds x over the row groups of the block (fixed order); threads of warp 0's first group hold the result.
template <int V, int NC>
__device__ __forceinline__ void add_over_block(float (&x)[NC][V], int lanes_per_row, float* scratch) {
    for (int o = lanes_per_row; o < 32; o <<= 1) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) x[c][e] += __shfl_xor_sync(kFullMask, x[c][e], o);
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane < lanes_per_row) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) scratch[((warp * NC + c) * 32 + lane) * V + e] = x[c][e];
    }
    __syncthreads();
    if (warp == 0 && lane < lanes_per_row) {
#pragma unroll
        for (int w = 1; w < kRowWarps; ++w)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) x[c][e] += scratch[((w * NC + c) * 32 + lane) * V + e];
    }
}

// The part of [begin, end) that split s of `splits` works on: equal parts, but none of fewer than 192 rows while there are
// more, so that the splits of a small cloud are few and those of a large one are not longer than need be.
__device__ __forceinline__ void split_range(int64_t& begin, int64_t& end, int s, int splits) {
    int64_t per = (end - begin + splits - 1) / splits;
    if (splits > 1 && per < 192) per = 192;
    const int64_t lo = begin + s * per, hi = lo + per;
    end = hi < end ? hi : end;
    begin = lo < end ? lo : end;
}

// ---- forward: block = one query x up to 8 key heads x one split of the keys -------------------------------------------
// A warp serves one key head (and GH query heads that share it): with several key heads the warps of a block walk the same
// rows side by side, so that a block reads whole rows; with fewer than eight the warps of a head take different keys.  A
// lane has the next kUnroll keys and values in flight while it works on the last ones, as raw 16-byte vectors.
// Without splits the output and lse are written; with splits the block leaves its unnormalised sum (relative to its own
// maximum), the maximum and the sum of the probabilities.
// V values held as packed pairs where there are pairs: two multiply-adds per instruction.
template <int V>
struct Lanes {
    static constexpr int kN = V > 1 ? V / 2 : 1;
    using Word = typename std::conditional<(V > 1), unsigned long long, float>::type;
    Word w[kN];
    __device__ __forceinline__ void set(const float (&x)[V]) {
        if constexpr (V > 1) {
#pragma unroll
            for (int i = 0; i < kN; ++i) w[i] = pack_f32x2(x[2 * i], x[2 * i + 1]);
        } else {
            w[0] = x[0];
        }
    }
    __device__ __forceinline__ void get(float (&x)[V]) const {
        if constexpr (V > 1) {
#pragma unroll
            for (int i = 0; i < kN; ++i) unpack_f32x2(w[i], x[2 * i], x[2 * i + 1]);
        } else {
            x[0] = w[0];
        }
    }
    // this += a * b, element by element
    __device__ __forceinline__ void add_product(const Lanes& a, const Lanes& b) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if constexpr (V > 1) w[i] = fma_f32x2(a.w[i], b.w[i], w[i]);
            else w[i] = fmaf(a.w[i], b.w[i], w[i]);
        }
    }
    __device__ __forceinline__ void add_scaled(const Lanes& a, float s) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if constexpr (V > 1) w[i] = fma_f32x2(a.w[i], pack_f32x2(s, s), w[i]);
            else w[i] = fmaf(a.w[i], s, w[i]);
        }
    }
    __device__ __forceinline__ void scale(float s) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if constexpr (V > 1) w[i] = mul_f32x2(w[i], pack_f32x2(s, s));
            else w[i] *= s;
        }
    }
    __device__ __forceinline__ float sum() const {
        float x[V], s = 0.f;
        get(x);
#pragma unroll
        for (int e = 0; e < V; ++e) s += x[e];
        return s;
    }
};

// Sums of U values over lanes_per_row lanes (at least U), each value's sum in its own part of the lanes: value `mine` in this one.
template <int U>
__device__ __forceinline__ float sum_and_spread(const float (&s)[U], int lanes_per_row, int in_row, int& mine) {
    static_assert(U == 2 || U == 4, "two or four values");
    int o = lanes_per_row >> 1;
    float v;
    if constexpr (U == 4) {
        const bool hi = in_row & o;
        float a = hi ? s[2] : s[0], b = hi ? s[3] : s[1];
        a += __shfl_xor_sync(kFullMask, hi ? s[0] : s[2], o);
        b += __shfl_xor_sync(kFullMask, hi ? s[1] : s[3], o);
        o >>= 1;
        const bool odd = in_row & o;
        v = (odd ? b : a) + __shfl_xor_sync(kFullMask, odd ? a : b, o);
        mine = (hi ? 2 : 0) + (odd ? 1 : 0);
    } else {
        const bool odd = in_row & o;
        v = (odd ? s[1] : s[0]) + __shfl_xor_sync(kFullMask, odd ? s[0] : s[1], o);
        mine = odd ? 1 : 0;
    }
    for (o >>= 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    return v;
}

// The end of a block: joins the row groups of a warp, then the warps of a head in ascending order, and writes.
template <class T, int V, int NC, int GH>
__device__ __forceinline__ void finish_rows(const AttentionCall& a, int64_t m, int h0, int lanes_per_row, int warp_heads, int splits,
                                            const float (&top)[GH], const float (&total)[GH], float (&acc)[GH][NC][V],
                                            T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part_out,
                                            float2* __restrict__ part_stat) {
    __shared__ float scratch[kRowWarps * NC * 32 * V];
    __shared__ float stat[kRowWarps][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slice = warp / warp_heads, split = blockIdx.z;
    const int group = a.heads / a.kv_heads, heads_here = min(GH, (h0 / group + 1) * group - h0);
#pragma unroll
    for (int g = 0; g < GH; ++g) {
        if (g >= heads_here) break;  // the same for the whole block
        float now = top[g];
        for (int o = lanes_per_row; o < 32; o <<= 1) now = fmaxf(now, __shfl_xor_sync(kFullMask, now, o));
        if (lane == 0) stat[warp][0] = now;
        __syncthreads();
        for (int w = warp % warp_heads; w < kRowWarps; w += warp_heads) now = fmaxf(now, stat[w][0]);
        const float from = now == -INFINITY ? 0.f : now;
        const float fade = exp2_fast(top[g] - from);
        float sum = total[g] * fade;
        sum = warp_sum(sum);
        if (lane == 0) stat[warp][1] = sum;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                acc[g][c][e] *= fade;
                for (int o = lanes_per_row; o < 32; o <<= 1) acc[g][c][e] += __shfl_xor_sync(kFullMask, acc[g][c][e], o);
                if (slice > 0 && lane < lanes_per_row) scratch[((warp * NC + c) * 32 + lane) * V + e] = acc[g][c][e];
            }
        __syncthreads();
        if (slice == 0) {
            for (int w = warp + warp_heads; w < kRowWarps; w += warp_heads) {
                sum += stat[w][1];
                if (lane < lanes_per_row) {
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int e = 0; e < V; ++e) acc[g][c][e] += scratch[((w * NC + c) * 32 + lane) * V + e];
                }
            }
            const int64_t at = m * a.heads + h0 + g;
            if (splits > 1) {
                const int64_t slot = (int64_t)split * a.num_queries * a.heads + at;
                if (lane == 0) part_stat[slot] = make_float2(now, sum);
                if (lane < lanes_per_row) {
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const int d = (c * lanes_per_row + lane) * V;
                        if (d < a.size) store_vec<float, V>(part_out + slot * a.size + d, acc[g][c]);
                    }
                }
            } else {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                if (lane == 0) lse[(int64_t)(h0 + g) * a.num_queries + m] = sum == 0.f ? -INFINITY : (now + log2f(sum)) * kLn2;
                if (lane < lanes_per_row) {
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const int d = (c * lanes_per_row + lane) * V;
#pragma unroll
                        for (int e = 0; e < V; ++e) acc[g][c][e] *= inv;
                        if (d < a.size) store_vec<T, V>(out + at * a.size + d, acc[g][c]);
                    }
                }
            }
        }
        __syncthreads();
    }
}

template <class T, int V, int NC, int GH>
__global__ void __launch_bounds__(kRowThreads)
attention_row_kernel(AttentionCall a, int lanes_per_row, int warp_heads, int splits, T* __restrict__ out, float* __restrict__ lse,
                     float* __restrict__ part_out, float2* __restrict__ part_stat) {
    constexpr int kUnroll = NC * V * GH > 32 ? 2 : 4;
    const int64_t m = blockIdx.x;
    const int group = a.heads / a.kv_heads, parts = (group + GH - 1) / GH;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slices = kRowWarps / warp_heads, slice = warp / warp_heads;
    const int kv = blockIdx.y / parts * warp_heads + warp % warp_heads, h0 = kv * group + (blockIdx.y % parts) * GH;
    const int heads_here = min(GH, (kv + 1) * group - h0), split = blockIdx.z;
    const int in_row = lane % lanes_per_row, sub = lane / lanes_per_row, per_warp = 32 / lanes_per_row;

    const int b = cloud_of_row(a.query_ends, a.clouds, m);
    int64_t begin = 0, end = 0;
    if (b < a.clouds) {
        begin = cloud_begin(a.key_ends, b, a.num_keys);
        end = cloud_end(a.key_ends, b, a.clouds, a.num_keys);
    }
    split_range(begin, end, split, splits);

    const float c2 = a.scale * kLog2e;
    Lanes<V> q[GH][NC], sums[GH][NC];
    float top[GH], total[GH];
#pragma unroll
    for (int g = 0; g < GH; ++g) {
        top[g] = -INFINITY;
        total[g] = 0.f;
        float x[NC][V];
        load_row<T, V, NC>((const T*)a.q.data + m * a.q.row + (h0 + min(g, heads_here - 1)) * a.q.head, in_row, lanes_per_row, a.size, x);
        const float zero[V] = {};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            q[g][c].set(x[c]);
            sums[g][c].set(zero);
        }
    }
    const T* keys = (const T*)a.k.data + kv * a.k.head;
    const T* values = (const T*)a.v.data + kv * a.v.head;
    const int step = slices * per_warp;
    RawVec<T, V> key[kUnroll][NC], val[kUnroll][NC];
    auto fetch = [&](int64_t first) {
        const T *k0 = keys + (first + sub) * a.k.row, *v0 = values + (first + sub) * a.v.row;
        const bool whole = first + (int64_t)step * (kUnroll - 1) + per_warp <= end;  // the same for the warp
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const bool in = whole || first + u * step + sub < end;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = (c * lanes_per_row + in_row) * V;
                if (in && d < a.size) {
                    key[u][c].load(k0 + d);
                    val[u][c].load(v0 + d);
                } else {
                    key[u][c].clear();
                    val[u][c].clear();
                }
            }
            k0 += step * a.k.row;
            v0 += step * a.v.row;
        }
    };
    // A logit is summed over the lanes of its row while the four of an iteration part: every lane ends with one of them, and
    // its exponential is taken once and handed round.  The kernel is bound by the instructions it issues (68% of the slots
    // with a full sum and exponential in every lane: 199 us for 400000 keys, 8 heads of 64, bf16, 16 queries; so 178 us).
    const int64_t start = begin + slice * per_warp;
    if (start < end) fetch(start);
    for (int64_t first = start; first < end; first += (int64_t)step * kUnroll) {  // the same for the warp's lanes
        float s[GH][kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            Lanes<V> x[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float f[V];
                key[u][c].widen(f);
                x[c].set(f);
            }
#pragma unroll
            for (int g = 0; g < GH; ++g) {
                const float zero[V] = {};
                Lanes<V> dot;
                dot.set(zero);
#pragma unroll
                for (int c = 0; c < NC; ++c) dot.add_product(q[g][c], x[c]);
                s[g][u] = dot.sum();
            }
        }
        RawVec<T, V> now_val[kUnroll][NC];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int c = 0; c < NC; ++c) now_val[u][c] = val[u][c];
        if (first + (int64_t)step * kUnroll < end) fetch(first + (int64_t)step * kUnroll);
#pragma unroll
        for (int g = 0; g < GH; ++g) {
            int mine;
            float v = sum_and_spread<kUnroll>(s[g], lanes_per_row, in_row, mine) * c2;
            if (first + mine * step + sub >= end) v = -INFINITY;
            float now = fmaxf(v, __shfl_xor_sync(kFullMask, v, lanes_per_row >> 1));
            if (kUnroll == 4) now = fmaxf(now, __shfl_xor_sync(kFullMask, now, lanes_per_row >> 2));
            now = fmaxf(top[g], now);
            const float from = now == -INFINITY ? 0.f : now;
            const float fade = exp2_fast(top[g] - from), p = exp2_fast(v - from);
            top[g] = now;
            total[g] = fmaf(total[g], fade, p);
#pragma unroll
            for (int c = 0; c < NC; ++c) sums[g][c].scale(fade);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int at = kUnroll == 4 ? (u >> 1) * (lanes_per_row >> 1) + (u & 1) * (lanes_per_row >> 2) : u * (lanes_per_row >> 1);
                s[g][u] = __shfl_sync(kFullMask, p, sub * lanes_per_row + at);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float f[V];
                now_val[u][c].widen(f);
                Lanes<V> x;
                x.set(f);
#pragma unroll
                for (int g = 0; g < GH; ++g) sums[g][c].add_scaled(x, s[g][u]);
            }
        }
    }
    float acc[GH][NC][V];
#pragma unroll
    for (int g = 0; g < GH; ++g) {
        total[g] *= (float)kUnroll / (float)lanes_per_row;  // a probability is held by that many lanes (a power of two)
#pragma unroll
        for (int c = 0; c < NC; ++c) sums[g][c].get(acc[g][c]);
    }
    finish_rows<T, V, NC, GH>(a, m, h0, lanes_per_row, warp_heads, splits, top, total, acc, out, lse, part_out, part_stat);
}

// d += a b for 16 rows (a), 8 columns (b) and 16 features of bf16: a0, a2 belong to the lane's first row, a1, a3 to the one eight behind.
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same for bf16 with the logits on the tensor cores: 16 keys are the rows of a product, lane (g, t) holds features of keys g
// and g + 8 as they lie in memory, and the queries of the heads that share them are its columns, repeated, so that every
// lane finds the logits of its own keys in its own registers: no sums over lanes, and softmax statistics per four lanes until the
// end.  The features of a product may come in any order as long as both sides have the same one.  Values are added as above.
template <int NC, int GH>
__global__ void __launch_bounds__(kRowThreads)
attention_row_products_kernel(AttentionCall a, int warp_heads, int splits, __nv_bfloat16* __restrict__ out, float* __restrict__ lse,
                              float* __restrict__ part_out, float2* __restrict__ part_stat) {
    using T = __nv_bfloat16;
    static_assert(GH == 1 || GH == 4, "a column's head is its own or its lane's neighbor's");
    constexpr int V = 8, kLanes = 4, kTiles = NC * GH > 1 ? 1 : 2;  // of 16 keys in flight; with two for heads of 64 and 1 block per SM 205 us, with one 175 us
    const int64_t m = blockIdx.x;
    const int group = a.heads / a.kv_heads, parts = (group + GH - 1) / GH;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slices = kRowWarps / warp_heads, slice = warp / warp_heads;
    const int kv = blockIdx.y / parts * warp_heads + warp % warp_heads, h0 = kv * group + (blockIdx.y % parts) * GH;
    const int heads_here = min(GH, (kv + 1) * group - h0), split = blockIdx.z;
    const int in_row = lane % kLanes, sub = lane / kLanes;

    const int b = cloud_of_row(a.query_ends, a.clouds, m);
    int64_t begin = 0, end = 0;
    if (b < a.clouds) {
        begin = cloud_begin(a.key_ends, b, a.num_keys);
        end = cloud_end(a.key_ends, b, a.clouds, a.num_keys);
    }
    split_range(begin, end, split, splits);

    const float c2 = a.scale * kLog2e;
    RawVec<T, V> q[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = (c * kLanes + in_row) * V;
        if (d < a.size) q[c].load((const T*)a.q.data + m * a.q.row + (h0 + min(sub % GH, heads_here - 1)) * a.q.head + d);
        else q[c].clear();
    }
    Lanes<V> sums[GH][NC];
    float top[GH], total[GH];
#pragma unroll
    for (int g = 0; g < GH; ++g) {
        top[g] = -INFINITY;
        total[g] = 0.f;
        const float zero[V] = {};
#pragma unroll
        for (int c = 0; c < NC; ++c) sums[g][c].set(zero);
    }
    const T* keys = (const T*)a.k.data + kv * a.k.head;
    const T* values = (const T*)a.v.data + kv * a.v.head;
    const int step = slices * 16;
    RawVec<T, V> key[kTiles][2][NC], val[kTiles][2][NC];
    auto fetch = [&](int64_t first) {
        const bool whole = first + (int64_t)step * (kTiles - 1) + 16 <= end;  // the same for the warp
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int64_t row = first + u * step + r * 8 + sub;
                const T *k0 = keys + row * a.k.row, *v0 = values + row * a.v.row;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int d = (c * kLanes + in_row) * V;
                    if ((whole || row < end) && d < a.size) {
                        key[u][r][c].load(k0 + d);
                        val[u][r][c].load(v0 + d);
                    } else {
                        key[u][r][c].clear();
                        val[u][r][c].clear();
                    }
                }
            }
    };
    const int64_t start = begin + slice * 16;
    if (start < end) fetch(start);
    for (int64_t first = start; first < end; first += (int64_t)step * kTiles) {  // the same for the warp's lanes
        float s[GH][kTiles][2];
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};  // keys (g, g, g + 8, g + 8), columns (2t, 2t + 1) twice
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                mma_16x8x16(d, key[u][0][c].v.x, key[u][1][c].v.x, key[u][0][c].v.y, key[u][1][c].v.y, q[c].v.x, q[c].v.y);
                mma_16x8x16(d, key[u][0][c].v.z, key[u][1][c].v.z, key[u][0][c].v.w, key[u][1][c].v.w, q[c].v.z, q[c].v.w);
            }
            if constexpr (GH == 1) {
                s[0][u][0] = d[0];
                s[0][u][1] = d[2];
            } else {  // an even lane has heads 0 and 1, an odd one 2 and 3
                const bool odd = lane & 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float other = __shfl_xor_sync(kFullMask, d[i], 1);
                    s[i & 1][u][i >> 1] = odd ? other : d[i];
                    s[2 + (i & 1)][u][i >> 1] = odd ? d[i] : other;
                }
            }
        }
        RawVec<T, V> now_val[kTiles][2][NC];
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                now_val[u][0][c] = val[u][0][c];
                now_val[u][1][c] = val[u][1][c];
            }
        if (first + (int64_t)step * kTiles < end) fetch(first + (int64_t)step * kTiles);
#pragma unroll
        for (int g = 0; g < GH; ++g) {
            float now = top[g];
#pragma unroll
            for (int u = 0; u < kTiles; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    s[g][u][r] = first + u * step + r * 8 + sub < end ? s[g][u][r] * c2 : -INFINITY;
                    now = fmaxf(now, s[g][u][r]);
                }
            const float from = now == -INFINITY ? 0.f : now;
            const float fade = exp2_fast(top[g] - from);
            top[g] = now;
            total[g] *= fade;
#pragma unroll
            for (int u = 0; u < kTiles; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    s[g][u][r] = exp2_fast(s[g][u][r] - from);
                    total[g] += s[g][u][r];
                }
#pragma unroll
            for (int c = 0; c < NC; ++c) sums[g][c].scale(fade);
        }
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    float f[V];
                    now_val[u][r][c].widen(f);
                    Lanes<V> x;
                    x.set(f);
#pragma unroll
                    for (int g = 0; g < GH; ++g) sums[g][c].add_scaled(x, s[g][u][r]);
                }
    }
    float acc[GH][NC][V];
#pragma unroll
    for (int g = 0; g < GH; ++g) {
        total[g] *= 1.f / kLanes;  // every probability is held by the lanes of its row
#pragma unroll
        for (int c = 0; c < NC; ++c) sums[g][c].get(acc[g][c]);
    }
    finish_rows<T, V, NC, GH>(a, m, h0, kLanes, warp_heads, splits, top, total, acc, out, lse, part_out, part_stat);
}

// Joins the splits of a query: W warps of a block per (query, head), each with every W-th split, joined in ascending order.
// Four splits are read at once, their statistics first: splits without keys have left no sum to read (one after
// the other: 8192 rows of 64 in 14 splits 18 us, so 10 us; 128 rows in 128 splits 11 us, so 7 us).  C: columns of a lane.
template <class T, int W, int C>
__global__ void __launch_bounds__(256)
attention_join_kernel(int64_t num_queries, int heads, int size, int splits, const float* __restrict__ part_out,
                      const float2* __restrict__ part_stat, T* __restrict__ out, float* __restrict__ lse) {
    constexpr int kRows = 8 / W, kAtOnce = 4;
    __shared__ float sums[W > 1 ? 8 : 1][C * 32 + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % W;
    const int64_t rows = num_queries * heads, row = (int64_t)blockIdx.x * kRows + warp / W;
    const bool live = row < rows;
    float top = -INFINITY;
    if (live)
        for (int s = lane; s < splits; s += 32) top = fmaxf(top, part_stat[s * rows + row].x);
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
    const float from = top == -INFINITY ? 0.f : top;
    float total = 0.f, acc[C];
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    if (live) {
        for (int s0 = part; s0 < splits; s0 += kAtOnce * W) {
            float2 st[kAtOnce];
            float x[kAtOnce][C];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) st[u] = s0 + u * W < splits ? part_stat[(s0 + u * W) * rows + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                for (int i = 0; i < C; ++i)
                    x[u][i] = st[u].y != 0.f && i * 32 + lane < size ? part_out[((s0 + u * W) * rows + row) * size + i * 32 + lane] : 0.f;
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const float f = exp2_fast(st[u].x - from);
                total += st[u].y * f;
#pragma unroll
                for (int i = 0; i < C; ++i) acc[i] = fmaf(f, x[u][i], acc[i]);
            }
        }
    }
    if (W > 1) {
#pragma unroll
        for (int i = 0; i < C; ++i) sums[warp][i * 32 + lane] = acc[i];
        if (lane == 0) sums[warp][C * 32] = total;
        __syncthreads();
        if (part != 0) return;
        for (int w = warp + 1; w < warp + W; ++w) {
            total += sums[w][C * 32];
#pragma unroll
            for (int i = 0; i < C; ++i) acc[i] += sums[w][i * 32 + lane];
        }
    }
    if (!live) return;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    if (lane == 0) lse[(row % heads) * num_queries + row / heads] = total == 0.f ? -INFINITY : (top + log2f(total)) * kLn2;
#pragma unroll
    for (int i = 0; i < C; ++i)
        if (i * 32 + lane < size) out[row * size + i * 32 + lane] = from_float<T>(acc[i] * inv);
}

// ---- backward ---------------------------------------------------------------------------------------------------
// delta[h, m] = sum_d out g: LPK lanes of a warp per (query, head), V elements each at a time.
template <class T, int V>
__global__ void __launch_bounds__(256)
attention_delta_kernel(int64_t num_queries, int heads, int size, int lanes_per_row, const T* __restrict__ out, HeadRows grads,
                       float* __restrict__ delta) {
    const int64_t rows = num_queries * heads, per_block = 256 / lanes_per_row;
    const int lane = threadIdx.x % lanes_per_row;
    for (int64_t first = blockIdx.x * per_block; first < rows; first += gridDim.x * per_block) {  // the same for the block
        const int64_t row = first + threadIdx.x / lanes_per_row;
        const int64_t m = row / heads;
        const int h = (int)(row - m * heads);
        float s = 0.f;
        if (row < rows) {
            const T* g = (const T*)grads.data + m * grads.row + h * grads.head;
            for (int d = lane * V; d < size; d += lanes_per_row * V) {
                float a[V], b[V];
                load_vec<T, V>(out + row * size + d, a);
                load_vec<T, V>(g + d, b);
#pragma unroll
                for (int e = 0; e < V; ++e) s = fmaf(a[e], b[e], s);
            }
        }
        s = sum_lanes(s, lanes_per_row);
        if (row < rows && lane == 0) delta[(int64_t)h * num_queries + m] = s;
    }
}

// Queries' gradient: block = one query and head x one split of its keys.
// DELTA: instead of the gradient, delta = sum_n p dp itself, for clouds of at most kDeltaKeys keys (splits = 1): the rounding of a
// bf16 output is a large part of dp - delta there (see attention_tc_grads_kernel).  Larger clouds keep what is in delta.
constexpr int kDeltaKeys = 256;
template <class T, int V, int NC, bool DELTA>
__global__ void __launch_bounds__(kRowThreads)
attention_query_grads_row_kernel(AttentionCall a, HeadRows grads, int lanes_per_row, int splits, const float* __restrict__ lse,
                                 float* __restrict__ delta, T* __restrict__ out, float* __restrict__ part) {
    __shared__ float scratch[kRowWarps * NC * 32 * V];
    const int64_t m = blockIdx.x;
    const int h = blockIdx.y, kv = h / (a.heads / a.kv_heads), split = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int in_row = lane % lanes_per_row, sub = lane / lanes_per_row, per_warp = 32 / lanes_per_row;
    const int b = cloud_of_row(a.query_ends, a.clouds, m);
    int64_t begin = 0, end = 0;
    if (b < a.clouds) {
        begin = cloud_begin(a.key_ends, b, a.num_keys);
        end = cloud_end(a.key_ends, b, a.clouds, a.num_keys);
    }
    if (DELTA && end - begin > kDeltaKeys) return;  // the same for the block
    split_range(begin, end, split, splits);
    const float c2 = a.scale * kLog2e;
    const float row_lse = lse[(int64_t)h * a.num_queries + m], base = row_lse == -INFINITY ? INFINITY : row_lse * kLog2e;
    const float row_delta = DELTA ? 0.f : delta[(int64_t)h * a.num_queries + m];
    float weighted = 0.f;
    float q[NC][V], g[NC][V], acc[NC][V];
    load_row<T, V, NC>((const T*)a.q.data + m * a.q.row + h * a.q.head, in_row, lanes_per_row, a.size, q);
    load_row<T, V, NC>((const T*)grads.data + m * grads.row + h * grads.head, in_row, lanes_per_row, a.size, g);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[c][e] = 0.f;
    const T* keys = (const T*)a.k.data + kv * a.k.head;
    const T* values = (const T*)a.v.data + kv * a.v.head;
    for (int64_t first = begin + warp * per_warp; first < end; first += kRowWarps * per_warp) {
        const int64_t n = first + sub;
        const bool in = n < end;
        float key[NC][V], val[NC][V];
        load_row<T, V, NC>(keys + (in ? n : begin) * a.k.row, in_row, lanes_per_row, a.size, key);
        load_row<T, V, NC>(values + (in ? n : begin) * a.v.row, in_row, lanes_per_row, a.size, val);
        const float s = sum_lanes(dot<V, NC>(q, key), lanes_per_row);
        const float dp = sum_lanes(dot<V, NC>(g, val), lanes_per_row);
        const float ds = exp2_fast(s * c2 - base) * (dp - row_delta);
        if (DELTA) {
            weighted += in && in_row == 0 ? ds : 0.f;
        } else if (in) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[c][e] = fmaf(ds, key[c][e], acc[c][e]);
        }
    }
    if constexpr (DELTA) {
        weighted = warp_sum(weighted);
        if (lane == 0) scratch[warp] = weighted;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kRowWarps; ++w) weighted += scratch[w];
            delta[(int64_t)h * a.num_queries + m] = weighted;
        }
        return;
    }
    add_over_block<V, NC>(acc, lanes_per_row, scratch);
    if (warp == 0 && lane < lanes_per_row) {
        const int64_t at = (m * a.heads + h) * a.size;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = (c * lanes_per_row + lane) * V;
            if (d >= a.size) break;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[c][e] *= a.scale;
            if (splits > 1) store_vec<float, V>(part + (int64_t)split * a.num_queries * a.heads * a.size + at + d, acc[c]);
            else store_vec<T, V>(out + at + d, acc[c]);
        }
    }
}

// Keys' and values' gradients: block = one key and its head x one split of the queries; the heads that share it are added.
template <class T, int V, int NC>
__global__ void __launch_bounds__(kRowThreads)
attention_key_grads_row_kernel(AttentionCall a, HeadRows grads, int lanes_per_row, int splits, const float* __restrict__ lse,
                               const float* __restrict__ delta, T* __restrict__ out_k, T* __restrict__ out_v,
                               float* __restrict__ part_k, float* __restrict__ part_v) {
    __shared__ float scratch[kRowWarps * NC * 32 * V];
    const int64_t n = blockIdx.x;
    const int kv = blockIdx.y, group = a.heads / a.kv_heads, split = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int in_row = lane % lanes_per_row, sub = lane / lanes_per_row, per_warp = 32 / lanes_per_row;
    const int b = cloud_of_row(a.key_ends, a.clouds, n);
    int64_t begin = 0, end = 0;
    if (b < a.clouds) {
        begin = cloud_begin(a.query_ends, b, a.num_queries);
        end = cloud_end(a.query_ends, b, a.clouds, a.num_queries);
    }
    split_range(begin, end, split, splits);
    const float c2 = a.scale * kLog2e;
    float key[NC][V], val[NC][V], dk[NC][V], dv[NC][V];
    load_row<T, V, NC>((const T*)a.k.data + n * a.k.row + kv * a.k.head, in_row, lanes_per_row, a.size, key);
    load_row<T, V, NC>((const T*)a.v.data + n * a.v.row + kv * a.v.head, in_row, lanes_per_row, a.size, val);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) dk[c][e] = dv[c][e] = 0.f;
    for (int h = kv * group; h < (kv + 1) * group; ++h) {
        const T* queries = (const T*)a.q.data + h * a.q.head;
        const T* g_rows = (const T*)grads.data + h * grads.head;
        for (int64_t first = begin + warp * per_warp; first < end; first += kRowWarps * per_warp) {
            const bool in = first + sub < end;
            const int64_t m = in ? first + sub : begin;
            float q[NC][V], g[NC][V];
            load_row<T, V, NC>(queries + m * a.q.row, in_row, lanes_per_row, a.size, q);
            load_row<T, V, NC>(g_rows + m * grads.row, in_row, lanes_per_row, a.size, g);
            const float row_lse = lse[(int64_t)h * a.num_queries + m];
            const float s = sum_lanes(dot<V, NC>(q, key), lanes_per_row);
            const float dp = sum_lanes(dot<V, NC>(g, val), lanes_per_row);
            const float p = exp2_fast(s * c2 - (row_lse == -INFINITY ? INFINITY : row_lse * kLog2e));
            const float ds = p * (dp - delta[(int64_t)h * a.num_queries + m]);
            if (in) {
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        dk[c][e] = fmaf(ds, q[c][e], dk[c][e]);
                        dv[c][e] = fmaf(p, g[c][e], dv[c][e]);
                    }
            }
        }
    }
    add_over_block<V, NC>(dk, lanes_per_row, scratch);
    __syncthreads();
    add_over_block<V, NC>(dv, lanes_per_row, scratch);
    if (warp == 0 && lane < lanes_per_row) {
        const int64_t at = (n * a.kv_heads + kv) * a.size, shift = (int64_t)split * a.num_keys * a.kv_heads * a.size;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = (c * lanes_per_row + lane) * V;
            if (d >= a.size) break;
#pragma unroll
            for (int e = 0; e < V; ++e) dk[c][e] *= a.scale;
            if (splits > 1) {
                store_vec<float, V>(part_k + shift + at + d, dk[c]);
                store_vec<float, V>(part_v + shift + at + d, dv[c]);
            } else {
                store_vec<T, V>(out_k + at + d, dk[c]);
                store_vec<T, V>(out_v + at + d, dv[c]);
            }
        }
    }
}

// out = the sum of the splits' parts, in ascending order.
template <class T>
__global__ void __launch_bounds__(256)
add_splits_kernel(int64_t count, int splits, const float* __restrict__ part, T* __restrict__ out) {
    for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < splits; ++s) v += part[s * count + i];
        out[i] = from_float<T>(v);
    }
}

// ---- host: choice of the kernel -----------------------------------------------------------------------------------
// 16-byte vectors need a head size and strides that are multiples of one and 16-byte aligned data; anything else goes
// element by element.
static bool vector_heads(const HeadRows& x, int v) { return aligned16(x.data) && x.row % v == 0 && x.head % v == 0; }

struct RowLayout {
    bool vectors;
    int chunks, lanes;
};
static RowLayout row_layout(const AttentionCall& a, const HeadRows* grads, bool outputs_aligned) {
    const int v = a.is_bf16 ? 8 : 4;
    RowLayout l;
    l.vectors = outputs_aligned && a.size % v == 0 && vector_heads(a.q, v) && vector_heads(a.k, v) && vector_heads(a.v, v) && (!grads || vector_heads(*grads, v));
    const int n = l.vectors ? a.size / v : a.size;
    l.lanes = 4;  // at least: the forward kernel spreads four keys over a row's lanes
    while (l.lanes < 32 && l.lanes < n) l.lanes *= 2;
    l.chunks = 1;
    while (l.chunks * l.lanes < n) l.chunks *= 2;
    return l;
}

// How many blocks share the `streamed` rows of a cloud (on average) when there are `units` blocks without a split: enough to
// give every SM about twelve blocks (clouds differ in size, and the last blocks should be short), as long as a block keeps
// at least 256 rows.
static int choose_splits(int64_t units, int64_t streamed_per_cloud, int blocks_per_sm = 12) {
    const int64_t want = (int64_t)sm_count() * blocks_per_sm;
    int64_t s = units > 0 ? (want + units - 1) / units : 1;
    const int64_t most = streamed_per_cloud / 256;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
}

static int64_t mean_rows(int64_t n, int clouds) { return n / (clouds > 0 ? clouds : 1); }

// GH heads that share keys are served by one pass over them where there are at least two.
static int forward_parts(const AttentionCall& a) {
    const int group = a.heads / a.kv_heads;
    return group >= 2 ? (group + 3) / 4 : 1;
}

// Key heads that a block of the forward kernel serves side by side, one (or several) warps each.
static int warp_heads(const AttentionCall& a) {
    int n = kRowWarps;
    while (a.kv_heads % n) n /= 2;
    return n;
}
// Logits on the tensor cores, for bf16 rows that are read in vectors: 16 queries, 400000 keys, 8 heads of 64 on 2: 185 us without, 135
// us with them and 95 us with three blocks per SM (six: 111 us); 6 heads of 32
// on 2: 127, 62 and 52 us; 8 heads of 64 that share none 178 and 175 us, 150 queries on 301 keys, 4 heads of 32 8.3 and 6.9 us.
// Heads of 128 that share none were slower with them (178 and 195 us), so wider ones stay with the plain kernel.
bool use_products(const AttentionCall& a) { return a.is_bf16 && a.size > 16 && a.size <= 64; }

static int forward_splits(const AttentionCall& a) {
    const bool shared = use_products(a) && a.heads > a.kv_heads;
    return choose_splits(a.num_queries * (a.kv_heads / warp_heads(a)) * forward_parts(a), mean_rows(a.num_keys, a.clouds), shared ? 3 : 12);
}
static int query_grad_splits(const AttentionCall& a) {
    return choose_splits(a.num_queries * a.heads, mean_rows(a.num_keys, a.clouds));
}
static int key_grad_splits(const AttentionCall& a) {
    return choose_splits(a.num_keys * a.kv_heads, mean_rows(a.num_queries, a.clouds));
}

template <class T, int C>
static int join_splits_as(const AttentionCall& a, int splits, const float* part, const float2* stat, void* out, float* lse, cudaStream_t s) {
    // one warp per row: with many splits (few rows) the whole block shares a row
    const int64_t rows = a.num_queries * a.heads;
    if (splits >= 16) attention_join_kernel<T, 8, C><<<(unsigned)rows, 256, 0, s>>>(a.num_queries, a.heads, a.size, splits, part, stat, (T*)out, lse);
    else attention_join_kernel<T, 1, C><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(a.num_queries, a.heads, a.size, splits, part, stat, (T*)out, lse);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}
template <class T>
static int join_splits_of(const AttentionCall& a, int splits, const float* part, const float2* stat, void* out, float* lse, cudaStream_t s) {
    if (a.size <= 64) return join_splits_as<T, 2>(a, splits, part, stat, out, lse, s);
    if (a.size <= 128) return join_splits_as<T, 4>(a, splits, part, stat, out, lse, s);
    return join_splits_as<T, 8>(a, splits, part, stat, out, lse, s);
}
int join_splits(const AttentionCall& a, int splits, const float* part, const float2* stat, void* out, float* lse, cudaStream_t s) {
    return a.is_bf16 ? join_splits_of<__nv_bfloat16>(a, splits, part, stat, out, lse, s) : join_splits_of<float>(a, splits, part, stat, out, lse, s);
}

template <class T, int V, int NC>
static int launch_rows(const AttentionCall& a, const RowLayout& l, void* out, float* lse, char* ws, cudaStream_t s) {
    const int splits = forward_splits(a);
    float2* stat = (float2*)ws;
    float* part = (float*)(ws + align_up((size_t)splits * a.num_queries * a.heads * sizeof(float2)));
    const int side_by_side = warp_heads(a);
    const dim3 grid((unsigned)a.num_queries, (unsigned)(a.kv_heads / side_by_side * forward_parts(a)), (unsigned)splits);
    if constexpr (sizeof(T) == 2 && V == 8) {
        if (use_products(a)) {
            const auto kernel = a.heads > a.kv_heads ? (a.size <= 32 ? attention_row_products_kernel<1, 4> : attention_row_products_kernel<2, 4>)
                                : a.size <= 32       ? attention_row_products_kernel<1, 1>
                                                     : attention_row_products_kernel<2, 1>;
            kernel<<<grid, kRowThreads, 0, s>>>(a, side_by_side, splits, (T*)out, lse, part, stat);
            PCCNN_LAUNCH_CHECK();
            return splits > 1 ? join_splits(a, splits, part, stat, out, lse, s) : PCCNN_OK;
        }
    }
    if (a.heads > a.kv_heads)
        attention_row_kernel<T, V, NC, 4><<<grid, kRowThreads, 0, s>>>(a, l.lanes, side_by_side, splits, (T*)out, lse, part, stat);
    else
        attention_row_kernel<T, V, NC, 1><<<grid, kRowThreads, 0, s>>>(a, l.lanes, side_by_side, splits, (T*)out, lse, part, stat);
    PCCNN_LAUNCH_CHECK();
    return splits > 1 ? join_splits(a, splits, part, stat, out, lse, s) : PCCNN_OK;
}

int add_splits(int is_bf16, int64_t count, int splits, const float* part, void* out, cudaStream_t s) {
    const unsigned blocks = grid_for(count, 256, 8);
    if (is_bf16) add_splits_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(count, splits, part, (__nv_bfloat16*)out);
    else add_splits_kernel<float><<<blocks, 256, 0, s>>>(count, splits, part, (float*)out);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

template <class T, int V, int NC>
static int launch_grad_rows(const AttentionCall& a, const HeadRows& grads, const RowLayout& l, const float* lse, float* delta,
                            void* dq, void* dk, void* dv, char* ws, cudaStream_t s) {
    float* part = (float*)ws;
    if (a.num_queries > 0) {
        const int splits = query_grad_splits(a);
        if constexpr (sizeof(T) == 2) {
            attention_query_grads_row_kernel<T, V, NC, true><<<dim3((unsigned)a.num_queries, (unsigned)a.heads), kRowThreads, 0, s>>>(
                a, grads, l.lanes, 1, lse, delta, (T*)dq, part);
            PCCNN_LAUNCH_CHECK();
        }
        attention_query_grads_row_kernel<T, V, NC, false><<<dim3((unsigned)a.num_queries, (unsigned)a.heads, (unsigned)splits), kRowThreads, 0, s>>>(
            a, grads, l.lanes, splits, lse, delta, (T*)dq, part);
        PCCNN_LAUNCH_CHECK();
        if (splits > 1)
            if (int rc = add_splits(a.is_bf16, a.num_queries * a.heads * a.size, splits, part, dq, s)) return rc;
    }
    if (a.num_keys > 0) {
        const int splits = key_grad_splits(a);
        const int64_t count = a.num_keys * a.kv_heads * a.size;
        attention_key_grads_row_kernel<T, V, NC><<<dim3((unsigned)a.num_keys, (unsigned)a.kv_heads, (unsigned)splits), kRowThreads, 0, s>>>(
            a, grads, l.lanes, splits, lse, delta, (T*)dk, (T*)dv, part, part + splits * count);
        PCCNN_LAUNCH_CHECK();
        if (splits > 1) {
            if (int rc = add_splits(a.is_bf16, count, splits, part, dk, s)) return rc;
            if (int rc = add_splits(a.is_bf16, count, splits, part + splits * count, dv, s)) return rc;
        }
    }
    return PCCNN_OK;
}

template <class T, class F>
static int dispatch_rows(const RowLayout& l, const F& f) {
    constexpr int kV = 16 / sizeof(T);
    if (l.vectors) {
        if constexpr (sizeof(T) == 2) return f.template run<T, kV, 1>();  // kMaxHeadSize is one vector of each lane
        else return l.chunks == 1 ? f.template run<T, kV, 1>() : f.template run<T, kV, 2>();
    }
    if (l.chunks == 1) return f.template run<T, 1, 1>();
    if (l.chunks == 2) return f.template run<T, 1, 2>();
    return l.chunks == 4 ? f.template run<T, 1, 4>() : f.template run<T, 1, 8>();
}

struct ForwardRows {
    const AttentionCall& a; RowLayout l; void* out; float* lse; char* ws; cudaStream_t s;
    template <class T, int V, int NC> int run() const { return launch_rows<T, V, NC>(a, l, out, lse, ws, s); }
};
struct BackwardRows {
    const AttentionCall& a; const HeadRows& grads; RowLayout l; const float* lse; float* delta; void *dq, *dk, *dv; char* ws; cudaStream_t s;
    template <class T, int V, int NC> int run() const { return launch_grad_rows<T, V, NC>(a, grads, l, lse, delta, dq, dk, dv, ws, s); }
};

static int launch_delta(const AttentionCall& a, const void* out, const HeadRows& grads, float* delta, cudaStream_t s) {
    const int v = a.is_bf16 ? 8 : 4;
    const bool vectors = a.size % v == 0 && aligned16(out) && vector_heads(grads, v);
    int lanes = 1;
    while (lanes < 32 && lanes * (vectors ? v : 1) < a.size) lanes *= 2;
    const unsigned blocks = grid_for(a.num_queries * a.heads * lanes, 256, 16);
    auto run = [&](auto kernel, auto* typed) { kernel<<<blocks, 256, 0, s>>>(a.num_queries, a.heads, a.size, lanes, typed, grads, delta); };
    if (a.is_bf16) run(vectors ? attention_delta_kernel<__nv_bfloat16, 8> : attention_delta_kernel<__nv_bfloat16, 1>, (const __nv_bfloat16*)out);
    else run(vectors ? attention_delta_kernel<float, 4> : attention_delta_kernel<float, 1>, (const float*)out);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

static int check_call(const char* who, const AttentionCall& a) {
    PCCNN_CHECK_ARG(a.num_queries >= 0 && a.num_queries < 0x7fffffffLL && a.num_keys >= 0 && a.num_keys < 0x7fffffffLL && a.clouds >= 0 && a.clouds < (1 << 30),
                    "%s: bad number of rows or clouds", who);
    PCCNN_CHECK_ARG(a.heads > 0 && a.heads <= 1024 && a.kv_heads > 0 && a.heads % a.kv_heads == 0,
                    "%s: %d heads cannot share %d key heads (at most 1024 heads, a multiple of the key heads)", who, a.heads, a.kv_heads);
    PCCNN_CHECK_ARG(a.size > 0 && a.size <= kMaxHeadSize, "%s: head size %d outside [1, %d]", who, a.size, kMaxHeadSize);
    PCCNN_CHECK_ARG(a.clouds == 0 || (a.query_ends && a.key_ends), "%s: null pointer", who);
    PCCNN_CHECK_ARG((a.num_queries == 0 || a.q.data) && (a.num_keys == 0 || (a.k.data && a.v.data)), "%s: null pointer", who);
    return PCCNN_OK;
}

// The stride of a dimension of one element means nothing: it becomes that of contiguous rows.
static HeadRows head_rows(const void* data, const int64_t* strides, int64_t rows, int heads, int size) {
    if (!strides) return {data, 0, 0};
    return {data, rows > 1 ? strides[0] : (int64_t)heads * size, heads > 1 ? strides[1] : size};
}

static AttentionCall describe(int64_t num_queries, int64_t num_keys, int clouds, int heads, int kv_heads, int size, int is_bf16,
                              const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                              const int64_t* v_strides, const int32_t* query_ends, const int32_t* key_ends, float scale) {
    AttentionCall a{num_queries, num_keys, clouds, heads, kv_heads, size, is_bf16, {q, 0, 0}, {k, 0, 0}, {v, 0, 0}, query_ends, key_ends, scale};
    a.q = head_rows(q, q_strides, num_queries, heads, size);
    a.k = head_rows(k, k_strides, num_keys, kv_heads, size);
    a.v = head_rows(v, v_strides, num_keys, kv_heads, size);
    return a;
}

}  // namespace pccnn

using namespace pccnn;

extern "C" {

size_t pccnn_cross_attention_workspace_bytes(int64_t num_queries, int64_t num_keys, int clouds, int heads, int kv_heads, int size,
                                             int is_bf16) {
    if (num_queries <= 0 || num_keys <= 0 || heads <= 0 || kv_heads <= 0 || size <= 0) return 256;
    const AttentionCall a = describe(num_queries, num_keys, clouds, heads, kv_heads, size, is_bf16, nullptr, nullptr, nullptr, nullptr,
                                     nullptr, nullptr, nullptr, nullptr, 1.f);
    const int splits = forward_splits(a);
    const size_t rows = splits > 1 ? (size_t)splits * num_queries * heads : 0;
    const size_t by_rows = align_up(rows * sizeof(float2)) + align_up(rows * size * 4) + 256, by_tiles = tc_shape(a) ? tc_forward_workspace(a) : 0;
    return by_rows > by_tiles ? by_rows : by_tiles;
}

int pccnn_cross_attention(int64_t num_queries, int64_t num_keys, int clouds, int heads, int kv_heads, int size, int is_bf16,
                          const void* queries, const int64_t* query_strides_host, const void* keys, const int64_t* key_strides_host,
                          const void* values, const int64_t* value_strides_host, const int32_t* query_ends, const int32_t* key_ends,
                          float scale, void* out, float* out_lse, void* workspace, size_t workspace_bytes, void* stream) {
    const AttentionCall a = describe(num_queries, num_keys, clouds, heads, kv_heads, size, is_bf16, queries, query_strides_host, keys,
                                     key_strides_host, values, value_strides_host, query_ends, key_ends, scale);
    if (int rc = check_call("cross_attention", a)) return rc;
    PCCNN_CHECK_ARG(query_strides_host && key_strides_host && value_strides_host, "cross_attention: null pointer");
    if (num_queries == 0) return PCCNN_OK;
    PCCNN_CHECK_ARG(out && out_lse, "cross_attention: null pointer");
    const size_t need = pccnn_cross_attention_workspace_bytes(num_queries, num_keys, clouds, heads, kv_heads, size, is_bf16);
    if (!workspace || workspace_bytes < need) {
        set_error("cross_attention: workspace of %zu bytes, need %zu", workspace_bytes, need);
        return PCCNN_ERR_WORKSPACE;
    }
    if (int rc = take_sticky_status("cross_attention")) return rc;  // an earlier call's tensor-core kernel gave up
    if (num_keys > 0 && tc_shape(a) && tc_layout(a, nullptr) && aligned16(out)) return tc_forward(a, out, out_lse, (char*)workspace, (cudaStream_t)stream);
    const ForwardRows f{a, row_layout(a, nullptr, aligned16(out)), out, out_lse, (char*)workspace, (cudaStream_t)stream};
    return is_bf16 ? dispatch_rows<__nv_bfloat16>(f.l, f) : dispatch_rows<float>(f.l, f);
}

size_t pccnn_cross_attention_grads_workspace_bytes(int64_t num_queries, int64_t num_keys, int clouds, int heads, int kv_heads, int size,
                                                   int is_bf16) {
    if (num_queries < 0 || num_keys < 0 || heads <= 0 || kv_heads <= 0 || size <= 0) return 256;
    const AttentionCall a = describe(num_queries, num_keys, clouds, heads, kv_heads, size, is_bf16, nullptr, nullptr, nullptr, nullptr,
                                     nullptr, nullptr, nullptr, nullptr, 1.f);
    const size_t sq = query_grad_splits(a), sk = key_grad_splits(a);
    const size_t pq = sq > 1 ? sq * num_queries * heads * size * 4 : 0, pk = sk > 1 ? 2 * sk * num_keys * kv_heads * size * 4 : 0;
    const size_t by_rows = align_up(pq > pk ? pq : pk), by_tiles = tc_grads_shape(a) ? tc_grads_workspace(a) : 0;
    return align_up((size_t)num_queries * heads * 4 + 256) + (by_rows > by_tiles ? by_rows : by_tiles);
}

int pccnn_cross_attention_grads(int64_t num_queries, int64_t num_keys, int clouds, int heads, int kv_heads, int size, int is_bf16,
                                const void* queries, const int64_t* query_strides_host, const void* keys,
                                const int64_t* key_strides_host, const void* values, const int64_t* value_strides_host,
                                const int32_t* query_ends, const int32_t* key_ends, float scale, const void* out, const float* lse,
                                const void* in_grads, const int64_t* grad_strides_host, void* out_query_grads, void* out_key_grads,
                                void* out_value_grads, void* workspace, size_t workspace_bytes, void* stream) {
    const AttentionCall a = describe(num_queries, num_keys, clouds, heads, kv_heads, size, is_bf16, queries, query_strides_host, keys,
                                     key_strides_host, values, value_strides_host, query_ends, key_ends, scale);
    if (int rc = check_call("cross_attention_grads", a)) return rc;
    PCCNN_CHECK_ARG(query_strides_host && key_strides_host && value_strides_host && grad_strides_host, "cross_attention_grads: null pointer");
    PCCNN_CHECK_ARG((num_queries == 0 || (out && lse && in_grads && out_query_grads)) && (num_keys == 0 || (out_key_grads && out_value_grads)),
                    "cross_attention_grads: null pointer");
    const size_t need = pccnn_cross_attention_grads_workspace_bytes(num_queries, num_keys, clouds, heads, kv_heads, size, is_bf16);
    if (!workspace || workspace_bytes < need) {
        set_error("cross_attention_grads: workspace of %zu bytes, need %zu", workspace_bytes, need);
        return PCCNN_ERR_WORKSPACE;
    }
    cudaStream_t s = (cudaStream_t)stream;
    if (int rc = take_sticky_status("cross_attention_grads")) return rc;
    const HeadRows grads = head_rows(in_grads, grad_strides_host, num_queries, heads, size);
    float* delta = (float*)workspace;
    char* rest = (char*)workspace + align_up((size_t)num_queries * heads * 4 + 256);
    if (num_queries > 0)
        if (int rc = launch_delta(a, out, grads, delta, s)) return rc;
    const bool outputs_aligned = aligned16(out_query_grads) && aligned16(out_key_grads) && aligned16(out_value_grads);
    if (num_queries > 0 && num_keys > 0 && tc_grads_shape(a) && tc_layout(a, &grads) && outputs_aligned)
        return tc_grads(a, grads, lse, delta, out_query_grads, out_key_grads, out_value_grads, rest, s);
    const BackwardRows b{a, grads, row_layout(a, &grads, outputs_aligned), lse, delta, out_query_grads, out_key_grads, out_value_grads, rest, s};
    return is_bf16 ? dispatch_rows<__nv_bfloat16>(b.l, b) : dispatch_rows<float>(b.l, b);
}

}  // extern "C"
