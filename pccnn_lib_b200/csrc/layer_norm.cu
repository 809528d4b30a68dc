// Layer norm over the channels of packed point features, forward and backward.
//
//   y = (x - mu) r w + b            mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps)
//   dx = r (g w - mean_c(g w) - xhat mean_c(g w xhat)),   dw = sum_n g xhat,   db = sum_n g,   xhat = (x - mu) r
//
// Both directions are bound by HBM: the forward pass reads x and writes y once, the backward pass reads x and g and writes dx
// once (500000 x 128 float: 78 us and 131 us, 102% and 91% of the measured copy bandwidth).  A row is held in the registers of TPR
// threads (a part of a warp, a warp, or a block), so the variance is taken around the finished mean without a second read.
// The backward kernel keeps the column sums of its rows in registers, every block writes one row of partial sums, and a
// second small kernel adds the blocks' rows in a fixed order: no atomics, the same bits on every run.  Statistics and sums are
// 32-bit floats whatever the features' type.  Rows of an odd number of bf16 channels are read two bytes at a time and are bound
// by instructions: 20011 x 1001 takes 31 us forward and 41 us backward, 2.6 and 2.9 TB/s.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "features.cuh"

namespace pccnn {

constexpr int kNormThreads = 256;

// Sums of R rows over the TPR consecutive threads that share them; every one of them gets the sums.  TPR = 256 uses shared
// memory and needs all threads of the block; consecutive calls alternate between the two halves of `slots`, so one barrier
// per call is enough.
template <int TPR, int R>
__device__ __forceinline__ void row_sums(float (&v)[R], float (*slots)[kNormThreads / 32][R]) {
    constexpr int kLanes = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < R; ++i) v[i] += __shfl_xor_sync(kFullMask, v[i], o);
    }
    if (TPR > 32) {
        if (lane_id() == 0) {
#pragma unroll
            for (int i = 0; i < R; ++i) (*slots)[threadIdx.x >> 5][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < R; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < kNormThreads / 32; ++w) v[i] += (*slots)[w][i];
        }
    }
}

// The E elements of a thread and row as pairs: one instruction works on two of them.  (With scalar arithmetic 200000 x 256
// bf16 took 44 us forward and 71% of the issue slots; so 34 us, 6.0 TB/s.)
template <int E>
struct Pairs {
    static constexpr int kN = (E + 1) / 2;
    unsigned long long w[kN];
    __device__ __forceinline__ void set(int e, float x) {  // element e (a constant after unrolling)
        float lo, hi;
        unpack_f32x2(w[e / 2], lo, hi);
        w[e / 2] = e % 2 ? pack_f32x2(lo, x) : pack_f32x2(x, hi);
    }
    __device__ __forceinline__ float get(int e) const {
        float lo, hi;
        unpack_f32x2(w[e / 2], lo, hi);
        return e % 2 ? hi : lo;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kN; ++i) w[i] = 0ull;
    }
};
__device__ __forceinline__ unsigned long long both(float x) { return pack_f32x2(x, x); }
__device__ __forceinline__ float sum_of(unsigned long long v) {
    float lo, hi;
    unpack_f32x2(v, lo, hi);
    return lo + hi;
}

// Vectors of V elements, K of them, into the pairs and back.
template <class T, int V, int K>
__device__ __forceinline__ void widen_row(const RawVec<T, V> (&raw)[K], Pairs<K * V>& x) {
    x.clear();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float f[V];
        raw[k].widen(f);
#pragma unroll
        for (int e = 0; e < V; ++e) x.set(k * V + e, f[e]);
    }
}
template <int V, int TPR, int K>
__device__ __forceinline__ void load_columns(const float* __restrict__ p, int t, int channels, Pairs<K * V>& x) {
    x.clear();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + t) * V;
        if (c < channels) {
            float f[V];
            load_vec<float, V>(p + c, f);
#pragma unroll
            for (int e = 0; e < V; ++e) x.set(k * V + e, f[e]);
        }
    }
}
template <class T, int V, int TPR, int K>
__device__ __forceinline__ void store_row(T* __restrict__ p, int t, int channels, const Pairs<K * V>& x) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + t) * V;
        if (c >= channels) break;
        float f[V];
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = x.get(k * V + e);
        store_vec<T, V>(p + c, f);
    }
}

// R rows per TPR threads at once, K vectors of V elements per thread and row.  The blocks are those resident at once and walk
// the rows; the next rows are on their way while the last ones are worked on.
template <class T, int V, int TPR, int K, int R>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_kernel(int64_t rows, int channels, const T* __restrict__ feats, int64_t ld, const float* __restrict__ weights,
                  const float* __restrict__ bias, float eps, T* __restrict__ out, float* __restrict__ out_mean,
                  float* __restrict__ out_rstd) {
    constexpr int kGroups = kNormThreads / TPR;
    using Row = Pairs<K * V>;
    __shared__ float slots[2][kNormThreads / 32][R];
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const int64_t stride = (int64_t)gridDim.x * kGroups * R;
    const bool ragged = channels < TPR * K * V;  // some elements of the threads lie behind the row
    const float inv = 1.f / (float)channels;
    RawVec<T, V> next[R][K];
    auto fetch = [&](int64_t row0) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * TPR + t) * V;
                if (row0 + i < rows && c < channels) next[i][k].load(feats + (row0 + i) * ld + c);
                else next[i][k].clear();
            }
    };
    fetch(((int64_t)blockIdx.x * kGroups + group) * R);
    constexpr bool kKeepColumns = K * V <= 4;  // weights and bias stay in registers where they are few
    Row w, b;
    if (kKeepColumns) {
        load_columns<V, TPR, K>(weights, t, channels, w);
        load_columns<V, TPR, K>(bias, t, channels, b);
    }
    for (int64_t base = (int64_t)blockIdx.x * kGroups * R; base < rows; base += stride) {  // the same for the block
        const int64_t row0 = base + group * R;
        Row x[R];
        float mean[R], rstd[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            widen_row<T, V, K>(next[i], x[i]);
            unsigned long long sum = x[i].w[0];
#pragma unroll
            for (int e = 1; e < Row::kN; ++e) sum = add_f32x2(sum, x[i].w[e]);
            mean[i] = sum_of(sum);
        }
        if (base + stride < rows) fetch(row0 + stride);
        row_sums<TPR, R>(mean, &slots[0]);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            mean[i] /= (float)channels;  // a division: the mean of equal values is that value wherever their sum is exact
            const unsigned long long m = both(mean[i]);
#pragma unroll
            for (int e = 0; e < Row::kN; ++e) x[i].w[e] = sub_f32x2(x[i].w[e], m);
            if (ragged) {
#pragma unroll
                for (int e = 0; e < K * V; ++e)
                    if (((e / V) * TPR + t) * V >= channels) x[i].set(e, 0.f);
            }
            if ((K * V) % 2) x[i].set(K * V, 0.f);
            unsigned long long sq = mul_f32x2(x[i].w[0], x[i].w[0]);
#pragma unroll
            for (int e = 1; e < Row::kN; ++e) sq = fma_f32x2(x[i].w[e], x[i].w[e], sq);
            rstd[i] = sum_of(sq);
        }
        row_sums<TPR, R>(rstd, &slots[1]);
        if (!kKeepColumns) {
            load_columns<V, TPR, K>(weights, t, channels, w);
            load_columns<V, TPR, K>(bias, t, channels, b);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            rstd[i] = rsqrtf(rstd[i] * inv + eps);
            if (row0 + i >= rows) break;
            if (t == 0) {
                out_mean[row0 + i] = mean[i];
                out_rstd[row0 + i] = rstd[i];
            }
            const unsigned long long r = both(rstd[i]);
#pragma unroll
            for (int e = 0; e < Row::kN; ++e) x[i].w[e] = fma_f32x2(mul_f32x2(x[i].w[e], r), w.w[e], b.w[e]);
            store_row<T, V, TPR, K>(out + (row0 + i) * channels, t, channels, x[i]);
        }
    }
}

// Sum over the block for the kernels of very wide rows.
__device__ __forceinline__ float block_sum(float v, float (*slots)[kNormThreads / 32][1]) {
    float s[1] = {v};
    row_sums<kNormThreads, 1>(s, slots);
    return s[0];
}

// Rows that do not fit the registers of a block: three passes over the row, which the first one leaves in the caches.
template <class T>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_wide_kernel(int channels, const T* __restrict__ feats, int64_t ld, const float* __restrict__ weights,
                       const float* __restrict__ bias, float eps, T* __restrict__ out, float* __restrict__ out_mean,
                       float* __restrict__ out_rstd) {
    __shared__ float slots[2][kNormThreads / 32][1];
    const int64_t row = blockIdx.x;
    const T* src = feats + row * ld;
    float sum = 0.f, sq = 0.f;
    for (int c = threadIdx.x; c < channels; c += kNormThreads) sum += to_float(src[c]);
    const float mean = block_sum(sum, &slots[0]) / (float)channels;
    for (int c = threadIdx.x; c < channels; c += kNormThreads) {
        const float d = to_float(src[c]) - mean;
        sq += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum(sq, &slots[1]) / (float)channels + eps);
    if (threadIdx.x == 0) {
        out_mean[row] = mean;
        out_rstd[row] = rstd;
    }
    for (int c = threadIdx.x; c < channels; c += kNormThreads)
        out[row * channels + c] = from_float<T>((to_float(src[c]) - mean) * rstd * weights[c] + bias[c]);
}

// Backward: the block's row groups walk the rows, R at a time, with a stride of the whole grid; column sums stay in registers
// and are added over the groups of the block, in ascending order, at the end.
template <class T, int V, int TPR, int K, int R>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_grads_kernel(int64_t rows, int channels, const T* __restrict__ feats, int64_t ld, const float* __restrict__ weights,
                        const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ grads,
                        int64_t ld_g, T* __restrict__ out, float* __restrict__ partial) {
    constexpr int kGroups = kNormThreads / TPR;
    extern __shared__ float sums[];  // [2][channels], where several rows share a block (at most 1024 channels: 8 KB)
    __shared__ float slots[2][kNormThreads / 32][2 * R];
    using Row = Pairs<K * V>;
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    Row w, dw, db;
    load_columns<V, TPR, K>(weights, t, channels, w);
    dw.clear();
    db.clear();
    const float inv = 1.f / (float)channels;
    const int64_t stride = (int64_t)gridDim.x * kGroups * R;
    RawVec<T, V> next_x[R][K], next_g[R][K];
    float next_mu[R], next_r[R];
    const bool ragged = channels < TPR * K * V;  // some elements of the threads lie behind the row
    auto fetch = [&](int64_t row0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool live = row0 + i < rows;  // every thread of the warp stays for the shuffles
            next_mu[i] = live ? mean[row0 + i] : 0.f;
            next_r[i] = live ? rstd[row0 + i] : 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * TPR + t) * V;
                if (live && c < channels) {
                    next_x[i][k].load(feats + (row0 + i) * ld + c);
                    next_g[i][k].load(grads + (row0 + i) * ld_g + c);
                } else {
                    next_x[i][k].clear();
                    next_g[i][k].clear();
                }
            }
        }
    };
    fetch(((int64_t)blockIdx.x * kGroups + group) * R);
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * kGroups * R; base < rows; base += stride, turn ^= 1) {
        const int64_t row0 = base + group * R;
        Row x[R], g[R];
        float r[R], s[2 * R];
        unsigned long long mu[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            mu[i] = both(next_mu[i]);
            r[i] = next_r[i];
            widen_row<T, V, K>(next_x[i], x[i]);
            widen_row<T, V, K>(next_g[i], g[i]);
            // behind the row x becomes the mean: (0 - mean) rstd may overflow, and an infinity times the zero gradient there would
            // reach the row's sums
            if (ragged) {
#pragma unroll
                for (int e = 0; e < K * V; ++e)
                    if (((e / V) * TPR + t) * V >= channels) x[i].set(e, next_mu[i]);
            }
            if ((K * V) % 2) x[i].set(K * V, next_mu[i]);
        }
        if (base + stride < rows) fetch(row0 + stride);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const unsigned long long rr = both(r[i]);
            unsigned long long s1 = 0ull, s2 = 0ull;
#pragma unroll
            for (int e = 0; e < Row::kN; ++e) {
                const unsigned long long hat = mul_f32x2(sub_f32x2(x[i].w[e], mu[i]), rr);
                dw.w[e] = fma_f32x2(g[i].w[e], hat, dw.w[e]);
                db.w[e] = add_f32x2(db.w[e], g[i].w[e]);
                x[i].w[e] = hat;
                g[i].w[e] = mul_f32x2(g[i].w[e], w.w[e]);
                s1 = add_f32x2(s1, g[i].w[e]);
                s2 = fma_f32x2(g[i].w[e], hat, s2);
            }
            s[2 * i] = sum_of(s1);
            s[2 * i + 1] = sum_of(s2);
        }
        row_sums<TPR, 2 * R>(s, &slots[turn]);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (row0 + i >= rows) break;
            const unsigned long long s1 = both(-s[2 * i] * inv), s2 = both(-s[2 * i + 1] * inv), rr = both(r[i]);
#pragma unroll
            for (int e = 0; e < Row::kN; ++e) x[i].w[e] = mul_f32x2(rr, fma_f32x2(x[i].w[e], s2, add_f32x2(g[i].w[e], s1)));
            store_row<T, V, TPR, K>(out + (row0 + i) * channels, t, channels, x[i]);
        }
    }
    float* dst = partial + (int64_t)blockIdx.x * 2 * channels;
    if constexpr (kGroups == 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * TPR + t) * V;
            if (c >= channels) break;
#pragma unroll
            for (int e = 0; e < V; ++e) dst[c + e] = dw.get(k * V + e), dst[channels + c + e] = db.get(k * V + e);
        }
    } else {
        for (int g = 0; g < kGroups; ++g) {
            if (group == g) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int c = (k * TPR + t) * V + e;
                        if (c < channels) {
                            sums[c] = g ? sums[c] + dw.get(k * V + e) : dw.get(k * V + e);
                            sums[channels + c] = g ? sums[channels + c] + db.get(k * V + e) : db.get(k * V + e);
                        }
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * channels; c += kNormThreads) dst[c] = sums[c];
    }
}

// Rows too wide for the registers: the block's row of partial sums is its accumulator.
template <class T>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_grads_wide_kernel(int64_t rows, int channels, const T* __restrict__ feats, int64_t ld,
                             const float* __restrict__ weights, const float* __restrict__ mean, const float* __restrict__ rstd,
                             const T* __restrict__ grads, int64_t ld_g, T* __restrict__ out, float* __restrict__ partial) {
    __shared__ float slots[2][kNormThreads / 32][1];
    float* dw = partial + (int64_t)blockIdx.x * 2 * channels;
    float* db = dw + channels;
    for (int c = threadIdx.x; c < channels; c += kNormThreads) dw[c] = db[c] = 0.f;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float mu = mean[row], r = rstd[row];
        const T *x = feats + row * ld, *g = grads + row * ld_g;
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < channels; c += kNormThreads) {
            const float hat = (to_float(x[c]) - mu) * r, gr = to_float(g[c]);
            dw[c] += gr * hat;  // a column belongs to one thread
            db[c] += gr;
            s1 += gr * weights[c];
            s2 += gr * weights[c] * hat;
        }
        s1 = block_sum(s1, &slots[0]) / (float)channels;
        s2 = block_sum(s2, &slots[1]) / (float)channels;
        for (int c = threadIdx.x; c < channels; c += kNormThreads) {
            const float hat = (to_float(x[c]) - mu) * r;
            out[row * channels + c] = from_float<T>(r * (to_float(g[c]) * weights[c] - s1 - hat * s2));
        }
    }
}

// Column sums of the blocks' rows: 32 columns x 32 row strides per block, added in a fixed order.
__global__ void __launch_bounds__(1024)
column_sums_kernel(int num_rows, int columns, const float* __restrict__ partial, int channels, float* __restrict__ weight_grads,
                   float* __restrict__ bias_grads) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float sum = 0.f;
    if (c < columns) {
#pragma unroll 8
        for (int r = slice; r < num_rows; r += 32) sum += partial[(int64_t)r * columns + c];
    }
    part[slice][lane] = sum;
    __syncthreads();
    sum = warp_sum(part[lane][slice]);  // warp s adds column s
    const int column = blockIdx.x * 32 + slice;
    if (lane == 0 && column < columns) {
        if (column < channels) weight_grads[column] = sum;
        else bias_grads[column - channels] = sum;
    }
}

constexpr int kNormMaxBlocksPerSm = 8;

// Blocks: what is resident at once (in the backward pass every block writes a row of partial sums), at most the rows' share.
template <class Kernel>
static int norm_blocks(Kernel kernel, size_t shared, int64_t rows, int rows_per_block) {
    const int64_t need = (rows + rows_per_block - 1) / rows_per_block;
    if (need <= sm_count()) return (int)(need < 1 ? 1 : need);
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kNormThreads, shared) != cudaSuccess || per_sm < 1) per_sm = 1;
    if (per_sm > kNormMaxBlocksPerSm) per_sm = kNormMaxBlocksPerSm;
    const int64_t cap = (int64_t)sm_count() * per_sm;
    return (int)(need < cap ? need : cap);
}

// Threads per row, vectors per thread and rows at once for rows of n vectors of V elements: few threads per row while that
// keeps it to a few vectors each, and then as many rows at once as keep 32 to 64 bytes of a thread in flight.  (A detour of
// unaligned rows through shared memory with 16-byte accesses was no faster: 20011 x 1001 bf16 36 us forward, 81 us backward,
// against 41 and 40 us.)
template <class T, int V, class Launch>
static int dispatch_rows_of(int n, const Launch& launch) {
    if constexpr (V * sizeof(T) >= 8) {
        if (n <= 8) return launch.template run<T, V, 8, 1, 4>();
        if (n <= 16) return launch.template run<T, V, 8, 2, 2>();
        if (n <= 32) return launch.template run<T, V, 32, 1, Launch::template warp_rows<T>()>();
        if (n <= 64) return launch.template run<T, V, 32, 2, 2>();
        if (n <= 128) return launch.template run<T, V, 32, 4, 1>();
        if (n <= 256) return launch.template run<T, V, 256, 1, 4>();
        if (n <= 1024) return launch.template run<T, V, 256, 4, 1>();
    } else {
        if (n <= 8) return launch.template run<T, V, 8, 1, 8>();
        if (n <= 16) return launch.template run<T, V, 8, 2, 4>();
        if (n <= 32) return launch.template run<T, V, 8, 4, 4>();
        if (n <= 64) return launch.template run<T, V, 32, 2, 4>();
        if (n <= 128) return launch.template run<T, V, 32, 4, 4>();
        if (n <= 256) return launch.template run<T, V, 32, 8, 2>();
        if (n <= 512) return launch.template run<T, V, 32, 16, 1>();
        if (n <= 1024) return launch.template run<T, V, 256, 4, 1>();
        if (n <= 4096) return launch.template run<T, V, 256, 16, 1>();
    }
    return launch.template wide<T>();
}
// `width`: the most elements of one access that every row of every tensor is aligned to.
template <class T, class Launch>
static int dispatch_norm(int channels, int width, const Launch& launch) {
    if constexpr (sizeof(T) == 2) {
        if (width >= 8) return dispatch_rows_of<T, 8>(channels / 8, launch);
    }
    if (width >= 4) return dispatch_rows_of<T, 4>(channels / 4, launch);
    if (width >= 2) return dispatch_rows_of<T, 2>(channels / 2, launch);
    return dispatch_rows_of<T, 1>(channels, launch);
}
// The largest power of two (at most 16 bytes) that divides the channels and the row stride and fits the address.
static int row_width(const void* p, int64_t ld, int channels, int element) {
    int v = 16 / element;
    while (v > 1 && (channels % v || ld % v || ((uintptr_t)p & (v * element - 1)))) v /= 2;
    return v;
}

// The same for float columns: 16-byte alignment serves vectors of 8 elements as well (two accesses).
static int column_width(const float* p, int channels) {
    const int v = row_width(p, channels, channels, 4);
    return v == 4 ? 8 : v;
}

struct NormForward {
    int64_t rows; int channels; const void* feats; int64_t ld; const float *weights, *bias; float eps;
    void* out; float *mean, *rstd; cudaStream_t s;
    // Rows at once of a warp with one vector per lane: three 32-bit ones (500000 x 128 78 us, 100000 x 128 16.6 us; with four
    // 90 and 17.7 us, with two 77 and 15.8 us, but 500001 x 100 69 against 66 us), four bf16 ones (200000 x 256 34.6 us;
    // with three 42.6, with two 39.0 us).
    template <class T> static constexpr int warp_rows() { return sizeof(T) == 4 ? 3 : 4; }
    template <class T, int V, int TPR, int K, int R> int run() const {
        const int blocks = norm_blocks(layer_norm_kernel<T, V, TPR, K, R>, 0, rows, kNormThreads / TPR * R);
        layer_norm_kernel<T, V, TPR, K, R><<<blocks, kNormThreads, 0, s>>>(rows, channels, (const T*)feats, ld, weights, bias,
                                                                                 eps, (T*)out, mean, rstd);
        PCCNN_LAUNCH_CHECK();
        return PCCNN_OK;
    }
    template <class T> int wide() const {
        layer_norm_wide_kernel<T><<<(unsigned)rows, kNormThreads, 0, s>>>(channels, (const T*)feats, ld, weights, bias, eps, (T*)out,
                                                                         mean, rstd);
        PCCNN_LAUNCH_CHECK();
        return PCCNN_OK;
    }
};

struct NormBackward {
    int64_t rows; int channels; const void* feats; int64_t ld; const float *weights, *mean, *rstd; const void* grads;
    int64_t ld_g; void* out; float *weight_grads, *bias_grads, *partial; cudaStream_t s;
    // Four of either type: 500001 x 100 float 100 us, 700000 x 96 132 us, 500000 x 128 131 us; with three 105, 141 and 121 us.
    template <class T> static constexpr int warp_rows() { return 4; }
    int sums(int blocks) const {
        column_sums_kernel<<<(2 * channels + 31) / 32, 1024, 0, s>>>(blocks, 2 * channels, partial, channels, weight_grads, bias_grads);
        PCCNN_LAUNCH_CHECK();
        return PCCNN_OK;
    }
    template <class T, int V, int TPR, int K, int R> int run() const {
        const size_t shared = TPR < kNormThreads ? (size_t)2 * channels * 4 : 0;
        const int blocks = norm_blocks(layer_norm_grads_kernel<T, V, TPR, K, R>, shared, rows, kNormThreads / TPR * R);
        layer_norm_grads_kernel<T, V, TPR, K, R><<<blocks, kNormThreads, shared, s>>>(
            rows, channels, (const T*)feats, ld, weights, mean, rstd, (const T*)grads, ld_g, (T*)out, partial);
        PCCNN_LAUNCH_CHECK();
        return sums(blocks);
    }
    template <class T> int wide() const {
        const int blocks = norm_blocks(layer_norm_grads_wide_kernel<T>, 0, rows, 1);
        layer_norm_grads_wide_kernel<T><<<blocks, kNormThreads, 0, s>>>(rows, channels, (const T*)feats, ld, weights, mean, rstd,
                                                                       (const T*)grads, ld_g, (T*)out, partial);
        PCCNN_LAUNCH_CHECK();
        return sums(blocks);
    }
};

}  // namespace pccnn

using namespace pccnn;

extern "C" {

int pccnn_layer_norm(int64_t rows, int channels, const void* feats, int64_t ld_feats, int is_bf16, const float* weights,
                     const float* bias, float eps, void* out, float* out_mean, float* out_rstd, void* stream) {
    PCCNN_CHECK_ARG(rows >= 0 && rows < 0x7fffffffLL && channels > 0 && channels <= (1 << 20),
                    "layer_norm: bad shape (%lld rows of %d channels)", (long long)rows, channels);
    PCCNN_CHECK_ARG(ld_feats >= channels || rows <= 1, "layer_norm: row stride %lld below the %d channels", (long long)ld_feats, channels);
    PCCNN_CHECK_ARG(eps >= 0.f, "layer_norm: eps must not be negative");
    if (rows == 0) return PCCNN_OK;
    PCCNN_CHECK_ARG(feats && weights && bias && out && out_mean && out_rstd, "layer_norm: null pointer");
    const NormForward f{rows, channels, feats, ld_feats, weights, bias, eps, out, out_mean, out_rstd, (cudaStream_t)stream};
    const int e = is_bf16 ? 2 : 4;
    const int width = std::min({row_width(feats, rows > 1 ? ld_feats : channels, channels, e), row_width(out, channels, channels, e),
                                column_width(weights, channels), column_width(bias, channels)});
    return is_bf16 ? dispatch_norm<__nv_bfloat16>(channels, width, f) : dispatch_norm<float>(channels, width, f);
}

size_t pccnn_layer_norm_grads_workspace_bytes(int64_t rows, int channels) {
    if (rows < 0 || channels <= 0) return 256;
    const int64_t cap = (int64_t)sm_count() * kNormMaxBlocksPerSm, blocks = rows < cap ? (rows > 0 ? rows : 1) : cap;
    return align_up((size_t)blocks * 2 * channels * 4);
}

int pccnn_layer_norm_grads(int64_t rows, int channels, const void* feats, int64_t ld_feats, int is_bf16, const float* weights,
                           const float* mean, const float* rstd, const void* in_grads, int64_t ld_grads, void* out_feat_grads,
                           float* out_weight_grads, float* out_bias_grads, void* workspace, size_t workspace_bytes, void* stream) {
    PCCNN_CHECK_ARG(rows >= 0 && rows < 0x7fffffffLL && channels > 0 && channels <= (1 << 20),
                    "layer_norm_grads: bad shape (%lld rows of %d channels)", (long long)rows, channels);
    PCCNN_CHECK_ARG((ld_feats >= channels && ld_grads >= channels) || rows <= 1, "layer_norm_grads: row strides below the %d channels",
                    channels);
    PCCNN_CHECK_ARG(out_weight_grads && out_bias_grads, "layer_norm_grads: null pointer");
    cudaStream_t s = (cudaStream_t)stream;
    if (rows == 0) {
        PCCNN_CUDA(cudaMemsetAsync(out_weight_grads, 0, (size_t)channels * 4, s));
        PCCNN_CUDA(cudaMemsetAsync(out_bias_grads, 0, (size_t)channels * 4, s));
        return PCCNN_OK;
    }
    PCCNN_CHECK_ARG(feats && weights && mean && rstd && in_grads && out_feat_grads, "layer_norm_grads: null pointer");
    if (!workspace || workspace_bytes < pccnn_layer_norm_grads_workspace_bytes(rows, channels)) {
        set_error("layer_norm_grads: workspace of %zu bytes, need %zu", workspace_bytes,
                  pccnn_layer_norm_grads_workspace_bytes(rows, channels));
        return PCCNN_ERR_WORKSPACE;
    }
    const NormBackward b{rows, channels, feats, ld_feats, weights, mean, rstd, in_grads, ld_grads, out_feat_grads,
                         out_weight_grads, out_bias_grads, (float*)workspace, s};
    const int e = is_bf16 ? 2 : 4;
    const int width = std::min({row_width(feats, rows > 1 ? ld_feats : channels, channels, e), row_width(out_feat_grads, channels, channels, e),
                                row_width(in_grads, rows > 1 ? ld_grads : channels, channels, e),
                                column_width(weights, channels)});
    return is_bf16 ? dispatch_norm<__nv_bfloat16>(channels, width, b) : dispatch_norm<float>(channels, width, b);
}

}  // extern "C"
