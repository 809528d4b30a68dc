// Rotary positions with several axes: pairs of a head's features are turned by angles that grow with the coordinates of
// the row's point.  Pair j of axis a: (x0, x1) -> (x0 cos t - x1 sin t, x0 sin t + x1 cos t), t = pts[n, a] f_j.  The first
// axis_pairs[0] pairs belong to axis 0, the next axis_pairs[1] to axis 1, and so on; features behind the last pair pass.
//
//   dx = the gradient turned by -t;      dpts[n, a] = sum_{j of a} f_j sum_h (g1 y0 - g0 y1),  y = the turned features
//
// Both directions are bound by HBM (150000 x 8 x 64 float, 30 pairs: 102 us forward, 170 us backward with the coordinates' gradient,
// 93% and 84% of the measured copy bandwidth).  The angle of a far position has no correct digit left in 32 bits, so the product (exact
// in 64 bits: 24 + 24 bits) and its reduction to a fraction of a turn are 64-bit, once per (row, pair) and not per head; the
// fraction is at most half a turn and its sine and cosine are taken in 32 bits.  A row belongs to 4 to 32 lanes of one warp,
// which compute the row's angles into shared memory and then walk its heads; the coordinates' gradient is a sum over
// those lanes in a fixed order.
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "features.cuh"

namespace pccnn {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryMaxSize = 1024;

struct RotaryAxes {
    int count;
    int last[kMaxDims];  // pairs of the axes up to and including this one
};

struct RotaryRows {
    int64_t row, head;  // strides in elements
};

__device__ __forceinline__ float2 turn_of(float coordinate, float frequency) {
    const double turns = (double)coordinate * (double)frequency * 0.15915494309189533577;  // 1 / (2 pi)
    float2 cs;
    sincospif((float)(2.0 * (turns - rint(turns))), &cs.y, &cs.x);
    return cs;
}

__device__ __forceinline__ int axis_of(const RotaryAxes& axes, int pair) {
    int a = 0;
#pragma unroll
    for (int i = 0; i < kMaxDims - 1; ++i) a += (i + 1 < axes.count && pair >= axes.last[i]) ? 1 : 0;
    return a;
}

// P > 1: one aligned access.  P = 1: two elements, of which the second may be absent (an odd head size).
template <class T, int P>
__device__ __forceinline__ void load_pairs(const T* __restrict__ p, bool whole, float (&x)[2 * P]) {
    if constexpr (P > 1) {
        load_vec<T, 2 * P>(p, x);
    } else {
        x[0] = to_float(p[0]);
        x[1] = whole ? to_float(p[1]) : 0.f;
    }
}

// P pairs per access, kAtOnce accesses of a lane in flight.  kAxes > 0: `in` is the gradient, turned back, and the
// coordinates' gradient (of at most kAxes axes) is taken from it and `feats` when pt_grads is given.
template <class T, int P, int kAxes>
__global__ void __launch_bounds__(kRotaryThreads)
rotary_kernel(int64_t rows, int heads, int size, const T* __restrict__ in, RotaryRows ld_in, const T* __restrict__ feats,
              RotaryRows ld_feats, const float* __restrict__ pts, const float* __restrict__ frequencies, RotaryAxes axes,
              int lanes_per_row, T* __restrict__ out, float* __restrict__ pt_grads) {
    constexpr bool kGrads = kAxes > 0;
    constexpr int kSums = kGrads ? kAxes : 1, kAtOnce = 4;
    extern __shared__ float2 table[];  // [pairs] (frequency, axis), then [rows of the block][pairs] (cosine, sine)
    const int pairs = axes.last[axes.count - 1];
    const int rows_per_block = kRotaryThreads / lanes_per_row;
    const int slot = threadIdx.x / lanes_per_row, lane = threadIdx.x % lanes_per_row;
    float2* cs = table + (1 + slot) * pairs;
    for (int j = threadIdx.x; j < pairs; j += kRotaryThreads) table[j] = make_float2(frequencies[j], __int_as_float(axis_of(axes, j)));
    __syncthreads();
    const int accesses = (size + 2 * P - 1) / (2 * P), total = heads * accesses;
    const bool both = kGrads && pt_grads;
    for (int64_t base = (int64_t)blockIdx.x * rows_per_block; base < rows; base += (int64_t)gridDim.x * rows_per_block) {
        const int64_t row = base + slot;
        const bool live = row < rows;
        float sum[kSums];
#pragma unroll
        for (int a = 0; a < kSums; ++a) sum[a] = 0.f;
        for (int first = 0; first < total; first += kAtOnce * lanes_per_row) {  // the same for the lanes of a warp
            float x[kAtOnce][2 * P], f[kGrads ? kAtOnce : 1][2 * P];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int i = first + u * lanes_per_row + lane;
                if (live && i < total) {
                    const int h = i / accesses, d = (i - h * accesses) * 2 * P;
                    const T* src = in + row * ld_in.row + h * ld_in.head + d;
                    const bool whole = P > 1 || d + 1 < size;  // P > 1: the size is a multiple of the access
                    load_pairs<T, P>(src, whole, x[u]);
                    if constexpr (kGrads) {
                        if (both) load_pairs<T, P>(feats + row * ld_feats.row + h * ld_feats.head + d, whole, f[u]);
                    }
                }
            }
            if (first == 0) {  // the row's angles, while its features are on their way
                if (live)
                    for (int j = lane; j < pairs; j += lanes_per_row) {
                        const float2 fa = table[j];
                        cs[j] = turn_of(pts[row * axes.count + __float_as_int(fa.y)], fa.x);
                    }
                __syncwarp();
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int i = first + u * lanes_per_row + lane;
                if (live && i < total) {
                    const int h = i / accesses, d = (i - h * accesses) * 2 * P;
                    T* dst = out + ((int64_t)row * heads + h) * size + d;
                    float y[2 * P];
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const int j = d / 2 + p;
                        const float x0 = x[u][2 * p], x1 = x[u][2 * p + 1];
                        y[2 * p] = x0;  // a pair that is not turned passes as it is, infinities included
                        y[2 * p + 1] = x1;
                        if (j < pairs) {
                            const float2 t = cs[j];
                            const float s = kGrads ? -t.y : t.y;
                            y[2 * p] = x0 * t.x - x1 * s;
                            y[2 * p + 1] = x0 * s + x1 * t.x;
                            if constexpr (kGrads) {
                                if (both) {
                                    const float2 fa = table[j];
                                    const float f0 = f[u][2 * p], f1 = f[u][2 * p + 1];
                                    const float term = (x1 * (f0 * t.x - f1 * t.y) - x0 * (f0 * t.y + f1 * t.x)) * fa.x;
#pragma unroll
                                    for (int a = 0; a < kSums; ++a) sum[a] += __float_as_int(fa.y) == a ? term : 0.f;
                                }
                            }
                        }
                    }
                    if constexpr (P > 1) {
                        store_vec<T, 2 * P>(dst, y);
                    } else {
                        dst[0] = from_float<T>(y[0]);
                        if (d + 1 < size) dst[1] = from_float<T>(y[1]);
                    }
                }
            }
        }
        if constexpr (kGrads) {
            if (both) {
#pragma unroll
                for (int a = 0; a < kSums; ++a) {
                    if (a >= axes.count) break;
                    float v = sum[a];
                    for (int o = lanes_per_row / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
                    if (live && lane == 0) pt_grads[row * axes.count + a] = v;
                }
            }
        }
        __syncwarp();  // the table is rewritten for the next row
    }
}

template <class T, int P, int kAxes>
static int launch_rotary(int64_t rows, int heads, int size, const void* in, RotaryRows ld_in, const void* feats, RotaryRows ld_feats,
                         const float* pts, const float* frequencies, const RotaryAxes& axes, void* out, float* pt_grads,
                         cudaStream_t s) {
    const int total = heads * ((size + 2 * P - 1) / (2 * P));
    int lanes = 4;
    while (lanes < 32 && lanes < total) lanes *= 2;
    const int pairs = axes.last[axes.count - 1];
    // the tables stay within 48 KB of shared memory: (1 + 8 rows) of 512 pairs are 36 KB
    while (lanes < 32 && (size_t)(1 + kRotaryThreads / lanes) * pairs * sizeof(float2) > 48 * 1024) lanes *= 2;
    const int per_block = kRotaryThreads / lanes;
    const size_t smem = (size_t)(1 + per_block) * pairs * sizeof(float2);
    const int64_t blocks = (rows + per_block - 1) / per_block, cap = (int64_t)sm_count() * 32;
    rotary_kernel<T, P, kAxes><<<(unsigned)(blocks < cap ? blocks : cap), kRotaryThreads, smem, s>>>(
        rows, heads, size, (const T*)in, ld_in, (const T*)feats, ld_feats, pts, frequencies, axes, lanes, (T*)out, pt_grads);
    PCCNN_LAUNCH_CHECK();
    return PCCNN_OK;
}

static bool vector_rows(const void* p, RotaryRows ld, int v) { return aligned16(p) && ld.row % v == 0 && ld.head % v == 0; }

template <bool kGrads>
static int rotary(const char* who, int64_t rows, int heads, int size, const void* in, RotaryRows ld_in, const void* feats,
                  RotaryRows ld_feats, int is_bf16, int num_axes, const float* pts, const float* frequencies,
                  const int32_t* axis_pairs_host, void* out, float* pt_grads, cudaStream_t s) {
    PCCNN_CHECK_ARG(rows >= 0 && rows < 0x7fffffffLL && heads > 0 && heads <= 65535 && size > 0 && size <= kRotaryMaxSize,
                    "%s: bad shape (%lld rows, %d heads of %d; a head has at most %d)", who, (long long)rows, heads, size, kRotaryMaxSize);
    PCCNN_CHECK_ARG(num_axes >= 1 && num_axes <= kMaxDims, "%s: %d axes, 1 to %d are supported", who, num_axes, kMaxDims);
    PCCNN_CHECK_ARG(axis_pairs_host, "%s: null pointer", who);
    RotaryAxes axes;
    axes.count = num_axes;
    int pairs = 0;
    for (int a = 0; a < num_axes; ++a) {
        PCCNN_CHECK_ARG(axis_pairs_host[a] >= 0 && axis_pairs_host[a] <= size / 2, "%s: axis %d has %d pairs of a head's %d", who, a,
                        axis_pairs_host[a], size / 2);
        pairs += axis_pairs_host[a];
        axes.last[a] = pairs;
    }
    for (int a = num_axes; a < kMaxDims; ++a) axes.last[a] = pairs;
    PCCNN_CHECK_ARG(pairs <= size / 2, "%s: %d pairs in all do not fit a head of %d", who, pairs, size);
    if (rows == 0) return PCCNN_OK;
    PCCNN_CHECK_ARG(in && pts && out && (frequencies || pairs == 0) && (!pt_grads || feats), "%s: null pointer", who);
    const int v = is_bf16 ? 8 : 4;
    const bool vec = size % v == 0 && vector_rows(in, ld_in, v) && aligned16(out) && (!pt_grads || vector_rows(feats, ld_feats, v));
    // the sums over the axes are unrolled for three of them, the usual case, or for all six
    auto launch = [&](auto type, auto pairs_at_once) {
        using T = decltype(type);
        constexpr int kP = decltype(pairs_at_once)::value;
        if constexpr (kGrads) {
            if (num_axes <= 3) return launch_rotary<T, kP, 3>(rows, heads, size, in, ld_in, feats, ld_feats, pts, frequencies, axes, out, pt_grads, s);
            return launch_rotary<T, kP, kMaxDims>(rows, heads, size, in, ld_in, feats, ld_feats, pts, frequencies, axes, out, pt_grads, s);
        } else {
            return launch_rotary<T, kP, 0>(rows, heads, size, in, ld_in, feats, ld_feats, pts, frequencies, axes, out, pt_grads, s);
        }
    };
    if (is_bf16) return vec ? launch(__nv_bfloat16(), std::integral_constant<int, 4>()) : launch(__nv_bfloat16(), std::integral_constant<int, 1>());
    return vec ? launch(0.f, std::integral_constant<int, 2>()) : launch(0.f, std::integral_constant<int, 1>());
}

}  // namespace pccnn

using namespace pccnn;

extern "C" {

int pccnn_rotary_positions(int64_t rows, int heads, int size, const void* feats, int64_t row_stride, int64_t head_stride,
                           int is_bf16, int num_axes, const float* pts, const float* frequencies, const int32_t* axis_pairs_host,
                           void* out, void* stream) {
    return rotary<false>("rotary_positions", rows, heads, size, feats, {row_stride, head_stride}, nullptr, {0, 0}, is_bf16,
                         num_axes, pts, frequencies, axis_pairs_host, out, nullptr, (cudaStream_t)stream);
}

int pccnn_rotary_positions_grads(int64_t rows, int heads, int size, const void* feats, int64_t row_stride, int64_t head_stride,
                                 int is_bf16, int num_axes, const float* pts, const float* frequencies,
                                 const int32_t* axis_pairs_host, const void* in_grads, int64_t grad_row_stride,
                                 int64_t grad_head_stride, void* out_feat_grads, float* out_pt_grads, void* stream) {
    return rotary<true>("rotary_positions_grads", rows, heads, size, in_grads, {grad_row_stride, grad_head_stride}, feats,
                        {row_stride, head_stride}, is_bf16, num_axes, pts, frequencies, axis_pairs_host, out_feat_grads,
                        out_pt_grads, (cudaStream_t)stream);
}

}  // extern "C"
