// What the kernels of cross attention on packed clouds share: the description of a call, the rows of a cloud, and the
// launchers that attention.cu chooses from.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace pccnn {

// [rows, heads, size] with any row and head stride (in elements) and contiguous features.
struct HeadRows {
    const void* data;
    int64_t row, head;
};

struct AttentionCall {
    int64_t num_queries, num_keys;
    int clouds, heads, kv_heads, size, is_bf16;
    HeadRows q, k, v;
    const int32_t *query_ends, *key_ends;
    float scale;
};

constexpr int kMaxSplits = 128;

// Whether the row kernel of the forward pass takes its logits from products of 16 keys (bf16).
bool use_products(const AttentionCall& a);

// Tensor-core kernels (attention_tc.cu).  Whether a call may use them goes by its shape (tc_shape: the workspace does not
// depend on anything else) and then by the layout of its tensors (tc_layout).
bool tc_shape(const AttentionCall& a);
bool tc_layout(const AttentionCall& a, const HeadRows* grads);
size_t tc_forward_workspace(const AttentionCall& a);
int tc_forward(const AttentionCall& a, void* out, float* lse, char* ws, cudaStream_t s);

bool tc_grads_shape(const AttentionCall& a);
size_t tc_grads_workspace(const AttentionCall& a);
int tc_grads(const AttentionCall& a, const HeadRows& grads, const float* lse, float* delta, void* dq, void* dk, void* dv, char* ws,
             cudaStream_t s);

// out = the sum of the splits' parts [splits, count].
int add_splits(int is_bf16, int64_t count, int splits, const float* part, void* out, cudaStream_t s);
// Joins the splits of every query: part_out [splits, queries, heads, size] relative to part_stat's (maximum in log2 units, sum).
int join_splits(const AttentionCall& a, int splits, const float* part_out, const float2* part_stat, void* out, float* lse, cudaStream_t s);

#ifdef __CUDACC__

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 2^x as the hardware computes it (relative error 2^-22, subnormal results become zero).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Rows of cloud b: [begin, end).  Whatever the end offsets hold, the range lies inside [0, n).  Cloud `clouds` is
// the rest: rows behind the last cloud.
__device__ __forceinline__ int64_t cloud_begin(const int32_t* __restrict__ ends, int b, int64_t n) {
    const int64_t e = b > 0 ? (int64_t)ends[b - 1] : 0;
    return e < 0 ? 0 : e < n ? e : n;
}
__device__ __forceinline__ int64_t cloud_end(const int32_t* __restrict__ ends, int b, int clouds, int64_t n) {
    if (b >= clouds) return n;
    const int64_t lo = cloud_begin(ends, b, n), e = (int64_t)ends[b];
    return e < lo ? lo : e < n ? e : n;
}

// First cloud whose end lies behind `row` (`clouds`: none).
__device__ __forceinline__ int cloud_of_row(const int32_t* __restrict__ ends, int clouds, int64_t row) {
    int lo = 0, hi = clouds;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)ends[mid] > row) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

#endif  // __CUDACC__

}  // namespace pccnn
