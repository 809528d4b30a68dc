// Host side of the tensor-core kernels of cross attention (attention_tc.cuh), and the kernel that brings 32-bit features into
// three bf16 planes.
#include <cuda.h>

#include <atomic>

#include "attention_tc.cuh"
#include "status.cuh"

namespace pccnn {

uint32_t tensor_core_poll_limit();
int tensor_core_withhold_from();
int make_heads_map(CUtensorMap* map, const void* base, int64_t rows, int heads, int size, int64_t row_stride, int64_t head_stride,
                   int box_rows);

// Dynamic shared memory above 48 KB has to be asked for once per kernel and device.
template <class Kernel>
static int allow_shared(Kernel kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    PCCNN_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load() & bit)) {
        PCCNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.fetch_or(bit);
    }
    return PCCNN_OK;
}

// x -> (h, m, l): planes [3][rows, heads, size] of bf16.  size is a multiple of 8; one thread per 8 features.
__global__ void __launch_bounds__(256)
split_planes_kernel(int64_t rows, int heads, int size, const float* __restrict__ src, int64_t row_stride, int64_t head_stride, bool vectors,
                    __nv_bfloat16* __restrict__ planes) {
    const int per_head = size / 8, per_row = heads * per_head;
    const int64_t total = rows * per_row, plane = rows * heads * size;
    for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per_row;
        const int in_row = (int)(i - r * per_row), h = in_row / per_head, c = (in_row - h * per_head) * 8;
        const float* p = src + r * row_stride + h * head_stride + c;
        float x[8];
        if (vectors) {
            load_vec<float, 8>(p, x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = p[e];
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
                x[2 * e] -= __uint_as_float(w[e] << 16);
                x[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
            }
            *reinterpret_cast<uint4*>(planes + k * plane + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// A tensor of heads as the kernels read it: its own data in bf16, or its three planes in the workspace.
struct TcOperand {
    TcRows rows;
    int64_t count;  // rows of one plane
    int heads;
};

static int tc_operand(TcOperand& o, const HeadRows& x, int64_t rows, int heads, int size, bool planes, char*& ws, cudaStream_t s) {
    o.count = rows;
    o.heads = heads;
    if (!planes) {
        o.rows = {(const __nv_bfloat16*)x.data, x.row, x.head, 0};
        return PCCNN_OK;
    }
    const int64_t plane = rows * heads * size;
    o.rows = {(const __nv_bfloat16*)ws, (int64_t)heads * size, size, plane};
    const bool vectors = aligned16(x.data) && x.row % 4 == 0 && x.head % 4 == 0;
    split_planes_kernel<<<grid_for(plane / 8, 256, 16), 256, 0, s>>>(rows, heads, size, (const float*)x.data, x.row, x.head, vectors,
                                                                    (__nv_bfloat16*)ws);
    PCCNN_LAUNCH_CHECK();
    ws += align_up((size_t)plane * 6);
    return PCCNN_OK;
}
static size_t operand_bytes(int64_t rows, int heads, int size, bool planes) {
    return planes ? align_up((size_t)rows * heads * size * 6) : 0;
}
static int operand_map(CUtensorMap* map, const TcOperand& o, int size, bool planes, int box_rows) {
    return make_heads_map(map, o.rows.data, planes ? 3 * o.count : o.count, o.heads, size, o.rows.row, o.rows.head, box_rows);
}

// ---- which calls ------------------------------------------------------------------------------------------------
// Tiles of 128 queries pay once a cloud has more than a handful of them; below that the row kernels read the keys once
// and do no product for absent rows.
bool tc_shape(const AttentionCall& a) {
    return a.size % 8 == 0 && a.size <= 128 && a.num_queries > 8 * (int64_t)a.clouds && a.num_keys > 0 && a.num_queries < 0x7fffffffLL / 3 &&
           a.num_keys < 0x7fffffffLL / 3;
}
static bool tc_heads(const HeadRows& x) { return aligned16(x.data) && x.row % 8 == 0 && x.head % 8 == 0; }
bool tc_layout(const AttentionCall& a, const HeadRows* grads) {
    return !a.is_bf16 || (tc_heads(a.q) && tc_heads(a.k) && tc_heads(a.v) && (!grads || tc_heads(*grads)));
}

// Splits of the streamed rows so that the blocks fill the GPU twice, as long as a split keeps at least four tiles (on average).
static int tc_splits(int64_t blocks, int64_t streamed_per_cloud, int tile) {
    int64_t s = (2 * (int64_t)sm_count() + blocks - 1) / (blocks > 0 ? blocks : 1);
    const int64_t most = streamed_per_cloud / (4 * tile);
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
}
static int64_t tc_blocks(int64_t rows, int per_block, int clouds) { return rows / per_block + clouds + 1; }

static int tc_forward_splits(const AttentionCall& a) {
    const int per_block = a.is_bf16 ? 256 : 128, clouds = a.clouds > 0 ? a.clouds : 1;
    const int64_t blocks = ((a.num_queries + per_block - 1) / per_block + clouds / 2) * a.heads;
    return tc_splits(blocks, a.num_keys / clouds, a.is_bf16 ? 128 : 64);
}

size_t tc_forward_workspace(const AttentionCall& a) {
    const bool planes = !a.is_bf16;
    const int splits = tc_forward_splits(a);
    const size_t rows = splits > 1 ? (size_t)splits * a.num_queries * a.heads : 0;
    return operand_bytes(a.num_queries, a.heads, a.size, planes) + 2 * operand_bytes(a.num_keys, a.kv_heads, a.size, planes) +
           align_up(rows * sizeof(float2)) + align_up(rows * a.size * 4) + 256;
}

static int tc_control(TcControl& ctl) {
    ctl = {tensor_core_poll_limit(), tensor_core_withhold_from(), sticky_status_device(), kOriginAttention << 8};
    return ctl.sticky ? PCCNN_OK : PCCNN_ERR_CUDA;
}

template <int GR, int BN, int NP, int QT, class T>
static int launch_forward(const AttentionCall& a, void* out, float* lse, char* ws, cudaStream_t s) {
    using Cfg = TcForward<GR, BN, NP, QT>;
    static std::atomic<uint64_t> done{0};
    const auto kernel = attention_tc_kernel<GR, BN, NP, QT, T>;
    if (int rc = allow_shared(kernel, Cfg::kBytes, done)) return rc;
    TcControl ctl;
    if (int rc = tc_control(ctl)) return rc;
    TcOperand q, k, v;
    if (int rc = tc_operand(q, a.q, a.num_queries, a.heads, a.size, NP == 3, ws, s)) return rc;
    if (int rc = tc_operand(k, a.k, a.num_keys, a.kv_heads, a.size, NP == 3, ws, s)) return rc;
    if (int rc = tc_operand(v, a.v, a.num_keys, a.kv_heads, a.size, NP == 3, ws, s)) return rc;
    CUtensorMap map_q, map_k, map_v, map_k8, map_v8;
    if (int rc = operand_map(&map_q, q, a.size, NP == 3, kTcRows)) return rc;
    if (int rc = operand_map(&map_k, k, a.size, NP == 3, BN)) return rc;
    if (int rc = operand_map(&map_v, v, a.size, NP == 3, BN)) return rc;
    if (int rc = operand_map(&map_k8, k, a.size, NP == 3, 8)) return rc;
    if (int rc = operand_map(&map_v8, v, a.size, NP == 3, 8)) return rc;
    const int splits = tc_forward_splits(a);
    float2* stat = (float2*)ws;
    float* part = (float*)(ws + align_up((size_t)splits * a.num_queries * a.heads * sizeof(float2)));
    const dim3 grid((unsigned)tc_blocks(a.num_queries, QT * kTcRows, a.clouds), (unsigned)a.heads, (unsigned)splits);
    kernel<<<grid, kTcThreads, Cfg::kBytes, s>>>(map_q, map_k, map_v, map_k8, map_v8, a, k.rows, v.rows, splits, (T*)out, lse, part, stat, ctl);
    PCCNN_LAUNCH_CHECK();
    return splits > 1 ? join_splits(a, splits, part, stat, out, lse, s) : PCCNN_OK;
}

int tc_forward(const AttentionCall& a, void* out, float* lse, char* ws, cudaStream_t s) {
    if (a.is_bf16)
        return a.size <= 64 ? launch_forward<1, 128, 1, 2, __nv_bfloat16>(a, out, lse, ws, s) : launch_forward<2, 64, 1, 2, __nv_bfloat16>(a, out, lse, ws, s);
    return a.size <= 64 ? launch_forward<1, 64, 3, 1, float>(a, out, lse, ws, s) : launch_forward<2, 32, 3, 1, float>(a, out, lse, ws, s);
}

// ---- backward -----------------------------------------------------------------------------------------------------
// The tiles that stay in shared memory: 32-bit heads of more than 64 features need 192 KB for them alone and take the row kernels.
// The streamed tiles of all heads that share a key head are counted in 32 bits.
bool tc_grads_shape(const AttentionCall& a) {
    return tc_shape(a) && (a.is_bf16 || a.size <= 64) && (a.num_queries / 64 + 1) * (a.heads / a.kv_heads) < 0x7fffffffLL;
}

static int tc_grad_splits(const AttentionCall& a, bool keys) {
    const int64_t rows = keys ? a.num_keys : a.num_queries, streamed = keys ? a.num_queries : a.num_keys;
    const int clouds = a.clouds > 0 ? a.clouds : 1;
    const int64_t blocks = ((rows + kTcRows - 1) / kTcRows + clouds / 2) * (keys ? a.kv_heads : a.heads);
    return tc_splits(blocks, streamed / clouds * (keys ? a.heads / a.kv_heads : 1), 64);
}

size_t tc_grads_workspace(const AttentionCall& a) {
    const bool planes = !a.is_bf16;
    const size_t sq = tc_grad_splits(a, false), sk = tc_grad_splits(a, true);
    const size_t pq = sq > 1 ? sq * a.num_queries * a.heads * a.size * 4 : 0, pk = sk > 1 ? 2 * sk * a.num_keys * a.kv_heads * a.size * 4 : 0;
    return 2 * operand_bytes(a.num_queries, a.heads, a.size, planes) + 2 * operand_bytes(a.num_keys, a.kv_heads, a.size, planes) +
           align_up(pq > pk ? pq : pk) + 256;
}

template <bool KEYS, int GR, int NP, class T>
static int launch_grads(const AttentionCall& a, const TcOperand& f1, const TcOperand& f2, const TcOperand& y1, const TcOperand& y2,
                        const float* lse, const float* delta, void* out1, void* out2, char* ws, cudaStream_t s) {
    using Cfg = TcBackward<KEYS, GR, NP>;
    static std::atomic<uint64_t> done{0};
    const auto kernel = attention_tc_grads_kernel<KEYS, GR, NP, T>;
    if (int rc = allow_shared(kernel, Cfg::kBytes, done)) return rc;
    TcControl ctl;
    if (int rc = tc_control(ctl)) return rc;
    CUtensorMap m[6];
    if (int rc = operand_map(&m[0], f1, a.size, NP == 3, kTcRows)) return rc;
    if (int rc = operand_map(&m[1], f2, a.size, NP == 3, kTcRows)) return rc;
    if (int rc = operand_map(&m[2], y1, a.size, NP == 3, Cfg::kBN)) return rc;
    if (int rc = operand_map(&m[3], y2, a.size, NP == 3, Cfg::kBN)) return rc;
    if (int rc = operand_map(&m[4], y1, a.size, NP == 3, 8)) return rc;
    if (int rc = operand_map(&m[5], y2, a.size, NP == 3, 8)) return rc;
    const int64_t rows = KEYS ? a.num_keys : a.num_queries;
    const int heads = KEYS ? a.kv_heads : a.heads, splits = tc_grad_splits(a, KEYS);
    const int64_t count = rows * heads * a.size;
    float* part = (float*)ws;
    const dim3 grid((unsigned)tc_blocks(rows, kTcRows, a.clouds), (unsigned)heads, (unsigned)splits);
    kernel<<<grid, kTcThreads, Cfg::kBytes, s>>>(m[0], m[1], m[2], m[3], m[4], m[5], a, y1.rows, y2.rows, splits, lse, delta, (T*)out1,
                                                 (T*)out2, part, part + splits * count, ctl);
    PCCNN_LAUNCH_CHECK();
    if (splits > 1) {
        if (int rc = add_splits(a.is_bf16, count, splits, part, out1, s)) return rc;
        if (KEYS) return add_splits(a.is_bf16, count, splits, part + splits * count, out2, s);
    }
    return PCCNN_OK;
}

template <int GR, int NP, class T>
static int launch_both_grads(const AttentionCall& a, const HeadRows& grads, const float* lse, const float* delta, void* dq, void* dk, void* dv,
                             char* ws, cudaStream_t s) {
    TcOperand q, k, v, g;
    if (int rc = tc_operand(q, a.q, a.num_queries, a.heads, a.size, NP == 3, ws, s)) return rc;
    if (int rc = tc_operand(g, grads, a.num_queries, a.heads, a.size, NP == 3, ws, s)) return rc;
    if (int rc = tc_operand(k, a.k, a.num_keys, a.kv_heads, a.size, NP == 3, ws, s)) return rc;
    if (int rc = tc_operand(v, a.v, a.num_keys, a.kv_heads, a.size, NP == 3, ws, s)) return rc;
    if (int rc = launch_grads<false, GR, NP, T>(a, q, g, k, v, lse, delta, dq, nullptr, ws, s)) return rc;
    return launch_grads<true, GR, NP, T>(a, k, v, q, g, lse, delta, dk, dv, ws, s);
}

int tc_grads(const AttentionCall& a, const HeadRows& grads, const float* lse, const float* delta, void* dq, void* dk, void* dv, char* ws,
             cudaStream_t s) {
    if (!a.is_bf16) return launch_both_grads<1, 3, float>(a, grads, lse, delta, dq, dk, dv, ws, s);
    return a.size <= 64 ? launch_both_grads<1, 1, __nv_bfloat16>(a, grads, lse, delta, dq, dk, dv, ws, s)
                        : launch_both_grads<2, 1, __nv_bfloat16>(a, grads, lse, delta, dq, dk, dv, ws, s);
}

}  // namespace pccnn
