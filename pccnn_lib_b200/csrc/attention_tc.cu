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

// x -> (h, m, l): planes [3][rows, heads, size] of bf16, for the tensors of one call (blockIdx.y).  size is a multiple of 8; one
// thread per 8 features.
struct SplitTensor {
    const float* src;
    int64_t row, head, rows;
    int heads;
    bool vectors;
    __nv_bfloat16* planes;
};
struct SplitTensors {
    SplitTensor t[4];
};
__global__ void __launch_bounds__(256)
split_planes_kernel(const __grid_constant__ SplitTensors all, int size) {
    const SplitTensor& x = all.t[blockIdx.y];
    const int per_head = size / 8, per_row = x.heads * per_head;
    const int64_t total = x.rows * per_row, plane = x.rows * x.heads * size;
    for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per_row;
        const int in_row = (int)(i - r * per_row), h = in_row / per_head, c = (in_row - h * per_head) * 8;
        const float* p = x.src + r * x.row + h * x.head + c;
        float v[8];
        if (x.vectors) {
            load_vec<float, 8>(p, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p[e];
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
                v[2 * e] -= __uint_as_float(w[e] << 16);
                v[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
            }
            *reinterpret_cast<uint4*>(x.planes + k * plane + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// A tensor of heads as the kernels read it: its own data in bf16, or its three planes in the workspace.
struct TcOperand {
    TcRows rows;
    int64_t count;  // rows of one plane
    int heads;
};

// Describes the tensors of a call, and brings 32-bit ones into planes (one launch for all of them).
struct TcOperands {
    TcOperand o[4];
    SplitTensors split;
    int n = 0;
    char* ws;
    int size;
    bool planes;

    TcOperands(char* ws_, int size_, bool planes_) : ws(ws_), size(size_), planes(planes_) {}
    const TcOperand& add(const HeadRows& x, int64_t rows, int heads) {
        TcOperand& r = o[n];
        r.count = rows;
        r.heads = heads;
        r.rows = {(const __nv_bfloat16*)x.data, x.row, x.head, 0};
        if (planes) {
            const int64_t plane = rows * heads * size;
            r.rows = {(const __nv_bfloat16*)ws, (int64_t)heads * size, size, plane};
            split.t[n] = {(const float*)x.data, x.row, x.head, rows, heads, aligned16(x.data) && x.row % 4 == 0 && x.head % 4 == 0, (__nv_bfloat16*)ws};
            ws += align_up((size_t)plane * 6);
        }
        return o[n++];
    }
    int make_planes(cudaStream_t s) const {
        if (!planes) return PCCNN_OK;
        int64_t most = 0;
        for (int i = 0; i < n; ++i) most = split.t[i].rows * split.t[i].heads > most ? split.t[i].rows * split.t[i].heads : most;
        split_planes_kernel<<<dim3(grid_for(most * (size / 8), 256, 8), (unsigned)n), 256, 0, s>>>(split, size);
        PCCNN_LAUNCH_CHECK();
        return PCCNN_OK;
    }
};
static size_t operand_bytes(int64_t rows, int heads, int size, bool planes) {
    return planes ? align_up((size_t)rows * heads * size * 6) : 0;
}
static int operand_map(CUtensorMap* map, const TcOperand& o, int size, bool planes, int box_rows) {
    return make_heads_map(map, o.rows.data, planes ? 3 * o.count : o.count, o.heads, size, o.rows.row, o.rows.head, box_rows);
}

// ---- which calls ------------------------------------------------------------------------------------------------
static bool tc_any_shape(const AttentionCall& a) {
    return a.size % 8 == 0 && a.size <= 128 && a.num_queries > 0 && a.num_keys > 0 && a.num_queries < 0x7fffffffLL / 3 && a.num_keys < 0x7fffffffLL / 3;
}
// Multiply-adds of one of the products, with the mean cloud's keys and heads that share keys counted once.
static double tc_work(const AttentionCall& a) {
    return (double)a.num_queries * ((double)a.num_keys / (a.clouds > 0 ? a.clouds : 1)) * a.kv_heads * a.size;
}
// Forward: tiles, except for
//  - small calls: 150 queries, 301 keys, 2 clouds, 4 heads of 32: 9.7 us with rows, 13.5 us with tiles in bf16, 11.7 and 20 us in
//    32 bits; one cloud of 64 queries, 300 keys, 4 heads of 64 (5e6 multiply-adds): 14.1 and 11.6, 21.2 and 19.3 us;
//  - few queries per cloud: one in bf16 (16 queries, 40000 keys, 8 heads of 64: 21 us with rows, 47 us with tiles; 32 queries 27 and
//    47 us, but with 400000 keys 239 and 191 us); three where heads share keys (48 queries, 8 heads on 2 of 64: 35 and 46 us with
//    40000 keys, 182 and 190 us with 400000; four queries per cloud: 48 and 47, 237 and 191 us), six for heads of up to 32 features
//    (96 queries, 4 heads on 1: 26 and 25, 88 and 100 us); four 32-bit ones, which would have to be split into planes first (64
//    queries, 40000 keys, 16 clouds, 8 heads: 146 and 183 us, with 256 queries 458 and 181 us).
bool tc_shape(const AttentionCall& a) {
    if (!tc_any_shape(a) || tc_work(a) < 4e6) return false;
    if (!a.is_bf16) return a.num_queries * (a.heads / a.kv_heads) > 4 * (int64_t)a.clouds;
    const int rows = use_products(a) && a.heads > a.kv_heads ? a.size > 32 ? 3 : 6 : 1;
    return a.num_queries > rows * (int64_t)a.clouds;
}
// What a tensor map describes: 16-byte aligned rows at positive strides below 2^40 bytes.  (A row or head that is repeated or runs
// backwards goes to the row kernels; 32-bit features are brought into planes first and may lie in any way.)
static bool tc_stride(int64_t s) { return s > 0 && s % 8 == 0 && s < (1ll << 39); }
static bool tc_heads(const HeadRows& x) { return aligned16(x.data) && tc_stride(x.row) && tc_stride(x.head); }
bool tc_layout(const AttentionCall& a, const HeadRows* grads) {
    return !a.is_bf16 || (tc_heads(a.q) && tc_heads(a.k) && tc_heads(a.v) && (!grads || tc_heads(*grads)));
}

// Splits of the streamed rows where the blocks do not fill the GPU twice: enough for two blocks per SM, as long as a split keeps at
// least 512 rows (on average).  A block costs several microseconds beside its units: 1024 latents on 120007 points took 209 us with
// two blocks per SM, 216 us with three and 252 us with six (203 us since).
static int tc_splits(int64_t blocks, int64_t streamed_per_cloud, int least_rows = kTcSplitRows) {
    if (blocks >= 2 * (int64_t)sm_count()) return 1;
    int64_t s = (2 * (int64_t)sm_count() + blocks - 1) / (blocks > 0 ? blocks : 1);
    const int64_t most = streamed_per_cloud / least_rows;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
}
static int64_t tc_blocks(int64_t rows, int per_block, int clouds) { return rows / per_block + clouds + 1; }

// Forward: a split's rows go by the mean cloud, and clouds of up to twice its keys make more splits instead of longer ones; splits
// that a cloud does not fill write nothing but their statistics.  (Against equal numbers for all clouds, clouds of a fifth to
// nine fifths of the mean: 1024 queries, 120007 keys, 8 heads on 4 of 64, 32 bits 650 us, so 554 us; 2000 queries, 200000 keys,
// 16 clouds, bf16 200 us, so 184 us; 1280 queries, 20000 keys, 5 clouds 51 us, so 57 us.)
struct TcForwardSplits {
    int count, rows;
};
static TcForwardSplits tc_forward_splits(const AttentionCall& a) {
    const int per_block = a.is_bf16 ? 256 : 128, clouds = a.clouds > 0 ? a.clouds : 1;
    const int64_t blocks = ((a.num_queries + per_block - 1) / per_block + clouds / 2) * a.heads, mean = a.num_keys / clouds;
    const int s = tc_splits(blocks, mean);
    if (s == 1 || clouds == 1) return {s, kTcSplitRows};
    const int64_t rows = (mean + s - 1) / s;
    return {2 * s < kMaxSplits ? 2 * s : kMaxSplits, (int)(rows > kTcSplitRows ? rows : kTcSplitRows)};
}

size_t tc_forward_workspace(const AttentionCall& a) {
    const bool planes = !a.is_bf16;
    const int splits = tc_forward_splits(a).count;
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
    TcOperands operands(ws, a.size, NP == 3);
    const TcOperand &q = operands.add(a.q, a.num_queries, a.heads), &k = operands.add(a.k, a.num_keys, a.kv_heads),
                    &v = operands.add(a.v, a.num_keys, a.kv_heads);
    if (int rc = operands.make_planes(s)) return rc;
    ws = operands.ws;
    CUtensorMap map_q, map_k, map_v, map_k8, map_v8;
    if (int rc = operand_map(&map_q, q, a.size, NP == 3, kTcRows)) return rc;
    if (int rc = operand_map(&map_k, k, a.size, NP == 3, BN)) return rc;
    if (int rc = operand_map(&map_v, v, a.size, NP == 3, BN)) return rc;
    if (int rc = operand_map(&map_k8, k, a.size, NP == 3, 8)) return rc;
    if (int rc = operand_map(&map_v8, v, a.size, NP == 3, 8)) return rc;
    const auto [splits, split_rows] = tc_forward_splits(a);
    float2* stat = (float2*)ws;
    float* part = (float*)(ws + align_up((size_t)splits * a.num_queries * a.heads * sizeof(float2)));
    const dim3 grid((unsigned)tc_blocks(a.num_queries, QT * kTcRows, a.clouds), (unsigned)a.heads, (unsigned)splits);
    kernel<<<grid, kTcThreads, Cfg::kBytes, s>>>(map_q, map_k, map_v, map_k8, map_v8, a, k.rows, v.rows, splits, split_rows, (T*)out, lse, part, stat, ctl);
    PCCNN_LAUNCH_CHECK();
    return splits > 1 ? join_splits(a, splits, part, stat, out, lse, s) : PCCNN_OK;
}

int tc_forward(const AttentionCall& a, void* out, float* lse, char* ws, cudaStream_t s) {
    if (a.is_bf16)
        return a.size <= 64 ? launch_forward<1, 128, 1, 2, __nv_bfloat16>(a, out, lse, ws, s) : launch_forward<2, 64, 1, 2, __nv_bfloat16>(a, out, lse, ws, s);
    return a.size <= 64 ? launch_forward<1, 64, 3, 1, float>(a, out, lse, ws, s) : launch_forward<2, 32, 3, 1, float>(a, out, lse, ws, s);
}

// ---- backward -----------------------------------------------------------------------------------------------------
// Backward: tiles, except for small 32-bit calls (150 queries, 301 keys, 2 clouds, 4 heads of 32: 24 us with rows, 40 us with
// tiles; 300 queries, 600 keys, 4 heads of 64: 107 and 65 us; in bf16 tiles are faster from one query on: 20.4 and 19.1 us for
// one query and 300 keys) and for 32-bit heads of more than 64 features: the two tiles that stay would take 2 x 192 columns of tensor
// memory, which leaves too few of the 512 for logits and accumulators.
// The streamed tiles of all heads that share a key head are counted in 32 bits.
bool tc_grads_shape(const AttentionCall& a) {
    return tc_any_shape(a) && (a.is_bf16 || (a.size <= 64 && tc_work(a) >= 6e6)) &&
           (a.num_queries / 32 + 1) * (a.heads / a.kv_heads) < 0x7fffffffLL;
}

// Streamed rows that a split has at least, for the host's choice and the kernel's ranges alike: kTcSplitRows, where a query counts
// once for every head that shares the block's keys, in whole tiles.  (With 512 queries a split whatever the heads, most of the
// splits that the host counted had none: both passes for 1000 queries, 300 keys, bf16 heads of 64, 8 on 1 85 us, so 56 us, 8 on 2 59
// and 45 us; 2000 queries, 1000 keys, 4 clouds, 8 on 1 90 and 60 us.  Where the splits run over into a second wave it is slower:
// 4000 queries, 300 keys, 8 on 4 59 and 66 us.)
static int tc_grad_split_rows(const AttentionCall& a, bool keys) {
    const int rows = kTcSplitRows / (keys ? a.heads / a.kv_heads : 1);
    return rows > kTcGradRows ? rows : kTcGradRows;
}

static int tc_grad_splits(const AttentionCall& a, bool keys) {
    const int64_t rows = keys ? a.num_keys : a.num_queries, streamed = keys ? a.num_queries : a.num_keys;
    const int clouds = a.clouds > 0 ? a.clouds : 1;
    const int64_t blocks = ((rows + kTcRows - 1) / kTcRows + clouds / 2) * (keys ? a.kv_heads : a.heads);
    const int s = tc_splits(blocks, streamed / clouds, tc_grad_split_rows(a, keys));
    if (clouds > 1 || s == 1) return s;
    // one cloud: as many splits as its tiles fill
    const int64_t tiles = (streamed + kTcGradRows - 1) / kTcGradRows, per = (tiles + s - 1) / s;
    return (int)((tiles + per - 1) / per);
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
                        const float* lse, float* delta, void* out1, void* out2, char* ws, cudaStream_t s) {
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
    kernel<<<grid, kTcThreads, Cfg::kBytes, s>>>(m[0], m[1], m[2], m[3], m[4], m[5], a, f1.rows, f2.rows, y1.rows, y2.rows, splits, tc_grad_split_rows(a, KEYS), lse, delta, (T*)out1,
                                                 (T*)out2, part, part + splits * count, ctl);
    PCCNN_LAUNCH_CHECK();
    if (splits > 1) {
        if (int rc = add_splits(a.is_bf16, count, splits, part, out1, s)) return rc;
        if (KEYS) return add_splits(a.is_bf16, count, splits, part + splits * count, out2, s);
    }
    return PCCNN_OK;
}

template <int GR, int NP, class T>
static int launch_both_grads(const AttentionCall& a, const HeadRows& grads, const float* lse, float* delta, void* dq, void* dk, void* dv,
                             char* ws, cudaStream_t s) {
    TcOperands operands(ws, a.size, NP == 3);
    const TcOperand &q = operands.add(a.q, a.num_queries, a.heads), &g = operands.add(grads, a.num_queries, a.heads),
                    &k = operands.add(a.k, a.num_keys, a.kv_heads), &v = operands.add(a.v, a.num_keys, a.kv_heads);
    if (int rc = operands.make_planes(s)) return rc;
    ws = operands.ws;
    if (int rc = launch_grads<false, GR, NP, T>(a, q, g, k, v, lse, delta, dq, nullptr, ws, s)) return rc;
    return launch_grads<true, GR, NP, T>(a, k, v, q, g, lse, delta, dk, dv, ws, s);
}

int tc_grads(const AttentionCall& a, const HeadRows& grads, const float* lse, float* delta, void* dq, void* dk, void* dv, char* ws,
             cudaStream_t s) {
    if (!a.is_bf16) return launch_both_grads<1, 3, float>(a, grads, lse, delta, dq, dk, dv, ws, s);
    return a.size <= 64 ? launch_both_grads<1, 1, __nv_bfloat16>(a, grads, lse, delta, dq, dk, dv, ws, s)
                        : launch_both_grads<2, 1, __nv_bfloat16>(a, grads, lse, delta, dq, dk, dv, ws, s);
}

}  // namespace pccnn
