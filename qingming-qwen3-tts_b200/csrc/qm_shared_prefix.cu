// Decode attention for streams that share a long prefix: groups of streams whose page tables begin with the same pages
// (one voice prompt behind many requests).  No counterpart in the reference, which serves one stream
// (launch_attention with query_length 1, 17.cu:17895); qm_decode_attention reads the shared pages once per stream.
//
// Two launches.  The first (qm_decode_splitkv_kernel with kShared, qm_decode.cu) has CTAs of two kinds: some attend the
// shared pages, each page once for up to 64 streams, on the tensor cores (qm_shared_prefix.cuh); the others the pages
// behind them, stream by stream, as qm_decode_attention does.  The plan gives both kinds about the same number of pages
// per CTA, so that they end together and HBM is busy to the end (as two launches, the second one's CTAs came up
// one by one where the first one's left, each with a full share still to do: 55 us against 43 for 64 streams behind 2048
// tokens with up to 1024 of their own).  The second, below, folds a row's partial results: up to
// a few dozen pieces of the shared part and one of its own, a CTA per pair of rows with its loads in flight together.
//
// Measured (8 KV heads): 64 streams behind 2048 tokens, up to 1024 of their own, 42 us (151 MB, 3.6 TB/s;
// qm_decode_attention 100 us); 83 streams behind five prefixes of up to 4288 tokens, 47-48 us (184 us); 32 streams behind 32 768
// tokens, 52-53 us (204 MB, 3.9 TB/s; 581 us); four streams behind 1024 tokens 11 us (11 us).  What is left above the bytes' 22 to
// 31 us: 1.3 to 2.1 us of plan, some 4 us until the first products, 7 to 9 us of fold and its launch, and CTAs with equal
// shares that end up to 10 us apart.
#include "qm_shared_prefix.cuh"

namespace {

constexpr int kCombineThreads = 128;
constexpr int kCombineWarps = kCombineThreads / 32;
constexpr int kOwnStride = kHeadDim + 2;      // m (natural log), l, o[128]
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void fold_into(float& m, float& l, float4& o, float m1, float l1, const float4& o1) {
    const float top = fmaxf(m, m1);
    const float w0 = fast_exp2(m - top), w1 = fast_exp2(m1 - top);
    l = fmaf(l, w0, l1 * w1);
    o.x = fmaf(o.x, w0, o1.x * w1);
    o.y = fmaf(o.y, w0, o1.y * w1);
    o.z = fmaf(o.z, w0, o1.z * w1);
    o.w = fmaf(o.w, w0, o1.w * w1);
    m = top;
}

// A CTA per (stream, KV head): the two query rows of the pair lie side by side in a piece's block.  Warp w folds the pieces
// w, w + 4, ..., a lane four elements of both rows; then warp r folds row r's four results and the stream's own part, in
// a fixed order.
__global__ void __launch_bounds__(kCombineThreads) qm_shared_combine_kernel(const SharedGroups g, const float* own, int kv_heads, uint16_t* out) {
    __shared__ float4 part_o[2][kCombineWarps][32];
    __shared__ float2 part_ml[2][kCombineWarps];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int stream = blockIdx.x / kv_heads, head = blockIdx.x - stream * kv_heads;
    const size_t row0 = (size_t)blockIdx.x * 2;
    int4 st = __ldcg(reinterpret_cast<const int4*>(g.streams + stream));     // base, splits, group_rows, row
    const bool has_own = (st.w & 1) != 0;
    st.w &= ~1;
    // the own part, fetched beside the descriptor; without one the place holds what some earlier call left there
    const float* mine = own + (row0 + (warp & 1)) * kOwnStride;
    const float2 own_ml = __ldcg(reinterpret_cast<const float2*>(mine));
    const float2 own_a = __ldcg(reinterpret_cast<const float2*>(mine + 2 + 4 * lane));
    const float2 own_b = __ldcg(reinterpret_cast<const float2*>(mine + 4 + 4 * lane));
    const int first = st.x + head * st.y * st.z;
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.0f, 0.0f};
    float4 o[2] = {};
    constexpr int kFlight = 4;
    for (int j0 = warp; j0 < st.y; j0 += kFlight * kCombineWarps) {
        float2 ml[kFlight][2];
        float4 po[kFlight][2];
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
            const int j = j0 + i * kCombineWarps;
            const size_t block = (size_t)(first + (j < st.y ? j : j0) * st.z);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                ml[i][r] = __ldcg(g.partial_ml + block + st.w + r);
                po[i][r] = __ldcg(g.partial_o + block * (kHeadDim / 4) + (size_t)lane * st.z + st.w + r);
            }
        }
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
            if (j0 + i * kCombineWarps >= st.y) break;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (j0 == warp && i == 0) {
                    m[r] = ml[i][r].x;
                    l[r] = ml[i][r].y;
                    o[r] = po[i][r];
                } else {
                    fold_into(m[r], l[r], o[r], ml[i][r].x, ml[i][r].y, po[i][r]);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        part_o[r][warp][lane] = o[r];
        if (lane == 0) part_ml[r][warp] = make_float2(m[r], l[r]);
    }
    __syncthreads();
    if (warp < 2) {
        float top = own_ml.x * kLog2e, sum = has_own ? own_ml.y : 0.0f;
        float4 acc = has_own ? make_float4(own_a.x, own_a.y, own_b.x, own_b.y) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        bool empty = !has_own;
#pragma unroll
        for (int w = 0; w < kCombineWarps; ++w) {
            if (w >= st.y) break;
            const float2 ml = part_ml[warp][w];
            if (empty) {
                top = ml.x;
                sum = ml.y;
                acc = part_o[warp][w][lane];
                empty = false;
            } else {
                fold_into(top, sum, acc, ml.x, ml.y, part_o[warp][w][lane]);
            }
        }
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        *reinterpret_cast<uint2*>(out + (row0 + warp) * kHeadDim + 4 * lane) =
            make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    }
}

// [batch][heads][128] bf16 viewed as {128, heads, batch}; boxes of 64 streams x 2 heads x 64 columns: row 2 * stream + head.
int32_t encode_pair_map(CUtensorMap* map, const void* base, int heads, uint64_t batch) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return qm_fail(QM_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3] = {(cuuint64_t)kHeadDim, (cuuint64_t)heads, batch};
    const cuuint64_t strides[2] = {(cuuint64_t)kHeadDim * 2, (cuuint64_t)kHeadDim * 2 * heads};
    const cuuint32_t box[3] = {64, 2, kStreamsPerTile};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUresult rc = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, elem,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return qm_fail(QM_ECUDA, "cuTensorMapEncodeTiled failed for the query tensor");
    return QM_OK;
}

// Partial rows of the shared part: there are no more pieces than CTAs, of 128 rows each, or one piece per (tile, head).
size_t partial_rows(int sm_count, int batch, int kv_heads) { return (size_t)(2 * sm_count) * 128 + (size_t)2 * batch * kv_heads; }

constexpr size_t kDescriptorBytes = (size_t)kSharedMaxBatch * sizeof(SharedStream);

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

extern "C" {

int64_t qm_decode_shared_workspace_bytes(const qm_kv_pool* pool, int32_t batch) {
    if (!pool || batch < 0) return 0;
    const int n = batch < kSharedMaxBatch ? batch : kSharedMaxBatch;
    const size_t rows = partial_rows(pool->sm_count, n, pool->kv_heads);
    return (int64_t)(align256((size_t)qm_decode_workspace_bytes(n, pool->kv_heads)) + kDescriptorBytes + align256(rows * sizeof(float2)) +
                     rows * kHeadDim * sizeof(float) + (size_t)n * 2 * pool->kv_heads * kOwnStride * sizeof(float));
}

int32_t qm_decode_attention_shared(qm_kv_pool* pool, int32_t layer, const uint16_t* q_rot, const int32_t* seq_lens,
                                   const int32_t* page_table, int32_t max_pages, int32_t batch, int32_t q_heads,
                                   const int32_t* group_starts, const int32_t* shared_pages, int32_t groups,
                                   int32_t max_shared_pages, uint16_t* out, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!pool) return qm_fail(QM_EINVAL, "pool is null");
    if (layer < 0 || layer >= pool->layers) return qm_fail(QM_EINVAL, "layer out of range");
    if (q_heads != 2 * pool->kv_heads)
        return qm_fail(QM_EINVAL, "decode attention needs q_heads == 2 * kv_heads (GQA group of 2)");
    if (batch < 0 || max_pages < 1 || groups < 0 || max_shared_pages < 0) return qm_fail(QM_EINVAL, "invalid geometry");
    if (batch > kSharedMaxBatch || groups > kSharedMaxBatch)
        return qm_fail(QM_ECAPACITY, "shared-prefix attention takes at most 256 streams and 256 groups per call");
    if (batch == 0) return QM_OK;                     // nothing to do; the tensors may then be null
    if (!q_rot || !seq_lens || !page_table || !out || !workspace || (groups > 0 && (!group_starts || !shared_pages)))
        return qm_fail(QM_EINVAL, "null tensor pointer");
    if ((reinterpret_cast<uintptr_t>(q_rot) & 15u) || (reinterpret_cast<uintptr_t>(workspace) & 15u) ||
        (reinterpret_cast<uintptr_t>(out) & 7u))
        return qm_fail(QM_EINVAL, "q_rot and workspace must be 16-byte aligned, out 8-byte aligned");
    if (workspace_bytes < qm_decode_shared_workspace_bytes(pool, batch))
        return qm_fail(QM_EINVAL, "workspace smaller than qm_decode_shared_workspace_bytes()");
    int device = -1;
    QM_CUDA_TRY(cudaGetDevice(&device), "get current device");
    if (device != pool->device) return qm_fail(QM_EINVAL, "the pool's device must be the current device");
    if (groups == 0 || max_shared_pages == 0)
        return qm_decode_attention(pool, layer, q_rot, seq_lens, page_table, max_pages, batch, q_heads, out, workspace,
                                   workspace_bytes, stream);

    unsigned char* ws = static_cast<unsigned char*>(workspace);
    const size_t rows = partial_rows(pool->sm_count, batch, pool->kv_heads);
    SharedGroups g{};
    g.starts = group_starts;
    g.pages = shared_pages;
    g.groups = groups;
    g.max_pages = max_shared_pages < max_pages ? max_shared_pages : max_pages;
    if (g.max_pages > 65535) g.max_pages = 65535;             // what lies behind is attended stream by stream
    size_t at = align256((size_t)qm_decode_workspace_bytes(batch, pool->kv_heads));
    g.streams = reinterpret_cast<SharedStream*>(ws + at);
    at += kDescriptorBytes;
    g.partial_ml = reinterpret_cast<float2*>(ws + at);
    at += align256(rows * sizeof(float2));
    g.partial_o = reinterpret_cast<float4*>(ws + at);
    at += rows * kHeadDim * sizeof(float);
    float* own = reinterpret_cast<float*>(ws + at);

    CUtensorMap q_map;
    int32_t rc = encode_pair_map(&q_map, q_rot, q_heads, (uint64_t)batch);
    if (rc != QM_OK) return rc;
    rc = qm_launch_decode_shared(pool, layer, q_rot, q_map, seq_lens, page_table, max_pages, batch, own, workspace, g,
                                 static_cast<cudaStream_t>(stream));
    if (rc != QM_OK) return rc;
    QM_CUDA_TRY(qm_launch(qm_shared_combine_kernel, dim3((unsigned)(batch * pool->kv_heads)), dim3(kCombineThreads), 0,
                          static_cast<cudaStream_t>(stream), g, own, (int)pool->kv_heads, out),
                "shared-prefix combine launch");
    return QM_OK;
}

}  // extern "C"
