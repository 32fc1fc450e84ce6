// Streams that share the first pages of their tables: what the prefix kernel and the split-KV kernel agree on.
//
// A stream takes part if it is long enough for all of its group's shared pages; then every shared key is visible to it
// and nothing needs a mask (a weight of zero would not hide a NaN behind a shorter stream's end).  A shorter stream, and
// one outside all groups, is attended page by page like any other.
#pragma once

#include "qm_common.cuh"

constexpr int kSharedMaxBatch = 256;       // streams (and groups) per call

// Where a stream's partial results over its group's shared pages lie: partial row
//   base + (kv_head * splits + split) * group_rows + 2 * (stream's place in its group) + query head of the pair.
struct SharedStream {
    int base;
    int splits;          // 0: nothing shared
    int group_rows;      // 2 * streams of the group
    int row;             // 2 * place in the group
};

struct SharedGroups {
    const int32_t* starts;       // [groups + 1]
    const int32_t* pages;        // [groups]
    int groups;
    int max_pages;               // entries of `pages` are cut to this
    SharedStream* streams;       // workspace [kSharedMaxBatch], written by the prefix kernel
    float* partial_o;            // workspace [rows][128], unnormalised
    float2* partial_ml;          // workspace [rows]: maximum (log2 domain) and sum of exponentials
};

// Group boundaries into shared memory, forced into order and into 0 .. batch whatever the array holds (so that every
// stream is in one group at most); streams outside all groups share nothing.  One warp.
__device__ __forceinline__ void load_group_starts(const SharedGroups& g, int batch, int* starts, uint32_t* status, int lane) {
    int carry = 0;
    bool bad = false;
    for (int base = 0; base <= g.groups; base += 32) {
        const int i = base + lane;
        int v = i <= g.groups ? g.starts[i] : 0;
        const int given = v;
        v = v < 0 ? 0 : (v > batch ? batch : v);
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= off) v = max(v, t);
        }
        v = max(v, carry);
        if (i <= g.groups) {
            starts[i] = v;
            bad |= v != given;
        }
        carry = __shfl_sync(0xffffffffu, v, 31);
    }
    if (bad) atomicOr(status, QM_DEVSTAT_BAD_POS);
}

// The group of a stream, or -1.
__device__ __forceinline__ int group_of_stream(const int* starts, int groups, int stream) {
    int lo = 0, hi = groups;                 // last g with starts[g] <= stream
    if (stream < starts[0] || stream >= starts[groups]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= stream) lo = mid; else hi = mid;
    }
    return lo;
}

// Pages of the group that a stream of `len` keys has attended for it.
__device__ __forceinline__ int shared_pages_of(const SharedGroups& g, int group, int len) {
    int p = g.pages[group];
    p = p < 0 ? 0 : (p > g.max_pages ? g.max_pages : p);
    return len / kPageTokens >= p ? p : 0;
}

// Folds a stream's partial results over the shared pages into (m, l, o): element d of query row `head2` (2 * kv head +
// query head of the pair).  Splits are folded in order.
__device__ __forceinline__ void fold_shared(const SharedGroups& g, const SharedStream& st, int kv_head, int qh, int d, float& m, float& l,
                                            float& o) {
    const int first = st.base + kv_head * st.splits * st.group_rows + st.row + qh;
    for (int j0 = 0; j0 < st.splits; j0 += 8) {
        float2 ml[8];
        float po[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const size_t r = (size_t)(first + (j0 + j < st.splits ? j0 + j : st.splits - 1) * st.group_rows);
            ml[j] = __ldcg(g.partial_ml + r);
            po[j] = __ldcg(g.partial_o + r * kHeadDim + d);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j0 + j < st.splits) {
                const float top = fmaxf(m, ml[j].x);
                const float w0 = fast_exp2(m - top), w1 = fast_exp2(ml[j].x - top);      // m = -inf so far: w0 = 0
                l = fmaf(l, w0, ml[j].y * w1);
                o = fmaf(o, w0, po[j] * w1);
                m = top;
            }
        }
    }
}

struct qm_kv_pool;
// Host: the split-KV launch over the pages behind the shared ones (qm_decode.cu).
int32_t qm_launch_decode_behind_shared(qm_kv_pool* pool, int32_t layer, const uint16_t* q_rot, const int32_t* seq_lens,
                                       const int32_t* page_table, int32_t max_pages, int32_t batch, uint16_t* out, void* workspace,
                                       const SharedGroups& groups, cudaStream_t stream);
