// Decode attention for streams that share a long prefix: groups of streams whose page tables begin with the same pages
// (one voice prompt behind many requests).  No counterpart in the reference, which serves one stream
// (launch_attention with query_length 1, 17.cu:17895); qm_decode_attention reads the shared pages once per stream.
//
// Softmax splits over any partition of the keys: with m_i, l_i, o_i the maximum, the sum of exponentials and the
// unnormalised output over part i,  out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i,  M = max_i m_i.  Here the parts
// are the shared pages, cut into pieces, and each stream's own pages:
//
//   qm_shared_prefix_kernel   the shared pages, every page read ONCE for up to 64 streams of a group: their 128 query rows
//                             of one KV head are the M rows of tcgen05.mma, so a 32 KB page pair (K and V of 64 keys)
//                             feeds 4.2 Mflop and HBM stays the bound; (m, l, o) of every piece go to the workspace
//   split-KV decode kernel    the pages behind them, stream by stream; the CTA that finishes a row folds the pieces'
//                             results into its own (qm_decode.cu, kShared)
//
// The second launch is let go as soon as every CTA of the first has seen what it waited for, so both stream from HBM
// together and only the folds wait.
//
// Per piece: S = Q K^T (128 x 64, both operands by TMA, double-buffered in TMEM), a thread per row for the softmax, P
// over S in bf16, O += P V with P as the TMEM operand.  P is rounded to bf16 (half a step is 2^-8 of each weight, and the
// errors of many keys average out); the sum of exponentials is taken before that rounding, in fp32.  Two CTAs fit an
// SM (96 KB of shared memory and 256 TMEM columns each), one's softmax beside the other's products.
#include <math_constants.h>

#include "qm_shared_groups.cuh"
#include "qm_tcgen05.cuh"

namespace {

constexpr int kThreads = 192;             // warps 0-3 softmax, warp 4 MMA issue, warp 5 TMA
constexpr int kStreamsPerTile = 64;
constexpr int kQBytes = 128 * kHeadDim * 2;
constexpr int kPageBytes = kTileBytes;    // K or V of one page and head
constexpr int kPageStages = 2;
constexpr uint32_t kTmemCols = 256;       // S 0-63, 64-127; O 128-255
constexpr float kRescale = 8.0f;

struct PrefixSmem {
    static constexpr int kQ = 0;
    static constexpr int kK = kQ + kQBytes;
    static constexpr int kV = kK + kPageStages * kPageBytes;
    static constexpr int kStarts = kV + kPageStages * kPageBytes;              // int[257] group boundaries
    static constexpr int kLens = kStarts + (kSharedMaxBatch + 4) * 4;          // int[256]
    static constexpr int kLeader = kLens + kSharedMaxBatch * 4;               // u32[256] the first stream that takes part, per group
    static constexpr int kItems = kLeader + kSharedMaxBatch * 4;              // int[257] first piece of each group
    static constexpr int kRows = kItems + (kSharedMaxBatch + 4) * 4;           // int[257] first partial row of each group
    static constexpr int kGroupPages = kRows + (kSharedMaxBatch + 4) * 4;      // int[256]
    static constexpr int kBars = kGroupPages + kSharedMaxBatch * 4;
    static constexpr int kTmemSlot = kBars + 16 * 8;
    static constexpr int kTotal = kTmemSlot + 16;
};
static_assert(2 * (PrefixSmem::kTotal + 1024 + 1024) <= 228 * 1024, "two CTAs per SM");

enum { BAR_Q = 0, BAR_QFREE = 1, BAR_KFULL = 2, BAR_KFREE = 4, BAR_VFULL = 6, BAR_VFREE = 8, BAR_S = 10, BAR_P = 12, BAR_O = 14 };

struct PrefixArgs {
    SharedGroups shared;
    const int32_t* seq_lens;
    const int32_t* page_table;
    uint32_t* status;
    int batch;
    int kv_heads;
    int max_pages;
    int num_pages;
    int target_items;        // pieces that the work is cut into, about
    int min_pages;           // pages of a piece, at least
};

// Inclusive prefix sum over the lanes.
__device__ __forceinline__ int warp_sum_scan(int v, int lane) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += t;
    }
    return v;
}

__global__ void __launch_bounds__(kThreads, 2)
qm_shared_prefix_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map, const PrefixArgs a) {
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw_addr = smem_addr(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    unsigned char* smem = smem_raw + pad;
    const uint32_t sbase = raw_addr + pad;
    const uint32_t bar0 = sbase + PrefixSmem::kBars;
    auto bar = [&](int i) { return bar0 + 8u * i; };
    int* starts = reinterpret_cast<int*>(smem + PrefixSmem::kStarts);
    int* lens = reinterpret_cast<int*>(smem + PrefixSmem::kLens);
    int* leader = reinterpret_cast<int*>(smem + PrefixSmem::kLeader);
    int* items = reinterpret_cast<int*>(smem + PrefixSmem::kItems);
    int* rows = reinterpret_cast<int*>(smem + PrefixSmem::kRows);
    int* group_pages = reinterpret_cast<int*>(smem + PrefixSmem::kGroupPages);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + PrefixSmem::kTmemSlot);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hkv = a.kv_heads, groups = a.shared.groups;

    if (tid == 0) {
        mbar_init(bar(BAR_Q), 1);
        mbar_init(bar(BAR_QFREE), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(BAR_KFULL + i), 1);
            mbar_init(bar(BAR_KFREE + i), 1);
            mbar_init(bar(BAR_VFULL + i), 1);
            mbar_init(bar(BAR_VFREE + i), 1);
            mbar_init(bar(BAR_S + i), 1);
            mbar_init(bar(BAR_P + i), 128);      // one per S buffer: a fast warp may be a page ahead of a slow one
            // One per parity of the page: when S of page n is there, P V of page n - 2 is done, that of n - 1 need not be.
            mbar_init(bar(BAR_O + i), 1);
        }
        fence_mbar_init();
    }
    if (warp == 4) {
        tmem_alloc(smem_addr(tmem_slot), kTmemCols);
        tmem_relinquish();
    }
    for (int g = tid; g < groups; g += kThreads) {
        leader[g] = kSharedMaxBatch;
        group_pages[g] = 0;
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();           // only now: the next launch reads what this wait has covered, and every CTA holds its TMEM
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

    // ---- the pieces: groups x tiles of 64 streams x KV heads x runs of pages
    const int cap = a.max_pages * kPageTokens;
    if (warp == 0) load_group_starts(a.shared, a.batch, starts, a.status, lane);
    for (int s = tid; s < a.batch; s += kThreads) {
        const int len = a.seq_lens[s];
        if (len > cap) atomicOr(a.status, QM_DEVSTAT_BAD_POS);
        lens[s] = len < 0 ? 0 : (len > cap ? cap : len);
    }
    __syncthreads();
    // a group's pages, and the stream whose table row is read for them: the first that takes part
    for (int s = tid; s < a.batch; s += kThreads) {
        const int g = group_of_stream(starts, groups, s);
        const int pages = g < 0 ? 0 : shared_pages_of(a.shared, g, lens[s]);
        if (pages > 0) {
            atomicMin(&leader[g], s);
            group_pages[g] = pages;          // the same value from every stream that takes part
        } else {
            lens[s] = 0;                     // from here on: 0 = takes no part
        }
    }
    __syncthreads();
    int total = 0;
    if (warp == 0) {
        for (int g = lane; g < groups; g += 32) total += (starts[g + 1] - starts[g] + kStreamsPerTile - 1) / kStreamsPerTile * hkv * group_pages[g];
        total = __reduce_add_sync(0xffffffffu, total);
        int piece = (total + a.target_items - 1) / a.target_items;
        piece = piece < a.min_pages ? a.min_pages : piece;
        int item_carry = 0, row_carry = 0;
        for (int base = 0; base < groups; base += 32) {
            const int g = base + lane;
            const int n = g < groups ? starts[g + 1] - starts[g] : 0;
            const int splits = g < groups && n > 0 ? (group_pages[g] + piece - 1) / piece : 0;
            const int my_items = (n + kStreamsPerTile - 1) / kStreamsPerTile * hkv * splits, my_rows = hkv * splits * 2 * n;
            const int item_sum = warp_sum_scan(my_items, lane), row_sum = warp_sum_scan(my_rows, lane);
            if (g < groups) {
                items[g] = item_carry + item_sum - my_items;
                rows[g] = row_carry + row_sum - my_rows;
            }
            item_carry += __shfl_sync(0xffffffffu, item_sum, 31);
            row_carry += __shfl_sync(0xffffffffu, row_sum, 31);
        }
        if (lane == 0) {
            items[groups] = item_carry;
            rows[groups] = piece;            // the last word carries the piece length
        }
    }
    __syncthreads();
    const int piece = rows[groups];
    const int n_items = items[groups];
    if (blockIdx.x == 0) {
        for (int s = tid; s < a.batch; s += kThreads) {
            const int g = group_of_stream(starts, groups, s);
            int4 w = make_int4(0, 0, 0, 0);
            if (g >= 0 && lens[s] > 0) w = make_int4(rows[g], (group_pages[g] + piece - 1) / piece, 2 * (starts[g + 1] - starts[g]), 2 * (s - starts[g]));
            *reinterpret_cast<int4*>(a.shared.streams + s) = w;
        }
    }
    struct Item {
        int group, tile, head, split, splits, page0, pages, table_row;
    };
    auto locate = [&](int item) {
        Item it;
        int lo = 0, hi = groups;             // last group with items[g] <= item (a group without pieces never is)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (items[mid] <= item) lo = mid; else hi = mid;
        }
        it.group = lo;
        it.splits = (group_pages[lo] + piece - 1) / piece;
        const int r = item - items[lo];
        it.split = r % it.splits;
        it.head = (r / it.splits) % hkv;
        it.tile = r / (it.splits * hkv);
        it.page0 = it.split * piece;
        it.pages = group_pages[lo] - it.page0 < piece ? group_pages[lo] - it.page0 : piece;
        it.table_row = leader[lo];
        return it;
    };
    bool dead = false;

    if (warp == 5) {
        // ------------------------------------------------------------- TMA loads
        if (lane == 0) {
            int n = 0, local = 0;
            for (int item = blockIdx.x; item < n_items; item += gridDim.x, ++local) {
                const Item it = locate(item);
                if (!mbar_wait_bounded(bar(BAR_QFREE), (local & 1) ^ 1, dead)) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
                mbar_arrive_expect_tx(bar(BAR_Q), kQBytes);
                for (int half = 0; half < 2; ++half)
                    tma_load_3d(sbase + PrefixSmem::kQ + half * (kQBytes / 2), &q_map, bar(BAR_Q), half * 64, 2 * it.head,
                                starts[it.group] + it.tile * kStreamsPerTile);
                const int32_t* table = a.page_table + (size_t)it.table_row * a.max_pages + it.page0;
                int next_id = table[0];
                for (int j = 0; j < it.pages; ++j, ++n) {
                    int id = next_id;
                    if (j + 1 < it.pages) next_id = table[j + 1];
                    if (id < 0 || id >= a.num_pages) {
                        atomicOr(a.status, QM_DEVSTAT_BAD_PAGE);
                        id = 0;
                    }
                    const int y = (id * hkv + it.head) * kPageTokens;
                    const int st = n % kPageStages;
                    const uint32_t parity = ((n / kPageStages) & 1) ^ 1;
                    if (!mbar_wait_bounded(bar(BAR_KFREE + st), parity, dead)) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
                    mbar_arrive_expect_tx(bar(BAR_KFULL + st), kPageBytes);
                    for (int half = 0; half < 2; ++half)
                        tma_load_2d(sbase + PrefixSmem::kK + st * kPageBytes + half * (kPageBytes / 2), &k_map, bar(BAR_KFULL + st),
                                    half * 64, y);
                    if (!mbar_wait_bounded(bar(BAR_VFREE + st), parity, dead)) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
                    mbar_arrive_expect_tx(bar(BAR_VFULL + st), kPageBytes);
                    for (int half = 0; half < 2; ++half)
                        tma_load_2d(sbase + PrefixSmem::kV + st * kPageBytes + half * (kPageBytes / 2), &v_map, bar(BAR_VFULL + st),
                                    half * 64, y);
                }
            }
            // every copy has landed (bounded) before this thread, and with it the CTA, goes
            bool gave_up = false;
            if (local > 0) mbar_wait_bounded(bar(BAR_Q), (local - 1) & 1, gave_up);
            for (int i = n > kPageStages ? n - kPageStages : 0; i < n; ++i) {
                mbar_wait_bounded(bar(BAR_KFULL + i % kPageStages), (i / kPageStages) & 1, gave_up);
                mbar_wait_bounded(bar(BAR_VFULL + i % kPageStages), (i / kPageStages) & 1, gave_up);
            }
        }
        __syncwarp();
    } else if (warp == 4) {
        // ------------------------------------------------------------- MMA issue
        if (lane == 0) {
            constexpr uint32_t idesc_qk = umma_instr_desc(128, kPageTokens, false);
            constexpr uint32_t idesc_pv = umma_instr_desc(128, kHeadDim, true);
            auto issue_s = [&](int n) {
                const uint32_t ka = sbase + PrefixSmem::kK + (n % kPageStages) * kPageBytes;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    mma_ss(tmem_base + (n & 1) * 64, smem_desc(sbase + PrefixSmem::kQ + (ks >> 2) * (kQBytes / 2) + (ks & 3) * 32, 16, 1024),
                           smem_desc(ka + (ks >> 2) * (kPageBytes / 2) + (ks & 3) * 32, 16, 1024), idesc_qk, ks > 0);
                tc_commit(bar(BAR_S + (n & 1)));
                tc_commit(bar(BAR_KFREE + n % kPageStages));
            };
            auto wait = [&](int which, uint32_t parity) {
                if (!mbar_wait_bounded(bar(which), parity, dead)) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
            };
            int n = 0, local = 0;
            for (int item = blockIdx.x; item < n_items; item += gridDim.x, ++local) {
                const int pages = locate(item).pages;
                wait(BAR_Q, local & 1);
                wait(BAR_KFULL + n % kPageStages, (n / kPageStages) & 1);
                tc_fence_after();
                issue_s(n);
                if (pages == 1) tc_commit(bar(BAR_QFREE));
                for (int j = 0; j < pages; ++j, ++n) {
                    // The next page's S goes ahead of this page's P V.  Its TMEM columns held the P of the page before,
                    // whose P V was issued earlier: the tensor pipe keeps that order.
                    if (j + 1 < pages) {
                        wait(BAR_KFULL + (n + 1) % kPageStages, ((n + 1) / kPageStages) & 1);
                        tc_fence_after();
                        issue_s(n + 1);
                        if (j + 2 == pages) tc_commit(bar(BAR_QFREE));
                    }
                    wait(BAR_VFULL + n % kPageStages, (n / kPageStages) & 1);
                    wait(BAR_P + (n & 1), (n >> 1) & 1);
                    tc_fence_after();
                    const uint32_t va = sbase + PrefixSmem::kV + (n % kPageStages) * kPageBytes;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        mma_ts(tmem_base + 128, tmem_base + (n & 1) * 64 + ks * 8, smem_desc(va + ks * 2048, kPageBytes / 2, 1024), idesc_pv,
                               (j > 0 || ks > 0) ? 1u : 0u);
                    tc_commit(bar(BAR_VFREE + n % kPageStages));
                    tc_commit(bar(BAR_O + (n & 1)));
                }
            }
        }
        __syncwarp();
    } else {
        // --------------------------------------------------------------- softmax, a thread per query row
        const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
        const float c = 1.4426950408889634f / sqrtf((float)kHeadDim);       // scale * log2(e)
        auto wait = [&](int which, uint32_t parity) {
            if (!mbar_wait_bounded(bar(which), parity, dead) && lane == 0) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
        };
        int n = 0;
        for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
            const Item it = locate(item);
            const int group_streams = starts[it.group + 1] - starts[it.group];
            const int place = it.tile * kStreamsPerTile + (tid >> 1);       // row = 2 * place in the tile + query head
            const bool real = place < group_streams && lens[starts[it.group] + place] > 0;       // other rows are not stored
            float m_used = -CUDART_INF_F, l = 0.0f;
            for (int j = 0; j < it.pages; ++j, ++n) {
                const uint32_t s_addr = tmem_base + lane_base + (n & 1) * 64;
                wait(BAR_S + (n & 1), (n >> 1) & 1);
                tc_fence_after();
                uint32_t sreg[2][32];
                tmem_ld32(s_addr, sreg[0]);
                tmem_ld32(s_addr + 32, sreg[1]);
                tmem_wait_ld();
                float mxa[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) mxa[i] = -CUDART_INF_F;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        mxa[(i >> 1) & 3] = fmax3(mxa[(i >> 1) & 3], __uint_as_float(sreg[h][i]), __uint_as_float(sreg[h][i + 1]));
                const float mx = fmaxf(fmax3(mxa[0], mxa[1], mxa[2]), mxa[3]);
                const float m_new = fmaxf(m_used, mx * c);
                const bool grow = m_new > m_used + kRescale;
                if (j == 0) {
                    m_used = m_new;
                } else if (__any_sync(0xffffffffu, grow)) {
                    wait(BAR_O + ((n - 1) & 1), ((n - 1) >> 1) & 1);
                    tc_fence_after();
                    const float factor = grow ? fast_exp2(m_used - m_new) : 1.0f;
                    if (grow) m_used = m_new;
                    l *= factor;
#pragma unroll 1
                    for (int cch = 0; cch < 8; ++cch) {
                        uint32_t oreg[16];
                        tmem_ld16(tmem_base + lane_base + 128 + cch * 16, oreg);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) oreg[i] = __float_as_uint(__uint_as_float(oreg[i]) * factor);
                        tmem_st16(tmem_base + lane_base + 128 + cch * 16, oreg);
                    }
                    tmem_wait_st();
                }
                float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                const float2 c2 = make_float2(c, c), negm2 = make_float2(-m_used, -m_used);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t preg[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 x = ffma2(make_float2(__uint_as_float(sreg[h][2 * i]), __uint_as_float(sreg[h][2 * i + 1])), c2, negm2);
                        const float2 p = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                        sum2[i & 1] = fadd2(sum2[i & 1], p);
                        preg[i] = pack_bf16x2(p.x, p.y);
                    }
                    tmem_st16(s_addr + h * 16, preg);
                }
                l += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(bar(BAR_P + (n & 1)));
            }
            // ---- (m, l, o) of this piece
            wait(BAR_O + ((n - 1) & 1), ((n - 1) >> 1) & 1);
            tc_fence_after();
            const size_t r = (size_t)rows[it.group] + (size_t)(it.head * it.splits + it.split) * (2 * group_streams) + 2 * place + (tid & 1);
#pragma unroll
            for (int cch = 0; cch < 4; ++cch) {
                uint32_t oreg[32];
                tmem_ld32(tmem_base + lane_base + 128 + cch * 32, oreg);
                tmem_wait_ld();
                if (real && !dead) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4*>(a.shared.partial_o + r * kHeadDim + cch * 32 + i) =
                            make_uint4(oreg[i], oreg[i + 1], oreg[i + 2], oreg[i + 3]);
                }
            }
            if (real && !dead) a.shared.partial_ml[r] = make_float2(m_used, l);
            tc_fence_before();
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
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

constexpr int kMinPages = 4;

// Pieces: no more than two per SM by length, plus one per (tile, head) for what rounding up leaves.  Every piece has
// 2 * streams rows, so rows <= pieces-by-length * 128 + 2 * batch per head.
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
                     rows * kHeadDim * sizeof(float));
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
    if (!q_rot || !seq_lens || !page_table || !out || !workspace || (groups > 0 && (!group_starts || !shared_pages)))
        return qm_fail(QM_EINVAL, "null tensor pointer");
    if ((reinterpret_cast<uintptr_t>(q_rot) & 15u) || (reinterpret_cast<uintptr_t>(workspace) & 15u) ||
        (reinterpret_cast<uintptr_t>(out) & 1u))
        return qm_fail(QM_EINVAL, "q_rot and workspace must be 16-byte aligned");
    if (workspace_bytes < qm_decode_shared_workspace_bytes(pool, batch))
        return qm_fail(QM_EINVAL, "workspace smaller than qm_decode_shared_workspace_bytes()");
    if (batch == 0) return QM_OK;
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
    g.partial_o = reinterpret_cast<float*>(ws + at);

    CUtensorMap q_map;
    const int32_t rc = encode_pair_map(&q_map, q_rot, q_heads, (uint64_t)batch);
    if (rc != QM_OK) return rc;
    const int smem_bytes = PrefixSmem::kTotal + 1024;
    static thread_local int attr_device = -1;
    if (attr_device != pool->device) {
        QM_CUDA_TRY(cudaFuncSetAttribute(qm_shared_prefix_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes),
                    "raise shared-prefix kernel shared memory");
        attr_device = pool->device;
    }
    PrefixArgs a{};
    a.shared = g;
    a.seq_lens = seq_lens;
    a.page_table = page_table;
    a.status = pool->status_dev;
    a.batch = batch;
    a.kv_heads = pool->kv_heads;
    a.max_pages = max_pages;
    a.num_pages = pool->num_pages;
    a.target_items = 2 * pool->sm_count;
    a.min_pages = kMinPages;
    // at most this many pieces: tiles of 64 streams (a partial one per group) x heads x pieces of kMinPages
    const long long tiles = batch / kStreamsPerTile + (groups < batch ? groups : batch);
    const long long pieces = tiles * pool->kv_heads * ((g.max_pages + kMinPages - 1) / kMinPages);
    const int grid = (int)(pieces < 2 * pool->sm_count ? pieces : 2 * pool->sm_count);
    QM_CUDA_TRY(qm_launch(qm_shared_prefix_kernel, dim3((unsigned)grid), dim3(kThreads), (size_t)smem_bytes,
                          static_cast<cudaStream_t>(stream), q_map, pool->key_maps[layer], pool->value_maps[layer], a),
                "shared-prefix attention launch");
    return qm_launch_decode_behind_shared(pool, layer, q_rot, seq_lens, page_table, max_pages, batch, out, workspace, g,
                                          static_cast<cudaStream_t>(stream));
}

}  // extern "C"
