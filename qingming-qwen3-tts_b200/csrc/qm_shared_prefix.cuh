// Streams that share the first pages of their tables: how the work of a launch is cut up, and the part of it that attends
// the shared pages.
//
// A stream takes part if it is long enough for all of its group's shared pages; then every shared key is visible to it
// and nothing needs a mask (a weight of zero would not hide a NaN behind a shorter stream's end).  A shorter stream, and
// one outside all groups, is attended page by page like any other.
#pragma once

#include <math_constants.h>

#include "qm_tcgen05.cuh"

constexpr int kSharedMaxBatch = 256;       // streams (and groups) per call
// The costs that the cut goes by, in the time of a stream's own page (measured with 8 KV heads only).  Measured, us, at
// 0.85 / 0.95 / 1.05 per shared page: 64 streams behind 2048 tokens 42.8 / 43.0 / 44.2, 32 behind 32 768 tokens 53.2 / 54.4 /
// 56.2; at 3 instead of 1 per piece 44.2 and 56.1.  Pieces of one page at least cost the first case 17.9 instead of 15.9 us of
// shared part alone.
constexpr float kSharedPageCost = 0.95f;   // a shared page (32 KB like an own one)
constexpr float kSharedPieceCost = 1.0f;   // a piece, besides its pages
constexpr int kOwnPartCost = 2;            // a stream's own part, besides its pages, per KV head (0 / 1 / 2: 83 streams behind five prefixes 50.7 / 48.0 / 47.5 us)
constexpr int kSharedMinPiece = 2;         // pages
constexpr int kStreamsPerTile = 64;        // streams whose 128 query rows of a KV head make one M tile

// Where a stream's partial results over its group's shared pages lie: partial row
//   base + (kv_head * splits + split) * group_rows + row + query head of the pair.
struct SharedStream {
    int base;
    int splits;          // 0: nothing shared
    int group_rows;      // 2 * streams of the group
    int row;             // 2 * place in the group; + 1: the stream has pages of its own, and so a partial result over them
};

struct SharedGroups {
    const int32_t* starts;       // [groups + 1]
    const int32_t* pages;        // [groups]
    int groups;
    int max_pages;               // entries of `pages` are cut to this
    SharedStream* streams;       // workspace [kSharedMaxBatch]
    // Workspace.  A piece's rows are a block of group_rows; in it the unnormalised outputs lie as [32][group_rows] float4
    // (four elements of every row, then the next four), so that the threads that hold a row each store side by side.
    float4* partial_o;
    float2* partial_ml;          // workspace [rows]: maximum (log2 domain) and sum of exponentials
};

// The cut of one launch.  Shared pages: pieces = groups x tiles of 64 streams x KV heads x runs of `piece` pages, dealt
// to the first `ctas` CTAs.  The rest of the grid has the streams' own pages.
struct SharedPlan {
    int* starts;         // [groups + 1] group boundaries
    int* part;           // [batch] 1: the stream takes part
    int* leader;         // [groups] the first stream that takes part: its table row is read
    int* pages;          // [groups] shared pages, 0 where no stream takes part
    int* items;          // [groups + 1] first piece of each group
    int* rows;           // [groups + 1] first partial row of each group
    int* words;          // ctas, piece, cost of the own parts, 1 where the boundaries were out of order
    int ctas, piece, n_items, groups;

    static constexpr int kBytes = (3 * (kSharedMaxBatch + 4) + 3 * kSharedMaxBatch + 4) * 4;
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

// Group boundaries forced into order and into 0 .. batch whatever they are (so that every stream is in one group at
// most); streams outside all groups share nothing.  One warp; returns whether it had to.
__device__ __forceinline__ bool order_group_starts(int groups, int batch, int* starts, int lane) {
    int carry = 0;
    bool bad = false;
    for (int base = 0; base <= groups; base += 32) {
        const int i = base + lane;
        int v = i <= groups ? starts[i] : 0;
        const int given = v;
        v = v < 0 ? 0 : (v > batch ? batch : v);
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= off) v = max(v, t);
        }
        v = max(v, carry);
        if (i <= groups) {
            starts[i] = v;
            bad |= v != given;
        }
        carry = __shfl_sync(0xffffffffu, v, 31);
    }
    return __any_sync(0xffffffffu, bad);
}

// The group of a stream, or -1.
__device__ __forceinline__ int group_of_stream(const int* starts, int groups, int stream) {
    if (stream < starts[0] || stream >= starts[groups]) return -1;
    int lo = 0, hi = groups;                 // last g with starts[g] <= stream
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= stream) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int tiles_of(int streams) { return (streams + kStreamsPerTile - 1) / kStreamsPerTile; }

// Small groups cost more than they save: a group is a 128-row tile however few its streams, and the search below walks
// all groups before any CTA has work.  256 streams behind 512 shared tokens with 300 of their own take 110 us in 16 groups, 134
// in 64, 176 in 128 and 243 in 256; qm_decode_attention over the same tables takes 129 to 132.
//
// Every CTA works the whole plan out for itself, from word `tid` of each array in thread `tid` (it may do so twice, from what
// it read before and after the launch in front has written them).  first_page[s] = pages of stream s that are attended for
// it.  `area`: SharedPlan::kBytes of shared memory.  All threads of the CTA; ends with a barrier.
__device__ __forceinline__ SharedPlan make_shared_plan(const SharedGroups& g, int len, int start, int shared_pages, int batch, int kv_heads,
                                                       int max_pages, int grid, unsigned char* area, uint16_t* first_page,
                                                       int tid) {
    SharedPlan p;
    p.starts = reinterpret_cast<int*>(area);
    p.items = p.starts + kSharedMaxBatch + 4;
    p.rows = p.items + kSharedMaxBatch + 4;
    p.part = p.rows + kSharedMaxBatch + 4;
    p.leader = p.part + kSharedMaxBatch;
    p.pages = p.leader + kSharedMaxBatch;
    p.words = p.pages + kSharedMaxBatch;
    p.groups = g.groups;
    const int lane = tid & 31, warp = tid >> 5;
    const int cap = max_pages * kPageTokens;
    len = tid >= batch || len < 0 ? 0 : (len > cap ? cap : len);
    if (tid <= g.groups) p.starts[tid] = start;
    if (tid < g.groups) {
        p.leader[tid] = kSharedMaxBatch;
        p.pages[tid] = 0;
        p.rows[tid] = shared_pages < 0 ? 0 : (shared_pages > g.max_pages ? g.max_pages : shared_pages);
    }
    __syncthreads();
    bool out_of_order = false;
    if (warp == 0) out_of_order = order_group_starts(g.groups, batch, p.starts, lane);
    if (tid < 4) p.words[tid] = tid == 3 && out_of_order ? 1 : 0;
    __syncthreads();
    int own = 0;
    if (tid < batch) {
        const int group = group_of_stream(p.starts, g.groups, tid);
        const int shared = group < 0 ? 0 : p.rows[group];
        const bool in = shared > 0 && len / kPageTokens >= shared;
        if (in) {
            atomicMin(&p.leader[group], tid);
            p.pages[group] = shared;             // the same value from every stream that takes part
        }
        p.part[tid] = in;
        first_page[tid] = (uint16_t)(in ? shared : 0);
        own = (len + kPageTokens - 1) / kPageTokens - (in ? shared : 0);
        own = own > 0 ? (own + kOwnPartCost) * kv_heads : 0;
    }
    own = __reduce_add_sync(0xffffffffu, own);
    if (lane == 0 && own) atomicAdd(&p.words[2], own);
    __syncthreads();
    if (warp == 0) {
        int most = 0;
        for (int i = lane; i < g.groups; i += 32) most = max(most, p.starts[i + 1] > p.starts[i] ? p.pages[i] : 0);
        most = __reduce_max_sync(0xffffffffu, most);
        const int own_cost = p.words[2];
        int ctas = 0, piece = 1;
        if (most > 0) {
            // Three lengths per lane: the longest prefix in 1 .. 32 and in 41 .. 320 parts, and 2 .. 33 pages.  One piece per
            // CTA; the call takes as long as the slower kind of CTA, a piece or an equal share of the own pages.
            float best = CUDART_INF_F;
            int best_piece = most, best_count = 0;
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const int parts = k == 0 ? lane + 1 : 9 * (lane + 1) + 32;
                const int length = k == 2 ? lane + kSharedMinPiece : max((most + parts - 1) / parts, kSharedMinPiece);
                int n = 0;
                for (int i = 0; i < g.groups; ++i)
                    n += tiles_of(p.starts[i + 1] - p.starts[i]) * kv_heads * ((p.pages[i] + length - 1) / length);
                const int left = grid - n;
                float time = (float)length * kSharedPageCost + kSharedPieceCost;
                if (own_cost > 0) time = fmaxf(time, left > 0 ? (float)own_cost / (float)left : CUDART_INF_F);
                if (left >= 0 && time < best) {
                    best = time;
                    best_piece = length;
                    best_count = n;
                }
            }
            float overall = best;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) overall = fminf(overall, __shfl_xor_sync(0xffffffffu, overall, off));
            if (overall < CUDART_INF_F) {
                const int from = __ffs(__ballot_sync(0xffffffffu, best == overall)) - 1;
                piece = __shfl_sync(0xffffffffu, best_piece, from);
                ctas = __shfl_sync(0xffffffffu, best_count, from);
            } else {
                // more tiles x heads than CTAs: whole prefixes go round the CTAs that their share of the pages gives them
                piece = most;
                long long total = 0;
                int n = 0;
                for (int i = 0; i < g.groups; ++i) {
                    const int lots = p.pages[i] > 0 ? tiles_of(p.starts[i + 1] - p.starts[i]) * kv_heads : 0;
                    n += lots;
                    total += (long long)lots * p.pages[i];
                }
                ctas = (int)((float)grid * (float)total / ((float)total + (float)own_cost));
                ctas = ctas < 1 ? 1 : (own_cost > 0 && ctas > grid - 1 ? grid - 1 : ctas);
                ctas = ctas < n ? ctas : n;
            }
        }
        int item_carry = 0, row_carry = 0;
        for (int base = 0; base < g.groups; base += 32) {
            const int i = base + lane;
            const int n = i < g.groups ? p.starts[i + 1] - p.starts[i] : 0;
            const int splits = i < g.groups ? (p.pages[i] + piece - 1) / piece : 0;
            const int my_items = tiles_of(n) * kv_heads * splits, my_rows = kv_heads * splits * 2 * n;
            const int item_sum = warp_sum_scan(my_items, lane), row_sum = warp_sum_scan(my_rows, lane);
            if (i < g.groups) {
                p.items[i] = item_carry + item_sum - my_items;
                p.rows[i] = row_carry + row_sum - my_rows;
            }
            item_carry += __shfl_sync(0xffffffffu, item_sum, 31);
            row_carry += __shfl_sync(0xffffffffu, row_sum, 31);
        }
        if (lane == 0) {
            p.items[g.groups] = item_carry;
            p.words[0] = ctas;
            p.words[1] = piece;
        }
    }
    __syncthreads();
    p.ctas = p.words[0];
    p.piece = p.words[1];
    p.n_items = p.items[g.groups];
    return p;
}

// Which partial results each stream will have and where, for the launch that folds them.  One CTA, once the plan is final;
// own_units: pages x KV heads that are attended for stream `tid` alone.  A stream without any has no partial result of its
// own, written by nobody (the whole grid may be at shared pieces then): the fold must not read one.
__device__ __forceinline__ void publish_shared_plan(const SharedPlan& p, const SharedGroups& g, int own_units, int batch, uint32_t* status,
                                                    int tid) {
    if (tid == 0 && p.words[3]) atomicOr(status, QM_DEVSTAT_BAD_POS);
    if (tid >= batch) return;
    int4 w = make_int4(0, 0, 0, 0);
    if (p.part[tid]) {
        const int group = group_of_stream(p.starts, g.groups, tid), first = p.starts[group];
        w = make_int4(p.rows[group], (p.pages[group] + p.piece - 1) / p.piece, 2 * (p.starts[group + 1] - first), 2 * (tid - first));
    }
    if (own_units > 0) w.w += 1;
    *reinterpret_cast<int4*>(g.streams + tid) = w;
}

// ---- the shared pages ----------------------------------------------------------------------------------------------
//
// Softmax splits over any partition of the keys: with m_i, l_i, o_i the maximum, the sum of exponentials and the
// unnormalised output over part i,  out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i,  M = max_i m_i.  A piece is such a
// part for up to 64 streams: their 128 query rows of one KV head are the M rows of tcgen05.mma, so a page's 32 KB of K
// and V feed 4.2 Mflop and HBM stays the bound.
//
// Per page: S = Q K^T (128 x 64, both operands by TMA, double-buffered in TMEM), a thread per row for the softmax, P
// over S in bf16, O += P V with P as the TMEM operand.  P is rounded to bf16 (half a step is 2^-8 of each weight, and
// the errors of many keys average out); the sum of exponentials is taken before that rounding, in fp32.  Against 64 bits a
// context is off by 0.0022-0.0023 of its norm where fp32 weights (qm_decode_attention) leave 0.0017, nearly all of that the
// rounding of the result.  P as a high and a low bf16 half, which has the 0.0017, was measured: 83 streams behind five
// prefixes 47.8 -> 56.0 us, 32 behind 32 768 tokens 52.7 -> 61.4 us (one voice, 42 us, and four streams, 11 us, within
// 0.6 us).  A row's O is only rescaled when its maximum grew by more than 2^8 since the value in use.  Two CTAs fit an SM,
// one's softmax beside the other's products.
constexpr int kPageBytes = kTileBytes;                 // K or V of one page and head
constexpr int kPrefixQBytes = 128 * kHeadDim * 2;
constexpr int kPageStages = 2;
constexpr int kPrefixTileBytes = kPrefixQBytes + 2 * kPageStages * kPageBytes;
constexpr int kPrefixBars = 16;
constexpr uint32_t kPrefixTmemCols = 256;              // S 0-63, 64-127; O 128-255
constexpr float kPrefixRescale = 8.0f;

enum { BAR_Q = 0, BAR_QFREE = 1, BAR_KFULL = 2, BAR_KFREE = 4, BAR_VFULL = 6, BAR_VFREE = 8, BAR_S = 10, BAR_P = 12, BAR_O = 14 };

constexpr int kPrefixTmemWarp = 4;
__device__ __forceinline__ void shared_prefix_tmem(uint32_t slot) {
    tmem_alloc(slot, kPrefixTmemCols);
    tmem_relinquish();
    tc_fence_before();
}

// warps 0-3 softmax, warp 4 MMA issue, warps 5 and 6 TMA; the CTA's other warps only wait at its barriers.  `smem`: kPrefixTileBytes
// on a 1024-byte boundary.
__device__ __forceinline__ void shared_prefix_role(const SharedPlan& plan, const SharedGroups& shared, const CUtensorMap& q_map,
                                                   const CUtensorMap& k_map, const CUtensorMap& v_map, unsigned char* smem, uint32_t bar0,
                                                   const int32_t* page_table, int max_pages, int num_pages, int hkv, uint32_t* status,
                                                   int cta, int tid, uint32_t tmem_base) {
    const uint32_t sbase = smem_addr(smem);
    const uint32_t q_at = sbase, k_at = sbase + kPrefixQBytes, v_at = k_at + kPageStages * kPageBytes;
    auto bar = [&](int i) { return bar0 + 8u * i; };
    const int warp = tid >> 5, lane = tid & 31;
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
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    struct Item {
        int group, tile, head, split, splits, page0, pages, table_row;
    };
    auto locate = [&](int item) {
        Item it;
        int lo = 0, hi = plan.groups;             // last group with items[g] <= item (a group without pieces never is)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (plan.items[mid] <= item) lo = mid; else hi = mid;
        }
        it.group = lo;
        it.splits = (plan.pages[lo] + plan.piece - 1) / plan.piece;
        const int r = item - plan.items[lo];
        it.split = r % it.splits;
        it.head = (r / it.splits) % hkv;
        it.tile = r / (it.splits * hkv);
        it.page0 = it.split * plan.piece;
        it.pages = plan.pages[lo] - it.page0 < plan.piece ? plan.pages[lo] - it.page0 : plan.piece;
        it.table_row = plan.leader[lo];
        return it;
    };
    bool dead = false;

    if (warp == 5 || warp == 6) {
        // --------------------------------------------- TMA loads: warp 5 queries and K, warp 6 V, neither behind the other
        if (lane == 0) {
            const bool keys = warp == 5;
            const int full = keys ? BAR_KFULL : BAR_VFULL, free = keys ? BAR_KFREE : BAR_VFREE;
            const uint32_t ring = keys ? k_at : v_at;
            const CUtensorMap* map = keys ? &k_map : &v_map;
            int n = 0, local = 0;
            for (int item = cta; item < plan.n_items; item += plan.ctas, ++local) {
                const Item it = locate(item);
                if (keys) {
                    if (!mbar_wait_bounded(bar(BAR_QFREE), (local & 1) ^ 1, dead)) atomicOr(status, QM_DEVSTAT_TIMEOUT);
                    mbar_arrive_expect_tx(bar(BAR_Q), kPrefixQBytes);
                    for (int half = 0; half < 2; ++half)
                        tma_load_3d(q_at + half * (kPrefixQBytes / 2), &q_map, bar(BAR_Q), half * 64, 2 * it.head,
                                    plan.starts[it.group] + it.tile * kStreamsPerTile);
                }
                const int32_t* table = page_table + (size_t)it.table_row * max_pages + it.page0;
                int next_id = table[0];
                for (int j = 0; j < it.pages; ++j, ++n) {
                    int id = next_id;
                    if (j + 1 < it.pages) next_id = table[j + 1];
                    if (id < 0 || id >= num_pages) {
                        atomicOr(status, QM_DEVSTAT_BAD_PAGE);
                        id = 0;
                    }
                    const int y = (id * hkv + it.head) * kPageTokens;
                    const int st = n % kPageStages;
                    if (!mbar_wait_bounded(bar(free + st), ((n / kPageStages) & 1) ^ 1, dead)) atomicOr(status, QM_DEVSTAT_TIMEOUT);
                    mbar_arrive_expect_tx(bar(full + st), kPageBytes);
                    for (int half = 0; half < 2; ++half)
                        tma_load_2d(ring + st * kPageBytes + half * (kPageBytes / 2), map, bar(full + st), half * 64, y);
                }
            }
            // every copy has landed (bounded) before this thread, and with it the CTA, goes
            bool gave_up = false;
            if (keys && local > 0) mbar_wait_bounded(bar(BAR_Q), (local - 1) & 1, gave_up);
            for (int i = n > kPageStages ? n - kPageStages : 0; i < n; ++i)
                mbar_wait_bounded(bar(full + i % kPageStages), (i / kPageStages) & 1, gave_up);
        }
        __syncwarp();
    } else if (warp == 4) {
        // ------------------------------------------------------------- MMA issue
        if (lane == 0) {
            constexpr uint32_t idesc_qk = umma_instr_desc(128, kPageTokens, false);
            constexpr uint32_t idesc_pv = umma_instr_desc(128, kHeadDim, true);
            auto issue_s = [&](int n) {
                const uint32_t ka = k_at + (n % kPageStages) * kPageBytes;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    mma_ss(tmem_base + (n & 1) * 64, smem_desc(q_at + (ks >> 2) * (kPrefixQBytes / 2) + (ks & 3) * 32, 16, 1024),
                           smem_desc(ka + (ks >> 2) * (kPageBytes / 2) + (ks & 3) * 32, 16, 1024), idesc_qk, ks > 0);
                tc_commit(bar(BAR_S + (n & 1)));
                tc_commit(bar(BAR_KFREE + n % kPageStages));
            };
            auto wait = [&](int which, uint32_t parity) {
                if (!mbar_wait_bounded(bar(which), parity, dead)) atomicOr(status, QM_DEVSTAT_TIMEOUT);
            };
            int n = 0, local = 0;
            for (int item = cta; item < plan.n_items; item += plan.ctas, ++local) {
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
                    const uint32_t va = v_at + (n % kPageStages) * kPageBytes;
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
    } else if (warp < 4) {
        // --------------------------------------------------------------- softmax, a thread per query row
        const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
        const float c = 1.4426950408889634f / sqrtf((float)kHeadDim);       // scale * log2(e)
        auto wait = [&](int which, uint32_t parity) {
            if (!mbar_wait_bounded(bar(which), parity, dead) && lane == 0) atomicOr(status, QM_DEVSTAT_TIMEOUT);
        };
        int n = 0;
        for (int item = cta; item < plan.n_items; item += plan.ctas) {
            const Item it = locate(item);
            const int group_streams = plan.starts[it.group + 1] - plan.starts[it.group];
            const int place = it.tile * kStreamsPerTile + (tid >> 1);       // row = 2 * place in the tile + query head
            const bool real = place < group_streams && plan.part[plan.starts[it.group] + place] != 0;       // other rows are not stored
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
                const bool grow = m_new > m_used + kPrefixRescale;
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
            const int group_rows = 2 * group_streams, row = 2 * place + (tid & 1);
            const size_t block = (size_t)plan.rows[it.group] + (size_t)(it.head * it.splits + it.split) * group_rows;
            float4* dst = shared.partial_o + block * (kHeadDim / 4) + row;
#pragma unroll
            for (int cch = 0; cch < 4; ++cch) {
                uint32_t oreg[32];
                tmem_ld32(tmem_base + lane_base + 128 + cch * 32, oreg);
                tmem_wait_ld();
                if (real && !dead) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        dst[(size_t)(cch * 8 + i / 4) * group_rows] = make_float4(__uint_as_float(oreg[i]), __uint_as_float(oreg[i + 1]),
                                                                                 __uint_as_float(oreg[i + 2]), __uint_as_float(oreg[i + 3]));
                }
            }
            if (real && !dead) shared.partial_ml[block + row] = make_float2(m_used, l);
            tc_fence_before();
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kPrefixTmemWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kPrefixTmemCols);
    }
}

// The launch that does both (qm_decode.cu): partial results of the shared pages into groups.partial_*, those of the
// streams' own pages into own_partials [batch][q_heads][130] as qm_decode_attention_partial has them.
int32_t qm_launch_decode_shared(qm_kv_pool* pool, int32_t layer, const uint16_t* q_rot, const CUtensorMap& q_map, const int32_t* seq_lens,
                                const int32_t* page_table, int32_t max_pages, int32_t batch, float* own_partials, void* workspace,
                                const SharedGroups& groups, cudaStream_t stream);
