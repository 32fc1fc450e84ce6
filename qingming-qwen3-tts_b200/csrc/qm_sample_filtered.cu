// Sampling from given uniform numbers with temperature, top-k, top-p and min-p, every row with parameters of its own.
//
// For a row of scores z (bf16 or fp32, up to 262 144 of them) with temperature T > 0:
//   w_i  = exp((z_i - max z) / T)
//   order: z descending, index ascending among equals
//   top-k  keeps the first k of that order
//   top-p  keeps, of those, every entry whose predecessors' weights sum to less than p times the sum over all of them
//   min-p  keeps, of those, w_i >= min_p  (the largest weight is 1)
//   draw   the lowest index i, in INDEX order, at which the kept weights up to and including w_i exceed u * their sum
// T <= 0 takes the first of the order.  No counterpart in the reference, whose sampler draws from at most 4096 codes with
// top-k only and a generator of its own (gpu_sample_topk_f32_kernel, 17.cu:7546); qm_final_head_sample is that one, and
// the processed scores it writes can be sampled here.
//
// Sums are whole numbers: a weight is worked out in double (to about 1e-13) and rounded to a multiple of 2^-45, so that
// sums over 2^18 weights fit 64 bits, are exact, and do not depend on the order of atomics; a weight below 2^-46 of the
// largest is zero and out of the game.
//
// A row is spread over a cluster of up to eight CTAs; the scores come from the L2 for every sweep after the first.
// Nothing is sorted as a whole: a sweep puts the entries (for top-p their weights too) into 1024 bins that are even in z,
// the CTAs add their bins up, a slice of them each, and every CTA finds the bin in which top-k (or top-p) ends by the
// same scan.  The few entries of that bin are gathered and put in order.  A bin with more than 512 entries
// (many equal scores) is first cut down by digits of the entries' keys, which contain the index and therefore differ.  Where
// top-k leaves few entries, they are gathered as a whole, and top-p, min-p and the draw need no sweep any more.
// What bounds it: in many bf16 rows with top-p, instructions (a weight is about 40, twelve of them in double precision; 143 warp
// instructions per 32 scores in all, at 2.1 of them per cycle); in few large fp32 rows and in small ones, the steps' latency (61
// per 32 scores at 0.95 per cycle).  Measured: one row of 2048 with top-k 6.7 us, 64
// rows of 2048 with everything 12 us, 32 rows of 131 072 fp32 44-45 us, 96 rows of 100 003 bf16 28 us without filters, 27 us
// with top-k 50 (and top-p and min-p behind it), 18 us with min-p, 81-82 us with top-p 0.7 to 1.  Tried and slower, when that took
// 92: the scores kept in shared memory (196 us; fewer CTAs fit), clusters of three with two CTAs on every SM (125 us), 512
// threads per CTA (103 us, though 45 instead of 50 us at 131 072).
#include <math_constants.h>

#include <cfloat>

#include "qm_cluster.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kBinsPerThread = kBins / kThreads;
constexpr int kList = 512;
constexpr int kIndexBits = 18;
constexpr int kMaxVocab = 1 << kIndexBits;
constexpr int kMaxCluster = 8;
constexpr int kCtasPerSm = 3;
constexpr int kTable = 16;                      // 128 bytes: lanes with different entries meet no bank twice
constexpr double kUnit = 35184372088832.0;      // 2^45: the whole number that stands for weight 1

typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    int64_t row_stride;          // elements
    const float* uniforms;
    const float* temperature;    // null: 1
    const int32_t* top_k;        // null or <= 0: off
    const float* top_p;          // null or not < 1: off
    const float* min_p;          // null or not > 0: off
    int32_t* tokens;
    float* probs;                // or null
    int vocab;
    int cluster;
};

// Behind the bins, a word per lane for the entries that are not in the game: adding them up there takes no branch.
struct Bins {
    uint32_t count[kBins + 32];
    uint32_t low[kBins + 32];    // sums of the weights, low and high 32 bits
    uint32_t high[kBins + 32];
};

struct Smem {
    Bins own, sum;               // of this CTA; of the cluster
    u64 list[kList];             // this CTA's entries of the chosen bin
    ulonglong2 all[kList];       // the cluster's: key, weight
    double table[kTable];        // 2^(j / 16) * 2^45
    u64 scan_mass[kWarps];
    float2 range[kMaxCluster];   // one from every CTA: largest and lowest score
    u64 totals[kMaxCluster];
    float2 scan_range[kWarps];
    uint32_t scan_count[kWarps];
    uint32_t list_count;
    uint32_t found;
    // the chosen bin
    u64 before_mass;
    uint32_t before_count, upto_count, bin;
};

__device__ __forceinline__ float fmin3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ u64 ld_cluster_u64(uint32_t addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr));
    return v;
}

// Larger is earlier in the order: monotone image of the score above the inverted index.
__device__ __forceinline__ u64 entry_key(float score, int index) {
    const uint32_t bits = __float_as_uint(score);
    const uint32_t image = (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
    return ((u64)image << kIndexBits) | (u64)(kMaxVocab - 1 - index);
}
__device__ __forceinline__ float key_score(u64 key) {
    const uint32_t image = (uint32_t)(key >> kIndexBits);
    return __uint_as_float((image & 0x80000000u) ? (image & 0x7fffffffu) : ~image);
}
__device__ __forceinline__ int key_index(u64 key) { return kMaxVocab - 1 - (int)(key & (kMaxVocab - 1)); }

// 2^45 exp((x - top) / T):  e = (x - top) / T = k ln2 / 16 + r with |r| <= ln2 / 32; 2^(k / 16) from a table, exp(r) by the first
// six terms of its series (the seventh is below 2e-13).  A float becomes a double by moving its fields, which is a third of
// the time of a conversion and takes a zero or a subnormal for a number below 2^-126; where T is so small that this could
// be seen, by conversion.  For NaN, infinities and scores below the cutoff the result means nothing: callers compare with it (above it e > -66, where
// the exponent's field cannot wrap, and below -31.9 the weight is less than half of 2^-45 and rounds to zero).
struct Weigher {
    const double* table;
    double top, inverse;         // 1 / T
    bool convert;
    bool infinite;               // top is +inf: only the scores equal to it have a weight

    __device__ __forceinline__ double exponential(double wide) const {
        const double e = (wide - top) * inverse;
        constexpr double kMagic = 6755399441055744.0;             // 1.5 * 2^52: the low word of a sum holds its rounding
        const double shifted = fma(e, 23.083120654223414219, kMagic);      // 16 / ln2
        const int k = __double2loint(shifted);
        const double r = fma(shifted - kMagic, -0.043321698784996581, e);  // ln2 / 16
        double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
        p = fma(p, r, 1.0 / 6.0);
        p = fma(p, r, 0.5);
        p = fma(p, r, 1.0);
        p = fma(p, r, 1.0);
        p *= table[k & (kTable - 1)];
        return __hiloint2double(__double2hiint(p) + (k >> 4) * (1 << 20), __double2loint(p));
    }
    __device__ __forceinline__ double common(float x) const {
        const uint32_t bits = __float_as_uint(x);
        return exponential(__hiloint2double((int)((bits & 0x80000000u) | (((bits & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(bits << 29)));
    }
    __device__ __noinline__ double rare(float x) const {
        if (infinite) return x == (float)top ? kUnit : 0.0;
        return exponential((double)x);
    }
    __device__ __forceinline__ double operator()(float x) const { return convert || infinite ? rare(x) : common(x); }
};

// The nearest whole number of 0 .. 2^45.
__device__ __forceinline__ u64 whole(double w) {
    const double d = w + 4503599627370496.0;                      // 2^52
    return ((u64)((uint32_t)__double2hiint(d) & 0xfffffu) << 32) | (uint32_t)__double2loint(d);
}

template <typename T>
__device__ __forceinline__ T warp_inclusive(T v, int lane) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const T t = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += t;
    }
    return v;
}

template <bool kFp32>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) qm_sample_filtered_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    Smem& s = *reinterpret_cast<Smem*>(raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cluster = a.cluster;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    const int row = blockIdx.x / cluster;
    const int slice = (a.vocab + cluster - 1) / cluster;
    const int begin = rank * slice < a.vocab ? rank * slice : a.vocab;
    const int n = (begin + slice < a.vocab ? begin + slice : a.vocab) - begin;
    const uint32_t self = smem_addr(raw);
    auto remote = [&](const void* mine, int r) { return map_to_rank(self + (uint32_t)((const unsigned char*)mine - raw), (uint32_t)r); };
    auto sync_all = [&]() {
        if (cluster > 1) cluster_sync_all();
        else __syncthreads();
    };

    pdl_trigger();
    if (cluster > 1) cluster_arrive_relaxed();    // "I have started": a CTA's shared memory is only written to after that
    if (tid < kTable) s.table[tid] = exp2((double)tid / kTable) * kUnit;
    for (int i = tid; i < kBins; i += kThreads) s.own.count[i] = s.own.low[i] = s.own.high[i] = 0u;
    pdl_wait();

    // The slice in blocks of 256 scores, eight to a lane, on 16-byte boundaries: `lead` scores of the first block and some of
    // the last belong to others and are filled with -inf.
    constexpr int kBytes = kFp32 ? 4 : 2;
    const unsigned char* base = static_cast<const unsigned char*>(a.logits) + ((size_t)row * a.row_stride + begin) * kBytes;
    const int lead = (int)((reinterpret_cast<uintptr_t>(base) & 15u) / kBytes);
    base -= lead * kBytes;
    const int blocks = (lead + n + 255) / 256;
    struct Eight {
        uint4 a, b;              // bf16: a alone
    };
    auto load = [&](int block) {
        Eight e;
        const int v = block * 256 + lane * 8;
        if (v >= lead && v + 8 <= lead + n) {
            e.a = *reinterpret_cast<const uint4*>(base + (size_t)v * kBytes);
            if (kFp32) e.b = *reinterpret_cast<const uint4*>(base + (size_t)v * kBytes + 16);
        } else {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = v + j >= lead && v + j < lead + n;
                if (kFp32) w[j] = in ? *reinterpret_cast<const uint32_t*>(base + (size_t)(v + j) * 4) : 0xff800000u;
                else w[j] = in ? *reinterpret_cast<const uint16_t*>(base + (size_t)(v + j) * 2) : 0xff80u;
            }
            if (kFp32) {
                e.a = make_uint4(w[0], w[1], w[2], w[3]);
                e.b = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
                e.a = make_uint4(w[0] | (w[1] << 16), w[2] | (w[3] << 16), w[4] | (w[5] << 16), w[6] | (w[7] << 16));
            }
        }
        return e;
    };
    auto score = [](const Eight& e, int j) {
        const uint32_t* w = kFp32 && j >= 4 ? reinterpret_cast<const uint32_t*>(&e.b) : reinterpret_cast<const uint32_t*>(&e.a);
        if (kFp32) return __uint_as_float(w[j & 3]);
        return __uint_as_float((j & 1) ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
    };
    // f(block, index of the lane's first score in the slice, the eight): a warp has every eighth block, one ahead in flight
    auto sweep = [&](auto f) {
        if (warp >= blocks) return;
        Eight next = load(warp);
        for (int block = warp; block < blocks; block += kWarps) {
            const Eight e = next;
            if (block + kWarps < blocks) next = load(block + kWarps);
            f(block, block * 256 + lane * 8 - lead, e);
        }
    };

    // ---- the largest score and the lowest above -inf, of the row
    float top = -CUDART_INF_F, lowest = CUDART_INF_F;
    sweep([&](int, int, const Eight& e) {         // neither is ever NaN
        float low = CUDART_INF_F;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            top = fmax3(top, score(e, j), score(e, j + 1));
            low = fmin3(low, score(e, j), score(e, j + 1));
        }
        if (low == -CUDART_INF_F) {
            low = CUDART_INF_F;
#pragma unroll
            for (int j = 0; j < 8; ++j) low = fminf(low, score(e, j) > -CUDART_INF_F ? score(e, j) : CUDART_INF_F);
        }
        lowest = fminf(lowest, low);
    });
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        lowest = fminf(lowest, __shfl_xor_sync(0xffffffffu, lowest, off));
    }
    if (lane == 0) s.scan_range[warp] = make_float2(top, lowest);
    __syncthreads();
    if (cluster > 1) cluster_wait();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        top = fmaxf(top, s.scan_range[w].x);
        lowest = fminf(lowest, s.scan_range[w].y);
    }
    if (cluster > 1) {
        if (tid < cluster)
            st_cluster_u64(remote(&s.range[rank], tid), ((u64)__float_as_uint(lowest) << 32) | __float_as_uint(top));
        cluster_sync_all();
        for (int r = 0; r < cluster; ++r) {
            top = fmaxf(top, s.range[r].x);
            lowest = fminf(lowest, s.range[r].y);
        }
    }
    top += 0.0f;                                  // -0 becomes +0
    const float temperature = a.temperature ? a.temperature[row] : 1.0f;
    if (top == -CUDART_INF_F || !(temperature > 0.0f)) {        // nothing to draw from, or nothing to draw
        if (top == -CUDART_INF_F) {
            if (rank == 0 && tid == 0) {
                a.tokens[row] = -1;
                if (a.probs) a.probs[row] = 0.0f;
            }
            return;
        }
        // the lowest index of the largest score
        uint32_t at = 0xffffffffu;
        sweep([&](int, int i0, const Eight& e) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (score(e, j) == top) at = min(at, (uint32_t)(begin + i0 + j));
        });
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) s.scan_count[warp] = at;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) at = min(at, s.scan_count[w]);
        if (cluster > 1) {
            if (tid < cluster) st_cluster_u64(remote(&s.totals[rank], tid), at);
            cluster_sync_all();
            for (int r = 0; r < cluster; ++r) at = min(at, (uint32_t)s.totals[r]);
        }
        if (rank == 0 && tid == 0) {
            a.tokens[row] = (int)at;
            if (a.probs) a.probs[row] = 1.0f;
        }
        return;
    }

    const Weigher weight{s.table, (double)top, 1.0 / (double)temperature, temperature < 0x1p-60f, top == CUDART_INF_F};
    // entries below this have no weight (a float next to it is either 32 T below the top, or no other float lies between)
    const float cutoff = top == CUDART_INF_F ? top : fmaxf(top - 32.5f * temperature, -FLT_MAX);
    // Bins even in z between the largest score and the lowest one that can matter.  Each operation is monotone, so a larger
    // score never has a larger bin; NaN (equal infinities, 0 * inf) comes only where all entries in question are equal or
    // the last of all, and is the last bin.
    const float range = fminf(top - lowest, 32.0f * temperature), per_bin = (float)kBins / range;
    auto bin_of = [&](float x) {
        return (int)(__float_as_uint(fminf((top - x) * per_bin, (float)(kBins - 1)) + 8388608.0f) & (kBins - 1));
    };
    // Eight weights without a branch between them, so that their chains of dependent operations overlap.
    auto weigh = [&](const Eight& e, u64 (&q)[8]) {
        if (weight.convert || weight.infinite) {
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = whole(weight.rare(score(e, j)));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = whole(weight.common(score(e, j)));
        }
    };
    float threshold = -CUDART_INF_F;              // what stays: scores above it, and at it the indices up to threshold_index
    int threshold_index = -1;                     // (of the slice)
    auto stays = [&](float x, int i) { return x > threshold || (x == threshold && i <= threshold_index); };

    // The first n entries of s.all into descending order of key & mask, by a bitonic network over the next power of two (returned;
    // what is behind the entries is zero).  A warp's pairs at distances up to 32 lie in 64 entries of its own.
    auto sort_list = [&](int n, u64 mask) {
        int size_all = 64;
        while (size_all < n) size_all *= 2;
        __syncthreads();
        for (int i = n + tid; i < size_all; i += kThreads) s.all[i] = make_ulonglong2(0ull, 0ull);      // behind every entry
        __syncthreads();
        for (int size = 2; size <= size_all; size *= 2) {
            for (int stride = size / 2; stride > 0; stride /= 2) {
                if (tid < size_all / 2) {
                    const int lo = 2 * tid - (tid & (stride - 1)), hi = lo + stride;
                    const ulonglong2 x = s.all[lo], y = s.all[hi];
                    if (((x.x & mask) < (y.x & mask)) == ((lo & size) == 0)) {
                        s.all[lo] = y;
                        s.all[hi] = x;
                    }
                }
                if (stride > 32 || (stride == 1 && size >= 64)) __syncthreads();
                else __syncwarp();
            }
        }
        return size_all;
    };
    // Sum over the block of a value of every thread, and of the threads before this one.
    auto scan_block = [&](u64 v, u64& total) {
        const u64 to = warp_inclusive(v, lane);
        __syncthreads();
        if (lane == 31) s.scan_mass[warp] = to;
        __syncthreads();
        u64 ahead = to - v;
        total = 0ull;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            ahead += w < warp ? s.scan_mass[w] : 0ull;
            total += s.scan_mass[w];
        }
        return ahead;
    };
    // The first n entries of s.all in descending order of key & mask: every entry, its place in the order and the weight in front of
    // it in some thread (two at most).  Up to 128 entries stay where they are and are counted, two to eight threads to an
    // entry; more are sorted.  Measured: a row of 2048 with top-k 50 counted 6.1, sorted 10.2 us; 96 rows with some 300 entries
    // at top-p's border counted 94, sorted 81 us (rows with 200 entries for top-k 43.7 and 39.4 us).
    struct Ordered {
        u64 key[2], weight[2], ahead[2];          // none: key ~0, weight 0
        int place[2], slot[2];                    // slot in s.all, or -1
    };
    auto order_list = [&](int n, u64 mask, Ordered& o) {
        u64 total;
        if (n > kThreads / 2) {
            const int sorted = sort_list(n, mask);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                o.slot[e] = o.place[e] = 2 * tid + e;
                const ulonglong2 entry = o.slot[e] < sorted ? s.all[o.slot[e]] : make_ulonglong2(0ull, 0ull);
                if (entry.x == 0ull) o.slot[e] = -1;
                o.key[e] = entry.x == 0ull ? ~0ull : entry.x;
                o.weight[e] = entry.y;
            }
            o.ahead[0] = scan_block(o.weight[0] + o.weight[1], total);
            o.ahead[1] = o.ahead[0] + o.weight[0];
            return total;
        }
        const int t = n <= kThreads / 8 ? 8 : (n <= kThreads / 4 ? 4 : 2), i = tid / t;
        const u64 key = i < n ? s.all[i].x : ~0ull;
        u64 ahead = 0ull;
        int place = 0;
#pragma unroll 4
        for (int j = tid & (t - 1); j < n; j += t) {
            const ulonglong2 other = s.all[j];
            const bool before = (other.x & mask) > (key & mask);
            place += before ? 1 : 0;
            ahead += before ? other.y : 0ull;
        }
        for (int off = 1; off < t; off <<= 1) {
            place += __shfl_xor_sync(0xffffffffu, place, off);
            ahead += __shfl_xor_sync(0xffffffffu, ahead, off);
        }
        const bool mine = i < n && (tid & (t - 1)) == 0;
        o = {{mine ? key : ~0ull, ~0ull}, {mine ? s.all[i].y : 0ull, 0ull}, {ahead, 0ull}, {place, 0}, {mine ? i : -1, -1}};
        scan_block(o.weight[0], total);
        return total;
    };
    static_assert(kList == 2 * kThreads, "two entries per thread");

    // The last entry of the order, among those that stay so far, whose predecessors count less than k (by_mass false) or
    // weigh less than p times all of them: the new threshold.
    // For a count, where the bin and all before it are few, they are listed (keys and weights, in the first CTA) and the rest
    // of the row's work is done there: returns their number, otherwise 0.  Few: what the list holds if p < 1, which saves the
    // sweeps of that search (96 rows of 100 003, top-k 200 and top-p 65.6 -> 40 us), otherwise what is counted and not
    // sorted (top-k 50 32.3 -> 26.5 us; for 200 the sweep of the draw takes 36.5 us, sorting 40).
    auto search = [&](bool by_mass, int k, float p, bool bins_are_clear) -> int {
        int shift = 64, bin = 0;                  // from the second round on: the chosen bin, keys that agree with prefix above `shift`
        u64 prefix = 0ull, limit = (u64)k;
        uint32_t ahead_count = 0;
        u64 ahead_mass = 0;
        int found = 0;
        constexpr int kShifts[6] = {40, 30, 20, 10, 0, 0};
        // entries of the chosen bin that agree with the digits so far
        auto matches = [&](float x, int i) {
            if (!(x >= cutoff) || bin_of(x) != bin || !stays(x, i)) return false;
            return shift >= 64 || (entry_key(x + 0.0f, begin + i) >> shift) == (prefix >> shift);
        };
        for (int round = 0; round < 6; ++round) {
            if (round > 0 || !bins_are_clear) {
                for (int i = tid; i < kBins; i += kThreads) s.own.count[i] = s.own.low[i] = s.own.high[i] = 0u;
                __syncthreads();
            }
            const int next = round > 0 ? kShifts[round - 1] : 0;
            sweep([&](int, int i0, const Eight& e) {
                int b[8];
                if (round == 0 && threshold == -CUDART_INF_F) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) b[j] = score(e, j) >= cutoff ? bin_of(score(e, j)) : kBins + lane;
                } else {
                    bool any = false;             // most blocks have nothing to add any more
#pragma unroll
                    for (int j = 0; j < 8; ++j) any |= score(e, j) >= threshold && score(e, j) >= cutoff;
                    if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float x = score(e, j);
                        const bool in = round > 0 ? matches(x, i0 + j) : x >= cutoff && stays(x, i0 + j);
                        const int digit = kBins - 1 - (int)((entry_key(x + 0.0f, begin + i0 + j) >> next) & (u64)(kBins - 1));
                        b[j] = in ? (round > 0 ? digit : bin_of(x)) : kBins + lane;
                    }
                }
                if (!by_mass) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) atomicAdd(&s.own.count[b[j]], 1u);
                    return;
                }
                // the low words first, all of them, then what carries into the high words
                u64 q[8];
                uint32_t old[8];
                weigh(e, q);
#pragma unroll
                for (int j = 0; j < 8; ++j) old[j] = atomicAdd(&s.own.low[b[j]], (uint32_t)q[j]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t hi = (uint32_t)(q[j] >> 32) + (old[j] + (uint32_t)q[j] < old[j] ? 1u : 0u);
                    if (hi) atomicAdd(&s.own.high[b[j]], hi);
                }
            });
            sync_all();
            const Bins* bins = &s.own;
            if (cluster > 1) {
                // this CTA adds up its slice of the bins and hands it to everyone
                bins = &s.sum;
                const int width = kBins / cluster;
                for (int b = rank * width + tid; b < (rank + 1) * width; b += kThreads) {
                    uint32_t c[kMaxCluster], lo[kMaxCluster], hi[kMaxCluster];
#pragma unroll
                    for (int r = 0; r < kMaxCluster; ++r) {
                        c[r] = lo[r] = hi[r] = 0u;
                        if (r < cluster) {
                            if (!by_mass) {
                                c[r] = ld_cluster_u32(remote(&s.own.count[b], r));
                            } else {
                                lo[r] = ld_cluster_u32(remote(&s.own.low[b], r));
                                hi[r] = ld_cluster_u32(remote(&s.own.high[b], r));
                            }
                        }
                    }
                    uint32_t count = 0;
                    u64 mass = 0;
#pragma unroll
                    for (int r = 0; r < kMaxCluster; ++r) {
                        count += c[r];
                        mass += ((u64)hi[r] << 32) + lo[r];
                    }
                    for (int r = 0; r < cluster; ++r) {
                        if (!by_mass) {
                            st_cluster_u32(remote(&s.sum.count[b], r), count);
                        } else {
                            st_cluster_u32(remote(&s.sum.low[b], r), (uint32_t)mass);
                            st_cluster_u32(remote(&s.sum.high[b], r), (uint32_t)(mass >> 32));
                        }
                    }
                }
                cluster_sync_all();
            }
            // the last bin with an entry whose predecessors measure less than the limit
            uint32_t c[kBinsPerThread], count = 0;
            u64 m[kBinsPerThread], mass = 0;
#pragma unroll
            for (int j = 0; j < kBinsPerThread; ++j) {
                const int b = tid * kBinsPerThread + j;
                c[j] = by_mass ? 0u : bins->count[b];
                m[j] = by_mass ? ((u64)bins->high[b] << 32) + bins->low[b] : 0ull;
                count += c[j];
                mass += m[j];
            }
            const uint32_t count_to = warp_inclusive(count, lane);
            const u64 mass_to = by_mass ? warp_inclusive(mass, lane) : 0ull;
            if (lane == 31) {
                s.scan_count[warp] = count_to;
                s.scan_mass[warp] = mass_to;
            }
            if (tid == 0) {
                s.found = 0u;
                s.list_count = 0u;
            }
            __syncthreads();
            uint32_t cb = ahead_count + count_to - count;
            u64 mb = ahead_mass + mass_to - mass, total = 0ull;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) {
                    cb += s.scan_count[w];
                    mb += s.scan_mass[w];
                }
                total += s.scan_mass[w];
            }
            if (by_mass && round == 0) {
                const double wanted = ceil((double)p * (double)total);
                limit = wanted > 1.0 ? (u64)wanted : 1ull;
            }
            int mine = -1;
            uint32_t my_count = 0, my_upto = 0;
            u64 my_mass = 0;
#pragma unroll
            for (int j = 0; j < kBinsPerThread; ++j) {
                if ((by_mass ? m[j] != 0ull && mb < limit : c[j] != 0u && (u64)cb < limit)) {
                    mine = tid * kBinsPerThread + j;
                    my_count = cb;
                    my_upto = cb + c[j];
                    my_mass = mb;
                }
                cb += c[j];
                mb += m[j];
            }
            if (mine >= 0) atomicMax(&s.found, (uint32_t)mine + 1u);
            __syncthreads();
            if (mine >= 0 && s.found == (uint32_t)mine + 1u) {
                s.bin = (uint32_t)mine;
                s.before_count = my_count;
                s.upto_count = my_upto;
                s.before_mass = my_mass;
            }
            __syncthreads();
            ahead_count = s.before_count;
            ahead_mass = s.before_mass;
            if (round == 0) {
                bin = (int)s.bin;
            } else {
                prefix |= (u64)(kBins - 1 - (int)s.bin) << next;
                shift = next;
            }
            // the bin's entries, from all CTAs into all CTAs, if the list holds them; most scores are ruled out by an interval
            // a hundredth of a bin wider than the bin on either side (bin_of's roundings are a ten-thousandth)
            float from = cutoff, to = CUDART_INF_F;
            const bool list_all = !by_mass && round == 0 && s.upto_count <= (uint32_t)(p < 1.0f ? kList : kThreads / 2);
            if (per_bin > 0.0f && per_bin < CUDART_INF_F) {
                const double width = (double)range * (1.0 / kBins);
                if (bin < kBins - 1) from = fmaxf(from, __double2float_rd((double)top - ((double)bin + 0.51) * width));
                if (!list_all) to = __double2float_ru((double)top - ((double)bin - 0.51) * width);
                if (!(to == to)) to = CUDART_INF_F;          // an infinite top or range
            }
            sweep([&](int, int i0, const Eight& e) {
                bool near = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) near |= score(e, j) >= from && score(e, j) <= to;
                if (!near) return;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = score(e, j);
                    if (list_all ? !(x >= cutoff) || bin_of(x) > bin : !matches(x, i0 + j)) continue;
                    const uint32_t at = atomicAdd(&s.list_count, 1u);
                    if (at < kList) s.list[at] = entry_key(x + 0.0f, begin + i0 + j);
                }
            });
            sync_all();
            found = 0;
            for (int r = 0; r < cluster && (!list_all || rank == 0); ++r) {
                const int there = (int)(cluster > 1 ? ld_cluster_u32(remote(&s.list_count, r)) : s.list_count);
                for (int i = tid; i < there && found + i < kList; i += kThreads) {
                    const u64 key = cluster > 1 ? ld_cluster_u64(remote(&s.list[i], r)) : s.list[i];
                    s.all[found + i] = make_ulonglong2(key, by_mass || list_all ? whole(weight(key_score(key))) : 1ull);
                }
                found += there;
            }
            if (list_all) return (int)s.upto_count;
            if (found <= kList) break;
            sync_all();                           // the others' lists have been looked at
        }
        __syncthreads();
        Ordered o;
        order_list(found, ~0ull, o);
        u64 last = ~0ull;
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (o.ahead[e] + (by_mass ? ahead_mass : (u64)ahead_count) < limit && o.key[e] < last) last = o.key[e];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            const u64 other = __shfl_xor_sync(0xffffffffu, last, off);
            last = other < last ? other : last;
        }
        __syncthreads();
        if (lane == 0) s.scan_mass[warp] = last;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) last = s.scan_mass[w] < last ? s.scan_mass[w] : last;
        __syncthreads();
        threshold = key_score(last);
        threshold_index = key_index(last) - begin;
        return 0;
    };

    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float min_p = a.min_p ? a.min_p[row] : 0.0f;
    const bool cut_k = k > 0 && k < a.vocab;
    const u64 least = min_p > 0.0f ? (u64)ceil((double)fminf(min_p, 2.0f) * kUnit) : 0ull;
    const double uniform = (double)a.uniforms[row];
    auto target_of = [&](u64 total) {
        const double wanted = uniform * (double)total;
        const u64 target = wanted > 0.0 ? (wanted < (double)total ? (u64)wanted : total - 1ull) : 0ull;
        return target < total ? target : total - 1ull;
    };
    const int listed = cut_k ? search(false, k, p, true) : 0;
    if (listed > 0) {
        // ---- all that can stay is in the first CTA's list: the remaining filters and the draw there
        sync_all();                               // the list is whole, and nobody's is needed any more
        if (rank != 0) return;
        Ordered o;
        order_list(listed, ~0ull, o);
        u64 total, sum = 0ull, limit = ~0ull;
#pragma unroll
        for (int e = 0; e < 2; ++e) sum += o.place[e] < k ? o.weight[e] : 0ull;
        scan_block(sum, total);
        if (p < 1.0f) {
            const double wanted = ceil((double)p * (double)total);
            limit = wanted > 1.0 ? (u64)wanted : 1ull;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (o.slot[e] >= 0 && (o.place[e] >= k || o.ahead[e] >= limit || (o.weight[e] < least && key_score(o.key[e]) != top)))
                s.all[o.slot[e]].y = 0ull;
        __syncthreads();
        total = order_list(listed, (u64)(kMaxVocab - 1), o);      // by index
        const u64 target = target_of(total);
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (target >= o.ahead[e] && target < o.ahead[e] + o.weight[e]) {
                a.tokens[row] = key_index(o.key[e]);
                if (a.probs) a.probs[row] = (float)(weight(key_score(o.key[e])) / (double)total);
            }
        return;
    }
    if (p < 1.0f) search(true, 0, p, !cut_k);

    // ---- the draw: kept weights in index order, summed by blocks (the bins' place is free again)
    // a score below this is out; above it min-p is compared exactly (the margin is far above the errors of logf, and of the
    // weights' own rounding where min_p is not tiny)
    float bound = cutoff;
    if (min_p >= 1.0e-6f) bound = fmaxf(bound, fminf(top, __double2float_rd((double)top + (double)temperature * ((double)logf(min_p) - 1.0e-4))));
    bound = fmaxf(bound, threshold);
    const bool filtered = threshold > -CUDART_INF_F || least > 0ull;
    auto stays_in = [&](float x, int i) { return x >= cutoff && stays(x, i); };
    auto kept = [&](float x, int i) -> u64 {
        const u64 q = whole(weight(x));
        return stays_in(x, i) && (q >= least || x == top) ? q : 0ull;
    };
    u64* block_sum = reinterpret_cast<u64*>(&s.own);
    static_assert((kMaxVocab / 256 + 1) * sizeof(u64) <= sizeof(Bins), "block sums lie where the bins were");
    __syncthreads();
    u64 mine = 0ull;
    float* few = reinterpret_cast<float*>(&s.sum) + warp * 256;          // a warp's scores that stay, of one block
    static_assert(kWarps * 256 * sizeof(float) <= sizeof(Bins), "they lie where the cluster's sums were");
    sweep([&](int block, int i0, const Eight& e) {
        u64 sum = 0ull;
        if (!filtered) {
            u64 q[8];
            weigh(e, q);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += score(e, j) >= cutoff ? q[j] : 0ull;
        } else {
            uint32_t in = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) in |= score(e, j) >= bound ? 1u << j : 0u;
            if (!__any_sync(0xffffffffu, in != 0u)) {
                if (lane == 0) block_sum[block] = 0ull;
                return;
            }
            // at the threshold itself the index decides
#pragma unroll
            for (int j = 0; j < 8; ++j) in &= score(e, j) != threshold || i0 + j <= threshold_index ? 0xffu : ~(1u << j);
            const int upto = warp_inclusive(__popc(in), lane), count = __shfl_sync(0xffffffffu, upto, 31);
            // side by side first, then a weight per lane (weighing all eight in place from 32, 64 or 128 of the 256 on: no faster)
            int at = upto - __popc(in);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (in >> j & 1u) few[at++] = score(e, j);
            __syncwarp();
            for (int i = lane; i < count; i += 32) {
                const float x = few[i];
                const u64 q = whole(weight(x));
                sum += q >= least || x == top ? q : 0ull;
            }
            __syncwarp();
        }
        mine += sum;
        // the warp's sum in two steps of 24 bits (eight weights stay below 2^49): 32 lanes of either fit 32 bits
        const u64 low = __reduce_add_sync(0xffffffffu, (uint32_t)sum & 0xffffffu), high = __reduce_add_sync(0xffffffffu, (uint32_t)(sum >> 24));
        if (lane == 0) block_sum[block] = (high << 24) + low;
    });
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
    if (lane == 0) s.scan_mass[warp] = mine;
    __syncthreads();
    u64 before = 0ull, own = 0ull;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) own += s.scan_mass[w];
    u64 total = own;
    if (cluster > 1) {
        if (tid < cluster) st_cluster_u64(remote(&s.totals[rank], tid), own);
        cluster_sync_all();
        total = 0ull;
        for (int r = 0; r < cluster; ++r) {
            if (r < rank) before += s.totals[r];
            total += s.totals[r];
        }
    }
    const u64 target = target_of(total);
    if (warp > 0 || target < before || target >= before + own) return;
    // The first warp of the CTA that has it: which block, which lane's eight, which of them.
    u64 sum = before;
    for (int block0 = 0; block0 < blocks; block0 += 32) {
        const u64 q = block0 + lane < blocks ? block_sum[block0 + lane] : 0ull;
        const u64 up_to = sum + warp_inclusive(q, lane);
        const unsigned past = __ballot_sync(0xffffffffu, target < up_to);
        if (!past) {
            sum = __shfl_sync(0xffffffffu, up_to, 31);
            continue;
        }
        const int which = __ffs(past) - 1;
        sum = __shfl_sync(0xffffffffu, up_to - q, which);
        const int i0 = (block0 + which) * 256 + lane * 8 - lead;
        const Eight e = load(block0 + which);
        u64 q8[8], eight = 0ull;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            q8[j] = kept(score(e, j), i0 + j);
            eight += q8[j];
        }
        const u64 to = sum + warp_inclusive(eight, lane);
        const unsigned beyond = __ballot_sync(0xffffffffu, target < to);
        if (lane == __ffs(beyond) - 1) {
            u64 at = to - eight;
            bool done = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                at += q8[j];
                if (!done && target < at) {
                    done = true;
                    a.tokens[row] = begin + i0 + j;
                    if (a.probs) a.probs[row] = (float)(weight(score(e, j)) / (double)total);
                }
            }
        }
        return;
    }
}

}  // namespace

extern "C" int32_t qm_sample_filtered(const void* logits, int32_t logits_are_fp32, int64_t row_stride, int32_t batch, int32_t vocab,
                                      const float* uniforms, const float* temperature, const int32_t* top_k, const float* top_p,
                                      const float* min_p, int32_t* tokens_out, float* probs_out, void* stream) {
    if (batch < 0 || vocab < 1 || vocab > kMaxVocab) return qm_fail(QM_EINVAL, "vocab must be between 1 and 262144");
    if (row_stride < 0) return qm_fail(QM_EINVAL, "row_stride must be >= 0");
    if (batch == 0) return QM_OK;
    if (!logits || !uniforms || !tokens_out) return qm_fail(QM_EINVAL, "null tensor pointer");
    const uintptr_t words = reinterpret_cast<uintptr_t>(uniforms) | reinterpret_cast<uintptr_t>(temperature) |
                            reinterpret_cast<uintptr_t>(top_k) | reinterpret_cast<uintptr_t>(top_p) | reinterpret_cast<uintptr_t>(min_p) |
                            reinterpret_cast<uintptr_t>(tokens_out) | reinterpret_cast<uintptr_t>(probs_out);
    if ((words & 3u) || (reinterpret_cast<uintptr_t>(logits) & (logits_are_fp32 ? 3u : 1u)))
        return qm_fail(QM_EINVAL, "misaligned tensor pointer");
    // As many CTAs per row as leave each 2048 scores, up to eight, and no more than fit the GPU at a time.
    const long long fit = (long long)kCtasPerSm * sm_count_of_current_device();
    int cluster = 1;
    while (cluster < kMaxCluster && vocab / (2 * cluster) >= 2048 && (long long)batch * 2 * cluster <= fit) cluster *= 2;
    if ((long long)batch * cluster > 0x7fffffffLL) return qm_fail(QM_ECAPACITY, "too many rows for one launch");
    SampleArgs a{};
    a.logits = logits;
    a.row_stride = row_stride;
    a.uniforms = uniforms;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.tokens = tokens_out;
    a.probs = probs_out;
    a.vocab = vocab;
    a.cluster = cluster;
    auto kernel = logits_are_fp32 ? qm_sample_filtered_kernel<true> : qm_sample_filtered_kernel<false>;
    static_assert(sizeof(Smem) <= 48 * 1024, "no opt-in to more shared memory");
    QM_CUDA_TRY(launch_cluster(kernel, dim3((unsigned)(batch * cluster)), dim3(kThreads), (unsigned)cluster, sizeof(Smem),
                               static_cast<cudaStream_t>(stream), a),
                "filtered sampling launch");
    return QM_OK;
}
