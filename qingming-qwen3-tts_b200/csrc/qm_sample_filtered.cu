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
// same scan.  The few entries of that bin are gathered and ranked by counting.  A bin with more than 512 entries
// (many equal scores) is first cut down by digits of the entries' keys, which contain the index and therefore differ.
// What bounds it: a weight takes eleven double-precision operations, and each step of the cluster a few microseconds of
// latency; rows are few, so as many CTAs as fit work on one wave of them.
#include <math_constants.h>

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
constexpr int kTable = 64;
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

struct Bins {
    uint32_t count[kBins];
    uint32_t low[kBins];         // sums of the weights, low and high 32 bits
    uint32_t high[kBins];
};

struct Smem {
    Bins own, sum;               // of this CTA; of the cluster
    u64 list[kList];             // this CTA's entries of the chosen bin
    ulonglong2 all[kList];       // the cluster's: key, weight
    double table[kTable];        // 2^(j / 64) * 2^45
    u64 scan_mass[kWarps];
    u64 best[kMaxCluster];       // one word from every CTA
    u64 totals[kMaxCluster];
    float lowest[kMaxCluster];
    uint32_t scan_count[kWarps];
    uint32_t list_count;
    uint32_t found;
    // the chosen bin
    u64 before_mass;
    uint32_t before_count, bin, population;
};

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

// 2^45 exp((x - top) / T):  e = (x - top) / T = k ln2 / 64 + r with |r| <= 2^-7.5; 2^(k / 64) from a table, exp(r) by the first
// five terms of its series (the sixth is below 1e-13).  A float becomes a double by moving its fields, which takes a
// zero or a subnormal for a number below 2^-126; where T is so small that this could be seen, by conversion.
struct Weigher {
    const double* table;
    double top, inverse;         // 1 / T
    float top_f;
    bool convert;

    __device__ __forceinline__ double operator()(float x) const {
        double wide;
        if (convert) {
            wide = (double)x;
        } else {
            const uint32_t bits = __float_as_uint(x);
            wide = __hiloint2double((int)((bits & 0x80000000u) | (((bits & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(bits << 29));
        }
        const double e = (wide - top) * inverse;
        constexpr double kMagic = 6755399441055744.0;             // 1.5 * 2^52: the low word of a sum holds its rounding
        const double shifted = fma(e, 92.332482616893656877, kMagic);      // 64 / ln2
        const int k = __double2loint(shifted);
        const double r = fma(shifted - kMagic, -0.010830424696249145, e);  // ln2 / 64
        double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
        p = fma(p, r, 0.5);
        p = fma(p, r, 1.0);
        p = fma(p, r, 1.0);
        p *= table[k & (kTable - 1)];
        const double w = __hiloint2double(__double2hiint(p) + (k >> 6) * (1 << 20), __double2loint(p));
        return x == top_f ? kUnit : (e > -31.9 ? w : 0.0);        // below -31.9: less than half of 2^-45; also NaN
    }
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
__global__ void __launch_bounds__(kThreads, 4) qm_sample_filtered_kernel(const SampleArgs a) {
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

    const uint16_t* row16 = static_cast<const uint16_t*>(a.logits) + (kFp32 ? 0 : (size_t)row * a.row_stride + begin);
    const float* row32 = static_cast<const float*>(a.logits) + (kFp32 ? (size_t)row * a.row_stride + begin : 0);
    // -0 becomes +0 (equal scores), NaN becomes -inf (never drawn)
    auto score_at = [&](int i) { return fmaxf((kFp32 ? row32[i] : bf16_bits_to_f32(row16[i])) + 0.0f, -CUDART_INF_F); };
    // f(score, index in the slice) for every entry above -inf
    auto sweep = [&](auto f) {
        constexpr int kFlight = 8;
        for (int i0 = tid; i0 < n; i0 += kThreads * kFlight) {
            float x[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u) x[u] = i0 + u * kThreads < n ? score_at(i0 + u * kThreads) : -CUDART_INF_F;
#pragma unroll
            for (int u = 0; u < kFlight; ++u)
                if (x[u] > -CUDART_INF_F) f(x[u], i0 + u * kThreads);
        }
    };

    // ---- the first of the order, and the lowest score above -inf
    u64 best = 0ull;
    float lowest = CUDART_INF_F;
    {
        float top = -CUDART_INF_F;
        int at = 0;
        sweep([&](float x, int i) {
            if (x > top) {                        // indices rise: the lower of equals stays
                top = x;
                at = i;
            }
            lowest = fminf(lowest, x);
        });
        if (top > -CUDART_INF_F) best = entry_key(top, begin + at);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, best, off);
        best = other > best ? other : best;
        lowest = fminf(lowest, __shfl_xor_sync(0xffffffffu, lowest, off));
    }
    if (lane == 0) {
        s.scan_mass[warp] = best;
        s.scan_count[warp] = __float_as_uint(lowest);
    }
    __syncthreads();
    if (cluster > 1) cluster_wait();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        best = s.scan_mass[w] > best ? s.scan_mass[w] : best;
        lowest = fminf(lowest, __uint_as_float(s.scan_count[w]));
    }
    if (cluster > 1) {
        if (tid < cluster) {
            st_cluster_u64(remote(&s.best[rank], tid), best);
            st_cluster_u32(remote(&s.lowest[rank], tid), __float_as_uint(lowest));
        }
        cluster_sync_all();
        for (int r = 0; r < cluster; ++r) {
            best = s.best[r] > best ? s.best[r] : best;
            lowest = fminf(lowest, s.lowest[r]);
        }
    }
    const float temperature = a.temperature ? a.temperature[row] : 1.0f;
    if (best == 0ull || !(temperature > 0.0f)) {  // nothing to draw from, or nothing to draw
        if (rank == 0 && tid == 0) {
            a.tokens[row] = best ? key_index(best) : -1;
            if (a.probs) a.probs[row] = best ? 1.0f : 0.0f;
        }
        return;
    }

    const float top = key_score(best);
    const Weigher weight{s.table, (double)top, 1.0 / (double)temperature, top, temperature < 0x1p-60f};
    // entries below this have no weight (a float next to it is either 32 T below the top, or no other float lies between)
    const float cutoff = top == CUDART_INF_F ? top : top - 32.5f * temperature;
    // Bins even in z between the largest score and the lowest one that can matter.  Each operation is monotone, so a larger
    // score never has a larger bin; NaN (equal infinities, 0 * inf) comes only where all entries in question are equal or
    // the last of all, and is the last bin.
    const float per_bin = (float)kBins / fminf(top - lowest, 32.0f * temperature);
    auto bin_of = [&](float x) {
        return (int)(__float_as_uint(fminf((top - x) * per_bin, (float)(kBins - 1)) + 8388608.0f) & (kBins - 1));
    };
    float threshold = -CUDART_INF_F;              // what stays: scores above it, and at it the indices up to threshold_index
    int threshold_index = -1;
    auto stays = [&](float x, int i) { return x > threshold || (x == threshold && begin + i <= threshold_index); };

    // The last entry of the order, among those that stay so far, whose predecessors count less than k (by_mass false) or
    // weigh less than p times all of them: the new threshold.
    auto search = [&](bool by_mass, int k, float p, bool bins_are_clear) {
        int shift = 64, bin = 0;                  // from the second round on: the chosen bin, keys that agree with prefix above `shift`
        u64 prefix = 0ull, limit = (u64)k;
        uint32_t ahead_count = 0;
        u64 ahead_mass = 0;
        constexpr int kShifts[6] = {40, 30, 20, 10, 0, 0};
        // entries of the chosen bin that agree with the digits so far
        auto matches = [&](float x, int i) {
            if (x < cutoff || bin_of(x) != bin || !stays(x, i)) return false;
            return shift >= 64 || (entry_key(x, begin + i) >> shift) == (prefix >> shift);
        };
        for (int round = 0; round < 6; ++round) {
            if (round > 0 || !bins_are_clear) {
                for (int i = tid; i < kBins; i += kThreads) s.own.count[i] = s.own.low[i] = s.own.high[i] = 0u;
                __syncthreads();
            }
            const int next = round > 0 ? kShifts[round - 1] : 0;
            sweep([&](float x, int i) {
                int b;
                if (round == 0) {
                    if (x < cutoff || !stays(x, i)) return;
                    b = bin_of(x);
                } else {
                    if (!matches(x, i)) return;
                    b = kBins - 1 - (int)((entry_key(x, begin + i) >> next) & (u64)(kBins - 1));
                }
                atomicAdd(&s.own.count[b], 1u);
                if (by_mass) {
                    const u64 q = whole(weight(x));
                    const uint32_t lo = (uint32_t)q;
                    const uint32_t old = atomicAdd(&s.own.low[b], lo);
                    const uint32_t hi = (uint32_t)(q >> 32) + (old + lo < lo ? 1u : 0u);
                    if (hi) atomicAdd(&s.own.high[b], hi);
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
                            c[r] = ld_cluster_u32(remote(&s.own.count[b], r));
                            if (by_mass) {
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
                        st_cluster_u32(remote(&s.sum.count[b], r), count);
                        if (by_mass) {
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
                c[j] = bins->count[b];
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
            uint32_t my_count = 0, my_population = 0;
            u64 my_mass = 0;
#pragma unroll
            for (int j = 0; j < kBinsPerThread; ++j) {
                if (c[j] && (by_mass ? mb : (u64)cb) < limit) {
                    mine = tid * kBinsPerThread + j;
                    my_population = c[j];
                    my_count = cb;
                    my_mass = mb;
                }
                cb += c[j];
                mb += m[j];
            }
            if (mine >= 0) atomicMax(&s.found, (uint32_t)mine + 1u);
            __syncthreads();
            if (mine >= 0 && s.found == (uint32_t)mine + 1u) {
                s.bin = (uint32_t)mine;
                s.population = my_population;
                s.before_count = my_count;
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
            if (s.population <= kList) break;
        }
        // ---- the bin's entries, from all CTAs into all CTAs
        sweep([&](float x, int i) {
            if (!matches(x, i)) return;
            const uint32_t at = atomicAdd(&s.list_count, 1u);
            if (at < kList) s.list[at] = entry_key(x, begin + i);
        });
        sync_all();
        int found = 0;
        for (int r = 0; r < cluster; ++r) {
            const int there = (int)(cluster > 1 ? ld_cluster_u32(remote(&s.list_count, r)) : s.list_count);
            for (int i = tid; i < there && found + i < kList; i += kThreads) {
                const u64 key = cluster > 1 ? ld_cluster_u64(remote(&s.list[i], r)) : s.list[i];
                s.all[found + i] = make_ulonglong2(key, by_mass ? whole(weight(key_score(key))) : 1ull);
            }
            found += there;
        }
        found = found < kList ? found : kList;
        __syncthreads();
        // rank by counting: what the larger keys measure
        u64 last = ~0ull;
        for (int e = tid; e < found; e += kThreads) {
            const u64 key = s.all[e].x;
            u64 before = by_mass ? ahead_mass : (u64)ahead_count;
            for (int j = 0; j < found; ++j) {
                const ulonglong2 other = s.all[j];
                before += other.x > key ? other.y : 0ull;
            }
            if (before < limit && key < last) last = key;
        }
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
        threshold_index = key_index(last);
    };

    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float min_p = a.min_p ? a.min_p[row] : 0.0f;
    const bool cut_k = k > 0 && k < a.vocab;
    if (cut_k) search(false, k, 1.0f, true);
    if (p < 1.0f) search(true, 0, p, !cut_k);

    // ---- the draw: kept weights in index order; a warp has a run of whole rows of 32 entries
    const u64 least = min_p > 0.0f ? (u64)ceil((double)fminf(min_p, 2.0f) * kUnit) : 0ull;
    auto kept = [&](float x, int i) -> double {
        if (x < cutoff || !stays(x, i)) return 0.0;
        const double w = weight(x);
        return whole(w) < least && x != top ? 0.0 : w;
    };
    const int run = (n + kWarps * 32 - 1) / (kWarps * 32) * 32;
    const int from = warp * run, to = from + run < n ? from + run : n;
    u64 mine = 0ull;
    {
        constexpr int kFlight = 8;
        for (int i0 = from + lane; i0 < to; i0 += 32 * kFlight) {
            float x[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u) x[u] = i0 + u * 32 < to ? score_at(i0 + u * 32) : -CUDART_INF_F;
#pragma unroll
            for (int u = 0; u < kFlight; ++u)
                if (x[u] > -CUDART_INF_F) mine += whole(kept(x[u], i0 + u * 32));
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
    if (lane == 0) s.scan_mass[warp] = mine;
    __syncthreads();
    u64 before = 0ull, total = 0ull;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s.scan_mass[w];
        total += s.scan_mass[w];
    }
    if (cluster > 1) {
        if (tid < cluster) st_cluster_u64(remote(&s.totals[rank], tid), total);
        cluster_sync_all();
        total = 0ull;
        for (int r = 0; r < cluster; ++r) {
            if (r < rank) before += s.totals[r];
            total += s.totals[r];
        }
    }
    const double wanted = (double)a.uniforms[row] * (double)total;
    u64 target = wanted > 0.0 ? (wanted < (double)total ? (u64)wanted : total - 1ull) : 0ull;
    if (target >= total) target = total - 1ull;
    if (target < before || target >= before + mine) return;
    // This warp's run holds it.  First which row of 32 entries: a lane adds up a row.  Then which entry: a lane has one.
    u64 sum = before;
    for (int row0 = from; row0 < to; row0 += 32 * 32) {
        u64 of_row = 0ull;
        const int first = row0 + lane * 32;
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
            const float x = first + i < to ? score_at(first + i) : -CUDART_INF_F;
            if (x > -CUDART_INF_F) of_row += whole(kept(x, first + i));
        }
        const u64 up_to = sum + warp_inclusive(of_row, lane);
        const unsigned past = __ballot_sync(0xffffffffu, target < up_to);
        if (past) {
            const int which = __ffs(past) - 1;
            sum = __shfl_sync(0xffffffffu, up_to - of_row, which);
            const int i = row0 + which * 32 + lane;
            const float x = i < to ? score_at(i) : -CUDART_INF_F;
            const double w = x > -CUDART_INF_F ? kept(x, i) : 0.0;
            const unsigned beyond = __ballot_sync(0xffffffffu, target < sum + warp_inclusive(whole(w), lane));
            if (lane == __ffs(beyond) - 1) {
                a.tokens[row] = begin + i;
                if (a.probs) a.probs[row] = (float)(w / (double)total);
            }
            return;
        }
        sum = __shfl_sync(0xffffffffu, up_to, 31);
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
    // As many CTAs per row as leave each 2048 scores, up to eight, and no more than fit the GPU at a time (four per SM).
    const long long fit = 4LL * sm_count_of_current_device();
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
