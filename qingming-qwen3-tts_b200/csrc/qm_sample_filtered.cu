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
// Sums are whole numbers: a weight is worked out in double (to about 1e-14) and rounded to a multiple of 2^-45, so that
// sums over 2^18 weights fit 64 bits, are exact, and do not depend on the order of atomics; a weight below 2^-46 of the
// largest is zero and out of the game.
//
// A row is spread over a cluster of up to eight CTAs that keep its scores in shared memory, so global memory is read
// once.  Nothing is sorted as a whole: one sweep puts count and sum of the weights into 2048 bins that are even in z; the
// bin in which top-k (or top-p) ends is found by a scan, its few entries are gathered in the first CTA and ordered
// there.  A bin with more than 2048 entries (many equal scores) is first cut down by 11-bit digits of the entries'
// keys, which contain the index and therefore differ.
#include <math_constants.h>

#include "qm_cluster.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kBinsPerThread = kBins / kThreads;
constexpr int kList = 2048;
constexpr int kIndexBits = 18;
constexpr int kMaxVocab = 1 << kIndexBits;
constexpr int kMaxCluster = 8;
constexpr int kSlice = 8192;                    // scores per CTA that a cluster is sized for, as far as eight CTAs go
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

// What the first CTA tells the others after each step.
struct Verdict {
    u64 key;             // end of a search: the last key that stays
    u64 mass;            //                  sum of the weights that stay
    u64 before_mass;     // during a search: sum and number of the entries ahead of the chosen bin,
    uint32_t before_count;
    uint32_t bin;        //                  the bin,
    uint32_t population; //                  and how many entries it has (0: the search ends past the last entry)
    uint32_t pad;
};
constexpr int kVerdictWords = sizeof(Verdict) / 8;

struct Smem {
    uint32_t count[kBins];
    uint32_t low[kBins];         // sums of the weights, low and high 32 bits
    uint32_t high[kBins];
    u64 list[kList];
    double table[16];            // 2^(j / 16)
    u64 scan_mass[kWarps];
    u64 exchange[kMaxCluster];   // one word from every CTA
    float exchange_low[kMaxCluster];
    Verdict verdict;
    uint32_t scan_count[kWarps];
    uint32_t list_count;
    uint32_t found;
};

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t atom_add_cluster(uint32_t addr, uint32_t v) {
    uint32_t old;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
    return old;
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

// exp((x - top) / T) as 2^y: y to the nearest sixteenth from a table, the rest (at most 2^-5 of ln 2) by six terms of
// the exponential's series, whose next term is below 5e-16.
struct Weigher {
    const double* table;
    double top;
    double per_unit;             // log2(e) / T
    float top_f;

    __device__ __forceinline__ double operator()(float x) const {
        if (x == top_f) return 1.0;
        const double y = ((double)x - top) * per_unit;
        if (!(y > -46.0)) return 0.0;                             // also -inf, and the NaN of -inf * 0
        const double shifted = fma(y, 16.0, 6755399441055744.0);  // 1.5 * 2^52: the low word holds round(16 y)
        const int k = __double2loint(shifted);
        const double r = fma(shifted - 6755399441055744.0, -0.0625, y) * 0.693147180559945309417;
        double p = fma(r, 1.0 / 720.0, 1.0 / 120.0);
        p = fma(p, r, 1.0 / 24.0);
        p = fma(p, r, 1.0 / 6.0);
        p = fma(p, r, 0.5);
        p = fma(p, r, 1.0);
        p = fma(p, r, 1.0);
        p *= table[k & 15];
        return __hiloint2double(__double2hiint(p) + (k >> 4) * (1 << 20), __double2loint(p));
    }
};

__device__ __forceinline__ u64 whole(double w) { return __double2ull_rn(w * kUnit); }

template <typename T>
__device__ __forceinline__ T warp_inclusive(T v, int lane) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const T t = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += t;
    }
    return v;
}

// Exclusive sums over the block of one count and one mass per thread.
__device__ __forceinline__ void block_exclusive(Smem& s, uint32_t& count, u64& mass, int warp, int lane) {
    const uint32_t ci = warp_inclusive(count, lane);
    const u64 mi = warp_inclusive(mass, lane);
    if (lane == 31) {
        s.scan_count[warp] = ci;
        s.scan_mass[warp] = mi;
    }
    __syncthreads();
    uint32_t cb = 0;
    u64 mb = 0;
    for (int w = 0; w < warp; ++w) {
        cb += s.scan_count[w];
        mb += s.scan_mass[w];
    }
    __syncthreads();
    count = cb + ci - count;
    mass = mb + mi - mass;
}

template <bool kFp32>
__global__ void __launch_bounds__(kThreads) qm_sample_filtered_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    Smem& s = *reinterpret_cast<Smem*>(raw);
    float* scores = reinterpret_cast<float*>(raw + sizeof(Smem));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_rank();
    const int row = blockIdx.x / a.cluster;
    // slices of whole 32s, so that a warp's run of entries starts at one
    const int slice = ((a.vocab + a.cluster - 1) / a.cluster + 31) / 32 * 32;
    const int begin = rank * slice < a.vocab ? rank * slice : a.vocab;
    const int n = (begin + slice < a.vocab ? begin + slice : a.vocab) - begin;
    const uint32_t smem_self = smem_addr(raw);
    auto remote = [&](const void* mine, int r) { return map_to_rank(smem_self + (uint32_t)((const unsigned char*)mine - raw), (uint32_t)r); };

    pdl_trigger();
    cluster_arrive_relaxed();                     // "I have started": a CTA's shared memory is only written to after that
    if (tid < 16) s.table[tid] = exp2((double)tid / 16.0);
    for (int i = tid; i < kBins; i += kThreads) s.count[i] = s.low[i] = s.high[i] = 0u;
    if (tid == 0) s.list_count = 0u;
    pdl_wait();

    // ---- scores into shared memory; the first of the order, the lowest finite score
    u64 best = 0ull;
    float lowest = CUDART_INF_F;
    {
        const uint16_t* row16 = static_cast<const uint16_t*>(a.logits) + (kFp32 ? 0 : (size_t)row * a.row_stride + begin);
        const float* row32 = static_cast<const float*>(a.logits) + (kFp32 ? (size_t)row * a.row_stride + begin : 0);
#pragma unroll 8
        for (int i = tid; i < n; i += kThreads) {
            float x = (kFp32 ? row32[i] : bf16_bits_to_f32(row16[i])) + 0.0f;      // -0 becomes +0: equal scores
            if (x != x) x = -CUDART_INF_F;                                         // NaN is never drawn
            scores[i] = x;
            if (x > -CUDART_INF_F) {
                const u64 key = entry_key(x, begin + i);
                best = key > best ? key : best;
                lowest = fminf(lowest, x);
            }
        }
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
    cluster_wait();
    if (tid < a.cluster) {
        for (int w = 0; w < kWarps; ++w) {
            best = s.scan_mass[w] > best ? s.scan_mass[w] : best;
            lowest = fminf(lowest, __uint_as_float(s.scan_count[w]));
        }
        st_cluster_u64(remote(&s.exchange[rank], tid), best);
        st_cluster_f32(remote(&s.exchange_low[rank], tid), lowest);
    }
    cluster_sync_all();
    best = 0ull;
    lowest = CUDART_INF_F;
    for (int r = 0; r < a.cluster; ++r) {
        best = s.exchange[r] > best ? s.exchange[r] : best;
        lowest = fminf(lowest, s.exchange_low[r]);
    }
    const float temperature = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    if (best == 0ull || greedy) {                 // nothing to draw from, or nothing to draw
        if (rank == 0 && tid == 0) {
            a.tokens[row] = best ? key_index(best) : -1;
            if (a.probs) a.probs[row] = best ? 1.0f : 0.0f;
        }
        return;
    }

    const float top = key_score(best);
    const Weigher weight{s.table, (double)top, 1.4426950408889634074 / (double)temperature, top};
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float min_p = a.min_p ? a.min_p[row] : 0.0f;
    const bool cut_k = k > 0 && k < a.vocab, cut_p = p < 1.0f;
    // Bins even in z between the largest score and the lowest one that can matter (32 T below, where weights round to
    // zero).  Each operation is monotone, so a larger score never has a larger bin.
    const float range = fminf(top - lowest, 32.0f * temperature);
    const float per_bin = (float)kBins / range;
    auto bin_of = [&](float x) {
        if (x == top) return 0;
        const float b = (top - x) * per_bin;
        return b < (float)(kBins - 1) ? (int)b : kBins - 1;       // NaN (0 * inf) cannot be: x differs from top
    };
    auto add = [&](int bin, u64 q) {
        atomicAdd(&s.count[bin], 1u);
        const uint32_t lo = (uint32_t)q;
        const uint32_t old = atomicAdd(&s.low[bin], lo);
        const uint32_t hi = (uint32_t)(q >> 32) + (old + lo < lo ? 1u : 0u);
        if (hi) atomicAdd(&s.high[bin], hi);
    };
    auto clear_bins = [&]() {
        for (int i = tid; i < kBins; i += kThreads) s.count[i] = s.low[i] = s.high[i] = 0u;
        __syncthreads();
    };
    auto announce = [&]() {                       // the first CTA's verdict to all
        __syncthreads();
        if (rank == 0 && tid < kVerdictWords * (a.cluster - 1)) {
            const int r = 1 + tid / kVerdictWords, w = tid % kVerdictWords;
            st_cluster_u64(remote(reinterpret_cast<u64*>(&s.verdict) + w, r), reinterpret_cast<const u64*>(&s.verdict)[w]);
        }
        cluster_sync_all();
    };
    bool summed = false;                          // the first CTA's bins hold the cluster's sums

    // The last non-empty bin whose entries in front (`ahead_*` and the bins before) measure less than `limit`.
    auto choose_bin = [&](bool by_mass, u64 limit, uint32_t ahead_count, u64 ahead_mass) {
        if (!summed) cluster_sync_all();
        if (rank == 0) {
            uint32_t c[kBinsPerThread];
            u64 m[kBinsPerThread];
            uint32_t count = 0;
            u64 mass = 0;
#pragma unroll
            for (int j = 0; j < kBinsPerThread; ++j) {
                const int b = tid * kBinsPerThread + j;
                c[j] = s.count[b];
                m[j] = ((u64)s.high[b] << 32) + s.low[b];
            }
            if (!summed) {
                for (int r = 1; r < a.cluster; ++r) {
#pragma unroll
                    for (int j = 0; j < kBinsPerThread; ++j) {
                        const int b = tid * kBinsPerThread + j;
                        c[j] += ld_cluster_u32(remote(&s.count[b], r));
                        m[j] += ((u64)ld_cluster_u32(remote(&s.high[b], r)) << 32) + ld_cluster_u32(remote(&s.low[b], r));
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kBinsPerThread; ++j) {
                const int b = tid * kBinsPerThread + j;
                s.count[b] = c[j];
                s.low[b] = (uint32_t)m[j];
                s.high[b] = (uint32_t)(m[j] >> 32);
                count += c[j];
                mass += m[j];
            }
            uint32_t cb = count;
            u64 mb = mass;
            block_exclusive(s, cb, mb, warp, lane);
            if (tid == 0) {
                s.found = 0u;
                s.verdict.population = 0u;
            }
            __syncthreads();
            cb += ahead_count;
            mb += ahead_mass;
            int mine = -1;
            uint32_t my_c = 0, my_population = 0;
            u64 my_m = 0;
#pragma unroll
            for (int j = 0; j < kBinsPerThread; ++j) {
                if (c[j] && (by_mass ? mb : (u64)cb) < limit) {
                    mine = tid * kBinsPerThread + j;
                    my_population = c[j];
                    my_c = cb;
                    my_m = mb;
                }
                cb += c[j];
                mb += m[j];
            }
            if (mine >= 0) atomicMax(&s.found, (uint32_t)mine + 1u);
            __syncthreads();
            if (mine >= 0 && s.found == (uint32_t)mine + 1u) {
                s.verdict.bin = (uint32_t)mine;
                s.verdict.population = my_population;
                s.verdict.before_count = my_c;
                s.verdict.before_mass = my_m;
            }
            if (tid == kThreads - 1) s.verdict.mass = mb;         // everything
        }
        summed = true;
        announce();
    };

    // The last entry, among those with key >= floor_key, whose predecessors measure less than `limit`; verdict.key and
    // verdict.mass (with it) say where it is.  The bins of the whole row are in place.
    auto search = [&](bool by_mass, u64 limit, u64 floor_key) {
        choose_bin(by_mass, limit, 0u, 0ull);
        const int bin = (int)s.verdict.bin;
        u64 prefix = 0ull;
        int shift = 64;                           // keys agree with prefix above this bit
        constexpr int kShifts[5] = {39, 28, 18, 9, 0};
        for (int digit = 0; digit < 5 && s.verdict.population > kList; ++digit) {
            const uint32_t ahead_count = s.verdict.before_count;
            const u64 ahead_mass = s.verdict.before_mass;
            const int next = kShifts[digit];
            const int digit_bins = 1 << ((digit == 0 ? 50 : kShifts[digit - 1]) - next);
            cluster_sync_all();                   // the first CTA has read the others' bins, everyone the verdict
            clear_bins();
            for (int i = tid; i < n; i += kThreads) {
                const float x = scores[i];
                if (!(x > -CUDART_INF_F) || bin_of(x) != bin) continue;
                const u64 key = entry_key(x, begin + i);
                if (key < floor_key || (shift < 64 && (key >> shift) != (prefix >> shift))) continue;
                add(digit_bins - 1 - (int)((key >> next) & (u64)(digit_bins - 1)), whole(weight(x)));
            }
            summed = false;
            choose_bin(by_mass, limit, ahead_count, ahead_mass);
            prefix |= (u64)(digit_bins - 1 - (int)s.verdict.bin) << next;
            shift = next;
        }
        // gather the bin's entries in the first CTA
        const uint32_t count_at = remote(&s.list_count, 0), list_at = remote(s.list, 0);
        for (int i = tid; i < n; i += kThreads) {
            const float x = scores[i];
            if (!(x > -CUDART_INF_F) || bin_of(x) != bin) continue;
            const u64 key = entry_key(x, begin + i);
            if (key < floor_key || (shift < 64 && (key >> shift) != (prefix >> shift))) continue;
            const uint32_t at = atom_add_cluster(count_at, 1u);
            if (at < kList) st_cluster_u64(list_at + 8u * at, key);
        }
        cluster_sync_all();
        if (rank == 0) {
            const int found = s.list_count < kList ? (int)s.list_count : kList;
            int size = 32;
            while (size < found) size <<= 1;
            for (int i = found + tid; i < size; i += kThreads) s.list[i] = 0ull;
            __syncthreads();
            for (int width = 2; width <= size; width <<= 1) {
                for (int stride = width >> 1; stride > 0; stride >>= 1) {
                    for (int i = tid; i < size / 2; i += kThreads) {
                        const int at = 2 * i - (i & (stride - 1));        // pairs (at, at + stride)
                        const bool down = (at & width) == 0;
                        const u64 x = s.list[at], y = s.list[at + stride];
                        if (down ? x < y : x > y) {
                            s.list[at] = y;
                            s.list[at + stride] = x;
                        }
                    }
                    __syncthreads();
                }
            }
            constexpr int kEach = kList / kThreads;
            u64 q[kEach], mass = 0;
            uint32_t count = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int i = tid * kEach + j;
                q[j] = i < found ? whole(weight(key_score(s.list[i]))) : 0ull;
                mass += q[j];
                count += i < found ? 1u : 0u;
            }
            block_exclusive(s, count, mass, warp, lane);
            count += s.verdict.before_count;
            mass += s.verdict.before_mass;
            if (tid == 0) s.found = 0u;
            __syncthreads();
            int last = -1;
            u64 with = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int i = tid * kEach + j;
                if (i < found && (by_mass ? mass : (u64)count) < limit) {
                    last = i;
                    with = mass + q[j];
                }
                mass += q[j];
                ++count;
            }
            if (last >= 0) atomicMax(&s.found, (uint32_t)last + 1u);
            __syncthreads();
            if (last >= 0 && s.found == (uint32_t)last + 1u) {
                s.verdict.key = s.list[last];
                s.verdict.mass = with;
            }
            if (tid == 0) s.list_count = 0u;
        }
        announce();
    };

    u64 threshold = 0ull;
    auto fill_bins = [&]() {
        for (int i = tid; i < n; i += kThreads) {
            const float x = scores[i];
            if (!(x > -CUDART_INF_F)) continue;
            const u64 q = whole(weight(x));
            if (q == 0ull) scores[i] = -CUDART_INF_F;             // out of the game
            else if (entry_key(x, begin + i) >= threshold) add(bin_of(x), q);
        }
    };
    if (cut_k || cut_p) {
        fill_bins();
        u64 total = 0ull;                        // known to the first CTA, which alone compares against the limit
        if (cut_k) {
            search(false, (u64)k, 0ull);
            threshold = s.verdict.key;
            if (rank == 0) total = s.verdict.mass;
        }
        if (cut_p) {
            if (!cut_k) {
                choose_bin(true, 1ull, 0u, 0ull);
                if (rank == 0) total = s.verdict.mass;
            } else {
                // bins now hold the whole row, or digits of the last search: once more, with what top-k left
                cluster_sync_all();
                clear_bins();
                fill_bins();
                summed = false;
            }
            const double limit = ceil((double)p * (double)total);
            search(true, limit > 1.0 ? (u64)limit : 1ull, threshold);
            threshold = s.verdict.key;
        }
    }

    // ---- the draw: kept weights in index order
    const bool lowest_weight = min_p > 0.0f;
    auto kept = [&](int i) -> double {
        const float x = scores[i];
        if (!(x > -CUDART_INF_F) || entry_key(x, begin + i) < threshold) return 0.0;
        const double w = weight(x);
        return lowest_weight && w < (double)min_p && x != top ? 0.0 : w;
    };
    const int run = (n + kWarps * 32 - 1) / (kWarps * 32) * 32;      // entries of one warp
    const int from = warp * run, to = from + run < n ? from + run : n;
    u64 mine = 0ull;
    for (int i = from + lane; i < to; i += 32) mine += whole(kept(i));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
    if (lane == 0) s.scan_mass[warp] = mine;
    __syncthreads();
    u64 before = 0ull, all = 0ull;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s.scan_mass[w];
        all += s.scan_mass[w];
    }
    cluster_sync_all();                          // everyone has read the first exchange
    if (tid < a.cluster) st_cluster_u64(remote(&s.exchange[rank], tid), all);
    cluster_sync_all();
    u64 total = 0ull;
    for (int r = 0; r < a.cluster; ++r) {
        if (r < rank) before += s.exchange[r];
        total += s.exchange[r];
    }
    const double wanted = (double)a.uniforms[row] * (double)total;
    u64 target = wanted > 0.0 ? (wanted < (double)total ? (u64)wanted : total - 1ull) : 0ull;
    if (target >= total) target = total - 1ull;
    if (target >= before && target < before + mine) {                // this warp's entries hold it
        u64 sum = before;
        for (int base = from; base < to; base += 32) {
            const int i = base + lane;
            const double w = i < to ? kept(i) : 0.0;
            const u64 up_to = sum + warp_inclusive(whole(w), lane);
            const unsigned past = __ballot_sync(0xffffffffu, target < up_to);
            if (past) {
                if (lane == __ffs(past) - 1) {
                    a.tokens[row] = begin + i;
                    if (a.probs) a.probs[row] = (float)(w * kUnit / (double)total);
                }
                break;
            }
            sum = __shfl_sync(0xffffffffu, up_to, 31);
        }
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
    int cluster = 1;
    while (cluster < kMaxCluster && (vocab + cluster - 1) / cluster > kSlice) cluster *= 2;
    if ((long long)batch * cluster > 0x7fffffffLL) return qm_fail(QM_ECAPACITY, "too many rows for one launch");
    const int slice = ((vocab + cluster - 1) / cluster + 31) / 32 * 32;
    const size_t smem = sizeof(Smem) + (size_t)slice * sizeof(float);
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
    constexpr size_t kMaxSmem = sizeof(Smem) + (size_t)(kMaxVocab / kMaxCluster) * sizeof(float);
    static_assert(kMaxSmem <= 227 * 1024, "the largest slice fits one CTA");
    QM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem),
                "raise sampling kernel shared memory");
    QM_CUDA_TRY(launch_cluster(kernel, dim3((unsigned)(batch * cluster)), dim3(kThreads), (unsigned)cluster, smem,
                               static_cast<cudaStream_t>(stream), a),
                "filtered sampling launch");
    return QM_OK;
}
