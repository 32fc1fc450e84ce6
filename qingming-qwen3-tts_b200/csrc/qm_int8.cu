// Projections with 8-bit integer operands: activations quantised per token row, weights per output channel.
//
//   s_x[r] = max_k |x[r][k]| / 127        q[r][k] = round(127 x[r][k] / max_k |x[r][k]|)      (ties to even)
//   out[r][n] = (sum_k q[r][k] w[n][k]) * s_x[r] * s_w[n]  (+ bias[n]) (+ residual[r][n])
//
// all of the second line after the sum in fp32, each operation rounded to it (the sum's conversion too, past 2^24), and the
// result to bf16.  The integer sums are exact (kind::i8 accumulates in 32 bits; |sum| <= 128^2 K stays below 2^31 for K up to 65 536),
// so neither the split of K over CTAs nor the order of the chunks can change a result.  No counterpart in the
// reference, whose projections are bf16 only (launch_linear_m1 17.cu:17646, launch_qkv_m1 :17691,
// launch_gate_up_swiglu_m1 :18020; the calls here have their shapes).  Against those, the weights are half the bytes,
// which is what a decode step streams, and the tensor pipe has twice the rate, which is what a prompt is bound by.
//
// Three kernels:
//   qm_quantize_rows_kernel   a CTA (many rows: a warp) per row; RMSNorm in front of the quantisation where a norm weight is given
//   qm_skinny_int8_kernel     up to 64 token rows: the weight tile is the M operand, K split over a cluster
//   qm_rows_int8_kernel       more rows: persistent 128-row tiles, two TMEM accumulators
// (the figures below: one B200, launches in a row in a CUDA graph)
#include <math_constants.h>

#include "qm_cluster.cuh"
#include "qm_tcgen05.cuh"

namespace {

// ---- quantisation of rows -----------------------------------------------------------------------------------------

constexpr int kQuantThreads = 256;             // CTA per row
constexpr int kQuantWarps = 8;                 // warp per row
constexpr int kQuantMaxDim = 24 * 1024;        // the row is staged in shared memory as bf16
constexpr int kMaxRows = 0x7fffff00;           // a row number rounded up to the next tile is an int too (rows of x and of weights)

// With a norm weight the value quantised is v[k] = x[k] * w[k] / rms; the rms divides out of q (q is a ratio of two such
// values) and enters the scale alone, so one sweep collects both the sum of squares and the largest |x w|, and x w is
// exact in fp32 (two 8-bit significands).  The largest magnitude is taken over the bit patterns, where an infinity or a
// NaN is larger than any number.
struct RowSweep {
    float sum;
    uint32_t big_bits;
};

struct QuantRow {
    float ratio;        // 127 / big where that is an ordinary number
    float big;
    float pre;          // exact power of two that keeps 127 * v and big inside fp32's range
    bool flat;          // nothing to quantise (all zero, or no scale): every q is zero
    bool plain;         // pre is 1
};

template <bool kNorm>
__device__ __forceinline__ void sweep_eight(const uint4& raw, const uint4& wv, RowSweep& s) {
    const uint32_t* rw = reinterpret_cast<const uint32_t*>(&raw);
    const uint32_t* ww = reinterpret_cast<const uint32_t*>(&wv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 v = bf16x2_to_float2(rw[i]);
        if (kNorm) {
            s.sum = fmaf(v.x, v.x, fmaf(v.y, v.y, s.sum));
            v = fmul2(v, bf16x2_to_float2(ww[i]));
        }
        s.big_bits = max(s.big_bits, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
    }
}

__device__ __forceinline__ QuantRow quant_row(uint32_t big_bits) {
    QuantRow r;
    r.flat = big_bits == 0u || big_bits >= 0x7f800000u;
    r.big = __uint_as_float(big_bits);
    r.pre = r.big > 1.0e30f ? 0x1p-64f : (r.big < 1.0e-30f ? 0x1p64f : 1.0f);
    r.plain = r.pre == 1.0f;
    r.ratio = r.flat ? 0.0f : 127.0f / r.big;
    return r;
}

__device__ __forceinline__ float row_scale(const QuantRow& r, float sum, bool norm, int dim, float epsilon) {
    if (r.big == 0.0f) return 0.0f;               // also without an epsilon, where the root below is infinite
    float s = r.big / 127.0f;
    if (norm) s *= rsqrtf(sum / (float)dim + epsilon);
    return r.flat ? CUDART_NAN_F : s;
}

// The correctly rounded quotient 127 v / big (the product is exact: at most 7 + 16 bits), to the nearest whole number.
__device__ __forceinline__ int quantize_exactly(float v, const QuantRow& r) {
    return (int)rintf(__fdiv_rn(127.0f * (v * r.pre), r.big * r.pre));
}

// Eight values at once.  fma(v, ratio, 1.5 * 2^23) leaves round(v * ratio) in the low bits; v * ratio is within 8e-6 of
// the quotient (ratio's own rounding), which can only change the rounding right beside a half step: if any of the
// eight is that near to one, all are divided.
template <bool kNorm>
__device__ __forceinline__ uint2 quantize_eight(const uint4& raw, const uint4& wv, const QuantRow& r) {
    if (r.flat) return make_uint2(0u, 0u);
    constexpr float kMagic = 12582912.0f;
    const uint32_t* rw = reinterpret_cast<const uint32_t*>(&raw);
    const uint32_t* ww = reinterpret_cast<const uint32_t*>(&wv);
    float v[8];
    uint32_t level[8];
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 e = bf16x2_to_float2(rw[i]);
        if (kNorm) e = fmul2(e, bf16x2_to_float2(ww[i]));
        v[2 * i] = e.x;
        v[2 * i + 1] = e.y;
        const float2 ratio2 = make_float2(r.ratio, r.ratio);
        const float2 m = ffma2(e, ratio2, make_float2(kMagic, kMagic));
        const float2 back = fadd2(make_float2(kMagic, kMagic), make_float2(-m.x, -m.y));
        const float2 d = ffma2(e, ratio2, back);
        off = fmax3(off, fabsf(d.x), fabsf(d.y));
        level[2 * i] = __float_as_uint(m.x);
        level[2 * i + 1] = __float_as_uint(m.y);
    }
    if (off > 0.49995f || !r.plain) {
#pragma unroll
        for (int i = 0; i < 8; ++i) level[i] = (uint32_t)quantize_exactly(v[i], r);
    }
    uint2 packed;
    packed.x = __byte_perm(__byte_perm(level[0], level[1], 0x0040), __byte_perm(level[2], level[3], 0x0040), 0x5410);
    packed.y = __byte_perm(__byte_perm(level[4], level[5], 0x0040), __byte_perm(level[6], level[7], 0x0040), 0x5410);
    return packed;
}

// A CTA per row: few rows, each as fast as it goes; any width and alignment (kVector = false).  Bound by latency: 2.2 us for
// one row of 2048, 3.4 us for 32 rows of 6144.
template <bool kVector, bool kNorm>
__global__ void __launch_bounds__(kQuantThreads) qm_quantize_rows_kernel(const uint16_t* __restrict__ x,
                                                                        const uint16_t* __restrict__ norm_weight,
                                                                        float epsilon, int8_t* __restrict__ q,
                                                                        float* __restrict__ scale, int dim) {
    extern __shared__ uint4 row_vectors[];
    __shared__ float warp_sum[kQuantThreads / 32];
    __shared__ uint32_t warp_big[kQuantThreads / 32];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t base = (size_t)blockIdx.x * dim;
    const uint4* weights = reinterpret_cast<const uint4*>(norm_weight);
    uint16_t* staged = reinterpret_cast<uint16_t*>(row_vectors);
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    RowSweep s = {0.0f, 0u};
    if (kVector) {
        for (int v = tid; v < dim / 8; v += kQuantThreads) {
            const uint4 raw = *reinterpret_cast<const uint4*>(x + base + 8 * v);
            row_vectors[v] = raw;
            sweep_eight<kNorm>(raw, kNorm ? __ldg(weights + v) : none, s);
        }
    } else {
        for (int c = tid; c < dim; c += kQuantThreads) {
            const uint16_t raw = x[base + c];
            staged[c] = raw;
            float v = bf16_bits_to_f32(raw);
            s.sum = fmaf(v, v, s.sum);
            if (kNorm) v *= bf16_bits_to_f32(norm_weight[c]);
            s.big_bits = max(s.big_bits, __float_as_uint(v) & 0x7fffffffu);
        }
    }
    s.big_bits = __reduce_max_sync(0xffffffffu, s.big_bits);
#pragma unroll
    for (int off = 16; off > 0 && kNorm; off >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, off);
    if (lane == 0) {
        warp_sum[warp] = s.sum;
        warp_big[warp] = s.big_bits;
    }
    __syncthreads();
    s = {0.0f, 0u};
#pragma unroll
    for (int w = 0; w < kQuantThreads / 32; ++w) {
        s.sum += warp_sum[w];
        s.big_bits = max(s.big_bits, warp_big[w]);
    }
    const QuantRow r = quant_row(s.big_bits);
    if (tid == 0) scale[blockIdx.x] = row_scale(r, s.sum, kNorm, dim, epsilon);
    if (kVector) {
        for (int v = tid; v < dim / 8; v += kQuantThreads)
            *reinterpret_cast<uint2*>(q + base + 8 * v) = quantize_eight<kNorm>(row_vectors[v], kNorm ? __ldg(weights + v) : none, r);
    } else {
        for (int c = tid; c < dim; c += kQuantThreads) {
            const float w = kNorm ? bf16_bits_to_f32(norm_weight[c]) : 1.0f;
            q[base + c] = r.flat ? (int8_t)0 : (int8_t)quantize_exactly(bf16_bits_to_f32(staged[c]) * w, r);
        }
    }
}

// A warp per row: many rows of up to 2048 values.  The row stays in registers (eight 16-byte pieces per lane, all
// requested at once), and there is nothing but shuffles between its two sweeps.  14.9 us for 9923 rows of 2048 (4.1 TB/s of
// the 9.4 us that HBM needs; 1.4 rounds of warps), 47.7 us for 40 099 (5.2 TB/s); with the norm 20.1 and 69.1 us, where a
// lane reads the norm weight twice from the L1 and three CTAs per SM are faster than four (22.7, 73.0).
constexpr int kManyRowsDim = 2048;

template <bool kNorm>
__global__ void __launch_bounds__(kQuantWarps * 32, kNorm ? 3 : 4) qm_quantize_many_rows_kernel(const uint16_t* __restrict__ x,
                                                                                const uint16_t* __restrict__ norm_weight,
                                                                                float epsilon, int8_t* __restrict__ q,
                                                                                float* __restrict__ scale, int dim, int rows) {
    constexpr int kPieces = kManyRowsDim / 8 / 32;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int row = blockIdx.x * kQuantWarps + (threadIdx.x >> 5);
    if (row >= rows) return;
    const uint4* src = reinterpret_cast<const uint4*>(x + (size_t)row * dim);
    const uint4* weights = reinterpret_cast<const uint4*>(norm_weight);
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    const int vectors = dim / 8;
    uint4 raw[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) raw[i] = lane + 32 * i < vectors ? src[lane + 32 * i] : none;
    RowSweep s = {0.0f, 0u};
#pragma unroll
    for (int i = 0; i < kPieces; ++i) sweep_eight<kNorm>(raw[i], kNorm && lane + 32 * i < vectors ? __ldg(weights + lane + 32 * i) : none, s);
    s.big_bits = __reduce_max_sync(0xffffffffu, s.big_bits);
#pragma unroll
    for (int off = 16; off > 0 && kNorm; off >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, off);
    const QuantRow r = quant_row(s.big_bits);
    if (lane == 0) scale[row] = row_scale(r, s.sum, kNorm, dim, epsilon);
    uint2* dst = reinterpret_cast<uint2*>(q + (size_t)row * dim);
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
        if (lane + 32 * i < vectors)
            dst[lane + 32 * i] = quantize_eight<kNorm>(raw[i], kNorm ? __ldg(weights + lane + 32 * i) : none, r);
}
// Measured, us, a CTA per row / a warp per row: 2048 columns, 2048 rows 6.5 / 7.5, 4096 rows 12.1 / 8.7, 9923 rows 24.1 / 14.9;
// other widths were not compared.  Wider rows have a CTA each whatever their number: 9923 rows of 6144 take 57 us, twice
// what their bytes need.
constexpr int kManyRows = 4096;

// ---- shared by the two products -----------------------------------------------------------------------------------

constexpr int kChunk = 128;                    // K columns (bytes) per ring stage: one 128-byte swizzle atom
constexpr int kSkinnyThreads = 192;            // warps 0-3 epilogue, warp 4 MMA issue, warp 5 TMA
constexpr int kWeightRows = 128;

// gate * sigmoid(gate) * up in fp32; the fast division is within 2 units in the last place (and gives 0 below a gate of
// -87, where the product is under 1e-36 of up)
__device__ __forceinline__ float gated(float gate, float up) { return __fdividef(gate, 1.0f + __expf(-gate)) * up; }

// The copying thread sees its last copies land (bounded) before it leaves, so that none is in flight into the shared
// memory of a CTA that has retired after some other thread's wait gave up.
template <typename FullBar>
__device__ __forceinline__ void drain_ring(FullBar full_bar, int loads, int stages) {
    bool gave_up = false;
    for (int i = loads > stages ? loads - stages : 0; i < loads; ++i)
        mbar_wait_bounded(full_bar(i % stages), (i / stages) & 1, gave_up);
}

struct Int8Args {
    const float* x_scale;            // [rows]
    const float* w_scale[3];         // [out_cols] of each weight matrix (gated: gate, up)
    const int8_t* weight[3];
    const uint16_t* bias[3];         // [out_cols] or null
    const uint16_t* residual;        // [rows][out_cols] or null (one matrix only)
    uint16_t* out[3];                // [rows][out_cols]
    int out_cols[3];
    int first_tile[3];               // first tile of each matrix
    uint32_t* status;
    int rows;
    int k_dim;
    int chunks;                      // ceil(k_dim / 128): the last chunk is filled up with zeros by the copy
    int split;                       // cluster size (skinny)
    int m_tiles, n_tiles;            // (many rows)
};

// ---- up to 64 token rows --------------------------------------------------------------------------------------------
//
// D^T[128 weight rows][token rows] accumulates in 16 / 32 / 64 TMEM columns; the CTAs of a cluster share a tile's K
// range and fold their integer sums through distributed shared memory.  While the launch waits for its predecessor
// (which writes the activations) it only asks the L2 for its weight slice: a weight matrix may be one that
// the previous launch has just quantised, so no weight byte is read into the SM before the wait.
//
// Bound by latency (launch, copies after the wait, the cluster's fold): 4.0 us for one row of 2048 -> 2048 (4 MB of weights,
// which HBM would bring in 0.64 us), 7.0 us for 32 rows of 6144 -> 2048, 9.1 us for 64 rows of 2048 -> 2 x 6144 gated.
template <int kMPad>
struct SkinnySmem {
    static constexpr int kStages = 4;
    static constexpr int kWeightBytes = kWeightRows * kChunk;
    static constexpr int kStageBytes = kWeightBytes + kMPad * kChunk;
    static constexpr int kReduce = 0;                                      // int32[kMPad][128], over the spent ring
    static constexpr int kBars = kStages * kStageBytes;                    // full[kStages], empty[kStages], acc
    static constexpr int kTmemSlot = kBars + (2 * kStages + 1) * 8;
    static constexpr int kTotal = kTmemSlot + 16;
    static_assert(kMPad * kWeightRows * 4 <= kStages * kStageBytes, "the reduction buffer lies inside the ring");
};

__device__ __forceinline__ int4 ld_cluster_s32x4(uint32_t remote_addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(remote_addr));
    return v;
}

template <int kMPad, bool kGated>
__global__ void __launch_bounds__(kSkinnyThreads)
qm_skinny_int8_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap w2_map,
                      const __grid_constant__ CUtensorMap w3_map, const __grid_constant__ CUtensorMap x_map, const Int8Args a) {
    using L = SkinnySmem<kMPad>;
    constexpr int kTmemCols = kMPad < 32 ? 32 : kMPad;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw_addr = smem_addr(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    unsigned char* smem = smem_raw + pad;
    const uint32_t sbase = raw_addr + pad;
    const uint32_t bar0 = sbase + L::kBars;
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (L::kStages + s); };
    const uint32_t acc_bar = bar0 + 8u * (2 * L::kStages);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmemSlot);
    int* reduce = reinterpret_cast<int*>(smem + L::kReduce);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int global_tile = blockIdx.x / a.split;
    const int seg = kGated ? 0 : (global_tile >= a.first_tile[2] ? 2 : (global_tile >= a.first_tile[1] ? 1 : 0));
    const int tile = global_tile - a.first_tile[seg];
    const CUtensorMap* seg_map = seg == 0 ? &w_map : (seg == 1 ? &w2_map : &w3_map);
    const int chunk_begin = (int)((long long)a.chunks * rank / a.split);
    const int chunk_end = (int)((long long)a.chunks * (rank + 1) / a.split);
    const int n_chunks = chunk_end - chunk_begin;

    if (warp == 5 && lane == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(acc_bar, 1);
        fence_mbar_init();
    }
    if (warp == 4) {
        tmem_alloc(smem_addr(tmem_slot), kTmemCols);
        tmem_relinquish();
    }
    if (warp < 4) {
        // one weight row's share of this CTA's K range per thread
        const int8_t* wbase = kGated ? (tid < 64 ? a.weight[0] : a.weight[1]) : a.weight[seg];
        const int wrow = kGated ? tile * 64 + (tid & 63) : tile * kWeightRows + tid;
        const int k0 = chunk_begin * kChunk;
        const int k1 = chunk_end * kChunk < a.k_dim ? chunk_end * kChunk : a.k_dim;
        if (wrow < a.out_cols[seg] && k1 > k0)
            bulk_prefetch_l2_hint(wbase + (size_t)wrow * a.k_dim + k0, (uint32_t)(k1 - k0), l2_policy_evict_last());
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    pdl_trigger();           // not before this CTA has its TMEM: the next launch's CTAs hold theirs while they wait for this one
    bool dead = false;
    pdl_wait();

    constexpr int kGroups = kGated ? 16 : 32;              // pieces of four columns in a tile
    const int n_cols = a.out_cols[seg];
    const int g = tid % kGroups;
    const int col = (kGated ? tile * 64 : tile * kWeightRows) + 4 * g;
    float sw[4], extra[4];                                 // column scales; the up scales (gated) or the bias
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = warp < 4 && col + i < n_cols;
        sw[i] = in ? a.w_scale[seg][col + i] : 0.0f;
        extra[i] = 0.0f;
        if (kGated) extra[i] = in ? a.w_scale[1][col + i] : 0.0f;
        else if (in && a.bias[seg]) extra[i] = bf16_bits_to_f32(a.bias[seg][col + i]);
    }

    if (warp == 5) {
        if (lane == 0) {
            const uint64_t weights_once = l2_policy_evict_first();
            for (int i = 0; i < n_chunks; ++i) {
                const int st = i % L::kStages;
                if (!mbar_wait_bounded(empty_bar(st), ((i / L::kStages) & 1) ^ 1, dead)) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
                const uint32_t dst = sbase + st * L::kStageBytes;
                const int col = (chunk_begin + i) * kChunk;
                mbar_arrive_expect_tx(full_bar(st), L::kStageBytes);
                tma_load_2d(dst + L::kWeightBytes, &x_map, full_bar(st), col, 0);
                if (kGated) {
                    tma_load_2d_hint(dst, &w_map, full_bar(st), col, tile * 64, weights_once);
                    tma_load_2d_hint(dst + L::kWeightBytes / 2, &w2_map, full_bar(st), col, tile * 64, weights_once);
                } else {
                    tma_load_2d_hint(dst, seg_map, full_bar(st), col, tile * kWeightRows, weights_once);
                }
            }
            drain_ring(full_bar, n_chunks, L::kStages);
        }
        __syncwarp();
    } else if (warp == 4) {
        if (lane == 0) {
            constexpr uint32_t idesc = umma_instr_desc_s8(kWeightRows, kMPad);
            for (int i = 0; i < n_chunks; ++i) {
                const int st = i % L::kStages;
                if (!mbar_wait_bounded(full_bar(st), (i / L::kStages) & 1, dead)) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
                tc_fence_after();
                const uint32_t wa = sbase + st * L::kStageBytes;
                const uint32_t xa = wa + L::kWeightBytes;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma_i8_ss(tmem_base, smem_desc(wa + ks * 32, 16, 1024), smem_desc(xa + ks * 32, 16, 1024), idesc,
                              (i > 0 || ks > 0) ? 1u : 0u);
                tc_commit(empty_bar(st));
            }
            tc_commit(acc_bar);
        }
        __syncwarp();
    } else {
        if (!mbar_wait_bounded(acc_bar, 0, dead) && lane == 0) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
        tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(warp * 32) << 16);
#pragma unroll
        for (int c = 0; c < kMPad / 16; ++c) {
            uint32_t v[16];
            if (n_chunks > 0) {
                tmem_ld16(taddr + c * 16, v);
                tmem_wait_ld();
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = 0u;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) reduce[(c * 16 + i) * kWeightRows + tid] = (int)v[i];
        }
    }
    cluster_sync_all();

    if (warp < 4) {
        // Rank r finishes the token rows r, r + split, ...; a thread keeps its four neighbouring weight rows of the tile
        // (whose scales and bias it fetched before the sums were ready) and walks those token rows.  All loads of a step
        // are issued before the first is used.
        const uint32_t reduce_addr = sbase + L::kReduce;
        uint32_t peer[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) peer[k] = map_to_rank(reduce_addr, (uint32_t)(k < a.split ? k : 0));
        for (int m = (int)rank + (tid / kGroups) * a.split; m < a.rows; m += (128 / kGroups) * a.split) {
            const uint32_t off = (uint32_t)(m * kWeightRows + 4 * g) * 4u;
            const size_t o = (size_t)m * n_cols + col;
            const float sx = a.x_scale[m];
            float res[4] = {0.f, 0.f, 0.f, 0.f};
            if (!kGated && a.residual) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + i < n_cols) res[i] = bf16_bits_to_f32(a.residual[o + i]);
            }
            int4 part[8], part2[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                part[k] = part2[k] = make_int4(0, 0, 0, 0);
                if (k < a.split) {
                    part[k] = ld_cluster_s32x4(peer[k] + off);
                    if (kGated) part2[k] = ld_cluster_s32x4(peer[k] + off + 64u * 4u);
                }
            }
            int acc[4] = {0, 0, 0, 0}, acc2[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                acc[0] += part[k].x; acc[1] += part[k].y; acc[2] += part[k].z; acc[3] += part[k].w;
                acc2[0] += part2[k].x; acc2[1] += part2[k].y; acc2[2] += part2[k].z; acc2[3] += part2[k].w;
            }
            uint32_t bits[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = (float)acc[i] * sx * sw[i];
                bits[i] = f32_to_bf16_bits(kGated ? gated(v, (float)acc2[i] * sx * extra[i]) : v + extra[i] + res[i]);
            }
            uint16_t* dst = a.out[seg] + o;
            if (col + 3 < n_cols && (reinterpret_cast<uintptr_t>(dst) & 7u) == 0) {
                *reinterpret_cast<uint2*>(dst) = make_uint2(bits[0] | (bits[1] << 16), bits[2] | (bits[3] << 16));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + i < n_cols) dst[i] = (uint16_t)bits[i];
            }
        }
    }

    cluster_arrive_relaxed();        // nobody leaves while a peer may still read its shared memory
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
    cluster_wait();
}

// ---- more token rows ------------------------------------------------------------------------------------------------
//
// One CTA per SM walks tiles of 128 token rows x kBN weight rows (gated: kBN / 2 gate rows and the same up rows); the
// MMA thread fills one TMEM accumulator while eight epilogue warps drain the other (two warps per quarter of the
// lanes, alternate blocks of 32 columns).  The tile's column scales and biases are fetched into shared memory while
// its products are still running; results leave through a 2 KB block per warp and TMA stores, which also clip the
// last tile.  kBN = 256 has the fewest operand bytes per operation; the narrower tiles are for calls whose 256-wide
// tiles would leave SMs without one.
//
// Bound by operand bytes from the L2 (48 KB per 128 columns of K and SM; 670 cycles against 512 of the tensor pipe) and,
// at small K, by the epilogue: 97 us = 2570 Tops for 9923 x 2048 x 6144, 187 us = 2940 Tops for 16384 x 4096 x 4096 (0.77
// and 0.88 of twice the measured bf16 rate).  Four epilogue warps with scattered 16-byte stores and the column scales
// read from global memory took 181 and 258 us.  Pairs of SMs on one tile of 256 x 256 (32 KB of operands instead of 48) were
// measured and lose 6 % between 1500 and 4000 rows to their longer start and end; above 9000 rows the difference is within
// what the chip's power limit does from run to run there (97 us, 115 after 0.3 s of such launches).  Walking the tiles in
// groups of 4 to 16 rows of tiles changes neither.
constexpr int kRowsThreads = 320;              // warps 0-7 epilogue, warp 8 MMA issue, warp 9 TMA loads
constexpr int kRowsEpilogue = 256;
constexpr int kStoreBytes = 32 * 32 * 2;       // 32 rows x 32 bf16 columns, 64-byte swizzle

template <int kBN>
struct RowsSmem {
    static constexpr int kStageA = 128 * kChunk;
    static constexpr int kStageBytes = kStageA + kBN * kChunk;
    static constexpr int kStages = kBN == 256 ? 4 : (kBN == 128 ? 6 : 8);
    static constexpr int kStore = kStages * kStageBytes;                   // one block per epilogue warp
    static constexpr int kColumns = kStore + 8 * kStoreBytes;              // float[2][3][kBN]: scale, up scale, bias
    static constexpr int kBars = kColumns + 2 * 3 * kBN * 4;               // full, empty, acc_full[2], acc_empty[2]
    static constexpr int kTmemSlot = kBars + (2 * kStages + 4) * 8;
    static constexpr int kTotal = kTmemSlot + 16;
    static_assert(kTotal + 1024 <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(x), "r"(y)
                 : "memory");
}

template <int kBN, bool kGated>
__global__ void __launch_bounds__(kRowsThreads, 1)
qm_rows_int8_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w0_map,
                    const __grid_constant__ CUtensorMap w1_map, const __grid_constant__ CUtensorMap out_map, const Int8Args a) {
    using L = RowsSmem<kBN>;
    constexpr int kCols = kGated ? kBN / 2 : kBN;           // output columns per tile
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw_addr = smem_addr(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    unsigned char* smem = smem_raw + pad;
    const uint32_t sbase = raw_addr + pad;
    const uint32_t bar0 = sbase + L::kBars;
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (L::kStages + s); };
    auto acc_full = [&](int b) { return bar0 + 8u * (2 * L::kStages + b); };
    auto acc_empty = [&](int b) { return bar0 + 8u * (2 * L::kStages + 2 + b); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmemSlot);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), kRowsEpilogue);
        }
        fence_mbar_init();
    }
    if (warp == 8) {
        tmem_alloc(smem_addr(tmem_slot), 2 * kBN);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    pdl_trigger();           // not before this CTA has its TMEM: the next launch's CTAs hold theirs while they wait for this one
    const int total_tiles = a.m_tiles * a.n_tiles;
    bool dead = false;
    pdl_wait();

    if (warp == 9) {
        if (lane == 0) {
            int it = 0;
            for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x) {
                const int m0 = (tile / a.n_tiles) * 128;
                const int n0 = (tile % a.n_tiles) * kCols;
                for (int kc = 0; kc < a.chunks; ++kc, ++it) {
                    const int st = it % L::kStages;
                    if (!mbar_wait_bounded(empty_bar(st), ((it / L::kStages) & 1) ^ 1, dead)) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
                    const uint32_t dst = sbase + st * L::kStageBytes;
                    mbar_arrive_expect_tx(full_bar(st), L::kStageBytes);
                    tma_load_2d(dst, &x_map, full_bar(st), kc * kChunk, m0);
                    tma_load_2d(dst + L::kStageA, &w0_map, full_bar(st), kc * kChunk, n0);
                    if (kGated)
                        tma_load_2d(dst + L::kStageA + kBN / 2 * kChunk, &w1_map, full_bar(st), kc * kChunk, n0);
                    else
                        tma_load_2d(dst + L::kStageA + kBN / 2 * kChunk, &w0_map, full_bar(st), kc * kChunk, n0 + kBN / 2);
                }
            }
            drain_ring(full_bar, it, L::kStages);
        }
        __syncwarp();
    } else if (warp == 8) {
        if (lane == 0) {
            constexpr uint32_t idesc = umma_instr_desc_s8(128, kBN);
            int it = 0, local = 0;
            for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++local) {
                const int buf = local & 1;
                if (!mbar_wait_bounded(acc_empty(buf), ((local >> 1) & 1) ^ 1, dead)) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
                tc_fence_after();
                uint32_t seen = mbar_probe(full_bar(it % L::kStages), (it / L::kStages) & 1);
                for (int kc = 0; kc < a.chunks; ++kc, ++it) {
                    const int st = it % L::kStages;
                    if (!mbar_wait_probed(seen, full_bar(st), (it / L::kStages) & 1, dead)) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
                    seen = kc + 1 < a.chunks ? mbar_probe(full_bar((it + 1) % L::kStages), ((it + 1) / L::kStages) & 1) : 0u;
                    tc_fence_after();
                    const uint32_t xa = sbase + st * L::kStageBytes;
                    const uint32_t wa = xa + L::kStageA;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        mma_i8_ss(tmem_base + buf * kBN, smem_desc(xa + ks * 32, 16, 1024), smem_desc(wa + ks * 32, 16, 1024), idesc,
                                  (kc > 0 || ks > 0) ? 1u : 0u);
                    tc_commit(empty_bar(st));
                }
                tc_commit(acc_full(buf));
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3;                      // which TMEM lanes this warp may read
        const int row_in_tile = quarter * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const int n_cols = a.out_cols[0];
        const bool wide = (n_cols & 7) == 0;               // rows are 16-byte multiples: TMA stores, 16-byte loads
        const uint32_t block = sbase + L::kStore + warp * kStoreBytes;
        const uint32_t my_row = block + lane * 64;
        const uint32_t swizzle = (uint32_t)((lane >> 1) & 3);       // 64-byte swizzle: 16-byte piece ^ (row / 2) % 4
        float* columns = reinterpret_cast<float*>(smem + L::kColumns);
        int local = 0;
        for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++local) {
            const int buf = local & 1;
            const int n0 = (tile % a.n_tiles) * kCols;
            const int m0 = (tile / a.n_tiles) * 128;
            const int row = m0 + row_in_tile;
            float* cs = columns + buf * 3 * kBN;           // two buffers: the other one may still be read
            if (tid < kCols) {
                const bool in = n0 + tid < n_cols;
                cs[tid] = in ? __ldg(a.w_scale[0] + n0 + tid) : 0.0f;
                if (kGated) cs[kBN + tid] = in ? __ldg(a.w_scale[1] + n0 + tid) : 0.0f;
                if (!kGated) cs[2 * kBN + tid] = in && a.bias[0] ? bf16_bits_to_f32(__ldg(a.bias[0] + n0 + tid)) : 0.0f;
            }
            const float sx = row < a.rows ? a.x_scale[row] : 0.0f;
            named_bar_sync(1, kRowsEpilogue);
            if (!mbar_wait_bounded(acc_full(buf), (local >> 1) & 1, dead) && lane == 0) atomicOr(a.status, QM_DEVSTAT_TIMEOUT);
            tc_fence_after();
            const uint32_t taddr = tmem_base + lane_base + buf * kBN;
#pragma unroll 1
            for (int c = warp >> 2; c < kCols / 32; c += 2) {
                const int col = n0 + c * 32;
                if (col >= n_cols) break;
                uint32_t acc[32], acc2[32];
                tmem_ld32(taddr + c * 32, acc);
                if (kGated) tmem_ld32(taddr + kBN / 2 + c * 32, acc2);
                const size_t o = (size_t)row * n_cols + col;
                uint4 res[4];
                const bool vector_residual = !kGated && wide && a.residual != nullptr;
#pragma unroll
                for (int p = 0; p < 4; ++p)
                    res[p] = vector_residual && row < a.rows && col + 8 * p < n_cols ? *(reinterpret_cast<const uint4*>(a.residual + o) + p)
                                                                                     : make_uint4(0u, 0u, 0u, 0u);
                tmem_wait_ld();
                uint32_t packed[16];
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 sw = *reinterpret_cast<const float2*>(cs + c * 32 + i);
                    float2 v = make_float2((float)(int)acc[i] * sx * sw.x, (float)(int)acc[i + 1] * sx * sw.y);
                    if (kGated) {
                        const float2 su = *reinterpret_cast<const float2*>(cs + kBN + c * 32 + i);
                        v.x = gated(v.x, (float)(int)acc2[i] * sx * su.x);
                        v.y = gated(v.y, (float)(int)acc2[i + 1] * sx * su.y);
                    } else {
                        const float2 bias = *reinterpret_cast<const float2*>(cs + 2 * kBN + c * 32 + i);
                        const uint32_t rw = reinterpret_cast<const uint32_t*>(res)[i >> 1];
                        v = make_float2(v.x + bias.x + bf16_lo(rw), v.y + bias.y + bf16_hi(rw));
                    }
                    if (wide) {
                        packed[i >> 1] = pack_bf16x2(v.x, v.y);
                    } else if (row < a.rows) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (col + i + h >= n_cols) continue;
                            float one = h ? v.y : v.x;
                            if (!kGated && a.residual) one += bf16_bits_to_f32(a.residual[o + i + h]);
                            a.out[0][o + i + h] = (uint16_t)f32_to_bf16_bits(one);
                        }
                    }
                }
                if (wide) {
                    // the warp's previous block has been read by its store
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
#pragma unroll
                    for (int p = 0; p < 4; ++p)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(my_row + (((uint32_t)p ^ swizzle) << 4)),
                                     "r"(packed[4 * p]), "r"(packed[4 * p + 1]), "r"(packed[4 * p + 2]), "r"(packed[4 * p + 3])
                                     : "memory");
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0 && m0 + quarter * 32 < a.rows) {
                        tma_store_2d(&out_map, block, col, m0 + quarter * 32);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            }
            tc_fence_before();
            mbar_arrive(acc_empty(buf));
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 2 * kBN);
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------

// [rows][cols] 8-bit row-major viewed as {cols, rows}; boxes of box_rows x 128 columns, 128-byte swizzle, zeros outside.
int32_t encode_byte_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint32_t box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return qm_fail(QM_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {cols};
    const cuuint32_t box[2] = {kChunk, box_rows};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult rc = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return qm_fail(QM_ECUDA, "cuTensorMapEncodeTiled failed for an 8-bit projection operand");
    return QM_OK;
}

// [rows][cols] bf16 results: blocks of 32 x 32, 64-byte swizzle.
int32_t encode_result_map(CUtensorMap* map, void* base, uint64_t rows, uint64_t cols) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return qm_fail(QM_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {cols * 2};
    const cuuint32_t box[2] = {32, 32};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult rc = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return qm_fail(QM_ECUDA, "cuTensorMapEncodeTiled failed for a projection result");
    return QM_OK;
}

struct Int8Segment {
    const int8_t* weight;
    const float* scale;
    const uint16_t* bias;
    uint16_t* out;
    int out_cols;
};

// CTAs that share a tile's K range, a power of two up to 8: doubled while that stays within two CTAs per SM and leaves
// each at least two chunks, or four where it would put a second CTA on SMs.  Measured, us, at 2048 -> 4096 (32 tiles, 16
// chunks) for 1 / 32 / 64 rows: split 2 6.0 / 7.5 / 9.4, split 4 5.0 / 5.8 / 6.9, split 8 5.1 / 6.5 / 7.7; at 4096 -> 4096
// (32 chunks) split 4 7.0 / 8.1 / 9.2, split 8 6.5 / 7.8 / 8.9.
int int8_split(int tiles, int chunks, int sms) {
    int split = 1;
    while (split < 8) {
        const int next = 2 * split;
        if (tiles * next > 2 * sms || chunks / next < (tiles * next > sms ? 4 : 2)) break;
        split = next;
    }
    return split;
}

// The opt-in to a kernel's shared memory, once per thread and device.
template <typename Kernel>
int32_t allow_smem(Kernel kernel, size_t bytes, int device, int& known_device, const char* what) {
    if (known_device == device) return QM_OK;
    QM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), what);
    known_device = device;
    return QM_OK;
}

template <int kMPad, bool kGated>
int32_t launch_skinny(const CUtensorMap* maps, const CUtensorMap& x_map, const Int8Args& a, unsigned grid, int device,
                      cudaStream_t stream, const char* what) {
    auto kernel = qm_skinny_int8_kernel<kMPad, kGated>;
    const size_t smem = SkinnySmem<kMPad>::kTotal + 1024;
    static thread_local int known_device = -1;
    const int32_t rc = allow_smem(kernel, smem, device, known_device, what);
    if (rc != QM_OK) return rc;
    QM_CUDA_TRY(launch_cluster(kernel, dim3(grid), dim3(kSkinnyThreads), (unsigned)a.split, smem, stream, maps[0], maps[1],
                               maps[2], x_map, a),
                what);
    return QM_OK;
}

template <int kBN, bool kGated>
int32_t launch_rows(const int8_t* x, const int8_t* w0, const int8_t* w1, Int8Args& a, int sms, int device, cudaStream_t stream,
                    const char* what) {
    constexpr int kCols = kGated ? kBN / 2 : kBN;
    CUtensorMap x_map, w0_map, w1_map, out_map{};
    int32_t rc = encode_byte_map(&x_map, x, (uint64_t)a.rows, (uint64_t)a.k_dim, 128);
    if (rc == QM_OK) rc = encode_byte_map(&w0_map, w0, (uint64_t)a.out_cols[0], (uint64_t)a.k_dim, kBN / 2);
    if (rc == QM_OK) rc = encode_byte_map(&w1_map, w1, (uint64_t)a.out_cols[0], (uint64_t)a.k_dim, kBN / 2);
    if (rc == QM_OK && a.out_cols[0] % 8 == 0) rc = encode_result_map(&out_map, a.out[0], (uint64_t)a.rows, (uint64_t)a.out_cols[0]);
    if (rc != QM_OK) return rc;
    a.n_tiles = (a.out_cols[0] + kCols - 1) / kCols;
    const long long tiles = (long long)a.m_tiles * a.n_tiles;
    if (tiles > kMaxRows) return qm_fail(QM_ECAPACITY, "too many output tiles for one launch");
    auto kernel = qm_rows_int8_kernel<kBN, kGated>;
    const size_t smem = RowsSmem<kBN>::kTotal + 1024;
    static thread_local int known_device = -1;
    rc = allow_smem(kernel, smem, device, known_device, what);
    if (rc != QM_OK) return rc;
    QM_CUDA_TRY(qm_launch(kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(kRowsThreads), smem, stream, x_map, w0_map,
                          w1_map, out_map, a),
                what);
    return QM_OK;
}

template <bool kGated>
int32_t run_int8(qm_kv_pool* pool, const int8_t* x, const float* x_scale, const Int8Segment* segs, int n_segs, const int8_t* up,
                 const float* up_scale, const uint16_t* residual, int rows, int k_dim, cudaStream_t stream, const char* what) {
    if (!pool) return qm_fail(QM_EINVAL, "pool is null");
    if (rows < 0 || rows > kMaxRows) return qm_fail(QM_EINVAL, "rows must be >= 0 and at most 2^31 - 256");
    if (k_dim < 16 || k_dim % 16 != 0 || k_dim > 65536)
        return qm_fail(QM_EINVAL, "reduction width must be a positive multiple of 16, at most 65536");
    for (int i = 0; i < n_segs; ++i)
        if (segs[i].out_cols < 1 || segs[i].out_cols > kMaxRows)
            return qm_fail(QM_EINVAL, "output width must be positive and at most 2^31 - 256");
    if (rows == 0) return QM_OK;                      // nothing to do; the row tensors may then be null
    if (!x || !x_scale || (kGated && (!up || !up_scale))) return qm_fail(QM_EINVAL, "null tensor pointer");
    uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(up) | reinterpret_cast<uintptr_t>(up_scale) |
                    reinterpret_cast<uintptr_t>(residual);
    for (int i = 0; i < n_segs; ++i) {
        if (!segs[i].weight || !segs[i].scale || !segs[i].out) return qm_fail(QM_EINVAL, "null tensor pointer");
        all |= reinterpret_cast<uintptr_t>(segs[i].weight) | reinterpret_cast<uintptr_t>(segs[i].scale) |
               reinterpret_cast<uintptr_t>(segs[i].bias) | reinterpret_cast<uintptr_t>(segs[i].out);
    }
    if ((all & 15u) || (reinterpret_cast<uintptr_t>(x_scale) & 3u))
        return qm_fail(QM_EINVAL, "8-bit projection operands must be 16-byte aligned");
    int device = -1;
    QM_CUDA_TRY(cudaGetDevice(&device), "get current device");
    if (device != pool->device) return qm_fail(QM_EINVAL, "the pool's device must be the current device");

    Int8Args a{};
    a.x_scale = x_scale;
    a.residual = residual;
    a.status = pool->status_dev;
    a.rows = rows;
    a.k_dim = k_dim;
    a.chunks = (k_dim + kChunk - 1) / kChunk;
    const int sms = pool->sm_count;
    if (rows <= 64) {
        const int rows_per_tile = kGated ? 64 : kWeightRows;
        CUtensorMap maps[3], x_map;
        int tiles = 0;
        for (int i = 0; i < 3; ++i) {
            const Int8Segment& sg = segs[i < n_segs ? i : n_segs - 1];
            const bool second = kGated && i == 1;
            a.weight[i] = second ? up : sg.weight;
            a.w_scale[i] = second ? up_scale : sg.scale;
            a.first_tile[i] = i < n_segs ? tiles : 0x7fffffff;
            if (i >= n_segs && !second) {          // unused: any valid map will do
                maps[i] = maps[i - 1];
                continue;
            }
            const int32_t rc = encode_byte_map(&maps[i], a.weight[i], (uint64_t)sg.out_cols, (uint64_t)k_dim, (uint32_t)rows_per_tile);
            if (rc != QM_OK) return rc;
            if (i < n_segs) {
                a.bias[i] = sg.bias;
                a.out[i] = sg.out;
                a.out_cols[i] = sg.out_cols;
                tiles += (sg.out_cols + rows_per_tile - 1) / rows_per_tile;
            }
        }
        const int m_pad = rows <= 16 ? 16 : (rows <= 32 ? 32 : 64);
        const int32_t rc = encode_byte_map(&x_map, x, (uint64_t)rows, (uint64_t)k_dim, (uint32_t)m_pad);
        if (rc != QM_OK) return rc;
        a.split = int8_split(tiles, a.chunks, sms);
        const unsigned grid = (unsigned)tiles * (unsigned)a.split;
        if (m_pad == 16) return launch_skinny<16, kGated>(maps, x_map, a, grid, device, stream, what);
        if (m_pad == 32) return launch_skinny<32, kGated>(maps, x_map, a, grid, device, stream, what);
        return launch_skinny<64, kGated>(maps, x_map, a, grid, device, stream, what);
    }
    a.m_tiles = (rows + 127) / 128;
    for (int i = 0; i < n_segs; ++i) {
        a.weight[0] = segs[i].weight;
        a.w_scale[0] = segs[i].scale;
        a.w_scale[1] = up_scale;
        a.bias[0] = segs[i].bias;
        a.out[0] = segs[i].out;
        a.out_cols[0] = segs[i].out_cols;
        // the widest tile that still gives every SM one
        auto enough = [&](int bn) {
            const int cols = kGated ? bn / 2 : bn;
            return (long long)a.m_tiles * ((segs[i].out_cols + cols - 1) / cols) >= sms;
        };
        const int8_t* second = kGated ? up : segs[i].weight;
        int32_t rc;
        if (enough(256)) rc = launch_rows<256, kGated>(x, segs[i].weight, second, a, sms, device, stream, what);
        else if (enough(128)) rc = launch_rows<128, kGated>(x, segs[i].weight, second, a, sms, device, stream, what);
        else rc = launch_rows<64, kGated>(x, segs[i].weight, second, a, sms, device, stream, what);
        if (rc != QM_OK) return rc;
    }
    return QM_OK;
}

}  // namespace

extern "C" {

int32_t qm_quantize_rows_int8(const uint16_t* x, const uint16_t* norm_weight, float epsilon, int8_t* q, float* scale, int32_t rows,
                              int32_t dim, void* stream) {
    if (rows < 0 || rows > kMaxRows) return qm_fail(QM_EINVAL, "rows must be >= 0 and at most 2^31 - 256");
    if (dim < 1 || dim > kQuantMaxDim) return qm_fail(QM_EINVAL, "dim must be between 1 and 24576");
    if (rows == 0) return QM_OK;
    if (!x || !q || !scale) return qm_fail(QM_EINVAL, "null tensor pointer");
    const uintptr_t bf16s = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(norm_weight);
    if ((bf16s & 1u) || (reinterpret_cast<uintptr_t>(scale) & 3u)) return qm_fail(QM_EINVAL, "misaligned tensor pointer");
    const size_t smem = ((size_t)dim * 2 + 15) / 16 * 16;
    const bool vector = dim % 8 == 0 && (bf16s & 15u) == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (vector && rows >= kManyRows && dim <= kManyRowsDim) {
        const dim3 grid((unsigned)((rows + kQuantWarps - 1) / kQuantWarps));
        QM_CUDA_TRY(qm_launch(norm_weight ? qm_quantize_many_rows_kernel<true> : qm_quantize_many_rows_kernel<false>, grid,
                              dim3(kQuantWarps * 32), 0, s, x, norm_weight, epsilon, q, scale, (int)dim, (int)rows),
                    "row quantisation launch");
        return QM_OK;
    }
    auto kernel = vector ? (norm_weight ? qm_quantize_rows_kernel<true, true> : qm_quantize_rows_kernel<true, false>)
                         : (norm_weight ? qm_quantize_rows_kernel<false, true> : qm_quantize_rows_kernel<false, false>);
    if (smem > 47 * 1024)         // the row and the static words together pass the 48 KB that need no opt-in
        QM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kQuantMaxDim * 2),
                    "raise row quantisation shared memory");
    QM_CUDA_TRY(qm_launch(kernel, dim3((unsigned)rows), dim3(kQuantThreads), smem, s, x, norm_weight, epsilon, q, scale, (int)dim),
                "row quantisation launch");
    return QM_OK;
}

int32_t qm_linear_int8(qm_kv_pool* pool, const int8_t* x, const float* x_scale, const int8_t* weight, const float* weight_scale,
                       const uint16_t* bias, const uint16_t* residual, uint16_t* out, int32_t rows, int32_t out_features,
                       int32_t in_features, void* stream) {
    const Int8Segment seg{weight, weight_scale, bias, out, out_features};
    return run_int8<false>(pool, x, x_scale, &seg, 1, nullptr, nullptr, residual, rows, in_features,
                           static_cast<cudaStream_t>(stream), "8-bit projection launch");
}

int32_t qm_qkv_linear_int8(qm_kv_pool* pool, const int8_t* x, const float* x_scale, const int8_t* q_weight, const float* q_scale,
                           const uint16_t* q_bias, const int8_t* k_weight, const float* k_scale, const uint16_t* k_bias,
                           const int8_t* v_weight, const float* v_scale, const uint16_t* v_bias, uint16_t* q_out, uint16_t* k_out,
                           uint16_t* v_out, int32_t rows, int32_t hidden, int32_t q_dim, int32_t kv_dim, void* stream) {
    const Int8Segment segs[3] = {{q_weight, q_scale, q_bias, q_out, q_dim},
                                 {k_weight, k_scale, k_bias, k_out, kv_dim},
                                 {v_weight, v_scale, v_bias, v_out, kv_dim}};
    return run_int8<false>(pool, x, x_scale, segs, 3, nullptr, nullptr, nullptr, rows, hidden, static_cast<cudaStream_t>(stream),
                           "8-bit QKV projection launch");
}

int32_t qm_gate_up_swiglu_int8(qm_kv_pool* pool, const int8_t* x, const float* x_scale, const int8_t* gate_weight,
                               const float* gate_scale, const int8_t* up_weight, const float* up_scale, uint16_t* out, int32_t rows,
                               int32_t hidden, int32_t intermediate, void* stream) {
    const Int8Segment seg{gate_weight, gate_scale, nullptr, out, intermediate};
    return run_int8<true>(pool, x, x_scale, &seg, 1, up_weight, up_scale, nullptr, rows, hidden, static_cast<cudaStream_t>(stream),
                          "8-bit gate/up/SwiGLU launch");
}

}  // extern "C"
