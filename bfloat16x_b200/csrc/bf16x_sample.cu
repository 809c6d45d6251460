// bf16x_sample.cu -- drawing the next token from a row of logits with
// temperature, top-k, top-p and min-p, from given random numbers.
//
// With l the logits of a row and top their maximum, token i has the weight
//   w_i = 2^-y_i,  y_i = (top - l_i) * log2(e) / temperature   (1 at the maximum).
// The tokens are ordered by logit, ties by index (the lower index first), and
//   top-k keeps the first k of that order,
//   top-p the shortest prefix whose weight reaches p times what top-k kept,
//   min-p the tokens with w_i >= min_p;
// the token drawn is the first of the kept ones, in index order, whose running
// sum exceeds u times their total.  Each filter keeps a prefix of the order,
// so all of them together are one cut: a key and how many of its ties stay.
//
// Which token a number u falls on must not depend on the order of a sum: the
// weights are computed in fp64 and held as 64-bit integers (2^-SH steps, SH
// such that the sum of a row cannot overflow), so every sum is exact and the
// same in any order.  With ~1e5 kept tokens, fp32 weights would move about
// one draw in a hundred to a neighbour.
//
// One cluster of C CTAs per row; each holds its part of the row as ordered
// 32-bit keys in shared memory and the logits are read once.
#include <algorithm>

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "bf16x_common.cuh"
#include "bf16x_status.cuh"

namespace cg = cooperative_groups;

namespace bf16x {

constexpr int kSampleWarps = 16;
constexpr int kSampleThreads = kSampleWarps * 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleMaxKeys = 40960;                 // keys per CTA (160 KB)
constexpr int kSampleMaxCluster = 8;
constexpr uint32_t kKeyNegInf = 0x007FFFFFu;          // key of -infinity

struct SampleParams {
    const void *logits;
    int64_t ld, V;
    int bf16, seg, sh;                                // elements per warp; fixed-point shift
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    float temperature0, top_p0, min_p0;
    int32_t top_k0;
    int64_t *tokens;
};

// 2^(-i/32)
__constant__ double c_exp2_tab[32] = {
    1, 0.97857206208770009, 0.9576032806985737, 0.93708381705514998,
    0.91700404320467122, 0.89735453750155358, 0.87812608018664973, 0.85930964906123897,
    0.8408964152537145, 0.82287773907698247, 0.80524516597462714, 0.78799042255394325,
    0.77110541270397037, 0.75458221379671142, 0.73841307296974967, 0.72259040348852333,
    0.70710678118654757, 0.69195494098191601, 0.67712777346844633, 0.66261832157987066,
    0.64841977732550482, 0.63452547859586661, 0.620928906036742, 0.60762367999023448,
    0.59460355750136051, 0.58186242938878874, 0.56939431737834578, 0.55719337129794622,
    0.54525386633262884, 0.53357020033841185, 0.52213689121370688, 0.51094857432705831};

// order-preserving key of a logit; NaN counts as -infinity, -0 as 0
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return kKeyNegInf;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// w = 2^-y in steps of 2^-sh: y = k/32 + g with |g| <= 1/64, so 2^-y =
// 2^(-k/32) e^(-g ln 2), the last factor by its Taylor series to the 6th power
// (|g ln 2| <= 0.0109: the rest is below 4e-18).
struct Weigher {
    double top, inv;                                  // maximum logit, log2(e) / temperature
    int sh;
    uint32_t top_key;
    const double *tab;
    __device__ __forceinline__ uint64_t operator()(uint32_t key) const {
        if (key == top_key) return 1ull << sh;
        const double y = (top - (double)logit_of(key)) * inv;
        if (!(y < (double)(sh + 2))) return 0;
        const double magic = 6755399441055744.0 / 32.0;            // 1.5 * 2^52 / 32: rounds to a multiple of 1/32
        const double yr = y + magic;
        const int k = (int)(__double_as_longlong(yr) & 0xFFFFFFFFll);
        const double x = ((yr - magic) - y) * 0.6931471805599453094;
        double p = 1.0 / 720.0;
        p = fma(p, x, 1.0 / 120.0);
        p = fma(p, x, 1.0 / 24.0);
        p = fma(p, x, 1.0 / 6.0);
        p = fma(p, x, 0.5);
        p = fma(p, x, 1.0);
        p = fma(p, x, 1.0);
        const double m = tab[k & 31] * p;                           // in (0.48, 1.02)
        const uint64_t v = (uint64_t)__double2ll_rn(m * (double)(1ull << sh));
        const int n = k >> 5;
        return n == 0 ? v : (v + (1ull << (n - 1))) >> n;
    }
};

struct SampleShared {
    uint32_t cnt[kSampleBins];
    uint32_t limb[3][kSampleBins];                    // 16-bit limbs of the weights, summed
    uint64_t tot_w[kSampleBins];
    uint32_t tot_c[kSampleBins];
    uint64_t scan_w[kSampleWarps];
    uint32_t scan_c[kSampleWarps];
    uint32_t red_key[kSampleWarps];
    uint64_t warp_w[kSampleWarps];
    uint32_t warp_c[kSampleWarps];
    uint64_t cta_w;
    uint32_t cta_c, cta_key;
    uint32_t pick_bin, pick_before_c;
    uint64_t pick_before_w;
    double tab[32];
};

// One digit of a search over the keys that agree with `prefix` above bit
// `shift + bits`: the bin that holds the cut, and what lies before it.
template <bool WEIGHT>
__device__ void sample_digit(cg::cluster_group &cl, int C, SampleShared &sm, const uint32_t *keys, int n,
                             const Weigher &weigh, uint32_t prefix, int shift, int bits, double target,
                             uint64_t &before_w, uint32_t &before_c, uint32_t &bin) {
    const int tid = threadIdx.x, nb = 1 << bits;
    for (int i = tid; i < kSampleBins; i += kSampleThreads) {
        sm.cnt[i] = 0;
        sm.limb[0][i] = sm.limb[1][i] = sm.limb[2][i] = 0;
    }
    __syncthreads();
    const int hi = shift + bits;
    for (int i = tid; i < n; i += kSampleThreads) {
        const uint32_t k = keys[i];
        if (hi < 32 && (k >> hi) != (prefix >> hi)) continue;
        const uint32_t d = (k >> shift) & (nb - 1);
        const uint64_t w = weigh(k);
        atomicAdd(&sm.cnt[d], 1u);
        if (w) {
            atomicAdd(&sm.limb[0][d], (uint32_t)(w & 0xFFFFu));
            atomicAdd(&sm.limb[1][d], (uint32_t)((w >> 16) & 0xFFFFu));
            atomicAdd(&sm.limb[2][d], (uint32_t)(w >> 32));
        }
    }
    cl.sync();
    // every CTA adds up all bins of the cluster
    for (int i = tid; i < nb; i += kSampleThreads) {
        uint32_t c = 0;
        uint64_t w = 0;
        for (int r = 0; r < C; ++r) {
            const SampleShared *o = cl.map_shared_rank(&sm, r);
            c += o->cnt[i];
            w += (uint64_t)o->limb[0][i] + ((uint64_t)o->limb[1][i] << 16) + ((uint64_t)o->limb[2][i] << 32);
        }
        sm.tot_c[i] = c;
        sm.tot_w[i] = w;
    }
    __syncthreads();
    if (tid == 0) {
        // from the largest digit down
        uint64_t bw = before_w;
        uint32_t bc = before_c;
        int i = nb - 1;
        int last = -1;
        uint64_t lw = 0;
        uint32_t lc = 0;
        for (; i >= 0; --i) {
            if (sm.tot_c[i] == 0) continue;
            last = i, lw = bw, lc = bc;
            if (WEIGHT ? (double)(bw + sm.tot_w[i]) >= target : (double)(bc + sm.tot_c[i]) >= target) break;
            bw += sm.tot_w[i];
            bc += sm.tot_c[i];
        }
        // never reached (rounding of the target, or fewer tokens than k): the last bin there is
        sm.pick_bin = (uint32_t)max(last, 0);
        sm.pick_before_w = lw;
        sm.pick_before_c = lc;
    }
    __syncthreads();
    bin = sm.pick_bin;
    before_w = sm.pick_before_w;
    before_c = sm.pick_before_c;
    cl.sync();                                        // the bins are read by all before they are cleared again
}

// The shortest prefix of the order that reaches the target: its last key, how
// many of that key's ties belong to it, and the weight of the prefix.
template <bool WEIGHT>
__device__ void sample_select(cg::cluster_group &cl, int C, SampleShared &sm, const uint32_t *keys, int n,
                              const Weigher &weigh, double target, uint32_t &cut, uint32_t &ties, uint64_t &sum) {
    uint64_t bw = 0;
    uint32_t bc = 0, bin, prefix = 0;
    sample_digit<WEIGHT>(cl, C, sm, keys, n, weigh, prefix, 21, 11, target, bw, bc, bin);
    prefix |= bin << 21;
    sample_digit<WEIGHT>(cl, C, sm, keys, n, weigh, prefix, 10, 11, target, bw, bc, bin);
    prefix |= bin << 10;
    sample_digit<WEIGHT>(cl, C, sm, keys, n, weigh, prefix, 0, 10, target, bw, bc, bin);
    prefix |= bin;
    const uint64_t w = weigh(prefix);
    const uint32_t have = sm.tot_c[bin];
    double need;
    if (WEIGHT) need = w ? ceil((target - (double)bw) / (double)w) : 1.0;
    else need = target - (double)bc;
    ties = (uint32_t)fmin(fmax(need, 1.0), (double)have);
    cut = prefix;
    sum = bw + (uint64_t)ties * w;
}

__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SampleShared &sm = *reinterpret_cast<SampleShared *>(smem_raw);
    uint32_t *keys = reinterpret_cast<uint32_t *>(smem_raw + sizeof(SampleShared));
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_launch_dependents();
    griddep_wait();
    const int64_t row = blockIdx.x / C;
    const int64_t chunk = (int64_t)p.seg * kSampleWarps, base = rank * chunk;
    const int n = (int)max((int64_t)0, min(chunk, p.V - base));
    if (tid < 32) sm.tab[tid] = c_exp2_tab[tid];
    // ---- the row's part as keys, and the maximum
    uint32_t top = 0;
    for (int i = tid; i < n; i += kSampleThreads) {
        const int64_t at = row * p.ld + base + i;
        const float x = p.bf16 ? bf16_bits_to_f32(static_cast<const uint16_t *>(p.logits)[at])
                               : static_cast<const float *>(p.logits)[at];
        const uint32_t k = key_of(x);
        keys[i] = k;
        top = max(top, k);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) sm.red_key[warp] = top;
    __syncthreads();
    if (tid == 0) {
        for (int w = 0; w < kSampleWarps; ++w) top = max(top, sm.red_key[w]);
        sm.cta_key = top;
    }
    cl.sync();
    top = 0;
    for (int r = 0; r < C; ++r) top = max(top, cl.map_shared_rank(&sm, r)->cta_key);
    const float temp = p.temperature ? p.temperature[row] : p.temperature0;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p0, min_p = p.min_p ? p.min_p[row] : p.min_p0;
    const int32_t top_k = p.top_k ? p.top_k[row] : p.top_k0;
    // ---- the cut
    Weigher weigh;
    weigh.top = (double)logit_of(top);
    weigh.inv = 1.4426950408889634074 / (double)temp;
    weigh.sh = p.sh;
    weigh.top_key = top;
    weigh.tab = sm.tab;
    uint32_t cut = kKeyNegInf, ties = 0;              // keep keys above the cut, and the first `ties` of its own
    uint64_t min_w = 1;
    const bool none = top <= kKeyNegInf;              // nothing to choose from
    if (none) {
        cut = 0xFFFFFFFFu;
    } else if (!(temp > 0.f) || top_k == 1) {
        cut = top;
        ties = 1;
    } else {
        uint64_t sum = 0;
        bool have_sum = false;
        if (top_k > 0 && top_k < p.V) {
            sample_select<false>(cl, C, sm, keys, n, weigh, (double)top_k, cut, ties, sum);
            have_sum = true;
        }
        if (top_p < 1.f) {
            if (!have_sum) {
                uint64_t w = 0;
                for (int i = tid; i < n; i += kSampleThreads) w += weigh(keys[i]);
                for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
                if (lane == 0) sm.warp_w[warp] = w;
                __syncthreads();
                if (tid == 0) {
                    w = 0;
                    for (int i = 0; i < kSampleWarps; ++i) w += sm.warp_w[i];
                    sm.cta_w = w;
                }
                cl.sync();
                for (int r = 0; r < C; ++r) sum += cl.map_shared_rank(&sm, r)->cta_w;
                cl.sync();
            }
            sample_select<true>(cl, C, sm, keys, n, weigh, (double)top_p * (double)sum, cut, ties, sum);
        }
        if (min_p > 0.f) min_w = max((uint64_t)1, (uint64_t)ceil(fmin((double)min_p, 1.0) * (double)(1ull << p.sh)));
    }
    // ---- ties before each warp's part, in index order
    const int s0 = warp * p.seg, s1 = min(n, s0 + p.seg);
    uint32_t c = 0;
    for (int i = s0 + lane; i < s1; i += 32) c += keys[i] == cut;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) sm.warp_c[warp] = c;
    __syncthreads();
    if (tid == 0) {
        c = 0;
        for (int w = 0; w < kSampleWarps; ++w) c += sm.warp_c[w];
        sm.cta_c = c;
    }
    cl.sync();
    uint32_t tie0 = 0;
    for (int r = 0; r < rank; ++r) tie0 += cl.map_shared_rank(&sm, r)->cta_c;
    for (int w = 0; w < warp; ++w) tie0 += sm.warp_c[w];
    // ---- the kept weight of each warp's part
    const auto kept = [&](int i, uint32_t &tie) -> uint64_t {       // whole warp; i may lie past the part's end
        const uint32_t k = i < s1 ? keys[i] : 0u;
        const uint32_t same = __ballot_sync(0xffffffffu, i < s1 && k == cut);
        const uint32_t before = tie + __popc(same & ((1u << lane) - 1u));
        tie += __popc(same);
        if (i >= s1 || k < cut || (k == cut && before >= ties)) return 0;
        const uint64_t w = weigh(k);
        return w >= min_w ? w : 0;
    };
    uint64_t w = 0;
    uint32_t tie = tie0;
    if (!none)
        for (int i = s0; i < s1; i += 32) w += kept(i + lane, tie);
    for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (lane == 0) sm.warp_w[warp] = w;
    __syncthreads();
    if (tid == 0) {
        w = 0;
        for (int i = 0; i < kSampleWarps; ++i) w += sm.warp_w[i];
        sm.cta_w = w;
    }
    cl.sync();
    uint64_t total = 0, before = 0;
    for (int r = 0; r < C; ++r) {
        const uint64_t x = cl.map_shared_rank(&sm, r)->cta_w;
        if (r < rank) before += x;
        total += x;
    }
    for (int i = 0; i < warp; ++i) before += sm.warp_w[i];
    w = sm.warp_w[warp];
    if (none) {
        if (rank == 0 && tid == 0) p.tokens[row] = -1;
    } else {
        // ---- the first token whose running sum exceeds u * total
        const double ut = fmax((double)p.u[row], 0.0) * (double)total;
        uint64_t target = ut < (double)total ? (uint64_t)ut : total;
        if (target >= total) target = total - 1;
        if (target >= before && target < before + w) {              // exactly one warp of the cluster
            uint64_t run = before;
            tie = tie0;
            for (int i = s0; i < s1; i += 32) {
                uint64_t x = kept(i + lane, tie);
                for (int o = 1; o < 32; o <<= 1) {
                    const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                const uint32_t over = __ballot_sync(0xffffffffu, run + x > target);
                if (over) {
                    if (lane == 0) p.tokens[row] = base + i + (__ffs(over) - 1);
                    break;
                }
                run += __shfl_sync(0xffffffffu, x, 31);
            }
        }
    }
    cl.sync();                                        // no CTA leaves while another reads its shared memory
}

}  // namespace bf16x

using namespace bf16x;

extern "C" int bf16x_sample(const void *logits, int dtype, int64_t ld, int64_t B, int64_t V, const float *u,
                            const float *temperature, float temperature0, const int32_t *top_k, int32_t top_k0,
                            const float *top_p, float top_p0, const float *min_p, float min_p0, int64_t *tokens,
                            void *stream) {
    if (dtype != BF16X_DTYPE_BF16 && dtype != BF16X_DTYPE_F32)
        return set_error(BF16X_ERR_INVALID, "bf16x_sample: logits must be bf16 or fp32");
    if (B < 0 || V < 1 || ld < V) return set_error(BF16X_ERR_INVALID, "bf16x_sample: bad shape");
    if (V > (int64_t)kSampleMaxCluster * kSampleMaxKeys)
        return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_sample: at most %d tokens", kSampleMaxCluster * kSampleMaxKeys);
    if (B > (1 << 24)) return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_sample: too many rows");
    if (B == 0) return BF16X_OK;
    if (!logits || !u || !tokens) return set_error(BF16X_ERR_INVALID, "bf16x_sample: null pointer");
    int C = 1;
    while (C < kSampleMaxCluster && (B * C < 148 || V > (int64_t)C * kSampleMaxKeys)) C *= 2;
    SampleParams p = {};
    p.logits = logits, p.ld = ld, p.V = V, p.bf16 = dtype == BF16X_DTYPE_BF16;
    p.seg = (int)((V + (int64_t)C * kSampleThreads - 1) / ((int64_t)C * kSampleThreads)) * 32;
    int lg = 0;
    while (((int64_t)1 << lg) < V) ++lg;
    p.sh = std::min(47, 62 - lg);                     // 16-bit limbs hold weights below 2^48
    p.u = u, p.temperature = temperature, p.top_p = top_p, p.min_p = min_p, p.top_k = top_k;
    p.temperature0 = temperature0, p.top_p0 = top_p0, p.min_p0 = min_p0, p.top_k0 = top_k0;
    p.tokens = tokens;
    const size_t smem = sizeof(SampleShared) + (size_t)p.seg * kSampleWarps * 4;
    cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return set_error(BF16X_ERR_CUDA, "bf16x_sample: shared memory: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * C));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)C;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, sample_kernel, p);
    if (e != cudaSuccess) return set_error(BF16X_ERR_CUDA, "bf16x_sample: launch: %s", cudaGetErrorString(e));
    return check_launch("sample_kernel");
}
