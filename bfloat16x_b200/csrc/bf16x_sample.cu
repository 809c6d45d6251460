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
// weights have some 31 correct bits and are held as 64-bit integers (2^-SH steps, SH
// such that the sum of a row cannot overflow), so every sum is exact and the
// same in any order.  With ~1e5 kept tokens, fp32 weights would move about
// one draw in a hundred to a neighbour.
//
// One cluster of C CTAs per row; each holds its part of the row as ordered
// 32-bit keys in shared memory and the logits are read once.  A histogram of
// (top - l) in 1/32 octaves of weight then says in which bin a cut lies.  If
// all tokens down to that bin are few, one CTA sorts them and finishes alone
// (the usual top-k, and top-p over a peaked row).  Otherwise the weight above
// the bin is summed exactly and only the bin's own tokens are sorted.
#include <algorithm>

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "bf16x_common.cuh"
#include "bf16x_status.cuh"

namespace cg = cooperative_groups;

namespace bf16x {

constexpr int kSampleWarps = 16;
constexpr int kSampleThreads = kSampleWarps * 32;
constexpr int kSampleBins = 1600;                     // 50 octaves: weights below 2^-49 are 0
constexpr int kSampleCap = 1024;                      // tokens that one CTA sorts
constexpr int kSampleMaxKeys = 40960;                 // tokens per CTA (81 keys per thread: 162 KB)
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

// 2^(62 - i/64)
__constant__ uint64_t c_exp2_tab[64] = {
    4611686018427387904ull, 4562008997483360349ull, 4512867096753504463ull, 4464254551929933550ull,
    4416165660797809419ull, 4368594782566476878ull, 4321536337207803251ull, 4274984804801645281ull,
    4228934724888366668ull, 4183380695828330266ull, 4138317374168289834ull, 4093739474014606996ull,
    4049641766413219908ull, 4006019078736290889ull, 3962866294075461077ull, 3920178350641640941ull,
    3877950241171266237ull, 3836177012338949768ull, 3794853764176460055ull, 3753975649497958757ull,
    3713537873331429433ull, 3673535692356230935ull, 3633964414346709481ull, 3594819397621804119ull,
    3556096050500581047ull, 3517789830763632898ull, 3479896245120279830ull, 3442410848681509921ull,
    3405329244438597040ull, 3368647082747335039ull, 3332360060817827770ull, 3296463922209775076ull,
    3260954456333195553ull, 3225827497954527522ull, 3191078926708050276ull, 3156704666612568285ull,
    3122700685593301682ull, 3089062995008926926ull, 3055787649183712190ull, 3022870744944692570ull,
    2990308421163830843ull, 2958096858305110056ull, 2926232277976504838ull, 2894710942486778865ull,
    2863529154407056491ull, 2832683256137117140ull, 2802169629476361550ull, 2771984695199399577ull,
    2742124912636209756ull, 2712586779256821376ull, 2683366830260470360ull, 2654461638169180747ull,
    2625867812425724110ull, 2597581998995909751ull, 2569600879975159024ull, 2541921173199317625ull,
    2514539631859660218ull, 2487453044122042215ull, 2460658232750154058ull, 2434152054732833796ull,
    2407931400915394245ull, 2381993195634921490ull, 2356334396359501942ull, 2330951993331335645ull};

// order-preserving key of a logit; NaN counts as -infinity, -0 as 0
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return kKeyNegInf;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// w = 2^-y in steps of 2^-sh.  The difference top - l is kept exactly as a sum
// of two fp32 numbers and multiplied by log2(e)/temperature in two parts, so y
// = k/64 + g has some 40 correct bits; then 2^-y = 2^(-k/64) (1 - u) with the
// first factor from a table of 62 bits and u = 1 - e^(-g ln 2) by its Taylor
// series to the 4th power in fp32 (|g ln 2| <= 0.0055: the rest is below 5e-14),
// which leaves a relative error of about 2^-31 without a sign of its own.  The
// same in fp64 took some 250 cycles per 32 tokens and scheduler, which was most
// of a call.
struct Weigher {
    float top, chi, clo;                              // maximum logit, log2(e) / temperature
    float limit;                                      // weights below half a step are 0
    int sh;
    uint32_t top_key;
    const uint64_t *tab;
    __device__ __forceinline__ float pos(uint32_t key) const { return __fmul_rn(__fsub_rn(top, logit_of(key)), chi); }
    __device__ __forceinline__ uint64_t operator()(uint32_t key) const {
        if (key == top_key) return 1ull << sh;
        const float l = logit_of(key), s = __fsub_rn(top, l), p = __fmul_rn(s, chi);
        if (!(p < limit)) return 0;
        const float bb = __fsub_rn(s, top), lo = __fsub_rn(__fsub_rn(top, __fsub_rn(s, bb)), __fadd_rn(l, bb));
        const float e = __fmaf_rn(lo, chi, __fmaf_rn(s, clo, __fmaf_rn(s, chi, -p)));
        const float m = __fmaf_rn(p, 64.f, 12582912.f);            // 1.5 * 2^23: rounds to a whole number
        const int k = (int)__float_as_uint(m) - 0x4B400000;
        const float x = 0.693147181f * __fadd_rn(__fmaf_rn(__fsub_rn(m, 12582912.f), -0.015625f, p), e);
        const float u = x * (1.f - x * (0.5f - x * (0.166666667f - x * 0.0416666667f)));
        const int64_t t = (int64_t)tab[k & 63];
        const int64_t w = t - (((int64_t)__float2int_rn(u * 0x1p38f) * (int64_t)(t >> 31)) >> 7);
        const int n = 62 - sh + (k >> 6);
        return (uint64_t)(w + (1ll << (n - 1))) >> n;
    }
    // which 1/32 octave below the maximum a key lies in: rounded fp32 operations, so it never falls as the logit does
    __device__ __forceinline__ int bin(uint32_t key) const {
        return key == top_key ? 0 : (int)fminf(pos(key) * 32.f, (float)(kSampleBins - 1));
    }
};

struct alignas(16) SampleShared {
    uint32_t cnt[kSampleBins];
    uint32_t low[kSampleBins];                        // sum over the bin of (1 - weight / weight at the bin's start) 2^21
    uint64_t list[kSampleCap];                        // this CTA's tokens of a bin; later the weights of `all`
    uint64_t all[kSampleCap];                         // the cluster's (first CTA)
    uint64_t red_w[2][kSampleWarps];
    uint32_t red_c[2][kSampleWarps];
    uint64_t cta_w[2];
    uint32_t cta_c[2];
    uint32_t n_list;
    uint64_t scan[kSampleWarps];
    uint32_t scan_c[kSampleWarps];
    // results of the first CTA, read by all
    uint64_t out_w;
    uint32_t out_key, out_idx;
    int out_move;
    int pick_bin;
    int last_bin;
    uint32_t pick_before, pick_count;
    uint64_t tab[64];
};

static_assert(sizeof(SampleShared) % 16 == 0, "the keys behind it are stored 16 bytes at a time");

struct SampleCtx {
    SampleShared &sm;
    const uint32_t *keys;
    int n, C, rank;
    int l0, per;                                      // this lane's part of them: per keys from l0 on (per odd: no bank conflicts)
    uint32_t base;
    int turn;                                         // of the two exchange slots
    Weigher weigh;
};

// Sums of w and c over the cluster; before_*: those of the CTAs and warps in
// front of this warp.  Two slots in turn: a slot is written again only after
// another cluster barrier, when everyone has read it.
__device__ __forceinline__ void cluster_sums(SampleCtx &x, uint64_t w, uint32_t c, uint64_t &tot_w, uint32_t &tot_c,
                                             uint64_t &before_w) {
    SampleShared &sm = x.sm;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, s = x.turn;
    x.turn ^= 1;
    for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) {
        sm.red_w[s][warp] = w;
        sm.red_c[s][warp] = c;
    }
    __syncthreads();
    if (warp == 0) {
        uint64_t a = lane < kSampleWarps ? sm.red_w[s][lane] : 0;
        uint32_t b = lane < kSampleWarps ? sm.red_c[s][lane] : 0;
        for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        b = __reduce_add_sync(0xffffffffu, b);
        if (lane == 0) {
            sm.cta_w[s] = a;
            sm.cta_c[s] = b;
        }
    }
    cl.sync();
    // lane r reads rank r: one remote access deep, not C
    uint64_t a = 0, f = 0;
    uint32_t n = 0;
    if (lane < x.C) {
        const SampleShared *o = cl.map_shared_rank(&sm, lane);
        a = o->cta_w[s];
        n = o->cta_c[s];
        f = lane < x.rank ? a : 0;
    }
    f += lane < warp ? sm.red_w[s][lane] : 0;
    for (int o = 16; o; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        f += __shfl_xor_sync(0xffffffffu, f, o);
    }
    tot_w = a;
    tot_c = __reduce_add_sync(0xffffffffu, n);
    before_w = f;
}

// Inclusive scan over the block (w in thread order).
__device__ __forceinline__ uint64_t block_scan(SampleShared &sm, uint64_t w) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    if (lane == 31) sm.scan[warp] = w;
    __syncthreads();
    for (int i = 0; i < warp; ++i) w += sm.scan[i];
    __syncthreads();
    return w;
}

// Ascending sort of a[0, n2), n2 a power of two >= 64, by the whole block.
// Pairs within a warp's own 64 elements need only the warp.
__device__ void block_sort(uint64_t *a, int n2) {
    const int tid = threadIdx.x;
    for (int size = 2; size <= n2; size <<= 1)
        for (int j = size >> 1; j; j >>= 1) {
            for (int p = tid; p < n2 / 2; p += kSampleThreads) {
                const int i = ((p & ~(j - 1)) << 1) | (p & (j - 1));
                const uint64_t u = a[i], v = a[i + j];
                const bool up = (i & size) == 0;
                if ((u > v) == up) {
                    a[i] = v;
                    a[i + j] = u;
                }
            }
            const int next = j > 1 ? j >> 1 : size;                 // distance of the following step
            if (j > 32 || next > 32) __syncthreads();
            else __syncwarp();
        }
    __syncthreads();
}

// The first CTA's `all` filled with the cluster's listed tokens, sorted into
// the order (key down, index up).  Called by all; returns their number there.
__device__ int gather_sorted(SampleCtx &x, int &n2) {
    SampleShared &sm = x.sm;
    cg::cluster_group cl = cg::this_cluster();
    const int lane = threadIdx.x & 31;
    const uint32_t mine = lane < x.C ? cl.map_shared_rank(&sm, lane)->n_list : 0u;
    uint32_t upto = mine;                                           // tokens of the ranks up to this lane's
    for (int o = 1; o < kSampleMaxCluster; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    const int m = (int)__shfl_sync(0xffffffffu, upto, x.C - 1);
    for (int i0 = 0; i0 < m; i0 += kSampleThreads) {
        const uint32_t i = (uint32_t)(i0 + (int)threadIdx.x);
        uint32_t r = 0, first = 0;
        for (int q = 0; q < x.C - 1; ++q) {
            const uint32_t end = __shfl_sync(0xffffffffu, upto, q);
            if (i >= end) r = q + 1, first = end;
        }
        if (i < (uint32_t)m) sm.all[i] = cl.map_shared_rank(&sm, r)->list[i - first];
    }
    n2 = 64;
    while (n2 < m) n2 <<= 1;
    for (int i = m + threadIdx.x; i < n2; i += kSampleThreads) sm.all[i] = ~0ull;
    __syncthreads();
    block_sort(sm.all, n2);
    return m;
}

// Token i of this CTA into its list, if `take` (called by whole warps).
__device__ __forceinline__ void list_tokens(SampleCtx &x, int i, bool take) {
    SampleShared &sm = x.sm;
    const uint32_t mask = __ballot_sync(0xffffffffu, take);
    if (mask == 0) return;
    const int lane = threadIdx.x & 31, lead = __ffs(mask) - 1;
    uint32_t at = 0;
    if (lane == lead) at = atomicAdd(&sm.n_list, (uint32_t)__popc(mask));
    at = __shfl_sync(0xffffffffu, at, lead) + __popc(mask & ((1u << lane) - 1u));
    if (take && at < kSampleCap) sm.list[at] = (uint64_t)(~x.keys[i]) << 32 | (x.base + (uint32_t)i);
}

// The first bin at which the running count reaches k (k > 0) or the running
// weight, as far as the histogram knows it, reaches target; the last occupied
// bin if none does.  Sets pick_bin, pick_before (tokens before the bin),
// pick_count (in it, 0 where none reaches it).
__device__ void find_bin(SampleCtx &x, uint32_t k, double target) {
    SampleShared &sm = x.sm;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t run_c = 0;
    uint64_t run_w = 0;
    if (tid == 0) sm.pick_bin = -1, sm.pick_before = 0, sm.pick_count = 0, sm.last_bin = 0;
    __syncthreads();
    for (int b0 = 0; b0 < kSampleBins; b0 += kSampleThreads) {
        const int b = b0 + tid;
        uint32_t c = 0;
        uint64_t lows = 0;
        if (b < kSampleBins) {
            uint32_t rc[kSampleMaxCluster], rl[kSampleMaxCluster];
#pragma unroll
            for (int r = 0; r < kSampleMaxCluster; ++r) {           // all asked for before the first is used
                const SampleShared *o = cl.map_shared_rank(&sm, r < x.C ? r : 0);
                rc[r] = o->cnt[b];
                rl[r] = o->low[b];
            }
#pragma unroll
            for (int r = 0; r < kSampleMaxCluster; ++r)
                if (r < x.C) c += rc[r], lows += rl[r];
        }
        const double start = (double)(x.weigh.tab[(2 * b) & 63] >> (62 - x.weigh.sh));
        uint64_t w = c ? (uint64_t)(start * ((double)c - (double)lows * 0x1p-21)) >> (b >> 5) : 0;
        // inclusive scans of c and w
        uint32_t sc = c;
        uint64_t sw = w;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t yc = __shfl_up_sync(0xffffffffu, sc, o);
            const uint64_t yw = __shfl_up_sync(0xffffffffu, sw, o);
            if (lane >= o) sc += yc, sw += yw;
        }
        if (lane == 31) sm.scan[warp] = sw, sm.scan_c[warp] = sc;
        __syncthreads();
        uint32_t all_c = run_c;
        uint64_t all_w = run_w;
        for (int i = 0; i < kSampleWarps; ++i) {
            if (i == warp) sc += all_c, sw += all_w;
            all_c += sm.scan_c[i];
            all_w += sm.scan[i];
        }
        const bool after = k ? sc >= k : (double)sw >= target, before = k ? sc - c >= k : (double)(sw - w) >= target;
        if (c && after && !before) {                                // one thread at most
            sm.pick_bin = b;
            sm.pick_before = sc - c;
            sm.pick_count = c;
        }
        if (c) atomicMax(&sm.last_bin, b);
        const int found = __syncthreads_or(c && after);
        run_c = all_c, run_w = all_w;
        if (found) return;
    }
    // not reached: the whole row
    if (tid == 0) {
        sm.pick_bin = sm.last_bin;
        sm.pick_before = run_c;
        sm.pick_count = 0;
    }
    __syncthreads();
}

// Bisection over keys, then over indices, for bins with more tokens than one
// CTA sorts (rows of a few distinct values): one exact sum over the cluster per
// step.  K: by count (target = tokens still to take from the bin), else by
// weight.  The cut and the weight of the bin's part before and with it.
template <bool K>
__device__ void bisect(SampleCtx &x, int b, double target, uint32_t &cut_key, uint32_t &cut_idx, uint64_t &part) {
    const int tid = threadIdx.x;
    uint32_t lo = 0, hi = x.weigh.top_key;
    uint64_t tw, bw;
    uint32_t tc;
    while (lo < hi) {                                               // the largest key down to which the target is reached
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        uint64_t w = 0;
        uint32_t c = 0;
        for (int i = tid; i < x.n; i += kSampleThreads) {
            const uint32_t k = x.keys[i];
            if (k >= mid && x.weigh.bin(k) == b) {
                if (K) ++c;
                else w += x.weigh(k);
            }
        }
        cluster_sums(x, w, c, tw, tc, bw);
        if (K ? (double)tc >= target : (double)tw >= target) lo = mid;
        else hi = mid - 1;
    }
    cut_key = lo;
    uint64_t w = 0;
    uint32_t c = 0;
    for (int i = tid; i < x.n; i += kSampleThreads) {
        const uint32_t k = x.keys[i];
        if (k > lo && x.weigh.bin(k) == b) ++c, w += x.weigh(k);
    }
    cluster_sums(x, w, c, tw, tc, bw);
    const uint64_t each = x.weigh(lo);
    const double need = K ? target - (double)tc : each ? ceil((target - (double)tw) / (double)each) : 1.0;
    const uint32_t want = (uint32_t)fmin(fmax(need, 1.0), 4294967295.0);
    uint32_t j0 = 0, j1 = 0xFFFFFFFFu;                              // the lowest index up to which `want` ties lie
    uint32_t ties = 0;
    while (j0 < j1) {
        const uint32_t mid = j0 + (j1 - j0) / 2;
        c = 0;
        for (int i = tid; i < x.n; i += kSampleThreads) c += x.keys[i] == lo && x.base + (uint32_t)i <= mid;
        uint64_t zero;
        cluster_sums(x, 0, c, zero, ties, bw);
        if (ties >= want) j1 = mid;
        else j0 = mid + 1;
    }
    cut_idx = j0;
    part = tw + (uint64_t)want * each;
}

// The occupied bin next to b in direction d (b where there is none).
__device__ int next_bin(SampleCtx &x, int b, int d) {
    cg::cluster_group cl = cg::this_cluster();
    for (int i = b + d; i >= 0 && i < kSampleBins; i += d)
        for (int r = 0; r < x.C; ++r)
            if (cl.map_shared_rank(&x.sm, r)->cnt[i]) return i;
    return b;
}

// The exact cut at or near bin b: K: the first `k` tokens of the order (`count`
// of them lie before the bin); else the shortest prefix that weighs `target`.
// `sum`: the weight of the prefix; `at_bin`, `below`: the bin, and this lane's
// weight in the bins before it (of its warp's part of the row).
template <bool K>
__device__ void resolve(SampleCtx &x, int b, uint32_t count, uint32_t k, double target,
                        uint32_t &cut_key, uint32_t &cut_idx, uint64_t &sum, int &at_bin, uint64_t &below) {
    SampleShared &sm = x.sm;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x;
    for (;;) {
        if (tid == 0) sm.n_list = 0;
        __syncthreads();
        uint64_t w = 0;
        uint32_t c = 0;
        for (int q = 0; q < x.per; ++q) {
            const int i = x.l0 + q;
            const uint32_t key = i < x.n ? x.keys[i] : 0u;
            const int kb = i < x.n ? x.weigh.bin(key) : kSampleBins;
            if (kb < b) w += x.weigh(key);
            if (kb == b) ++c;
            list_tokens(x, min(i, x.n - 1), kb == b);
        }
        at_bin = b;
        below = w;
        uint64_t before, skip;
        uint32_t m;
        cluster_sums(x, w, c, before, m, skip);
        if (m > (uint32_t)kSampleCap) {
            uint64_t part;
            double need = K ? (double)(k - count) : target - (double)before;
            if (!K) {                                               // whether the cut lies in this bin at all
                uint64_t bin_w = 0, t2, s2;
                uint32_t c2;
                for (int i = tid; i < x.n; i += kSampleThreads)
                    if (x.weigh.bin(x.keys[i]) == b) bin_w += x.weigh(x.keys[i]);
                cluster_sums(x, bin_w, 0, t2, c2, s2);
                const int to = need <= 0.0 ? next_bin(x, b, -1) : need > (double)t2 ? next_bin(x, b, 1) : b;
                if (to != b) {
                    b = to;
                    continue;
                }
                need = fmin(need, (double)t2);
            }
            bisect<K>(x, b, need, cut_key, cut_idx, part);
            sum = before + part;
            return;
        }
        if (x.rank == 0) {
            int n2;
            const int got = gather_sorted(x, n2);
            // prefix weights, n2 / 512 tokens per thread
            const int per = (n2 + kSampleThreads - 1) / kSampleThreads;
            uint64_t mine[kSampleCap / kSampleThreads], s = 0;
#pragma unroll
            for (int q = 0; q < kSampleCap / kSampleThreads; ++q) {
                const int e = tid * per + q;
                mine[q] = q < per && e < got ? x.weigh(~(uint32_t)(sm.all[e] >> 32)) : 0;
                s += mine[q];
            }
            uint64_t run = block_scan(sm, s) - s;
            if (tid == 0) sm.out_move = got == 0 || (!K && target <= (double)before) ? -1 : 1;
            __syncthreads();
            const bool down = sm.out_move < 0;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < kSampleCap / kSampleThreads; ++q) {
                const int e = tid * per + q;
                if (q >= per || e >= got) break;
                const uint64_t upto = before + run + mine[q];
                const bool hit = K ? (uint32_t)e + 1 == k - count
                                   : !down && (double)upto >= target && (double)(before + run) < target;
                if (hit) {
                    sm.out_move = 0;
                    sm.out_key = ~(uint32_t)(sm.all[e] >> 32);
                    sm.out_idx = (uint32_t)sm.all[e];
                    sm.out_w = upto;
                }
                run += mine[q];
            }
            __syncthreads();
        }
        cl.sync();
        const SampleShared *o = cl.map_shared_rank(&sm, 0);
        const int move = o->out_move;
        cut_key = o->out_key, cut_idx = o->out_idx, sum = o->out_w;
        cl.sync();
        if (move == 0) return;
        const int to = next_bin(x, b, move);
        if (to == b) {                                              // no such bin: the cut is at the end of the row
            cut_key = move < 0 ? x.weigh.top_key : kKeyNegInf, cut_idx = 0xFFFFFFFFu;
            return;
        }
        b = to;
    }
}

__global__ void __launch_bounds__(kSampleThreads, 1) sample_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SampleShared &sm = *reinterpret_cast<SampleShared *>(smem_raw);
    uint32_t *keys = reinterpret_cast<uint32_t *>(smem_raw + sizeof(SampleShared));
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_launch_dependents();
    if (tid < 64) sm.tab[tid] = c_exp2_tab[tid];
    for (int i = tid; i < kSampleBins; i += kSampleThreads) sm.cnt[i] = sm.low[i] = 0;
    if (tid == 0) sm.n_list = 0;
    griddep_wait();
    const int64_t row = blockIdx.x / C;
    const int64_t chunk = (int64_t)p.seg * kSampleWarps, base = rank * chunk;
    const int n = (int)max((int64_t)0, min(chunk, p.V - base));
    // ---- the row's part as keys, and the maximum
    uint32_t top = 0;
    {
        const uint8_t *src = static_cast<const uint8_t *>(p.logits) + (row * p.ld + base) * (p.bf16 ? 2 : 4);
        const bool vec = ((uintptr_t)src & 15) == 0;
        int done = 0;
        if (vec && p.bf16) {
            done = n & ~7;
#pragma unroll 4
            for (int i = 8 * tid; i < done; i += 8 * kSampleThreads) {
                const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(src + 2 * i));
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                uint32_t k[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    k[2 * j] = key_of(__uint_as_float(w[j] << 16));
                    k[2 * j + 1] = key_of(__uint_as_float(w[j] & 0xFFFF0000u));
                    top = max(top, max(k[2 * j], k[2 * j + 1]));
                }
                *reinterpret_cast<uint4 *>(keys + i) = make_uint4(k[0], k[1], k[2], k[3]);
                *reinterpret_cast<uint4 *>(keys + i + 4) = make_uint4(k[4], k[5], k[6], k[7]);
            }
        } else if (vec) {
            done = n & ~3;
#pragma unroll 8
            for (int i = 4 * tid; i < done; i += 4 * kSampleThreads) {
                const float4 v = __ldcs(reinterpret_cast<const float4 *>(src + 4 * i));
                const uint4 k = make_uint4(key_of(v.x), key_of(v.y), key_of(v.z), key_of(v.w));
                top = max(max(top, max(k.x, k.y)), max(k.z, k.w));
                *reinterpret_cast<uint4 *>(keys + i) = k;
            }
        }
        for (int i = done + tid; i < n; i += kSampleThreads) {
            const float v = p.bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(src)[i])
                                   : reinterpret_cast<const float *>(src)[i];
            const uint32_t k = key_of(v);
            keys[i] = k;
            top = max(top, k);
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) sm.red_c[0][warp] = top;
    __syncthreads();
    if (warp == 0) {
        top = __reduce_max_sync(0xffffffffu, lane < kSampleWarps ? sm.red_c[0][lane] : 0u);
        if (lane == 0) sm.cta_c[0] = top;
    }
    cl.sync();
    top = __reduce_max_sync(0xffffffffu, lane < C ? cl.map_shared_rank(&sm, lane)->cta_c[0] : 0u);
    const float temp = p.temperature ? p.temperature[row] : p.temperature0;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p0, min_p = p.min_p ? p.min_p[row] : p.min_p0;
    const int32_t top_k = p.top_k ? p.top_k[row] : p.top_k0;
    const float u = p.u[row];
    const int per = p.seg / 32, l0 = warp * p.seg + lane * per;
    SampleCtx x = {sm, keys, n, C, rank, l0, per, (uint32_t)base, 1, {}};
    Weigher &weigh = x.weigh;
    const double inv = 1.4426950408889634074 / (double)temp;
    weigh.top = logit_of(top);
    weigh.chi = (float)inv;
    weigh.clo = (float)(inv - (double)weigh.chi);
    weigh.limit = (float)p.sh + 1.5f;
    weigh.sh = p.sh;
    weigh.top_key = top;
    weigh.tab = sm.tab;
    const bool none = top <= kKeyNegInf, greedy = !(temp > 0.f) || top_k == 1;
    if (none || greedy) {
        // ---- the lowest index of the maximum
        uint32_t at = 0xFFFFFFFFu;
        if (!none)
            for (int i = tid; i < n; i += kSampleThreads)
                if (keys[i] == top) {
                    at = (uint32_t)base + (uint32_t)i;
                    break;
                }
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) sm.red_c[1][warp] = at;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < kSampleWarps; ++w) at = min(at, sm.red_c[1][w]);
            sm.cta_c[1] = at;
        }
        cl.sync();
        if (rank == 0 && warp == 0) {
            at = __reduce_min_sync(0xffffffffu, lane < C ? cl.map_shared_rank(&sm, lane)->cta_c[1] : 0xFFFFFFFFu);
            if (lane == 0) p.tokens[row] = none ? -1 : (int64_t)at;
        }
        cl.sync();
        return;
    }
    const uint64_t min_w =
        min_p > 0.f ? max((uint64_t)1, (uint64_t)ceil(fmin((double)min_p, 1.0) * (double)(1ull << p.sh))) : 1ull;
    int at_bin = -1;                                                // the cut's bin, where it was resolved
    uint64_t below = 0;
    uint32_t cut_key = kKeyNegInf, cut_idx = 0xFFFFFFFFu;           // keep keys above the cut, and its own up to an index
    const bool by_k = top_k > 0 && top_k < p.V, by_p = top_p < 1.f;
    if (by_k || by_p) {
        // ---- the histogram, and the row's whole weight where top-p needs it
        uint64_t w = 0, total, skip;
        for (int i = tid; i < n; i += kSampleThreads) {
            const uint32_t k = keys[i];
            const float f = k == top ? 0.f : weigh.pos(k) * 32.f;
            if (!(f < (float)(kSampleBins - 1))) continue;
            const int b = (int)f;
            atomicAdd(&sm.cnt[b], 1u);
            if (by_p) {
                float r;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((f - (float)b) * -0.03125f));
                atomicAdd(&sm.low[b], (uint32_t)((1.f - r) * 2097152.f));
                if (!by_k) w += weigh(k);
            }
        }
        uint32_t c;
        cluster_sums(x, w, 0, total, c, skip);
        find_bin(x, by_k ? (uint32_t)top_k : 0u, fmax((double)top_p * (double)total, 1.0));
        int b = sm.pick_bin;
        uint32_t before = sm.pick_before, count = sm.pick_count;
        const bool few = before + count <= (uint32_t)kSampleCap && b < kSampleBins - 1;
        bool finish = false;
        if (few) {
            // ---- all that can be kept on one CTA
            for (int i0 = 0; i0 < n; i0 += kSampleThreads) {
                const int i = i0 + tid;
                list_tokens(x, min(i, n - 1), i < n && weigh.bin(keys[i]) <= b);
            }
            cl.sync();
            if (rank == 0) {
                int n2;
                const int m = gather_sorted(x, n2);
                const int per = (n2 + kSampleThreads - 1) / kSampleThreads;
                uint64_t mine[kSampleCap / kSampleThreads], s = 0;
#pragma unroll
                for (int q = 0; q < kSampleCap / kSampleThreads; ++q) {
                    const int e = tid * per + q;
                    const bool in = q < per && e < m && (!by_k || e < top_k);
                    mine[q] = in ? weigh(~(uint32_t)(sm.all[e] >> 32)) : 0;
                    s += mine[q];
                }
                const uint64_t upto = block_scan(sm, s);
                if (tid == kSampleThreads - 1) sm.out_w = upto;
                __syncthreads();
                const uint64_t listed = sm.out_w;
                const double target = fmax((double)top_p * (double)(by_k ? listed : total), 1.0);
                // top-p alone: the histogram's estimate may have missed the cut
                finish = !(by_p && !by_k && (double)listed < target);
                if (finish) {
                    uint64_t run = upto - s, kept = 0;
#pragma unroll
                    for (int q = 0; q < kSampleCap / kSampleThreads; ++q) {
                        const int e = tid * per + q;
                        if (q >= per || e >= n2) break;
                        const uint64_t one = (by_p && (double)run >= target && e > 0) || mine[q] < min_w ? 0 : mine[q];
                        run += mine[q];
                        kept += one;
                        sm.list[e] = one;
                    }
                    __syncthreads();
                    for (int e = tid; e < n2; e += kSampleThreads)
                        sm.all[e] = e < m && sm.list[e] ? sm.all[e] << 32 | (uint32_t)e : ~0ull;    // by index
                    kept = block_scan(sm, kept);
                    if (tid == kSampleThreads - 1) sm.out_w = kept;
                    __syncthreads();
                    const uint64_t sum = sm.out_w;
                    block_sort(sm.all, n2);
                    const double ut = fmax((double)u, 0.0) * (double)sum;
                    const uint64_t goal = min(ut < (double)sum ? (uint64_t)ut : sum - 1, sum - 1);
                    s = 0;
#pragma unroll
                    for (int q = 0; q < kSampleCap / kSampleThreads; ++q) {
                        const int e = tid * per + q;
                        mine[q] = q < per && e < n2 && sm.all[e] != ~0ull ? sm.list[(uint32_t)sm.all[e]] : 0;
                        s += mine[q];
                    }
                    run = block_scan(sm, s) - s;
#pragma unroll
                    for (int q = 0; q < kSampleCap / kSampleThreads; ++q) {
                        if (goal >= run && goal < run + mine[q])     // exactly one
                            p.tokens[row] = (int64_t)(sm.all[tid * per + q] >> 32);
                        run += mine[q];
                    }
                }
                if (tid == 0) sm.out_move = finish ? 1 : 0;
            }
            cl.sync();
            finish = cl.map_shared_rank(&sm, 0)->out_move == 1;
            cl.sync();
            if (finish) return;
        }
        uint64_t sum = total;
        if (by_k && count > 0) {
            resolve<true>(x, b, before, (uint32_t)top_k, 0.0, cut_key, cut_idx, sum, at_bin, below);
        } else if (by_k && by_p) {                                  // k reaches past every weight
            uint64_t all = 0;
            for (int i = tid; i < n; i += kSampleThreads) all += weigh(keys[i]);
            cluster_sums(x, all, 0, sum, c, skip);
        }
        if (by_p) {
            const double target = fmax((double)top_p * (double)sum, 1.0);
            if (by_k) {
                find_bin(x, 0u, target);
                b = sm.pick_bin;
                __syncthreads();
            }
            resolve<false>(x, b, 0, 0, target, cut_key, cut_idx, sum, at_bin, below);
        }
    }
    // ---- the kept weight of each lane's part
    const auto kept = [&](int i) -> uint64_t {
        const uint32_t k = keys[i];
        if (k < cut_key || (k == cut_key && (uint32_t)base + (uint32_t)i > cut_idx)) return 0;
        const uint64_t w = weigh(k);
        return w >= min_w ? w : 0;
    };
    const int l1 = min(n, l0 + per);
    uint64_t w = 0, total, before;
    uint32_t c;
    if (at_bin >= 0 && min_w == 1) {                                // only the cut's bin is left to look at
        w = below;
        for (int i = l0; i < l1; ++i)
            if (weigh.bin(keys[i]) == at_bin) w += kept(i);
    } else {
#pragma unroll 2
        for (int i = l0; i < l1; ++i) w += kept(i);
    }
    cluster_sums(x, w, 0, total, c, before);
    // ---- the first token whose running sum exceeds u * total: its lane's part, then the token
    const double ut = fmax((double)u, 0.0) * (double)total;
    const uint64_t goal = min(ut < (double)total ? (uint64_t)ut : total - 1, total - 1);
    uint64_t upto = w;
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t z = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += z;
    }
    upto += before;
    const uint32_t over = __ballot_sync(0xffffffffu, upto > goal);
    if (goal >= before && over) {                                   // exactly one warp of the cluster
        const int who = __ffs(over) - 1;
        uint64_t run = __shfl_sync(0xffffffffu, upto - w, who);
        const int i0 = warp * p.seg + who * per;
        for (int q = 0; q < per; q += 32) {
            const int i = i0 + q + lane;
            uint64_t y = q + lane < per && i < n ? kept(i) : 0;
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t z = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= o) y += z;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, run + y > goal);
            if (hit) {
                if (lane == 0) p.tokens[row] = base + i0 + q + (__ffs(hit) - 1);
                break;
            }
            run += __shfl_sync(0xffffffffu, y, 31);
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
    while (C < kSampleMaxCluster && (B * C < 2 * 148 || V > (int64_t)C * kSampleMaxKeys)) C *= 2;
    SampleParams p = {};
    p.logits = logits, p.ld = ld, p.V = V, p.bf16 = dtype == BF16X_DTYPE_BF16;
    p.seg = (int)(((V + (int64_t)C * kSampleThreads - 1) / ((int64_t)C * kSampleThreads)) | 1) * 32;
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
