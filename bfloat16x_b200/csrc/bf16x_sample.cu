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
// weights have some 30 correct bits and are held as 64-bit integers (2^-SH steps, SH
// such that the sum of a row cannot overflow), so every sum is exact and the
// same in any order.  With ~1e5 kept tokens, fp32 weights would move about
// one draw in a hundred to a neighbour.
//
// One cluster of C CTAs per row; each holds its part of the row as fp32 logits
// in shared memory, so the row is read once.  A histogram of
// (top - l) in 1/64 octaves of weight then says in which bin a cut lies.  If
// all tokens down to that bin are few, one CTA sorts them and finishes alone
// (the usual top-k, and top-p over a peaked row).  Otherwise the weight above
// the bin is summed exactly and only the bin's own tokens are sorted.
//
// Bound by latency for few rows (up to a dozen exchanges over the cluster of 0.5
// to 2 us each), by instructions for many (some 40 for a weight, of which each
// token needs one without filters and, for top-p, one before the cut is known
// and one if it is kept).  A row of 128256 bf16 logits: greedy 4.7 us, without
// filters 10.6, top-k 50 with or without top-p 13, top-p 0.9 alone 31; 16 rows
// (fp32): 5.6, 16, 17, 39; 129 rows of 73448: 12, 36, 35, 76 (38 MB: reading
// alone takes 6).
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "bf16x_common.cuh"
#include "bf16x_status.cuh"

namespace cg = cooperative_groups;

namespace bf16x {

constexpr int kSampleBins = 3200;                     // 50 octaves: weights below 2^-49 are 0
constexpr int kSampleMaxKeys = 40960;                 // tokens per CTA (160 KB)
constexpr int kSampleMaxCluster = 8;

struct SampleParams {
    const void *logits;
    int64_t ld, V;
    int bf16, per, sh;                                // tokens per thread; fixed-point shift
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    float temperature0, top_p0, min_p0;
    int32_t top_k0;
    int64_t *tokens;
};

// 2^(31 - i/64), and 2^(31 - (i - 1/2)/64): where the bin of that step begins
__constant__ uint32_t c_step[64] = {
    2147483648u, 2124350982u, 2101467502u, 2078830522u, 2056437387u, 2034285470u, 2012372174u, 1990694927u,
    1969251188u, 1948038440u, 1927054196u, 1906295993u, 1885761398u, 1865448001u, 1845353420u, 1825475297u,
    1805811301u, 1786359126u, 1767116489u, 1748081133u, 1729250827u, 1710623359u, 1692196547u, 1673968228u,
    1655936265u, 1638098541u, 1620452965u, 1602997467u, 1585730000u, 1568648537u, 1551751076u, 1535035634u,
    1518500250u, 1502142985u, 1485961921u, 1469955159u, 1454120821u, 1438457051u, 1422962010u, 1407633882u,
    1392470869u, 1377471191u, 1362633090u, 1347954824u, 1333434672u, 1319070932u, 1304861917u, 1290805962u,
    1276901417u, 1263146652u, 1249540052u, 1236080024u, 1222764986u, 1209593378u, 1196563654u, 1183674286u,
    1170923762u, 1158310587u, 1145833280u, 1133490379u, 1121280436u, 1109202018u, 1097253708u, 1085434106u};
__constant__ uint32_t c_bin[64] = {
    2159144272u, 2135885998u, 2112878262u, 2090118366u, 2067603638u, 2045331439u, 2023299156u, 2001504204u,
    1979944027u, 1958616096u, 1937517909u, 1916646992u, 1896000896u, 1875577199u, 1855373507u, 1835387448u,
    1815616678u, 1796058879u, 1776711757u, 1757573041u, 1738640488u, 1719911875u, 1701385007u, 1683057710u,
    1664927835u, 1646993254u, 1629251865u, 1611701585u, 1594340357u, 1577166143u, 1560176931u, 1543370725u,
    1526745556u, 1510299473u, 1494030547u, 1477936870u, 1462016553u, 1446267730u, 1430688553u, 1415277195u,
    1400031848u, 1384950723u, 1370032052u, 1355274085u, 1340675091u, 1326233356u, 1311947188u, 1297814910u,
    1283834865u, 1270005413u, 1256324931u, 1242791816u, 1229404479u, 1216161350u, 1203060876u, 1190101520u,
    1177281762u, 1164600099u, 1152055042u, 1139645120u, 1127368878u, 1115224875u, 1103211687u, 1091327906u};

// order-preserving key of a logit (no NaN, no -0)
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
constexpr float kNegInf = -__builtin_huge_valf();
// a logit as it is held: NaN counts as -infinity, -0 as 0
__device__ __forceinline__ float plain_logit(float x) { return x == x ? x + 0.f : kNegInf; }

// w = 2^-y in steps of 2^-sh.  The difference top - l is kept exactly as a sum
// of two fp32 numbers and multiplied by log2(e)/temperature in two parts, so y
// = k/64 + g has some 40 correct bits; then 2^-y = 2^(-k/64) (1 - u) with the
// first factor from a table and u = 1 - e^(-g ln 2) by its Taylor series to the
// 4th power in fp32 (|g ln 2| <= 0.0055: the rest is below 5e-14), to 30 bits:
// a relative error of about 2^-30 without a sign of its own.  Some 40
// instructions, all of 32 bits but the last sum: fp64, and 64-bit shifts, cost
// 250 and 100 cycles per 32 tokens and scheduler.
struct Weigher {
    float top, chi, clo;                              // maximum logit, log2(e) / temperature
    float limit;                                      // weights of less than about half a step are 0
    int sh;
    const uint32_t *step;
    // y (p), and k = y in 1/64 octaves, rounded, as a number and an integer; false for weights of 0.  Each fp32
    // operation is rounded by itself, so k never falls as the logit does.
    __device__ __forceinline__ bool place(float l, float &s, float &p, float &kf, int &k) const {
        s = l == top ? 0.f : __fsub_rn(top, l);                     // (infinity less infinity)
        p = __fmul_rn(s, chi);
        const bool ok = p < limit;
        p = ok ? p : 0.f;
        const float m = __fmaf_rn(p, 64.f, 12582912.f);            // 1.5 * 2^23: rounds to a whole number
        kf = __fsub_rn(m, 12582912.f);
        k = (int)__float_as_uint(m) - 0x4B400000;
        return ok;
    }
    // the bin of one step, the last one for weights of 0
    __device__ __forceinline__ int bin(float l) const {
        float s, p, kf;
        int k;
        return place(l, s, p, kf, k) ? k : kSampleBins - 1;
    }
    // the weight of a logit that counts as mant * 2^(-31 - (k >> 6))
    __device__ __forceinline__ uint32_t mantissa(float l, float s, float p, float kf, int k) const {
        const float bb = __fsub_rn(s, top), lo = __fsub_rn(__fsub_rn(top, __fsub_rn(s, bb)), __fadd_rn(l, bb));
        const float e = __fmaf_rn(lo, chi, __fmaf_rn(s, clo, __fmaf_rn(s, chi, -p)));
        const float x = 0.693147181f * __fadd_rn(__fmaf_rn(kf, -0.015625f, p), e);
        const float u = x * (1.f - x * (0.5f - x * (0.166666667f - x * 0.0416666667f)));
        const int q = (int)__float_as_uint(__fmaf_rn(u, 0x1p29f, 12582912.f)) - 0x4B400000;       // u 2^29, below 2^22
        const uint32_t t = step[k & 63];
        return l == top ? 0x80000000u : t - (uint32_t)__mulhi((int)(t >> 1), q * 16);
    }
    // acc + mant * 2^(sh - 31 - (k >> 6)), rounded
    __device__ __forceinline__ uint64_t add(uint64_t acc, uint32_t mant, int k) const {
        const int e = sh - 31 - (k >> 6), r = max(-e, 0);
        const uint32_t m = (mant >> r) + ((mant << 1) >> r & (r ? 1u : 0u));
        return acc + (uint64_t)m * (1u << max(e, 0));
    }
    __device__ __forceinline__ uint64_t add(uint64_t acc, float l, bool take = true) const {
        float s, p, kf;
        int k;
        const bool ok = place(l, s, p, kf, k) && take;              // no branch: four of these overlap
        const uint32_t m = mantissa(l, s, p, kf, k);
        return add(acc, ok ? m : 0u, k);
    }
    __device__ __forceinline__ uint64_t operator()(float l) const { return add(0, l); }
};

// W warps per CTA, a listed token per thread.
template <int W>
struct alignas(16) SampleShared {
    static constexpr int kThreads = W * 32;
    uint32_t cnt[kSampleBins];
    uint32_t low[kSampleBins];                        // sum over the bin of (weight at its start - weight), 2^-21 of the octave's
    uint64_t list[W * 32];                        // this CTA's tokens of a bin; later the weights of `all`
    uint64_t all[W * 32];                         // the cluster's (first CTA)
    uint64_t red_w[2][W];
    uint32_t red_c[2][W];
    uint64_t peer_w[2][kSampleMaxCluster];        // each CTA's sums, written by it
    uint32_t peer_c[2][kSampleMaxCluster];
    uint32_t n_list;
    uint64_t scan[W];
    uint32_t scan_c[W];
    // results of the first CTA
    uint64_t out_w;
    uint32_t out_key, out_idx;
    int out_move;
    // the same, in every CTA
    uint64_t got_w;
    uint32_t got_key, got_idx;
    int got_move;
    int pick_bin;
    int last_bin;
    uint32_t pick_before, pick_count;
    uint32_t step[64], start[64];
};
static_assert(sizeof(SampleShared<16>) % 16 == 0 && sizeof(SampleShared<32>) % 16 == 0,
              "the logits behind it are stored 16 bytes at a time");

template <int W>
struct SampleCtx {
    SampleShared<W> &sm;
    const float *logits;                              // this lane's: `per` of them (odd: no bank conflicts), padded
    int per, C, rank;                                 // with -infinity behind the row
    uint32_t first;                                   // index in the row of this lane's first one
    int turn;                                         // of the two exchange slots
    Weigher weigh;
};

// f(logit, q) for this lane's logits, four at a time: the weights' chains overlap.
template <int W, typename F>
__device__ __forceinline__ void for_logits(const SampleCtx<W> &x, F f) {
    int q = 0;
    for (; q + 4 <= x.per; q += 4) {
        float l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) l[i] = x.logits[q + i];
#pragma unroll
        for (int i = 0; i < 4; ++i) f(l[i], q + i);
    }
    for (; q < x.per; ++q) f(x.logits[q], q);
}

__device__ __forceinline__ uint64_t warp_sum(uint64_t w) {          // in limbs of 26 bits: 32 of them fit a word
    const uint64_t a = __reduce_add_sync(0xffffffffu, (uint32_t)w & 0x3FFFFFFu),
                   b = __reduce_add_sync(0xffffffffu, (uint32_t)(w >> 26) & 0x3FFFFFFu),
                   c = __reduce_add_sync(0xffffffffu, (uint32_t)(w >> 52));
    return a + (b << 26) + (c << 52);
}
__device__ __forceinline__ uint64_t warp_scan(uint64_t w) {         // inclusive
    const int lane = threadIdx.x & 31;
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    return w;
}

// Sums of w and c over the cluster; before_*: those of the CTAs and warps in
// front of this warp.  A CTA writes its sums to all others before the barrier,
// so that they are read at home.  Two slots in turn: a slot is written again
// only after another cluster barrier, when everyone has read it.
template <int W>
__device__ __forceinline__ void cluster_sums(SampleCtx<W> &x, uint64_t w, uint32_t c, uint64_t &tot_w, uint32_t &tot_c,
                                             uint64_t &before_w) {
    SampleShared<W> &sm = x.sm;
    cg::cluster_group cl = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, s = x.turn;
    x.turn ^= 1;
    w = warp_sum(w);
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) {
        sm.red_w[s][warp] = w;
        sm.red_c[s][warp] = c;
    }
    __syncthreads();
    if (warp == 0) {
        const uint64_t a = warp_sum(lane < W ? sm.red_w[s][lane] : 0);
        const uint32_t b = __reduce_add_sync(0xffffffffu, lane < W ? sm.red_c[s][lane] : 0u);
        if (lane < x.C) {
            SampleShared<W> *o = cl.map_shared_rank(&sm, lane);
            o->peer_w[s][x.rank] = a;
            o->peer_c[s][x.rank] = b;
        }
    }
    cl.sync();
    const uint64_t a = lane < x.C ? sm.peer_w[s][lane] : 0;
    const uint32_t n = lane < x.C ? sm.peer_c[s][lane] : 0u;
    const uint64_t f = (lane < warp ? sm.red_w[s][lane] : 0) + (lane < x.rank ? a : 0);
    tot_w = warp_sum(a);
    tot_c = __reduce_add_sync(0xffffffffu, n);
    before_w = warp_sum(f);
}

// Inclusive scan over the block (in thread order), and the block's total.
template <int W>
__device__ __forceinline__ uint64_t block_scan(SampleShared<W> &sm, uint64_t w, uint64_t &total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    w = warp_scan(w);
    if (lane == 31) sm.scan[warp] = w;
    __syncthreads();
    const uint64_t all = lane < W ? sm.scan[lane] : 0;
    w += warp_sum(lane < warp ? all : 0);
    total = warp_sum(all);
    __syncthreads();
    return w;
}

// Ascending sort of one number per thread of the first n2 threads (a power of
// two >= 64): shuffles within warps, shared memory (`all`) between them.
template <int W>
__device__ uint64_t block_sort(SampleShared<W> &sm, uint64_t a, int n2) {
    const int tid = threadIdx.x;
    for (int size = 2; size <= n2; size <<= 1)
        for (int j = size >> 1; j; j >>= 1) {
            uint64_t b;
            if (j >= 32) {
                __syncthreads();
                sm.all[tid] = a;
                __syncthreads();
                b = sm.all[tid ^ j];
            } else {
                b = __shfl_xor_sync(0xffffffffu, a, j);
            }
            const bool low = ((tid & j) == 0) == ((tid & size) == 0);
            a = (a < b) == low ? a : b;
        }
    __syncthreads();
    return a;
}

// The cluster's listed tokens in the first CTA, one per thread: ~key << 32 |
// index, so that they ascend in the order (logit down, index up), all ones
// behind the last.  Returns their number.
template <int W>
__device__ __forceinline__ int gather(SampleCtx<W> &x, uint64_t &token) {
    cg::cluster_group cl = cg::this_cluster();
    const int lane = threadIdx.x & 31;
    const uint32_t mine = lane < x.C ? cl.map_shared_rank(&x.sm, lane)->n_list : 0u;
    uint32_t upto = mine;                                           // tokens of the ranks up to this lane's
    for (int o = 1; o < kSampleMaxCluster; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    const int m = (int)__shfl_sync(0xffffffffu, upto, x.C - 1);
    const uint32_t i = threadIdx.x;
    uint32_t r = 0, first = 0;
#pragma unroll
    for (int q = 0; q < kSampleMaxCluster - 1; ++q) {
        const uint32_t end = __shfl_sync(0xffffffffu, upto, q);
        if (q < x.C - 1 && i >= end) r = q + 1, first = end;
    }
    token = i < (uint32_t)m ? cl.map_shared_rank(&x.sm, r)->list[i - first] : ~0ull;
    return m;
}
__device__ __forceinline__ int sort_size(int m) { return m <= 64 ? 64 : 1 << (32 - __clz(m - 1)); }

// Where few tokens are listed, n threads count for each what a sort would
// find: `before`: how many of `tok` are smaller, and what those weigh.
__device__ __forceinline__ void count_before(const uint64_t *tok, const uint64_t *weight, int m, int n, uint64_t mine,
                                             int &before, uint64_t &before_w) {
    before = 0, before_w = 0;
#pragma unroll 4
    for (int j = threadIdx.x & (n - 1); j < m; j += n) {
        const bool less = tok[j] < mine;
        before += less;
        before_w += less ? weight[j] : 0;
    }
    for (int o = 1; o < n; o <<= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        before_w += __shfl_xor_sync(0xffffffffu, before_w, o);
    }
}

// This lane's logits q0 .. q0 + 31, a bit each: those in bins before b, and in b.
template <int W>
__device__ __forceinline__ void mark_bins(const SampleCtx<W> &x, int q0, int b, uint32_t &before, uint32_t &at) {
    before = at = 0;
    const int n = min(32, x.per - q0);
    const auto mark = [&](float l, int i) {
        const int k = x.weigh.bin(l);
        before |= (k < b ? 1u : 0u) << i;
        at |= (k == b ? 1u : 0u) << i;
    };
    int i = 0;
    for (; i + 4 <= n; i += 4) {
        float l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) l[j] = x.logits[q0 + i + j];
#pragma unroll
        for (int j = 0; j < 4; ++j) mark(l[j], i + j);
    }
    for (; i < n; ++i) mark(x.logits[q0 + i], i);
}

// The marked ones into the CTA's list.
template <int W>
__device__ __forceinline__ void list_tokens(SampleCtx<W> &x, int q0, uint32_t marks) {
    if (!marks) return;
    SampleShared<W> &sm = x.sm;
    uint32_t at = atomicAdd(&sm.n_list, (uint32_t)__popc(marks));
    for (; marks; marks &= marks - 1, ++at) {
        const int q = q0 + __ffs(marks) - 1;
        if (at < W * 32) sm.list[at] = (uint64_t)(~key_of(x.logits[q])) << 32 | (x.first + (uint32_t)q);
    }
}

// The first bin at which the running count reaches k (k > 0) or the running
// weight, as far as the histogram knows it, reaches target; the last occupied
// bin if none does.  Sets pick_bin, pick_before (tokens before the bin),
// pick_count (in it, 0 where none reaches it).
template <int W>
__device__ void find_bin(SampleCtx<W> &x, uint32_t k, double target) {
    SampleShared<W> &sm = x.sm;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t run_c = 0;
    uint64_t run_w = 0;
    if (tid == 0) sm.pick_bin = -1, sm.pick_before = 0, sm.pick_count = 0, sm.last_bin = 0;
    for (int b0 = 0; b0 < kSampleBins; b0 += (W * 32)) {
        const int b = b0 + tid;
        uint32_t c = 0;
        uint64_t lows = 0;
        if (b < kSampleBins) {
            uint32_t rc[kSampleMaxCluster], rl[kSampleMaxCluster];
#pragma unroll
            for (int r = 0; r < kSampleMaxCluster; ++r) {           // all asked for before the first is used
                const SampleShared<W> *o = cl.map_shared_rank(&sm, r < x.C ? r : 0);
                rc[r] = o->cnt[b];
                rl[r] = k ? 0u : o->low[b];
            }
#pragma unroll
            for (int r = 0; r < kSampleMaxCluster; ++r)
                if (r < x.C) c += rc[r], lows += rl[r];
        }
        uint64_t w = 0;
        if (!k && c) {
            // 2^-31 of the octave's weight -> 2^-sh of the maximum's
            const uint64_t v = (uint64_t)c * sm.start[b & 63] - (lows << 10);
            const int e = x.weigh.sh - 31 - (b >> 6);
            w = e >= 0 ? v << e : v >> -e;
        }
        uint32_t sc = c;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, sc, o);
            if (lane >= o) sc += y;
        }
        uint64_t sw = k ? 0 : warp_scan(w);
        if (lane == 31) sm.scan[warp] = sw, sm.scan_c[warp] = sc;
        __syncthreads();
        const uint64_t aw = lane < W ? sm.scan[lane] : 0;
        const uint32_t ac = lane < W ? sm.scan_c[lane] : 0u;
        sc += run_c + __reduce_add_sync(0xffffffffu, lane < warp ? ac : 0u);
        run_c += __reduce_add_sync(0xffffffffu, ac);
        if (!k) {
            sw += run_w + warp_sum(lane < warp ? aw : 0);
            run_w += warp_sum(aw);
        }
        const bool after = k ? sc >= k : (double)sw >= target, before = k ? sc - c >= k : (double)(sw - w) >= target;
        if (c && after && !before) {                                // one thread at most
            sm.pick_bin = b;
            sm.pick_before = sc - c;
            sm.pick_count = c;
        }
        if (c) atomicMax(&sm.last_bin, b);
        if (__syncthreads_or(c && after)) return;
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
template <bool K, int W>
__device__ void bisect(SampleCtx<W> &x, int b, double target, float &cut, uint32_t &cut_idx, uint64_t &part) {
    uint32_t lo = 0, hi = key_of(x.weigh.top);
    uint64_t tw, bw;
    uint32_t tc;
    while (lo < hi) {                                               // the largest key down to which the target is reached
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        uint64_t w = 0;
        uint32_t c = 0;
        for_logits(x, [&](float l, int) {
            if (key_of(l) >= mid && x.weigh.bin(l) == b) {
                if (K) ++c;
                else w = x.weigh.add(w, l);
            }
        });
        cluster_sums(x, w, c, tw, tc, bw);
        if (K ? (double)tc >= target : (double)tw >= target) lo = mid;
        else hi = mid - 1;
    }
    cut = logit_of(lo);
    uint64_t w = 0;
    uint32_t c = 0;
    for_logits(x, [&](float l, int) {
        if (key_of(l) > lo && x.weigh.bin(l) == b) ++c, w = x.weigh.add(w, l);
    });
    cluster_sums(x, w, c, tw, tc, bw);
    const uint64_t each = x.weigh(cut);
    const double need = K ? target - (double)tc : each ? ceil((target - (double)tw) / (double)each) : 1.0;
    const uint32_t want = (uint32_t)fmin(fmax(need, 1.0), 4294967295.0);
    uint32_t j0 = 0, j1 = 0xFFFFFFFFu;                              // the lowest index up to which `want` ties lie
    uint32_t ties = 0;
    while (j0 < j1) {
        const uint32_t mid = j0 + (j1 - j0) / 2;
        c = 0;
        for_logits(x, [&](float l, int q) { c += key_of(l) == lo && x.first + (uint32_t)q <= mid; });
        uint64_t zero;
        cluster_sums(x, 0, c, zero, ties, bw);
        if (ties >= want) j1 = mid;
        else j0 = mid + 1;
    }
    cut_idx = j0;
    part = tw + (uint64_t)want * each;
}

// The occupied bin next to b in direction d (b where there is none).
template <int W>
__device__ int next_bin(SampleCtx<W> &x, int b, int d) {
    cg::cluster_group cl = cg::this_cluster();
    for (int i = b + d; i >= 0 && i < kSampleBins; i += d)
        for (int r = 0; r < x.C; ++r)
            if (cl.map_shared_rank(&x.sm, r)->cnt[i]) return i;
    return b;
}

// The exact cut at or near bin b: K: the first `k` tokens of the order (`count`
// of them lie before the bin); else the shortest prefix that weighs `target`.
// `sum`: the weight of the prefix; `at_bin`, `below`: the bin, and the weight
// of this lane's tokens in the bins before it; `at_lo`, `at_hi`: its first and
// last one in the bin.
template <bool K, int W>
__device__ void resolve(SampleCtx<W> &x, int b, uint32_t count, uint32_t k, double target, float &cut,
                        uint32_t &cut_idx, uint64_t &sum, int &at_bin, uint64_t &below, int &at_lo, int &at_hi) {
    SampleShared<W> &sm = x.sm;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x;
    for (;;) {
        if (tid == 0) sm.n_list = 0;
        __syncthreads();
        uint64_t w = 0;
        uint32_t c = 0;
        at_lo = x.per, at_hi = -1;
        for (int q0 = 0; q0 < x.per; q0 += 32) {
            uint32_t less, at;
            mark_bins(x, q0, b, less, at);
            for (; less; less &= less - 1) w = x.weigh.add(w, x.logits[q0 + __ffs(less) - 1]);
            list_tokens(x, q0, at);
            if (at) {
                c += __popc(at);
                at_lo = min(at_lo, q0 + __ffs(at) - 1);
                at_hi = q0 + 31 - __clz(at);
            }
        }
        at_bin = b;
        below = w;
        uint64_t before, skip;
        uint32_t m;
        cluster_sums(x, w, c, before, m, skip);
        if (m > (uint32_t)(W * 32)) {
            uint64_t part;
            double need = K ? (double)(k - count) : target - (double)before;
            if (!K) {                                               // whether the cut lies in this bin at all
                uint64_t bin_w = 0, t2, s2;
                uint32_t c2;
                for_logits(x, [&](float l, int) {
                    if (x.weigh.bin(l) == b) bin_w = x.weigh.add(bin_w, l);
                });
                cluster_sums(x, bin_w, 0, t2, c2, s2);
                const int to = need <= 0.0 ? next_bin(x, b, -1) : need > (double)t2 ? next_bin(x, b, 1) : b;
                if (to != b) {
                    b = to;
                    continue;
                }
                need = fmin(need, (double)t2);
            }
            bisect<K>(x, b, need, cut, cut_idx, part);
            sum = before + part;
            return;
        }
        if (x.rank == 0) {
            uint64_t token, all;
            const int got = gather(x, token);
            int place = tid;                                        // in the order
            uint64_t mine, upto;
            bool lead = tid < got;
            if (got <= W * 16) {                                    // two threads or more per token
                const int n = got <= W * 4 ? 8 : got <= W * 8 ? 4 : 2, i = tid / n;
                if (tid < got) {
                    sm.all[tid] = token;
                    sm.list[tid] = x.weigh(logit_of(~(uint32_t)(token >> 32)));
                }
                __syncthreads();
                token = i < got ? sm.all[i] : ~0ull;
                mine = i < got ? sm.list[i] : 0;
                lead = i < got && tid % n == 0;
                count_before(sm.all, sm.list, got, n, token, place, upto);
                upto += before + mine;
            } else {
                token = block_sort(sm, token, sort_size(got));
                mine = tid < got ? x.weigh(logit_of(~(uint32_t)(token >> 32))) : 0;
                upto = before + block_scan(sm, mine, all);
            }
            if (tid == 0) sm.out_move = got == 0 || (!K && target <= (double)before) ? -1 : 1;
            __syncthreads();
            const bool down = sm.out_move < 0;
            __syncthreads();
            const bool hit = K ? (uint32_t)place + 1 == k - count
                               : !down && (double)upto >= target && (double)(upto - mine) < target;
            if (lead && hit) {                                      // one thread at most
                sm.out_move = 0;
                sm.out_key = ~(uint32_t)(token >> 32);
                sm.out_idx = (uint32_t)token;
                sm.out_w = upto;
            }
        }
        if (x.rank == 0) {
            __syncthreads();
            if (tid < x.C) {
                SampleShared<W> *o = cl.map_shared_rank(&sm, tid);
                o->got_move = sm.out_move, o->got_key = sm.out_key, o->got_idx = sm.out_idx, o->got_w = sm.out_w;
            }
        }
        cl.sync();
        const int move = sm.got_move;
        cut = logit_of(sm.got_key), cut_idx = sm.got_idx, sum = sm.got_w;
        if (move == 0) return;
        const int to = next_bin(x, b, move);
        if (to == b) {                                              // no such bin: the cut is at the end of the row
            cut = move < 0 ? x.weigh.top : kNegInf, cut_idx = 0xFFFFFFFFu;
            at_bin = -1;
            return;
        }
        b = to;
    }
}

template <int W>
__global__ void __launch_bounds__(W * 32, W == 16 ? 2 : 1) sample_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SampleShared<W> &sm = *reinterpret_cast<SampleShared<W> *>(smem_raw);
    float *logits = reinterpret_cast<float *>(smem_raw + sizeof(SampleShared<W>));
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_launch_dependents();
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");       // this CTA runs: others may write to it
    if (tid < 64) sm.step[tid] = c_step[tid], sm.start[tid] = c_bin[tid];
    for (int i = tid; i < kSampleBins; i += (W * 32)) sm.cnt[i] = sm.low[i] = 0;
    if (tid == 0) sm.n_list = 0;
    const int64_t row = blockIdx.x / C;
    const int64_t chunk = (int64_t)p.per * (W * 32), base = rank * chunk;
    const int n = (int)max((int64_t)0, min(chunk, p.V - base));
    for (int i = n + tid; i < (int)chunk; i += (W * 32)) logits[i] = kNegInf;
    griddep_wait();
    // ---- the row's part, and the maximum
    float top = kNegInf;
    {
        const uint8_t *src = static_cast<const uint8_t *>(p.logits) + (row * p.ld + base) * (p.bf16 ? 2 : 4);
        const bool vec = ((uintptr_t)src & 15) == 0;
        int done = 0;
        if (vec && p.bf16) {
            done = n & ~7;
#pragma unroll 4
            for (int i = 8 * tid; i < done; i += 8 * (W * 32)) {
                const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(src + 2 * i));
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                float l[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    l[2 * j] = plain_logit(__uint_as_float(w[j] << 16));
                    l[2 * j + 1] = plain_logit(__uint_as_float(w[j] & 0xFFFF0000u));
                    top = fmaxf(top, fmaxf(l[2 * j], l[2 * j + 1]));
                }
                *reinterpret_cast<float4 *>(logits + i) = make_float4(l[0], l[1], l[2], l[3]);
                *reinterpret_cast<float4 *>(logits + i + 4) = make_float4(l[4], l[5], l[6], l[7]);
            }
        } else if (vec) {
            done = n & ~3;
#pragma unroll 8
            for (int i = 4 * tid; i < done; i += 4 * (W * 32)) {
                const float4 v = __ldcs(reinterpret_cast<const float4 *>(src + 4 * i));
                const float4 l = make_float4(plain_logit(v.x), plain_logit(v.y), plain_logit(v.z), plain_logit(v.w));
                top = fmaxf(fmaxf(top, fmaxf(l.x, l.y)), fmaxf(l.z, l.w));
                *reinterpret_cast<float4 *>(logits + i) = l;
            }
        }
        for (int i = done + tid; i < n; i += (W * 32)) {
            const float l = plain_logit(p.bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(src)[i])
                                               : reinterpret_cast<const float *>(src)[i]);
            logits[i] = l;
            top = fmaxf(top, l);
        }
    }
    const float temp = p.temperature ? p.temperature[row] : p.temperature0;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p0, min_p = p.min_p ? p.min_p[row] : p.min_p0;
    const int32_t top_k = p.top_k ? p.top_k[row] : p.top_k0;
    const float u = p.u[row];
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    uint32_t high = __reduce_max_sync(0xffffffffu, key_of(top));
    if (lane == 0) sm.red_c[0][warp] = high;
    __syncthreads();
    if (warp == 0) {
        high = __reduce_max_sync(0xffffffffu, lane < W ? sm.red_c[0][lane] : 0u);
        if (lane < C) cl.map_shared_rank(&sm, lane)->peer_c[0][rank] = high;
    }
    cl.sync();
    top = logit_of(__reduce_max_sync(0xffffffffu, lane < C ? sm.peer_c[0][lane] : 0u));
    SampleCtx<W> x = {sm, logits + tid * p.per, p.per, C, rank, (uint32_t)(base + tid * p.per), 1, {}};
    Weigher &weigh = x.weigh;
    const double inv = 1.4426950408889634074 / (double)temp;
    weigh.top = top;
    weigh.chi = (float)inv;
    weigh.clo = (float)(inv - (double)weigh.chi);
    weigh.limit = (float)p.sh + 0.75f;
    weigh.sh = p.sh;
    weigh.step = sm.step;
    // (a temperature whose reciprocal leaves fp32 is the limit of 0)
    const bool none = top == kNegInf, greedy = !(temp > 0.f) || top_k == 1 || !(weigh.chi < __int_as_float(0x7f800000));
    if (none || greedy) {
        // ---- the lowest index of the maximum
        uint32_t at = 0xFFFFFFFFu;
        if (!none)
            for (int q = p.per - 1; q >= 0; --q)
                if (x.logits[q] == top) at = x.first + (uint32_t)q;
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) sm.red_c[1][warp] = at;
        __syncthreads();
        if (warp == 0) {
            at = __reduce_min_sync(0xffffffffu, lane < W ? sm.red_c[1][lane] : 0xFFFFFFFFu);
            if (lane == 0) cl.map_shared_rank(&sm, 0)->peer_c[1][rank] = at;
        }
        cl.sync();
        if (rank == 0 && warp == 0) {
            at = __reduce_min_sync(0xffffffffu, lane < C ? sm.peer_c[1][lane] : 0xFFFFFFFFu);
            if (lane == 0) p.tokens[row] = none ? -1 : (int64_t)at;
        }
        return;
    }
    const uint64_t min_w =
        min_p > 0.f ? max((uint64_t)1, (uint64_t)ceil(fmin((double)min_p, 1.0) * (double)(1ull << p.sh))) : 1ull;
    int at_bin = -1;                                                // the cut's bin, where it was resolved
    uint64_t below = 0;
    int at_lo = 0, at_hi = -1;
    float cut = kNegInf;                                            // keep logits above the cut, and equal ones up to an index
    uint32_t cut_idx = 0xFFFFFFFFu;
    const bool by_k = top_k > 0 && top_k < p.V, by_p = top_p < 1.f;
    if (by_k || by_p) {
        // ---- the histogram (behind top-k only of counts: mostly few tokens are left), and the row's whole weight
        uint64_t w = 0, total = 0, skip;
        for_logits(x, [&](float l, int) {
            float d, y, kf;
            int k;
            const bool ok = weigh.place(l, d, y, kf, k);
            if (by_k) {
                if (ok) atomicAdd(&sm.cnt[k], 1u);
                return;
            }
            const uint32_t m = weigh.mantissa(l, d, y, kf, k);
            w = weigh.add(w, ok ? m : 0u, k);
            if (ok) {
                atomicAdd(&sm.cnt[k], 1u);
                atomicAdd(&sm.low[k], (uint32_t)max((int)(sm.start[k & 63] - m), 0) >> 10);
            }
        });
        uint32_t c;
        if (by_k) cl.sync();
        else cluster_sums(x, w, 0, total, c, skip);
        find_bin(x, by_k ? (uint32_t)top_k : 0u, fmax((double)top_p * (double)total, 1.0));
        int b = sm.pick_bin;
        uint32_t before = sm.pick_before, count = sm.pick_count;
        if (before + count <= (uint32_t)(W * 32) && b < kSampleBins - 1) {
            // ---- all that can be kept on one CTA, one token per thread
            for (int q0 = 0; q0 < x.per; q0 += 32) {
                uint32_t less, at;
                mark_bins(x, q0, b + 1, less, at);
                list_tokens(x, q0, less);
            }
            cl.sync();
            bool finish = false;
            if (rank == 0) {
                uint64_t token, listed, sum;
                const int m = gather(x, token);
                const int top_n = by_k ? min(top_k, m) : m;         // of the order
                if (m <= W * 4) {                                   // eight threads per token
                    if (tid < m) {
                        sm.all[tid] = token;
                        sm.list[tid] = weigh(logit_of(~(uint32_t)(token >> 32)));
                    }
                    __syncthreads();
                    const int i = tid >> 3;
                    const bool lead = i < m && (tid & 7) == 0;
                    uint64_t mine = i < m ? sm.list[i] : 0, less;
                    token = i < m ? sm.all[i] : ~0ull;
                    int place;
                    count_before(sm.all, sm.list, m, 8, token, place, less);
                    if (lead && place == top_n - 1) sm.out_w = less + mine;
                    __syncthreads();
                    listed = sm.out_w;
                    const double target = fmax((double)top_p * (double)(by_k ? listed : total), 1.0);
                    // top-p alone: the histogram's estimate may have missed the cut
                    finish = !(by_p && !by_k && (double)listed < target);
                    const bool keep = lead && place < top_n && (!by_p || (double)less < target || place == 0) && mine >= min_w;
                    const int kept_n = __syncthreads_count(keep);
                    if (lead) {
                        sm.all[i] = token << 32;                    // by index
                        sm.list[i] = keep ? mine : 0;
                        if (place == kept_n - 1) sm.out_w = less + mine;
                    }
                    __syncthreads();
                    sum = sm.out_w;
                    token <<= 32;
                    mine = i < m ? sm.list[i] : 0;
                    count_before(sm.all, sm.list, m, 8, token, place, less);
                    const double ut = fmax((double)u, 0.0) * (double)sum;
                    const uint64_t goal = min(ut < (double)sum ? (uint64_t)ut : sum - 1, sum - 1);
                    if (finish && lead && goal >= less && goal < less + mine) p.tokens[row] = (int64_t)(token >> 32);
                } else {
                    const int n2 = sort_size(m);
                    token = block_sort(sm, token, n2);
                    const uint64_t mine = tid < top_n ? weigh(logit_of(~(uint32_t)(token >> 32))) : 0;
                    const uint64_t upto = block_scan(sm, mine, listed);
                    const double target = fmax((double)top_p * (double)(by_k ? listed : total), 1.0);
                    finish = !(by_p && !by_k && (double)listed < target);
                    if (finish) {
                        const uint64_t keep = (by_p && (double)(upto - mine) >= target && tid > 0) || mine < min_w ? 0 : mine;
                        block_scan(sm, keep, sum);
                        sm.list[tid] = keep;
                        // by index
                        token = block_sort(sm, keep ? token << 32 | (uint32_t)tid : ~0ull, n2);
                        const uint64_t one = token != ~0ull ? sm.list[(uint32_t)token] : 0;
                        uint64_t skip2;
                        const uint64_t run = block_scan(sm, one, skip2);
                        const double ut = fmax((double)u, 0.0) * (double)sum;
                        const uint64_t goal = min(ut < (double)sum ? (uint64_t)ut : sum - 1, sum - 1);
                        if (goal < run && goal >= run - one) p.tokens[row] = (int64_t)(token >> 32);     // exactly one
                    }
                }
                if (tid < C) cl.map_shared_rank(&sm, tid)->got_move = finish;
            }
            cl.sync();
            finish = sm.got_move;
            if (finish) return;
        }
        uint64_t sum = total;
        if (by_k && count > 0) {
            resolve<true>(x, b, before, (uint32_t)top_k, 0.0, cut, cut_idx, sum, at_bin, below, at_lo, at_hi);
        } else if (by_k && by_p) {                                  // k reaches past every weight
            uint64_t all = 0;
            for_logits(x, [&](float l, int) { all = weigh.add(all, l); });
            cluster_sums(x, all, 0, sum, c, skip);
        }
        if (by_p) {
            const double target = fmax((double)top_p * (double)sum, 1.0);
            if (by_k) {
                for_logits(x, [&](float l, int) {                   // the histogram's weights
                    float d, y, kf;
                    int k;
                    const bool ok = weigh.place(l, d, y, kf, k);
                    const uint32_t m = weigh.mantissa(l, d, y, kf, k);
                    if (ok) atomicAdd(&sm.low[k], (uint32_t)max((int)(sm.start[k & 63] - m), 0) >> 10);
                });
                cl.sync();
                find_bin(x, 0u, target);
                b = sm.pick_bin;
                __syncthreads();
            }
            resolve<false>(x, b, 0, 0, target, cut, cut_idx, sum, at_bin, below, at_lo, at_hi);
        }
    }
    // ---- the kept weight of each lane's part
    const auto kept = [&](uint64_t acc, float l, uint32_t index) -> uint64_t {
        const uint64_t w = weigh.add(0, l, l > cut || (l == cut && index <= cut_idx));
        return acc + (w >= min_w ? w : 0);
    };
    uint64_t w = 0, total, before;
    uint32_t c;
    if (at_bin >= 0 && min_w == 1) {                                // only the cut's bin is left to look at
        w = below;
        for (int q = at_lo; q <= at_hi; ++q)
            if (weigh.bin(x.logits[q]) == at_bin) w = kept(w, x.logits[q], x.first + (uint32_t)q);
    } else {
        for_logits(x, [&](float l, int q) { w = kept(w, l, x.first + (uint32_t)q); });
    }
    cluster_sums(x, w, 0, total, c, before);
    // ---- the first token whose running sum exceeds u * total: its lane, then the token
    const double ut = fmax((double)u, 0.0) * (double)total;
    const uint64_t goal = min(ut < (double)total ? (uint64_t)ut : total - 1, total - 1);
    const uint64_t upto = before + warp_scan(w);
    const uint32_t over = __ballot_sync(0xffffffffu, upto > goal);
    if (goal >= before && over) {                                   // exactly one warp of the cluster: it shares the lane's tokens
        const int lead = __ffs(over) - 1;
        const float *l = logits + (tid - lane + lead) * p.per;
        const uint32_t first = (uint32_t)(base + (tid - lane + lead) * p.per);
        uint64_t run = __shfl_sync(0xffffffffu, upto - w, lead);
        for (int q0 = 0; q0 < p.per; q0 += 32) {
            const uint32_t index = first + (uint32_t)(q0 + lane);
            run += warp_scan(q0 + lane < p.per ? kept(0, l[q0 + lane], index) : 0);
            const uint32_t hit = __ballot_sync(0xffffffffu, run > goal);
            if (hit) {
                if (lane == __ffs(hit) - 1) p.tokens[row] = (int64_t)index;
                break;
            }
            run = __shfl_sync(0xffffffffu, run, 31);
        }
    }
}

// CTAs per row, and warps per CTA: 32, one CTA per SM, or 16, two per SM, which
// fill each other's waits.  The pair with the least (waves of clusters) * (40 +
// tokens per thread): a thread's start, exchanges and searches cost about as much
// as 40 tokens (16 without filters, 70 for top-p).  A wave of 32 warps takes 0.9
// of one of 2 x 16; a last wave of 16 that leaves every CTA its SM 0.6, as the
// SMs come free one by one, and a first one that is nearly empty 0.75.  How many
// clusters run at once is the device's to say: clusters of 8 with one CTA per SM
// leave SMs out, and 16 of them took two waves.  Measured, 32 warps against 16
// with twice the CTAs: 129 rows of 73448, top-p: 77 us and 88 (two full waves
// each); 40 rows of 128256: 79 and 68 (the second wave nearly empty).  With
// settings per row, rows take different times and the next begin as one ends:
// no wave is rounded up (16 such rows of 128256: 37 us with 8 CTAs, of which 14
// clusters run at once, and 53 with 4; 16 rows of one setting, top-p: 50 and 39).
struct SampleShape {
    int ctas, warps;
};
template <int W>
static int sample_slots(int dev, int lg) {              // clusters of 2^lg CTAs that run at once
    static std::atomic<int> known[64][4];
    if (dev < 64)
        if (const int n = known[dev][lg].load(std::memory_order_relaxed)) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << lg);
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = W == 32 ? 200 * 1024 : 112 * 1024;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1u << lg;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, sample_kernel<W>, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = std::max(1, (W == 32 ? 148 : 296) >> lg);
    }
    if (dev < 64) known[dev][lg].store(n, std::memory_order_relaxed);
    return n;
}
static SampleShape sample_shape(int dev, int64_t B, int64_t V, bool mixed) {
    SampleShape best = {kSampleMaxCluster, 32};
    int64_t least = INT64_MAX;
    for (int warps = 32; warps >= 16; warps /= 2)
        for (int lg = 0; 1 << lg <= kSampleMaxCluster; ++lg) {
            const int64_t threads = (int64_t)warps * 32 << lg, per = ((V + threads - 1) / threads) | 1;
            const int64_t smem = per * warps * 128 + (int64_t)(warps == 32 ? sizeof(SampleShared<32>) : sizeof(SampleShared<16>));
            if (V > (int64_t)kSampleMaxKeys << lg || smem > (warps == 32 ? 227 : 112) * 1024) continue;
            const int64_t slots = warps == 32 ? sample_slots<32>(dev, lg) : sample_slots<16>(dev, lg);
            const int64_t full = B / slots, rest = B % slots;
            const int64_t waves = mixed         ? std::max<int64_t>(100, 100 * B / slots) * (warps == 32 ? 90 : 100) / 100
                                  : warps == 32 ? (full + (rest > 0)) * 90
                                              : full * 100 + (rest == 0               ? 0
                                                              : full && 2 * rest <= slots ? 60
                                                              : 4 * rest <= slots     ? 75
                                                                                      : 100);
            if (waves * (40 + per) < least) {
                least = waves * (40 + per);
                best = {1 << lg, warps};
            }
        }
    return best;
}

template <int W>
static int sample_launch(SampleParams p, int64_t B, int C, cudaStream_t st) {
    p.per = (int)((p.V + (int64_t)C * W * 32 - 1) / ((int64_t)C * W * 32)) | 1;
    const size_t smem = sizeof(SampleShared<W>) + (size_t)p.per * W * 32 * 4;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * C));
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)C;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<W>, p);
    if (e != cudaSuccess) return set_error(BF16X_ERR_CUDA, "bf16x_sample: launch: %s", cudaGetErrorString(e));
    return check_launch("sample_kernel");
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
    static std::atomic<uint64_t> raised{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (e == cudaSuccess && !(raised.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(sample_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_kernel<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e == cudaSuccess) raised.fetch_or(bit, std::memory_order_relaxed);
    }
    if (e != cudaSuccess) return set_error(BF16X_ERR_CUDA, "bf16x_sample: shared memory: %s", cudaGetErrorString(e));
    const SampleShape shape = sample_shape(dev, B, V, temperature || top_k || top_p || min_p);
    SampleParams p = {};
    p.logits = logits, p.ld = ld, p.V = V, p.bf16 = dtype == BF16X_DTYPE_BF16;
    int lg = 0;
    while (((int64_t)1 << lg) < V) ++lg;
    p.sh = std::min(47, 62 - lg);                     // a row's sum fits 64 bits
    p.u = u, p.temperature = temperature, p.top_p = top_p, p.min_p = min_p, p.top_k = top_k;
    p.temperature0 = temperature0, p.top_p0 = top_p0, p.min_p0 = min_p0, p.top_k0 = top_k0;
    p.tokens = tokens;
    return shape.warps == 32 ? sample_launch<32>(p, B, shape.ctas, (cudaStream_t)stream)
                             : sample_launch<16>(p, B, shape.ctas, (cudaStream_t)stream);
}
