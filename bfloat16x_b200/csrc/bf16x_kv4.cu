// bf16x_kv4.cu -- writing the 4-bit key/value cache, reading it back, and
// attention of few query rows over it (decode steps, a few guessed tokens).
#include <algorithm>

#include <cuda_runtime.h>

#include "bf16x_kv4.cuh"
#include "bf16x_kv4_rows.cuh"

namespace bf16x {

// --------------------------------------------------------------------- write
// y = the head's channel pairs (2i, 2i+1) turned by the angle of the position
// (q and k), rounded to bf16; then for every 32 channels of k and v
//   m = min y,  d = (max y - m) / 15 rounded up to bf16,  code = rint((y - m) / d).
// d is rounded up so that no code exceeds 15, and m is a bf16 value already.
// A group that holds an infinity or a NaN gets d = NaN, m = 0: it reads as NaN
// and m stays finite, so a masked position cannot reach another row's sums.
// A group of one value has codes 0, so its d is free: 2^-13 |m|, which gives
// the attention the group's magnitude.
// Every operation is rounded by itself (no fused multiply-add), so the codes
// do not depend on how the compiler contracts.
//
// A CTA per token: D/8 lanes per head, 8 channels each (a 16-byte load, and the
// whole K word of a lane), over the heads in turn, so that the angles of the
// position are loaded once.  4 x 2047 tokens of the 8B heads (32 + 2 * 8 of 128
// channels, 190 MB) take 48 us, 4.0 TB/s; one token 3.4 us, all latency.  Bound
// by instructions (0.78 per cycle and scheduler, memory at a third), one value
// each: arithmetic on fp32 pairs and minima of bf16 pairs would be fewer and
// round the same.  Rounding by a division per value took 118 us.
template <int D>
__device__ __forceinline__ void kv4_quantize8(const float (&y)[8], float &d, float &m, uint32_t &codes) {
    float lo = y[0], hi = y[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = fmin_nan(lo, y[i]);
        hi = fmax_nan(hi, y[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fmin_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmax_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const float span = __fdiv_rn(__fsub_rn(hi, lo), 15.f);
    d = __uint_as_float((__float_as_uint(span) + 0xFFFFu) & 0xFFFF0000u);
    m = lo;
    codes = 0;
    if (!(fabsf(span) < __int_as_float(0x7f800000))) {            // infinity or NaN in the group
        d = __int_as_float(0x7fc00000);
        m = 0.f;
    } else if (d == 0.f) {                                        // a constant group: m, with any d; one near m's
        d = __uint_as_float(__float_as_uint(fabsf(lo) * 0x1p-13f) & 0xFFFF0000u);      // own scale suits the reader
    } else if (d < 0x1p-100f || d > 0x1p100f) {                   // 1/d may leave fp32
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = rintf(__fdiv_rn(__fsub_rn(y[i], lo), d));
            codes |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * i);
        }
    } else {
        // the nearest whole number to a / d without a division: n from a * (1/d),
        // which may miss by one, and a - n d, which is exact (n d has 12 bits),
        // against d / 2; halves go to the even n.  a / d <= 15, so n is a code.
        const float inv = __frcp_rn(d), half = 0.5f * d, more = __uint_as_float(__float_as_uint(half) + 1u);
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            const float a = __fsub_rn(y[i], lo), t = __fmaf_rn(a, inv, 12582912.f), rest = __fmaf_rn(-__fsub_rn(t, 12582912.f), d, a);
            uint32_t n = __float_as_uint(t) & 0x1Fu;
            if (fabsf(rest) >= (n & 1u ? half : more)) n += rest > 0.f ? 1u : ~0u;
            codes = codes * 16u + n;
        }
    }
}

struct Kv4AppendParams {
    const uint16_t *qkv;
    int64_t ld_b, ld_t;                 // elements
    int T, H, KV, pos_stride;
    const int64_t *pos0;
    const float *cos_t, *sin_t;         // NULL: no rotation
    uint16_t *q_out;
    uint8_t *blocks;
    int64_t max_seq, nblk;
};

template <int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4AppendParams p) {
    using L = KvLayout<D>;
    constexpr int LPH = D / 8;                                      // lanes per head
    griddep_launch_dependents();
    griddep_wait();
    // a token per CTA: its threads keep their channels' angles and go over the heads
    constexpr int STEP = 256 / LPH;
    const int heads = p.H + 2 * p.KV, l = threadIdx.x % LPH;
    const int64_t tok = blockIdx.x;
    const uint32_t b = blockIdx.x / (uint32_t)p.T, t = blockIdx.x - b * (uint32_t)p.T;
    const int64_t pos = p.pos0[(int64_t)b * p.pos_stride] + t;
    const bool inside = pos >= 0 && pos < p.max_seq, turn = p.cos_t != nullptr && inside;
    if (pos >= p.max_seq && threadIdx.x == 0) atomicOr(&g_status, kErrBadIndex);
    const uint16_t *src = p.qkv + (int64_t)b * p.ld_b + (int64_t)t * p.ld_t + 8 * l;
    int head = (int)threadIdx.x / LPH;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (head < heads) raw = *reinterpret_cast<const uint4 *>(src + head * D);
    float c[4] = {}, s[4] = {};
    if (turn) {
        const float4 c4 = *reinterpret_cast<const float4 *>(p.cos_t + pos * (D / 2) + 4 * l);
        const float4 s4 = *reinterpret_cast<const float4 *>(p.sin_t + pos * (D / 2) + 4 * l);
        c[0] = c4.x, c[1] = c4.y, c[2] = c4.z, c[3] = c4.w;
        s[0] = s4.x, s[1] = s4.y, s[2] = s4.z, s[3] = s4.w;
    }
    const int r = (int)pos & 15, grp = l / 4, t4 = l % 4;
    uint8_t *blocks = p.blocks + ((int64_t)b * p.KV * p.nblk + (pos >> 4)) * L::kBytes;        // of kv head 0; used if inside
    uint16_t *q_out = p.q_out + tok * p.H * D + 8 * l;
    for (int base = 0; base < heads; base += STEP, head += STEP) {  // whole warps: the quantiser shuffles
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if (head + STEP < heads) raw = *reinterpret_cast<const uint4 *>(src + (head + STEP) * D);
        const bool live = head < heads;
        uint32_t o[4] = {w[0], w[1], w[2], w[3]};
        if (turn && head < p.H + p.KV) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = bf_lo(w[i]), y = bf_hi(w[i]);
                o[i] = pack_bf16x2(__fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i])),
                                   __fadd_rn(__fmul_rn(x, s[i]), __fmul_rn(y, c[i])));
            }
        }
        if (live && head < p.H)                                     // a position outside the cache: zeros
            *reinterpret_cast<uint4 *>(q_out + head * D) = inside ? make_uint4(o[0], o[1], o[2], o[3]) : make_uint4(0, 0, 0, 0);
        if (!__any_sync(0xffffffffu, live && head >= p.H)) continue;
        float y[8], d, m;
        uint32_t codes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[2 * i] = bf_lo(o[i]);
            y[2 * i + 1] = bf_hi(o[i]);
        }
        kv4_quantize8<D>(y, d, m, codes);
        if (!live || head < p.H || !inside) continue;
        const bool is_v = head >= p.H + p.KV;
        const int kvh = head - p.H - (is_v ? p.KV : 0);
        uint8_t *blk = blocks + (int64_t)kvh * p.nblk * L::kBytes;
        const uint16_t db = (uint16_t)(__float_as_uint(d) >> 16), mb = (uint16_t)(__float_as_uint(m) >> 16);
        if (!is_v) {
            *reinterpret_cast<uint32_t *>(blk + ((r * 4 + t4) * L::NG + grp) * 4) = codes;
            if (t4 == 0) {
                *reinterpret_cast<uint16_t *>(blk + L::kKd + (r * L::NG + grp) * 2) = db;
                *reinterpret_cast<uint16_t *>(blk + L::kKm + (r * L::NG + grp) * 2) = mb;
            }
        } else {
            const int pp = r / 8, tt = (r % 8) / 2, h = r % 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int g = 2 * t4 + i;                           // channels 32 grp + 4 g ..
                *reinterpret_cast<uint16_t *>(blk + L::kV + (((pp * 8 + g) * 4 + tt) * L::NG + grp) * 4 + 2 * h) =
                    (uint16_t)(codes >> (16 * i));
            }
            if (t4 == 0) {
                *reinterpret_cast<uint16_t *>(blk + L::kVd + (r * L::NG + grp) * 2) = db;
                *reinterpret_cast<uint16_t *>(blk + L::kVm + (((r / 2) * L::NG + grp) * 2 + h) * 2) = mb;
            }
        }
    }
}

// ---------------------------------------------------------------------- read
// The values that positions *pos0 .. *pos0 + T - 1 stand for, d * code + m in
// fp32 rounded to bf16; a position outside the cache reads as zeros.
// Four tokens' heads of K and V per CTA, whole warps for K or V, all loads of a
// thread before its first use: 4 x 2047 tokens of 8 heads of 128 channels (44
// MB, most of it written) take 10.2 us, 4.3 TB/s (one token per CTA 13.7, eight
// 9.7; K and V in turn within a warp, and a conversion per code, 14.7 with one).
// Bound by instructions (0.75 per cycle and scheduler, one value each) and its
// start.
struct Kv4ReadParams {
    const uint8_t *blocks;
    int64_t max_seq, nblk;
    int T, KV, pos_stride;
    const int64_t *pos0;
    uint16_t *k_out, *v_out;
};

constexpr int kReadTokens = 4;

template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p) {
    using L = KvLayout<D>;
    constexpr int LPH = D / 8;
    griddep_launch_dependents();
    griddep_wait();
    const int part = (int)(blockIdx.y * (256 / LPH) + threadIdx.x / LPH), l = threadIdx.x % LPH;        // K's heads, V's heads
    if (part >= 2 * p.KV) return;
    const bool is_v = part >= p.KV;
    const int kvh = is_v ? part - p.KV : part;
    const uint32_t chunks = ((uint32_t)p.T + kReadTokens - 1) / kReadTokens, b = blockIdx.x / chunks;
    const int t0 = (int)(blockIdx.x - b * chunks) * kReadTokens, n = min(kReadTokens, p.T - t0);
    const int64_t pos0 = p.pos0[(int64_t)b * p.pos_stride] + t0;
    if (pos0 + n > p.max_seq && l == 0) atomicOr(&g_status, kErrBadIndex);
    const uint8_t *head = p.blocks + ((int64_t)b * p.KV + kvh) * p.nblk * L::kBytes;
    const int grp = l / 4, t4 = l % 4;
    uint32_t codes[kReadTokens];
    uint16_t db[kReadTokens], mb[kReadTokens];
#pragma unroll
    for (int i = 0; i < kReadTokens; ++i) {                         // all loads before the first is used
        const int64_t pos = pos0 + i;
        const uint8_t *blk = head + (pos >> 4) * L::kBytes;
        const int r = (int)pos & 15;
        codes[i] = 0, db[i] = mb[i] = 0;
        if (i >= n || pos < 0 || pos >= p.max_seq) continue;
        if (!is_v) {
            codes[i] = *reinterpret_cast<const uint32_t *>(blk + ((r * 4 + t4) * L::NG + grp) * 4);
            db[i] = *reinterpret_cast<const uint16_t *>(blk + L::kKd + (r * L::NG + grp) * 2);
            mb[i] = *reinterpret_cast<const uint16_t *>(blk + L::kKm + (r * L::NG + grp) * 2);
        } else {
            const int pp = r / 8, tt = (r % 8) / 2, h = r % 2;
            const uint8_t *at = blk + L::kV + (((pp * 8 + 2 * t4) * 4 + tt) * L::NG + grp) * 4 + 2 * h;
            codes[i] = *reinterpret_cast<const uint16_t *>(at) |
                       (uint32_t)*reinterpret_cast<const uint16_t *>(at + 16 * L::NG) << 16;
            db[i] = *reinterpret_cast<const uint16_t *>(blk + L::kVd + (r * L::NG + grp) * 2);
            mb[i] = *reinterpret_cast<const uint16_t *>(blk + L::kVm + (((r / 2) * L::NG + grp) * 2 + h) * 2);
        }
    }
    uint16_t *out = (is_v ? p.v_out : p.k_out) + (((int64_t)b * p.T + t0) * p.KV + kvh) * D + 8 * l;
#pragma unroll
    for (int i = 0; i < kReadTokens; ++i) {
        if (i >= n) break;
        const float d = bf16_bits_to_f32(db[i]), m = bf16_bits_to_f32(mb[i]);
        float y[8];
        if (d >= 0x1p-100f && d <= 0x1p100f) {
            // 2^23 + 16^j code by an OR; times d / 16^j less 2^23 d / 16^j, both exact: d * code, rounded once
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float s = d * (1.f / (float)(1 << (4 * (k & 3))));
                const uint32_t f = ((k < 4 ? codes[i] : codes[i] >> 16) & (15u << (4 * (k & 3)))) | 0x4B000000u;
                y[k] = __fadd_rn(__fmaf_rn(__uint_as_float(f), s, s * -8388608.f), m);
            }
        } else {                        // (outside the cache too: zeros)
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = __fadd_rn(__fmul_rn(d, (float)((codes[i] >> (4 * k)) & 15u)), m);
        }
        *reinterpret_cast<uint4 *>(out + (int64_t)i * p.KV * D) = make_uint4(
            pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
    }
}

// -------------------------------------------------------------------- attend
// What a warp does with its rows and blocks is in bf16x_kv4_rows.cuh; here is which
// warp does which, and how the parts come together.
//
// The schedule.  A unit is one row tile of one (sequence, kv head); its work is
// the blocks that its sequence holds, plus kUnitCost blocks for starting and
// ending a unit.  The units' work, one after the other, is cut into equal
// shares, one for each warp of the grid: sequences of any lengths load the GPU
// evenly, no warp waits for another, and lengths are read on the device, so a
// captured call follows them.  A warp writes a unit that it has alone; of
// others it writes its part, at most one that began before its share (slot 0)
// and one that goes on after it (slot 1), and a second kernel joins the parts.
//
// Bound by latency: some 290 instructions per block of 16 positions at 128
// channels (unpacking codes, softmax, the weights times the scales, four mma per
// 32 channels) follow one another in one chain per warp, and the three warps per
// scheduler that the registers allow issue 0.54 per cycle; DRAM is at half.  About
// 8 us of a call are its start, the first loads and the
// join.  8B heads: one sequence of 131071 positions (168 MB) 44 us, 3.8 TB/s;
// 16 sequences of 17 to 16384 positions (168 MB) 41 us, 4.1 TB/s; one of 300
// positions 9.6 us; 8 x 4 tokens behind 900 to 5001 positions at 64 channels
// 19 us (20 with 8 warps per CTA instead of 12).
template <int D, int NT>
struct AttendCfg {
    static constexpr int kWarps = NT == 1 || D == 64 ? 12 : 8;      // per CTA and SM: what the registers allow
    static constexpr int kNB = NT == 1 ? 2 : 1;                     // blocks per stage
    static constexpr int kDepth = NT == 1 ? 3 : 5;                  // stages in flight per warp
};
constexpr int kUnitCost = 4;
constexpr int kMinShare = 4;

template <int D, int NT>
struct AttendSmem {
    static constexpr int W = AttendCfg<D, NT>::kWarps;
    uint8_t ring[W][AttendCfg<D, NT>::kDepth][AttendCfg<D, NT>::kNB * KvLayout<D>::kBytes];
    uint4 frag[W][NT][D / 32][32];
    uint64_t full[W][AttendCfg<D, NT>::kDepth];
    float2 ml[W][8 * NT];               // of the warps' parts of one unit, whose sums lie in the rings
    int merge[W][2];                    // how many of them (0: not so), and the slot of their sum
    static_assert(sizeof(ring[0]) >= 8 * NT * D * 4, "a part's sums");
};

__device__ __forceinline__ int64_t kv4_blocks_of(const Kv4AttendParams &p, int64_t pos0) {
    const int64_t n = min(pos0 + p.T, p.max_seq);
    return n > 0 ? (n + kKvBlock - 1) / kKvBlock : 0;
}

// a / b and its remainder, in 32 bits where that is enough (64-bit division takes some hundred instructions)
__device__ __forceinline__ int64_t quot(int64_t a, int64_t b) {
    return ((uint64_t)a | (uint64_t)b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

struct Kv4Plan {                        // how the work is cut
    int64_t total, shares, q, r;        // the first r shares have q + 1, the others q
    __device__ __forceinline__ Kv4Plan(int64_t total_, int64_t warps) : total(total_) {
        shares = max((int64_t)1, min(warps, quot(total, kMinShare)));
        q = quot(total, shares);
        r = total - q * shares;
    }
    __device__ __forceinline__ int64_t start(int64_t c) const { return q * c + min(c, r); }
    __device__ __forceinline__ int64_t share_of(int64_t at) const {
        const int64_t big = (q + 1) * r;
        return at < big ? quot(at, q + 1) : r + quot(at - big, q);
    }
};

// Work of all sequences, and of those before sequence `b` (one warp).
__device__ __forceinline__ int64_t kv4_work(const Kv4AttendParams &p, int64_t per_seq, int64_t b, int64_t &before) {
    int64_t x = 0, y = 0;
    for (int64_t i = threadIdx.x & 31; i < p.B; i += 32) {
        const int64_t k = kv4_blocks_of(p, p.pos0[i * p.pos_stride]);
        const int64_t w = k ? k + kUnitCost : 0;
        y += w;
        if (i < b) x += w;
    }
    for (int o = 16; o; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    before = x * per_seq;
    return y * per_seq;
}

// Walks a share, unit by unit.
struct Kv4Walk {
    int64_t b, pos0, nb;                // the unit's sequence and its blocks
    int kvh, tile;
    int64_t blk, end;                   // blocks of the unit in this share: [blk, end)
    int64_t left;                       // work of the share after this unit

    // at: where in the unit's work the share begins; work: what the share still has
    __device__ __forceinline__ void enter(int64_t at, int64_t work) {
        const int64_t stop = min(at + work, nb + kUnitCost);
        left = work - (stop - at);
        blk = max(at - kUnitCost, (int64_t)0);
        end = max(stop - kUnitCost, (int64_t)0);
    }
    __device__ __forceinline__ void next(const Kv4AttendParams &p) {       // left > 0
        if (++tile == p.tiles) {
            tile = 0;
            if (++kvh == p.KV) {
                kvh = 0;
                do {
                    ++b;
                    pos0 = p.pos0[b * p.pos_stride];
                    nb = kv4_blocks_of(p, pos0);
                } while (nb == 0);
            }
        }
        enter(0, left);
    }
};

template <int D, int NT>
__global__ void __launch_bounds__(AttendCfg<D, NT>::kWarps * 32, 1)
    kv4_attend_kernel(const __grid_constant__ Kv4AttendParams p) {
    using L = KvLayout<D>;
    using Cfg = AttendCfg<D, NT>;
    constexpr int NG = L::NG, C = 8 * NT, DEPTH = Cfg::kDepth, NB = Cfg::kNB;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    AttendSmem<D, NT> &sm = *reinterpret_cast<AttendSmem<D, NT> *>(smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    griddep_launch_dependents();
    if (lane == 0)
        for (int i = 0; i < DEPTH; ++i) mbar_init(&sm.full[warp][i], 1);
    fence_mbar_init();
    __syncwarp();
    griddep_wait();
    const int64_t per_seq = (int64_t)p.KV * p.tiles;
    Kv4Walk con;
    int64_t total, skip;
    if (p.B == 1) {
        con.b = 0;
        con.pos0 = p.pos0[0];
        con.nb = kv4_blocks_of(p, con.pos0);
        total = con.nb ? (con.nb + kUnitCost) * per_seq : 0;
    } else {
        total = kv4_work(p, per_seq, 0, skip);
    }
    if (total == 0) return;
    const Kv4Plan plan(total, p.warps);
    // ---- this warp's share: the CTAs in turn; or, of few units, equally many one after the other
    const uint32_t s0 = (uint32_t)plan.shares * blockIdx.x / gridDim.x,
                   s1 = (uint32_t)plan.shares * (blockIdx.x + 1) / gridDim.x;
    const int64_t share = p.few_units ? s0 + warp : (uint32_t)warp * gridDim.x + blockIdx.x;
    if (share >= (p.few_units ? s1 : plan.shares)) return;
    int64_t at = plan.start(share);
    const int64_t next_at = plan.start(share + 1), work = next_at - at;     // in the cut order
    if (p.B > 1) {
        // the sequence in which the share begins
        for (int64_t b0 = 0;; b0 += 32) {                           // ends: the share lies within the total
            const int64_t b = b0 + lane;
            const int64_t pos = b < p.B ? p.pos0[b * p.pos_stride] : -(int64_t)p.T;
            const int64_t nb = kv4_blocks_of(p, pos), mine = nb ? (nb + kUnitCost) * per_seq : 0;
            int64_t x = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, at < x);
            if (hit == 0 && b0 + 32 < p.B) {
                at -= __shfl_sync(0xffffffffu, x, 31);
                continue;
            }
            const int who = hit ? __ffs(hit) - 1 : 31;
            con.b = b0 + who;
            con.pos0 = __shfl_sync(0xffffffffu, pos, who);
            con.nb = __shfl_sync(0xffffffffu, nb, who);
            at -= __shfl_sync(0xffffffffu, x - mine, who);
            break;
        }
    }
    {
        const int64_t unit = quot(at, con.nb + kUnitCost);
        con.kvh = (int)quot(unit, p.tiles);
        con.tile = (int)(unit - (int64_t)con.kvh * p.tiles);
        at -= unit * (con.nb + kUnitCost);
        con.enter(at, work);
    }
    // One unit has all of this CTA's shares (and blocks in each): its warps join
    // their parts before they go to memory, as long contexts of few sequences
    // have hundreds of parts per unit (131072 positions of one sequence, 8B
    // heads: 1776 parts, of which the second kernel took 12 us).
    if (lane == 0) {                    // (not kept in registers over the loop)
        const int64_t unit_at = plan.start(share) - at;
        const bool merge = p.few_units && s1 - s0 > 1 && plan.q > kUnitCost && unit_at <= plan.start(s0) &&
                           plan.start(s1) <= unit_at + con.nb + kUnitCost;
        sm.merge[warp][0] = merge ? (int)(s1 - s0) : 0;
        sm.merge[warp][1] = (int)s0 * 2 + (plan.start(s0) - unit_at <= kUnitCost ? 1 : 0);
    }
    __syncwarp();
    // ---- the ring: stages of NB blocks
    const Kv4Lane<D> ln;
    const uint32_t ring0 = smem_u32(sm.ring[warp][0]), bar0 = smem_u32(&sm.full[warp][0]);
    uint32_t slot = 0, parity = 0;      // of the next stage to be read
    const uint8_t *src = nullptr;       // the next stage to be asked for
    int asked = 0, stages = 0, last_bytes = 0;
    const auto issue = [&](uint32_t to) {
        if (lane == 0) {
            const uint32_t bytes = asked == stages - 1 ? last_bytes : NB * L::kBytes;
            asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}"
                         :: "r"(bar0 + 8 * to), "r"(bytes) : "memory");
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         :: "r"(ring0 + to * NB * L::kBytes), "l"(src), "r"(bytes), "r"(bar0 + 8 * to) : "memory");
        }
        src += NB * L::kBytes;
        ++asked;
    };
    const auto start = [&]() {          // the first stages of the unit's part; every slot is free
        const int count = (int)(con.end - con.blk);
        stages = (count + NB - 1) / NB;
        last_bytes = (count - (stages - 1) * NB) * L::kBytes;
        src = p.blocks + ((con.b * p.KV + con.kvh) * p.nblk + con.blk) * L::kBytes;
        asked = 0;
        uint32_t to = slot;
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            if (asked < stages) issue(to);
            if (++to == DEPTH) to = 0;
        }
    };
    start();
    bool alive = true;
    for (;;) {
        // ---- one unit's part; positions from here on relative to its first one
        const int64_t b = con.b, pos0 = con.pos0, origin = con.blk * kKvBlock;
        const int kvh = con.kvh, row0 = con.tile * C;
        const bool began = con.blk == 0, ends = con.end == con.nb, any = con.end > con.blk;
        if (began && any && lane == 0) {
            // a unit that goes on after this share: its last block lies nb - end blocks past the share's end
            p.held[(b * p.KV + kvh) * p.tiles + con.tile] =
                make_int2((int)share, ends ? (int)share : (int)plan.share_of(next_at + (con.nb - con.end) - 1));
        }
        const int64_t lim = min(pos0 + min(row0 + C - 1, p.R - 1) / p.G + 1, p.max_seq);
        const int part = (int)(con.end - con.blk) * kKvBlock;
        const int n_keys = (int)max(min(lim - origin, (int64_t)part), (int64_t)0);
        // (a tile with a row past the cache goes masked throughout: that row sees nothing, its last one lies furthest)
        const bool past = pos0 + min(row0 + C - 1, p.R - 1) / p.G >= p.max_seq;
        const int all_see = past ? 0 : (int)max(min(pos0 + row0 / p.G + 1 - origin, (int64_t)n_keys), (int64_t)0);
        Kv4Acc<D, NT> acc;
        kv4_acc_init(acc);
        if (any) {
            Kv4Rows<D, NT> rows;
            kv4_load_rows<D, NT>(p, b, kvh, row0, pos0, origin, sm.frag[warp], rows);
            int key0 = 0;
            for (int i = 0; i < stages; ++i) {
                if (alive) alive = mbar_wait(&sm.full[warp][slot], parity, &g_status);
                if (alive) {
                    const uint32_t blk = ring0 + slot * NB * L::kBytes;
                    if (key0 + NB * kKvBlock > all_see || !kv4_block<D, NT, NB, false>(blk, key0, n_keys, ln, rows, acc)) {
                        for (int n = 0; n < NB; ++n)
                            if (key0 + n * kKvBlock < n_keys)
                                kv4_block<D, NT, 1, true>(blk + n * L::kBytes, key0 + n * kKvBlock, n_keys, ln, rows, acc);
                    }
                    __syncwarp();
                    if (asked < stages) issue(slot);
                }
                key0 += NB * kKvBlock;
                if (++slot == DEPTH) slot = 0, parity ^= 1;
            }
        }
        const bool more = con.left > 0;
        if (more) {                     // the next unit's first stages come in while this one's rows are written
            con.next(p);
            if (alive) start();
        }
        if (any) {
            const bool merge = sm.merge[warp][0] != 0;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float l[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    l[i] = acc.l[nt][i];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
                }
                float mt[2][NG];
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) mt[i][j] = __shfl_sync(0xffffffffu, acc.mt[nt][i], 4 * j + t);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int c = 8 * nt + 2 * t + i, r = row0 + c;
                    if (r >= p.R) continue;
                    if (merge) {
                        float *sums = reinterpret_cast<float *>(sm.ring[warp][0]) + c * D + 4 * g;
#pragma unroll
                        for (int j = 0; j < NG; ++j)
                            *reinterpret_cast<float4 *>(sums + 32 * j) = kv4_sums(acc, nt, i, j, mt[i][j], 1.f);
                        if (g == 0) sm.ml[warp][c] = make_float2(acc.M[nt][i], l[i]);
                        continue;
                    }
                    const bool whole = began && ends;
                    const float f = !whole ? 1.f : l[i] != 0.f ? 1.f / l[i] : 0.f;
                    const int tok = r / p.G, hh = r - tok * p.G;
                    uint16_t *dst = p.out + ((b * p.T + tok) * p.H + kvh * p.G + hh) * D + 4 * g;
                    const int64_t slot_at = (share * 2 + (began ? 1 : 0)) * C + c;
#pragma unroll
                    for (int j = 0; j < NG; ++j) {
                        // a result that is 0 of nothing seen is 0, not what an empty sum left
                        const float4 o = kv4_sums(acc, nt, i, j, mt[i][j], f);
                        if (whole)
                            *reinterpret_cast<uint2 *>(dst + 32 * j) =
                                make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
                        else
                            *reinterpret_cast<float4 *>(p.part_o + slot_at * D + 32 * j + 4 * g) = o;
                    }
                    if (!whole && g == 0) p.part_ml[slot_at] = make_float2(acc.M[nt][i], l[i]);
                }
            }
        }
        if (!more) break;
        __syncwarp();
    }
    if (const int n = sm.merge[warp][0]; n) {                       // into the first warp's part; the others' are empty
        asm volatile("bar.sync 1, %0;" :: "r"(n * 32) : "memory");
        const int64_t to = (int64_t)sm.merge[warp][1] * C;
        const int row0 = con.tile * C;
        for (int i = threadIdx.x; i < C * (D / 4); i += n * 32) {
            const int c = i / (D / 4), ch = i % (D / 4) * 4;
            if (row0 + c >= p.R) break;
            float top = kNoMax;
            for (int w = 0; w < n; ++w) top = fmaxf(top, sm.ml[w][c].x);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            float l = 0.f;
#pragma unroll 4
            for (int w = 0; w < n; ++w) {
                const float f = ex2(sm.ml[w][c].x - top);
                const float4 y = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(sm.ring[w][0]) + c * D + ch);
                l += sm.ml[w][c].y * f;
                o = make_float4(fmaf(y.x, f, o.x), fmaf(y.y, f, o.y), fmaf(y.z, f, o.z), fmaf(y.w, f, o.w));
            }
            *reinterpret_cast<float4 *>(p.part_o + (to + c) * D + ch) = o;
            if (ch == 0) p.part_ml[to + c] = make_float2(top, l);
        }
        if (warp > 0 && lane < C) p.part_ml[share * 2 * C + lane] = make_float2(kNoMax, 0.f);
    }
    if (!alive)                         // a copy that was late: every slot's bounded once more before the memory goes
        for (int i = 0; i < DEPTH; ++i) mbar_wait(&sm.full[warp][(slot + i) % DEPTH], parity ^ (slot + i >= DEPTH), &g_status);
}

// N numbers, or zeros; loads that are written one after the other are issued so.
template <int N>
__device__ __forceinline__ void load_if(const float *src, bool take, float (&v)[N]) {
    if constexpr (N == 4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\t"
                     "mov.b32 %3, 0;\n\t@p ld.global.v4.f32 {%0, %1, %2, %3}, [%4];\n\t}"
                     : "=&f"(v[0]), "=&f"(v[1]), "=&f"(v[2]), "=&f"(v[3]) : "l"(src), "r"((uint32_t)take) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\t"
                     "@p ld.global.v2.f32 {%0, %1}, [%2];\n\t}"
                     : "=&f"(v[0]), "=&f"(v[1]) : "l"(src), "r"((uint32_t)take) : "memory");
}

// Units of which several warps had a part, joined in order, and rows of
// sequences that hold nothing.  WPR warps per row: a row of few units has many
// parts, rows of many units have few.
template <int D, int NT, int WPR>
__global__ void __launch_bounds__(WPR > 8 ? WPR * 32 : 256) kv4_join_kernel(const __grid_constant__ Kv4AttendParams p) {
    constexpr int V = D / 32, C = 8 * NT, W = WPR > 8 ? WPR : 8;
    __shared__ float s_acc[WPR > 1 ? W : 1][D];
    __shared__ float s_l[WPR > 1 ? W : 1];
    griddep_launch_dependents();
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WPR;
    const int64_t row = (int64_t)blockIdx.x * (W / WPR) + warp / WPR;       // (b * KV + kvh) * R + r
    const bool live = row < (int64_t)p.B * p.KV * p.R;
    const int64_t item = live ? quot(row, p.R) : 0;
    const int r = live ? (int)(row - item * p.R) : 0;
    const int64_t b = quot(item, p.KV);
    const int kvh = (int)(item - b * p.KV), tile = r / C;
    const int64_t pos0 = p.pos0[b * p.pos_stride];
    const int2 held = p.held[item * p.tiles + tile];                // not written for a sequence that holds nothing
    const int64_t nb = kv4_blocks_of(p, pos0);
    const int tok = r / p.G, hh = r - tok * p.G;
    if (live && sub == 0 && lane == 0 && pos0 + tok >= p.max_seq) atomicOr(&g_status, kErrBadIndex);
    float acc[V], l = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    const bool parts = live && nb > 0 && held.x != held.y, write = live && (nb == 0 || parts);
    if (parts) {
        const int c0 = held.x, c1 = held.y;
        const auto slot = [&](int c) { return ((int64_t)c * 2 + (c == c0 ? 1 : 0)) * C + (r - tile * C); };
        float top = kNoMax;
        for (int base = c0; base <= c1; base += 128) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = base + 32 * i + lane;
                x[i] = c <= c1 ? p.part_ml[slot(c)].x : kNoMax;
            }
            top = fmaxf(fmaxf(fmaxf(top, x[0]), fmaxf(x[1], x[2])), x[3]);
        }
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // several parts' loads at a time whatever their number (one after the other they are most of the time), in short
        // code: it is never in the instruction cache
        constexpr int N = WPR == 32 ? 8 : 4;
        constexpr int64_t kStep = (int64_t)WPR * 2 * C;
        for (int base = c0 + sub; base <= c1; base += N * WPR) {
            const int64_t at = (int64_t)base * 2 * C + (r - tile * C);          // slot 0; the first part lies in slot 1
            const int64_t at0 = at + (base == c0 ? C : 0);
            float x[N][2], y[N][V];
#pragma unroll
            for (int i = 0; i < N; ++i) load_if<2>(reinterpret_cast<const float *>(p.part_ml + (i ? at : at0) + kStep * i), base + WPR * i <= c1, x[i]);
#pragma unroll
            for (int i = 0; i < N; ++i)                             // (M and l of 0: no such part, or nothing was written there)
                load_if<V>(p.part_o + ((i ? at : at0) + kStep * i) * D + lane * V, x[i][1] != 0.f || (x[i][0] != 0.f && x[i][0] != kNoMax), y[i]);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float f = ex2(fminf(x[i][0] - top, 0.f));     // (above the maximum only where there is no part)
                l += x[i][1] * f;
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] = fmaf(y[i][k], f, acc[k]);
            }
        }
    }
    if constexpr (WPR > 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) s_acc[warp][lane * V + i] = acc[i];
        if (lane == 0) s_l[warp] = l;
        __syncthreads();
        if (sub) return;
#pragma unroll 4
        for (int w = 1; w < WPR; ++w) {
            l += s_l[warp + w];
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += s_acc[warp + w][lane * V + i];
        }
    }
    if (!write) return;
    const float inv = l != 0.f ? 1.f / l : 0.f;
    uint16_t *dst = p.out + ((b * p.T + tok) * p.H + kvh * p.G + hh) * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; i += 2)
        *reinterpret_cast<uint32_t *>(dst + i) = pack_bf16x2(acc[i] * inv, acc[i + 1] * inv);
}

// Rows per kv head up to which the kernel of this file takes a call; above, the
// prompt kernel.  8B heads (4 per kv head): 8 tokens (32 rows) of 4 sequences of
// 8192 positions take 39 us here and 55 us there, 12 tokens (48 rows) of one
// sequence 22 and 27 us, 16 tokens (64 rows) of 4 sequences 66 and 55 us.
constexpr int64_t kFewRows = 48;

// Column tiles of 8 rows that one warp takes, and the grid.
static int attend_tiles(int64_t R) { return R > 8 ? 2 : 1; }
constexpr int kAttendGrid = 148;
static int attend_warps(int nt, int64_t D) {
    return kAttendGrid * (D == 64   ? nt == 1 ? AttendCfg<64, 1>::kWarps : AttendCfg<64, 2>::kWarps
                          : nt == 1 ? AttendCfg<128, 1>::kWarps
                                    : AttendCfg<128, 2>::kWarps);
}

template <int D, int NT>
static int attend_launch(const Kv4AttendParams &p, cudaStream_t st) {
    const int64_t rows = (int64_t)p.B * p.KV * p.R, units = (int64_t)p.B * p.KV * p.tiles;
    const int rc = launch_kv4<kv4_attend_kernel<D, NT>>(dim3(kAttendGrid), AttendCfg<D, NT>::kWarps * 32,
                                                        sizeof(AttendSmem<D, NT>), st, "kv4_attend_kernel", p);
    if (rc != BF16X_OK) return rc;
    // a row has up to p.warps / units parts; 32 warps for each of few rows (384 rows of 24 units: 26 us in all, 19 with 8)
    if (p.few_units && rows <= 2 * 148)
        return launch_kv4<kv4_join_kernel<D, NT, 32>>(dim3((unsigned)rows), 1024, 0, st, "kv4_join_kernel", p);
    if (units * 8 <= p.warps || p.few_units)
        return launch_kv4<kv4_join_kernel<D, NT, 8>>(dim3((unsigned)rows), 256, 0, st, "kv4_join_kernel", p);
    return launch_kv4<kv4_join_kernel<D, NT, 1>>(dim3((unsigned)((rows + 7) / 8)), 256, 0, st, "kv4_join_kernel", p);
}

static int check_shape(const char *what, int64_t B, int64_t T, int64_t KV, int64_t D, int64_t max_seq) {
    if (B < 0 || T < 0 || KV <= 0 || max_seq <= 0) return set_error(BF16X_ERR_INVALID, "%s: bad shape", what);
    if (D != 64 && D != 128) return set_error(BF16X_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", what);
    if (B > 65535 || KV > 4096 || T > (1 << 24) || max_seq > ((int64_t)1 << 30) || B * KV > 65535)
        return set_error(BF16X_ERR_UNSUPPORTED, "%s: at most 65535 heads in the batch and 2^30 positions", what);
    return BF16X_OK;
}

}  // namespace bf16x

using namespace bf16x;

extern "C" int64_t bf16x_kv4_block_bytes(int64_t head_dim) { return head_dim == 64 || head_dim == 128 ? 20 * head_dim : 0; }

extern "C" int bf16x_kv4_append(const uint16_t *qkv, int64_t ld_b, int64_t ld_t, int64_t B, int64_t T, int64_t H,
                                int64_t KV, int64_t D, const int64_t *pos0, int pos_stride, const float *cos_t,
                                const float *sin_t, uint16_t *q_out, uint8_t *blocks, int64_t max_seq, void *stream) {
    const int rc = check_shape("bf16x_kv4_append", B, T, KV, D, max_seq);
    if (rc != BF16X_OK) return rc;
    if (H < 0 || H > 65536) return set_error(BF16X_ERR_INVALID, "bf16x_kv4_append: bad number of heads");
    if (B == 0 || T == 0) return BF16X_OK;
    if (!qkv || !pos0 || !blocks || (H && !q_out) || (!cos_t != !sin_t))
        return set_error(BF16X_ERR_INVALID, "bf16x_kv4_append: null pointer");
    if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)blocks | (uintptr_t)cos_t | (uintptr_t)sin_t) & 15 ||
        (ld_b | ld_t) % 8)
        return set_error(BF16X_ERR_INVALID, "bf16x_kv4_append: pointers must be 16-byte aligned, strides multiples of 8");
    Kv4AppendParams p = {qkv, ld_b, ld_t, (int)T, (int)H, (int)KV, pos_stride, pos0, cos_t, sin_t, q_out, blocks,
                         max_seq, (max_seq + kKvBlock - 1) / kKvBlock};
    if (B * T > 0x7fffffffLL) return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_kv4_append: too many tokens");
    const dim3 grid((unsigned)(B * T));
    return D == 64 ? launch_kv4<kv4_append_kernel<64>>(grid, 256, 0, (cudaStream_t)stream,
                                "kv4_append_kernel", p)
                   : launch_kv4<kv4_append_kernel<128>>(grid, 256, 0, (cudaStream_t)stream,
                                "kv4_append_kernel", p);
}

extern "C" int bf16x_kv4_read(const uint8_t *blocks, int64_t max_seq, int64_t B, int64_t T, int64_t KV, int64_t D,
                              const int64_t *pos0, int pos_stride, uint16_t *k_out, uint16_t *v_out, void *stream) {
    const int rc = check_shape("bf16x_kv4_read", B, T, KV, D, max_seq);
    if (rc != BF16X_OK) return rc;
    if (B == 0 || T == 0) return BF16X_OK;
    if (!blocks || !pos0 || !k_out || !v_out) return set_error(BF16X_ERR_INVALID, "bf16x_kv4_read: null pointer");
    if (((uintptr_t)blocks | (uintptr_t)k_out | (uintptr_t)v_out) & 15)
        return set_error(BF16X_ERR_INVALID, "bf16x_kv4_read: pointers must be 16-byte aligned");
    Kv4ReadParams p = {blocks, max_seq, (max_seq + kKvBlock - 1) / kKvBlock, (int)T, (int)KV, pos_stride, pos0,
                       k_out, v_out};
    if (B * T > 0x7fffffffLL) return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_kv4_read: too many tokens");
    const dim3 grid((unsigned)(B * ((T + kReadTokens - 1) / kReadTokens)), (unsigned)((2 * KV * (D / 8) + 255) / 256));
    return D == 64 ? launch_kv4<kv4_read_kernel<64>>(grid, 256, 0, (cudaStream_t)stream,
                                "kv4_read_kernel", p)
                   : launch_kv4<kv4_read_kernel<128>>(grid, 256, 0, (cudaStream_t)stream,
                                "kv4_read_kernel", p);
}

extern "C" int64_t bf16x_kv4_attend_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t KV, int64_t D,
                                                    int64_t max_seq) {
    if (B <= 0 || T <= 0 || H <= 0 || KV <= 0 || H % KV || max_seq <= 0) return 0;
    if (T * (H / KV) > kFewRows) return kv4_prefill_workspace(B, KV, T * (H / KV), T, D, max_seq);
    const int nt = attend_tiles(T * (H / KV));
    const int64_t units = B * KV * ((T * (H / KV) + 8 * nt - 1) / (8 * nt));
    return (int64_t)attend_warps(nt, D) * 2 * 8 * nt * (D * 4 + 8) + units * 8;
}

extern "C" int bf16x_kv4_attend(const uint16_t *q, int64_t ldq_b, int64_t ldq_t, int64_t ldq_h, int64_t B, int64_t T,
                                int64_t H, int64_t KV, int64_t D, const int64_t *pos0, int pos_stride, float scale,
                                const uint8_t *blocks, int64_t max_seq, uint16_t *out, void *workspace,
                                int64_t workspace_bytes, void *stream) {
    const int rc = check_shape("bf16x_kv4_attend", B, T, KV, D, max_seq);
    if (rc != BF16X_OK) return rc;
    if (H <= 0 || H % KV || H > 65536)
        return set_error(BF16X_ERR_INVALID, "bf16x_kv4_attend: heads must be a multiple of kv_heads");
    if (B == 0 || T == 0) return BF16X_OK;
    if (!q || !pos0 || !blocks || !out) return set_error(BF16X_ERR_INVALID, "bf16x_kv4_attend: null pointer");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)blocks | (uintptr_t)workspace) & 15 ||
        (ldq_b | ldq_t | ldq_h) % 8)
        return set_error(BF16X_ERR_INVALID, "bf16x_kv4_attend: pointers must be 16-byte aligned, strides multiples of 8");
    const int64_t need = bf16x_kv4_attend_workspace_bytes(B, T, H, KV, D, max_seq);
    if (need && (!workspace || workspace_bytes < need))
        return set_error(BF16X_ERR_INVALID, "bf16x_kv4_attend: workspace too small (%lld bytes needed)", (long long)need);
    const int64_t G = H / KV, R = T * G, nblk = (max_seq + kKvBlock - 1) / kKvBlock;
    if (R > 0x7fffff00LL || B * KV * R > ((int64_t)1 << 32)) return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_kv4_attend: too many query rows");
    const int nt = attend_tiles(R);
    Kv4AttendParams p = {};
    p.q = q, p.ldq_b = ldq_b, p.ldq_t = ldq_t, p.ldq_h = ldq_h;
    p.B = (int)B, p.T = (int)T, p.H = (int)H, p.KV = (int)KV, p.G = (int)G, p.R = (int)R;
    p.tiles = (int)((R + 8 * nt - 1) / (8 * nt)), p.warps = attend_warps(nt, D);
    p.few_units = B * KV * p.tiles * 64 <= p.warps;
    p.pos_stride = pos_stride, p.pos0 = pos0, p.scale_log2 = scale * 1.44269504088896340736f;
    p.blocks = blocks, p.max_seq = max_seq, p.nblk = nblk, p.out = out;
    if (R > kFewRows) return kv4_prefill(p, D, workspace, (cudaStream_t)stream);
    p.part_o = (float *)workspace;
    p.part_ml = (float2 *)((uint8_t *)workspace + (int64_t)p.warps * 2 * 8 * nt * D * 4);
    p.held = (int2 *)(p.part_ml + (int64_t)p.warps * 2 * 8 * nt);
    cudaStream_t st = (cudaStream_t)stream;
    if (D == 64) return nt == 1 ? attend_launch<64, 1>(p, st) : attend_launch<64, 2>(p, st);
    return nt == 1 ? attend_launch<128, 1>(p, st) : attend_launch<128, 2>(p, st);
}
