// bf16x_kv4.cu -- writing the 4-bit key/value cache, reading it back, and
// attention of few query rows over it (decode steps, a few guessed tokens).
#include <algorithm>

#include <cuda_runtime.h>

#include "bf16x_kv4.cuh"

namespace bf16x {

// --------------------------------------------------------------------- write
// y = the head's channel pairs (2i, 2i+1) turned by the angle of the position
// (q and k), rounded to bf16; then for every 32 channels of k and v
//   m = min y,  d = (max y - m) / 15 rounded up to bf16,  code = rint((y - m) / d).
// d is rounded up so that no code exceeds 15, and m is a bf16 value already.
// A group that holds an infinity or a NaN gets d = NaN, m = 0: it reads as NaN
// and m stays finite, so a masked position cannot reach another row's sums.
// Every operation is rounded by itself (no fused multiply-add), so the codes
// do not depend on how the compiler contracts.
//
// D/8 lanes per (token, head), 8 channels each: a 16-byte load, and the whole
// K word of a lane.  Bound by memory traffic for prompts, by latency for steps.
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
    } else if (d > 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = rintf(__fdiv_rn(__fsub_rn(y[i], lo), d));
            codes |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * i);
        }
    }
}

struct Kv4AppendParams {
    const uint16_t *qkv;
    int64_t ld_b, ld_t;                 // elements
    int64_t tokens;
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
    const int heads = p.H + 2 * p.KV;
    const int64_t unit_raw = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPH;
    const int64_t n_units = p.tokens * heads;
    const bool live = unit_raw < n_units;                           // the warp stays whole for the shuffles
    const int64_t unit = live ? unit_raw : n_units - 1;
    const int l = threadIdx.x % LPH;
    const int64_t tok = unit / heads;
    const int head = (int)(unit - tok * heads);
    const int64_t b = tok / p.T;
    const int t = (int)(tok - b * p.T);
    const int64_t pos = p.pos0[b * p.pos_stride] + t;
    const bool inside = pos >= 0 && pos < p.max_seq;
    if (live && pos >= p.max_seq && head == 0 && l == 0) atomicOr(&g_status, kErrBadIndex);
    const uint4 raw = *reinterpret_cast<const uint4 *>(p.qkv + b * p.ld_b + t * p.ld_t + (int64_t)head * D + 8 * l);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[2 * i] = bf_lo(w[i]);
        y[2 * i + 1] = bf_hi(w[i]);
    }
    if (head < p.H + p.KV && p.cos_t != nullptr && inside) {
        const float4 c4 = *reinterpret_cast<const float4 *>(p.cos_t + pos * (D / 2) + 4 * l);
        const float4 s4 = *reinterpret_cast<const float4 *>(p.sin_t + pos * (D / 2) + 4 * l);
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = __fsub_rn(__fmul_rn(y[2 * i], c[i]), __fmul_rn(y[2 * i + 1], s[i]));
            const float e = __fadd_rn(__fmul_rn(y[2 * i], s[i]), __fmul_rn(y[2 * i + 1], c[i]));
            const uint32_t r = pack_bf16x2(a, e);
            y[2 * i] = bf_lo(r);
            y[2 * i + 1] = bf_hi(r);
        }
    }
    float d, m;
    uint32_t codes;
    kv4_quantize8<D>(y, d, m, codes);                               // shuffles: every lane takes part
    if (!live) return;
    if (head < p.H) {
        uint4 o = make_uint4(0, 0, 0, 0);                           // a position outside the cache: zeros
        if (inside)
            o = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                           pack_bf16x2(y[6], y[7]));
        *reinterpret_cast<uint4 *>(p.q_out + (tok * p.H + head) * D + 8 * l) = o;
        return;
    }
    if (!inside) return;
    const bool is_v = head >= p.H + p.KV;
    const int kvh = head - p.H - (is_v ? p.KV : 0);
    uint8_t *blk = p.blocks + ((b * p.KV + kvh) * p.nblk + pos / kKvBlock) * L::kBytes;
    const int r = (int)(pos % kKvBlock), grp = l / 4, t4 = l % 4;
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
            const int g = 2 * t4 + i;                               // channels 32 grp + 4 g ..
            *reinterpret_cast<uint16_t *>(blk + L::kV + (((pp * 8 + g) * 4 + tt) * L::NG + grp) * 4 + 2 * h) =
                (uint16_t)(codes >> (16 * i));
        }
        if (t4 == 0) {
            *reinterpret_cast<uint16_t *>(blk + L::kVd + (r * L::NG + grp) * 2) = db;
            *reinterpret_cast<uint16_t *>(blk + L::kVm + (((r / 2) * L::NG + grp) * 2 + h) * 2) = mb;
        }
    }
}

// ---------------------------------------------------------------------- read
// The values that positions *pos0 .. *pos0 + T - 1 stand for, d * code + m in
// fp32 rounded to bf16; a position outside the cache reads as zeros.
struct Kv4ReadParams {
    const uint8_t *blocks;
    int64_t max_seq, nblk, tokens;
    int T, KV, pos_stride;
    const int64_t *pos0;
    uint16_t *k_out, *v_out;
};

template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p) {
    using L = KvLayout<D>;
    constexpr int LPH = D / 8;
    griddep_launch_dependents();
    griddep_wait();
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPH;
    const int l = threadIdx.x % LPH;
    if (unit >= p.tokens * p.KV * 2) return;
    const int64_t row = unit >> 1;                                  // token * KV + head
    const bool is_v = unit & 1;
    const int64_t tok = row / p.KV;
    const int kvh = (int)(row - tok * p.KV);
    const int64_t b = tok / p.T;
    const int64_t pos = p.pos0[b * p.pos_stride] + (tok - b * p.T);
    uint4 o = make_uint4(0, 0, 0, 0);
    if (pos >= p.max_seq && l == 0) atomicOr(&g_status, kErrBadIndex);
    if (pos >= 0 && pos < p.max_seq) {
        const uint8_t *blk = p.blocks + ((b * p.KV + kvh) * p.nblk + pos / kKvBlock) * L::kBytes;
        const int r = (int)(pos % kKvBlock), grp = l / 4, t4 = l % 4;
        uint32_t codes;
        uint16_t db, mb;
        if (!is_v) {
            codes = *reinterpret_cast<const uint32_t *>(blk + ((r * 4 + t4) * L::NG + grp) * 4);
            db = *reinterpret_cast<const uint16_t *>(blk + L::kKd + (r * L::NG + grp) * 2);
            mb = *reinterpret_cast<const uint16_t *>(blk + L::kKm + (r * L::NG + grp) * 2);
        } else {
            const int pp = r / 8, tt = (r % 8) / 2, h = r % 2;
            codes = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                codes |= (uint32_t)*reinterpret_cast<const uint16_t *>(
                             blk + L::kV + (((pp * 8 + 2 * t4 + i) * 4 + tt) * L::NG + grp) * 4 + 2 * h) << (16 * i);
            db = *reinterpret_cast<const uint16_t *>(blk + L::kVd + (r * L::NG + grp) * 2);
            mb = *reinterpret_cast<const uint16_t *>(blk + L::kVm + (((r / 2) * L::NG + grp) * 2 + h) * 2);
        }
        const float d = bf16_bits_to_f32(db), m = bf16_bits_to_f32(mb);
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __fadd_rn(__fmul_rn(d, (float)((codes >> (4 * i)) & 15u)), m);
        o = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                       pack_bf16x2(y[6], y[7]));
    }
    *reinterpret_cast<uint4 *>((is_v ? p.v_out : p.k_out) + row * D + 8 * l) = o;
}

// -------------------------------------------------------------------- attend
// Rows r = t * G + h of one kv head's G query heads and T tokens, 8 per mma
// column tile.  Per block of 16 positions a warp computes
//   S^T [16 positions][8 rows] = K Q^T,  P = 2^(S' - M),  O^T [D][8 rows] += V^T P^T
// with the codes as fp16 operands: per 32-channel group j
//   S  += dK_j (codes Q_j) + mK_j sum(Q_j),   O_j += codes (P dV_j),  O_j += mV_j P.
// The minima go through one more mma each (bf16, exact on the m side, the
// other side split into two or three bf16 parts).
// P dV has to fit fp16 whatever the scale of V, so the running reference M of
// a row is the maximum of S' + log2(max_j dV_j), not of S' alone; it is
// raised only when a term exceeds it by more than 2^8.
struct Kv4AttendParams {
    const uint16_t *q;
    int64_t ldq_b, ldq_t, ldq_h;
    int B, T, H, KV, G, R;
    int pos_stride, nsplit;
    const int64_t *pos0;
    float scale_log2;                   // softmax scale * log2(e)
    const uint8_t *blocks;
    int64_t max_seq, nblk;
    uint16_t *out;
    float *part_o;                      // [item][row][split][D]
    float2 *part_ml;                    // [item][row][split]
};

constexpr float kRescale = 8.f;         // log2 of how far a term may exceed the reference
constexpr float kNoMax = -3.0e38f;

template <int D, int NT>
struct Kv4Rows {
    static constexpr int NG = D / 32;
    uint32_t qb[NT][NG][4];             // B fragments: pairs (0,4) (1,5)/16 (2,6) (3,7)/16 of each 8 channels
    uint32_t qm[NT][2];                 // B fragment of the minima's mma: sums of Q per group, split in bf16 parts
    float c1[NT][2];                    // turns the sums of columns 2t, 2t+1 into log2 units
    int64_t last[NT][2];                // last position that columns 2t, 2t+1 see, -1: none
};

// This lane's row of the tile (row g of each column tile): its pointer, or null.
template <int D, int NT>
__device__ __forceinline__ void kv4_load_rows(const Kv4AttendParams &p, int64_t b, int kvh, int row0, int64_t pos0,
                                              Kv4Rows<D, NT> &rows) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = row0 + 8 * nt + g;
        const bool have = r < p.R;
        const int tok = have ? r / p.G : 0, hh = have ? r - tok * p.G : 0;
        const uint16_t *src = p.q + b * p.ldq_b + (int64_t)tok * p.ldq_t + (int64_t)(kvh * p.G + hh) * p.ldq_h;
        float x[NG][8];
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            uint4 raw = make_uint4(0, 0, 0, 0);
            if (have) raw = *reinterpret_cast<const uint4 *>(src + 32 * j + 8 * t);
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[j][2 * i] = bf_lo(w[i]);
                x[j][2 * i + 1] = bf_hi(w[i]);
                top = fmaxf(top, fmaxf(fabsf(x[j][2 * i]), fabsf(x[j][2 * i + 1])));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the row scaled by 2^e to a largest value in [2^13, 2^14): bf16 values are then exact in fp16
        const int ex = (int)(__float_as_uint(top) >> 23) - 127;
        const int e = top > 0.f && ex < 128 ? min(max(13 - ex, -110), 110) : 0;
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        float sum[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[j][i] *= up;
                s += x[j][i];
            }
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            sum[j] = s * 0x1p-24f;                                  // in the units of the codes' sums
            rows.qb[nt][j][0] = pack_f16x2(x[j][0], x[j][4]);
            rows.qb[nt][j][1] = pack_f16x2(x[j][1] * 0.0625f, x[j][5] * 0.0625f);
            rows.qb[nt][j][2] = pack_f16x2(x[j][2], x[j][6]);
            rows.qb[nt][j][3] = pack_f16x2(x[j][3] * 0.0625f, x[j][7] * 0.0625f);
        }
        // the group sums in three bf16 parts (24 bits): k index 4 part + j (NG = 4) or 2 part + j (NG = 2)
        float part[3][NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            float rest = sum[j];
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                part[i][j] = bf_lo(pack_bf16x2(rest, 0.f) & 0xFFFFu);
                rest -= part[i][j];
            }
        }
        if constexpr (NG == 4) {
            const uint32_t a[3][2] = {{pack_bf16x2(part[0][0], part[0][1]), pack_bf16x2(part[0][2], part[0][3])},
                                      {pack_bf16x2(part[1][0], part[1][1]), pack_bf16x2(part[1][2], part[1][3])},
                                      {pack_bf16x2(part[2][0], part[2][1]), pack_bf16x2(part[2][2], part[2][3])}};
            rows.qm[nt][0] = t == 0 ? a[0][0] : t == 1 ? a[0][1] : t == 2 ? a[1][0] : a[1][1];
            rows.qm[nt][1] = t == 0 ? a[2][0] : t == 1 ? a[2][1] : 0u;
        } else {
            const uint32_t a[3] = {pack_bf16x2(part[0][0], part[0][1]), pack_bf16x2(part[1][0], part[1][1]),
                                   pack_bf16x2(part[2][0], part[2][1])};
            rows.qm[nt][0] = t == 0 ? a[0] : t == 1 ? a[1] : t == 2 ? a[2] : 0u;
            rows.qm[nt][1] = 0u;
        }
        const float c1 = p.scale_log2 * __uint_as_float((uint32_t)(127 + 24 - e) << 23);
        int64_t last = have ? pos0 + tok : -1;
        if (last >= p.max_seq) last = -1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            rows.c1[nt][i] = __shfl_sync(0xffffffffu, c1, 4 * (2 * t + i));
            rows.last[nt][i] = __shfl_sync(0xffffffffu, last, 4 * (2 * t + i));
        }
    }
}

template <int D, int NT>
struct Kv4Acc {
    float o[NT][D / 16][4];             // O^T: [2 j + i]: channels 32 j + 4 g + 2 i (c0, c1) and + 1 (c2, c3, times 16)
    float mt[NT][4];                    // sums of mV P: group g (g < NG), columns 2t, 2t+1 (c0, c1)
    float l[NT][2], M[NT][2];
};

template <int D, int NT>
__device__ __forceinline__ void kv4_acc_init(Kv4Acc<D, NT> &a) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) a.o[nt][i][k] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) a.mt[nt][k] = 0.f;
        a.l[nt][0] = a.l[nt][1] = 0.f;
        a.M[nt][0] = a.M[nt][1] = kNoMax;
    }
}

template <int NG>
__device__ __forceinline__ void kv4_expand(const uint8_t *at, float (&d)[NG]) {     // NG bf16 values
    if constexpr (NG == 4) {
        const uint2 w = *reinterpret_cast<const uint2 *>(at);
        d[0] = bf_lo(w.x);
        d[1] = bf_hi(w.x);
        d[2] = bf_lo(w.y);
        d[3] = bf_hi(w.y);
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(at);
        d[0] = bf_lo(w);
        d[1] = bf_hi(w);
    }
}

template <int NG>
__device__ __forceinline__ void kv4_words(const uint8_t *at, uint32_t (&w)[NG]) {   // NG words of codes
    if constexpr (NG == 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(at);
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2 *>(at);
        w[0] = v.x;
        w[1] = v.y;
    }
}

// log2 of a position's largest V scale for the reference: not below -100, so
// that P <= 2^108 and its sums stay finite; a position whose groups are all
// constant has no code part, and -20 keeps m P finite too (where d is not 0, m
// is at most 2^12 d: the values are bf16).
__device__ __forceinline__ float kv4_ref_exp(float d) { return d > 0.f ? fmaxf(lg2(d), -100.f) : -20.f; }

// One block at `blk`, whose first position is key0.  MASK: some row of the
// tile does not see all of it; positions from n_keys on are not read as numbers.
template <int D, int NT, bool MASK>
__device__ __forceinline__ void kv4_block(const uint8_t *blk, int64_t key0, int64_t n_keys, const Kv4Rows<D, NT> &rows,
                                          Kv4Acc<D, NT> &acc) {
    using L = KvLayout<D>;
    constexpr int NG = L::NG;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const bool ok0 = !MASK || key0 + g < n_keys, ok1 = !MASK || key0 + g + 8 < n_keys;
    // ---- scores
    uint32_t k0[NG], k1[NG];
    float d0[NG], d1[NG];
    kv4_words<NG>(blk + (g * 4 + t) * NG * 4, k0);
    kv4_words<NG>(blk + ((g + 8) * 4 + t) * NG * 4, k1);
    kv4_expand<NG>(blk + L::kKd + g * NG * 2, d0);
    kv4_expand<NG>(blk + L::kKd + (g + 8) * NG * 2, d1);
    const int tm = NG == 4 ? (t & 1) * 4 : 0;
    uint32_t m0 = *reinterpret_cast<const uint32_t *>(blk + L::kKm + g * NG * 2 + tm);
    uint32_t m1 = *reinterpret_cast<const uint32_t *>(blk + L::kKm + (g + 8) * NG * 2 + tm);
    if (MASK) {
        m0 = ok0 ? m0 : 0u;
        m1 = ok1 ? m1 : 0u;
    }
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
        mma_bf16(s[nt], m0, m1, m0, m1, rows.qm[nt][0], rows.qm[nt][1]);
    }
#pragma unroll
    for (int j = 0; j < NG; ++j) {
        const uint32_t h0 = k0[j] >> 8, h1 = k1[j] >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            mma_f16(c, k0[j] & 0x000F000Fu, k1[j] & 0x000F000Fu, k0[j] & 0x00F000F0u, k1[j] & 0x00F000F0u,
                    rows.qb[nt][j][0], rows.qb[nt][j][1]);
            mma_f16(c, h0 & 0x000F000Fu, h1 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x00F000F0u, rows.qb[nt][j][2],
                    rows.qb[nt][j][3]);
            s[nt][0] = fmaf(d0[j], c[0], s[nt][0]);
            s[nt][1] = fmaf(d0[j], c[1], s[nt][1]);
            s[nt][2] = fmaf(d1[j], c[2], s[nt][2]);
            s[nt][3] = fmaf(d1[j], c[3], s[nt][3]);
        }
    }
    // ---- V's scales, and the reference of each row
    float v0[NG], v1[NG];
    kv4_expand<NG>(blk + L::kVd + g * NG * 2, v0);
    kv4_expand<NG>(blk + L::kVd + (g + 8) * NG * 2, v1);
    if (MASK) {
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            v0[j] = ok0 ? v0[j] : 0.f;
            v1[j] = ok1 ? v1[j] : 0.f;
        }
    }
    float e0 = fmaxf(v0[0], v0[1]), e1 = fmaxf(v1[0], v1[1]);
    if constexpr (NG == 4) {
        e0 = fmaxf(e0, fmaxf(v0[2], v0[3]));
        e1 = fmaxf(e1, fmaxf(v1[2], v1[3]));
    }
    e0 = kv4_ref_exp(e0);
    e1 = kv4_ref_exp(e1);
    bool raise = false;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[nt][i] *= rows.c1[nt][i & 1];
            if (MASK) {
                const int64_t key = key0 + g + (i & 2 ? 8 : 0);
                if (key > rows.last[nt][i & 1]) s[nt][i] = -__int_as_float(0x7f800000);
            }
        }
        top[nt][0] = fmaxf(s[nt][0] + e0, s[nt][2] + e1);
        top[nt][1] = fmaxf(s[nt][1] + e0, s[nt][3] + e1);
        raise |= top[nt][0] > acc.M[nt][0] + kRescale || top[nt][1] > acc.M[nt][1] + kRescale;
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float a[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = top[nt][i];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                x = fmaxf(x, acc.M[nt][i]);
                a[i] = ex2(acc.M[nt][i] - x);
                acc.M[nt][i] = x;
                acc.l[nt][i] *= a[i];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                acc.mt[nt][k] *= a[k & 1];
#pragma unroll
                for (int i = 0; i < D / 16; ++i) acc.o[nt][i][k] *= a[k & 1];
            }
        }
    }
    // ---- P, and O
    uint32_t w0[NG], w1[NG];
    kv4_words<NG>(blk + L::kV + (g * 4 + t) * NG * 4, w0);
    kv4_words<NG>(blk + L::kV + ((8 + g) * 4 + t) * NG * 4, w1);
    uint32_t vm0 = 0, vm1 = 0;
    if (g < NG) {
        vm0 = *reinterpret_cast<const uint32_t *>(blk + L::kVm + (t * NG + g) * 4);
        vm1 = *reinterpret_cast<const uint32_t *>(blk + L::kVm + ((4 + t) * NG + g) * 4);
        if (MASK) {
            const int64_t a = key0 + 2 * t, c = a + 8;
            vm0 = a + 1 < n_keys ? vm0 : a < n_keys ? vm0 & 0xFFFFu : 0u;
            vm1 = c + 1 < n_keys ? vm1 : c < n_keys ? vm1 & 0xFFFFu : 0u;
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = ex2(s[nt][i] - acc.M[nt][i & 1]);
        acc.l[nt][0] += pr[0] + pr[2];
        acc.l[nt][1] += pr[1] + pr[3];
        {
            const uint32_t a = pack_bf16x2(pr[0], pr[1]), c = pack_bf16x2(pr[2], pr[3]);
            mma_bf16(acc.mt[nt], vm0, 0u, vm1, 0u, movmatrix(a), movmatrix(c));
            const uint32_t al = pack_bf16x2(pr[0] - bf_lo(a), pr[1] - bf_hi(a)),
                           cl = pack_bf16x2(pr[2] - bf_lo(c), pr[3] - bf_hi(c));
            mma_bf16(acc.mt[nt], vm0, 0u, vm1, 0u, movmatrix(al), movmatrix(cl));
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            float x[4] = {pr[0] * v0[j], pr[1] * v0[j], pr[2] * v1[j], pr[3] * v1[j]};
            if (MASK) {                                             // 0 * NaN: a masked position stays out of its row
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = s[nt][i] == -__int_as_float(0x7f800000) ? 0.f : x[i];
            }
            const uint32_t b0 = movmatrix(pack_f16x2(x[0], x[1])), b1 = movmatrix(pack_f16x2(x[2], x[3]));
            const uint32_t h0 = w0[j] >> 8, h1 = w1[j] >> 8;
            mma_f16(acc.o[nt][2 * j], w0[j] & 0x000F000Fu, w0[j] & 0x00F000F0u, w1[j] & 0x000F000Fu,
                    w1[j] & 0x00F000F0u, b0, b1);
            mma_f16(acc.o[nt][2 * j + 1], h0 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x000F000Fu, h1 & 0x00F000F0u, b0,
                    b1);
        }
    }
}

constexpr int kAttendWarps = 8;

template <int D, int NT>
struct AttendSmem {
    float o[kAttendWarps][8 * NT][D + 4];
    float M[kAttendWarps][8 * NT], l[kAttendWarps][8 * NT];
};

template <int D, int NT>
__global__ void __launch_bounds__(kAttendWarps * 32) kv4_attend_kernel(const Kv4AttendParams p) {
    using L = KvLayout<D>;
    constexpr int NG = L::NG, W = kAttendWarps, C = 8 * NT;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    AttendSmem<D, NT> &sm = *reinterpret_cast<AttendSmem<D, NT> *>(smem_raw);
    griddep_launch_dependents();
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, row0 = blockIdx.y * C;
    const int64_t item = blockIdx.z;
    const int64_t b = item / p.KV;
    const int kvh = (int)(item - b * p.KV);
    const int64_t pos0 = p.pos0[b * p.pos_stride];
    // positions that some row of the tile sees: rows are ordered by token
    const int tok_last = min(row0 + C - 1, p.R - 1) / p.G;
    int64_t n_keys = pos0 + tok_last + 1;
    if (n_keys > p.max_seq) {                                       // tokens past the cache's end see nothing
        if (threadIdx.x == 0) atomicOr(&g_status, kErrBadIndex);
        n_keys = p.max_seq;
    }
    n_keys = max(n_keys, (int64_t)0);
    const int64_t first_last = pos0 + row0 / p.G;                   // last position that the tile's first row sees
    const int64_t nb = (n_keys + kKvBlock - 1) / kKvBlock;
    const int64_t b0 = nb * split / p.nsplit, b1 = nb * (split + 1) / p.nsplit;
    Kv4Rows<D, NT> rows;
    kv4_load_rows<D, NT>(p, b, kvh, row0, pos0, rows);
    Kv4Acc<D, NT> acc;
    kv4_acc_init(acc);
    const uint8_t *base = p.blocks + (b * p.KV + kvh) * p.nblk * L::kBytes;
    for (int64_t i = b0 + warp; i < b1; i += W) {
        const int64_t key0 = i * kKvBlock;
        if (key0 + kKvBlock - 1 <= first_last && key0 + kKvBlock <= n_keys)
            kv4_block<D, NT, false>(base + i * L::kBytes, key0, n_keys, rows, acc);
        else
            kv4_block<D, NT, true>(base + i * L::kBytes, key0, n_keys, rows, acc);
    }
    // ---- the warps' sums joined: each scaled to the largest reference
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float l = acc.l[nt][i];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (g == 0) {
                sm.M[warp][8 * nt + 2 * t + i] = acc.M[nt][i];
                sm.l[warp][8 * nt + 2 * t + i] = l;
            }
        }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float top = kNoMax;
            for (int w = 0; w < W; ++w) top = fmaxf(top, sm.M[w][8 * nt + 2 * t + i]);
            f[i] = ex2(acc.M[nt][i] - top);
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const float mt0 = __shfl_sync(0xffffffffu, acc.mt[nt][0], 4 * j + t),
                        mt1 = __shfl_sync(0xffffffffu, acc.mt[nt][1], 4 * j + t);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float(&o)[4] = acc.o[nt][2 * j + i];
                const int ch = 32 * j + 4 * g + 2 * i, c = 8 * nt + 2 * t;
                *reinterpret_cast<float2 *>(&sm.o[warp][c][ch]) =
                    make_float2((o[0] * 0x1p24f + mt0) * f[0], (o[2] * 0x1p20f + mt0) * f[0]);
                *reinterpret_cast<float2 *>(&sm.o[warp][c + 1][ch]) =
                    make_float2((o[1] * 0x1p24f + mt1) * f[1], (o[3] * 0x1p20f + mt1) * f[1]);
            }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < C * (D / 2); e += W * 32) {
        const int c = e / (D / 2), ch = 2 * (e - c * (D / 2)), r = row0 + c;
        if (r >= p.R) continue;
        float top = kNoMax, l = 0.f;
        for (int w = 0; w < W; ++w) top = fmaxf(top, sm.M[w][c]);
        float2 o = make_float2(0.f, 0.f);
        for (int w = 0; w < W; ++w) {
            l += sm.l[w][c] * ex2(sm.M[w][c] - top);
            const float2 a = *reinterpret_cast<const float2 *>(&sm.o[w][c][ch]);
            o.x += a.x;
            o.y += a.y;
        }
        if (p.nsplit == 1) {
            const float inv = l != 0.f ? 1.f / l : 0.f;
            const int tok = r / p.G, hh = r - tok * p.G;
            *reinterpret_cast<uint32_t *>(p.out + ((b * p.T + tok) * p.H + kvh * p.G + hh) * D + ch) =
                pack_bf16x2(o.x * inv, o.y * inv);
        } else {
            const int64_t at = (item * p.R + r) * p.nsplit + split;
            *reinterpret_cast<float2 *>(p.part_o + at * D + ch) = o;
            if (ch == 0) p.part_ml[at] = make_float2(top, l);
        }
    }
}

// One warp per row: the splits' sums joined in order.
template <int D>
__global__ void __launch_bounds__(128) kv4_join_kernel(const Kv4AttendParams p) {
    constexpr int V = D / 32;
    griddep_launch_dependents();
    griddep_wait();
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);      // item * R + r
    const int lane = threadIdx.x & 31;
    if (row >= (int64_t)p.B * p.KV * p.R) return;
    const float2 *ml = p.part_ml + row * p.nsplit;
    float top = kNoMax;
    for (int s = lane; s < p.nsplit; s += 32) top = fmaxf(top, ml[s].x);
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float l = 0.f, acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int s = 0; s < p.nsplit; ++s) {
        const float2 x = ml[s];
        const float f = ex2(x.x - top);
        l += x.y * f;
        const float *src = p.part_o + (row * p.nsplit + s) * D + lane * V;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(src[i], f, acc[i]);
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const int64_t item = row / p.R;
    const int r = (int)(row - item * p.R), tok = r / p.G, hh = r - tok * p.G;
    const int64_t b = item / p.KV;
    const int kvh = (int)(item - b * p.KV);
    uint16_t *dst = p.out + ((b * p.T + tok) * p.H + kvh * p.G + hh) * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; i += 2)
        *reinterpret_cast<uint32_t *>(dst + i) = pack_bf16x2(acc[i] * inv, acc[i + 1] * inv);
}

template <typename P>
static int launch_kv4(void (*kern)(P), dim3 grid, unsigned block, size_t smem, cudaStream_t st, const char *what,
                      const P &params) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return set_error(BF16X_ERR_CUDA, "%s: shared memory: %s", what, cudaGetErrorString(e));
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, params);
    if (e != cudaSuccess) return set_error(BF16X_ERR_CUDA, "%s: launch: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

// Column tiles of 8 rows that one CTA takes, and the splits of the positions.
static int attend_tiles(int64_t R) { return R > 16 ? 4 : R > 8 ? 2 : 1; }
static int attend_splits(int64_t items, int64_t row_tiles, int64_t nblk) {
    const int64_t want = (2 * 148 + items * row_tiles - 1) / (items * row_tiles);
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, nblk / kAttendWarps), 148));
}

template <int D, int NT>
static int attend_launch(const Kv4AttendParams &p, int64_t row_tiles, cudaStream_t st) {
    const int64_t items = (int64_t)p.B * p.KV;
    int rc = launch_kv4(kv4_attend_kernel<D, NT>, dim3((unsigned)p.nsplit, (unsigned)row_tiles, (unsigned)items),
                        kAttendWarps * 32, sizeof(AttendSmem<D, NT>), st, "kv4_attend_kernel", p);
    if (rc != BF16X_OK || p.nsplit == 1) return rc;
    return launch_kv4(kv4_join_kernel<D>, dim3((unsigned)((items * p.R + 3) / 4)), 128, 0, st, "kv4_join_kernel", p);
}

static int check_shape(const char *what, int64_t B, int64_t T, int64_t KV, int64_t D, int64_t max_seq) {
    if (B < 0 || T < 0 || KV <= 0 || max_seq <= 0) return set_error(BF16X_ERR_INVALID, "%s: bad shape", what);
    if (D != 64 && D != 128) return set_error(BF16X_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", what);
    if (B > 65535 || KV > 4096 || T > (1 << 24) || max_seq > ((int64_t)1 << 40) || B * KV > 65535)
        return set_error(BF16X_ERR_UNSUPPORTED, "%s: batch * kv_heads must be at most 65535", what);
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
    Kv4AppendParams p = {qkv, ld_b, ld_t, B * T, (int)T, (int)H, (int)KV, pos_stride, pos0, cos_t, sin_t, q_out, blocks,
                         max_seq, (max_seq + kKvBlock - 1) / kKvBlock};
    const int64_t threads = B * T * (H + 2 * KV) * (D / 8), grid = (threads + 255) / 256;
    if (grid > 0x7fffffffLL) return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_kv4_append: too many tokens");
    return D == 64 ? launch_kv4(kv4_append_kernel<64>, dim3((unsigned)grid), 256, 0, (cudaStream_t)stream,
                                "kv4_append_kernel", p)
                   : launch_kv4(kv4_append_kernel<128>, dim3((unsigned)grid), 256, 0, (cudaStream_t)stream,
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
    Kv4ReadParams p = {blocks, max_seq, (max_seq + kKvBlock - 1) / kKvBlock, B * T, (int)T, (int)KV, pos_stride, pos0,
                       k_out, v_out};
    const int64_t threads = B * T * 2 * KV * (D / 8), grid = (threads + 255) / 256;
    if (grid > 0x7fffffffLL) return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_kv4_read: too many tokens");
    return D == 64 ? launch_kv4(kv4_read_kernel<64>, dim3((unsigned)grid), 256, 0, (cudaStream_t)stream,
                                "kv4_read_kernel", p)
                   : launch_kv4(kv4_read_kernel<128>, dim3((unsigned)grid), 256, 0, (cudaStream_t)stream,
                                "kv4_read_kernel", p);
}

extern "C" int64_t bf16x_kv4_attend_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t KV, int64_t D,
                                                    int64_t max_seq) {
    if (B <= 0 || T <= 0 || H <= 0 || KV <= 0 || H % KV || max_seq <= 0) return 0;
    const int64_t R = T * (H / KV), C = 8 * attend_tiles(R), items = B * KV;
    const int n = attend_splits(items, (R + C - 1) / C, (max_seq + kKvBlock - 1) / kKvBlock);
    return n == 1 ? 0 : items * R * n * (D * 4 + 8);
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
    const int64_t G = H / KV, R = T * G, nblk = (max_seq + kKvBlock - 1) / kKvBlock, items = B * KV;
    const int nt = attend_tiles(R);
    const int64_t row_tiles = (R + 8 * nt - 1) / (8 * nt);
    if (row_tiles > 65535) return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_kv4_attend: too many query rows");
    Kv4AttendParams p = {};
    p.q = q, p.ldq_b = ldq_b, p.ldq_t = ldq_t, p.ldq_h = ldq_h;
    p.B = (int)B, p.T = (int)T, p.H = (int)H, p.KV = (int)KV, p.G = (int)G, p.R = (int)R;
    p.pos_stride = pos_stride, p.pos0 = pos0, p.scale_log2 = scale * 1.44269504088896340736f;
    p.blocks = blocks, p.max_seq = max_seq, p.nblk = nblk, p.out = out;
    p.nsplit = attend_splits(items, row_tiles, nblk);
    p.part_o = (float *)workspace;
    p.part_ml = (float2 *)((uint8_t *)workspace + items * R * p.nsplit * D * 4);
    cudaStream_t st = (cudaStream_t)stream;
    if (D == 64)
        return nt == 1 ? attend_launch<64, 1>(p, row_tiles, st)
                       : nt == 2 ? attend_launch<64, 2>(p, row_tiles, st) : attend_launch<64, 4>(p, row_tiles, st);
    return nt == 1 ? attend_launch<128, 1>(p, row_tiles, st)
                   : nt == 2 ? attend_launch<128, 2>(p, row_tiles, st) : attend_launch<128, 4>(p, row_tiles, st);
}
