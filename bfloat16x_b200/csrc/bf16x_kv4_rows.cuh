// bf16x_kv4_rows.cuh -- one warp's attention of 8 or 16 query rows over blocks of
// the 4-bit cache in shared memory, by mma.sync: all of the work for few rows
// (bf16x_kv4.cu), and what the prompt kernel's fp16 tiles cannot hold
// (bf16x_kv4_prefill.cu).
#pragma once

#include "bf16x_kv4.cuh"

namespace bf16x {

// Rows r = t * G + h of one kv head's G query heads and T tokens, 8 per mma
// column tile.  Per block of 16 positions a warp computes
//   S^T [16 positions][8 rows] = K Q^T,  P = 2^(S' - M),  O^T [D][8 rows] += V^T P^T
// with the codes as operands: per 32-channel group j
//   S  += dK_j (codes Q_j) + mK_j sum(Q_j),   O_j += codes (P dV_j),  O_j += mV_j P.
// Q, each row scaled by a power of two, is exact in fp16 (but for channels below
// 2^-26 of the row's largest, which are off by 2^-34 of that at most); P dV is
// rounded to fp16.  The minima go through one more mma each (bf16, exact on the m side, the
// other side split into three or two bf16 parts).  (fp8 operands for the K codes
// would halve their mma's, but sm_100a's mma.sync widens e4m3 to fp16 first.)
// P dV has to fit fp16 whatever the scale of V, so the running reference M of
// a row is that of the maximum of S' + log2(max_j dV_j), not of S' alone, and is
// raised only when a term exceeds it by too much (kRescale).  A group of channels
// whose scale is 2^-8 of its position's largest or less would lose bits of P dV_j,
// in the end all of them, to fp16's subnormals: blocks that hold such a position
// take each group's products apart, P dV_j scaled by a power of two of the row
// and group, and add them in fp32 (kv4_add_apart).  Looking for it costs 1 % of a
// call whose groups are alike.
template <int D, int NT>
struct Kv4Rows {
    static constexpr int NG = D / 32;
    uint32_t q;                         // shared address of this lane's B fragments [NT][NG][32 lanes] x 16 bytes:
                                        // pairs (0,4) (1,5)/16 (2,6) (3,7)/16 of each 8 channels
    uint32_t qm[NT][2];                 // B fragment of the minima's mma: sums of Q per group, split in bf16 parts
    float c1[NT][2];                    // turns the sums of columns 2t, 2t+1 into log2 units
    int last[NT][2];                    // last position that columns 2t, 2t+1 see, from the origin of the walk
};

// The rows of a tile: lane (g, t) takes channels 8 t .. 8 t + 7 of every group of row g.
template <int D, int NT>
__device__ __forceinline__ void kv4_load_rows(const Kv4AttendParams &p, int64_t b, int kvh, int row0, int64_t pos0,
                                              int64_t origin, uint4 (*frag)[D / 32][32], Kv4Rows<D, NT> &rows) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    rows.q = smem_u32(&frag[0][0][lane]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = row0 + 8 * nt + g;
        const bool have = r < p.R;
        const int tok = have ? r / p.G : 0, hh = have ? r - tok * p.G : 0;
        const uint16_t *src = p.q + b * p.ldq_b + (int64_t)tok * p.ldq_t + (int64_t)(kvh * p.G + hh) * p.ldq_h;
        uint4 raw[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j)
            raw[j] = have ? *reinterpret_cast<const uint4 *>(src + 32 * j + 8 * t) : make_uint4(0, 0, 0, 0);
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(bf_lo(w[i])), fabsf(bf_hi(w[i]))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the row scaled by 2^e to a largest value in [2^13, 2^14): bf16 values are then exact in fp16
        const int ex = (int)(__float_as_uint(top) >> 23) - 127;
        const int e = top > 0.f && ex < 128 ? min(max(13 - ex, -100), 110) : 0;
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        float part[3][NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
            float x[8], s = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = bf_lo(w[i]) * up;
                x[2 * i + 1] = bf_hi(w[i]) * up;
                s += x[2 * i] + x[2 * i + 1];
            }
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            frag[nt][j][lane] =
                make_uint4(pack_f16x2(x[0], x[4]), pack_f16x2(x[1] * 0.0625f, x[5] * 0.0625f), pack_f16x2(x[2], x[6]),
                           pack_f16x2(x[3] * 0.0625f, x[7] * 0.0625f));
            // the group sums, in the units of the codes' sums, in three bf16 parts (24 bits):
            // k index 4 part + j (NG = 4) or 2 part + j (NG = 2)
            float rest = s * 0x1p-24f;
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
        // negative: sees nothing (padding, past the cache, no row)
        const int64_t at = have ? pos0 + tok : -1;
        const int last = at < 0 || at >= p.max_seq ? -0x40000000 : (int)max(at - origin, (int64_t)-0x40000000);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            rows.c1[nt][i] = __shfl_sync(0xffffffffu, c1, 4 * (2 * t + i));
            rows.last[nt][i] = __shfl_sync(0xffffffffu, last, 4 * (2 * t + i));
        }
    }
    __syncwarp();
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

// Channels 32 j + 4 g .. + 3 of column 2t + i, times f; mt: the minima's part.
template <int D, int NT>
__device__ __forceinline__ float4 kv4_sums(const Kv4Acc<D, NT> &a, int nt, int i, int j, float mt, float f) {
    return make_float4(fmaf(a.o[nt][2 * j][i], 0x1p24f, mt) * f, fmaf(a.o[nt][2 * j][2 + i], 0x1p20f, mt) * f,
                       fmaf(a.o[nt][2 * j + 1][i], 0x1p24f, mt) * f, fmaf(a.o[nt][2 * j + 1][2 + i], 0x1p20f, mt) * f);
}

template <int NG>
__device__ __forceinline__ void kv4_expand(uint32_t at, float (&d)[NG]) {           // NG bf16 values
    if constexpr (NG == 4) {
        const uint2 w = lds64(at);
        d[0] = bf_lo(w.x);
        d[1] = bf_hi(w.x);
        d[2] = bf_lo(w.y);
        d[3] = bf_hi(w.y);
    } else {
        const uint32_t w = lds32(at);
        d[0] = bf_lo(w);
        d[1] = bf_hi(w);
    }
}

template <int NG>
__device__ __forceinline__ void kv4_words(uint32_t at, uint32_t (&w)[NG]) {         // NG words of codes
    if constexpr (NG == 4) {
        const uint4 v = lds128(at);
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
    } else {
        const uint2 v = lds64(at);
        w[0] = v.x;
        w[1] = v.y;
    }
}

// log2 of a position's largest V scale for the reference: not below -92, so
// that P <= 2^107 and its sums stay finite.
__device__ __forceinline__ float kv4_ref_exp(float d) { return fmaxf(lg2(d), -92.f); }
constexpr int kSpreadBits = 8 << 23;    // ratio of a position's V scales above which its groups are taken apart, as fp32 bits

// One group's products with x = P dV_j (positions g, g + 8; columns 2t, 2t+1),
// scaled so that each column's largest is in [2^14, 2^15).
__device__ __forceinline__ void kv4_add_apart(float (&o0)[4], float (&o1)[4], uint32_t w0, uint32_t w1, float (&x)[4]) {
    float back[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float top = fmaxf(x[i], x[2 + i]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 15);
        const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
        x[i] *= up;
        x[2 + i] *= up;
        back[i] = __uint_as_float((uint32_t)(127 - 14 + ex) << 23);
    }
    const uint32_t b0 = movmatrix(pack_f16x2(x[0], x[1])), b1 = movmatrix(pack_f16x2(x[2], x[3]));
    const uint32_t h0 = w0 >> 8, h1 = w1 >> 8;
    float c[4];
    mma_f16(c, w0 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x000F000Fu, w1 & 0x00F000F0u, b0, b1, 0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) o0[k] = fmaf(c[k], back[k & 1], o0[k]);
    mma_f16(c, h0 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x000F000Fu, h1 & 0x00F000F0u, b0, b1, 0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) o1[k] = fmaf(c[k], back[k & 1], o1[k]);
}

// Where this lane's parts of a block lie.
template <int D>
struct Kv4Lane {
    uint32_t codes, row, kmin, vmin;    // byte offsets
    int g, t;
    __device__ __forceinline__ Kv4Lane() {
        constexpr int NG = D / 32;
        const int lane = threadIdx.x & 31;
        g = lane >> 2, t = lane & 3;
        codes = lane * NG * 4;
        row = 16 * D + g * NG * 2;
        kmin = 17 * D + g * NG * 2 + (NG == 4 ? (t & 1) * 4 : 0);
        vmin = 19 * D + (t * NG + min(g, NG - 1)) * 4;
        // kept in registers, not worked out again for every block
        asm volatile("" : "+r"(codes), "+r"(row), "+r"(kmin), "+r"(vmin));
    }
};

// The weights P = 2^(S' - M) of kv4_block, and what they add to the sums; APART:
// each group's products by themselves.
template <int D, int NT, int NB, bool MASK, bool APART>
__device__ __forceinline__ void kv4_products(uint32_t blk, int key0, int n_keys, const Kv4Lane<D> &ln, const float (&s)[NB][NT][4],
                                             const float (&v)[NB][2][D / 32], const float (&unit)[NT][2], Kv4Acc<D, NT> &acc) {
    using L = KvLayout<D>;
    constexpr int NG = L::NG;
    constexpr float kInf = __builtin_huge_valf();
    const int t = ln.t;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const uint32_t at = blk + n * L::kBytes;
        uint32_t w0[NG], w1[NG];
        kv4_words<NG>(at + ln.codes + L::kV, w0);
        kv4_words<NG>(at + ln.codes + L::kV + 32 * NG * 4, w1);
        // rows g >= NG of this mma are not used: they may hold any finite numbers (the last group's minima)
        uint32_t vm0 = lds32(at + ln.vmin), vm1 = lds32(at + ln.vmin + 16 * NG);
        if (MASK) {
            const int a = key0 + 16 * n + 2 * t, c = a + 8;
            vm0 = a + 1 < n_keys ? vm0 : a < n_keys ? vm0 & 0xFFFFu : 0u;
            vm1 = c + 1 < n_keys ? vm1 : c < n_keys ? vm1 & 0xFFFFu : 0u;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float pr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pr[i] = ex2(fmaf(s[n][nt][i], unit[nt][i & 1], -acc.M[nt][i & 1]));
            acc.l[nt][0] += pr[0] + pr[2];
            acc.l[nt][1] += pr[1] + pr[3];
            const uint32_t a = pack_bf16x2(pr[0], pr[1]), c = pack_bf16x2(pr[2], pr[3]);
            const uint32_t al = pack_bf16x2(pr[0] - bf_lo(a), pr[1] - bf_hi(a)),
                           cl = pack_bf16x2(pr[2] - bf_lo(c), pr[3] - bf_hi(c));
            mma_bf16(acc.mt[nt], vm0, vm0, vm1, vm1, movmatrix(a), movmatrix(c));
            mma_bf16(acc.mt[nt], vm0, vm0, vm1, vm1, movmatrix(al), movmatrix(cl));
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                float x[4] = {pr[0] * v[n][0][j], pr[1] * v[n][0][j], pr[2] * v[n][1][j], pr[3] * v[n][1][j]};
                if (MASK) {                                         // 0 * NaN: a masked position stays out of its row
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = s[n][nt][i] == -kInf ? 0.f : x[i];
                }
                if constexpr (APART) {
                    kv4_add_apart(acc.o[nt][2 * j], acc.o[nt][2 * j + 1], w0[j], w1[j], x);
                } else {
                    const uint32_t b0 = movmatrix(pack_f16x2(x[0], x[1])), b1 = movmatrix(pack_f16x2(x[2], x[3]));
                    const uint32_t h0 = w0[j] >> 8, h1 = w1[j] >> 8;
                    mma_f16(acc.o[nt][2 * j], w0[j] & 0x000F000Fu, w0[j] & 0x00F000F0u, w1[j] & 0x000F000Fu,
                            w1[j] & 0x00F000F0u, b0, b1);
                    mma_f16(acc.o[nt][2 * j + 1], h0 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x000F000Fu,
                            h1 & 0x00F000F0u, b0, b1);
                }
            }
        }
    }
}

// NB consecutive blocks at shared address `blk`, the first position of the
// first at key0 (relative to the tile's first row, like rows.last).  MASK: some
// row of the tile does not see all of them; positions from n_keys on are not
// read as numbers.  Without MASK, blocks whose groups need to be taken apart are
// left undone (false): short code is what most of them need.
template <int D, int NT, int NB, bool MASK>
__device__ __forceinline__ bool kv4_block(uint32_t blk, int key0, int n_keys, const Kv4Lane<D> &ln,
                                          const Kv4Rows<D, NT> &rows, Kv4Acc<D, NT> &acc) {
    using L = KvLayout<D>;
    constexpr int NG = L::NG;
    constexpr float kInf = __builtin_huge_valf();
    const int g = ln.g, t = ln.t;
    float s[NB][NT][4];
    bool ok[NB][2];
    // ---- scores
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const uint32_t at = blk + n * L::kBytes;
        ok[n][0] = !MASK || key0 + 16 * n + g < n_keys;
        ok[n][1] = !MASK || key0 + 16 * n + g + 8 < n_keys;
        uint32_t k0[NG], k1[NG];
        float d0[NG], d1[NG];
        kv4_words<NG>(at + ln.codes, k0);
        kv4_words<NG>(at + ln.codes + 32 * NG * 4, k1);
        kv4_expand<NG>(at + ln.row, d0);
        kv4_expand<NG>(at + ln.row + 8 * NG * 2, d1);
        uint32_t m0 = lds32(at + ln.kmin), m1 = lds32(at + ln.kmin + 8 * NG * 2);
        if (MASK) {
            m0 = ok[n][0] ? m0 : 0u;
            m1 = ok[n][1] ? m1 : 0u;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            mma_bf16(s[n][nt], m0, m1, m0, m1, rows.qm[nt][0], rows.qm[nt][1], 0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const uint32_t h0 = k0[j] >> 8, h1 = k1[j] >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float c[4];
                const uint4 q = lds128(rows.q + (nt * NG + j) * 512);
                mma_f16(c, k0[j] & 0x000F000Fu, k1[j] & 0x000F000Fu, k0[j] & 0x00F000F0u, k1[j] & 0x00F000F0u, q.x,
                        q.y, 0.f, 0.f, 0.f, 0.f);
                mma_f16(c, h0 & 0x000F000Fu, h1 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x00F000F0u, q.z, q.w);
                s[n][nt][0] = fmaf(d0[j], c[0], s[n][nt][0]);
                s[n][nt][1] = fmaf(d0[j], c[1], s[n][nt][1]);
                s[n][nt][2] = fmaf(d1[j], c[2], s[n][nt][2]);
                s[n][nt][3] = fmaf(d1[j], c[3], s[n][nt][3]);
            }
        }
    }
    // ---- V's scales, and the reference of each row
    float v[NB][2][NG], e[NB][2];
    int spread = 0;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            kv4_expand<NG>(blk + n * L::kBytes + ln.row + 2 * D + i * 8 * NG * 2, v[n][i]);
            if (MASK) {
#pragma unroll
                for (int j = 0; j < NG; ++j) v[n][i][j] = ok[n][i] ? v[n][i][j] : 0.f;
            }
            float lo = fminf(v[n][i][0], v[n][i][1]);
            e[n][i] = fmaxf(v[n][i][0], v[n][i][1]);
            if constexpr (NG == 4) {
                lo = min3(lo, v[n][i][2], v[n][i][3]);
                e[n][i] = max3(e[n][i], v[n][i][2], v[n][i][3]);
            }
            spread = max(spread, __float_as_int(e[n][i]) - __float_as_int(lo));
            e[n][i] = kv4_ref_exp(e[n][i]);
        }
    const bool apart = spread > kSpreadBits;
    bool raise = false;
    float top[NT][2], unit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (MASK) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[n][nt][i] *= rows.c1[nt][i & 1];
                    if (key0 + 16 * n + g + (i & 2 ? 8 : 0) > rows.last[nt][i & 1]) s[n][nt][i] = -kInf;
                }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            unit[nt][i] = MASK ? 1.f : rows.c1[nt][i];
            top[nt][i] = fmaxf(fmaf(s[0][nt][i], unit[nt][i], e[0][0]), fmaf(s[0][nt][2 + i], unit[nt][i], e[0][1]));
            if constexpr (NB == 2)
                top[nt][i] = fmaxf(top[nt][i], fmaxf(fmaf(s[NB - 1][nt][i], unit[nt][i], e[NB - 1][0]),
                                                     fmaf(s[NB - 1][nt][2 + i], unit[nt][i], e[NB - 1][1])));
            raise |= top[nt][i] > acc.M[nt][i] + kRescale;
        }
    }
    bool any_apart = false;
    if (__any_sync(0xffffffffu, raise || apart)) {                  // (one vote for two rare cases)
        any_apart = __any_sync(0xffffffffu, apart);
        if (!MASK && any_apart) return false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float a[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = top[nt][i];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                x = fmaxf(x - kRefTerm, acc.M[nt][i]);
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
    if constexpr (MASK) {
        if (any_apart) {
            kv4_products<D, NT, NB, MASK, true>(blk, key0, n_keys, ln, s, v, unit, acc);
            return true;
        }
    }
    kv4_products<D, NT, NB, MASK, false>(blk, key0, n_keys, ln, s, v, unit, acc);
    return true;
}

}  // namespace bf16x
