// bf16x_kv4_prefill.cu -- attention of many query rows over the 4-bit cache
// (prompts, chunks of prompts) on the 5th-generation tensor cores.
//
// Rows r = t * G + h of one kv head, 256 per unit (two groups of 128), walk
// over the cache in tiles of 128 positions:
//   S[128][128] = Q K^T,  P = 2^(S c - M),  O[128][D] += P V
// with S, P and O in tensor memory (all 512 columns at D = 128: P takes the
// place of S) and Q, K and V^T as fp16 operands in shared memory.  13 warps:
//   0..3, 4..7  one softmax group per 128 rows, one thread per row: scores out
//               of tensor memory, maximum, 2^x, P back as fp16
//   8..11       K and V from 4 bits to fp16 (loaded one tile ahead into
//               registers), one thread per position, into two stages each
//   12          issues the MMAs
// While one group works on its scores, the tensor cores work for the other.
// The softmax goes over tensor memory twice in short loops: holding a row's 128
// scores in registers took 700 cycles more per tile, as its straight code does
// not stay in an instruction cache that three roles share; steps of 64 with two
// S per group took a third more, since an MMA of 64 columns takes as long as
// one of 128.  A CTA goes over several units (the longest first), so that the
// next one's K and V are ready when a unit ends.
//
// fp16 operands hold any scale: a row of Q is scaled by a power of two into
// [2^13, 2^14), exact; the values of a tile by 2^-dk (K) and 2^-dv (V) to at
// most 2^-6, so that d * 2^24 fits fp16 and one fused multiply-add per pair
// turns codes (subnormal fp16, see bf16x_kv4.cuh) into values, rounded once (2^-12).
// dk enters the scores' factor.  dv enters the exponent, P' = 2^(S c + dv - M),
// and its inverse the sum l of the P'; M is raised, and O scaled, only when a
// term exceeds it by too much (kRescale).  dk and dv are one number per tile, unless
// its positions differ by more than 2^6 in size, or their groups of channels by
// more than 2^7: then each position has its own (fp16 would lose the small ones),
// which makes the softmax slow (12000 cycles a tile, not 3200).  A group that is 2^-7 of its own
// position's largest or less falls into fp16's subnormals with any dv.  A piece of a
// unit that holds such a position is done once more behind the others, by mma.sync
// on the codes (bf16x_kv4_rows.cuh), which takes any sizes.
//
// A V group that is not finite reads as zeros here, and the rows that see its
// position get NaN in its 32 channels at the end: 0 * NaN would reach the rows
// that do not.
//
// Bound: per tile and 256 rows at D = 128 the MMAs take 2048 cycles and 2^x
// (16 per cycle and SM) takes 2048; a tile takes 5600, the chain of one group:
// scores to weights 3100 (maxima 700, weights 2000), then the product and the
// next scores, 1000 each, half of that the time until an MMA's end is seen.
// (At 64 channels P has columns of its own, so the next scores need not wait
// for the product: 4700.)  A call's start and end take 12 us.  8B heads: a
// prompt of 2048 tokens 62 us, 556 TFLOP/s of the useful half; 512 tokens behind
// 7680 109 us, 610 TFLOP/s.  3 x 511 tokens of 8 heads of 64 channels behind up
// to 7003 positions 46 us, 234 TFLOP/s.
#include <algorithm>

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "bf16x_kv4.cuh"
#include "bf16x_kv4_rows.cuh"
#include "bf16x_umma.cuh"
#include "bf16x_wait.cuh"

namespace bf16x {

constexpr int kPreRows = 256;                         // rows per unit
constexpr int kPreKeys = 128;                         // positions per tile
constexpr int kPreThreads = 13 * 32;
constexpr int kPreCut = 4 * 148;                      // units, up to which they may be cut
constexpr int kPreUnitCost = 2;                       // of a unit's start and end, in tiles
constexpr int kPreRedo = 1024;                        // (of more pieces per CTA some are done again without need)
// log2 of where a row's largest term lies when M is set.  It may grow by 2^8 before M is raised: to raise it costs a wait
// for the product and a pass over O (from 2^11, with 2^4 to go, 2048 tokens of the 8B heads took 66 us instead of 62).
constexpr float kPreTerm = kRescale - 8.f;
constexpr int kPreSpread = 7;                         // log2 of how far groups of channels may differ in size

template <int D>
struct PreSmem {
    static constexpr int NG = D / 32;
    // columns of tensor memory: S of both groups, O of both groups, and P, apart from S if there is room
    static constexpr bool kApart = D == 64;
    static constexpr int kPCol = kApart ? 256 + 2 * D : 0, kPStep = kApart ? 64 : 128;
    static constexpr int kSubK = kPreKeys * 128;      // [128 rows][64 columns] fp16
    static constexpr int kSubV = D * 128;             // [D rows][64 positions] fp16
    static constexpr int kK = 2 * (D / 64) * kSubK;   // offsets: Q of both groups first
    static constexpr int kKStage = (D / 64) * kSubK;
    static constexpr int kV = kK + 2 * kKStage;
    static constexpr int kVStage = 2 * kSubV;
    static constexpr int kScale = kV + 2 * kVStage;   // fp16, two buffers: V's d [NG][128], m [NG][128]
    static constexpr int kScaleBytes = 2 * kPreKeys * NG * 2;
    static constexpr int kMisc = kScale + 2 * kScaleBytes;
    static constexpr int kPlan = kMisc + 7424;        // PrePlan
    static constexpr int kBytes = kPlan + 2560 + 1024;              // alignment slack
};

struct PreMisc {
    uint64_t q_ready[2], k_full[2], k_empty[2], v_full[2], v_empty[2], drain;
    uint64_t s_full[2], p_full[2], pv_done[2];                      // per group
    uint64_t dq[2], m_full[4];                        // the converting warps among themselves; a tile's numbers below
    uint32_t tmem;
    int abort_flag;
    int red[2][4][8];
    int uneven[4];                                    // of tile j at j % 4: 1: each position has its own dk and dv, 2: fp16 is not enough
    float k_fac[4][kPreKeys], v_exp[4][kPreKeys], v_inv[4][kPreKeys];      // 2^dk, dv, 2^-dv; else the first only
    uint32_t any_bad[4];
    uint32_t bad[4][kPreKeys / 4];                    // per position a byte: its V groups that are not finite
    uint32_t redo[kPreRedo / 32], any_redo;           // pieces that fp16 is not enough for: piece n of the CTA at n % kPreRedo
};
static_assert(sizeof(PreMisc) <= 7424, "PreMisc");
struct PrePlan {
    int start[kPreCut + 1];                           // of the units, each nt + kPreUnitCost long
    int sum[kPreThreads / 32];
};
static_assert(sizeof(PrePlan) <= 2560, "PrePlan");

__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(a)
        : "memory");
}
// Loads that are asked for now and waited for together; the waits name the
// registers, so that nothing reads them before.
__device__ __forceinline__ void tmem_ask32(uint32_t a, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_got32(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                   "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23])
                 :
                 : "memory");
    asm volatile("" : "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :: "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t a, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        :: "r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
           "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t a, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 :: "r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// fp16 operands, fp32 sums, M = 128: A and B from shared memory, or A from tensor memory.
template <int N>
__host__ __device__ constexpr uint32_t umma_idesc_f16() {
    return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ bool finite_bits(uint32_t b) { return (b & 0x7F800000u) != 0x7F800000u; }

// A tile that every row of the warp sees whole, with one dk and dv: the maximum
// of a row's scores.
__device__ __forceinline__ float pre_top(uint32_t t_s) {
    float mx[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) mx[q] = -__builtin_huge_valf();
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {
        uint32_t v[2][32];
        tmem_ask32(t_s + 64 * c, v[0]);
        tmem_ask32(t_s + 64 * c + 32, v[1]);
        tmem_got32(v[0]);
        tmem_got32(v[1]);
#pragma unroll
        for (int i = 0; i < 16; i += 2)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                mx[q] = max3(mx[q], __uint_as_float(v[q >> 1][16 * (q & 1) + i]), __uint_as_float(v[q >> 1][16 * (q & 1) + i + 1]));
    }
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

// Its weights P = 2^(S fac + off), as fp16, over S if P has no place of its own
// (a chunk's P lies over scores that were read before); returns their sum.
__device__ __forceinline__ void pre_chunk(const uint32_t (&v)[32], uint32_t t_p, uint64_t f2, uint64_t o2, uint64_t (&sum2)[4]) {
    uint32_t o[16];
#pragma unroll
    for (int h = 0; h < 32; h += 8) {                               // eight at a time: enough to overlap, few registers
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            unpack2(fma2(pack2(__uint_as_float(v[h + i]), __uint_as_float(v[h + i + 1])), f2, o2), x[i], x[i + 1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ex2(x[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum2[i] = add2(sum2[i], pack2(x[2 * i], x[2 * i + 1]));
            o[h / 2 + i] = pack_f16x2(x[2 * i], x[2 * i + 1]);
        }
    }
    tmem_st16(t_p, o);
}
__device__ __forceinline__ float pre_weights(uint32_t t_s, uint32_t t_p, float fac, float off) {
    const uint64_t f2 = pack2(fac, fac), o2 = pack2(off, off);
    uint64_t sum2[4] = {};
    uint32_t a[32], b[32];
    tmem_ask32(t_s, a);
    tmem_got32(a);
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {                                   // the next chunk comes in while one is worked on
        tmem_ask32(t_s + 64 * c + 32, b);
        pre_chunk(a, t_p + 32 * c, f2, o2, sum2);
        tmem_got32(b);
        if (c == 0) tmem_ask32(t_s + 64, a);
        pre_chunk(b, t_p + 32 * c + 16, f2, o2, sum2);
        if (c == 0) tmem_got32(a);
    }
    float x, y;
    unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), x, y);
    return x + y;
}

// The scores that a row does not see become -inf in tensor memory.
__device__ __forceinline__ void pre_mask(uint32_t t_s, int vis) {
#pragma unroll 1
    for (int c = 0; c < kPreKeys; c += 16) {
        if (!__any_sync(0xffffffffu, vis < c + 16)) continue;
        uint32_t v[16];
        tmem_ld16(t_s + c, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = c + i < vis ? v[i] : 0xFF800000u;
        tmem_st16(t_s + c, v);
    }
    tmem_wait_st();
}

// The same for any tile: rows that see only `vis` of its positions, a dk and dv
// for each position.  (Slow: 12000 cycles for a tile, against 3200.)
__device__ __forceinline__ float pre_top_any(uint32_t t_s, const PreMisc &ms, int slot, bool uneven, float c_row, int vis) {
    float mx = -__builtin_huge_valf();
#pragma unroll 1
    for (int c = 0; c < 8; ++c) {
        uint32_t v[16];
        tmem_ld16(t_s + 16 * c, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int k = 16 * c + i, n = uneven ? k : 0;
            const float x = fmaf(__uint_as_float(v[i]), c_row * ms.k_fac[slot][n], ms.v_exp[slot][n]);
            if (k < vis) mx = fmaxf(mx, x);
        }
    }
    return mx;
}
__device__ __forceinline__ float pre_weights_any(uint32_t t_s, uint32_t t_p, const PreMisc &ms, int slot, bool uneven, float c_row,
                                                 float M, int vis) {
    float sum = 0.f;
#pragma unroll 1
    for (int c = 0; c < 8; ++c) {
        uint32_t v[16], o[8];
        tmem_ld16(t_s + 16 * c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float x[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = 16 * c + 2 * i + h, n = uneven ? k : 0;
                x[h] = ex2(fmaf(__uint_as_float(v[2 * i + h]), c_row * ms.k_fac[slot][n], ms.v_exp[slot][n] - M));
                x[h] = k < vis ? x[h] : 0.f;
                sum = fmaf(x[h], ms.v_inv[slot][n], sum);
            }
            o[i] = pack_f16x2(x[0], x[1]);
        }
        tmem_st8(t_p + 8 * c, o);
    }
    return sum;
}

struct PreParams {
    Kv4AttendParams a;
    int items, row_tiles, units;
    int *held;                          // units that may be cut: whether units are cut, then first and last CTA of each
};

// Unit u: 256 rows of one kv head; the row tiles that see most come first.  A
// piece of it: nt tiles of positions from tile t0 on.
struct PreUnit {
    int b, kvh, row0, t0, nt, groups;
    int slot;                           // where the piece's sums go; -1: it is the whole unit
    int64_t pos0, n_keys;               // positions that some row sees
    __device__ __forceinline__ void set(const PreParams &pp, int u) {
        const Kv4AttendParams &p = pp.a;
        const int tile = u / pp.items, item = u - tile * pp.items;
        b = item / p.KV;
        pos0 = p.pos0[(int64_t)b * p.pos_stride];
        kvh = item - b * p.KV;
        row0 = (pp.row_tiles - 1 - tile) * kPreRows;
        n_keys = max(min(pos0 + min(row0 + kPreRows - 1, p.R - 1) / p.G + 1, p.max_seq), (int64_t)0);
        groups = p.R - row0 > 128 ? 2 : 1;
        slot = -1;
        t0 = 0;
        nt = (int)((n_keys + kPreKeys - 1) / kPreKeys);
    }
};

// The pieces of a CTA.  Whole units: CTA c of n takes units c, 2 n - 1 - c,
// 2 n + c, ..., so that one of the longest goes with one of the shortest.  Or
// all units in a row, cut into equal shares, one per CTA.
struct PreWalk {
    int share;                          // 0: whole units
    int i;
    const int *start;
    __device__ __forceinline__ PreWalk(const PreParams &pp, const PrePlan &plan, int share_) : share(share_), i(0), start(plan.start) {
        if (share) {                    // the last unit that starts at or before the share
            int hi = pp.units;
            while (hi - i > 1) {
                const int mid = (i + hi) >> 1;
                if (start[mid] <= (int)blockIdx.x * share) i = mid;
                else hi = mid;
            }
        }
    }
    __device__ __forceinline__ bool next(const PreParams &pp, PreUnit &un) {
        if (!share) {
            const int n = (int)gridDim.x, c = (int)blockIdx.x, u = i & 1 ? (i + 1) * n - 1 - c : i * n + c;
            if (u >= pp.units) return false;
            ++i;
            un.set(pp, u);
            return true;
        }
        for (; i < pp.units && start[i] < ((int)blockIdx.x + 1) * share; ++i) {
            const int a = (int)blockIdx.x * share - start[i], all = start[i + 1] - start[i] - kPreUnitCost;
            const int lo = max(a - kPreUnitCost, 0), hi = min(a + share - kPreUnitCost, all);
            if (hi <= lo && (all > 0 || a > 0)) continue;           // (a unit without tiles is zeros, from where it starts)
            un.set(pp, i++);
            un.t0 = lo;
            un.nt = max(hi - lo, 0);
            if (un.nt < all) un.slot = 2 * (int)blockIdx.x + (lo == 0);
            return true;
        }
        return false;
    }
};

// How the units go over the CTAs: 0 for whole units, else a CTA's share.  Units
// are cut when that ends earlier by more than what it costs to write the sums
// of the pieces and to join them.
__device__ __forceinline__ int pre_plan(const PreParams &pp, PrePlan &plan) {
    constexpr int kJoinCost = 2;
    const int tid = threadIdx.x, lane = tid & 31, n = (int)gridDim.x;
    int before = 0;
    for (int u0 = 0; u0 < pp.units; u0 += kPreThreads) {            // running sum of the units' costs
        int cost = 0;
        if (u0 + tid < pp.units) {
            PreUnit un;
            un.set(pp, u0 + tid);
            cost = un.nt + kPreUnitCost;
        }
        int x = cost;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) plan.sum[tid >> 5] = x;
        __syncthreads();
        int all = before;
        for (int w = 0; w < kPreThreads / 32; ++w) {
            if (w < tid >> 5) x += plan.sum[w];
            all += plan.sum[w];
        }
        if (u0 + tid < pp.units) plan.start[u0 + tid] = before + x - cost;
        before = all;
        __syncthreads();
    }
    if (tid == 0) plan.start[pp.units] = before;
    __syncthreads();
    const int share = max((before + n - 1) / n, 2 * kPreUnitCost);
    int load = 0;
    if (tid < n)
        for (int i = 0, u = tid; u < pp.units; ++i, u = i & 1 ? (i + 1) * n - 1 - tid : i * n + tid)
            load += plan.start[u + 1] - plan.start[u];
    const bool cut = __syncthreads_or(load > share + kJoinCost);
    if (blockIdx.x == 0) {
        for (int u = tid; u < pp.units; u += kPreThreads) {
            const int first = plan.start[u] + kPreUnitCost, last = max(plan.start[u + 1] - 1, first);
            reinterpret_cast<int2 *>(pp.held)[1 + u] = make_int2(first / share, last / share);
        }
        if (tid == 0) pp.held[0] = cut;
    }
    return cut ? share : 0;
}

// A piece once more, by mma.sync: its rows eight at a time, one warp each, over
// rings of blocks where Q, K and V were.  (A function of its own: within the kernel
// its registers made the tiles' loops spill.)  2048 tokens of the 8B heads take 470
// us if all of their pieces need it for their keys, 680 for their values, 61
// without; looking for such positions costs 1 %.
template <int D>
struct PreRing {
    static constexpr int kDepth = 3;
    uint8_t block[kDepth][KvLayout<D>::kBytes];
    uint4 frag[1][D / 32][32];
};
template <int D>
__device__ __noinline__ void pre_redo(const Kv4AttendParams &p, const PreUnit &un, PreRing<D> &ring) {
    using L = KvLayout<D>;
    constexpr int NG = L::NG, DEPTH = PreRing<D>::kDepth;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t origin = (int64_t)un.t0 * kPreKeys;
    const uint8_t *src = p.blocks + (((int64_t)un.b * p.KV + un.kvh) * p.nblk + (int64_t)un.t0 * (kPreKeys / kKvBlock)) * L::kBytes;
    const Kv4Lane<D> ln;
    for (int row0 = un.row0 + 8 * warp; row0 < min(un.row0 + kPreRows, p.R); row0 += 8 * (kPreThreads / 32)) {
        Kv4Rows<D, 1> rows;
        kv4_load_rows<D, 1>(p, un.b, un.kvh, row0, un.pos0, origin, ring.frag, rows);
        Kv4Acc<D, 1> acc;
        kv4_acc_init(acc);
        const int64_t lim = min(un.pos0 + min(row0 + 7, p.R - 1) / p.G + 1, p.max_seq) - origin;
        const int n_keys = (int)max(min(lim, (int64_t)un.nt * kPreKeys), (int64_t)0), count = (n_keys + kKvBlock - 1) / kKvBlock;
        const auto ask = [&](int i) {
            if (i < count)
                for (int c = lane; c < L::kBytes / 16; c += 32)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                 :: "r"(smem_u32(ring.block[i % DEPTH]) + 16 * c), "l"(src + (int64_t)i * L::kBytes + 16 * c) : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int i = 0; i < DEPTH; ++i) ask(i);
        for (int i = 0; i < count; ++i) {
            asm volatile("cp.async.wait_group %0;" :: "n"(DEPTH - 1) : "memory");
            __syncwarp();
            kv4_block<D, 1, 1, true>(smem_u32(ring.block[i % DEPTH]), i * kKvBlock, n_keys, ln, rows, acc);
            __syncwarp();
            ask(i + DEPTH);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float l = acc.l[0][i];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            float mt[NG];
#pragma unroll
            for (int j = 0; j < NG; ++j) mt[j] = __shfl_sync(0xffffffffu, acc.mt[0][i], 4 * j + t);
            const int r = row0 + 2 * t + i;
            if (r >= p.R) continue;
            const bool part = un.slot >= 0;
            const int64_t in_slot = (int64_t)un.slot * kPreRows + r - un.row0;
            const int tok = r / p.G, hh = r - tok * p.G;
            uint16_t *dst = p.out + (((int64_t)un.b * p.T + tok) * p.H + un.kvh * p.G + hh) * D + 4 * g;
            const float f = part ? 1.f : l != 0.f ? 1.f / l : 0.f;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const float4 o = kv4_sums(acc, 0, i, j, mt[j], f);
                if (part) *reinterpret_cast<float4 *>(p.part_o + in_slot * D + 32 * j + 4 * g) = o;
                else *reinterpret_cast<uint2 *>(dst + 32 * j) = make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
            }
            if (part && g == 0) p.part_ml[in_slot] = make_float2(acc.M[0][i], l);
        }
        __syncwarp();                   // (the rows' fragments and the ring are used again)
    }
}

template <int D>
__global__ void __launch_bounds__(kPreThreads, 1) kv4_prefill_kernel(const __grid_constant__ PreParams pp) {
    using L = KvLayout<D>;
    using SM = PreSmem<D>;
    constexpr int NG = L::NG, NH = NG / 2, SUBS = D / 64;
    constexpr bool kApart = SM::kApart;
    const Kv4AttendParams &p = pp.a;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    PreMisc &ms = *reinterpret_cast<PreMisc *>(smem + SM::kMisc);
    volatile int *abort_flag = &ms.abort_flag;
    PrePlan &plan = *reinterpret_cast<PrePlan *>(smem + SM::kPlan);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ms.q_ready[i], 4);
            mbar_init(&ms.k_full[i], 4);
            mbar_init(&ms.k_empty[i], 1);
            mbar_init(&ms.v_full[i], 4);
            mbar_init(&ms.v_empty[i], 1);
            mbar_init(&ms.s_full[i], 1);
            mbar_init(&ms.p_full[i], 4);
            mbar_init(&ms.pv_done[i], 1);
        }
        mbar_init(&ms.drain, 1);
        for (int i = 0; i < 2; ++i) mbar_init(&ms.dq[i], 4);
        for (int i = 0; i < 4; ++i) mbar_init(&ms.m_full[i], 4);
        ms.abort_flag = 0;
        ms.any_redo = 0;
        fence_mbar_init();
    }
    if (tid < kPreRedo / 32) ms.redo[tid] = 0;
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&ms.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ms.tmem;
    const uint32_t base = smem_u32(smem);
    griddep_wait();
    const int share = pp.held ? pre_plan(pp, plan) : 0;

    if (warp < 8) {
        // ------------------------------------------------------------ softmax
        const int grp = warp >> 2, rl = (warp & 3) * 32 + lane;
        const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + t_lane + grp * 128, t_o = tmem + t_lane + 256 + grp * D,
                       t_p = tmem + t_lane + SM::kPCol + grp * SM::kPStep;
        bool ok = true;
        int tiles = 0, mine = 0;                                    // tiles before this unit: of all, and of this group
        int piece = 0;
        PreWalk walk(pp, plan, share);
        for (PreUnit un; ok && walk.next(pp, un); ++piece) {
            const int row = un.row0 + grp * 128 + rl;
            const bool have = row < p.R;
            const int tok = have ? row / p.G : 0, hh = have ? row - tok * p.G : 0;
            if (un.t0 == 0 && un.kvh == 0 && have && hh == 0 && un.pos0 + tok >= p.max_seq)
                atomicOr(&g_status, kErrBadIndex);
            if (grp >= un.groups) {
                tiles += un.nt;
                continue;
            }
            // ---- Q, scaled by 2^e (and the softmax scale's sign), in the K codes' channel order.  D / 8 lanes fetch a
            // row together, into its place; then each lane changes its own row there.  Short loops: straight code that
            // runs once per unit waits for its instructions (this took 5 us, and the way out another 5)
            float c_row = 0.f;
            if (un.nt > 0) {
                constexpr int LPR = D / 8, RPL = 32 / LPR;          // lanes per row, rows at a time
                const int64_t off = have ? (int64_t)un.b * p.ldq_b + (int64_t)tok * p.ldq_t + (int64_t)(un.kvh * p.G + hh) * p.ldq_h : -1;
                const uint32_t q_at = base + grp * SUBS * SM::kSubK + (warp & 3) * 4096;
                const int c = lane % LPR;
#pragma unroll 4
                for (int i = 0; i < LPR; ++i) {
                    const int r = i * RPL + lane / LPR;
                    const int64_t from = __shfl_sync(0xffffffffu, off, r);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                 :: "r"(q_at + (c >> 3) * SM::kSubK + r * 128 + (((c ^ r) & 7) << 4)),
                                    "l"(p.q + (from >= 0 ? from : 0) + 8 * c), "r"(from >= 0 ? 16 : 0) : "memory");
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
                const uint32_t q_row = q_at + lane * 128;
                uint32_t m2 = 0;                                    // largest magnitudes of the row, as bf16 bits
#pragma unroll 4
                for (int i = 0; i < LPR; ++i) {
                    const uint4 x = lds128(q_row + (i >> 3) * SM::kSubK + (((i ^ lane) & 7) << 4));
                    m2 = __vmaxu2(m2, __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu),
                                               __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu)));
                }
                const uint32_t top = max(m2 & 0xFFFFu, m2 >> 16);
                const int ex = (int)(top >> 7) - 127;
                const int e = top && ex < 128 ? min(max(13 - ex, -100), 110) : 0;
                const float up = __uint_as_float((uint32_t)(127 + e) << 23) * (p.scale_log2 < 0.f ? -1.f : 1.f);
#pragma unroll 1
                for (int n = 0; n < LPR; n += 4) {
                    uint4 w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = lds128(q_row + (n >> 3) * SM::kSubK + ((((n + i) ^ lane) & 7) << 4));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 x = w[i];                       // channels (0 4) (1 5) (2 6) (3 7)
                        sts128(q_row + (n >> 3) * SM::kSubK + ((((n + i) ^ lane) & 7) << 4),
                               pack_f16x2(bf_lo(x.x) * up, bf_lo(x.z) * up), pack_f16x2(bf_hi(x.x) * up, bf_hi(x.z) * up),
                               pack_f16x2(bf_lo(x.y) * up, bf_lo(x.w) * up), pack_f16x2(bf_hi(x.y) * up, bf_hi(x.w) * up));
                    }
                }
                c_row = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(127 - e) << 23);
                fence_proxy_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ms.q_ready[grp]);
            }
            // positions that this row sees, from the first tile on
            const int64_t at = have ? un.pos0 + tok : -1;
            const int64_t sees = at < 0 || at >= p.max_seq ? 0 : max(at + 1 - (int64_t)un.t0 * kPreKeys, (int64_t)0);
            // a row that sees nothing here (padding, no row) goes along as if it saw all, and is zeros at the end
            float M = kNoMax, l = 0.f;
            uint32_t bad = 0;
            int redo = 0;
            for (int j = 0; j < un.nt; ++j) {
                const int g = tiles + j, slot = g & 3;
                // (the scores first: a group that sat out a unit may be phases ahead of m_full)
                if (!role_wait(&ms.s_full[grp], (mine + j) & 1, abort_flag) ||
                    !role_wait(&ms.m_full[slot], (g >> 2) & 1, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const int vis = sees ? (int)min(max(sees - (int64_t)j * kPreKeys, (int64_t)0), (int64_t)kPreKeys) : kPreKeys;
                const float fac = c_row * ms.k_fac[slot][0], dv = ms.v_exp[slot][0];
                // (a factor of zero would make NaN of the scores that are masked by -inf)
                const int sizes = ms.uneven[slot];
                redo |= sizes & 2;
                const bool uneven = sizes & 1, plain = !uneven && !__any_sync(0xffffffffu, !(fac > 0.f));
                if (plain && __any_sync(0xffffffffu, vis < kPreKeys)) pre_mask(t_s, vis);
                const float x_top = plain ? fmaf(pre_top(t_s), fac, dv) : pre_top_any(t_s, ms, slot, uneven, c_row, vis);
                if (__any_sync(0xffffffffu, x_top > M + kRescale)) {
                    const float to = fmaxf(x_top - kPreTerm, M), a = ex2(M - to);
                    M = to;
                    l *= a;
                    if (j > 0) {                                    // O is complete up to the last tile: its PV is done
                        if (!role_wait(&ms.pv_done[grp], (mine + j - 1) & 1, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(t_o + 16 * c, o);
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * a);
                            tmem_st16(t_o + 16 * c, o);
                        }
                    }
                }
                if (kApart && j > 0 && !role_wait(&ms.pv_done[grp], (mine + j - 1) & 1, abort_flag)) {         // P is free
                    ok = false;
                    break;
                }
                l += plain ? pre_weights(t_s, t_p, fac, dv - M) * ms.v_inv[slot][0]
                           : pre_weights_any(t_s, t_p, ms, slot, uneven, c_row, M, vis);
                // (read before P is handed over: the slot is used again after that)
                if (ms.any_bad[slot])
                    for (int k = 0; k < vis; ++k) bad |= (ms.bad[slot][k >> 2] >> (8 * (k & 3))) & 0xFFu;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ms.p_full[grp]);
            }
            tiles += un.nt;
            mine += un.nt;
            if (ok && un.nt > 0) ok = role_wait(&ms.pv_done[grp], (mine - 1) & 1, abort_flag);
            if (!ok) break;
            if (redo && tid == 0) {
                ms.redo[piece / 32 % (kPreRedo / 32)] |= 1u << (piece % 32);
                ms.any_redo = 1;
            }
            tc_fence_after();
            // ---- out, by way of Q's place (its products are done): 128 bytes of 4 rows per store
            const bool part = un.slot >= 0;
            const int64_t in_slot = (int64_t)un.slot * kPreRows + grp * 128 + rl;
            int64_t off = -1;                                       // bytes of this row from the start
            if (have) off = part ? in_slot * D * 4 : (((int64_t)un.b * p.T + tok) * p.H + un.kvh * p.G + hh) * D * 2;
            if (have && part) p.part_ml[in_slot] = make_float2(sees ? M : kNoMax, sees ? l : 0.f);
            uint8_t *dst = part ? reinterpret_cast<uint8_t *>(p.part_o) : reinterpret_cast<uint8_t *>(p.out);
            const float inv = part ? 1.f : l != 0.f ? 1.f / l : 0.f;
            const int per = part ? 2 : 4;                  // 16 channels each: together 128 bytes, a piece
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
                const int piece = c / per, nth = c % per;
                const float f = (bad >> (c >> 1)) & 1u ? __int_as_float(0x7fc00000) : inv;
                uint32_t v[16];
                tmem_ld16(t_o + 16 * c, v);
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = sees ? __float_as_uint(__uint_as_float(v[k]) * f) : 0u;
                const uint32_t at = base + (grp * SUBS + piece % SUBS) * SM::kSubK + (warp & 3) * 4096;
                if (part) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        sts128(at + lane * 128 + (((4 * nth + i) ^ lane) & 7) * 16, v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            w[k] = pack_bf16x2(__uint_as_float(v[8 * i + 2 * k]), __uint_as_float(v[8 * i + 2 * k + 1]));
                        sts128(at + lane * 128 + (((2 * nth + i) ^ lane) & 7) * 16, w[0], w[1], w[2], w[3]);
                    }
                }
                if (nth + 1 < per) continue;
                __syncwarp();
#pragma unroll 2
                for (int i = 0; i < 8; ++i) {
                    const int r = 4 * i + (lane >> 3);
                    const int64_t to = __shfl_sync(0xffffffffu, off, r);
                    const uint4 x = lds128(at + r * 128 + (((lane ^ r) & 7) << 4));
                    if (to >= 0) *reinterpret_cast<uint4 *>(dst + to + piece * 128 + (lane & 7) * 16) = x;
                }
                __syncwarp();
            }
        }
        tc_fence_before();
    } else if (warp < 12) {
        // ------------------------------------------------- K and V to fp16
        // K: thread = position.  V: thread = 8 positions (vp) x 4 channels of
        // each group (vg); the scales of all positions through shared memory.
        // Scales are prepared one tile ahead of the codes, and the tile's
        // largest exponents before that, so the warps meet once per tile, long
        // after they have arrived.
        // The tiles of all pieces follow one another; the loads look ahead.
        const int dw = warp - 8, key = tid - 256, vp = (dw >> 1) * 8 + (lane & 7), vg = (dw & 1) * 4 + (lane >> 3);
        struct Tile {                                               // where a tile lies
            const uint8_t *cache;                                   // its head's blocks
            int64_t blk;                                            // its first block
            int live;                                               // positions that some row sees; 0: no more tiles
        };
        struct Feed {                                               // the tiles of this CTA's pieces, one after the other
            PreWalk walk;
            int left;                                               // tiles left of this piece
            Tile tl;
            int64_t keys;                                           // positions left of its unit
        } feed = {PreWalk(pp, plan, share), 0, {p.blocks, 0, 0}, 0};
        const auto next_tile = [&]() -> Tile {
            PreUnit un;
            while (feed.left == 0 && feed.walk.next(pp, un)) {
                feed.left = un.nt;
                feed.tl.cache = p.blocks + ((int64_t)un.b * p.KV + un.kvh) * p.nblk * L::kBytes;
                feed.tl.blk = (int64_t)un.t0 * (kPreKeys / kKvBlock);
                feed.keys = un.n_keys - (int64_t)un.t0 * kPreKeys;
            }
            Tile t = feed.tl;
            t.live = feed.left ? (int)min(feed.keys, (int64_t)kPreKeys) : 0;
            if (feed.left) {
                --feed.left;
                feed.tl.blk += kPreKeys / kKvBlock;
                feed.keys -= kPreKeys;
            }
            return t;
        };
        uint32_t kc[4][NG], vc[4][NG];                              // codes of a tile
        uint32_t rk[NH], rkm[NH], rv[NH], rvm[NH];                  // raw scales and minima of this position, in pairs
        const auto words = [](const uint8_t *at, uint32_t (&w)[NG]) {
            if constexpr (NG == 4) {
                const uint4 x = *reinterpret_cast<const uint4 *>(at);
                w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2 *>(at);
                w[0] = x.x, w[1] = x.y;
            }
        };
        const auto halves = [](const uint8_t *at, uint32_t (&w)[NH]) {
            if constexpr (NH == 2) {
                const uint2 x = *reinterpret_cast<const uint2 *>(at);
                w[0] = x.x, w[1] = x.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t *>(at);
            }
        };
        const auto load_k = [&](const Tile &tl) {                   // nothing past the cache is read
            const uint8_t *cache = tl.cache;
            const int64_t blk = tl.blk + (key >> 4);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int g = 0; g < NG; ++g) kc[t][g] = 0;
                if (blk < p.nblk) words(cache + blk * L::kBytes + ((key & 15) * 4 + t) * NG * 4, kc[t]);
            }
        };
        const auto load_v = [&](const Tile &tl) {
            const uint8_t *cache = tl.cache;
            const int64_t blk = tl.blk + (vp >> 1);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int g = 0; g < NG; ++g) vc[t][g] = 0;
                if (blk < p.nblk) words(cache + blk * L::kBytes + L::kV + (((vp & 1) * 8 + vg) * 4 + t) * NG * 4, vc[t]);
            }
        };
        const auto load_scales = [&](const Tile &tl) {
            const uint8_t *cache = tl.cache;
            const int64_t blk = tl.blk + (key >> 4);
            const int r = key & 15;
#pragma unroll
            for (int i = 0; i < NH; ++i) rk[i] = rkm[i] = rv[i] = rvm[i] = 0;
            if (tl.live > 0 && blk < p.nblk) {
                const uint8_t *at = cache + blk * L::kBytes;
                halves(at + L::kKd + r * NG * 2, rk);
                halves(at + L::kKm + r * NG * 2, rkm);
                halves(at + L::kVd + r * NG * 2, rv);
                uint32_t m[NG];                                     // pairs of positions, one word per group
                words(at + L::kVm + (r >> 1) * NG * 4, m);
#pragma unroll
                for (int i = 0; i < NH; ++i) rvm[i] = prmt(m[2 * i], m[2 * i + 1], r & 1 ? 0x7632u : 0x5410u);
            }
        };
        // numbers of a tile's position, ready to be scaled
        float kd[NG], km[NG], vd[NG], vm[NG];
        uint32_t bad_k = 0, bad_v = 0;
        constexpr int kNone = 1 << 20;
        int ke = kNone, ve = kNone;                                 // 2^e is above the position's largest value
        const auto survey = [&](int j, int live) {                  // the raw scales of tile j; writes the warp's exponents
            float kmax = 0.f, vmax = 0.f;
            uint32_t kmin = ~0u, vmin = ~0u;                        // of the groups that are not zeros: bits - 1
            bad_k = bad_v = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const auto pick = [&](const uint32_t (&w)[NH]) { return g & 1 ? bf_hi(w[g >> 1]) : bf_lo(w[g >> 1]); };
                kd[g] = pick(rk), km[g] = pick(rkm), vd[g] = pick(rv), vm[g] = pick(rvm);
                if (key >= live) kd[g] = km[g] = vd[g] = vm[g] = 0.f;           // behind the last position: zeros
                if (!finite_bits(__float_as_uint(kd[g])) || !finite_bits(__float_as_uint(km[g]))) {
                    bad_k |= 1u << g;
                    kd[g] = km[g] = 0.f;
                }
                if (!finite_bits(__float_as_uint(vd[g])) || !finite_bits(__float_as_uint(vm[g]))) {
                    bad_v |= 1u << g;
                    vd[g] = vm[g] = 0.f;
                }
                const float kt = fmaxf(fabsf(km[g]), fabsf(fmaf(15.f, kd[g], km[g]))),
                            vt = fmaxf(fabsf(vm[g]), fabsf(fmaf(15.f, vd[g], vm[g])));
                kmax = fmaxf(kmax, kt), vmax = fmaxf(vmax, vt);
                kmin = min(kmin, __float_as_uint(kt) - 1u), vmin = min(vmin, __float_as_uint(vt) - 1u);
            }
            // (V not below 2^-96: 2^-dv times the weights' sum stays finite)
            const auto exponent = [](uint32_t bits, int least) { return min(max((int)(bits >> 23) - 126, least), 110); };
            ke = kmax > 0.f ? exponent(__float_as_uint(kmax), -100) : kNone;
            ve = vmax > 0.f ? exponent(__float_as_uint(vmax), -96) : kNone;
            const int kg = kmax > 0.f ? exponent(kmin + 1u, -100) : kNone, vg = vmax > 0.f ? exponent(vmin + 1u, -96) : kNone;
            const int a = __reduce_max_sync(0xffffffffu, ke == kNone ? -100 : ke), c = __reduce_min_sync(0xffffffffu, ke),
                      d = __reduce_max_sync(0xffffffffu, ve == kNone ? -100 : ve), f = __reduce_min_sync(0xffffffffu, ve);
            const int k = __reduce_min_sync(0xffffffffu, kg), v = __reduce_min_sync(0xffffffffu, vg);
            const bool far = __any_sync(0xffffffffu, ke - kg > kPreSpread || ve - vg > kPreSpread);
            if (lane == 0) {
                int *red = ms.red[j & 1][dw];
                red[0] = a, red[1] = c, red[2] = d, red[3] = f, red[4] = k, red[5] = v, red[6] = far;
            }
            ms.bad[j & 3][lane] = 0;                                // every warp the same
            if (lane == 0) ms.any_bad[j & 3] = 0;
            __syncwarp();
        };
        uint32_t kd24[NH], kmh[NH];                                 // K's scales * 2^24 and minima of this position, fp16 pairs
        const auto scale = [&](int j) {                             // after all warps' exponents of tile j
            const int slot = j & 3;
            int k_hi = -100, k_lo = kNone, v_hi = -100, v_lo = kNone, k_grp = kNone, v_grp = kNone, far = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int *red = ms.red[j & 1][i];
                k_hi = max(k_hi, red[0]), k_lo = min(k_lo, red[1]), v_hi = max(v_hi, red[2]), v_lo = min(v_lo, red[3]);
                k_grp = min(k_grp, red[4]), v_grp = min(v_grp, red[5]), far |= red[6];
            }
            const bool uneven = !far && (k_hi - k_lo > 6 || v_hi - v_lo > 6 || k_hi - k_grp > kPreSpread || v_hi - v_grp > kPreSpread);
            // 2^-dk times the largest value is at most 2^-6
            const int dk = (uneven && ke != kNone ? ke : k_hi) + 6, dv = (uneven && ve != kNone ? ve : v_hi) + 6;
            const float k0 = __uint_as_float((uint32_t)(127 - dk) << 23), k24 = k0 * 0x1p24f,
                        v0 = __uint_as_float((uint32_t)(127 - dv) << 23), v24 = v0 * 0x1p24f;
            uint16_t *a = reinterpret_cast<uint16_t *>(smem + SM::kScale + (j & 1) * SM::kScaleBytes);
#pragma unroll
            for (int i = 0; i < NH; ++i) {
                kd24[i] = pack_f16x2(kd[2 * i] * k24, kd[2 * i + 1] * k24) | (bad_k >> (2 * i) & 1 ? 0x7FFFu : 0u) |
                          (bad_k >> (2 * i + 1) & 1 ? 0x7FFF0000u : 0u);
                kmh[i] = pack_f16x2(km[2 * i] * k0, km[2 * i + 1] * k0);
                const uint32_t d = pack_f16x2(vd[2 * i] * v24, vd[2 * i + 1] * v24), m = pack_f16x2(vm[2 * i] * v0, vm[2 * i + 1] * v0);
                a[2 * i * kPreKeys + key] = (uint16_t)d;
                a[(2 * i + 1) * kPreKeys + key] = (uint16_t)(d >> 16);
                a[(NG + 2 * i) * kPreKeys + key] = (uint16_t)m;
                a[(NG + 2 * i + 1) * kPreKeys + key] = (uint16_t)(m >> 16);
            }
            if (bad_v) {
                atomicOr(&ms.bad[slot][key >> 2], bad_v << (8 * (key & 3)));
                ms.any_bad[slot] = 1;
            }
            if (key == 0) ms.uneven[slot] = (int)uneven | far << 1;
            if (uneven || key == 0) {
                ms.k_fac[slot][key] = __uint_as_float((uint32_t)(127 + dk) << 23);
                ms.v_exp[slot][key] = (float)dv;
                ms.v_inv[slot][key] = ex2((float)-dv);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms.m_full[slot]);
        };
        Tile now = next_tile(), ahead = next_tile();               // tile j and tile j + 1
        load_scales(now);
        load_k(now);
        load_v(now);
        survey(0, now.live);
        if (lane == 0) mbar_arrive(&ms.dq[1]);
        load_scales(ahead);
        bool ok = role_wait(&ms.dq[1], 0, abort_flag);
        if (ok && now.live) scale(0);
        for (int j = 0; now.live && ok; ++j) {
            const int st = j & 1;
            const uint32_t wait_parity = ((j >> 1) & 1) ^ 1;
            // ---- arrive with the scales of this tile and the exponents of the next
            survey(j + 1, ahead.live);
            if (lane == 0) mbar_arrive(&ms.dq[0]);
            const Tile later = next_tile();
            load_scales(later);
            // ---- K: 16-byte chunks of 8 channels, [128 positions][64 channels] swizzled
            if (!role_wait(&ms.k_empty[st], wait_parity, abort_flag)) break;
            const uint32_t k_row = base + SM::kK + st * SM::kKStage + key * 128;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t sel = g & 1 ? 0x3232u : 0x1010u;
                const uint32_t d24 = prmt(kd24[g >> 1], 0u, sel), m = prmt(kmh[g >> 1], 0u, sel);
                const uint32_t d20 = hmul2(d24, 0x2C002C00u);       // / 16
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t w = kc[t][g], h = w >> 8;
                    const int c = g * 4 + t;                        // chunk of the row
                    sts128(k_row + (c >> 3) * SM::kSubK + (((c ^ key) & 7) << 4), hfma2(w & 0x000F000Fu, d24, m),
                           hfma2(w & 0x00F000F0u, d20, m), hfma2(h & 0x000F000Fu, d24, m), hfma2(h & 0x00F000F0u, d20, m));
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms.k_full[st]);
            if (ahead.live) load_k(ahead);
            // ---- V^T: 16-byte chunks of 8 positions, [D channels][64 positions] swizzled
            if (!role_wait(&ms.dq[0], j & 1, abort_flag) || !role_wait(&ms.v_empty[st], wait_parity, abort_flag)) break;
            const uint32_t v_tile = base + SM::kV + st * SM::kVStage + (vp >> 3) * SM::kSubV;
            const uint32_t v_scale = base + SM::kScale + (j & 1) * SM::kScaleBytes + vp * 16;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint4 d4 = lds128(v_scale + g * kPreKeys * 2), m4 = lds128(v_scale + (NG + g) * kPreKeys * 2);
                const uint32_t d24[4] = {d4.x, d4.y, d4.z, d4.w}, m[4] = {m4.x, m4.y, m4.z, m4.w};
                uint32_t x[4][4];                                   // [channel][position pair]
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t w = vc[t][g], h = w >> 8, d20 = hmul2(d24[t], 0x2C002C00u);
                    x[0][t] = hfma2(w & 0x000F000Fu, d24[t], m[t]);
                    x[1][t] = hfma2(w & 0x00F000F0u, d20, m[t]);
                    x[2][t] = hfma2(h & 0x000F000Fu, d24[t], m[t]);
                    x[3][t] = hfma2(h & 0x00F000F0u, d20, m[t]);
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int ch = 32 * g + 4 * vg + n;
                    sts128(v_tile + ch * 128 + (((vp ^ ch) & 7) << 4), x[n][0], x[n][1], x[n][2], x[n][3]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms.v_full[st]);
            if (ahead.live) {
                load_v(ahead);
                scale(j + 1);
            }
            now = ahead;
            ahead = later;
        }
    } else if (lane == 0) {
        // ------------------------------------------------------------ MMAs
        constexpr uint32_t id_s = umma_idesc_f16<kPreKeys>(), id_o = umma_idesc_f16<D>();
        const auto qk = [&](int g, int st) {                        // the scores of the tile in stage st
            uint64_t a = umma_desc_sw128(base + g * SUBS * SM::kSubK), bd = umma_desc_sw128(base + SM::kK + st * SM::kKStage);
#pragma unroll 1
            for (int s = 0; s < SUBS; ++s) {
#pragma unroll
                for (int k = 0; k < 4; ++k)                         // 16 channels each: 32 bytes along the row
                    umma_f16_ss(tmem + g * 128, a + 2u * k, bd + 2u * k, id_s, (s | k) != 0);
                a += SM::kSubK >> 4;
                bd += SM::kSubK >> 4;
            }
            umma_commit(&ms.s_full[g]);
        };
        bool ok = true;
        int tiles = 0, mine[2] = {0, 0}, units[2] = {0, 0};         // so far: tiles, and tiles and units of each group
        PreWalk walk(pp, plan, share);
        for (PreUnit un; ok && walk.next(pp, un);) {
            if (un.nt == 0) continue;
            for (int g = 0; g < un.groups && ok; ++g) ok = role_wait(&ms.q_ready[g], units[g]++ & 1, abort_flag);
            ok = ok && role_wait(&ms.k_full[tiles & 1], (tiles >> 1) & 1, abort_flag);
            if (ok) {
                tc_fence_after();
                for (int g = 0; g < un.groups; ++g) qk(g, tiles & 1);
                umma_commit(&ms.k_empty[tiles & 1]);
            }
            for (int j = 0; j < un.nt && ok; ++j) {
                const int t = tiles + j, st = t & 1;
                for (int g = 0; g < un.groups && ok; ++g) {
                    const bool last = g == un.groups - 1;
                    if (kApart) ok = role_wait(&ms.p_full[g], (mine[g] + j) & 1, abort_flag);
                    if (kApart && ok && j + 1 < un.nt) {            // the scores were read: the next ones
                        if (g == 0) ok = role_wait(&ms.k_full[st ^ 1], ((t + 1) >> 1) & 1, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        qk(g, st ^ 1);
                        if (last) umma_commit(&ms.k_empty[st ^ 1]);
                    }
                    if (ok && g == 0) ok = role_wait(&ms.v_full[st], (t >> 1) & 1, abort_flag);
                    if (!kApart) ok = ok && role_wait(&ms.p_full[g], (mine[g] + j) & 1, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    uint64_t bd = umma_desc_sw128(base + SM::kV + st * SM::kVStage);
                    uint32_t pa = tmem + SM::kPCol + g * SM::kPStep;
#pragma unroll 1
                    for (int s = 0; s < 2; ++s) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)                 // 16 positions each: 8 columns of P
                            umma_f16_ts(tmem + 256 + g * D, pa + 8 * k, bd + 2u * k, id_o, (j | s | k) != 0);
                        pa += 32;
                        bd += SM::kSubV >> 4;
                    }
                    umma_commit(&ms.pv_done[g]);
                    if (last) umma_commit(&ms.v_empty[st]);
                    if (kApart || j + 1 == un.nt) continue;
                    // the next scores take the place of P: after its product is done
                    if (g == 0) ok = role_wait(&ms.k_full[st ^ 1], ((t + 1) >> 1) & 1, abort_flag);
                    ok = ok && role_wait(&ms.pv_done[g], (mine[g] + j) & 1, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    qk(g, st ^ 1);
                    if (last) umma_commit(&ms.k_empty[st ^ 1]);
                }
            }
            tiles += un.nt;
            for (int g = 0; g < un.groups; ++g) mine[g] += un.nt;
        }
        // nothing in flight when tensor memory goes
        umma_commit(&ms.drain);
        mbar_wait(&ms.drain, 0, &g_status);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512) : "memory");
    }
    // ---- pieces that fp16 is not enough for
    static_assert(sizeof(PreRing<D>) % 16 == 0 && sizeof(PreRing<D>) * (kPreThreads / 32) <= SM::kScale, "PreRing");
    if (!ms.any_redo || ms.abort_flag) return;
    PreWalk walk(pp, plan, share);
    int piece = 0;
    for (PreUnit un; walk.next(pp, un); ++piece)
        if (ms.redo[piece / 32 % (kPreRedo / 32)] >> (piece % 32) & 1u) pre_redo<D>(p, un, reinterpret_cast<PreRing<D> *>(smem)[warp]);
}

// The sums of the units that were cut, joined: one warp per row.
template <int D>
__global__ void __launch_bounds__(256) kv4_prefill_join_kernel(const __grid_constant__ PreParams pp) {
    constexpr int V = D / 32;
    const Kv4AttendParams &p = pp.a;
    const int lane = threadIdx.x & 31;
    griddep_launch_dependents();
    griddep_wait();
    if (!pp.held[0]) return;
    for (int task = blockIdx.x; task < pp.units * (kPreRows / 8); task += gridDim.x) {
        const int u = task / (kPreRows / 8), tile = u / pp.items, item = u - tile * pp.items;
        const int in_unit = task % (kPreRows / 8) * 8 + (threadIdx.x >> 5), r = (pp.row_tiles - 1 - tile) * kPreRows + in_unit;
        const int2 held = reinterpret_cast<const int2 *>(pp.held)[1 + u];
        if (held.x == held.y || r >= p.R) continue;
        const int n = held.y - held.x + 1;
        const auto slot = [&](int s) { return (int64_t)(2 * (held.x + s) + (s == 0)) * kPreRows + in_unit; };
        float top = kNoMax;
        for (int s = lane; s < n; s += 32) top = fmaxf(top, p.part_ml[slot(s)].x);
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float acc[V], l = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 8
        for (int s = 0; s < n; ++s) {
            const float2 x = p.part_ml[slot(s)];
            const float f = ex2(x.x - top);
            l += x.y * f;
            const float *src = p.part_o + slot(s) * D + lane * V;
            if constexpr (V == 4) {
                const float4 y = *reinterpret_cast<const float4 *>(src);
                acc[0] = fmaf(y.x, f, acc[0]);
                acc[1] = fmaf(y.y, f, acc[1]);
                acc[2] = fmaf(y.z, f, acc[2]);
                acc[3] = fmaf(y.w, f, acc[3]);
            } else {
                const float2 y = *reinterpret_cast<const float2 *>(src);
                acc[0] = fmaf(y.x, f, acc[0]);
                acc[1] = fmaf(y.y, f, acc[1]);
            }
        }
        const float inv = l != 0.f ? 1.f / l : 0.f;
        const int64_t b = item / p.KV;
        const int kvh = item - (int)b * p.KV, tok = r / p.G, hh = r - tok * p.G;
        uint16_t *dst = p.out + ((b * p.T + tok) * p.H + kvh * p.G + hh) * D + lane * V;
#pragma unroll
        for (int i = 0; i < V; i += 2)
            *reinterpret_cast<uint32_t *>(dst + i) = pack_bf16x2(acc[i] * inv, acc[i + 1] * inv);
    }
}

static int64_t prefill_units(int64_t B, int64_t KV, int64_t R) { return B * KV * ((R + kPreRows - 1) / kPreRows); }

// Units may be cut where whole ones can leave CTAs idle: fewer units than CTAs,
// or up to four per CTA over a long cache.  A prompt from its first token on (a
// cache of at most twice its tokens) with more units than CTAs goes well in whole
// units, of which the longest go with the shortest: planning and a second kernel
// made 2048 tokens of the 8B heads 3 us slower (61 -> 64); 3 x 511 tokens of 8
// heads of 64 channels behind 333 to 7003 positions, 48 units, went from 63 us
// with equal cuts of each unit to 47.  (The costs' sum has to fit 31 bits.)
static bool prefill_may_cut(int64_t B, int64_t KV, int64_t R, int64_t T, int64_t max_seq) {
    const int64_t units = prefill_units(B, KV, R);
    return units <= kPreCut && (units < 148 || max_seq > 2 * T) &&
           units * (max_seq / kPreKeys + 1 + kPreUnitCost) <= (1 << 30);
}

// Two pieces per CTA that are not whole units, and who holds what.
int64_t kv4_prefill_workspace(int64_t B, int64_t KV, int64_t R, int64_t T, int64_t D, int64_t max_seq) {
    return !prefill_may_cut(B, KV, R, T, max_seq) ? 0 : 2 * 148 * kPreRows * (D * 4 + 8) + (kPreCut + 1) * 8;
}

int kv4_prefill(Kv4AttendParams p, int64_t D, void *workspace, cudaStream_t st) {
    PreParams pp = {};
    const int64_t units = prefill_units(p.B, p.KV, p.R);
    if (units > 0x3fffffffLL) return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_kv4_attend: too many query rows");
    pp.items = p.B * p.KV;
    pp.row_tiles = (p.R + kPreRows - 1) / kPreRows;
    pp.units = (int)units;
    const bool may_cut = prefill_may_cut(p.B, p.KV, p.R, p.T, p.max_seq);
    if (may_cut) {
        const int64_t rows = 2 * 148 * kPreRows;
        p.part_o = (float *)workspace;
        p.part_ml = (float2 *)((uint8_t *)workspace + rows * D * 4);
        pp.held = (int *)((uint8_t *)workspace + rows * (D * 4 + 8));
    }
    pp.a = p;
    const dim3 grid(148);
    const int rc = D == 64 ? launch_kv4<kv4_prefill_kernel<64>>(grid, kPreThreads, PreSmem<64>::kBytes, st, "kv4_prefill_kernel", pp)
                           : launch_kv4<kv4_prefill_kernel<128>>(grid, kPreThreads, PreSmem<128>::kBytes, st, "kv4_prefill_kernel", pp);
    if (rc != BF16X_OK || !may_cut) return rc;
    const dim3 jgrid((unsigned)std::min(pp.units * (kPreRows / 8), 148 * 8));
    return D == 64 ? launch_kv4<kv4_prefill_join_kernel<64>>(jgrid, 256, 0, st, "kv4_prefill_join_kernel", pp)
                   : launch_kv4<kv4_prefill_join_kernel<128>>(jgrid, 256, 0, st, "kv4_prefill_join_kernel", pp);
}

}  // namespace bf16x
