// bf16x_kv4_prefill.cu -- attention of many query rows over the 4-bit cache
// (prompts, chunks of prompts) on the 5th-generation tensor cores.
//
// Rows r = t * G + h of one kv head, 256 per CTA (two groups of 128), walk
// over the cache in tiles of 128 positions:
//   S[128][128] = Q K^T,  P = 2^(S c - M),  O[128][D] += P V
// with S, P and O in tensor memory (P takes the place of S) and Q, K and V^T as
// fp16 operands in shared memory.  17 warps:
//   0..3, 4..7  one softmax group per 128 rows, one thread per row: scores out
//               of tensor memory, maximum, 2^x, P back as fp16
//   8..15       K and V of the next tile from 4 bits to fp16 (loaded one tile
//               ahead into registers), into two stages each
//   16          issues the MMAs
// While one group works on its scores, the tensor cores work for the other.
//
// fp16 operands hold any scale: a row of Q is scaled by a power of two into
// [2^13, 2^14), exact; the values of a tile by 2^-dk (K) and 2^-dv (V) to at
// most 2^-6, so that d * 2^24 fits fp16 and one fused multiply-add per pair
// turns codes (subnormal fp16, see bf16x_kv4.cuh) into values, rounded once (2^-12).
// dk enters the scores' factor.  dv enters the exponent, P' = 2^(S c + dv - M),
// and its inverse the sum l of the P'; M is raised, and O scaled, only when a
// term exceeds it by more than 2^8.  dk and dv are one number per tile, unless
// its positions differ by more than 2^6 in size: then each position has its own
// (fp16 would lose the small ones), which costs the softmax a third more work.
//
// A V group that is not finite reads as zeros here, and the rows that see its
// position get NaN in its 32 channels at the end: 0 * NaN would reach the rows
// that do not.
//
// Bound: per tile and 256 rows at D = 128 the MMAs take 2048 cycles and 2^x
// (16 per cycle and SM) takes 2048.
#include <algorithm>

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "bf16x_kv4.cuh"
#include "bf16x_umma.cuh"
#include "bf16x_wait.cuh"

namespace bf16x {

constexpr int kPreRows = 256;                         // rows per CTA
constexpr int kPreKeys = 128;                         // positions per tile
constexpr int kPreThreads = 17 * 32;

template <int D>
struct PreSmem {
    static constexpr int NG = D / 32;
    static constexpr int kSubK = kPreKeys * 128;      // [128 rows][64 columns] fp16
    static constexpr int kSubV = D * 128;             // [D rows][64 positions] fp16
    static constexpr int kK = 2 * (D / 64) * kSubK;   // offsets: Q of both groups first
    static constexpr int kKStage = (D / 64) * kSubK;
    static constexpr int kV = kK + 2 * kKStage;
    static constexpr int kVStage = 2 * kSubV;
    static constexpr int kScale = kV + 2 * kVStage;   // fp16: kd [128][NG], km [128][NG], vd [NG][128], vm [NG][128]
    static constexpr int kScaleBytes = 4 * kPreKeys * NG * 2;
    static constexpr int kMisc = kScale + kScaleBytes;
    static constexpr int kBytes = kMisc + 7424 + 1024;              // alignment slack
};

struct PreMisc {
    uint64_t q_ready[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], pv_done[2], drain;
    uint64_t dq[2], m_full[4];                        // the converting warps among themselves; a tile's numbers below
    uint32_t tmem;
    int abort_flag;
    int red[8][4];
    int uneven[4];                                    // of tile j at j % 4: each position has its own dk and dv
    float k_fac[4][kPreKeys], v_exp[4][kPreKeys], v_inv[4][kPreKeys];      // 2^dk, dv, 2^-dv; else the first only
    uint32_t any_bad[4];
    uint32_t bad[4][kPreKeys / 4];                    // per position a byte: its V groups that are not finite
};
static_assert(sizeof(PreMisc) <= 7424, "PreMisc");

__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(a));
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        :: "r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
           "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
           "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
           "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        :: "r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
           "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
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

// The maximum of a row's terms S c + dv over the `vis` positions that it sees.
template <bool UNEVEN, bool MASK>
__device__ __forceinline__ float pre_top(uint32_t t_s, const PreMisc &ms, int slot, float c_row, int vis) {
    float mx = -__builtin_huge_valf();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        tmem_ld32(t_s + 32 * c, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float x = __uint_as_float(v[i]);
            if (UNEVEN) x = fmaf(x, c_row * ms.k_fac[slot][32 * c + i], ms.v_exp[slot][32 * c + i]);
            if (!MASK || 32 * c + i < vis) mx = fmaxf(mx, x);
        }
    }
    return UNEVEN ? mx : fmaf(mx, c_row * ms.k_fac[slot][0], ms.v_exp[slot][0]);
}

// P = 2^(S c + dv - M) as fp16 over S; returns the sum of 2^-dv P.
template <bool UNEVEN, bool MASK>
__device__ __forceinline__ float pre_weights(uint32_t t_s, const PreMisc &ms, int slot, float c_row, float M, int vis) {
    const float fac = c_row * ms.k_fac[slot][0], off = ms.v_exp[slot][0] - M;
    const uint64_t f2 = pack2(fac, fac), o2 = pack2(off, off);
    uint64_t sum2 = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t v[32], o[16];
        tmem_ld32(t_s + 32 * c, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int k = 32 * c + 2 * i;
            float x, y;
            if (UNEVEN) {
                x = fmaf(__uint_as_float(v[2 * i]), c_row * ms.k_fac[slot][k], ms.v_exp[slot][k] - M);
                y = fmaf(__uint_as_float(v[2 * i + 1]), c_row * ms.k_fac[slot][k + 1], ms.v_exp[slot][k + 1] - M);
            } else {
                unpack2(fma2(pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), f2, o2), x, y);
            }
            x = ex2(x);
            y = ex2(y);
            if (MASK) {
                x = k < vis ? x : 0.f;
                y = k + 1 < vis ? y : 0.f;
            }
            sum2 = UNEVEN ? fma2(pack2(x, y), pack2(ms.v_inv[slot][k], ms.v_inv[slot][k + 1]), sum2)
                          : add2(sum2, pack2(x, y));
            o[i] = pack_f16x2(x, y);
        }
        tmem_st16(t_s + 16 * c, o);
    }
    float x, y;
    unpack2(sum2, x, y);
    return UNEVEN ? x + y : (x + y) * ms.v_inv[slot][0];
}

struct PreParams {
    Kv4AttendParams a;
    int items, nsplit, row_tiles;
};

template <int D>
__global__ void __launch_bounds__(kPreThreads, 1) kv4_prefill_kernel(const __grid_constant__ PreParams pp) {
    using L = KvLayout<D>;
    using SM = PreSmem<D>;
    constexpr int NG = L::NG, NH = NG / 2, SUBS = D / 64;
    const Kv4AttendParams &p = pp.a;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    PreMisc &ms = *reinterpret_cast<PreMisc *>(smem + SM::kMisc);
    volatile int *abort_flag = &ms.abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_launch_dependents();
    griddep_wait();
    // ---- this CTA's rows and positions; the row tiles that see most come first
    const int item = blockIdx.x % pp.items, tile = pp.row_tiles - 1 - blockIdx.x / pp.items, split = blockIdx.y;
    const int b = item / p.KV, kvh = item - b * p.KV, row0 = tile * kPreRows;
    const int64_t pos0 = p.pos0[(int64_t)b * p.pos_stride];
    const int tok_last = min(row0 + kPreRows - 1, p.R - 1) / p.G;
    if (tid == 0 && pos0 + tok_last >= p.max_seq) atomicOr(&g_status, kErrBadIndex);
    const int64_t n_keys = max(min(pos0 + tok_last + 1, p.max_seq), (int64_t)0);
    const int64_t all = (n_keys + kPreKeys - 1) / kPreKeys;
    const int64_t t0 = all * split / pp.nsplit, t1 = all * (split + 1) / pp.nsplit;
    const int nt = (int)(t1 - t0);
    const int groups = p.R - row0 > 128 ? 2 : 1;
    const int64_t part0 = ((int64_t)item * pp.nsplit + split) * p.R;          // first row of this part
    // ---- a thread's row (softmax groups)
    const int grp = warp >> 2, row = row0 + (grp & 1) * 128 + (warp & 3) * 32 + lane;
    const bool have = warp < 8 && row < p.R;
    const int tok = have ? row / p.G : 0, hh = have ? row - tok * p.G : 0;
    const auto write_row = [&](int c0, const float (&o)[32], float M, float l) {       // channels c0 .. c0 + 31
        if (!have) return;
        if (pp.nsplit > 1) {
            float *dst = p.part_o + (part0 + row) * D + c0;
#pragma unroll
            for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4 *>(dst + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            if (c0 == 0) p.part_ml[part0 + row] = make_float2(M, l);
        } else {
            const float inv = l != 0.f ? 1.f / l : 0.f;
            uint16_t *dst = p.out + (((int64_t)b * p.T + tok) * p.H + kvh * p.G + hh) * D + c0;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
                *reinterpret_cast<uint4 *>(dst + i) =
                    make_uint4(pack_bf16x2(o[i] * inv, o[i + 1] * inv), pack_bf16x2(o[i + 2] * inv, o[i + 3] * inv),
                               pack_bf16x2(o[i + 4] * inv, o[i + 5] * inv), pack_bf16x2(o[i + 6] * inv, o[i + 7] * inv));
        }
    };
    if (nt == 0) {
        const float zero[32] = {};
        for (int c0 = 0; c0 < D; c0 += 32) write_row(c0, zero, kNoMax, 0.f);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ms.q_ready[i], 4);
            mbar_init(&ms.k_full[i], 8);
            mbar_init(&ms.k_empty[i], 1);
            mbar_init(&ms.v_full[i], 8);
            mbar_init(&ms.v_empty[i], 1);
            mbar_init(&ms.s_full[i], 1);
            mbar_init(&ms.p_full[i], 4);
            mbar_init(&ms.pv_done[i], 1);
        }
        mbar_init(&ms.drain, 1);
        for (int i = 0; i < 2; ++i) mbar_init(&ms.dq[i], 8);
        for (int i = 0; i < 4; ++i) mbar_init(&ms.m_full[i], 8);
        ms.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&ms.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ms.tmem;
    const uint32_t base = smem_u32(smem);

    if (warp < 8) {
        // ------------------------------------------------------------ softmax
        if (grp < groups) {
            const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t t_s = tmem + t_lane + grp * 128, t_o = tmem + t_lane + 256 + grp * D;
            // ---- this row of Q, scaled by 2^e (and the softmax scale's sign), in the K codes' channel order
            const uint16_t *src = p.q + (int64_t)b * p.ldq_b + (int64_t)tok * p.ldq_t + (int64_t)(kvh * p.G + hh) * p.ldq_h;
            float top = 0.f;
            for (int c = 0; c < D / 8; ++c) {
                const uint4 raw = have ? *reinterpret_cast<const uint4 *>(src + 8 * c) : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(bf_lo(w[i])), fabsf(bf_hi(w[i]))));
            }
            const int ex = (int)(__float_as_uint(top) >> 23) - 127;
            const int e = top > 0.f && ex < 128 ? min(max(13 - ex, -100), 110) : 0;
            const float up = __uint_as_float((uint32_t)(127 + e) << 23) * (p.scale_log2 < 0.f ? -1.f : 1.f);
            const int rl = (warp & 3) * 32 + lane;
            const uint32_t q_row = base + grp * SUBS * SM::kSubK + rl * 128;
            for (int c = 0; c < D / 8; ++c) {
                const uint4 raw = have ? *reinterpret_cast<const uint4 *>(src + 8 * c) : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
                float x[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[2 * i] = bf_lo(w[i]) * up;
                    x[2 * i + 1] = bf_hi(w[i]) * up;
                }
                sts128(q_row + (c >> 3) * SM::kSubK + (((c ^ rl) & 7) << 4), pack_f16x2(x[0], x[4]),
                       pack_f16x2(x[1], x[5]), pack_f16x2(x[2], x[6]), pack_f16x2(x[3], x[7]));
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms.q_ready[grp]);
            const float c_row = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(127 - e) << 23);
            // positions that this row sees, from the first tile on
            const int64_t at = have ? pos0 + tok : -1;
            const int64_t sees = at < 0 || at >= p.max_seq ? 0 : max(at + 1 - t0 * kPreKeys, (int64_t)0);
            float M = kNoMax, l = 0.f;
            uint32_t bad = 0;
            bool ok = true;
            for (int j = 0; j < nt; ++j) {
                if (!role_wait(&ms.m_full[j & 3], (j >> 2) & 1, abort_flag) ||
                    !role_wait(&ms.s_full[grp], j & 1, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const int vis = (int)min(max(sees - (int64_t)j * kPreKeys, (int64_t)0), (int64_t)kPreKeys);
                const bool masked = __any_sync(0xffffffffu, vis < kPreKeys), uneven = ms.uneven[j & 3];
                const float x_top = uneven   ? pre_top<true, true>(t_s, ms, j & 3, c_row, vis)
                                    : masked ? pre_top<false, true>(t_s, ms, j & 3, c_row, vis)
                                             : pre_top<false, false>(t_s, ms, j & 3, c_row, vis);
                if (__any_sync(0xffffffffu, x_top > M + kRescale)) {
                    const float to = x_top > M ? x_top : M;
                    const float a = ex2(M - to);
                    M = to;
                    l *= a;
                    if (j > 0) {                                    // O is complete up to the last tile: its PV is done
                        if (!role_wait(&ms.pv_done[grp], (j - 1) & 1, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t v[32];
                            tmem_ld32(t_o + 32 * c, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * a);
                            tmem_st32(t_o + 32 * c, v);
                        }
                    }
                }
                const float sum = uneven   ? pre_weights<true, true>(t_s, ms, j & 3, c_row, M, vis)
                                  : masked ? pre_weights<false, true>(t_s, ms, j & 3, c_row, M, vis)
                                           : pre_weights<false, false>(t_s, ms, j & 3, c_row, M, vis);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ms.p_full[grp]);
                l += sum;
                if (ms.any_bad[j & 3])
                    for (int i = 0; i < vis; ++i) bad |= (ms.bad[j & 3][i >> 2] >> (8 * (i & 3))) & 0xFFu;
            }
            if (ok && role_wait(&ms.pv_done[grp], (nt - 1) & 1, abort_flag)) {
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t v[32];
                    tmem_ld32(t_o + 32 * c, v);
                    tmem_wait_ld();
                    float o[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        o[i] = (bad >> c) & 1u ? __int_as_float(0x7fc00000) : __uint_as_float(v[i]);
                    write_row(32 * c, o, M, l);
                }
            }
            tc_fence_before();
        }
    } else if (warp < 16) {
        // ------------------------------------------------- K and V to fp16
        const int dw = warp - 8, dt = tid - 256;
        // K: 8 positions x 2 halves of the channels' words x 2; V: 8 half blocks x 2 halves of the groups x 2
        const int part = (lane >> 3) & 1, key = dw * 16 + (lane >> 4) * 8 + (lane & 7);
        const int vp = (dw >> 2) * 8 + (lane & 7), vg = (dw & 3) * 2 + (lane >> 4);
        const uint8_t *cache = p.blocks + ((int64_t)b * p.KV + kvh) * p.nblk * L::kBytes;
        struct Raw {
            uint32_t k[2][NG], v[4][NH], kd, km, vd, vm;                    // codes; two groups' scales and minima
        } raw;
        const auto load = [&](int j) {                              // this thread's part of tile j; nothing past the cache
            const int64_t blk0 = (t0 + j) * (kPreKeys / kKvBlock);
            const int64_t kb = blk0 + dw, vb = blk0 + (vp >> 1);
            raw = Raw{};
            if (kb < p.nblk) {
                const uint8_t *at = cache + kb * L::kBytes;
                const int r = key & 15;
#pragma unroll
                for (int i = 0; i < NH; ++i)
                    raw.vm |= (uint32_t)*reinterpret_cast<const uint16_t *>(
                                  at + L::kVm + (((r >> 1) * NG + part * NH + i) * 2 + (r & 1)) * 2) << (16 * i);
                if constexpr (NG == 4) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(at + (r * 4 + 2 * part) * 16);
                    const uint4 y = *reinterpret_cast<const uint4 *>(at + (r * 4 + 2 * part + 1) * 16);
                    raw.k[0][0] = x.x, raw.k[0][1] = x.y, raw.k[0][2] = x.z, raw.k[0][3] = x.w;
                    raw.k[1][0] = y.x, raw.k[1][1] = y.y, raw.k[1][2] = y.z, raw.k[1][3] = y.w;
                    raw.kd = *reinterpret_cast<const uint32_t *>(at + L::kKd + r * 8 + part * 4);
                    raw.km = *reinterpret_cast<const uint32_t *>(at + L::kKm + r * 8 + part * 4);
                    raw.vd = *reinterpret_cast<const uint32_t *>(at + L::kVd + r * 8 + part * 4);
                } else {
                    const uint4 x = *reinterpret_cast<const uint4 *>(at + (r * 4 + 2 * part) * 8);
                    raw.k[0][0] = x.x, raw.k[0][1] = x.y, raw.k[1][0] = x.z, raw.k[1][1] = x.w;
                    raw.kd = *reinterpret_cast<const uint16_t *>(at + L::kKd + r * 4 + part * 2);
                    raw.km = *reinterpret_cast<const uint16_t *>(at + L::kKm + r * 4 + part * 2);
                    raw.vd = *reinterpret_cast<const uint16_t *>(at + L::kVd + r * 4 + part * 2);
                }
            }
            if (vb < p.nblk) {
                const uint8_t *at = cache + vb * L::kBytes + L::kV + (((vp & 1) * 8 + vg) * 4) * NG * 4 + part * NH * 4;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if constexpr (NG == 4) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(at + t * 16);
                        raw.v[t][0] = x.x, raw.v[t][1] = x.y;
                    } else {
                        raw.v[t][0] = *reinterpret_cast<const uint32_t *>(at + t * 8);
                    }
                }
            }
        };
        load(0);
        const uint32_t s_kd = base + SM::kScale, s_km = s_kd + kPreKeys * NG * 2, s_vd = s_km + kPreKeys * NG * 2,
                       s_vm = s_vd + kPreKeys * NG * 2;
        for (int j = 0; j < nt; ++j) {
            const int st = j & 1, slot = j & 3;
            const uint32_t wait_parity = ((j >> 1) & 1) ^ 1;
            // ---- scales and minima; positions from n_keys on are zeros
            const int64_t key0 = (t0 + j) * kPreKeys;
            const int live = (int)min(n_keys - key0, (int64_t)kPreKeys);
            float kd[2], km[2], vd[2], vm[2];
            kd[0] = bf_lo(raw.kd), kd[1] = bf_hi(raw.kd);
            km[0] = bf_lo(raw.km), km[1] = bf_hi(raw.km);
            vd[0] = bf_lo(raw.vd), vd[1] = bf_hi(raw.vd);
            vm[0] = bf_lo(raw.vm), vm[1] = bf_hi(raw.vm);
            uint32_t bad_k = 0, bad_v = 0;
            float kmax = 0.f, vmax = 0.f;                           // no value of this position is larger
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (key >= live) kd[i] = km[i] = vd[i] = vm[i] = 0.f;
                if (!finite_bits(__float_as_uint(kd[i])) || !finite_bits(__float_as_uint(km[i]))) {
                    bad_k |= 1u << i;
                    kd[i] = km[i] = 0.f;
                }
                if (!finite_bits(__float_as_uint(vd[i])) || !finite_bits(__float_as_uint(vm[i]))) {
                    bad_v |= 1u << i;
                    vd[i] = vm[i] = 0.f;
                }
                kmax = fmaxf(kmax, fmaxf(fabsf(km[i]), fabsf(fmaf(15.f, kd[i], km[i]))));
                vmax = fmaxf(vmax, fmaxf(fabsf(vm[i]), fabsf(fmaf(15.f, vd[i], vm[i]))));
            }
            kmax = fmaxf(kmax, __shfl_xor_sync(0xffffffffu, kmax, 8));          // the position's other groups
            vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 8));
            // exponents: 2^e is above the largest value; a position of zeros has none
            constexpr int kNone = 1 << 20;
            const int ke = kmax > 0.f ? min(max((int)(__float_as_uint(kmax) >> 23) - 126, -100), 110) : kNone,
                      ve = vmax > 0.f ? min(max((int)(__float_as_uint(vmax) >> 23) - 126, -100), 110) : kNone;
            int k_hi = __reduce_max_sync(0xffffffffu, ke == kNone ? -100 : ke), k_lo = __reduce_min_sync(0xffffffffu, ke),
                v_hi = __reduce_max_sync(0xffffffffu, ve == kNone ? -100 : ve), v_lo = __reduce_min_sync(0xffffffffu, ve);
            if (lane == 0) {
                ms.red[dw][0] = k_hi;
                ms.red[dw][1] = k_lo;
                ms.red[dw][2] = v_hi;
                ms.red[dw][3] = v_lo;
            }
            if (dt < kPreKeys / 4) ms.bad[slot][dt] = 0;
            if (dt == 0) ms.any_bad[slot] = 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms.dq[0]);
            if (!role_wait(&ms.dq[0], j & 1, abort_flag)) break;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                k_hi = max(k_hi, ms.red[i][0]);
                k_lo = min(k_lo, ms.red[i][1]);
                v_hi = max(v_hi, ms.red[i][2]);
                v_lo = min(v_lo, ms.red[i][3]);
            }
            const bool uneven = k_hi - k_lo > 6 || v_hi - v_lo > 6;
            // 2^-dk times the largest value is at most 2^-6
            const int dk = (uneven && ke != kNone ? ke : k_hi) + 6, dv = (uneven && ve != kNone ? ve : v_hi) + 6;
            {
                const float k24 = __uint_as_float((uint32_t)(127 + 24 - dk) << 23), v24 = __uint_as_float((uint32_t)(127 + 24 - dv) << 23);
                const uint32_t kdh = pack_f16x2(kd[0] * k24, kd[1] * k24), kmh = pack_f16x2(km[0] * k24 * 0x1p-24f, km[1] * k24 * 0x1p-24f);
                const uint32_t vdh = pack_f16x2(vd[0] * v24, vd[1] * v24), vmh = pack_f16x2(vm[0] * v24 * 0x1p-24f, vm[1] * v24 * 0x1p-24f);
                const uint32_t nan_k = (bad_k & 1 ? 0x7FFFu : 0u) | (bad_k & 2 ? 0x7FFF0000u : 0u);
                uint16_t *a = reinterpret_cast<uint16_t *>(smem + SM::kScale);
                constexpr int PART = kPreKeys * NG;
                const int g0 = part * NH;
#pragma unroll
                for (int i = 0; i < NH; ++i) {
                    a[key * NG + g0 + i] = (uint16_t)((kdh | nan_k) >> (16 * i));
                    a[PART + key * NG + g0 + i] = (uint16_t)(kmh >> (16 * i));
                    a[2 * PART + (g0 + i) * kPreKeys + key] = (uint16_t)(vdh >> (16 * i));
                    a[3 * PART + (g0 + i) * kPreKeys + key] = (uint16_t)(vmh >> (16 * i));
                    if (bad_v >> i & 1) {
                        atomicOr(&ms.bad[slot][key >> 2], (1u << (g0 + i)) << (8 * (key & 3)));
                        ms.any_bad[slot] = 1;
                    }
                }
                if (dt == 0) ms.uneven[slot] = uneven;
                if (part == 0 && (uneven || key == 0)) {
                    ms.k_fac[slot][key] = __uint_as_float((uint32_t)(127 + dk) << 23);
                    ms.v_exp[slot][key] = (float)dv;
                    ms.v_inv[slot][key] = ex2((float)-dv);
                }
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ms.dq[1]);
                mbar_arrive(&ms.m_full[slot]);
            }
            if (!role_wait(&ms.dq[1], j & 1, abort_flag)) break;
            const Raw now = raw;
            if (j + 1 < nt) load(j + 1);
            // ---- K: 16-byte chunks of 8 channels, [128 positions][64 channels] swizzled
            if (!role_wait(&ms.k_empty[st], wait_parity, abort_flag)) break;
            {
                const uint32_t k_row = base + SM::kK + st * SM::kKStage + key * 128;
                uint32_t dw_[NH], mw[NH];                           // this position's groups, in pairs
#pragma unroll
                for (int i = 0; i < NH; ++i) {
                    dw_[i] = lds32(s_kd + key * NG * 2 + 4 * i);
                    mw[i] = lds32(s_km + key * NG * 2 + 4 * i);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t sel = g & 1 ? 0x3232u : 0x1010u;
                    const uint32_t d24 = prmt(dw_[g >> 1], 0u, sel), m = prmt(mw[g >> 1], 0u, sel);
                    const uint32_t d20 = hmul2(d24, 0x2C002C00u);   // / 16
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t w = now.k[i][g], h = w >> 8;
                        const int c = g * 4 + 2 * part + i;         // chunk of the row
                        sts128(k_row + (c >> 3) * SM::kSubK + (((c ^ key) & 7) << 4), hfma2(w & 0x000F000Fu, d24, m),
                               hfma2(w & 0x00F000F0u, d20, m), hfma2(h & 0x000F000Fu, d24, m),
                               hfma2(h & 0x00F000F0u, d20, m));
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms.k_full[st]);
            // ---- V^T: 16-byte chunks of 8 positions, [D channels][64 positions] swizzled
            if (!role_wait(&ms.v_empty[st], wait_parity, abort_flag)) break;
            {
                const uint32_t v_tile = base + SM::kV + st * SM::kVStage + (vp >> 3) * SM::kSubV;
#pragma unroll
                for (int i = 0; i < NH; ++i) {
                    const int g = part * NH + i;
                    const uint4 d4 = lds128(s_vd + (g * kPreKeys + vp * 8) * 2), m4 = lds128(s_vm + (g * kPreKeys + vp * 8) * 2);
                    const uint32_t d24[4] = {d4.x, d4.y, d4.z, d4.w}, m[4] = {m4.x, m4.y, m4.z, m4.w};
                    uint32_t x[4][4];                               // [channel][position pair]
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t w = now.v[t][i], h = w >> 8, d20 = hmul2(d24[t], 0x2C002C00u);
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
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms.v_full[st]);
        }
    } else if (lane == 0) {
        // ------------------------------------------------------------ MMAs
        constexpr uint32_t id_s = umma_idesc_f16<kPreKeys>(), id_o = umma_idesc_f16<D>();
        bool ok = true;
        const auto qk = [&](int g, int j) {
            const uint32_t qa = base + g * SUBS * SM::kSubK, ka = base + SM::kK + (j & 1) * SM::kKStage;
#pragma unroll
            for (int s = 0; s < SUBS; ++s) {
                const uint64_t a = umma_desc_sw128(qa + s * SM::kSubK), bd = umma_desc_sw128(ka + s * SM::kSubK);
#pragma unroll
                for (int k = 0; k < 4; ++k)                         // 16 channels each: 32 bytes along the row
                    umma_f16_ss(tmem + g * 128, a + 2u * k, bd + 2u * k, id_s, (s | k) != 0);
            }
            umma_commit(&ms.s_full[g]);
        };
        for (int g = 0; g < groups && ok; ++g) ok = role_wait(&ms.q_ready[g], 0, abort_flag);
        ok = ok && role_wait(&ms.k_full[0], 0, abort_flag);
        if (ok) {
            tc_fence_after();
            for (int g = 0; g < groups; ++g) qk(g, 0);
            umma_commit(&ms.k_empty[0]);
        }
        for (int j = 0; j < nt && ok; ++j) {
            for (int g = 0; g < groups && ok; ++g) {
                if (g == 0) ok = role_wait(&ms.v_full[j & 1], (j >> 1) & 1, abort_flag);
                ok = ok && role_wait(&ms.p_full[g], j & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t va = base + SM::kV + (j & 1) * SM::kVStage;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint64_t bd = umma_desc_sw128(va + s * SM::kSubV);
#pragma unroll
                    for (int k = 0; k < 4; ++k)                     // 16 positions each: 8 columns of P
                        umma_f16_ts(tmem + 256 + g * D, tmem + g * 128 + 32 * s + 8 * k, bd + 2u * k, id_o,
                                    (j | s | k) != 0);
                }
                umma_commit(&ms.pv_done[g]);
                if (g == groups - 1) umma_commit(&ms.v_empty[j & 1]);
                if (j + 1 == nt) continue;
                // the next scores take the place of P: after its product is done
                if (g == 0) ok = role_wait(&ms.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, abort_flag);
                ok = ok && role_wait(&ms.pv_done[g], j & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                qk(g, j + 1);
                if (g == groups - 1) umma_commit(&ms.k_empty[(j + 1) & 1]);
            }
        }
        // nothing in flight when tensor memory goes
        umma_commit(&ms.drain);
        mbar_wait(&ms.drain, 0, &g_status);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512) : "memory");
    }
}

// The splits of the positions joined, one warp per row.
template <int D>
__global__ void __launch_bounds__(256) kv4_prefill_join_kernel(const __grid_constant__ PreParams pp) {
    constexpr int V = D / 32;
    const Kv4AttendParams &p = pp.a;
    griddep_launch_dependents();
    griddep_wait();
    const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);        // item * R + r
    const int lane = threadIdx.x & 31;
    if (at >= (int64_t)pp.items * p.R) return;
    const int64_t item = at / p.R;
    const int r = (int)(at - item * p.R);
    const auto slot = [&](int s) { return (item * pp.nsplit + s) * p.R + r; };
    float top = kNoMax;
    for (int s = lane; s < pp.nsplit; s += 32) top = fmaxf(top, p.part_ml[slot(s)].x);
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float acc[V], l = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 8
    for (int s = 0; s < pp.nsplit; ++s) {
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
    const int kvh = (int)(item - b * p.KV), tok = r / p.G, hh = r - tok * p.G;
    uint16_t *dst = p.out + ((b * p.T + tok) * p.H + kvh * p.G + hh) * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; i += 2)
        *reinterpret_cast<uint32_t *>(dst + i) = pack_bf16x2(acc[i] * inv, acc[i + 1] * inv);
}

// Splits of the positions: where there are fewer row tiles than SMs, at least
// two tiles of positions each.
static int prefill_splits(int64_t ctas, int64_t max_seq) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(148 / ctas, max_seq / (2 * kPreKeys)));
}

int64_t kv4_prefill_workspace(int64_t B, int64_t KV, int64_t R, int64_t D, int64_t max_seq) {
    const int64_t items = B * KV;
    const int n = prefill_splits(items * ((R + kPreRows - 1) / kPreRows), max_seq);
    return n == 1 ? 0 : items * n * R * (D * 4 + 8);
}

int kv4_prefill(Kv4AttendParams p, int64_t D, void *workspace, cudaStream_t st) {
    PreParams pp = {};
    pp.items = p.B * p.KV;
    pp.row_tiles = (p.R + kPreRows - 1) / kPreRows;
    const int64_t ctas = (int64_t)pp.items * pp.row_tiles;
    if (ctas > 0x7fffffffLL) return set_error(BF16X_ERR_UNSUPPORTED, "bf16x_kv4_attend: too many query rows");
    pp.nsplit = prefill_splits(ctas, p.max_seq);
    p.part_o = (float *)workspace;
    p.part_ml = (float2 *)((uint8_t *)workspace + (int64_t)pp.items * pp.nsplit * p.R * D * 4);
    pp.a = p;
    const dim3 grid((unsigned)ctas, (unsigned)pp.nsplit);
    const int rc = D == 64 ? launch_kv4<kv4_prefill_kernel<64>>(grid, kPreThreads, PreSmem<64>::kBytes, st, "kv4_prefill_kernel", pp)
                           : launch_kv4<kv4_prefill_kernel<128>>(grid, kPreThreads, PreSmem<128>::kBytes, st, "kv4_prefill_kernel", pp);
    if (rc != BF16X_OK || pp.nsplit == 1) return rc;
    const dim3 jgrid((unsigned)(((int64_t)pp.items * p.R + 7) / 8));
    return D == 64 ? launch_kv4<kv4_prefill_join_kernel<64>>(jgrid, 256, 0, st, "kv4_prefill_join_kernel", pp)
                   : launch_kv4<kv4_prefill_join_kernel<128>>(jgrid, 256, 0, st, "kv4_prefill_join_kernel", pp);
}

}  // namespace bf16x
