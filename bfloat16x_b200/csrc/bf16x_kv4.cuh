// bf16x_kv4.cuh -- the 4-bit key/value cache: its layout and the warp-level
// pieces shared by the kernels that write, read and attend to it.
//
// The cache of one layer is a byte array [batch][kv_heads][ceil(max_seq/16)]
// of blocks of 20 * D bytes.  A block holds 16 positions of one kv head.  Each
// group of 32 neighbouring channels of a position has a scale d >= 0 and a
// minimum m (bf16), and its 4-bit codes stand for d * code + m: 5 bits per
// value.  With NG = D / 32 groups, the parts of a block are
//
//   K codes  [16 r][4 t][NG j][8 n]          position r, channel 32 j + 8 t + n
//   V codes  [2 p][8 g][4 t][NG j][2 h][4 n] position 8 p + 2 t + h, channel 32 j + 4 g + n
//   K scales [16 r][NG], K minima [16 r][NG], V scales [16 r][NG]   bf16
//   V minima [8 pairs][NG][2]                bf16, positions 2 pair, 2 pair + 1
//
// The order is that of the mma.sync fragments: lane (g, t) = (lane / 4,
// lane % 4) of a warp reads its K codes of row g with one 16-byte access (D =
// 128) and its V codes of each half p with another, both contiguous over the
// warp.  A nibble that sits in bits 0..3 or 4..7 of a 16-bit half is, read as
// fp16, the subnormal number code * 2^-24 or code * 2^-20: exact, so one AND
// turns a packed pair of codes into a matrix operand, and the powers of two
// are taken out of the other operand (K) or of the sums (V).
#pragma once

#include <atomic>

#include "bf16x_common.cuh"
#include "bf16x_status.cuh"

namespace bf16x {

constexpr int kKvBlock = 16;                   // positions per block

template <int D>
struct KvLayout {
    static constexpr int NG = D / 32;
    static constexpr int kV = 8 * D;           // byte offset of each part
    static constexpr int kKd = 16 * D;
    static constexpr int kKm = 17 * D;
    static constexpr int kVd = 18 * D;
    static constexpr int kVm = 19 * D;
    static constexpr int kBytes = 20 * D;
};

__device__ __forceinline__ float fmin_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float fmax_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float lg2(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// bf16 in the low / high half of a word, as fp32
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// D[16][8] = A[16][16] B[16][8] + C, fp32 sums
#define BF16X_MMA(NAME, TYPE)                                                                                         \
    __device__ __forceinline__ void NAME(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,           \
                                         uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {          \
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "     \
                     "{%8,%9}, {%10,%11,%12,%13};"                                                                    \
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                 \
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));     \
    }                                                                                                                 \
    __device__ __forceinline__ void NAME(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,           \
                                         uint32_t b0, uint32_t b1) {                                                  \
        NAME(c, a0, a1, a2, a3, b0, b1, c[0], c[1], c[2], c[3]);                                                      \
    }
BF16X_MMA(mma_f16, "f16")
BF16X_MMA(mma_bf16, "bf16")
#undef BF16X_MMA

// transposed 8x8 tile of 16-bit values: row g, columns 2t, 2t+1 -> row 2t.. as column
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}

// shared-memory loads by 32-bit address
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
    return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 r;
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
    return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
    return r;
}

// Arguments of the attention kernels.  Rows of one kv head: r = t * G + h.
struct Kv4AttendParams {
    const uint16_t *q;
    int64_t ldq_b, ldq_t, ldq_h;
    int B, T, H, KV, G, R;
    int pos_stride, tiles, warps;       // row tiles per head; warps of the grid
    int few_units;                      // a unit has the shares of several CTAs
    const int64_t *pos0;
    float scale_log2;                   // softmax scale * log2(e)
    const uint8_t *blocks;
    int64_t max_seq, nblk;
    uint16_t *out;
    float *part_o;                      // [share][2][row of the tile][D]
    float2 *part_ml;                    // [share][2][row of the tile]
    int2 *held;                         // [unit]: the first and last share that hold blocks of it
};

// A row's reference M is kept so that its largest term P dV is 2^kRefTerm when M
// is set and at most 2^kRescale before it is raised: fp16 is used from the top, so
// that a term of 2^-25 of the largest still has its 11 bits, and a long tail of
// smaller ones (2^17 positions) is off by 2^-19 of the largest at most.
constexpr float kRefTerm = 11.f, kRescale = 15.f;
constexpr float kNoMax = -3.0e38f;

// Launch as a programmatic dependent of the previous kernel of the stream.  The
// shared-memory limit of a kernel is raised once per device.
template <auto Kern, typename P>
static int launch_kv4(dim3 grid, unsigned block, size_t smem, cudaStream_t st, const char *what, const P &params) {
    cudaError_t e;
    if (smem > 48 * 1024) {
        static std::atomic<uint64_t> raised{0};
        int dev = 0;
        e = cudaGetDevice(&dev);
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (e == cudaSuccess && !(raised.load(std::memory_order_relaxed) & bit)) {
            e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e == cudaSuccess) raised.fetch_or(bit, std::memory_order_relaxed);
        }
        if (e != cudaSuccess) return set_error(BF16X_ERR_CUDA, "%s: shared memory: %s", what, cudaGetErrorString(e));
    }
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
    e = cudaLaunchKernelEx(&cfg, Kern, params);
    if (e != cudaSuccess) return set_error(BF16X_ERR_CUDA, "%s: launch: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

// Attention of many rows per kv head (bf16x_kv4_prefill.cu): its workspace, and its launch.
int64_t kv4_prefill_workspace(int64_t B, int64_t KV, int64_t R, int64_t T, int64_t D, int64_t max_seq);
int kv4_prefill(Kv4AttendParams p, int64_t D, void *workspace, cudaStream_t st);

}  // namespace bf16x
