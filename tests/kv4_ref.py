"""The 4-bit cache in plain numpy/torch (64 bits, CPU), for the tests: every
code looked up by its place in the block (the layout of csrc/bf16x_kv4.cuh)."""
import math

import torch


def _up_bf16(x):
    """fp32 >= 0 -> the next bf16 at or above it, as fp32."""
    return ((x.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)


def quantize(x):
    """x [..., D] (bf16 values) -> codes (long), d, m (fp64) per group of 32; non-finite groups read as NaN."""
    g = x.float().unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    d = _up_bf16((hi - lo) / torch.full_like(hi, 15.0))
    q = torch.where(d > 0, torch.round((g - lo) / d), torch.zeros_like(g))
    bad = ~torch.isfinite(hi - lo)
    q = torch.where(bad, torch.zeros_like(q), q).clamp(0, 15)
    d = torch.where(bad, torch.full_like(d, math.nan), d)
    m = torch.where(bad, torch.zeros_like(lo), lo)
    return q.flatten(-2).long(), d.squeeze(-1).double(), m.squeeze(-1).double()


def value(q, d, m):
    return (q.double().unflatten(-1, (-1, 32)) * d[..., None] + m[..., None]).flatten(-2)


def unpack(blocks):
    """blocks (uint8 [B, KV, NB, 20 D]) -> (codes, d, m) of K and of V: [B, KV, 16 NB, D], [.., NG] fp64."""
    blocks = blocks.cpu()
    B, KV, NB, size = blocks.shape
    D = size // 20
    NG = D // 32
    r = torch.arange(16)[:, None]
    c = torch.arange(D)[None, :]
    j = c // 32
    nib = torch.stack((blocks & 15, blocks >> 4), -1).flatten(-2).long()             # [B, KV, NB, 40 D]
    kc = nib[..., ((r * 4 + c % 32 // 8) * NG + j) * 8 + c % 8]
    vc = nib[..., 16 * D + (((((r // 8) * 8 + c % 32 // 4) * 4 + r % 8 // 2) * NG + j) * 2 + r % 2) * 4 + c % 4]
    half = blocks.contiguous().view(torch.bfloat16).double()                          # [.., 10 D]
    jj = torch.arange(NG)[None, :]
    kd, km, vd = (half[..., (16 + i) * D // 2 + r * NG + jj] for i in range(3))
    vm = half[..., 19 * D // 2 + ((r // 2) * NG + jj) * 2 + r % 2]

    def flat(x):
        return x.reshape(B, KV, NB * 16, -1)

    return (flat(kc), flat(kd), flat(km)), (flat(vc), flat(vd), flat(vm))


def attend(q, blocks, pos0, scale, max_seq):
    """(out, bound) fp64 [B, T, H, D]: attention in 64 bits and what the kernels' roundings can add to it."""
    K, V = unpack(blocks)
    B, T, H, D = q.shape
    KV = blocks.shape[1]
    G = H // KV
    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    q = q.cpu().double()
    for b in range(B):
        for t in range(T):
            n = int(pos0[b]) + t + 1
            if n <= 0 or n > max_seq:
                continue
            for h in range(H):
                kv = h // G
                kc, kd, km = (a[b, kv, :n] for a in K)
                vc, vd, vm = (a[b, kv, :n] for a in V)
                k, v = value(kc, kd, km), value(vc, vd, vm)
                s = scale * (k @ q[b, t, h])
                p = torch.softmax(s, 0)
                o = p @ v
                mags = (kc.double().unflatten(-1, (-1, 32)) * kd[..., None] + km.abs()[..., None]).flatten(-2)
                # largest sum of magnitudes of a score: |scale q k| <= |scale| |q| |k|, whatever the scale's sign
                s_abs = abs(scale) * float((mags @ q[b, t, h].abs()).max())
                vmag = (vc.double().unflatten(-1, (-1, 32)) * vd[..., None] + vm.abs()[..., None]).flatten(-2)
                # bf16 result; the weights times the scales in fp16 (a half step 2^-11) and in two bf16 parts;
                # the scores' error in the exponent: fp32 sums of at most 40 terms and the final products
                out[b, t, h] = o
                bound[b, t, h] = 2.0 ** -8 * o.abs() + (p @ vmag) * (2.0 ** -11 + 2.0 ** -15 + 2.0 ** -17 * (1 + s_abs))
    return out, bound
