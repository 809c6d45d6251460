"""Cases of the decoder's serving operators: writing keys and values into a
4-bit cache, attention over that cache, and drawing the next token.

``run`` computes one pass, either in a plain form (elementary torch operations
in 32 bits, 64 where it matters) or, where ``own`` is true, through the
framework's entry points; ``exact`` says what the pass is in 64 bits.

The 4-bit cache is one uint8 tensor ``blocks`` [batch, kv_heads, max_seq / 16,
20 * head_dim].  A block holds 16 positions of one head.  Each group of 32
neighbouring channels of a position has a scale d and a minimum m (bf16) and
stands for d * code + m.  With NG = head_dim / 32 the parts of a block are

    K codes   [16 positions][4 t][NG groups][8 n]     4 bits, channel 32 group + 8 t + n
    V codes   [2 p][8 g][4 t][NG groups][2 h][4 n]    4 bits, position 8 p + 2 t + h, channel 32 group + 4 g + n
    K scales  [16][NG] bf16,  K minima [16][NG] bf16
    V scales  [16][NG] bf16,  V minima [8 pairs][NG][2 of a pair] bf16

(the order in which a warp's matrix fragments take them).
"""
from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 16
GROUP = 32


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's cache write at batch 1 (the 1B decoder's heads): latency
        dict(name="append-step-b1", op="append", batch=1, tokens=1, heads=16, kv_heads=8, head_dim=128,
             first=1000, step=0, max_seq=2048),
        # a batch of prompts entering the cache at uneven positions (the 8B decoder's heads)
        dict(name="append-prompt-b4", op="append", batch=4, tokens=2047, heads=32, kv_heads=8, head_dim=128,
             first=5, step=131, max_seq=4096),
        # single-stream decoding early in a conversation (the 1B decoder's heads): latency
        dict(name="decode-b1-short", op="attend", batch=1, tokens=1, heads=16, kv_heads=8, head_dim=128,
             shortest=300, longest=300),
        # single-stream decoding over a long document (the 8B decoder's heads)
        dict(name="decode-b1-long", op="attend", batch=1, tokens=1, heads=32, kv_heads=8, head_dim=128,
             shortest=131071, longest=131071),
        # a serving batch of sequences of very different lengths
        dict(name="decode-b16-ragged", op="attend", batch=16, tokens=1, heads=32, kv_heads=8, head_dim=128,
             shortest=17, longest=16384),
        # four guessed tokens checked at once, with the small decoder's head size
        dict(name="verify-b8-t4-d64", op="attend", batch=8, tokens=4, heads=32, kv_heads=8, head_dim=64,
             shortest=900, longest=5001),
        # a whole prompt (the prefill benchmark's 2048 tokens, the 8B decoder's heads)
        dict(name="prefill-b1-t2048", op="attend", batch=1, tokens=2048, heads=32, kv_heads=8, head_dim=128,
             shortest=2048, longest=2048),
        # a later chunk of a long prompt, left-padded in the shortest sequence, without head sharing at 64 channels
        dict(name="prefill-b3-chunk-d64", op="attend", batch=3, tokens=511, heads=8, kv_heads=8, head_dim=64,
             shortest=333, longest=7003),
        # one token of one stream: all filters, logits on the bf16 grid of the projection (the 8B decoder's vocabulary)
        dict(name="sample-b1-filters", op="sample", batch=1, vocab=128256, dtype="bfloat16", temperature=0.8,
             top_k=50, top_p=0.95, min_p=0.02, mixed=False),
        # a serving batch in which every sequence has its own settings
        dict(name="sample-b16-mixed", op="sample", batch=16, vocab=128256, dtype="float32", temperature=1.0,
             top_k=0, top_p=1.0, min_p=0.0, mixed=True),
        # many short samples with top-p only (the 1B decoder's vocabulary, an odd batch)
        dict(name="sample-b129-top-p", op="sample", batch=129, vocab=73448, dtype="float32", temperature=1.1,
             top_k=0, top_p=0.9, min_p=0.0, mixed=False),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng: random.Random):
    kind = rng.choice(("append", "decode", "decode", "prefill", "sample", "sample"))
    kv_heads, group = rng.choice(((8, 4), (8, 2), (8, 1), (2, 2), (1, 8), (4, 3), (2, 16)))
    head_dim = rng.choice((64, 128, 128))
    heads = dict(heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim)
    if kind == "append":
        batch = _log_int(rng, 1, 16)
        tokens = _log_int(rng, 1, max(1, 8000 // batch))
        first, step = rng.randint(-3, 300), rng.randint(0, 60)
        room = max(1, first + step * (batch - 1) + tokens)
        return dict(op="append", batch=batch, tokens=tokens, first=first, step=step,
                    max_seq=room + rng.randint(0, 40), **heads)
    if kind == "decode":
        batch, tokens = _log_int(rng, 1, 32), rng.choice((1, 1, 1, 2, 5))
        longest = _log_int(rng, tokens, min(131072, 262144 // batch))
        return dict(op="attend", batch=batch, tokens=tokens, shortest=rng.randint(0, longest), longest=longest, **heads)
    if kind == "prefill":
        batch = _log_int(rng, 1, 4)
        tokens = _log_int(rng, 33, 2048 // batch)
        longest = tokens + rng.choice((0, _log_int(rng, 1, 6000 // batch)))
        return dict(op="attend", batch=batch, tokens=tokens, shortest=rng.randint(1, longest), longest=longest, **heads)
    return dict(op="sample", batch=_log_int(rng, 1, 128), vocab=_log_int(rng, 1000, 128256),
                dtype=rng.choice(("float32", "bfloat16")), temperature=round(rng.uniform(0.3, 1.5), 3),
                top_k=rng.choice((0, 1, 40, 1000)), top_p=rng.choice((1.0, 0.95, 0.6)),
                min_p=rng.choice((0.0, 0.05)), mixed=rng.random() < 0.3)


def _spread(case, lo, hi):
    """One whole number per sequence, evenly from lo to hi."""
    n = case["batch"]
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case):
    return _spread(case, case["shortest"], case["longest"])


def work(case):
    if case["op"] == "append":
        tok = case["batch"] * case["tokens"]
        d, kv, h = case["head_dim"], case["kv_heads"], case["heads"]
        # the projections, the angles, the rotated queries, the 4-bit rows, and the rows read back (4 bits in, bf16 out)
        row = 5 * d // 4
        bytes_ = tok * (2 * d * (h + 2 * kv) + 4 * d + 2 * d * h + 2 * kv * row + 4 * d * kv)
        return {"bytes": bytes_, "flops": tok * d * (3 * (h + kv) + 6 * 2 * kv)}
    if case["op"] == "attend":
        d, kv, h, t = case["head_dim"], case["kv_heads"], case["heads"], case["tokens"]
        pairs = keys = 0
        for n in _lengths(case):
            keys += max(n, 0)
            seen = min(t, max(n, 0))                               # queries at positions n - seen .. n - 1
            pairs += seen * (2 * n - seen + 1) // 2
        bytes_ = keys * kv * (5 * d // 4) + 4 * case["batch"] * t * h * d
        return {"bytes": bytes_, "flops": 4 * pairs * h * d}
    size = 2 if case["dtype"] == "bfloat16" else 4
    return {"bytes": case["batch"] * (case["vocab"] * size + 4 + 8), "flops": 4 * case["batch"] * case["vocab"]}


# -------------------------------------------------------------------- inputs
def _quantize(x):
    """x [..., channels] bf16 values (fp32) -> codes, scales, minima of its groups of 32."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    d = (hi - lo) / torch.full_like(hi, 15.0)      # a true division: a product with 1/15 can miss an exact quotient
    d = ((d.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)      # up to the next bf16: no code above 15
    q = torch.where(d > 0, torch.round((g - lo) / d), torch.zeros_like(g)).clamp(0, 15)
    return q.flatten(-2).to(torch.uint8), d.squeeze(-1), lo.squeeze(-1)


def _pack(kq, kd, km, vq, vd, vm):
    """Codes [B, H, S, D] and scales, minima [B, H, S, NG] -> blocks [B, H, S/16, 20 D]."""
    B, H, S, D = kq.shape
    ng, nb = D // GROUP, S // BLOCK

    def nibbles(x):
        x = x.reshape(B, H, nb, -1, 2)
        return x[..., 0] | (x[..., 1] << 4)

    k = nibbles(kq.view(B, H, nb, 16, ng, 4, 8).transpose(4, 5).contiguous())
    v = nibbles(vq.view(B, H, nb, 2, 4, 2, ng, 8, 4).permute(0, 1, 2, 3, 7, 4, 6, 5, 8).contiguous())

    def raw(x):
        return x.to(torch.bfloat16).contiguous().view(torch.uint8).reshape(B, H, nb, -1)

    vmin = vm.view(B, H, nb, 8, 2, ng).transpose(4, 5)
    return torch.cat([k, v, raw(kd), raw(km), raw(vd), raw(vmin)], -1).contiguous()


def _generator(case, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _keys_values(case, seq, g):
    """Keys with a few strong channels, as rotated keys have them, and values; bf16 values in fp32."""
    B, KV, D = case["batch"], case["kv_heads"], case["head_dim"]
    loud = 1.0 + 3.0 * (torch.rand(KV, 1, D, generator=g, device="cuda") > 0.95)
    shift = torch.randn(KV, 1, D, generator=g, device="cuda") * 0.5
    k = torch.randn(B, KV, seq, D, generator=g, device="cuda") * loud + shift
    v = torch.randn(B, KV, seq, D, generator=g, device="cuda") * 0.7
    return k.to(torch.bfloat16).float(), v.to(torch.bfloat16).float()


def prepare(case, seed):
    g = _generator(case, seed)
    B = case["batch"]
    if case["op"] == "sample":
        V, dt = case["vocab"], getattr(torch, case["dtype"])
        # a few likely tokens over a broad floor; rounded to bf16 as the projection gives them
        x = torch.randn(B, V, generator=g, device="cuda") * 2.2
        hot = torch.randint(0, V, (B, 24), generator=g, device="cuda")
        x.scatter_add_(1, hot, torch.rand(B, 24, generator=g, device="cuda") * 9.0)
        x = x.to(torch.bfloat16).to(dt) if case["mixed"] or case["dtype"] == "bfloat16" else x.to(dt)
        u = torch.rand(B, generator=g, device="cuda")
        s = {"op": "sample", "logits": x, "u": u}
        for name, t in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32),
                        ("min_p", torch.float32)):
            if case["mixed"]:
                pool = {"temperature": (1.0, 0.7, 0.0, 1.3), "top_k": (0, 20, 0, 400, 1), "top_p": (1.0, 0.9, 0.5),
                        "min_p": (0.0, 0.1)}[name]
                s[name] = torch.tensor([pool[i % len(pool)] for i in range(B)], dtype=t, device="cuda")
            else:
                s[name] = case[name]
        return s
    H, KV, D, T = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
    if case["op"] == "append":
        S = case["max_seq"]
        qkv = torch.randn(B, T, (H + 2 * KV) * D, generator=g, device="cuda").to(torch.bfloat16)
        inv = 1.0 / (500000.0 ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float32) / D))
        f = torch.outer(torch.arange(S, device="cuda", dtype=torch.float32), inv)
        pos0 = torch.tensor([case["first"] + case["step"] * b for b in range(B)], dtype=torch.long, device="cuda")
        blocks = torch.zeros(B, KV, -(-S // BLOCK), 20 * D, dtype=torch.uint8, device="cuda")
        return {"op": "append", "qkv": qkv, "cos": torch.cos(f), "sin": torch.sin(f), "pos0": pos0, "blocks": blocks,
                "heads": H, "max_seq": S, "tokens": T}
    lengths = _lengths(case)
    S = -(-max(max(lengths), 1) // BLOCK) * BLOCK
    k, v = _keys_values(case, S, g)
    blocks = _pack(*_quantize(k), *_quantize(v))
    q = (torch.randn(B, T, H, D, generator=g, device="cuda") * 1.3).to(torch.bfloat16)
    pos0 = torch.tensor([n - T for n in lengths], dtype=torch.long, device="cuda")
    return {"op": "attend", "q": q, "pos0": pos0, "blocks": blocks, "max_seq": S}


# -------------------------------------------------------------- plain forms
def _unpack(blocks):
    """blocks -> K and V [B, H, S, D] in fp32, the values that they stand for."""
    B, H, nb, size = blocks.shape
    D = size // 20
    ng = D // GROUP

    def nibbles(x):
        return torch.stack((x & 15, x >> 4), -1).flatten(-2)

    def half(x):
        return x.contiguous().view(torch.bfloat16).float()

    k = nibbles(blocks[..., :8 * D]).view(B, H, nb, 16, 4, ng, 8).transpose(4, 5)
    v = nibbles(blocks[..., 8 * D:16 * D]).view(B, H, nb, 2, 8, 4, ng, 2, 4).permute(0, 1, 2, 3, 5, 7, 6, 4, 8)
    kd, km, vd = (half(blocks[..., (16 + i) * D:(17 + i) * D]).view(B, H, nb, 16, ng, 1, 1) for i in range(3))
    vm = half(blocks[..., 19 * D:]).view(B, H, nb, 8, ng, 2).transpose(4, 5).reshape(B, H, nb, 16, ng, 1, 1)
    k = k.float() * kd + km
    v = v.reshape(B, H, nb, 16, ng, 8, 4).float() * vd + vm
    return k.reshape(B, H, nb * 16, D), v.reshape(B, H, nb * 16, D)


def _plain_append(s):
    qkv, T, S = s["qkv"], s["tokens"], s["max_seq"]
    B, KV = s["blocks"].shape[:2]
    D = s["blocks"].shape[3] // 20
    H = s["heads"]
    pos = s["pos0"][:, None] + torch.arange(T, device=qkv.device)
    inside = (pos >= 0) & (pos < S)
    at = pos.clamp(0, S - 1)
    c, n = s["cos"][at][:, :, None, :], s["sin"][at][:, :, None, :]
    x = qkv.float().view(B, T, H + 2 * KV, D)
    x1, x2 = x[:, :, :H + KV, 0::2], x[:, :, :H + KV, 1::2]
    r = torch.stack((x1 * c - x2 * n, x1 * n + x2 * c), -1).flatten(-2).to(torch.bfloat16)
    q = torch.where(inside[:, :, None, None], r[:, :, :H], torch.zeros((), dtype=r.dtype, device=r.device))
    out = [q]
    for y in (r[:, :, H:].float(), x[:, :, H + KV:]):
        codes, d, m = _quantize(y)
        y = codes.float().unflatten(-1, (-1, GROUP)) * d[..., None] + m[..., None]
        out.append(torch.where(inside[:, :, None, None], y.flatten(-2), torch.zeros_like(m[..., :1])).to(torch.bfloat16))
    return {"q": out[0], "k": out[1], "v": out[2]}


def _plain_attend(s):
    q, pos0 = s["q"], s["pos0"]
    B, T, H, D = q.shape
    k, v = _unpack(s["blocks"])
    KV, S = k.shape[1], k.shape[2]
    pos = pos0[:, None] + torch.arange(T, device=q.device)
    seen = torch.arange(S, device=q.device) <= pos[:, :, None]                  # [B, T, S]
    qg = q.float().view(B, T, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, D)
    x = torch.matmul(qg, k.transpose(-1, -2)).view(B, KV, H // KV, T, S) / math.sqrt(D)
    x = x.masked_fill(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, torch.ones_like(total))).view(B, KV, -1, S)
    o = torch.matmul(p, torch.where(seen.any(1)[:, None, :, None], v, torch.zeros((), device=v.device)))
    return o.view(B, KV, H // KV, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(q.dtype)


def _row(x, like, dtype):
    return x if isinstance(x, torch.Tensor) else torch.full((like.shape[0],), x, dtype=dtype, device=like.device)


def _plain_sample(s):
    x = s["logits"].double()
    B, V = x.shape
    t = _row(s["temperature"], x, torch.float32).double()[:, None]
    kk = _row(s["top_k"], x, torch.int32).long()[:, None]
    pp = _row(s["top_p"], x, torch.float32).double()[:, None]
    mp = _row(s["min_p"], x, torch.float32).double()[:, None]
    srt, idx = torch.sort(x, dim=1, descending=True, stable=True)
    top = srt[:, :1]
    w = torch.where(srt == top, torch.ones_like(srt), torch.exp((srt - top) / torch.where(t > 0, t, torch.ones_like(t))))
    rank = torch.arange(V, device=x.device)[None]
    keep = (kk <= 0) | (rank < kk)
    w = w * keep
    cum = torch.cumsum(w, 1)
    keep &= (pp >= 1) | (cum - w < pp * cum[:, -1:])
    keep &= w >= mp
    keep[:, 0] = True
    keep &= (t > 0) | (rank == 0)
    w = torch.zeros_like(w).scatter_(1, idx, w * keep)
    cum = torch.cumsum(w, 1)
    target = s["u"].double()[:, None] * cum[:, -1:]
    return (cum <= target).sum(1)


def run(state):
    if state["op"] == "append":
        if not own:
            return _plain_append(state)
        from bfloat16x_b200.kv4 import Kv4Cache
        cache = Kv4Cache(state["blocks"], state["max_seq"])
        q = cache.append(state["qkv"], state["pos0"], state["heads"], state["cos"], state["sin"])
        k, v = cache.read(state["pos0"], state["tokens"])
        return {"q": q, "k": k, "v": v}
    if state["op"] == "attend":
        if not own:
            return _plain_attend(state)
        from bfloat16x_b200.kv4 import Kv4Cache
        return Kv4Cache(state["blocks"], state["max_seq"]).attend(state["q"], state["pos0"])
    if not own:
        return _plain_sample(state)
    from bfloat16x_b200.sampling import sample
    return sample(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                  top_p=state["top_p"], min_p=state["min_p"])


# --------------------------------------------------- the definition, 64 bits
def _exact_rows(blocks, b, h, count):
    """K and V [count, D] of one head in fp64, each value looked up by its place in the block."""
    D = blocks.shape[3] // 20
    ng = D // 32
    dev = blocks.device
    i = torch.arange(count, device=dev)[:, None]
    c = torch.arange(D, device=dev)[None, :]
    flat = blocks[b, h].reshape(-1)
    base, r, grp = (i // 16) * (20 * D), i % 16, c // 32

    def code(part, place):
        byte = flat[base + part + place // 2].long()
        return torch.where(place % 2 == 0, byte % 16, byte // 16).double()

    half = flat.view(torch.bfloat16)

    def number(part, place):
        return half[(base + part) // 2 + place].double()

    kc = code(0, ((r * 4 + (c % 32) // 8) * ng + grp) * 8 + c % 8)
    pair = r // 2
    vc = code(8 * D, (((((r // 8) * 8 + (c % 32) // 4) * 4 + pair % 4) * ng + grp) * 2 + r % 2) * 4 + c % 4)
    k = kc * number(16 * D, r * ng + grp) + number(17 * D, r * ng + grp)
    v = vc * number(18 * D, r * ng + grp) + number(19 * D, (pair * ng + grp) * 2 + r % 2)
    return k, v


def _exact_attend(case, s):
    q = s["q"].double()
    B, T, H, D = q.shape
    KV = case["kv_heads"]
    G = H // KV
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=q.device)
    for b, n in enumerate(_lengths(case)):
        if n <= 0:
            continue
        pos = torch.arange(n - T, n, device=q.device)
        live = (pos >= 0).nonzero()[:, 0]
        for h in range(KV):
            k, v = _exact_rows(s["blocks"], b, h, n)
            for t in live.split(512):
                x = torch.einsum("tgd,nd->tgn", q[b, t, h * G:(h + 1) * G], k) / math.sqrt(D)
                x.masked_fill_((torch.arange(n, device=q.device)[None] > pos[t][:, None])[:, None], -math.inf)
                out[b, t, h * G:(h + 1) * G] = torch.softmax(x, -1) @ v
    return out


def _exact_append(case, s):
    B, T, H, KV, D = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    x = s["qkv"].double().view(B, T, H + 2 * KV, D)
    q = torch.zeros(B, T, H, D, dtype=torch.float64, device=x.device)
    k, v = torch.zeros(B, T, KV, D, dtype=torch.float64, device=x.device), None
    v = torch.zeros_like(k)
    for b in range(B):
        p0 = case["first"] + case["step"] * b
        t = torch.tensor([i for i in range(T) if 0 <= p0 + i < case["max_seq"]], device=x.device, dtype=torch.long)
        angle = torch.complex(s["cos"][p0 + t].double(), s["sin"][p0 + t].double())[:, None]
        turned = torch.view_as_real(torch.view_as_complex(x[b, t, :H + KV].unflatten(-1, (-1, 2)).contiguous()) * angle)
        turned = turned.flatten(-2)
        q[b, t] = turned[:, :H]
        for y, to in ((turned[:, H:].to(torch.bfloat16).double(), k), (x[b, t, H + KV:], v)):
            y = y.unflatten(-1, (-1, 32))
            low = y.min(-1, keepdim=True).values
            span = y.max(-1, keepdim=True).values - low
            span = span / torch.full_like(span, 15.0)
            e = torch.floor(torch.log2(torch.where(span > 0, span, torch.ones_like(span)))) - 7
            d = torch.ceil(span * torch.exp2(-e)) * torch.exp2(e)             # eight significant bits, upwards
            y = torch.where(d > 0, torch.round((y - low) / torch.where(d > 0, d, torch.ones_like(d))) * d, 0.0) + low
            to[b, t] = y.flatten(-2)
    return {"q": q, "k": k, "v": v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    return None        # tokens are whole numbers: equal or not
