"""The 4-bit key/value cache on the GPU: writing (codes bit for bit), reading
back and attention, against plain 64-bit formulas on the CPU."""
import pytest
import torch

from bfloat16x_b200 import _lib
from bfloat16x_b200.kv4 import Kv4Cache, kv4_blocks
from bfloat16x_b200.llama_e2e import _rope_tables
from tests import kv4_ref

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _filled(B, KV, D, S, seed, k_scale=1.0, v_scale=1.0, stale=False):
    """A cache of S random positions (written by append); stale: random bytes first, as an earlier use leaves them."""
    g = _gen(seed)
    cache = Kv4Cache.empty(B, S, KV, D, "cuda")
    if stale:
        cache.blocks.copy_(torch.randint(0, 256, cache.blocks.shape, generator=g, dtype=torch.uint8))
    kv = torch.randn(B, S, 2 * KV, D, generator=g)
    kv[:, :, :KV] *= k_scale
    kv[:, :, :KV] += 0.5 * torch.randn(KV, D, generator=g)
    kv[:, :, KV:] *= v_scale
    qkv = kv.to(torch.bfloat16).reshape(B, S, -1).cuda()
    cache.append(qkv, torch.zeros(1, dtype=torch.long, device="cuda"), 0)
    return cache


def _check(cache, q, pos0, scale=None, out=None):
    got = cache.attend(q.cuda() if not q.is_cuda else q, pos0.cuda(), scale)
    assert got.dtype == torch.bfloat16 and got.shape == q.shape
    B = q.shape[0]
    p = pos0.reshape(-1).tolist()
    p = p * B if len(p) == 1 else p
    ref, bound = kv4_ref.attend(q, cache.blocks, p, q.shape[3] ** -0.5 if scale is None else scale, cache.max_seq)
    err = (got.cpu().double() - ref).abs()
    assert bool((err <= bound + 1e-30).all()), f"off by {float((err - bound).max())} over the bound"
    return got


# ------------------------------------------------------------------ write, read
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,H,KV,S,pos", [(1, 1, 4, 2, 5, [4]), (1, 37, 2, 1, 60, [11]), (3, 18, 6, 2, 64, [0, 13, -7]),
                                            (2, 1, 1, 1, 33, [15, 16]), (2, 5, 0, 3, 40, [-9, 35])])
def test_append_and_read(D, B, T, H, KV, S, pos):
    g = _gen(100 * D + T)
    qkv = (torch.randn(B, T, (H + 2 * KV) * D, generator=g) * torch.rand(B, T, 1, generator=g).exp2()).to(torch.bfloat16)
    cos, sin = _rope_tables(D, S + 3, 10000.0, "cpu")
    cache = Kv4Cache.empty(B, S, KV, D, "cuda")
    cache.blocks.fill_(0xA5)
    before = cache.blocks.clone()
    p0 = torch.tensor(pos, dtype=torch.long)
    q = cache.append(qkv.cuda(), p0.cuda(), H, cos.cuda(), sin.cuda())
    k, v = cache.read(p0.cuda(), T)
    _lib.check_device_status()
    K, V = kv4_ref.unpack(cache.blocks)
    written = torch.zeros(B, cache.blocks.shape[2] * 16, dtype=torch.bool)
    for b in range(B):
        for t in range(T):
            at = pos[b] + t
            if at < 0:
                assert not q[b, t].any() and not k[b, t].any() and not v[b, t].any()
                continue
            written[b, at] = True
            x = qkv[b, t].float().view(H + 2 * KV, D)
            x1, x2 = x[:H + KV, 0::2], x[:H + KV, 1::2]
            y = torch.stack((x1 * cos[at] - x2 * sin[at], x1 * sin[at] + x2 * cos[at]), -1).flatten(-2).to(torch.bfloat16)
            assert torch.equal(q[b, t].cpu(), y[:H])
            for part, ref, back in ((K, y[H:], k), (V, x[H + KV:], v)):
                c, d, m = kv4_ref.quantize(ref)
                assert torch.equal(part[0][b, :, at], c)
                assert torch.equal(part[1][b, :, at], d) and torch.equal(part[2][b, :, at], m)
                assert torch.equal(back[b, t].cpu(), kv4_ref.value(c, d, m).float().to(torch.bfloat16))
    # every other position of the cache as it was
    K0, V0 = kv4_ref.unpack(before)
    for new, old in zip(K + V, K0 + V0):
        assert torch.equal(new.transpose(1, 2)[~written].nan_to_num(7.0), old.transpose(1, 2)[~written].nan_to_num(7.0))


def test_append_special_values():
    """Constant groups, the largest values, denormals; an infinity or NaN makes its group NaN and no other."""
    D = 64
    x = torch.randn(1, 6, 2 * D, generator=_gen(3))
    x[0, 0, :32] = 3.25
    x[0, 1, 32:64] = 0.0
    x[0, 2, :32] = torch.linspace(-1.5e38, 1.5e38, 32)
    x[0, 2, 32:64] *= 1e-39
    x[0, 3, 5] = float("inf")
    x[0, 4, 70] = float("nan")
    x[0, 5, 100] = float("-inf")
    x = x.to(torch.bfloat16)
    cache = Kv4Cache.empty(1, 6, 1, D, "cuda")
    zero = torch.zeros((), dtype=torch.long, device="cuda")
    cache.append(x.cuda(), zero, 0)
    k, v = cache.read(zero, 6)
    for got, ref in ((k, x[0, :, :D]), (v, x[0, :, D:])):
        want = kv4_ref.value(*kv4_ref.quantize(ref))
        got = got[0, :, 0].cpu().double()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0), want.float().to(torch.bfloat16).double().nan_to_num(0.0))
    assert int(k.isnan().sum()) == 32 and int(v.isnan().sum()) == 64


def test_append_strided_and_unaligned_input():
    D, KV, H = 64, 2, 2
    g = _gen(5)
    wide = torch.randn(2, 7, 3 * (H + 2 * KV) * D + 3, generator=g).to(torch.bfloat16).cuda()
    n = (H + 2 * KV) * D
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    for view in (wide[:, :, 8:8 + n], wide[:, :, 3:3 + n], wide[:, ::2, n:2 * n], wide[:, :, :n].transpose(0, 1)[:2]):
        if view.shape[0] != 2:
            continue
        a, b = Kv4Cache.empty(2, 7, KV, D, "cuda"), Kv4Cache.empty(2, 7, KV, D, "cuda")
        qa, qb = a.append(view, zero, H), b.append(view.contiguous().clone(), zero, H)
        assert torch.equal(qa, qb) and torch.equal(a.blocks, b.blocks)


def test_position_past_the_cache_is_reported():
    D, KV = 64, 1
    cache = Kv4Cache.empty(1, 20, KV, D, "cuda")
    x = torch.randn(1, 3, 3 * D, generator=_gen(6)).to(torch.bfloat16).cuda()
    p = torch.tensor([18], device="cuda")
    q = cache.append(x, p, 1)
    assert _lib.device_status() & 16
    assert q[0, :2].any() and not q[0, 2].any()
    k, _ = cache.read(p, 3)
    assert _lib.device_status() & 16
    assert k[0, 1].any() and not k[0, 2].any()
    o = cache.attend(x.view(1, 3, 3, D), p)
    assert _lib.device_status() & 16
    assert o[0, 1].any() and not o[0, 2].any()


# ---------------------------------------------------------------------- attend
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KV", [(1, 1), (4, 4), (8, 2), (6, 2), (8, 1), (17, 1), (48, 2)])
def test_attend_single_token(D, H, KV):
    for n in (1, 2, 15, 16, 17, 33, 200):
        cache = _filled(2, KV, D, n + 5, seed=n, stale=True)
        q = torch.randn(2, 1, H, D, generator=_gen(n + H)).to(torch.bfloat16)
        _check(cache, q, torch.tensor([n - 1, n // 2]))
    _lib.check_device_status()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,H,KV,pos", [(2, 4, 2, [0, 30]), (5, 4, 1, [-2, 91]), (3, 8, 8, [-3, -1]), (9, 6, 2, [7, 64]),
                                        (40, 4, 2, [-20, 50]), (33, 1, 1, [0, 0]), (70, 5, 1, [1, 26])])
def test_attend_many_tokens(D, T, H, KV, pos):
    cache = _filled(2, KV, D, 100, seed=T, stale=True)
    q = torch.randn(2, T, H, D, generator=_gen(T + D)).to(torch.bfloat16)
    _check(cache, q, torch.tensor(pos))
    _lib.check_device_status()


@pytest.mark.parametrize("B,T,H,KV,S,pos", [
    (20, 64, 32, 8, 64, (0, 0)),            # more units of rows than CTAs, each row tile whole
    (40, 75, 8, 2, 120, (-75, 44)),         # two row tiles, the last with few rows; sequences that see nothing
    (20, 64, 32, 8, 400, (-64, 336)),       # a long cache, units cut between CTAs
    (3, 130, 4, 2, 1500, (-130, 1370)),     # few units, very different lengths
    (3, 50, 4, 2, 3000, (-3, 2950)),        # units of one group of rows
    (1, 130, 1, 1, 4500, (4370, 4370)),
    (2, 520, 2, 1, 2000, (1, 1480))])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_schedules(D, B, T, H, KV, S, pos):
    cache = _filled(B, KV, D, S, seed=T + S, stale=True)
    q = torch.randn(B, T, H, D, generator=_gen(T + B)).to(torch.bfloat16)
    _check(cache, q, torch.linspace(pos[0], pos[1], B).round().long())
    _lib.check_device_status()


@pytest.mark.parametrize("n", [1000, 4099])
@pytest.mark.parametrize("T", [1, 3, 150])
def test_attend_long(n, T):
    if T == 150 and n > 1000:
        n = 1500
    D, H, KV = 128, 4, 1
    cache = _filled(1, KV, D, n + T, seed=n, k_scale=1.5)
    q = (torch.randn(1, T, H, D, generator=_gen(n)) * 1.5).to(torch.bfloat16)
    _check(cache, q, torch.tensor(n))


@pytest.mark.parametrize("D,T,H,KV,pos", [(64, 1, 4, 2, [80001]), (64, 1, 3, 1, [70000, 90000]), (128, 1, 8, 8, [20479]),
                                          (128, 1, 1, 1, [-1, 150000, 17]), (64, 3, 4, 1, [99990]), (128, 4, 12, 3, [35000, 4])])
def test_attend_few_sequences_of_many_blocks(D, T, H, KV, pos):
    """Several CTAs per kv head: their warps join their parts before the second kernel does."""
    cache = _filled(len(pos), KV, D, max(pos) + T, seed=KV)
    q = (torch.randn(len(pos), T, H, D, generator=_gen(D + T)) * 1.5).to(torch.bfloat16)
    _check(cache, q, torch.tensor(pos))
    _lib.check_device_status()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 6, 50])
@pytest.mark.parametrize("qs,ks,vs", [(1.0, 1.0, 1e-30), (1.0, 1.0, 1e25), (1e-20, 1e20, 1.0), (1e15, 1e-15, 3e4),
                                      (1e-30, 1.0, 1e-3), (30.0, 3.0, 1.0)])
def test_attend_magnitudes(D, T, qs, ks, vs):
    """fp16 operands inside: keys, queries and values of any bf16 magnitude."""
    cache = _filled(1, 2, D, 64, seed=9, k_scale=ks, v_scale=vs)
    if ks < 1e-10:                                    # _filled adds a shift of order one to the keys
        cache = Kv4Cache.empty(1, 64, 2, D, "cuda")
        kv = torch.randn(1, 64, 4, D, generator=_gen(10))
        kv[:, :, :2] *= ks
        kv[:, :, 2:] *= vs
        cache.append(kv.to(torch.bfloat16).reshape(1, 64, -1).cuda(), torch.zeros(1, dtype=torch.long, device="cuda"), 0)
    q = (torch.randn(1, T, 4, D, generator=_gen(11)) * qs).to(torch.bfloat16)
    _check(cache, q, torch.tensor(64 - T))


@pytest.mark.parametrize("T", [1, 40])
def test_attend_values_of_uneven_scale(T):
    """Positions whose values differ by powers of ten, constant groups (d = 0) and strong single scores."""
    D = 128
    kv = torch.randn(1, 96, 2, D, generator=_gen(21))
    kv[:, :, 1] *= 10.0 ** torch.randint(-6, 7, (96, 1), generator=_gen(22))
    kv[:, 10:20, 1] = 2.5
    kv[:, 50, 0] *= 6
    cache = Kv4Cache.empty(1, 96, 1, D, "cuda")
    cache.append(kv.to(torch.bfloat16).reshape(1, 96, -1).cuda(), torch.zeros(1, dtype=torch.long, device="cuda"), 0)
    q = (torch.randn(1, T, 3, D, generator=_gen(23)) * 2).to(torch.bfloat16)
    _check(cache, q, torch.tensor(96 - T))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [3, 9, 60])
def test_nan_reaches_only_rows_that_see_it(D, T):
    n = 64
    g = _gen(31)
    kv = torch.randn(1, n, 2, D, generator=g)
    bad = n - 2
    for part, ch in ((0, 3), (1, D - 1)):
        x = kv.clone()
        x[0, bad, part, ch] = float("inf") if part else float("nan")
        cache = Kv4Cache.empty(1, n, 1, D, "cuda")
        cache.append(x.to(torch.bfloat16).reshape(1, n, -1).cuda(), torch.zeros(1, dtype=torch.long, device="cuda"), 0)
        q = torch.randn(1, T, 2, D, generator=g).to(torch.bfloat16)
        got = cache.attend(q.cuda(), torch.tensor([n - T], device="cuda")).cpu()
        clean = [t for t in range(T) if n - T + t < bad]
        assert not got[:, clean].isnan().any()
        ref, bound = kv4_ref.attend(q[:, :len(clean)], cache.blocks, [n - T], D ** -0.5, n)
        assert bool(((got[:, clean].double() - ref).abs() <= bound).all())
        assert got[:, len(clean):].isnan().any()


def test_attend_scale_strides_out_and_empty():
    D, H, KV = 128, 4, 2
    cache = _filled(2, KV, D, 50, seed=41)
    wide = torch.randn(2, 3, H, D + 8, generator=_gen(42)).to(torch.bfloat16).cuda()
    p = torch.tensor([20, 40])
    a = _check(cache, wide[..., :D].cpu(), p, scale=0.31)
    assert torch.equal(cache.attend(wide[..., :D], p.cuda(), 0.31), a)                      # row pitch D + 8
    assert torch.equal(cache.attend(wide[..., 1:D + 1].contiguous(), p.cuda()), cache.attend(wide[..., 1:D + 1], p.cuda()))
    t = wide[..., :D].contiguous().transpose(1, 2).contiguous().transpose(1, 2)             # heads outside tokens
    assert torch.equal(cache.attend(t, p.cuda(), 0.31), a)
    out = torch.empty(2, 3, H, D, dtype=torch.bfloat16, device="cuda")
    assert cache.attend(t, p.cuda(), 0.31, out=out) is out and torch.equal(out, a)
    assert cache.attend(wide[:, :0, :, :D], p.cuda()).shape == (2, 0, H, D)
    pos2 = torch.tensor([[20, 0], [40, 0]], device="cuda")[:, 0]                            # a strided vector of positions
    assert torch.equal(cache.attend(t, pos2, 0.31), a)
    both = torch.zeros(2, 2, 3, H, D, dtype=torch.bfloat16, device="cuda")
    both[0] = t
    assert torch.equal(cache.attend(both[0], p.cuda(), 0.31, out=both[1]), a)
    for bad in (both[0], both.view(-1)[H * D:][:a.numel()].view_as(a)):
        with pytest.raises(ValueError, match="overlap"):
            cache.attend(both[0], p.cuda(), 0.31, out=bad)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30])
@pytest.mark.parametrize("T", [1, 3, 60])
def test_attend_unusual_scales(T, scale):
    cache = _filled(2, 2, 64, 150, seed=43, stale=True)
    q = torch.randn(2, T, 4, 64, generator=_gen(44)).to(torch.bfloat16)
    _check(cache, q, torch.tensor([90, -1]), scale=scale)


@pytest.mark.parametrize("T,S", [(60, 200), (96, 1500)])
def test_attend_prompts_on_two_streams_and_in_graphs(T, S):
    """The prompt kernel, its units cut and whole: two calls at once, and one captured call with moved positions."""
    D, H, KV = 128, 8, 2
    caches = [_filled(3, KV, D, S, seed=60 + i) for i in range(2)]
    q = torch.randn(3, T, H, D, generator=_gen(62)).to(torch.bfloat16).cuda()
    pos = torch.tensor([0, S - T, 50], device="cuda")
    want = [c.attend(q, pos) for c in caches]
    _check(caches[0], q.cpu(), pos.cpu())
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in caches], [[], []]
    for _ in range(4):
        for i, c in enumerate(caches):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.attend(q, pos))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for g, w in zip(got, want) for o in g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = caches[0].attend(q, pos)
    for p in ([S - T] * 3, [-T, 3, S // 2], [-5, -6, -7]):
        pos.copy_(torch.tensor(p))
        graph.replay()
        assert torch.equal(out, caches[0].attend(q, pos))
    _lib.check_device_status()


def test_attend_layer_slices_streams_and_graphs():
    """Caches that are slices of one tensor, a side stream, and two captured graphs replayed with moved positions."""
    D, H, KV, S = 64, 4, 2, 600
    store = torch.stack([kv4_blocks(1, S, KV, D, "cuda") for _ in range(3)])
    caches = [Kv4Cache(store[i], S) for i in range(3)]
    g = _gen(51)
    zero = torch.zeros((), dtype=torch.long, device="cuda")
    for c in caches:
        c.append(torch.randn(1, S, 2 * KV * D, generator=g).to(torch.bfloat16).cuda(), zero, 0)
    q = torch.randn(1, 1, H, D, generator=g).to(torch.bfloat16).cuda()
    pos = torch.tensor(599, device="cuda")
    want = [_check(c, q.cpu(), torch.tensor(599)) for c in caches]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [c.attend(q, pos) for c in caches]
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for c in caches[:2]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(c.attend(q, pos))
        graphs.append(gr)
    for p in (0, 17, 599):
        pos.fill_(p)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for c, o in zip(caches, outs):
            assert torch.equal(o, c.attend(q, pos))
