"""Attention over the 4-bit cache where sizes differ within a position: groups
of channels of keys and of values that differ by powers of ten, and long tails
of small weights behind one strong score, against the 64-bit formulas and the
same per-channel bound as everywhere."""
import pytest
import torch

from bfloat16x_b200 import _lib
from bfloat16x_b200.kv4 import Kv4Cache
from tests import kv4_ref

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cache(k, v):
    """k, v [B, S, KV, D] -> a cache that holds them."""
    B, S, KV, D = k.shape
    cache = Kv4Cache.empty(B, S, KV, D, "cuda")
    kv = torch.cat((k, v), 2).to(torch.bfloat16).reshape(B, S, -1).cuda()
    cache.append(kv, torch.zeros(1, dtype=torch.long, device="cuda"), 0)
    return cache


def _check(cache, q, pos0, scale=None):
    got = cache.attend(q.cuda(), torch.tensor(pos0, device="cuda"), scale)
    scale = q.shape[3] ** -0.5 if scale is None else scale
    ref, bound = kv4_ref.attend(q, cache.blocks, pos0, scale, cache.max_seq)
    over = (got.cpu().double() - ref).abs() / bound.clamp(min=1e-300)
    worst = float(over.max())
    assert worst <= 1, f"{worst} of the bound"
    assert torch.equal(got, cache.attend(q.cuda(), torch.tensor(pos0, device="cuda"), scale))
    _lib.check_device_status()


def _groups(S, D, how, seed):
    """Powers of ten for the groups of a position [S, 1, D]: the same in all positions, or drawn for each."""
    n = D // 32
    if how == "fixed":
        e = torch.tensor([0, -3, -5, -2][:n]).expand(S, n)
    elif how == "wide":
        e = torch.tensor([0, -24, 3, -13][:n]).expand(S, n)             # 2^-80 and 2^10 beside 1
    else:
        e = torch.tensor([0, -3, -5, -20])[torch.randint(0, 3 if how == "drawn" else 4, (S, n), generator=_gen(seed))]
    return (10.0 ** e.double()).repeat_interleave(32, 1)[:, None]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 6, 60])
@pytest.mark.parametrize("how", ["fixed", "drawn", "far", "wide"])
def test_value_groups_of_uneven_size(D, T, how):
    S, KV = 150, 2
    k, v = torch.randn(2, S, KV, D, generator=_gen(1)), torch.randn(2, S, KV, D, generator=_gen(2))
    v = v.double() * _groups(S, D, how, 3)
    q = (torch.randn(2, T, 4, D, generator=_gen(4)) * 2).to(torch.bfloat16)
    _check(_cache(k, v), q, [S - T, S // 2 - T + 1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 6, 60])
@pytest.mark.parametrize("values", [False, True])
def test_key_groups_of_uneven_size(D, T, values):
    """Each group has its share of the scores: the queries are large where the keys are small."""
    S, KV = 150, 2
    k, v = torch.randn(2, S, KV, D, generator=_gen(5)), torch.randn(2, S, KV, D, generator=_gen(6))
    size = _groups(1, D, "fixed", 0)
    q = torch.randn(2, T, 4, D, generator=_gen(7)).double()
    if values:
        v = v * size
    _check(_cache(k * size, v), (q / size).to(torch.bfloat16), [S - T, S // 2 - T + 1])


@pytest.mark.parametrize("T", [1, 60])
def test_key_groups_drawn(T):
    """Positions whose large groups differ: most weight lies where a large query meets a large key."""
    S, D = 150, 128
    k, v = torch.randn(1, S, 1, D, generator=_gen(8)), torch.randn(1, S, 1, D, generator=_gen(9))
    q = torch.randn(1, T, 4, D, generator=_gen(10)).double() * _groups(1, D, "drawn", 11)
    _check(_cache(k * _groups(S, D, "drawn", 12), v), q.to(torch.bfloat16), [S - T], 0.3)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,S", [(1, 100000), (3, 40000), (60, 12000)])
@pytest.mark.parametrize("down", [(0, 3, 6, 8), (0, 5, 7, 12), (20, 0, 10, 15)])
def test_long_tail_behind_a_strong_score(D, T, S, down):
    """One position 2^20 above all others, which together weigh as much as S / 2^20; groups of 2^-down."""
    n = D // 32
    k = torch.zeros(1, S, 1, D)
    k[0, 0] = 1.0
    strong = 20 * 0.693147 / D
    size = (2.0 ** -torch.tensor(down[:n], dtype=torch.float64)).repeat_interleave(32)
    v = (1 + torch.rand(1, 1, 1, D, generator=_gen(13))).expand(1, S, 1, D).double().clone()
    v[0, 0] = torch.randn(1, D, generator=_gen(14)) * 1e-3
    q = torch.full((1, T, 2, D), 1.0)
    q[:, :, 1] = 0.9
    _check(_cache(k, v * size), q.to(torch.bfloat16), [S - T], strong)


# (B, T, H, KV, S, first positions): units that go whole and cut, some sequences with groups far apart and some without,
# in the first tiles only or in the last ones
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,H,KV,S,pos", [(20, 64, 32, 8, 64, (0, 0)), (40, 75, 8, 2, 120, (-75, 44)), (3, 130, 4, 2, 1500, (-130, 1370)),
                                            (1, 300, 4, 1, 2500, (2200, 2200)), (2, 520, 2, 1, 2000, (1, 1480))])
def test_prompts_of_which_parts_have_groups_far_apart(D, B, T, H, KV, S, pos):
    k, v = torch.randn(B, S, KV, D, generator=_gen(21)), torch.randn(B, S, KV, D, generator=_gen(22))
    far = torch.rand(B, 1, KV, 1, generator=_gen(23)) < 0.5
    at = torch.arange(S)[None, :, None, None]
    v[..., 32:64] *= torch.where(far & (at < 100), 2.0 ** -12, 1.0)
    k[..., :32] *= torch.where(far & (at >= max(S - 140, 100)), 2.0 ** -11, 1.0)
    q = torch.randn(B, T, H, D, generator=_gen(24)).to(torch.bfloat16)
    _check(_cache(k, v), q, torch.linspace(pos[0], pos[1], B).round().long().tolist())


@pytest.mark.parametrize("T", [60, 130])
def test_captured_prompt_follows_the_sizes_in_the_cache(T):
    """One captured call over a cache whose groups are alike, then far apart, then alike."""
    D, H, KV, S = 128, 4, 2, 600
    k, v = torch.randn(1, S, KV, D, generator=_gen(25)), torch.randn(1, S, KV, D, generator=_gen(26))
    w = v.clone()
    w[..., 64:96] *= 1e-4
    cache, other = _cache(k, v), _cache(k, w)
    plain = cache.blocks.clone()
    q = torch.randn(1, T, H, D, generator=_gen(27)).to(torch.bfloat16).cuda()
    pos = torch.tensor(S - T, device="cuda")
    want = [cache.attend(q, pos), other.attend(q, pos)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, pos)
    for i, blocks in enumerate((plain, other.blocks, plain, other.blocks)):
        cache.blocks.copy_(blocks)
        graph.replay()
        assert torch.equal(out, want[i % 2])
    _lib.check_device_status()


def test_many_pieces_of_a_cta_some_of_them_far_apart():
    """24 units per CTA: every third sequence has groups far apart; a few sequences of each kind against the formulas."""
    B, KV, T, H, D = 300, 4, 130, 16, 64
    k, v = torch.randn(B, T, KV, D, generator=_gen(31)), torch.randn(B, T, KV, D, generator=_gen(32))
    v[1::3, ..., 32:] *= 2.0 ** -12
    cache = _cache(k, v)
    q = torch.randn(B, T, H, D, generator=_gen(33)).to(torch.bfloat16)
    got = cache.attend(q.cuda(), torch.zeros(1, dtype=torch.long, device="cuda")).cpu()
    for b in (0, 1, 151, B - 2):
        ref, bound = kv4_ref.attend(q[b:b + 1], cache.blocks[b:b + 1], [0], D ** -0.5, T)
        worst = float(((got[b:b + 1].double() - ref).abs() / bound).max())
        assert worst <= 1, f"sequence {b}: {worst} of the bound"
    _lib.check_device_status()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [3, 9, 60])
@pytest.mark.parametrize("part", [0, 1])
def test_nan_beside_groups_far_apart(D, T, part):
    """An infinity in the keys or values of a position reaches only the rows that see it, in whatever form they go."""
    n = 200
    kv = torch.randn(1, n, 2, D, generator=_gen(34))
    kv[:, :, 1, :32] *= 2.0 ** -12
    kv[0, n - 2, part, D - 1] = float("inf")
    cache = _cache(kv[:, :, :1], kv[:, :, 1:])
    q = torch.randn(1, T, 2, D, generator=_gen(35)).to(torch.bfloat16)
    got = cache.attend(q.cuda(), torch.tensor([n - T], device="cuda")).cpu()
    ref, bound = kv4_ref.attend(q[:, :T - 2], cache.blocks, [n - T], D ** -0.5, n)
    assert bool(((got[:, :T - 2].double() - ref).abs() <= bound).all())
    seen = got[:, T - 2:].isnan()
    assert bool(seen.all()) if part == 0 else bool(seen[..., D - 32:].all() and not seen[..., :D - 32].any())
    _lib.check_device_status()
