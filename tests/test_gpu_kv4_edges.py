"""Attention over the 4-bit cache at its edges: rows at and past the end of a
cache that is full, against the plain 64-bit formulas on the CPU."""
import pytest
import torch

from bfloat16x_b200 import _lib
from bfloat16x_b200.kv4 import Kv4Cache
from tests import kv4_ref

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _full(B, KV, D, S, seed):
    """A cache with every one of its S positions written."""
    cache = Kv4Cache.empty(B, S, KV, D, "cuda")
    kv = torch.randn(B, S, 2 * KV * D, generator=_gen(seed)).to(torch.bfloat16).cuda()
    cache.append(kv, torch.zeros(1, dtype=torch.long, device="cuda"), 0)
    return cache


def _check(cache, q, pos0, scale=None):
    got = cache.attend(q.cuda(), torch.tensor(pos0, device="cuda"), scale).cpu()
    scale = q.shape[3] ** -0.5 if scale is None else scale
    ref, bound = kv4_ref.attend(q, cache.blocks, pos0, scale, cache.max_seq)
    err = (got.double() - ref).abs()
    over = float((err - bound).max())
    assert over <= 0, f"off by {over} over the bound"
    return got


# rows inside the cache and past it, in one tile and in tiles of their own; 40000 positions of one
# sequence: its parts are joined within the CTAs first; 60 tokens: the prompt kernel
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,T,H,KV,pos", [
    (64, 1, 4, 2, [64, 63]), (61, 1, 4, 2, [61, 60]), (61, 1, 1, 1, [1000, 0]), (64, 1, 8, 1, [1 << 40, 5]),
    (400, 1, 12, 1, [400, 399]), (64, 3, 2, 2, [62, 61]), (61, 3, 4, 1, [59, 58]), (300, 6, 4, 2, [296, 300, 120]),
    (40000, 1, 4, 1, [40000]), (40000, 2, 4, 1, [39999]), (100, 60, 2, 2, [70, 100, 40])])
def test_rows_past_a_full_cache_are_zeros(D, S, T, H, KV, pos):
    cache = _full(len(pos), KV, D, S, seed=S + T)
    q = torch.randn(len(pos), T, H, D, generator=_gen(T + D)).to(torch.bfloat16)
    got = _check(cache, q, pos)
    past = [(b, t) for b, p in enumerate(pos) for t in range(T) if p + t >= S]
    assert past and not any(bool(got[b, t].any()) for b, t in past)
    assert _lib.device_status() & 16


# the end of the cache within rows 0..127 and 128..255 of a unit of the prompt kernel; 1500 and 400 positions may be
# cut between CTAs, 200 tokens of 150 sequences go in whole units
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S,T,H,KV,pos", [(2, 1500, 60, 4, 1, [1460, 1400]), (1, 400, 200, 1, 1, [250]),
                                            (1, 400, 200, 1, 1, [399]), (1, 400, 70, 4, 1, [331]),
                                            (150, 210, 200, 1, 1, [0] * 149 + [60])])
def test_attend_alone_reports_rows_past_the_cache(D, B, S, T, H, KV, pos):
    cache = _full(B, KV, D, S, seed=S + T)
    assert _lib.device_status() == 0
    q = torch.randn(B, T, H, D, generator=_gen(T + D)).to(torch.bfloat16)
    got = cache.attend(q.cuda(), torch.tensor(pos, device="cuda"))
    assert _lib.device_status() == 16
    for b, p in enumerate(pos):
        assert not got[b, max(S - p, 0):].any() and bool(got[b, :S - p].any())
    inside = [p - max(0, p + T - S) for p in pos]                   # the same, all inside: nothing to report
    cache.attend(q.cuda(), torch.tensor(inside, device="cuda"))
    assert _lib.device_status() == 0
