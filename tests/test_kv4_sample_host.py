"""Refusals of the 4-bit cache and of sampling that need no GPU: wrong shapes,
types and devices raise before anything is launched."""
import ctypes
import types

import pytest
import torch

from bfloat16x_b200 import _lib, llama_e2e
from bfloat16x_b200.kv4 import Kv4Cache, kv4_blocks
from bfloat16x_b200.llama_e2e import NextToken
from bfloat16x_b200.sampling import SamplingParams, sample


def test_block_sizes():
    L = _lib.lib()
    assert [L.bf16x_kv4_block_bytes(d) for d in (64, 128, 96, 0)] == [1280, 2560, 0, 0]
    assert kv4_blocks(2, 33, 3, 64, "cpu").shape == (2, 3, 3, 1280)
    c = Kv4Cache.empty(2, 33, 3, 128, "cpu")
    assert (c.batch, c.kv_heads, c.max_seq, c.head_dim, c.nbytes()) == (2, 3, 33, 128, 2 * 3 * 3 * 2560)
    assert Kv4Cache(c.blocks).max_seq == 48


@pytest.mark.parametrize("args", [(1, 16, 1, 96), (0, 16, 1, 64), (1, 0, 1, 64), (1, 16, 0, 64)])
def test_bad_cache_sizes(args):
    with pytest.raises(ValueError):
        kv4_blocks(*args, "cpu")


def test_bad_blocks():
    b = kv4_blocks(1, 32, 2, 64, "cpu")
    for bad in (b.float(), b[0], b[..., :100], b.transpose(1, 2), b[:, :, :, ::2]):
        with pytest.raises(ValueError):
            Kv4Cache(bad)
    for n in (16, 33, 0):
        with pytest.raises(ValueError, match="positions"):
            Kv4Cache(b, n)


def test_cpu_tensors_are_refused():
    c = Kv4Cache.empty(1, 32, 2, 64, "cpu")
    p = torch.zeros(1, dtype=torch.long)
    with pytest.raises(_lib.Bf16xError, match="CUDA"):
        c.append(torch.zeros(1, 1, 5 * 64, dtype=torch.bfloat16), p, 1)
    with pytest.raises(_lib.Bf16xError, match="CUDA"):
        c.attend(torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), p)
    with pytest.raises(_lib.Bf16xError, match="CUDA"):
        c.read(p, 1)
    with pytest.raises(_lib.Bf16xError, match="CUDA"):
        sample(torch.zeros(1, 5), torch.zeros(1))


def test_tensor_parallel_ranks_must_draw_alike():
    with pytest.raises(ValueError, match="same seed"):
        NextToken(2, "cpu", SamplingParams(), None, tp=2)
    a, b = (NextToken(2, "cpu", SamplingParams(), torch.Generator().manual_seed(5), tp=2) for _ in range(2))
    a.draw()
    b.draw()
    assert torch.equal(a.u, b.u) and NextToken(2, "cpu", None, None, tp=2).sampling is None


def test_rows_without_a_token_are_fed_an_index_and_reported(monkeypatch):
    """What sample() gives for rows of NaN never goes on to the embedding."""
    drawn = iter([[5, 0, 3], [-1, 2, -1], [1, 1, 1], [4, 4, 4]])
    monkeypatch.setattr(llama_e2e, "sample", lambda *a: torch.tensor(next(drawn)))
    c = NextToken(3, "cpu", SamplingParams())
    logits = torch.zeros(3, 8)
    assert c.choose(logits).tolist() == [[5], [0], [3]]
    c.check()
    assert c.choose(logits).tolist() == [[0], [2], [0]]
    assert c.choose(logits).tolist() == [[1], [1], [1]]
    with pytest.raises(_lib.Bf16xError, match=r"sequences \[0, 2\]"):
        c.check()
    c.check()                                        # reported once
    c.choose(logits)
    c.check()
    greedy = NextToken(3, "cpu")
    assert greedy.choose(torch.full((3, 8), float("nan"))).lt(8).all()
    greedy.check()


def test_generate_refuses_what_does_not_fit_the_4bit_cache():
    model = types.SimpleNamespace(cache_kv4=[None], max_seq=24, tp=1)       # refused before the model is called
    prompt = torch.zeros(2, 20, dtype=torch.long)
    for new, lengths in ((5, None), (400, None), (8, [17, 3]), (5, [1, 20])):
        with pytest.raises(ValueError, match="do not fit"):
            llama_e2e.generate(model, prompt, new, lengths=lengths)


def _err():
    return _lib.lib().bf16x_last_error().decode()


def test_c_entry_points_refuse():
    """Checked on the host, before any launch (the pointers are never followed)."""
    L, v, odd = _lib.lib(), ctypes.c_void_p(256), ctypes.c_void_p(264)

    def append(qkv=v, ld_b=640, ld_t=320, B=1, T=2, H=1, KV=2, D=64, pos=v, cos=v, sin=v, q=v, blocks=v, S=32):
        return L.bf16x_kv4_append(qkv, ld_b, ld_t, B, T, H, KV, D, pos, 1, cos, sin, q, blocks, S, None)

    for kw, word in (({"D": 96}, "head_dim"), ({"KV": 0}, "shape"), ({"S": 0}, "shape"), ({"T": -1}, "shape"),
                     ({"qkv": None}, "null"), ({"pos": None}, "null"), ({"cos": None}, "null"), ({"sin": None}, "null"),
                     ({"blocks": odd}, "aligned"), ({"ld_t": 321}, "multiples"), ({"H": -1}, "heads"),
                     ({"B": 65536}, "65535")):
        assert append(**kw) < 0, kw
        assert word in _err(), (kw, _err())
    assert append(B=0) == 0 and append(T=0) == 0

    assert L.bf16x_kv4_read(v, 32, 1, 1, 2, 64, v, 1, v, None, None) < 0 and "null" in _err()
    assert L.bf16x_kv4_read(v, 32, 1, 1, 2, 80, v, 1, v, v, None) < 0 and "head_dim" in _err()

    def attend(q=v, B=1, T=1, H=4, KV=2, D=64, S=4096, out=v, ws=v, n=1 << 40, ldq=256):
        return L.bf16x_kv4_attend(q, ldq, ldq, 64, B, T, H, KV, D, v, 1, 0.1, v, S, out, ws, n, None)

    for kw, word in (({"H": 3}, "multiple"), ({"H": 0}, "multiple"), ({"D": 32}, "head_dim"), ({"q": None}, "null"),
                     ({"out": odd}, "aligned"), ({"ldq": 4}, "multiples"), ({"ws": None, "n": 0}, "workspace"),
                     ({"n": 8}, "workspace")):
        assert attend(**kw) < 0, kw
        assert word in _err(), (kw, _err())
    assert attend(B=0) == 0 and attend(T=0) == 0

    def smp(x=v, dt=1, ld=100, B=1, V=100, u=v, out=v):
        return L.bf16x_sample(x, dt, ld, B, V, u, None, 1.0, None, 0, None, 1.0, None, 0.0, out, None)

    for kw, word in (({"dt": 2}, "bf16 or fp32"), ({"V": 0}, "shape"), ({"ld": 99}, "shape"), ({"x": None}, "null"),
                     ({"u": None}, "null"), ({"out": None}, "null"), ({"V": 400000, "ld": 400000}, "at most")):
        assert smp(**kw) < 0, kw
        assert word in _err(), (kw, _err())
    assert smp(B=0) == 0
