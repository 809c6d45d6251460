"""The decoder with the 4-bit cache and sampling: logits against the same model
with torch's attention over the quantised values, prompts of different lengths
against each alone, captured decode against eager decode, fixed random numbers."""
import pytest
import torch
import torch.nn.functional as F

from bfloat16x_b200 import _lib, llama_e2e
from bfloat16x_b200.kv4 import Kv4Cache
from bfloat16x_b200.llama_e2e import CONFIGS, LlamaModel, NextToken, SamplingParams, generate, pack_model
from tests.gpu_util import rel_l2

pytestmark = pytest.mark.gpu
TOL = 2e-2           # the decoder tests' tolerance: bf16 activations on both sides
# Where the projections run at another number of rows, keys and values differ in
# their last bf16 bit (up to 2^-8 of the value) before they are quantised, and a
# value that crosses a border moves by a whole step d.  With 32 normal values
# per group d is 4.1 sigma / 15 = 0.27 sigma; a value of 0.8 sigma crosses with
# probability 2^-8 * 0.8 / 0.27 = 1.2 %, which is sqrt(0.012) * 0.27 = 3 % of the
# keys' and values' norm if every value differs.  Two layers, keys and values:
# 2 * 3 % on the attention's part of the stream at most, beside TOL.
TOL_STEPS = 8e-2


def _prompt(B, P, vocab, seed=1):
    return torch.randint(0, vocab, (B, P), generator=torch.Generator().manual_seed(seed)).cuda()


class _Quantised(Kv4Cache):
    """The same cache, attended to by torch over the values read back."""
    __slots__ = ()

    def attend(self, q, pos0, scale=None, out=None):
        B, T, H, D = q.shape
        k, v = self.read(torch.zeros((), dtype=torch.long, device=q.device), self.max_seq)
        pos = pos0.reshape(-1, 1) + torch.arange(T, device=q.device)
        mask = (torch.arange(self.max_seq, device=q.device) <= pos.expand(B, T)[..., None])[:, None]
        return F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), attn_mask=mask,
                                              enable_gqa=True).transpose(1, 2)


def test_model_with_4bit_cache_matches_torch_attention():
    cfg = CONFIGS["tiny"]
    prompt = _prompt(2, 40, cfg.vocab)
    model = LlamaModel(cfg, 64, "cuda", seed=3, batch=2, kv_bits=4)
    pack_model(model)
    zero = torch.zeros((), dtype=torch.long, device="cuda")
    step = torch.tensor(40, device="cuda")
    tok = _prompt(2, 1, cfg.vocab, 9)
    got = [model(prompt, zero), model(tok, step)]
    model.cache_kv4 = [_Quantised(torch.zeros_like(c.blocks), 64) for c in model.cache_kv4]
    ref = [model(prompt, zero), model(tok, step)]
    for a, b in zip(got, ref):
        assert rel_l2(a.cpu().numpy(), b.cpu().numpy()) < TOL
    _lib.check_device_status()


def test_prompts_of_different_lengths():
    cfg = CONFIGS["tiny"]
    lengths = [5, 33, 20]
    P = max(lengths)
    model = LlamaModel(cfg, 48, "cuda", seed=4, batch=3, kv_bits=4)
    pack_model(model)
    prompt = _prompt(3, P, cfg.vocab, 2)
    pos0 = torch.tensor([n - P for n in lengths], device="cuda")
    first = model(prompt, pos0)
    nxt = model(prompt[:, :1], torch.tensor(lengths, device="cuda"))
    one = LlamaModel(cfg, 48, "cuda", seed=4, batch=1, kv_bits=4)
    pack_model(one)
    for i, n in enumerate(lengths):
        a = one(prompt[i:i + 1, P - n:], torch.zeros((), dtype=torch.long, device="cuda"))
        b = one(prompt[i:i + 1, :1], torch.tensor(n, device="cuda"))
        assert rel_l2(first[i].cpu().numpy(), a[0].cpu().numpy()) < TOL_STEPS
        assert rel_l2(nxt[i].cpu().numpy(), b[0].cpu().numpy()) < TOL_STEPS
    _lib.check_device_status()


@pytest.mark.parametrize("sampling", [None, SamplingParams(temperature=0.8, top_k=20, top_p=0.9, min_p=0.01)])
def test_graph_decode_matches_eager(sampling):
    cfg = CONFIGS["tiny"]
    lengths = [30, 12]
    prompt = _prompt(2, 30, cfg.vocab, 5)
    toks = []
    for use_graph in (True, False):
        model = LlamaModel(cfg, 64, "cuda", seed=6, batch=2, kv_bits=4)
        pack_model(model)
        gen = torch.Generator(device="cuda").manual_seed(77)
        toks.append(generate(model, prompt, 12, use_graph, sampling, gen, lengths)[0])
    assert torch.equal(*toks)
    _lib.check_device_status()


def test_sampling_with_the_bf16_cache_and_refusals():
    cfg = CONFIGS["tiny"]
    model = LlamaModel(cfg, 64, "cuda", seed=6)
    prompt = _prompt(1, 20, cfg.vocab, 5)
    greedy = generate(model, prompt, 8)[0]
    cold = generate(model, prompt, 8, sampling=SamplingParams(temperature=0.0))[0]
    assert torch.equal(greedy, cold)
    gens = [torch.Generator(device="cuda").manual_seed(s) for s in (1, 1, 2)]
    hot = [generate(model, prompt, 16, sampling=SamplingParams(temperature=3.0), generator=g)[0] for g in gens]
    assert torch.equal(hot[0], hot[1]) and not torch.equal(hot[0], hot[2])
    with pytest.raises(ValueError, match="4-bit"):
        generate(model, prompt, 1, lengths=[20])
    with pytest.raises(ValueError, match="4-bit"):
        model(prompt, torch.zeros(1, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError, match="kv_bits"):
        llama_e2e.LlamaModel(cfg, 64, "cuda", kv_bits=8)


@pytest.mark.parametrize("kv_bits", [4, 16])
@pytest.mark.parametrize("use_graph", [True, False])
def test_logits_of_nan_raise(kv_bits, use_graph):
    """No token can be drawn: token 0 is fed instead, and the call raises."""
    cfg = CONFIGS["tiny"]
    model = LlamaModel(cfg, 64, "cuda", seed=6, batch=2, kv_bits=kv_bits)
    prompt = _prompt(2, 20, cfg.vocab, 5)
    chooser = NextToken(2, "cuda", SamplingParams(temperature=0.7))
    logits = torch.randn(2, cfg.vocab, generator=torch.Generator().manual_seed(3)).cuda()
    logits[1] = float("nan")
    tok = chooser.choose(logits)
    assert tok.shape == (2, 1) and int(tok[1]) == 0
    with pytest.raises(_lib.Bf16xError, match=r"sequences \[1\]"):
        chooser.check()
    with torch.no_grad():
        model.norm.weight.fill_(float("nan"))
    with pytest.raises(_lib.Bf16xError, match=r"sequences \[0, 1\]"):
        generate(model, prompt, 4, use_graph, SamplingParams(temperature=0.7, top_k=5))
    with torch.no_grad():
        model.norm.weight.fill_(1.0)
    a, b = (generate(model, prompt, 4, g, SamplingParams(temperature=0.7, top_k=1))[0] for g in (use_graph, True))
    assert torch.equal(a, b)
    _lib.check_device_status()


def test_generation_up_to_the_last_position():
    cfg = CONFIGS["tiny"]
    prompt = _prompt(2, 20, cfg.vocab, 5)
    long, short = (LlamaModel(cfg, n, "cuda", seed=6, batch=2, kv_bits=4) for n in (64, 25))
    assert torch.equal(generate(long, prompt, 5)[0], generate(short, prompt, 5)[0])
    assert torch.equal(generate(long, prompt, 13, lengths=[12, 7])[0], generate(short, prompt, 13, lengths=[12, 7])[0])
    _lib.check_device_status()
    with pytest.raises(ValueError, match="do not fit"):
        generate(short, prompt, 6)
    with pytest.raises(ValueError, match="do not fit"):
        generate(short, prompt, 14, lengths=[12, 7])
    _lib.check_device_status()
