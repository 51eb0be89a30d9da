"""GPU: the model over the key/value cache (RatchetGPT.forward_cached) and generate().

Bars: against the uncached forward with its keys and values put through the same 8-bit blocks in 64
bits, a dense fp32 model agrees to fp32 rounding through a few layers: 1e-4 of the logits' norm.  A
code within rounding of the middle between two may fall either way, one step in 127 of a few of 10^6
values, which is below that.  Against the plain uncached forward, keys and values are off by a uniform
rounding of one step = max / 127, about 3 / 127 / sqrt(12) = 0.7 % of their norm; two layers of the int8
model, whose activations are themselves rounded to 8 bits by row, stay within 5 %.
"""

from __future__ import annotations

import pytest
import torch

from local_ai_training_b200 import model as model_module
from local_ai_training_b200.generate import cache_for, choose, generate
from local_ai_training_b200.kv_cache import QUANT_BLOCK
from local_ai_training_b200.model import ModelConfig, build_seeded_model

pytestmark = pytest.mark.gpu


def _model(dev, mode="fp32", **kw):
    config = ModelConfig(vocab_size=384, block_size=256, n_layer=2, n_head=4, n_embd=256,
                         matmul_mode=mode, int8_backward=mode == "int8", **kw)
    return build_seeded_model(config, max_code=None if mode == "fp32" else 2, seed=3).to(dev).eval()


def _blocked(x):
    """[B, H, T, D] through blocks of 16 tokens and a head in 8 bits, in 64 bits."""
    b, h, t, d = x.shape
    pad = -t % QUANT_BLOCK
    y = torch.nn.functional.pad(x.double(), (0, 0, 0, pad)).view(b, h, -1, QUANT_BLOCK, d)
    s = (y.abs().amax((-1, -2), keepdim=True) / 127).clamp_min(torch.finfo(torch.float32).tiny)
    return ((y / s).round() * s).view(b, h, -1, d)[:, :, :t].to(x.dtype)


def _tokens(dev, *shape, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randint(0, 384, shape, device=dev, generator=g)


def _uncached(model, tokens, monkeypatch):
    plain = torch.nn.functional.scaled_dot_product_attention
    with monkeypatch.context() as m:
        m.setattr(model_module.F, "scaled_dot_product_attention",
                  lambda q, k, v, **kw: plain(q, _blocked(k), _blocked(v), **kw))
        with torch.no_grad():
            return model(tokens)[0]


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


def test_forward_cached_equals_the_uncached_forward_on_8_bit_keys(cuda_device, monkeypatch):
    model = _model(cuda_device)
    texts = [_tokens(cuda_device, n, seed=n) for n in (200, 1, 77)]
    want = [_uncached(model, t[None], monkeypatch)[0] for t in texts]
    cache = cache_for(model, 1024)
    seqs = [cache.new_sequence() for _ in texts]
    batch = cache.reserve(seqs, [len(t) for t in texts])
    got = model.forward_cached(torch.cat(texts), cache, batch, last_only=False)
    assert _rel(got, torch.cat(want)) <= 1e-4
    # the same text in pieces of whole blocks: the same codes, so the same logits
    seq = cache.new_sequence()
    at = 0
    for n in (32, 128, 16, 24):
        batch = cache.reserve([seq], n)
        piece = model.forward_cached(texts[0][at:at + n], cache, batch, last_only=False)
        assert _rel(piece, want[0][at:at + n]) <= 1e-4
        at += n


def test_int8_model_decodes_token_by_token(cuda_device):
    model = _model(cuda_device, "int8")
    text = _tokens(cuda_device, 2, 90)
    with torch.no_grad():
        want = model(text)[0]
    cache = cache_for(model, 512)
    seqs = [cache.new_sequence(), cache.new_sequence()]
    batch = cache.reserve(seqs, 60)
    got = model.forward_cached(text[:, :60].reshape(-1), cache, batch, last_only=False)
    assert _rel(got.view(2, 60, -1), want[:, :60]) <= 0.05
    for i in range(60, 90):
        batch = cache.reserve(seqs)
        got = model.forward_cached(text[:, i].contiguous(), cache, batch)
        assert got.shape == (2, 384) and _rel(got, want[:, i]) <= 0.05


@pytest.mark.parametrize("mode", ["fp32", "int8"])
def test_generate_samples_share_prompts_and_give_pages_back(cuda_device, mode):
    model = _model(cuda_device, mode)
    prompts = [_tokens(cuda_device, n, seed=n).tolist() for n in (70, 3, 128)]
    cache = cache_for(model, 64 * 40)
    kept = cache.new_sequence()
    cache.reserve([kept], 10)
    free = cache.free_pages
    greedy = generate(model, prompts, 20, samples=3, cache=cache)
    assert cache.free_pages == free and cache.length(kept) == 10
    for per_prompt in greedy:
        assert len(per_prompt) == 3 and all(len(t) == 20 for t in per_prompt)
        assert per_prompt[0] == per_prompt[1] == per_prompt[2]
    draws = [generate(model, prompts, 12, samples=2, temperature=1.5,
                      generator=torch.Generator(device=cuda_device).manual_seed(s)) for s in (1, 1, 2)]
    assert draws[0] == draws[1] != draws[2]
    assert any(p[0] != p[1] for p in draws[0])


def test_generate_greedy_follows_the_model(cuda_device):
    """Each greedy token is the largest logit of forward_cached on the text so far."""
    model = _model(cuda_device)
    prompt = _tokens(cuda_device, 50).tolist()
    out = generate(model, [prompt], 30)[0][0]
    cache = cache_for(model, 256)
    seq = cache.new_sequence()
    logits = model.forward_cached(torch.tensor(prompt, device=cuda_device), cache,
                                  cache.reserve([seq], len(prompt)))
    for token in out:
        assert token == logits.argmax().item()
        logits = model.forward_cached(torch.tensor([token], device=cuda_device), cache, cache.reserve([seq]))
    stop = out[4]
    cut = generate(model, [prompt], 30, stop_token=stop)[0][0]
    assert cut == out[:out.index(stop) + 1]


def test_generate_refusals(cuda_device):
    model = _model(cuda_device)
    assert generate(model, [], 4) == [] and generate(model, [[1]], 0) == [[[]]]
    with pytest.raises(ValueError, match="at least one token"):
        generate(model, [[1], []], 4)
    with pytest.raises(ValueError, match="block_size"):
        generate(model, [[1] * 250], 7)
    with pytest.raises(ValueError, match="temperature"):
        generate(model, [[1]], 2, temperature=-1.0)
    with pytest.raises(ValueError, match="samples"):
        generate(model, [[1]], 2, samples=0)
    with pytest.raises(RuntimeError, match="pages needed"):
        generate(model, [[1] * 200], 2, cache=cache_for(model, 64))
    cache = cache_for(model, 64)
    seq = cache.new_sequence()
    batch = cache.reserve([seq], 3)
    one = torch.zeros(3, device=cuda_device, dtype=torch.long)
    with pytest.raises(ValueError, match="newest tokens"):
        model.forward_cached(one[:2], cache, batch)
    other = cache_for(_model(cuda_device), 64)
    other.n_layer = 1
    with pytest.raises(ValueError, match="must be the model's"):
        model.forward_cached(one, other, batch)
    with pytest.raises(RuntimeError, match="evaluation mode"):
        model.train().forward_cached(one, cache, batch)
    with pytest.raises(RuntimeError, match="evaluation mode"):
        generate(model, [[1]], 2)


def test_choose(cuda_device):
    logits = torch.tensor([[0.0, 2.0, 2.0], [5.0, 1.0, 0.0]], device=cuda_device)
    assert choose(logits).tolist() == [1, 0]
    g = torch.Generator(device=cuda_device).manual_seed(0)
    assert choose(logits * 1e4, 1.0, g)[1].item() == 0
