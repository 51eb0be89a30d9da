"""Text generation with a RatchetGPT over the paged int8 key/value cache (kv_cache.py).

The reference generates by running the whole window again for every token (generate.py:137); here a
prompt runs once, every further token runs alone over the cache, and several samples of one prompt
share the prompt's pages (forks; a shared page is copied when a sample writes into it).

    from local_ai_training_b200.generate import generate
    texts = generate(model.eval(), [prompt_tokens], max_new_tokens=64, samples=4, temperature=0.8)

    python -m local_ai_training_b200.generate        # a small random decoder, greedy and sampled
"""

from __future__ import annotations

import torch
from torch import Tensor

from .kv_cache import PagedKVCache
from .model import RatchetGPT


def cache_for(model: RatchetGPT, tokens: int, *, page_size: int = 64, extra_pages: int = 0) -> PagedKVCache:
    """A cache of the model's layers and heads with room for `tokens` tokens in whole pages."""
    config = model.config
    return PagedKVCache(len(model.blocks), config.n_head, config.n_embd // config.n_head,
                        n_pages=-(-tokens // page_size) + extra_pages, page_size=page_size,
                        device=model.position_encoding.device)


def choose(logits: Tensor, temperature: float = 0.0, generator: torch.Generator | None = None) -> Tensor:
    """Next tokens [rows] of logits [rows, vocab]: the largest (lowest index of equals) at temperature 0,
    else one drawn from softmax(logits / temperature)."""
    if temperature < 0:
        raise ValueError("temperature must be >= 0")
    if temperature == 0:
        return logits.argmax(dim=-1)
    return torch.multinomial(torch.softmax(logits.float() / temperature, dim=-1), 1,
                             generator=generator)[:, 0]


@torch.no_grad()
def generate(model: RatchetGPT, prompts: list[list[int]], max_new_tokens: int, *, samples: int = 1,
             temperature: float = 0.0, stop_token: int | None = None,
             generator: torch.Generator | None = None, cache: PagedKVCache | None = None
             ) -> list[list[list[int]]]:
    """The new tokens of `samples` continuations of each prompt, [prompts][samples][tokens].

    A continuation ends with stop_token (which is kept) or after max_new_tokens.  All prompts are
    prefilled as one ragged batch; the unfinished continuations of all of them decode as one batch.
    `cache`: a cache of the model to use (its other sequences are left alone); by default one is made
    for the call."""
    if model.training:
        raise RuntimeError("generate requires evaluation mode (model.eval())")
    if max_new_tokens < 0 or samples < 1:
        raise ValueError("max_new_tokens must be >= 0 and samples >= 1")
    if not all(prompts):
        raise ValueError("every prompt needs at least one token")
    longest = max((len(p) for p in prompts), default=0) + max_new_tokens
    if longest > model.config.block_size:
        raise ValueError(f"prompt and new tokens ({longest}) exceed configured block_size "
                         f"({model.config.block_size})")
    device = model.position_encoding.device
    texts: list[list[list[int]]] = [[[] for _ in range(samples)] for _ in prompts]
    if not prompts or max_new_tokens == 0:
        return texts
    if cache is None:
        page = 64
        # the prompts' pages, and a page for each sample's copy of the last plus its own new ones
        own = -(-max_new_tokens // page) + 1
        cache = cache_for(model, sum(-(-len(p) // page) * page for p in prompts), page_size=page,
                          extra_pages=len(prompts) * samples * own)
    live: list[tuple[int, int, int]] = []  # (sequence, prompt, sample)
    try:
        firsts = []
        for i in range(len(prompts)):
            firsts.append(cache.new_sequence())
            live.append((firsts[i], i, 0))
        batch = cache.reserve(firsts, [len(p) for p in prompts])
        tokens = torch.tensor([t for p in prompts for t in p], device=device)
        logits = model.forward_cached(tokens, cache, batch)
        for i, seq in enumerate(firsts):
            live += [(cache.fork(seq), i, s) for s in range(1, samples)]
        logits = logits[torch.tensor([i for _, i, _ in live], device=device)]
        for step in range(max_new_tokens):
            tokens = choose(logits, temperature, generator)
            keep = []
            for row, ((seq, i, s), token) in enumerate(zip(live, tokens.tolist())):
                texts[i][s].append(token)
                if token != stop_token:
                    keep.append(row)
            for row in set(range(len(live))) - set(keep):
                cache.free(live[row][0])
            live = [live[row] for row in keep]
            if not live or step + 1 == max_new_tokens:
                break
            if len(keep) < tokens.shape[0]:
                tokens = tokens[torch.tensor(keep, device=device)]
            logits = model.forward_cached(tokens, cache, cache.reserve([seq for seq, _, _ in live]))
    finally:
        for seq, _, _ in live:
            cache.free(seq)
    return texts


def main() -> None:
    from .model import ModelConfig, build_seeded_model

    config = ModelConfig(vocab_size=8192, block_size=512, n_layer=8, n_head=8, n_embd=512,
                         matmul_mode="int8", int8_backward=True)
    model = build_seeded_model(config, max_code=2, seed=1337).cuda().eval()
    prompts = [list(range(100, 140)), [7, 8, 9]]
    print("greedy ", generate(model, prompts, 16))
    draw = torch.Generator(device="cuda").manual_seed(1)
    print("sampled", generate(model, prompts, 16, samples=3, temperature=1.0, generator=draw))


if __name__ == "__main__":
    main()
