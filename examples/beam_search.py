"""A beam search as a server runs it: prompts of different lengths in one packed call, then for several beams of each the best
continuations, token by token, over 4-bit caches whose pages the beams share.

    python examples/beam_search.py

Prints each request's best sequences, and how far their scores are from those of the whole sequences at once with 16-bit keys and values.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from forge_amd import ops  # noqa: E402
from forge_amd.nn import DecoderAttention, Int4Linear, PagedBeams  # noqa: E402


class Decoder(torch.nn.Module):
    """Attention blocks between an embedding and a projection to the vocabulary, with random weights."""

    def __init__(self, vocab=1000, hidden=256, layers=2, heads=8, kv_heads=2, head_dim=64, device="cuda:0", seed=0):
        super().__init__()
        torch.manual_seed(seed)
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self.embed = torch.nn.Parameter(torch.randn(vocab, hidden).half(), requires_grad=False)
        self.blocks = torch.nn.ModuleList(DecoderAttention(hidden, heads, kv_heads, head_dim, 4096, 64) for _ in range(layers))
        self.head = Int4Linear(hidden, vocab, False, 64)
        self.to(device)
        for layer in [self.head] + [x for b in self.blocks for x in (b.qkv, b.out)]:
            layer.quantize_weight(torch.randn((layer.out_features, layer.in_features), device=device) * layer.in_features ** -0.5)

    def caches(self, pages, page_size):
        device = self.embed.device
        return [torch.zeros(ops.cache4_shape(pages, page_size, self.kv_heads, self.head_dim), dtype=torch.uint8, device=device)
                for _ in self.blocks]

    @torch.no_grad()
    def prompt(self, tokens, cu, positions, caches, slots):
        """Logits of packed prompts, whose keys and values go into the caches (pairs of 16-bit caches, or 4-bit ones)."""
        x = self.embed[tokens]
        for block, cache in zip(self.blocks, caches):
            k, v = cache if isinstance(cache, tuple) else (cache, None)
            x = x + block.prompt(x, cu, positions, k, v, slots)
        return self.head(x)

    @torch.no_grad()
    def next(self, tokens, caches, beams):
        """Logits of each row's newest token, which goes to beams.slots."""
        x = self.embed[tokens.clamp_min(0)][:, None]
        for block, cache in zip(self.blocks, caches):
            x = x + block.cached(x, beams.lens, cache, None, beams.slots, beams.table, beams.lens)
        return self.head(x[:, 0])


def search(model, prompts, width, steps, end_token, page_size=16):
    """prompts: lists of tokens. Returns each request's beams, best first: sequences behind the prompt (requests, beams, steps), and
    their scores."""
    device = model.embed.device
    lens = [len(p) for p in prompts]
    longest = max(lens) + steps
    per_row = longest // page_size + 2
    beams = PagedBeams(len(prompts), width, 2 * len(prompts) * width * per_row, page_size, longest, device)
    caches = model.caches(beams.refs.shape[0], page_size)
    slots = beams.start(lens)
    cu = torch.tensor([0] + lens, device=device).cumsum(0).to(torch.int32)
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).to(device)
    logits = model.prompt(torch.tensor(sum(prompts, []), device=device), cu, positions, caches, slots)
    logits = logits[(cu[1:] - 1).long()][:, None].expand(-1, width, -1)          # only the first row of each counts yet
    found = torch.zeros((len(prompts), width, 0), dtype=torch.int32, device=device)
    for i in range(steps):
        tokens, parents = beams.step(logits, caches, end_token)
        found = torch.cat([found.gather(1, parents.clamp_min(0).long()[..., None].expand(-1, -1, i)), tokens[..., None]], -1)
        if i + 1 < steps:
            logits = model.next(tokens.flatten(), caches, beams).view(len(prompts), width, -1)
    return found, beams.scores


def score(model, prompt, tokens, end_token):
    """The score of one sequence behind its prompt, from all of it at once with 16-bit keys and values."""
    device = model.embed.device
    if end_token in tokens:
        tokens = tokens[:tokens.index(end_token) + 1]
    whole = prompt + tokens
    n, page = len(whole), 16
    at = torch.arange(n, dtype=torch.int32, device=device)
    shape = ((n + page - 1) // page, page, model.kv_heads, model.head_dim)
    caches = [(torch.zeros(shape, dtype=torch.float16, device=device), torch.zeros(shape, dtype=torch.float16, device=device))
              for _ in model.blocks]
    logits = model.prompt(torch.tensor(whole, device=device), torch.tensor([0, n], dtype=torch.int32, device=device), at, caches, at)
    logp = torch.log_softmax(logits.double(), -1)
    return sum(logp[len(prompt) - 1 + i, t].item() for i, t in enumerate(tokens))


def main():
    model = Decoder()
    torch.manual_seed(1)
    prompts = [torch.randint(1000, (n,)).tolist() for n in (37, 5, 130)]
    found, scores = search(model, prompts, 4, 12, end_token=7)
    worst = 0.0
    for b, prompt in enumerate(prompts):
        best = found[b, 0].tolist()
        print(f"request {b}: score {scores[b, 0].item():.3f}, tokens {best}")
        for w in range(found.shape[1]):
            worst = max(worst, abs(score(model, prompt, found[b, w].tolist(), 7) - scores[b, w].item()))
    print("largest difference to the scores of whole sequences with 16-bit keys and values: %.3f" % worst)
    return found, scores, worst


if __name__ == "__main__":
    main()
