"""A decoder's attention block as a server runs it: prompts of different lengths in one packed call, then tokens one
at a time, then trees of drafted tokens verified in one call, all over one paged cache.

    python examples/decoder_attention.py

Prints, for each phase, how far it is from the same block over each whole sequence at once.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from forge_amd.nn import DecoderAttention, tree_masks  # noqa: E402


class Pages:
    """A paged cache: hands out pages in any order and knows where each sequence's tokens lie."""

    def __init__(self, sequences, max_len, page, kv_heads, head_dim, dtype, device):
        width = (max_len + page - 1) // page
        self.page = page
        self.k = torch.zeros((sequences * width, page, kv_heads, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.table = torch.randperm(sequences * width).view(sequences, width).to(torch.int32).to(device)

    def slots(self, sequence, positions):
        """Cache rows of positions (int64, on the device) of a sequence."""
        return (self.table[sequence, positions // self.page].long() * self.page + positions % self.page).to(torch.int32)


def run(block, x, prompt_lens, steps, parents, device):
    """x: per sequence a (prompt + steps + drafts, hidden) tensor of token vectors. Returns the outputs of the
    prompts (packed), of the single steps (B, steps, hidden) and of the drafts (B, T, hidden)."""
    B, T = parents.shape
    lens = torch.tensor(prompt_lens, device=device)
    cache = Pages(B, max(prompt_lens) + steps + T, 16, block.kv_heads, block.head_dim, x[0].dtype, device)

    def at(first, n):
        """positions and slots of n tokens of each sequence from position first[b] on, as (B * n,) tensors."""
        pos = first[:, None] + torch.arange(n, device=device)
        return pos.flatten().to(torch.int32), torch.stack([cache.slots(b, pos[b]) for b in range(B)]).flatten()

    # the prompts, packed
    cu = torch.zeros(B + 1, dtype=torch.int32, device=device)
    cu[1:] = lens.cumsum(0)
    pos = torch.cat([torch.arange(n, device=device) for n in prompt_lens])
    slots = torch.cat([cache.slots(b, torch.arange(n, device=device)) for b, n in enumerate(prompt_lens)])
    prompt = block.prompt(torch.cat([t[:n] for t, n in zip(x, prompt_lens)]), cu, pos.to(torch.int32), cache.k, cache.v, slots)

    # one token at a time
    outs = []
    for i in range(steps):
        now = torch.stack([t[n + i] for t, n in zip(x, prompt_lens)])[:, None]
        pos, slots = at(lens + i, 1)
        outs.append(block.cached(now, pos, cache.k, cache.v, slots, cache.table, (lens + i).to(torch.int32)))

    # a tree of drafts per sequence: a draft's position is its depth in the tree
    depth = torch.zeros((B, T), dtype=torch.int64)
    for b in range(B):
        for t in range(T):
            depth[b, t] = depth[b, parents[b, t]] + 1 if parents[b, t] >= 0 else 0
    first = lens + steps
    _, slots = at(first, T)
    pos = (first[:, None] + depth.to(device)).flatten().to(torch.int32)
    now = torch.stack([t[n + steps:n + steps + T] for t, n in zip(x, prompt_lens)])
    drafts = block.cached(now, pos, cache.k, cache.v, slots, cache.table, first.to(torch.int32), tree_masks(parents).to(device))
    return prompt, torch.cat(outs, 1) if outs else None, drafts


def make(device, dtype=torch.float16, hidden=512, heads=8, kv_heads=2, head_dim=64, group_size=64, seed=0):
    """A block with random weights."""
    torch.manual_seed(seed)
    block = DecoderAttention(hidden, heads, kv_heads, head_dim, 4096, group_size, dtype=dtype).to(device)
    for layer in (block.qkv, block.out):
        layer.quantize_weight(torch.randn((layer.out_features, layer.in_features), device=device) * layer.in_features ** -0.5)
    with torch.no_grad():
        for w in (block.q_norm, block.k_norm):
            w.copy_(torch.rand(head_dim) + 0.5)
    return block


def whole(block, x, device):
    """The block over one sequence at once."""
    n = x.shape[0]
    cache = Pages(1, n, 16, block.kv_heads, block.head_dim, x.dtype, device)
    pos = torch.arange(n, device=device)
    cu = torch.tensor([0, n], dtype=torch.int32, device=device)
    return block.prompt(x, cu, pos.to(torch.int32), cache.k, cache.v, cache.slots(0, pos))


def main():
    device = torch.device("cuda:0")
    block = make(device)
    prompt_lens, steps = [37, 300, 1, 130], 5
    parents = torch.tensor([[-1, 0, 0, 1, 1, 2, 5]] * 4)
    x = [torch.randn((n + steps + parents.shape[1], block.qkv.in_features), device=device).half() for n in prompt_lens]
    prompt, single, drafts = run(block, x, prompt_lens, steps, parents, device)
    worst = [0.0, 0.0, 0.0]
    start = 0
    for b, n in enumerate(prompt_lens):
        full = whole(block, x[b][:n + steps], device)
        worst[0] = max(worst[0], (prompt[start:start + n] - full[:n]).abs().max().item())
        worst[1] = max(worst[1], (single[b] - full[n:]).abs().max().item())
        start += n
        for t in range(parents.shape[1]):           # a draft sees the sequence and its own ancestors
            path = [t]
            while parents[b, path[0]] >= 0:
                path.insert(0, int(parents[b, path[0]]))
            branch = torch.cat([x[b][:n + steps], x[b][[n + steps + p for p in path]]])
            worst[2] = max(worst[2], (drafts[b, t] - whole(block, branch, device)[-1]).abs().max().item())
    print("largest output %.3f; largest difference to the whole sequence at once: prompts %.4f, single tokens %.4f, "
          "drafts %.4f" % (prompt.abs().max().item(), *worst))
    return worst


if __name__ == "__main__":
    main()
