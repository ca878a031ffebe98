"""Greedy decoding with drafted trees over a paged key/value cache.

A small decoder (random weights) answers a batch of prompts twice: token by token,
and with a tree of drafted tokens per step, of which the longest path that greedy
decoding would have taken is kept.  Both give the same tokens.  Run it on a B200:

    python examples/speculative_decode.py
"""

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "techjam-kernel_b200"))

from b200_attention import check_device_errors  # noqa: E402
from b200_attention.transformer import Decoder, DecoderConfig, init_normal_  # noqa: E402


def logits(model, hidden):
    return hidden.float() @ model.embed.weight.float().t()


def feed_prompts(model, cache, prompts):
    """Commit the prompts and return each one's next token."""
    batch, length = prompts.shape
    dev = prompts.device
    if int(cache.reserve(length)) != 0:
        raise RuntimeError("no pages for the prompts")
    hidden = model.cached_forward(prompts, cache)
    keep = torch.arange(length, dtype=torch.int32, device=dev).expand(batch, length).contiguous()
    cache.accept(keep, torch.full((batch,), length, dtype=torch.int32, device=dev))
    return logits(model, hidden[:, -1]).argmax(-1)


def decode(model, prompts, new_tokens):
    """One token a step."""
    batch, length = prompts.shape
    cache = model.new_cache(batch, length + new_tokens + 1)
    token = feed_prompts(model, cache, prompts)
    answer = [token]
    first = torch.zeros(batch, 1, dtype=torch.int32, device=prompts.device)
    one = torch.ones(batch, dtype=torch.int32, device=prompts.device)
    for _ in range(new_tokens - 1):
        cache.reserve(1)
        hidden = model.cached_forward(token[:, None], cache)
        cache.accept(first, one)
        token = logits(model, hidden[:, 0]).argmax(-1)
        answer.append(token)
    return torch.stack(answer, 1)


def tree(branches, depth, device):
    """Parents, depths and ancestor mask of a root with ``branches`` chains of ``depth``."""
    parent, level = [-1], [0]
    for b in range(branches):
        for d in range(depth):
            parent.append(0 if d == 0 else len(parent) - 1)
            level.append(d + 1)
    n = len(parent)
    mask = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        if parent[i] >= 0:
            mask[i] = mask[parent[i]]
        mask[i, i] = True
    return parent, level, mask.to(device)


def speculate(model, prompts, new_tokens, draft, branches=3, depth=3):
    """A tree of drafted tokens a step.  ``draft(tokens, branches, depth)`` proposes
    continuations [batch, branches, depth] of the last tokens [batch]."""
    batch, length = prompts.shape
    dev = prompts.device
    parent, _, mask = tree(branches, depth, dev)
    nodes = len(parent)
    cache = model.new_cache(batch, length + new_tokens + nodes + depth + 1)
    token = feed_prompts(model, cache, prompts)
    answers = [[int(t)] for t in token]
    steps = 0
    while min(len(a) for a in answers) < new_tokens:
        drafted = torch.cat([token[:, None], draft(token, branches, depth).reshape(batch, -1)], 1)
        if int(cache.reserve(nodes)) != 0:
            raise RuntimeError("no pages left")
        hidden = model.cached_forward(drafted, cache, mask)
        best = logits(model, hidden).argmax(-1).tolist()
        told = drafted.tolist()
        paths = torch.zeros(batch, depth + 1, dtype=torch.int32)
        counts = torch.zeros(batch, dtype=torch.int32)
        for b in range(batch):
            if len(answers[b]) >= new_tokens:
                continue
            path = [0]  # the root is the model's own last token
            while True:
                at = path[-1]
                answers[b].append(best[b][at])
                child = [i for i in range(nodes) if parent[i] == at and told[b][i] == best[b][at]]
                if not child or len(answers[b]) >= new_tokens:
                    break
                path.append(child[0])
            paths[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
            counts[b] = len(path)
        cache.accept(paths.to(dev), counts.to(dev))
        token = torch.tensor([a[-1] for a in answers], device=dev)
        steps += 1
    check_device_errors(dev)
    return torch.tensor([a[:new_tokens] for a in answers], device=dev), steps


def main():
    dev = torch.device("cuda")
    config = DecoderConfig(batch_size=4, seq_len=48, d_model=256, num_heads=4, ffn_dim=512,
                           num_layers=3, causal=True, vocab_size=97)
    model = init_normal_(Decoder(config), std=0.2, seed=0).to(dev).eval()
    prompts = torch.randint(0, 97, (4, 48), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        plain = decode(model, prompts, 40)
        # a drafter that knows half of the answer: the true continuation on one branch
        follows = {}
        for row in plain.tolist():
            for x, y in zip(row, row[1:]):
                follows.setdefault(x, []).append(y)

        def draft(tokens, branches, depth):
            out = torch.zeros(len(tokens), branches, depth, dtype=torch.long)
            for i, t in enumerate(tokens.tolist()):
                for b in range(branches):
                    at = t
                    for d in range(depth):
                        known = follows.get(at, [0])
                        at = known[b % len(known)]
                        out[i, b, d] = at
            return out.to(dev)

        fast, steps = speculate(model, prompts, 40, draft)
    print(f"{plain.shape[1]} tokens in {steps} tree steps; same tokens: {torch.equal(plain, fast)}")
    return 0 if torch.equal(plain, fast) else 1


if __name__ == "__main__":
    sys.exit(main())
