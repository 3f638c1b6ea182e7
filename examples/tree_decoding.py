"""Generation with drafted trees over the paged NVFP4 cache, checked against generation token by token.

A small random transformer generates for a ragged batch in two ways with the
same random numbers (one per position):

* token by token: append the last token's K and V, attend, sample;
* with trees: a drafter proposes a tree of continuations; its tokens' K and V are appended,
  ``tree_attention`` attends with the tree's mask, ``sample`` says what the model
  says after every node, ``accept_tree`` walks the tree as far as it agrees,
  and ``compact`` keeps the accepted tokens and frees the pages of the rest.

Nothing in a step waits for the host.  A token's K, V and query are quantized by
themselves and P is not quantized, so what else was drafted changes a token's
output in its last places only (the order of sums and the maximum that weights
are rounded under are those of the call): both ways generate the same tokens
unless a random number lies that near a boundary between two.  The beam at the
end forks a sequence (its full pages are shared) and frees it.

    python examples/tree_decoding.py [--steps 48] [--nodes 9]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from fp4_attn_b200.paged_cache import PagedNVFP4Cache, tree_attention, tree_mask  # noqa: E402
from fp4_attn_b200.sampling import accept_tree, sample  # noqa: E402

HEAD_DIM = 128


class Model:
    """A random decoder: RMS norm, attention with grouped heads and RoPE, gated MLP; fp32."""

    def __init__(self, layers=2, hidden=256, heads=4, kv_heads=2, vocab=101, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g) / s[-1] ** 0.5).to(device)  # noqa: E731
        self.heads, self.kv_heads, self.vocab, self.device = heads, kv_heads, vocab, torch.device(device, 0)
        self.embed, self.head = w(vocab, hidden) * hidden ** 0.5, w(vocab, hidden) * 2.0
        self.layers = [dict(q=w(heads * HEAD_DIM, hidden), k=w(kv_heads * HEAD_DIM, hidden),
                            v=w(kv_heads * HEAD_DIM, hidden), o=w(hidden, heads * HEAD_DIM),
                            up=w(2 * hidden, hidden), gate=w(2 * hidden, hidden), down=w(hidden, 2 * hidden))
                       for _ in range(layers)]
        self.freq = 10000.0 ** (-torch.arange(0, HEAD_DIM, 2, device=device) / HEAD_DIM)

    def caches(self, batch, tokens, page_size=16):
        per = -(-tokens // page_size)
        return [PagedNVFP4Cache(num_pages=2 * batch * per, page_size=page_size, num_kv_heads=self.kv_heads,
                                head_dim=HEAD_DIM, max_seqs=2 * batch, max_pages_per_seq=per, device=self.device)
                for _ in self.layers]

    def rope(self, x, positions):  # [B, N, H, D]
        a = positions[:, :, None, None] * self.freq
        x1, x2 = x.chunk(2, -1)
        return torch.cat((x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()), -1)

    def forward(self, tokens, positions, caches, mask=None, counts=None):
        """Appends tokens [B, N] (row b: its first counts[b]) to the caches; logits [B, N, vocab]."""
        norm = lambda x: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
        B, N = tokens.shape
        x = self.embed[tokens]
        for w, cache in zip(self.layers, caches):
            y = norm(x)
            q = self.rope((y @ w["q"].T).view(B, N, self.heads, HEAD_DIM), positions)
            k = self.rope((y @ w["k"].T).view(B, N, self.kv_heads, HEAD_DIM), positions)
            v = (y @ w["v"].T).view(B, N, self.kv_heads, HEAD_DIM)
            cache.append(k.transpose(1, 2), v.transpose(1, 2), counts=counts)
            o = tree_attention(q.transpose(1, 2), cache, mask=mask, counts=counts)
            x = x + o.flatten(2) @ w["o"].T
            y = norm(x)
            x = x + (torch.nn.functional.silu(y @ w["gate"].T) * (y @ w["up"].T)) @ w["down"].T
        return norm(x) @ self.head.T


SAMPLING = dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.01)


def prefill(model, prompt, lengths, caches, u):
    """The prompts enter the caches in one call; the token after each is sampled."""
    B, T = prompt.shape
    positions = torch.arange(T, device=prompt.device).expand(B, T)
    # the ragged prompts' nodes are their sequences' last tokens: all of them, at the front of the row
    logits = model.forward(prompt, positions, caches, counts=lengths)
    last = logits.gather(1, (lengths.long() - 1)[:, None, None].expand(B, 1, model.vocab))
    return sample(last[:, 0], u.gather(1, lengths.long()[:, None])[:, 0], **SAMPLING)[0]


def token_by_token(model, prompt, lengths, u, steps):
    B, T = prompt.shape
    caches = model.caches(B, T + steps + 2)
    token = prefill(model, prompt, lengths, caches, u)
    out = [token]
    for _ in range(steps - 1):
        pos = caches[0].lens[:B].long()[:, None]
        logits = model.forward(token[:, None], pos, caches)
        token = sample(logits[:, 0], u.gather(1, pos + 1)[:, 0], **SAMPLING)[0]
        out.append(token)
    for c in caches:
        c.check()
    return torch.stack(out, 1), caches


def with_trees(model, prompt, lengths, u, steps, draft, nodes):
    """draft(context positions [B]) -> (tokens [B, nodes - 1], parents [B, nodes]); returns (tokens [B, steps], calls)."""
    B, T = prompt.shape
    caches = model.caches(B, T + steps + 2 * nodes + 2)
    token = prefill(model, prompt, lengths, caches, u)
    out = torch.full((B, steps + nodes + 1), -1, dtype=torch.long, device=prompt.device)
    out[:, 0] = token
    done = torch.ones(B, dtype=torch.long, device=prompt.device)  # tokens generated
    calls = 0
    while int(done.min()) < steps:  # the loop's own end is the only thing that the host waits for
        drafted, parents = draft(done)
        tokens = torch.cat((token[:, None], drafted), 1)
        mask = tree_mask(parents)
        pos = caches[0].lens[:B].long()[:, None] + mask.sum(-1) - 1
        logits = model.forward(tokens, pos, caches, mask=mask)
        said, _ = sample(logits, u.gather(1, pos + 1), **SAMPLING)
        keep, n, token = accept_tree(parents, tokens, said)
        # a row that has enough keeps its root only, so that its cache stays in bounds
        full = done >= steps
        n = torch.where(full, 0, n)
        for c in caches:
            c.compact(keep, n)
        # what the kept nodes said: the accepted tokens and the one after them
        got = said.gather(1, keep.long())
        j = torch.arange(nodes, device=prompt.device)
        at = torch.where(j < n[:, None], done[:, None] + j, out.shape[1] - 1)
        out.scatter_(1, at, got)
        done = done + n
        calls += 1
    for c in caches:
        c.check()
    return out[:, :steps], calls


def drafter(truth, nodes, vocab, hit=0.7, seed=1):
    """Trees around a guess that is right with probability `hit`: a chain of guesses with a wrong sibling at each level."""
    B, steps = truth.shape
    g = torch.Generator(device=truth.device).manual_seed(seed)
    parents = torch.full((B, nodes), -1, dtype=torch.int32, device=truth.device)
    parents[:, 1:3] = 0
    for j in range(3, nodes):
        parents[:, j] = 1 + 2 * ((j - 1) // 2 - 1)  # under the last level's guess

    def draft(done):
        j = torch.arange(1, nodes, device=truth.device)
        level = (j - 1) // 2
        guess = truth.gather(1, (done[:, None] + level).clamp(max=steps - 1))
        wrong = torch.randint(vocab, guess.shape, generator=g, device=truth.device)
        right = (torch.rand(guess.shape, generator=g, device=truth.device) < hit) & (j % 2 == 1)
        return torch.where(right, guess, wrong), parents

    return draft


def run(steps=48, nodes=9, batch=3, device="cuda"):
    """-> (tokens token by token, tokens with trees, calls with trees)."""
    model = Model(device=device)
    g = torch.Generator().manual_seed(7)
    lengths = torch.tensor([21, 5, 40, 33, 1, 18][:batch], dtype=torch.int32)
    prompt = torch.randint(model.vocab, (batch, int(lengths.max())), generator=g).to(device)
    u = torch.rand(batch, 40 + steps + 3 * nodes, generator=g).to(device)
    lengths = lengths.to(device)
    one, caches = token_by_token(model, prompt, lengths, u, steps)
    trees, calls = with_trees(model, prompt, lengths, u, steps, drafter(one, nodes, model.vocab), nodes)
    # a beam: sequence 0 continues as sequence `batch` too, on the same pages, and goes again
    ids = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    for c in caches:
        held = int((c.refs > 0).sum())
        c.fork(ids(0), ids(batch))
        shared = int((c.refs > 1).sum())
        c.release(ids(batch))
        c.check()
        assert shared == int(c.lens[0]) // c.page_size and int((c.refs > 0).sum()) == held
    return one, trees, calls


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=48)
    ap.add_argument("--nodes", type=int, default=9)
    args = ap.parse_args()
    one, trees, calls = run(args.steps, args.nodes)
    print(f"{args.steps} tokens for each of {one.shape[0]} sequences: {args.steps} calls token by token, {calls} with trees "
          f"of {args.nodes}; the same tokens: {bool(torch.equal(one, trees))}")
