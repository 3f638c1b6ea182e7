"""The paged cache and the attention over it beyond the first block of everything: more rows than a warp and than a block
looks at together, one list entry over more CTAs than a warp has lanes, chunks of hundreds of tokens over a cache that is
not empty, more pages and rows than the plan's block has threads.  Tolerances as in test_tree_attention_gpu.py."""
import random

import pytest
import torch

from test_tree_attention_gpu import build, check, rand_q

pytestmark = pytest.mark.gpu

D = 128
DEV = "cuda:0"


def i32(v):
    return torch.tensor(list(v), dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("B,N,dtype", [(33, 1, torch.bfloat16), (64, 5, torch.bfloat16), (100, 2, torch.float32),
                                       (300, 1, torch.float32), (300, 3, torch.float16)])
def test_batches(B, N, dtype):
    from fp4_attn_b200.paged_cache import tree_attention
    rng = random.Random(B * N)
    lens = [rng.choice([0, 1, 2, 17, rng.randint(3, 90), rng.randint(90, 700)]) for _ in range(B)]
    lens[0] = lens[31] = lens[-1] = 0
    c = build(lens, 2, 16, seed=B)
    q = rand_q(B, 6, N, dtype)
    counts = [min(N, n) for n in lens]
    o = tree_attention(q, c, counts=i32(counts))
    check(o, q, c, counts=counts)
    order = list(range(B))
    rng.shuffle(order)
    p = tree_attention(q[order], c, counts=i32(counts[s] for s in order), seqs=i32(order))
    check(p, q[order], c, counts=[counts[s] for s in order], seqs=order)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G,N", [(4, 1), (4, 20)])
def test_one_sequence_over_many_ctas(G, N, dtype):
    from fp4_attn_b200.paged_cache import tree_attention
    c = build([20011], 1, 64, seed=N)
    q = rand_q(1, G, N, dtype)
    check(tree_attention(q, c), q, c)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("page", [16, 128])
def test_a_chunk_of_a_prompt_over_a_cache(page, dtype):
    from fp4_attn_b200.paged_cache import tree_attention
    N = 700
    c = build([1100, 700, 2049], 2, page, seed=page)
    q = rand_q(3, 8, N, dtype)
    counts = [N, 333, N]
    check(tree_attention(q, c, counts=i32(counts)), q, c, counts=counts)


def test_more_pages_than_a_plan_reads_at_once():
    """The lowest free pages, behind more than 16384 that are taken; holes are filled first."""
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    c = PagedNVFP4Cache(40000, 16, 1, D, 3, 33000, DEV)
    T = 33000 * 16 - 5
    k = torch.zeros(1, 1, 1, D, device=DEV).expand(1, 1, T, D)
    c.append(k, k, seqs=i32([1]))
    c.check()
    assert torch.equal(c.page_table[1].cpu(), torch.arange(33000, dtype=torch.int32))
    t = torch.randn(1, 1, 200, D, device=DEV)
    c.append(t, t, seqs=i32([0]))
    c.check()
    assert c.page_table[0, :14].tolist() == list(range(33000, 33013)) + [-1]
    c.truncate(i32([20000 * 16]), seqs=i32([1]))
    c.append(t, t, seqs=i32([2]))
    c.check()
    assert c.page_table[2, :14].tolist() == list(range(20000, 20013)) + [-1]
    assert int((c.refs > 0).sum()) == 20000 + 13 + 13
    c.release(i32([0]))
    c.fork(i32([1]), i32([0]))
    c.check()
    assert torch.equal(c.page_table[0, :20000], c.page_table[1, :20000]) and int((c.refs == 2).sum()) == 20000
    for a, b in zip(c.gather(200, seqs=i32([2])), c.gather(200, seqs=i32([2]))):
        assert torch.equal(a, b) and a.any()


@pytest.mark.parametrize("R", [1024, 1025, 2500])
def test_more_rows_than_a_plan_takes_at_once(R):
    """Pages in order of (row, position), forks and compactions of all of them."""
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    rng = random.Random(R)
    c = PagedNVFP4Cache(8 * R, 16, 1, D, 2 * R, 4, DEV)
    g = torch.Generator(device=DEV).manual_seed(R)
    k, v = (torch.randn(R, 1, 40, D, generator=g, device=DEV) for _ in range(2))
    rows = list(range(R))
    rng.shuffle(rows)
    counts = [rng.choice([0, 1, 15, 16, 17, 40]) for _ in rows]
    c.append(k, v, seqs=i32(rows), counts=i32(counts))
    c.check()
    at = 0
    table = c.page_table.tolist()
    for s, n in zip(rows, counts):
        m = -(-n // 16)
        assert table[s] == list(range(at, at + m)) + [-1] * (4 - m)
        at += m
    dense = c.gather(40, seqs=i32(rows))
    c.fork(i32(rows), i32(R + s for s in rows))
    c.check()
    for a, b in zip(c.gather(40, seqs=i32(R + s for s in rows)), dense):
        assert torch.equal(a, b)
    refs = c.refs.tolist()
    assert sum(refs) == 2 * at and sum(r == 2 for r in refs) == sum(n // 16 for n in counts)
    # the last token of each copy, and nothing else of its last page
    tails = [min(n % 16, 3) for n in counts]
    keep = torch.tensor([[max(t - 1, 0), 0, 0] for t in tails], dtype=torch.int32, device=DEV)
    c.compact(keep, i32(min(t, 1) for t in tails), seqs=i32(R + s for s in rows), tails=i32(tails))
    c.check()
    after = c.gather(40, seqs=i32(R + s for s in rows))
    for i in range(0, R, 97):
        n, t = counts[i], tails[i]
        m = n - t + min(t, 1)
        assert int(c.lens[R + rows[i]]) == m
        for a, b in zip(after, dense):
            assert torch.equal(a[i, :, :n - t], b[i, :, :n - t]) and not a[i, :, m:].any()
            assert t == 0 or torch.equal(a[i, :, n - t], b[i, :, n - 1])
