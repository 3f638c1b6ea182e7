"""Calls of the paged cache on several sequences that share pages: what one row does to a page's count is not seen by
another row of the same call."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
DEV = "cuda:0"
POOLS = ("k_codes", "k_scales", "k_g", "v_codes", "v_scales", "v_g")


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make(seqs, pages=600, page=16, H=2, per_seq=8):
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    return PagedNVFP4Cache(pages, page, H, D, seqs, per_seq, DEV)


def fill(c, s, T, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    k, v = (torch.randn(1, c.num_kv_heads, T, D, generator=g, device=DEV) for _ in range(2))
    c.append(k, v, seqs=i32(s))


@pytest.mark.parametrize("moving_first", [False, True])
@pytest.mark.parametrize("pairs", [1, 40])
def test_compact_refuses_a_shared_page_whatever_the_other_rows_drop(pairs, moving_first):
    """Sequences 2i and 2i + 1 hold the same two full pages.  In one call 2i drops the second page, which 2i + 1 would
    have to move tokens in: 2i + 1 is refused and stays as it was, in either order of the rows, every time."""
    for attempt in range(20):
        c = make(2 * pairs)
        for i in range(pairs):
            fill(c, 2 * i, 32, seed=i)
        c.fork(i32(*range(0, 2 * pairs, 2)), i32(*range(1, 2 * pairs, 2)))
        c.check()
        before = c.gather(32)
        table = c.page_table.clone()
        rows = [s for i in range(pairs) for s in ((2 * i + 1, 2 * i) if moving_first else (2 * i, 2 * i + 1))]
        keep = torch.zeros(2 * pairs, 16, dtype=torch.int32, device=DEV)
        keep[:, 0] = 3  # of the second page, token 3 ...
        counts = i32(*(s % 2 for s in rows))  # ... in 2i + 1; nothing in 2i
        c.compact(keep, counts, seqs=i32(*rows))
        with pytest.raises(RuntimeError, match="shared page"):
            c.check()
        assert c.lens.tolist() == [16, 32] * pairs, attempt
        assert torch.equal(c.page_table[1::2], table[1::2])
        assert (c.page_table[0::2, 1] == -1).all() and torch.equal(c.page_table[0::2, 0], table[0::2, 0])
        assert sorted(c.refs.tolist())[-2 * pairs:] == [1] * pairs + [2] * pairs
        for x, y in zip(c.gather(32), before):
            assert torch.equal(x[1::2], y[1::2]) and torch.equal(x[0::2, :, :16], y[0::2, :, :16])


def test_compact_of_no_tokens():
    """keep of width 0: tails say how much is dropped; a tail longer than the sequence is refused."""
    c = make(3)
    for s in range(3):
        fill(c, s, 20, seed=s)
    keep = torch.zeros(3, 0, dtype=torch.int32, device=DEV)
    c.compact(keep, i32(0, 0, 0), tails=i32(5, 21, 0))
    with pytest.raises(RuntimeError, match="keep list"):
        c.check()
    assert c.lens.tolist() == [15, 20, 20] and (c.refs > 0).sum() == 5
