"""Which sequences a call names: indexes out of range and sequences named twice."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
DEV = "cuda:0"


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make(lens, pages=64, page=16, H=2, per_seq=8):
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    c = PagedNVFP4Cache(pages, page, H, D, len(lens), per_seq, DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn(len(lens), H, max(lens), D, generator=g, device=DEV) for _ in range(2))
    c.append(k, v, counts=i32(*lens))
    c.check()
    return c


@pytest.mark.parametrize("bad", [3, -1, 1 << 30])
def test_reads_of_a_sequence_out_of_range(bad):
    """tree_attention and gather give zeros for it, the others' rows, and the error bit."""
    from fp4_attn_b200.paged_cache import tree_attention
    c = make([40, 20, 33])
    q = torch.randn(3, 4, 2, D, device=DEV)
    want = tree_attention(q, c, seqs=i32(2, 0, 1))
    kw, vw = c.gather(40, seqs=i32(2, 0, 1))
    c.check()
    o = tree_attention(q, c, seqs=i32(2, bad, 1))
    with pytest.raises(RuntimeError, match="out of range"):
        c.check()
    assert torch.equal(o[[0, 2]], want[[0, 2]]) and not o[1].any()
    k, v = c.gather(40, seqs=i32(2, bad, 1))
    with pytest.raises(RuntimeError, match="out of range"):
        c.check()
    for x, y in ((k, kw), (v, vw)):
        assert torch.equal(x[[0, 2]], y[[0, 2]]) and not x[1].any()
    # several rows may read one sequence
    o = tree_attention(q, c, seqs=i32(2, 2, 1))
    c.check()
    assert torch.equal(o[[0, 2]], want[[0, 2]])


POOLS = ("k_codes", "k_scales", "k_g", "v_codes", "v_scales", "v_g")


def state(c):
    return [getattr(c, n).clone() for n in POOLS + ("page_table", "lens", "refs")]


@pytest.mark.parametrize("many", [0, 1500])
def test_a_sequence_named_twice_by_a_call_that_changes_it(many):
    """append and fork are refused as a whole, truncate, release and compact for the sequence named twice; the calls
    after it find the cache in order."""
    lens = [40, 20, 33] + [0] * (many + 3)
    c = make(lens, pages=64 + many)
    empty = list(range(5, 5 + many))  # further rows, so that the two are far apart
    rows = i32(1, *empty, 0, 1)

    def refused(call):
        call()
        with pytest.raises(RuntimeError, match="named twice"):
            c.check()

    was = state(c)
    n = len(rows)
    t = torch.randn(n, 2, 3, D, device=DEV)
    refused(lambda: c.append(t, t, seqs=rows))
    refused(lambda: c.append(t, t, seqs=rows, counts=i32(3, *([0] * (n - 1)))))
    refused(lambda: c.fork(i32(*([0] * n)), i32(3, *empty, 4, 3)))
    refused(lambda: c.fork(i32(*([0] * n)), i32(3, *empty, 4, 3), deep=True))
    assert all(torch.equal(a, b) for a, b in zip(was, state(c)))
    refused(lambda: c.truncate(i32(2, *([0] * many), 40, 1), seqs=rows))
    refused(lambda: c.release(i32(1, *empty, 1)))
    keep = torch.zeros(n, 4, dtype=torch.int32, device=DEV)
    keep[:, 0] = 2
    counts = i32(1, *([0] * many), 0, 1)
    refused(lambda: c.compact(keep, counts, seqs=rows, tails=i32(4, *([0] * many), 0, 4)))
    assert all(torch.equal(a, b) for a, b in zip(was, state(c)))
    # the rows beside the two are carried out
    refused(lambda: c.truncate(i32(2, *([0] * many), 17, 1), seqs=rows))
    assert c.lens.tolist()[:3] == [17, 20, 33] and int(c.page_table[0, 2]) == -1
    assert (c.refs > 0).sum() == 2 + 2 + 3 and (c.refs >= 0).all()
    # each once, in any order
    c.truncate(i32(2, *([0] * many), 1), seqs=i32(1, *empty, 0))
    c.append(t[:many + 2], t[:many + 2], seqs=i32(1, *empty, 0), counts=i32(1, *([0] * many), 3))
    c.compact(keep[:2], i32(1, 1), seqs=i32(2, 0), tails=i32(4, 3))
    c.fork(i32(1, *([4] * many), 2), i32(3, *empty, 4))
    c.check()
    assert c.lens.tolist()[:5] == [2, 3, 30, 3, 30] and (c.refs >= 0).all()
