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
