"""The C entries of the paged cache, its attention and sampling refuse bad arguments with a status and a message,
before any CUDA work (no GPU needed)."""
import ctypes

import pytest

P = ctypes.c_void_p(256)


def lib():
    from fp4_attn_b200 import _lib
    return _lib.load()


def cache(**kw):
    from fp4_attn_b200.paged_cache import _Struct
    v = dict(k_codes=256, k_scales=256, k_g=256, v_codes=256, v_scales=256, v_g=256, page_table=256, lens=256, refs=256,
             status=256, work=256, num_pages=10, page_size=16, num_kv_heads=2, head_dim=128, max_seqs=4, max_pages=8)
    v.update(kw)
    return _Struct(**v)


def ref(c):
    return ctypes.addressof(c)


@pytest.mark.parametrize("kw,code,message", [
    (dict(k_codes=None), 1, b"null"), (dict(lens=None), 1, b"null"), (dict(v_g=260), 1, b"aligned"),
    (dict(head_dim=64), 3, b"head_dim"), (dict(page_size=48), 1, b"page_size"), (dict(num_pages=0), 1, b"shape"),
    (dict(num_kv_heads=0), 1, b"shape"), (dict(max_pages=1 << 28), 1, b"2^31")])
def test_every_entry_checks_the_cache(kw, code, message):
    L = lib()
    c = cache(**kw)
    for call in (lambda: L.fp4paged_append(ref(c), P, P, 1, 1, 1, 0, 0, 0, 0, 0, 0, None, None, None),
                 lambda: L.fp4paged_truncate(ref(c), None, None, 1, None),
                 lambda: L.fp4paged_compact(ref(c), P, P, None, None, 1, 1, None),
                 lambda: L.fp4paged_fork(ref(c), P, P, 1, 0, None),
                 lambda: L.fp4paged_gather(ref(c), P, P, 1, None, 1, 1, None),
                 lambda: L.fp4paged_attention(ref(c), P, 1, 1, 2, 1, 0, 0, 0, None, 0, 0, 0, None, None, 0.1, P, 1, P,
                                              1 << 30, None)):
        assert call() == code
        assert message in L.fp4attn_last_error()
    assert L.fp4paged_truncate(None, None, None, 1, None) == 1 and b"cache is null" in L.fp4attn_last_error()


def test_arguments():
    L = lib()
    c = cache()
    assert L.fp4paged_work_size(10, 4) == 3 * 4 + 4 + 2 * 10 and L.fp4paged_work_size(0, 4) == -1
    assert L.fp4paged_append(ref(c), None, P, 1, 1, 1, 0, 0, 0, 0, 0, 0, None, None, None) == 1
    assert L.fp4paged_append(ref(c), P, P, 7, 1, 1, 0, 0, 0, 0, 0, 0, None, None, None) == 1
    assert b"dtype" in L.fp4attn_last_error()
    assert L.fp4paged_append(ref(c), P, P, 1, 5, 1, 0, 0, 0, 0, 0, 0, None, None, None) == 1  # more rows than sequences
    assert L.fp4paged_append(ref(c), P, P, 1, 0, 1, 0, 0, 0, 0, 0, 0, None, None, None) == 0  # nothing to do
    assert L.fp4paged_compact(ref(c), None, P, None, None, 1, 1, None) == 1
    assert L.fp4paged_fork(ref(c), None, P, 1, 0, None) == 1
    assert L.fp4paged_gather(ref(c), P, ctypes.c_void_p(264), 1, None, 1, 1, None) == 1

    def attend(B=1, Hq=4, N=1, q=P, out=P, ws=P, size=1 << 30, dt=1, odt=1):
        return L.fp4paged_attention(ref(c), q, dt, B, Hq, N, 0, 0, 0, None, 0, 0, 0, None, None, 0.1, out, odt, ws, size,
                                    None)

    assert attend(Hq=3) == 1 and b"query heads" in L.fp4attn_last_error()
    assert attend(q=None) == 1 and attend(out=None) == 1 and attend(ws=None) == 1
    assert attend(dt=3) == 1 and attend(odt=-1) == 1 and b"dtype" in L.fp4attn_last_error()
    need = L.fp4paged_attention_workspace_size(1, 4, 2, 1)
    assert need > 0 and attend(size=need - 1) == 1 and b"workspace" in L.fp4attn_last_error()
    assert attend(ws=ctypes.c_void_p(264)) == 1 and attend(N=0) == 0
    assert L.fp4paged_attention_workspace_size(1, 3, 2, 1) == -1


def test_sampling_arguments():
    L = lib()

    def go(x=P, dt=0, R=1, V=10, ld=10, u=P, tokens=P):
        return L.fp4_sample(x, dt, R, V, ld, u, None, None, None, None, tokens, None, None)

    assert go(x=None) == 1 and go(u=None) == 1 and go(tokens=None) == 1 and b"null" in L.fp4attn_last_error()
    assert go(V=0) == 1 and go(R=-1) == 1 and go(ld=-1) == 1
    assert go(V=262145, ld=262145) == 3 and b"logits" in L.fp4attn_last_error()
    assert go(dt=5) == 1 and go(R=0) == 0
    assert L.fp4_accept_tree(None, P, P, None, 1, 1, P, P, P, None) == 1
    assert L.fp4_accept_tree(P, P, P, None, 1, 0, P, P, P, None) == 1
    assert L.fp4_accept_tree(P, P, P, None, 0, 1, P, P, P, None) == 0


def test_python_refuses_cpu_tensors():
    import torch
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    from fp4_attn_b200.sampling import accept_tree, sample
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedNVFP4Cache(4, 16, 1, 128, 1, 1, "cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        sample(torch.zeros(1, 4), torch.zeros(1))
    z = torch.zeros(1, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        accept_tree(z.int(), z, z)


def test_tree_mask_follows_the_parents():
    import torch
    from fp4_attn_b200.paged_cache import tree_mask
    parents = torch.tensor([[-1, 0, 0, 1, 3, 2], [-1, 0, 1, 2, 3, 4]])
    m = tree_mask(parents)
    assert m[0, 4].tolist() == [True, True, False, True, True, False]
    assert m[0, 5].tolist() == [True, False, True, False, False, True]
    assert torch.equal(m[1], torch.ones(6, 6, dtype=torch.bool).tril())
