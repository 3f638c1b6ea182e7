"""Attention of drafted tokens over the paged cache against the formula in 64 bits.

Tolerance, element by element, from the formula o = sum p v:
  |o - ref| <= u |ref| + e sum p |v| + T f max(p g)
with u the unit roundoff of the output type and e what p may be off by, relative:
the rounding of p to one fp16 (2^-12; fp32 outputs: two fp16, 2^-22) and the
error of the exponent, whose argument |S| log2(e) has a few 32-bit roundings
(2^-21 max|S| log2(e) covers three), doubled for the sum in the denominator.
The products p g_v (g_v: the token's global scale, at least its |v|) are held
in fp16, scaled so that the row's largest is 2^9 to 2^15: half of fp16's smallest
step is then 2^-34 to 2^-40 of it.  f = 2^-36 a token, since T such roundings do
not all go one way; they add up to T f of the largest.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}


def build(lens, H, page, seed=0, spare=5, per_seq=None):
    """A cache whose sequences have lens tokens in scattered pages (filled in rounds that interleave sequences)."""
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    g = torch.Generator(device=DEV).manual_seed(seed)
    per = per_seq or max(1, max(-(-n // page) for n in lens))
    c = PagedNVFP4Cache(sum(-(-n // page) for n in lens) + spare, page, H, D, len(lens), per, DEV)
    done = [0] * len(lens)
    while any(d < n for d, n in zip(done, lens)):
        T = max(1, min(max(lens), 4 * page + 3))
        cnt = [min(T, n - d) for d, n in zip(done, lens)]
        k = torch.randn(len(lens), T, H, D, generator=g, device=DEV).transpose(1, 2)
        v = (torch.randn(len(lens), T, H, D, generator=g, device=DEV) *
             torch.exp(torch.randn(len(lens), T, 1, 1, generator=g, device=DEV))).transpose(1, 2)
        c.append(k, v, counts=torch.tensor(cnt, dtype=torch.int32, device=DEV))
        done = [d + n for d, n in zip(done, cnt)]
    c.check()
    return c


def quant64(q):
    """The NVFP4 values of q's tokens ([B, Hq, N, D], per token over all heads) in 64 bits."""
    from oracle import quant as oq
    B, H, N, _ = q.shape
    x = q.transpose(1, 2).reshape(B * N, H * D).float().cpu().numpy()
    out = oq.fused_qdq(x, "row", "float32")[0]
    return torch.from_numpy(out).double().view(B, N, H, D).transpose(1, 2).to(DEV)


def reference(q, c, mask, counts, scaling, seqs=None):
    """(ref, sum p |v|, T max(p g), max |S|) in 64 bits, [B, N, Hq, D]."""
    B, Hq, N, _ = q.shape
    H = c.num_kv_heads
    qh = quant64(q)
    ref = torch.zeros(B, N, Hq, D, dtype=torch.float64, device=DEV)
    size, top = torch.zeros_like(ref), torch.zeros_like(ref)
    smax = 0.0
    K, V = c.gather(max(1, int(c.lens.max())))
    for b in range(B):
        s = b if seqs is None else seqs[b]
        n = N if counts is None else counts[b]
        L = int(c.lens[s])
        k, v = K[s, :, :L].double().repeat_interleave(Hq // H, 0), V[s, :, :L].double().repeat_interleave(Hq // H, 0)
        S = qh[b, :, :n] @ k.transpose(1, 2) * scaling
        seen = torch.ones(n, L, dtype=torch.bool, device=DEV)
        if n:
            m = torch.ones(n, n, dtype=torch.bool, device=DEV).tril() if mask is None else \
                (mask if mask.dim() == 2 else mask[b])[:n, :n]
            seen[:, L - n:] = m
        S = S.masked_fill(~seen, -math.inf)
        if L and n:
            smax = max(smax, float(torch.where(torch.isfinite(S), S, 0.0).abs().max()))
            p = torch.nan_to_num(torch.softmax(S, -1), 0.0)
            ref[b, :n] = (p @ v).transpose(0, 1)
            size[b, :n] = (p @ v.abs()).transpose(0, 1)
            top[b, :n] = L * (p * V[s, :, :L].double().abs().amax((0, 2))).amax(-1).transpose(0, 1)[..., None]
    return ref, size, top, smax


def check(o, q, c, mask=None, counts=None, scaling=D ** -0.5, seqs=None):
    from fp4_attn_b200.gemm import device_status
    assert device_status() == 0
    ref, size, top, smax = reference(q, c, mask, counts, scaling, seqs)
    e = (2.0 ** -11 if o.dtype != torch.float32 else 2.0 ** -20) + 2.0 ** -20 * smax * 1.4427
    tol = U[o.dtype] * ref.abs() + e * size + 2.0 ** -36 * top + 2.0 ** -24 * (o.dtype == torch.float16)
    err = (o.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-30)).max())


def rand_q(B, Hq, N, dtype, seed=1, scale=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (scale * torch.randn(B, Hq, N, D, generator=g, device=DEV)).to(dtype)


@pytest.mark.parametrize("Hq,H,N,lens,page,dtype", [
    (1, 1, 1, [1], 16, torch.float32),
    (4, 1, 1, [1, 2, 127, 128, 129, 700], 16, torch.bfloat16),
    (32, 8, 1, [777], 64, torch.bfloat16),
    (16, 1, 3, [3, 5, 300], 128, torch.float16),
    (14, 2, 9, [100, 9, 260, 1025], 32, torch.float32),
    (5, 5, 16, [16, 140, 400], 16, torch.bfloat16),
    (28, 4, 27, [27, 355, 128 + 27], 16, torch.float16),
    (6, 2, 50, [50, 500], 64, torch.float32),
    (64, 8, 64, [64, 1111], 128, torch.bfloat16),
    (3, 1, 200, [200, 333, 513], 32, torch.bfloat16),
    (40, 2, 70, [260], 16, torch.float32),
])
def test_chain(Hq, H, N, lens, page, dtype):
    from fp4_attn_b200.paged_cache import tree_attention
    c = build(lens, H, page, seed=N)
    q = rand_q(len(lens), Hq, N, dtype)
    o = tree_attention(q, c)
    assert o.dtype == dtype and o.shape == (len(lens), N, Hq, D)
    check(o, q, c)
    assert torch.equal(o, tree_attention(q, c))  # repeatable bit for bit


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Hq,H,N,lens,page", [(8, 2, 13, [13, 600, 141], 16), (8, 1, 33, [33, 1500], 128),
                                              (7, 7, 64, [64, 200], 32)])
def test_trees_and_ragged_counts(Hq, H, N, lens, page, dtype):
    from fp4_attn_b200.paged_cache import tree_attention, tree_mask
    g = torch.Generator().manual_seed(N)
    B = len(lens)
    c = build(lens, H, page, seed=N)
    q = rand_q(B, Hq, N, dtype)
    parents = torch.tensor([[-1] + [int(torch.randint(0, j, (1,), generator=g)) for j in range(1, N)] for _ in lens],
                           device=DEV)
    mask = tree_mask(parents)
    for b in range(B):  # the mask is what following the parents gives
        for i in (0, N // 2, N - 1):
            seen, at = set(), i
            while at >= 0:
                seen.add(at)
                at = int(parents[b, at])
            assert set(mask[b, i].nonzero().flatten().tolist()) == seen
    check(tree_attention(q, c, mask=mask), q, c, mask)
    check(tree_attention(q, c, mask=mask[0]), q, c, mask[0])
    t = mask.transpose(1, 2).contiguous().transpose(1, 2)  # another order of its axes
    assert torch.equal(tree_attention(q, c, mask=t), tree_attention(q, c, mask=mask))
    counts = [max(0, N - 4 * b * b - 1) if b else 0 for b in range(B)]
    ct = torch.tensor(counts, dtype=torch.int32, device=DEV)
    for m in (None, mask):
        o = tree_attention(q, c, mask=m, counts=ct)
        check(o, q, c, m, counts)
        for b in range(B):
            assert not o[b, counts[b]:].any()


def test_rows_that_see_nothing():
    """A mask that shows a node no key, on a sequence that has only its drafted tokens, gives 0; a node that sees one
    key gives that key's value."""
    from fp4_attn_b200.paged_cache import tree_attention
    c = build([6, 30], 2, 16)
    q = rand_q(2, 8, 6, torch.float32)
    mask = torch.zeros(6, 6, dtype=torch.bool, device=DEV)
    mask[2, 4] = True
    o = tree_attention(q, c, mask=mask)
    check(o, q, c, mask)
    assert not o[0, [0, 1, 3, 4, 5]].any()
    v = c.gather(6)[1][0, :, 4]
    assert torch.allclose(o[0, 2], v.repeat_interleave(4, 0), rtol=2.0 ** -20, atol=0)
    assert o[1].any(-1).all()


def test_sequences_and_empty_ones():
    from fp4_attn_b200.paged_cache import tree_attention
    c = build([300, 5, 140, 77], 2, 32)
    c.release(torch.tensor([1], dtype=torch.int32, device=DEV))
    q = rand_q(3, 4, 1, torch.bfloat16)
    seqs = [3, 1, 0]
    o = tree_attention(q, c, seqs=torch.tensor(seqs, dtype=torch.int32, device=DEV))
    assert not o[1].any()
    check(o[0::2], q[0::2], c, seqs=seqs[0::2])


def test_not_finite_tokens_stay_where_they_are_seen():
    """A NaN token of the cache reaches the nodes that see it and no other; a NaN query token only its own rows."""
    from fp4_attn_b200.paged_cache import tree_attention
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    for x in (0, 1):
        c = PagedNVFP4Cache(40, 16, 2, D, 1, 30, DEV)
        t = [torch.randn(1, 2, 200, D, device=DEV) for _ in range(2)]
        t[x][0, 1, 198, 3] = float("nan")  # node 2 of 4
        t[1 - x][0, 0, 199, 7] = float("inf")  # node 3
        c.append(*t)
        q = rand_q(1, 4, 4, torch.float32)
        mask = torch.eye(4, dtype=torch.bool, device=DEV)
        o = tree_attention(q, c, mask=mask)
        assert torch.isfinite(o[0, :2]).all() and torch.isnan(o[0, 2:]).all()
        c2 = PagedNVFP4Cache(40, 16, 2, D, 1, 30, DEV)
        for y in t:
            y[0, :, 198:] = 1.0
        c2.append(*t)
        assert torch.equal(tree_attention(q, c2, mask=mask)[0, :2], o[0, :2])
    q[0, 2, 1, 0] = float("nan")
    o = tree_attention(q, c2, mask=mask)
    assert torch.isnan(o[0, 1]).all() and torch.isfinite(o[0, [0, 2, 3]]).all()


def test_sharp_flat_and_shifting_scores():
    """One key far above the rest, equal scores, scores that grow along the sequence (the running maximum moves in
    every tile), values of very different sizes."""
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache, tree_attention
    T = 1500
    for case in range(4):
        g = torch.Generator(device=DEV).manual_seed(case)
        k = torch.randn(1, 1, T, D, generator=g, device=DEV)
        v = torch.randn(1, 1, T, D, generator=g, device=DEV)
        q = rand_q(1, 2, 1, torch.float32, seed=case)
        if case == 0:
            k[0, 0, 777] = 8 * q[0, 0, 0]
        elif case == 1:
            k[:] = 1.0
        elif case == 2:
            k = q[:, :1] * torch.linspace(-4, 4, T, device=DEV)[:, None] / 8
        else:
            v = v * torch.exp2(torch.linspace(-60, 60, T, device=DEV)[:, None])
        c = PagedNVFP4Cache(100, 16, 1, D, 1, 100, DEV)
        c.append(k, v)
        for dt in (torch.float32, torch.float32 if case == 3 else torch.float16):
            check(tree_attention(q, c, out_dtype=dt), q, c)


def test_strides_out_and_scaling():
    from fp4_attn_b200.paged_cache import tree_attention
    c = build([150, 90], 2, 64)
    q = rand_q(2, 6, 5, torch.bfloat16)
    ref = tree_attention(q, c, scaling=0.2)
    check(ref, q, c, scaling=0.2)
    for other in (q.transpose(1, 2).contiguous().transpose(1, 2), q.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0),
                  torch.empty(2, 6, 5, D + 3, dtype=q.dtype, device=DEV)[..., 3:].copy_(q)):
        assert torch.equal(tree_attention(other, c, scaling=0.2), ref)
    out = torch.full((2, 5, 6, D), float("nan"), device=DEV)
    assert tree_attention(q, c, scaling=0.2, out=out) is out
    check(out, q, c, scaling=0.2)


def test_captured_in_a_graph_with_growing_lengths():
    """Lengths are read on the device: a captured call follows the cache as it grows."""
    from fp4_attn_b200.paged_cache import tree_attention
    c = build([120, 3], 1, 16, per_seq=20, spare=30)
    q = rand_q(2, 4, 2, torch.float32)
    out = torch.empty(2, 2, 4, D, device=DEV)
    tree_attention(q, c, out=out)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        with torch.cuda.graph(g, stream=st):
            tree_attention(q, c, out=out)
    for i in range(3):
        c.append(torch.randn(2, 1, 70, D, device=DEV), torch.randn(2, 1, 70, D, device=DEV))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(out, q, c)


def test_refusals():
    from fp4_attn_b200.paged_cache import tree_attention
    c = build([20, 20], 2, 16)
    q = rand_q(2, 4, 3, torch.bfloat16)
    ok = torch.ones(3, 3, dtype=torch.bool, device=DEV)
    for args, kw in (((q[:, :3], c), {}), ((q[..., :64], c), {}), ((q.double(), c), {}), ((q, c), dict(mask=ok.float())),
                     ((q, c), dict(mask=ok[:2])), ((q, c), dict(counts=torch.ones(2, device=DEV))),
                     ((q, c), dict(out_dtype=torch.float64)), ((q, c), dict(out=torch.empty(2, 3, 4, 64, device=DEV))),
                     ((rand_q(3, 4, 1, torch.bfloat16), c), {})):
        with pytest.raises(ValueError):
            tree_attention(*args, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        tree_attention(q.cpu(), c)
    with pytest.raises(RuntimeError, match="workspace"):
        tree_attention(q, c, workspace=torch.empty(64, dtype=torch.uint8, device=DEV))
    assert tree_attention(q[:, :, :0], c).shape == (2, 0, 4, D)
    assert tree_attention(q[:0], c).shape == (0, 3, 4, D)
