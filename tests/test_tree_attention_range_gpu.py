"""Attention of drafted tokens over the paged cache at the ends of its range, against the formula in 64 bits.

Tolerances are those of test_tree_attention_gpu.py; where one key (or several equal ones) has all the weight the
exponents' error drops out, and what is left of e is the rounding of W (fp16, 2^-12 relative; fp32 outputs two planes,
2^-22) and of the row's sum, doubled.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
E = {torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -11}


def cache_of(k, v, page=16):
    """k, v [B, H, T, D] in a cache of their own."""
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    B, H, T, _ = k.shape
    per = -(-T // page)
    c = PagedNVFP4Cache(B * per, page, H, D, B, per, DEV)
    c.append(k, v)
    c.check()
    return c


def quantized(q):
    """The NVFP4 values of q's tokens ([B, Hq, N, D], per token over all heads) in 64 bits."""
    from oracle import quant as oq
    B, H, N, _ = q.shape
    out = oq.fused_qdq(q.transpose(1, 2).reshape(B * N, H * D).float().cpu().numpy(), "row", "float32")[0]
    return torch.from_numpy(out).double().view(B, N, H, D).transpose(1, 2).to(DEV)


def formula(q, c, b=0, g0=0.0):
    """(o, sum p |v|, T max(p g) with g0 for tokens without a value, max |S|) of sequence b under a causal mask, in 64 bits;
    the first three [N, Hq, D]."""
    Hq, N = q.shape[1:3]
    L, G = int(c.lens[b]), Hq // c.num_kv_heads
    K, V = (t[b].double() for t in c.gather(L))
    k, v = (t.repeat_interleave(G, 0) for t in (K, V))
    S = quantized(q)[b] @ k.transpose(1, 2) * D ** -0.5
    smax = float(S.abs().max())
    S[:, :, L - N:].masked_fill_(torch.ones(N, N, dtype=torch.bool, device=DEV).triu(1), -math.inf)
    p = torch.softmax(S, -1)
    top = L * (p * V.abs().amax((0, 2)).clamp(min=g0)).amax(-1)
    return (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1), top.transpose(0, 1)[..., None], smax


def ended():
    from fp4_attn_b200.gemm import device_status
    assert device_status() == 0


# ------------------------------------------------------------- large scores
@pytest.mark.parametrize("exponent,dtype", [(20, torch.float32), (25, torch.float16), (26, torch.bfloat16), (27, torch.float32),
                                            (28, torch.float16), (28, torch.float32), (31, torch.bfloat16),
                                            (40, torch.float32), (64, torch.bfloat16), (100, torch.float32), (120, torch.float32)])
@pytest.mark.parametrize("N,G", [(1, 2), (20, 4)])
def test_large_finite_scores(exponent, dtype, N, G):
    """Scores up to 2^exponent (times log2 e), far apart (quantized, neighbours differ by parts in a thousand): the key with
    the largest has all the weight, equal ones share it; growing along the sequence they move the maximum in every tile."""
    from fp4_attn_b200.paged_cache import tree_attention
    T = 700
    g = torch.Generator(device=DEV).manual_seed(exponent)
    d = torch.randn(D, generator=g, device=DEV)
    size = float(2.0 ** exponent / (float(d.square().sum()) * D ** -0.5 * math.log2(math.e))) ** 0.5
    for kind in ("one", "two", "growing"):
        c = torch.rand(T, generator=g, device=DEV) * 1.4 - 0.9  # (-0.9, 0.5)
        if kind == "growing":
            c = torch.linspace(-1, 1, T, device=DEV)
        top = {"one": [333], "two": [100, 601], "growing": [T - N - 1]}[kind]
        c[top] = 1.0
        if kind == "growing":
            c[T - N:] = -1.0
        k = (c[:, None] * d * size).to(dtype).view(1, 1, T, D)
        v = torch.randn(1, 1, T, D, generator=g, device=DEV).clamp(-3.0, 3.0)
        v[..., 0] = 4.0  # the same g for all: log2(g_v) is in x, of which it is too small a part to tell equal ones apart
        v = v.to(dtype)
        q = (d * size * (1 + torch.rand(1, G, N, 1, generator=g, device=DEV))).to(dtype) / 2
        cache = cache_of(k, v)
        o = tree_attention(q, cache)
        ended()
        ref, share, _, _ = formula(q, cache)
        assert (o[0].double() - ref).abs().le(U[dtype] * ref.abs() + E[dtype] * share + 2.0 ** -24).all(), (kind, exponent)


# ------------------------------------------------- V tokens without a value
@pytest.mark.parametrize("largest", [False, True])
@pytest.mark.parametrize("exponent,dtype", [(0, torch.float32), (-10, torch.float16), (-10, torch.float32), (-25, torch.bfloat16),
                                            (-25, torch.float32), (-40, torch.bfloat16), (-40, torch.float32),
                                            (15, torch.float16), (40, torch.float32)])
@pytest.mark.parametrize("N,G", [(1, 2), (9, 4)])
def test_zero_values_among_small_ones(exponent, dtype, largest, N, G):
    """Tokens whose V is 0 (or below 2^-100) take their share of the softmax and nothing else: the others' values keep
    their precision, whatever their size, also where a token without a value has the largest score.  Such a token
    counts as one of 2^-64 where m is made, which adds T f 2^-64 p to what W is rounded by."""
    from fp4_attn_b200.paged_cache import tree_attention
    T = 900
    g = torch.Generator(device=DEV).manual_seed(exponent + 100)
    k = torch.randn(1, 2, T, D, generator=g, device=DEV)
    v = torch.randn(1, 2, T, D, generator=g, device=DEV) * 2.0 ** exponent
    v[:, :, 5::7] = 0
    v[:, :, 6::50] = 2.0 ** -110
    v[:, :, :300] = 0  # a whole tile of them
    q = 2.0 * torch.randn(1, 2 * G, N, D, generator=g, device=DEV)
    if largest:  # node 0's own direction, at places without a value
        for h in range(2):
            k[0, h, [40, 5 + 7 * 100]] = q[0, h * G, 0] * 1.2
    cache = cache_of(k, v)
    o = tree_attention(q, cache, out_dtype=dtype)
    ended()
    ref, share, top, smax = formula(q, cache, g0=2.0 ** -64)
    e = E[dtype] + 2.0 ** -20 * smax * 1.4427
    tol = U[dtype] * ref.abs() + e * share + 2.0 ** -36 * top + 2.0 ** -24 * (dtype == torch.float16)
    err = (o[0].double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


def test_a_workspace_elsewhere_is_refused():
    from fp4_attn_b200.paged_cache import tree_attention
    cache = cache_of(*(torch.randn(1, 2, 9, D, device=DEV) for _ in range(2)))
    q = torch.randn(1, 4, 2, D, device=DEV)
    size = 1 << 22
    for w in (torch.empty(size, dtype=torch.uint8), torch.empty(size, 2, dtype=torch.uint8, device=DEV)[:, 0]):
        with pytest.raises(ValueError, match="workspace"):
            tree_attention(q, cache, workspace=w)
    good = torch.empty(size, dtype=torch.uint8, device=DEV)
    assert torch.equal(tree_attention(q, cache, workspace=good), tree_attention(q, cache))
