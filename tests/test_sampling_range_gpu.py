"""Sampling where it can go wrong besides its formula: clusters that start late, thresholds at a band's edge, parameters
beyond their usual range.  Compared with the definition in 64 bits, or with the same rows by themselves, to the bit."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def logits(R, V, dtype=torch.float32, seed=0, spread=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(R, V, generator=g, device=DEV) * spread
    return x.to(dtype), torch.rand(R, generator=g, device=DEV)


def test_rows_held_by_clusters_on_a_busy_gpu():
    """Clusters of up to 16 CTAs that come to run one after the other, next to other work on other streams."""
    from fp4_attn_b200.sampling import sample
    cases = [logits(R, V, dt, seed=V) for R, V, dt in ((8, 262144, torch.float32), (16, 100003, torch.bfloat16),
                                                       (32, 50001, torch.float32), (3, 32000, torch.float16))]
    kw = dict(temperature=0.8, top_k=60, top_p=0.9)
    alone = [sample(x, u, **kw) for x, u in cases]
    torch.cuda.synchronize()
    a = torch.randn(2048, 2048, device=DEV, dtype=torch.bfloat16)
    streams = [torch.cuda.Stream() for _ in range(5)]
    got = []
    for i in range(30):
        for j, (x, u) in enumerate(cases):
            with torch.cuda.stream(streams[j]):
                got.append((j, sample(x, u, **kw)))
        with torch.cuda.stream(streams[4]):
            a @ a
    torch.cuda.synchronize()
    for j, (tok, lp) in got:
        assert torch.equal(tok, alone[j][0]) and torch.equal(lp, alone[j][1])


def band_edge(seed):
    """(max, T, a logit 7 T below the maximum up to rounding, in 32 bits) such that max - logit <= 7 T but logit is below
    max - 7 T - |max| 2.4e-7."""
    F = np.float32
    rng = np.random.RandomState(seed)
    while True:
        mx, T = F(rng.uniform(0.05, 3.0)), F(rng.uniform(1.2, 3.0))
        reach = F(F(7.0) * T)
        low = F(F(mx - reach) - F(mx * F(2.4e-7)))
        v = np.nextafter(low, F(-np.inf))
        if F(mx - v) <= reach:
            return mx, T, v


@pytest.mark.parametrize("R,V", [(1, 3001), (40, 60001), (160, 60001)])
def test_a_logit_at_a_bands_edge(R, V):
    """top_k ends at a logit that lies on the first band's edge: it counts, and the next one is dropped."""
    k = 40
    x = np.full((R, V), -60.0, np.float32)
    T = np.zeros(R, np.float32)
    for r in range(R):
        mx, T[r], v = band_edge(R + r)
        x[r, 5:5 + k - 2] = mx - np.float32(0.5)
        x[r, 2], x[r, 3] = mx, v
        x[r, V - 7] = v - np.float32(0.01)  # the first that top_k drops, the last in index order
    t = torch.from_numpy(x).to(DEV)
    u = torch.full((R,), float(np.nextafter(np.float32(1), np.float32(0))), device=DEV)
    from fp4_attn_b200.sampling import sample
    tok, _ = sample(t, u, temperature=torch.from_numpy(T).to(DEV), top_k=k)
    assert tok.tolist() == [5 + k - 3] * R


@pytest.mark.parametrize("R,V,dtype", [(1, 5000, torch.float32), (40, 60001, torch.float32), (100, 60001, torch.float32),
                                       (200, 90001, torch.bfloat16)])
def test_the_whole_range_of_logits(R, V, dtype):
    """Logits down to the type's lowest value under a temperature of their size: no band ends above them."""
    from fp4_attn_b200.sampling import sample
    far = torch.finfo(dtype).min
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (-1e38 - torch.rand(R, V, generator=g, device=DEV) * 2.4e38).clamp(min=far).to(dtype)
    x[:, 7:9], x[:, 100:200], x[:, 30] = far, float("-inf"), -1e38
    u = torch.rand(R, generator=g, device=DEV)
    for kw in (dict(top_k=40), dict(top_p=0.7), dict(top_k=300, top_p=0.5)):
        tok, lp = sample(x, u, temperature=3e38, **kw)
        for r in range(0, R, 17):
            d = x[r].double()
            order = torch.sort(-d, stable=True).indices
            p = torch.exp((d - d.max()) / float(np.float32(3e38)))[order]
            n = kw.get("top_k", V)
            eps = 56 * 2.0 ** -23 + V * 2.0 ** -35
            fine = False
            c = p[:n].cumsum(0)
            sizes = [n] if "top_p" not in kw else [max(1, int((c - p[:n] < (kw["top_p"] + e) * c[-1]).sum())) for e in (-eps, eps)]
            for m in range(sizes[0], sizes[-1] + 1):
                q = torch.zeros(V, dtype=torch.float64, device=DEV).index_copy(0, order[:m], p[:m] / p[:m].sum())
                t = q.cumsum(0)[int(tok[r])]
                fine |= bool(q[int(tok[r])] > 0 and t - q[int(tok[r])] <= float(u[r]) + 2 * eps and t >= float(u[r]) - 2 * eps)
            assert fine, (r, kw)


@pytest.mark.parametrize("R", [1, 200])
@pytest.mark.parametrize("min_p", [1.5, float("inf"), float("nan")])
def test_min_p_that_nothing_reaches_keeps_the_first(R, min_p):
    """No weight is min_p times the largest: what is left is the first of the largest logits, whatever u; with min_p 1
    all of the largest are kept."""
    from fp4_attn_b200.sampling import sample
    x, u = logits(R, 20000, torch.bfloat16, seed=R)
    x[:, [77, 500, 19999]] = 40.0
    u[0] = 0.9
    for kw in ({}, dict(top_k=9), dict(top_p=0.9)):
        tok, lp = sample(x, u, temperature=0.7, min_p=min_p, **kw)
        assert (tok == 77).all()
        want = -torch.logsumexp((x.double() - 40.0) / float(np.float32(0.7)), 1)
        assert (lp.double() - want).abs().max() < 2.0 ** -21
        assert int(sample(x, u, temperature=0.7, min_p=1.0, **kw)[0][0]) == 19999
