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
