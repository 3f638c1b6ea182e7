"""Sampling against the definition in 64 bits.

The token is where the running sum of the kept weights passes u.  In 32 bits a
weight exp((x - max) / T) is off by its argument's rounding and exp's: at most
(|arg| + 4) 2^-23 of itself, and |arg| < 24 where the weight, in multiples of
2^-34, is not 0; V half units are V 2^-35 of the largest weight.  A share of a
sum of such weights is off by at most 56 * 2^-23 + V 2^-35 =: eps.  So: the token
belongs to the kept set for top_p widened by eps, and u lies within 2 eps of
its interval for one of the sets that a threshold within eps of top_p gives.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def kept_count(p, k, top_p, min_p):
    """How many of the sorted probabilities are kept."""
    n = len(p)
    if k > 0:
        n = min(n, k)
    if top_p < 1:
        c = np.cumsum(p[:n])
        n = max(1, int(np.sum(c - p[:n] < top_p * c[-1])))
    return max(1, min(n, int(np.sum(p >= min_p * p[0]))))


def check_row(x, u, T, k, top_p, min_p, token, logprob):
    x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), np.finfo(np.float32).max))
    V = len(x)
    if not np.isfinite(x.max()):
        assert token == -1 and logprob == -np.inf
        return
    order = np.argsort(-x, kind="stable")
    t = T if T > 0 else 1.0
    w = np.exp((x - x.max()) / t)
    want = (x[token] - x.max()) / t - np.log(w.sum())
    # (x - max) / T and the log are rounded to 32 bits each, the sum once more
    assert abs(logprob - want) <= 2.0 ** -22 * (abs((x[token] - x.max()) / t) + abs(np.log(w.sum())) + 1)
    if T <= 0:
        assert token == order[0]
        return
    eps = 56 * 2.0 ** -23 + V * 2.0 ** -35
    ws = w[order]
    fine = False
    for n in range(kept_count(ws, k, top_p - eps, min_p * (1 + eps)) if top_p < 1 else kept_count(ws, k, top_p, min_p * (1 + eps)),
                   kept_count(ws, k, top_p + eps if top_p < 1 else 1.0, min_p * (1 - eps)) + 1):
        q = np.zeros(V)
        q[order[:n]] = ws[:n] / ws[:n].sum()
        c = np.cumsum(q)
        if q[token] > 0 and c[token] - q[token] <= u + 2 * eps and c[token] >= u - 2 * eps:
            fine = True
            break
    assert fine, (V, u, T, k, top_p, min_p, token)


def run(x, u, T=1.0, k=0, p=1.0, m=0.0):
    from fp4_attn_b200.sampling import sample
    tok, lp = sample(x, u, temperature=T, top_k=k, top_p=p, min_p=m)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32
    R = x.shape[0]
    full = lambda v: v.tolist() if isinstance(v, torch.Tensor) else [v] * R  # noqa: E731
    xs = x.float().cpu().numpy()
    for r, (t, l, uu, T1, k1, p1, m1) in enumerate(zip(tok.tolist(), lp.tolist(), u.tolist(), full(T), full(k), full(p), full(m))):
        check_row(xs[r], uu, T1, k1, p1, m1, t, l)
    t2, l2 = sample(x, u, temperature=T, top_k=k, top_p=p, min_p=m)
    assert torch.equal(tok, t2) and torch.equal(lp, l2)
    return tok, lp


def logits(R, V, dtype=torch.float32, seed=0, spread=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(R, V, generator=g, device=DEV) * spread
    return x.to(dtype), torch.rand(R, generator=g, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (5, 31), (4, 1000), (7, 1025), (3, 32000), (2, 50001), (2, 131072),
                                 (1, 262144), (200, 333)])
def test_filters(R, V, dtype):
    x, u = logits(R, V, dtype, seed=V)
    run(x, u)
    run(x, u, T=0.7, k=50)
    run(x, u, p=0.9)
    run(x, u, T=1.5, m=0.05)
    run(x, u, T=0.8, k=40, p=0.95, m=0.01)
    run(x, u, T=0.0)


def test_parameters_of_each_row():
    x, u = logits(64, 5003, torch.float16, seed=9)
    r = torch.arange(64, device=DEV)
    run(x, u, T=(0.25 * (r % 6)).float(), k=(r * 7 % 60 - 3).int(), p=(1.05 - 0.1 * (r % 9)).float(), m=(0.02 * (r % 4)).float())


@pytest.mark.parametrize("k", [1, 2, 3, 5, 64, 700, 999])
def test_ties_go_to_the_lowest_index(k):
    """bf16 rows full of equal logits: top_k keeps the first of them."""
    g = torch.Generator(device=DEV).manual_seed(k)
    x = torch.randint(-2, 3, (40, 1000), generator=g, device=DEV).bfloat16()
    u = torch.rand(40, generator=g, device=DEV)
    run(x, u, k=k)
    run(x, u, k=k, p=0.5)
    run(x, u, p=0.3)
    flat = torch.zeros(40, 1000, device=DEV)
    flat[:, ::2] = -0.0
    tok, _ = run(flat, u, k=k)
    assert torch.equal(tok, torch.floor(u.double() * k).long())
    tok, _ = run(flat, u, T=0.0)
    assert not tok.any()


def test_ends_of_u_and_masked_tokens():
    x, _ = logits(4, 300)
    x[:, :7] = float("-inf")
    x[:, -9:] = float("-inf")
    one = float(np.nextafter(np.float32(1), np.float32(0)))
    tok, _ = run(x, torch.tensor([0.0, one, 0.0, one], device=DEV))
    assert tok.tolist()[0] == 7 and tok.tolist()[1] == 290
    tok, _ = run(x, torch.tensor([0.0, one, 0.0, one], device=DEV), k=300, p=0.999999)
    assert ((tok >= 7) & (tok < 291)).all()


def test_rows_that_are_not_finite():
    x, u = logits(6, 400)
    x[0] = float("-inf")
    x[1] = float("nan")
    x[2, 5] = float("nan")
    x[3, [70, 90]] = float("inf")
    x[4, 1:] = float("-inf")
    x[5] = torch.finfo(torch.float32).min
    x[5, 33] = torch.finfo(torch.float32).max
    for kw in ({}, dict(k=3), dict(p=0.5), dict(T=0.0), dict(T=0.3, k=7, p=0.9, m=0.1)):
        tok, lp = run(x, u, **kw)
        assert tok[:2].tolist() == [-1, -1] and tok[3] in (70, 90) and tok[4] == 0 and tok[5] == 33
        assert lp[4] == 0


@pytest.mark.parametrize("rows", [3, 320])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_in_masked_places(rows, dtype):
    """Whole stretches of NaN, at the start among them, weigh nothing."""
    V = 60001
    x, u = logits(rows, V, dtype, seed=rows)
    x[:, :20000] = float("nan")
    x[:, 30000::7] = float("nan")
    for kw in ({}, dict(m=0.05), dict(k=40, p=0.7), dict(T=0.0)):
        u[0] = 0.0
        tok, _ = run(x[:3], u[:3], **kw)
        from fp4_attn_b200.sampling import sample
        many = sample(x, u, temperature=kw.get("T", 1.0), top_k=kw.get("k", 0), top_p=kw.get("p", 1.0), min_p=kw.get("m", 0.0))
        assert torch.equal(many[0][:3].cpu(), torch.as_tensor(tok).cpu())
        assert (many[0] >= 20000).all() and torch.isfinite(x.gather(1, many[0][:, None])).all()


@pytest.mark.parametrize("kind", ["normal", "steps", "peaks"])
@pytest.mark.parametrize("R,V,dtype", [(20, 131072, torch.float32), (40, 60001, torch.float32), (70, 100003, torch.bfloat16),
                                       (130, 200001, torch.float16), (160, 33333, torch.bfloat16)])
def test_many_long_rows_like_single_ones(R, V, dtype, kind):
    """Rows that are not held on chip give what each gives alone, to the bit; the first ones what the definition says."""
    from fp4_attn_b200.sampling import sample
    if kind == "normal":
        x, u = logits(R, V, dtype, seed=V + R)
    else:
        g = torch.Generator(device=DEV).manual_seed(V - R)
        u = torch.rand(R, generator=g, device=DEV)
        if kind == "steps":  # many equal logits
            x = torch.randint(-3, 4, (R, V), generator=g, device=DEV).to(dtype)
        else:  # a few far above the rest, which top_k goes down to
            x = torch.randn(R, V, generator=g, device=DEV)
            x[:, ::V // 5] += 30.0
            x = x.to(dtype)
    x[:, V // 2:V // 2 + 100] = float("-inf")
    r = torch.arange(R, device=DEV)
    kw = dict(T=(0.3 * (r % 8)).float(), k=(r * 53 % 400 - 20).int(), p=(1.06 - 0.11 * (r % 7)).float(), m=(0.02 * (r % 3)).float())
    run(x[:12], u[:12], **{a: b[:12] for a, b in kw.items()})
    tok, lp = sample(x, u, temperature=kw["T"], top_k=kw["k"], top_p=kw["p"], min_p=kw["m"])
    for i in range(R):
        s = slice(i, i + 1)
        t1, l1 = sample(x[s], u[s], temperature=kw["T"][s], top_k=kw["k"][s], top_p=kw["p"][s], min_p=kw["m"][s])
        assert torch.equal(tok[s], t1) and torch.equal(lp[s], l1), i


def test_strides_shapes_and_streams():
    from fp4_attn_b200.sampling import sample
    x, u = logits(6, 777, torch.bfloat16, seed=3)
    ref = sample(x, u, top_p=0.8)
    wide = torch.zeros(6, 1501, dtype=x.dtype, device=DEV)
    for off in (0, 1, 5):
        v = wide[:, off:off + 777]
        v.copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(sample(v, u, top_p=0.8), ref))
    got = sample(x.view(2, 3, 777), u.view(2, 3), top_p=0.8)
    assert got[0].shape == (2, 3) and torch.equal(got[0].view(-1), ref[0])
    assert torch.equal(sample(x.t().contiguous().t(), u, top_p=0.8)[0], ref[0])
    assert int(sample(x[2], u[2], top_p=0.8)[0]) == int(ref[0][2])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a = sample(x, u, top_p=0.8)
    st.synchronize()
    assert torch.equal(a[0], ref[0])
    assert sample(x[:0], u[:0])[0].shape == (0,)


def test_frequencies():
    """Evenly spaced u draw each token as often as its probability says, within one draw of either end."""
    from fp4_attn_b200.sampling import sample
    x, _ = logits(1, 50, seed=11, spread=1.0)
    n = 4096
    u = (torch.arange(n, device=DEV) + 0.5) / n
    tok, _ = sample(x.expand(n, 50), u, temperature=0.9)
    p = torch.softmax(x[0].double() / 0.9, 0)
    assert ((torch.bincount(tok, minlength=50) - p * n).abs() <= 1.0 + 1e-3).all()


def test_refusals():
    from fp4_attn_b200.sampling import accept_tree, sample
    x, u = logits(2, 10)
    for args, kw in (((x.double(), u), {}), ((x, u[:1]), {}), ((x, u.double()), {}), ((x, u), dict(top_p=u.double())),
                     ((x, u), dict(top_k=torch.ones(2, device=DEV))), ((x[:, :0], u), {})):
        with pytest.raises(ValueError):
            sample(*args, **kw)
    with pytest.raises(NotImplementedError):
        sample(torch.zeros(1, 262145, device=DEV), u[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        sample(x.cpu(), u.cpu())
    t = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError):
        accept_tree(t, t, t)
    with pytest.raises(ValueError):
        accept_tree(t.int(), t, t[:, :2])


@pytest.mark.parametrize("N", [1, 2, 13, 64, 300])
def test_accept_tree(N):
    from fp4_attn_b200.sampling import accept_tree
    rng = np.random.RandomState(N)
    B = 9
    parents = np.full((B, N), -1, np.int32)
    for j in range(1, N):
        parents[:, j] = rng.randint(max(0, j - 4), j, B)
    tokens, sampled = rng.randint(0, 3, (B, N)), rng.randint(0, 3, (B, N))
    counts = np.array([N, 0, 1] + [rng.randint(1, N + 1) for _ in range(B - 3)], np.int32)
    for cnt in (None, counts):
        keep, n, nxt = accept_tree(torch.from_numpy(parents).to(DEV), torch.from_numpy(tokens).to(DEV),
                                   torch.from_numpy(sampled).to(DEV), None if cnt is None else torch.from_numpy(cnt).to(DEV))
        for b in range(B):
            c = N if cnt is None else cnt[b]
            path, want = [], -1
            at = 0 if c else None
            while at is not None:
                path.append(at)
                want = sampled[b, at]
                at = next((j for j in range(at + 1, c) if parents[b, j] == at and tokens[b, j] == want), None)
            assert int(n[b]) == len(path) and int(nxt[b]) == want
            assert keep[b].tolist() == path + [N - 1] * (N - len(path))
