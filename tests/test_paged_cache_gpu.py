"""The paged NVFP4 cache: appended tokens against the C oracle's row quantizer bit for bit, page bookkeeping
against a model in plain Python, moves and copies byte for byte, and the refusals."""
import random

import numpy as np
import pytest
import torch

from oracle import quant as oq

pytestmark = pytest.mark.gpu

D = 128
POOLS = ("k_codes", "k_scales", "k_g", "v_codes", "v_scales", "v_g")
DEV = "cuda:0"


def make(num_pages=64, page=16, H=2, seqs=4, per_seq=12):
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    return PagedNVFP4Cache(num_pages, page, H, D, seqs, per_seq, DEV)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def token(c, x, s, t):
    """(codes [H, D/2], scales [H, D/16], g) of token t of sequence s."""
    page, slot = int(c.page_table[s, t // c.page_size]), t % c.page_size
    assert page >= 0
    return (getattr(c, x + "_codes")[page, :, slot].cpu(), getattr(c, x + "_scales")[page, :, slot].cpu(),
            getattr(c, x + "_g")[page, slot].cpu())


def same(a, b):
    return all(torch.equal(x.reshape(-1).view(torch.uint8), y.reshape(-1).view(torch.uint8)) for x, y in zip(a, b))


class Model:
    """Page bookkeeping in plain Python: the lowest-numbered free pages, in order of (row, position)."""

    def __init__(self, c):
        self.P, self.tables, self.lens, self.refs = c.page_size, [[] for _ in range(c.max_seqs)], \
            [0] * c.max_seqs, [0] * c.num_pages

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def append(self, s, n):
        self.lens[s] += n
        while len(self.tables[s]) * self.P < self.lens[s]:
            self.tables[s].append(self.take())

    def shorten(self, s, n):
        self.lens[s] = min(self.lens[s], n)
        while len(self.tables[s]) > -(-self.lens[s] // self.P):
            self.refs[self.tables[s].pop()] -= 1

    def fork(self, pairs, deep):
        for s, d in pairs:
            full = 0 if deep else self.lens[s] // self.P
            self.tables[d] = self.tables[s][:full]
            for p in self.tables[d]:
                self.refs[p] += 1
        for s, d in pairs:
            while len(self.tables[d]) < len(self.tables[s]):
                self.tables[d].append(self.take())
            self.lens[d] = self.lens[s]

    def check(self, c):
        c.check()
        assert c.lens.tolist() == self.lens
        assert c.refs.tolist() == self.refs
        for s, t in enumerate(c.page_table.tolist()):
            assert t == self.tables[s] + [-1] * (len(t) - len(self.tables[s]))


def kv(B, H, T, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(B, T, H, D, generator=g) * torch.exp(torch.randn(B, T, 1, 1, generator=g))).to(dtype)
            .to(DEV).transpose(1, 2) for _ in range(2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,T,page", [(1, 1, 16), (3, 37, 32), (4, 20, 64), (8, 150, 128), (9, 33, 16), (40, 18, 16)])
def test_append_is_the_row_quantizer(dtype, H, T, page):
    c = make(num_pages=40, page=page, H=H, seqs=3, per_seq=12)
    k, v = kv(3, H, T, dtype, seed=H * T)
    counts = i32(T, max(1, T // 2), 0)
    c.append(k, v, counts=counts)
    c.append(k[:, :, :1], v[:, :, :1])  # one more, behind ragged ends
    c.check()
    assert c.lens.tolist() == [T + 1, max(1, T // 2) + 1, 1]
    for x, t in (("k", k), ("v", v)):
        for s in range(3):
            src = torch.cat((t[s, :, :int(counts[s])], t[s, :, :1]), 1).transpose(0, 1).float().cpu()
            n = src.shape[0]
            out, codes, scales, g = oq.fused_qdq(src.reshape(n, H * D).numpy(), "row", "float32")
            got = [token(c, x, s, i) for i in range(n)]
            assert np.array_equal(torch.stack([a[0].reshape(-1) for a in got]).numpy(), codes)
            assert np.array_equal(torch.stack([a[1].reshape(-1) for a in got]).numpy(), scales)
            assert np.array_equal(torch.stack([a[2] for a in got]).numpy(), g)
            dense = c.gather(n)[0 if x == "k" else 1][s].transpose(0, 1).reshape(n, -1)
            assert np.array_equal(dense.cpu().numpy(), out)


def test_append_strides_and_alignment():
    """Other orders of the axes, rows that are not 16-byte aligned and a last axis that is not contiguous give the
    same bytes."""
    k, v = kv(2, 3, 21)
    ref = make(H=3)
    ref.append(k, v)
    odd = torch.empty(2, 3, 21, D + 1, dtype=k.dtype, device=DEV)[..., 1:]
    for kk, vv in ((k.contiguous(), v.contiguous()), (odd.copy_(k), v),
                   (k.transpose(2, 3).contiguous().transpose(2, 3), v.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3))):
        c = make(H=3)
        c.append(kk, vv)
        c.check()
        for n in POOLS:
            assert torch.equal(getattr(c, n), getattr(ref, n)), n


def test_append_zero_tiny_and_not_finite_tokens():
    k, v = kv(1, 2, 6, torch.float32)
    k, v = k.contiguous(), v.contiguous()
    k[0, :, 0] = 0
    v[0, 1, 1] = 1e-39  # subnormal next to ordinary values: rounds to 0 under the token's g
    v[0, :, 2] = 1e-39  # g itself subnormal: the token stands for 0
    k[0, 1, 3, 5] = float("inf")
    v[0, 0, 4, 7] = float("nan")
    c = make(H=2)
    c.append(k, v)
    c.check()
    K, V = c.gather(6, B=1)
    assert (K[0, :, 0] == 0).all() and (V[0, :, 2] == 0).all() and (V[0, 1, 1] == 0).all()
    for x, t in (("k", 3), ("v", 4)):
        codes, scales, g = token(c, x, 0, t)
        assert torch.isnan(g) and not codes.any() and not scales.any()
    assert torch.isnan(K[0, :, 3]).all() and torch.isnan(V[0, :, 4]).all()
    assert torch.isfinite(K[0, :, [0, 1, 2, 4, 5]]).all() and torch.isfinite(V[0, :, [0, 1, 2, 3, 5]]).all()


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_bookkeeping_against_a_model(page):
    """Random appends, truncations, compactions, forks and releases; every token keeps its bytes."""
    rng = random.Random(page)
    c = make(num_pages=90, page=page, H=1, seqs=6, per_seq=9)
    m = Model(c)
    held = [[] for _ in range(6)]  # bytes of every token
    for step in range(60):
        op = rng.choice(["append", "append", "append", "compact", "truncate", "fork", "release"])
        rows = rng.sample(range(6), rng.randint(1, 6))
        seqs = i32(*rows)
        if op == "append":
            T = rng.choice([1, 3, page, 2 * page + 1])
            counts = [rng.randint(0, T) for _ in rows]
            if any(m.lens[s] + n > 9 * page for s, n in zip(rows, counts)):
                continue
            shared = [s for s, n in zip(rows, counts) if n and m.lens[s] % page and m.refs[m.tables[s][m.lens[s] // page]] > 1]
            if shared:
                continue
            k, v = kv(len(rows), 1, T, seed=step)
            c.append(k, v, seqs=seqs, counts=i32(*counts))
            for s, n in zip(rows, counts):
                t0 = m.lens[s]
                m.append(s, n)
                held[s] += [[token(c, x, s, t) for x in "kv"] for t in range(t0, t0 + n)]
        elif op == "truncate":
            lens = [rng.randint(0, 9 * page) for _ in rows]
            c.truncate(i32(*lens), seqs=seqs)
            for s, n in zip(rows, lens):
                m.shorten(s, n)
                held[s] = held[s][:n]
        elif op == "release":
            c.release(seqs)
            for s in rows:
                m.shorten(s, 0)
                held[s] = []
        elif op == "compact":
            tails = [rng.randint(0, m.lens[s]) for s in rows]
            keeps = [sorted(rng.sample(range(t), rng.randint(0, t))) for t in tails]
            bad = any(k != j and m.refs[m.tables[s][(m.lens[s] - t + j) // page]] > 1
                      for s, t, ks in zip(rows, tails, keeps) for j, k in enumerate(ks))
            if bad:
                continue
            N = max(1, max(tails))
            keep = torch.tensor([ks + [0] * (N - len(ks)) for ks in keeps], dtype=torch.int32, device=DEV)
            c.compact(keep, i32(*(len(k) for k in keeps)), seqs=seqs, tails=i32(*tails))
            for s, t, ks in zip(rows, tails, keeps):
                base = m.lens[s] - t
                held[s] = held[s][:base] + [held[s][base + k] for k in ks]
                m.shorten(s, base + len(ks))
        else:
            empty = [s for s in range(6) if m.lens[s] == 0]
            full = [s for s in range(6) if m.lens[s] > 0]
            if not empty or not full:
                continue
            pairs = [(rng.choice(full), d) for d in empty[:rng.randint(1, 3)]]
            deep = rng.random() < 0.5
            c.fork(i32(*(s for s, _ in pairs)), i32(*(d for _, d in pairs)), deep=deep)
            m.fork(pairs, deep)
            for s, d in pairs:
                held[d] = list(held[s])
        m.check(c)
        for s in range(6):
            for t, h in enumerate(held[s]):
                if rng.random() < 0.1:
                    assert all(same(token(c, x, s, t), h[i]) for i, x in enumerate("kv")), (step, op, s, t)


def test_compact_long_list_over_many_pages():
    c = make(num_pages=64, page=16, H=2, seqs=1, per_seq=60)
    k, v = kv(1, 2, 900)
    c.append(k, v)
    before = [token(c, x, 0, t) for x in "kv" for t in range(900)]
    keep = [t for t in range(850) if t % 3 != 1]  # of the last 850
    c.compact(i32(*keep + [0] * (850 - len(keep))).view(1, -1), i32(len(keep)))
    c.check()
    assert int(c.lens[0]) == 50 + len(keep) and int((c.refs > 0).sum()) == -(-(50 + len(keep)) // 16)
    for i, x in enumerate("kv"):
        for j, t in enumerate(list(range(50)) + [50 + t for t in keep]):
            if j % 7 == 0:
                assert same(token(c, x, 0, j), before[i * 900 + t])


def test_errors_leave_the_cache_alone():
    c = make(num_pages=8, page=16, H=1, seqs=3, per_seq=6)
    k, v = kv(1, 1, 40)
    c.append(k, v, seqs=i32(1))
    c.check()

    def state():
        return [getattr(c, n).clone() for n in POOLS + ("page_table", "lens", "refs")]

    def refused(what, call):
        was = state()
        call()
        with pytest.raises(RuntimeError, match=what):
            c.check()
        c.check()  # reported once
        assert all(torch.equal(a, b) for a, b in zip(was, state()))

    big = kv(2, 1, 48)
    refused("free pages", lambda: c.append(*big, seqs=i32(0, 2)))
    refused("row of the page table", lambda: c.append(*kv(1, 1, 60), seqs=i32(1)))
    refused("out of range", lambda: c.append(*kv(1, 1, 1), seqs=i32(3)))
    refused("keep list", lambda: c.compact(i32(3, 3).view(1, 2), i32(2), seqs=i32(1), tails=i32(9)))
    refused("keep list", lambda: c.compact(i32(3, 9).view(1, 2), i32(2), seqs=i32(1), tails=i32(9)))
    refused("keep list", lambda: c.compact(i32(0, 1).view(1, 2), i32(2), seqs=i32(1), tails=i32(41)))
    refused("not empty", lambda: c.fork(i32(1), i32(1)))
    refused("free pages", lambda: c.fork(i32(1, 1), i32(0, 2), deep=True))
    c.fork(i32(1), i32(0))
    c.truncate(i32(20), seqs=i32(0))
    c.check()
    refused("shared page", lambda: c.append(*kv(1, 1, 1), seqs=i32(0)))  # position 20: a page that 1 holds too
    refused("shared page", lambda: c.compact(i32(1).view(1, 1), i32(1), seqs=i32(0), tails=i32(4)))


def test_argument_refusals():
    from fp4_attn_b200.paged_cache import PagedNVFP4Cache
    with pytest.raises(ValueError, match="page_size"):
        PagedNVFP4Cache(8, 48, 1, D, 1, 1, DEV)
    with pytest.raises(NotImplementedError, match="head_dim"):
        PagedNVFP4Cache(8, 16, 1, 64, 1, 1, DEV)
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedNVFP4Cache(8, 16, 1, D, 1, 1, "cpu")
    c = make(H=2, seqs=2)
    k, v = kv(2, 2, 3)
    for args, kw in (((k[:, :1], v[:, :1]), {}), ((k, v[:, :, :2]), {}), ((k, v.float()), {}), ((k.double(), v.double()), {}),
                     ((k, v), dict(counts=i32(1))), ((k, v), dict(counts=torch.tensor([1, 2], device=DEV))),
                     ((k, v), dict(seqs=torch.tensor([0, 1], dtype=torch.int32))), (kv(3, 2, 1), {})):
        with pytest.raises(ValueError):
            c.append(*args, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.append(k.cpu(), v.cpu())
    with pytest.raises(ValueError):
        c.gather(-1)
    c.append(k[:, :, :0], v[:, :, :0])
    assert c.gather(0)[0].shape == (2, 2, 0, D)
    c.check()


def test_on_another_stream_and_in_a_graph():
    """A verify step's calls captured in a CUDA graph and replayed give what the plain calls give."""
    a, b = make(seqs=2), make(seqs=2)
    k, v = kv(2, 2, 5)
    keep, counts, lens0 = i32(0, 2, 4, 0, 0, 1, 2, 3, 0, 0).view(2, 5), i32(3, 3), i32(7, 4)
    for c in (a, b):
        c.append(*kv(2, 2, 7, seed=4), counts=i32(7, 4))

    def step(c):
        c.truncate(lens0)
        c.append(k, v)
        c.compact(keep, counts)
    step(a)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        with torch.cuda.graph(g, stream=st):
            step(b)
        for _ in range(3):
            g.replay()
    st.synchronize()
    a.check(), b.check()
    assert torch.equal(a.lens, b.lens) and torch.equal(a.page_table, b.page_table)
    for x, y in zip(a.gather(20), b.gather(20)):
        assert torch.equal(x, y)
