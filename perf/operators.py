"""The serving operators of the paged NVFP4 cache, as measured: attention of drafted tokens over the cache,
the cache's page operations, and sampling.

Each case runs in two forms.  Where ``own`` is false: elementary torch operations in 32 bits.  Where it is
true: the calls that a user makes of ``fp4_attn_b200.paged_cache`` and ``fp4_attn_b200.sampling``.

A token of the cache is stored by itself: per (token, K or V) a global scale g over all heads' channels, one
E4M3 scale per 16 channels and E2M1 codes, two per byte (the first channel in the low nibble):
    g = max|x| (0 where that is subnormal; NaN where it is not finite, with codes and scales 0)
    s = e4m3(max|x * (1/g)| over the block * (1/6)),  code = e2m1(x * (1/g) * (1/s)),  value = code * s * g.
"""
import math
import random

import torch

own = False

D = 128
TINY = 2.0 ** -126
SIXTH = 1.0 / 6.0
POOLS = ("k_codes", "k_scales", "k_g", "v_codes", "v_scales", "v_g")
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one sequence, one new token, a short context: the smallest decode call, where launches and latency count
        dict(name="decode 1x1 t777", op="attention", B=1, Hq=32, Hkv=8, N=1, T=777, ragged=False, page=64,
             tree=False, dtype="bfloat16"),
        # a batch of long contexts, one new token each: an ordinary serving step, bound by the cache's bytes
        dict(name="decode 8x1 t32768", op="attention", B=8, Hq=64, Hkv=8, N=1, T=32768, ragged=False, page=128,
             tree=False, dtype="bfloat16"),
        # verification of drafted trees of odd size in a ragged batch, 7 query heads per KV head
        dict(name="tree 6x27 ragged t5003", op="attention", B=6, Hq=28, Hkv=4, N=27, T=5003, ragged=True, page=16,
             tree=True, dtype="float16"),
        # the largest: whole trees of 64 drafted tokens over very long contexts
        dict(name="tree 2x64 t65536", op="attention", B=2, Hq=64, Hkv=8, N=64, T=65536, ragged=False, page=128,
             tree=True, dtype="bfloat16"),
        # a chain of drafted tokens with fp32 queries and outputs, one KV head per query head
        dict(name="chain 4x5 fp32 t2900", op="attention", B=4, Hq=32, Hkv=32, N=5, T=2900, ragged=True, page=32,
             tree=False, dtype="float32"),
        # after a verification: the drafted tokens are appended, the accepted ones kept, the rest's pages freed
        dict(name="commit 8x13", op="commit", B=8, Hkv=8, N=13, T=500, page=16, dtype="bfloat16"),
        # prompts enter the cache: ragged chunks of long prompts are quantized into newly taken pages
        dict(name="prompt 3x8192", op="prompt", B=3, Hkv=8, N=8192, page=64, dtype="bfloat16"),
        # beams: every sequence is forked eight times, full pages shared, the last page copied
        dict(name="fork 4 to 32", op="fork", B=4, copies=8, Hkv=8, T=5001, page=128, deep=False),
        # whole copies of long sequences (a sequence that is to be rewritten in place)
        dict(name="copy 8 x 16384", op="fork", B=8, copies=1, Hkv=8, T=16384, page=64, deep=True),
        # one row of logits of a small vocabulary: the smallest sampling call
        dict(name="sample 1x32000", op="sample", R=1, V=32000, dtype="bfloat16", filters="k+p"),
        # a serving batch, an odd vocabulary, parameters of each row's own, greedy rows among them
        dict(name="sample 64x100003", op="sample", R=64, V=100003, dtype="float16", filters="mixed"),
        # the rows of a large batch's drafted trees
        dict(name="sample 512x131072", op="sample", R=512, V=131072, dtype="float32", filters="p+min"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "commit", "prompt", "fork", "sample", "sample"])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    if op == "attention":
        Hkv = rng.choice([1, 2, 4, 8])
        G = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        N = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 64)])
        B = _log(rng, 1, 32)
        T = max(N, _log(rng, 1, 65536))
        while B > 1 and (B * T * Hkv > 2 ** 20 or B * T * Hkv * G * N > 2 ** 26):
            B //= 2
        while T * Hkv > 2 ** 20 or B * T * Hkv * G * N > 2 ** 26:
            T = max(N, T // 2)
        return dict(op=op, B=B, Hq=Hkv * G, Hkv=Hkv, N=N, T=T, ragged=rng.random() < 0.7, page=page,
                    tree=rng.random() < 0.5, dtype=dtype)
    Hkv = rng.choice([1, 2, 4, 8])
    if op == "commit":
        N = _log(rng, 1, 64)
        return dict(op=op, B=_log(rng, 1, 32), Hkv=Hkv, N=N, T=_log(rng, N + 1, 700), page=page, dtype=dtype)
    if op == "prompt":
        return dict(op=op, B=_log(rng, 1, 6), Hkv=Hkv, N=_log(rng, 1, 4096), page=page, dtype=dtype)
    if op == "fork":
        return dict(op=op, B=_log(rng, 1, 8), copies=_log(rng, 1, 4), Hkv=Hkv, T=_log(rng, 1, 4096), page=page,
                    deep=rng.random() < 0.5)
    return dict(op=op, R=_log(rng, 1, 200), V=_log(rng, 100, 131072), dtype=dtype,
                filters=rng.choice(["none", "k", "p", "k+p", "p+min", "mixed"]))


def _lens(case):
    """Cached tokens of each sequence, the drafted ones included."""
    B, T = case["B"], case["T"]
    if case["op"] == "attention" and not case["ragged"]:
        return [T] * B
    low = case["N"] if case["op"] == "attention" else 1
    return [max(low, int(T * (1.0 - 0.7 * ((b * 0.6180339887) % 1.0)))) for b in range(B)]


def _prompt_counts(case):
    return [max(1, int(case["N"] * (1.0 - 0.45 * ((b * 0.6180339887) % 1.0)))) for b in range(case["B"])]


def work(case):
    op = case["op"]
    if op == "sample":
        size = {"float32": 4}.get(case["dtype"], 2)
        return {"bytes": case["R"] * (case["V"] * size + 32), "flops": 2 * case["R"] * case["V"]}
    Hkv = case["Hkv"]
    token = 2 * (Hkv * (D // 2 + D // 16) + 4)  # stored bytes of a token
    if op == "attention":
        size = {"float32": 4}.get(case["dtype"], 2)
        total = sum(_lens(case))
        return {"bytes": total * token + 2 * case["B"] * case["N"] * case["Hq"] * D * size,
                "flops": 4 * D * case["Hq"] * case["N"] * total}
    if op == "commit":  # drafted tokens in, their packed form out, the kept ones moved, all gathered as bf16
        size = {"float32": 4}.get(case["dtype"], 2)
        n = case["B"] * case["N"]
        kept = sum(_lens(case)) + n // 2
        return {"bytes": n * (2 * Hkv * D * size + 2 * token) + kept * (token + 2 * Hkv * D * 2),
                "flops": 8 * n * Hkv * D}
    if op == "prompt":
        size = {"float32": 4}.get(case["dtype"], 2)
        n = sum(_prompt_counts(case))
        return {"bytes": n * (2 * Hkv * D * size + 2 * token) + 2 * case["B"] * case["N"] * Hkv * D * 2,
                "flops": 8 * n * Hkv * D}
    P, c = case["page"], case["copies"]
    copied = sum((-(-n // P) if case["deep"] else (n % P > 0)) for n in _lens(case)) * c
    pages = sum(-(-n // P) for n in _lens(case))
    return {"bytes": 2 * copied * P * token + (2 * c + 1) * pages * 8 + 64, "flops": 0}


# ------------------------------------------------------------------ inputs
def _pack(x):
    """[..., n] values -> codes [..., n/2], E4M3 scale bytes [..., n/16], g [...] of the last axis (see above)."""
    x = x.float()
    g = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(g)
    g = torch.where(g < TINY, 0.0, g)
    y = torch.where(bad, 0.0, x * torch.where(g == 0, 0.0, 1.0 / g))
    y = y.unflatten(-1, (-1, 16))
    s8 = (y.abs().amax(-1, keepdim=True) * torch.tensor(SIXTH, device=x.device)).to(torch.float8_e4m3fn)
    s = s8.float()
    z = (y * torch.where(s == 0, 0.0, 1.0 / s)).clamp(-6.0, 6.0)
    a = z.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.round(a / step) * step
    code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4)) + torch.where(z < 0, 8.0, 0.0)
    code = code.flatten(-2).to(torch.uint8)
    g = torch.where(bad, float("nan"), g).squeeze(-1)
    return code[..., 0::2] | (code[..., 1::2] << 4), s8.squeeze(-1).view(torch.uint8), g


def _tree_parents(B, N, gen, device):
    """Parents of B random trees of N nodes: node 0 is the root, a node's parent comes before it."""
    r = torch.rand(B, N, generator=gen, device=device)
    j = torch.arange(N, device=device)
    return torch.where(j == 0, -1, torch.minimum((r * j).long(), (j - 1).clamp(min=0)))


def _ancestors(parents):
    """[B, N, N] truth values: node j is node i or one of its ancestors."""
    B, N = parents.shape
    seen = torch.eye(N, dtype=torch.bool, device=parents.device).expand(B, N, N).clone()
    at = parents.clone()
    for _ in range(N - 1):
        seen |= (at[..., None] == torch.arange(N, device=parents.device))
        at = torch.where(at >= 0, parents.gather(1, at.clamp(min=0)), at)
    return seen


class State(dict):
    __getattr__ = dict.__getitem__


def _new_cache(pages, P, Hkv, seqs, per_seq, device):
    if own:
        from fp4_attn_b200.paged_cache import PagedNVFP4Cache
        return PagedNVFP4Cache(num_pages=pages, page_size=P, num_kv_heads=Hkv, head_dim=D, max_seqs=seqs,
                               max_pages_per_seq=per_seq, device=device)
    u8 = dict(dtype=torch.uint8, device=device)
    c = State(page_table=torch.full((seqs, per_seq), -1, dtype=torch.int32, device=device),
              lens=torch.zeros(seqs, dtype=torch.int32, device=device),
              refs=torch.zeros(pages, dtype=torch.int32, device=device), page_size=P)
    for x in "kv":
        c[x + "_codes"] = torch.zeros(pages, Hkv, P, D // 2, **u8)
        c[x + "_scales"] = torch.zeros(pages, Hkv, P, D // 16, **u8)
        c[x + "_g"] = torch.zeros(pages, P, device=device)
    return c


def _fill(cache, lens, gen, order=None):
    """Sequences 0.. of the cache get lens[b] tokens of random K and V, in pages of a random order."""
    pages, Hkv, P, _ = cache.k_codes.shape
    dev = cache.k_codes.device
    for x in "kv":
        t = torch.randn(pages, P, Hkv * D, generator=gen, device=dev)
        t *= torch.exp(0.3 * torch.randn(pages, P, 1, generator=gen, device=dev))
        codes, scales, g = _pack(t)
        del t
        getattr(cache, x + "_codes").copy_(codes.view(pages, P, Hkv, -1).transpose(1, 2))
        getattr(cache, x + "_scales").copy_(scales.view(pages, P, Hkv, -1).transpose(1, 2))
        getattr(cache, x + "_g").copy_(g)
    used = [-(-n // P) for n in lens]
    ids = torch.randperm(pages, generator=gen, device=dev)[:sum(used)].int() if order is None else order
    at = 0
    for b, n in enumerate(used):
        cache.page_table[b, :n] = ids[at:at + n]
        at += n
    cache.lens[:len(lens)] = torch.tensor(lens, dtype=torch.int32, device=dev)
    cache.refs[ids.long()] = 1


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    dtype = DTYPES[case.get("dtype", "float32")]
    s = State(op=op, case=case)
    if op == "sample":
        R, V = case["R"], case["V"]
        x = torch.randn(R, V, generator=gen, device=dev) * 2.5
        x += 8.0 * torch.rand(R, V, generator=gen, device=dev).pow(300.0)  # a few likely tokens
        x[:, -max(1, V // 50):] = float("-inf")  # tokens that the vocabulary does not use
        f = case["filters"]
        s.update(logits=x.to(dtype), u=torch.rand(R, generator=gen, device=dev))
        row = torch.arange(R, device=dev)
        flat = lambda v: torch.full((R,), v, device=dev)  # noqa: E731
        s.temperature = flat(0.8) if f != "mixed" else 0.25 * (row % 7)
        s.top_k = flat(50).int() if "k" in f else (row * 37 % 300).int() if f == "mixed" else flat(0).int()
        s.top_p = flat(0.9) if "p" in f else 1.0 - 0.05 * (row % 5) if f == "mixed" else flat(1.0)
        s.min_p = flat(0.02) if "min" in f else 0.01 * (row % 3) if f == "mixed" else flat(0.0)
        s.temperature, s.top_p, s.min_p = (t.float() for t in (s.temperature, s.top_p, s.min_p))
        return s
    P, Hkv, B = case["page"], case["Hkv"], case["B"]
    if op == "attention":
        lens = _lens(case)
        per = -(-case["T"] // P)
        used = sum(-(-n // P) for n in lens)
        s.cache = _new_cache(used + max(1, used // 16), P, Hkv, B, per, dev)
        _fill(s.cache, lens, gen)
        s.q = (2.0 * torch.randn(B, case["Hq"], case["N"], D, generator=gen, device=dev)).to(dtype)
        s.mask = _ancestors(_tree_parents(B, case["N"], gen, dev)) if case["tree"] else None
        return s
    if op == "commit":
        lens, N = _lens(case), case["N"]
        per = -(-(case["T"] + N) // P)
        s.cache = _new_cache(B * per + 8, P, Hkv, B, per, dev)
        _fill(s.cache, lens, gen)
        s.lens0 = s.cache.lens.clone()
        r = torch.rand(B, N, generator=gen, device=dev) < 0.5
        s.counts = r.sum(1).int()
        j = torch.arange(N, device=dev)
        s.keep = torch.where(r, j, N).sort(1).values.clamp(max=N - 1).int()  # the kept nodes, in order, come first
    elif op == "prompt":
        N = case["N"]
        per = -(-N // P)
        s.cache = _new_cache(B * per + 8, P, Hkv, B, per, dev)
        s.counts = torch.tensor(_prompt_counts(case), dtype=torch.int32, device=dev)
    else:
        lens, c = _lens(case), case["copies"]
        per = -(-case["T"] // P)
        used = [-(-n // P) for n in lens]
        new = sum(used) * c if case["deep"] else B * c
        s.cache = _new_cache(sum(used) + new + 8, P, Hkv, B * (1 + c), per, dev)
        _fill(s.cache, lens, gen)
        s.src = torch.arange(B * c, device=dev).div(c, rounding_mode="floor").int()
        s.dst = (B + torch.arange(B * c, device=dev)).int()
        return s
    s.k = torch.randn(B, case["N"], Hkv, D, generator=gen, device=dev).to(dtype).transpose(1, 2)
    s.v = torch.randn(B, case["N"], Hkv, D, generator=gen, device=dev).to(dtype).transpose(1, 2)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    if s.op == "attention":
        from fp4_attn_b200.paged_cache import tree_attention
        return tree_attention(s.q, s.cache, mask=s.mask)
    if s.op == "sample":
        from fp4_attn_b200.sampling import sample
        return sample(s.logits, s.u, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p, min_p=s.min_p)
    c = s.cache
    if s.op == "commit":
        c.truncate(s.lens0)
        c.append(s.k, s.v)
        c.compact(s.keep, s.counts)
        k, v = c.gather(s.case["T"] + s.case["N"], dtype=torch.bfloat16)
        return k, v, c.page_table, c.lens, c.refs
    if s.op == "prompt":
        c.release()
        c.append(s.k, s.v, counts=s.counts)
        k, v = c.gather(s.case["N"], dtype=torch.bfloat16)
        return k, v, c.page_table, c.lens, c.refs
    c.release(s.dst)
    c.fork(s.src, s.dst, deep=s.case["deep"])
    return [getattr(c, n) for n in POOLS] + [c.page_table, c.lens, c.refs]


def _run_plain(s):
    if s.op == "attention":
        return _plain_attention(s)
    if s.op == "sample":
        return _plain_sample(s)
    c = s.cache
    rows = torch.arange(c.lens.shape[0], device=c.lens.device)
    if s.op == "commit":
        _plain_shorten(c, rows, torch.minimum(c.lens, s.lens0))
        _plain_append(c, s.k, s.v, torch.full_like(c.lens, s.case["N"]))
        base = c.lens - s.case["N"]
        _plain_move(c, base, s.keep, s.counts)
        _plain_shorten(c, rows, base + s.counts)
        return *_plain_gather(c, s.case["T"] + s.case["N"]), c.page_table, c.lens, c.refs
    if s.op == "prompt":
        _plain_shorten(c, rows, torch.zeros_like(c.lens))
        _plain_append(c, s.k, s.v, s.counts)
        return *_plain_gather(c, s.case["N"]), c.page_table, c.lens, c.refs
    _plain_shorten(c, s.dst.long(), torch.zeros_like(s.dst))
    _plain_fork(c, s.src.long(), s.dst.long(), s.case["deep"])
    return [c[n] for n in POOLS] + [c.page_table, c.lens, c.refs]


def _values(codes, scales):
    """code * s of packed rows: [..., n/2], [..., n/16] -> [..., n] in 32 bits."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat((grid, -grid))
    byte = torch.arange(256, device=codes.device)
    pair = torch.stack((grid[byte & 15], grid[byte >> 4]), -1)
    x = pair[codes.int()].flatten(-2).unflatten(-1, (-1, 16))
    return (x * scales.view(torch.float8_e4m3fn).float()[..., None]).flatten(-2)


def _plain_dense(c, x):
    """[S, Hkv, T, D] values of every sequence's tokens, T the page table's whole width (unused pages: page 0)."""
    ids = c["page_table"].clamp(min=0).int()
    y = _values(c[x + "_codes"][ids], c[x + "_scales"][ids]) * c[x + "_g"][ids][:, :, None, :, None]
    return y.transpose(1, 2).flatten(2, 3)


def _plain_attention(s):
    c, q = s.cache, s.q
    B, Hq, N, _ = q.shape
    Hkv = c.k_codes.shape[1]
    codes, scales, g = _pack(q.transpose(1, 2).reshape(B, N, Hq * D))
    qh = (_values(codes, scales) * g[..., None]).view(B, N, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    S = torch.matmul(qh.reshape(B, Hkv, -1, D), _plain_dense(c, "k").transpose(-1, -2)) * D ** -0.5
    S = S.view(B, Hkv, Hq // Hkv, N, -1)
    pos = torch.arange(S.shape[-1], device=q.device)
    node = pos - (c.lens[:, None].long() - N)  # [B, T]: < 0 before the drafted tokens
    i = torch.arange(N, device=q.device)
    if s.mask is None:
        seen = node[:, None, :] <= i[:, None]
    else:
        at = node.clamp(0, N - 1)[:, None, :].expand(B, N, -1)
        seen = (node < 0)[:, None, :] | (s.mask.gather(2, at) & (node < N)[:, None, :])
    S = torch.where(seen[:, None, None], S, float("-inf"))
    e = torch.exp(S - S.amax(-1, keepdim=True))
    o = torch.matmul((e / e.sum(-1, keepdim=True)).flatten(2, 3), _plain_dense(c, "v"))
    return o.view(B, Hq, N, D).transpose(1, 2).to(q.dtype)


def _plain_shorten(c, rows, lens):
    """Sequences `rows` keep lens tokens; pages that no sequence holds any more are free (refs 0)."""
    have = c.page_table[rows]
    drop = (torch.arange(have.shape[1], device=have.device) * c.page_size >= lens[:, None]) & (have >= 0)
    c.refs.index_add_(0, have.clamp(min=0).flatten().long(), -drop.flatten().int())
    c.page_table[rows] = torch.where(drop, -1, have)
    c.lens[rows] = lens


def _plain_take(c, rows, want):
    """Sequences `rows` get pages up to want each: the lowest free ones, in order."""
    have = c.page_table[rows]
    j = torch.arange(have.shape[1], device=have.device)
    new = (have < 0) & (j < want[:, None])
    free = torch.argsort((c.refs > 0).int(), stable=True).int()
    ids = free[(new.flatten().cumsum(0) - 1).clamp(min=0)].view(have.shape)
    c.page_table[rows] = torch.where(new, ids, have)
    c.refs.index_add_(0, ids.flatten().long(), new.flatten().int())


def _plain_slots(c, pos):
    """(page, slot in the page) of positions pos [B, n] of sequences 0..B-1."""
    P = c.page_size
    page = c.page_table[:pos.shape[0]].gather(1, (pos // P).clamp(0, c.page_table.shape[1] - 1).long())
    return page.long(), (pos % P).long()


def _plain_append(c, k, v, counts):
    B, Hkv, N, _ = k.shape
    rows = torch.arange(B, device=k.device)
    P = c.page_size
    _plain_take(c, rows, (c.lens[:B] + counts + P - 1) // P)
    j = torch.arange(N, device=k.device, dtype=torch.int32)
    page, slot = _plain_slots(c, c.lens[:B, None] + j)
    live = j < counts[:, None]
    page, slot = page[live], slot[live]
    for x, t in (("k", k), ("v", v)):
        codes, scales, g = _pack(t.transpose(1, 2).reshape(B, N, Hkv * D)[live])
        c[x + "_codes"][page, :, slot] = codes.view(-1, Hkv, D // 2)
        c[x + "_scales"][page, :, slot] = scales.view(-1, Hkv, D // 16)
        c[x + "_g"][page, slot] = g
    c.lens[:B] += counts


def _plain_move(c, base, keep, counts):
    B, N = keep.shape
    j = torch.arange(N, device=keep.device, dtype=torch.int32)
    live = j < counts[:, None]
    p0, s0 = (t[live] for t in _plain_slots(c, base[:, None] + keep))
    p1, s1 = (t[live] for t in _plain_slots(c, base[:, None] + j))
    for x in POOLS:
        if x.endswith("_g"):
            c[x][p1, s1] = c[x][p0, s0]
        else:
            c[x][p1, :, s1] = c[x][p0, :, s0]


def _plain_gather(c, T):
    live = (torch.arange(T, device=c.lens.device) < c.lens[:, None])[:, None, :, None]
    return [torch.where(live, _plain_dense(c, x)[:, :, :T], 0.0).to(torch.bfloat16) for x in "kv"]


def _plain_fork(c, src, dst, deep):
    P = c.page_size
    lens, from_ = c.lens[src], c.page_table[src]
    j = torch.arange(from_.shape[1], device=src.device)
    held = from_ >= 0
    shared = held & ((j + 1) * P <= lens[:, None]) & (not deep)
    c.page_table[dst] = torch.where(shared, from_, -1)
    c.refs.index_add_(0, from_.clamp(min=0).flatten().long(), shared.flatten().int())
    # the rest gets pages of its own: all are missing, the shared ones are not
    _plain_take(c, dst, held.sum(1))
    copied = held & ~shared
    p0, p1 = from_[copied].long(), c.page_table[dst][copied].long()
    for x in POOLS:
        c[x][p1] = c[x][p0]
    c.lens[dst] = lens


ONE = 2.0 ** 34  # weights are held as whole multiples of 2^-34 of the largest one, so that sums have no order


def _plain_sample(s):
    x = s.logits.float()
    R, V = x.shape
    x = torch.where(torch.isnan(x), float("-inf"), x).clamp(max=torch.finfo(torch.float32).max)
    m = x.amax(1, keepdim=True)
    greedy = (s.temperature <= 0)[:, None]
    T = torch.where(greedy, 1.0, s.temperature[:, None])
    w = torch.where(x == float("-inf"), 0.0, torch.exp((x - m) / T))
    W = torch.round(w * ONE).long()
    Z = W.sum(1, keepdim=True)
    xs, order = x.sort(dim=1, descending=True, stable=True)  # equal logits: lowest index first
    Ws = W.gather(1, order)
    rank = torch.arange(V, device=x.device)
    k = s.top_k[:, None]
    kept = (rank < k) | (k <= 0)
    before = (Ws * kept).cumsum(1) - Ws * kept
    mass = (Ws * kept).sum(1, keepdim=True)
    kept &= (before.double() < s.top_p[:, None].double() * mass.double()) | (rank == 0) | (s.top_p[:, None] >= 1)
    kept &= (Ws.double() >= s.min_p[:, None].double() * ONE) | (rank == 0)
    kept = torch.zeros_like(kept).scatter(1, order, kept)
    c = (W * kept).cumsum(1)
    target = torch.floor(s.u[:, None].double() * c[:, -1:].double()).long()
    over = (c > torch.minimum(target, c[:, -1:] - 1)) & kept
    token = torch.where(greedy[:, 0], order[:, 0], over.int().argmax(1))
    got = x.gather(1, token[:, None])
    logprob = (got - m) / T - torch.log(Z.double() / ONE).float()
    none = m[:, 0] == float("-inf")  # a row without a possible token
    return torch.where(none, -1, token), torch.where(none, float("-inf"), logprob[:, 0])


# ------------------------------------------------------------------ the definitions in 64 bits
def _unpack64(codes, scales):
    low, high = (codes & 15).long(), (codes >> 4).long()
    nib = torch.stack((low, high), -1).flatten(-2)
    e, frac, sign = (nib >> 1) & 3, nib & 1, 1 - 2 * (nib >> 3)
    mag = torch.where(e == 0, 0.5 * frac.double(), (1 + 0.5 * frac.double()) * 2.0 ** (e - 1).double())
    b = scales.long()
    se, sf = b >> 3, b & 7
    sc = torch.where(se == 0, sf.double() * 2.0 ** -9, (1 + sf.double() / 8) * 2.0 ** (se - 7).double())
    return sign * mag * sc.repeat_interleave(16, -1)


def exact(case, seed):
    if case["op"] == "sample":
        return _exact_sample(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, seed)
    if case["op"] in ("prompt", "commit"):
        return _exact_appended(case, seed)
    return None  # bytes that are moved: they have to be equal


def _exact_attention(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c, P = s.cache, case["page"]
    B, Hq, N, _ = s.q.shape
    Hkv, G = case["Hkv"], case["Hq"] // case["Hkv"]
    # the quantizer's definition has the 32-bit roundings of its steps
    codes, scales, g = _pack(s.q.transpose(1, 2).reshape(B, N, Hq * D))
    qh = (_unpack64(codes, scales) * g.double()[..., None]).view(B, N, Hkv, G, D)
    out = torch.empty(B, N, Hkv, G, D, dtype=torch.float64, device=s.q.device)
    for b, n in enumerate(_lens(case)):
        ids = c.page_table[b, :-(-n // P)].long()
        for h in range(Hkv):
            dense = []
            for x in "kv":
                y = _unpack64(c[x + "_codes"][ids, h], c[x + "_scales"][ids, h]) * c[x + "_g"][ids].double()[..., None]
                dense.append(y.reshape(-1, D)[:n])
            S = torch.einsum("igd,td->igt", qh[b, :, h], dense[0]) / math.sqrt(D)
            seen = torch.ones(N, n, dtype=torch.bool, device=S.device)
            seen[:, n - N:] = s.mask[b] if s.mask is not None else seen[:, n - N:].tril()
            S.masked_fill_(~seen[:, None], float("-inf"))
            out[b, :, h] = torch.softmax(S, -1) @ dense[1]
    return out.view(B, N, Hq, D)


def _exact_appended(case, seed):
    """K and V of every sequence after a prompt's append, or after a commit of the kept nodes."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c, P, B = s.cache, case["page"], case["B"]
    commit = case["op"] == "commit"
    out = []
    for x, t in (("k", s.k), ("v", s.v)):
        y = torch.zeros(B, case["Hkv"], case["N"] + (case["T"] if commit else 0), D, dtype=torch.float64,
                        device=t.device)
        for b in range(B):
            new, first = t[b].transpose(0, 1), 0
            if commit:
                first = _lens(case)[b]
                ids = c.page_table[b, :-(-first // P)].long()
                old = _unpack64(c[x + "_codes"][ids], c[x + "_scales"][ids])
                old = old * c[x + "_g"][ids].double()[:, None, :, None]
                y[b, :, :first] = old.transpose(0, 1).flatten(1, 2)[:, :first]
                new = new[s.keep[b, :int(s.counts[b])].long()]
            else:
                new = new[:_prompt_counts(case)[b]]
            n = new.shape[0]
            codes, scales, g = _pack(new.reshape(n, -1))
            val = _unpack64(codes, scales) * g.double()[:, None]
            y[b, :, first:first + n] = val.view(n, case["Hkv"], D).transpose(0, 1)
        out.append(y)
    return *out, None, None, None


def _exact_sample(case, seed):
    s = prepare(case, seed)  # the same inputs in both forms
    x = s.logits.double()
    tokens, logprobs = [], []
    for r in range(case["R"]):
        T = float(s.temperature[r])
        z = x[r] / (T if T > 0 else 1.0)
        p = torch.softmax(z, 0)
        order = torch.argsort(-x[r], stable=True)
        n, k, top_p, min_p = case["V"], int(s.top_k[r]), float(s.top_p[r]), float(s.min_p[r])
        n = min(n, k) if k > 0 else n
        ps = p[order]
        if top_p < 1:
            cum = ps[:n].cumsum(0)
            n = max(1, int(((cum - ps[:n]) < top_p * cum[-1]).sum()))
        n = max(1, min(n, int((ps >= min_p * ps[0]).sum())))
        if T <= 0:
            n = 1
        kept = torch.zeros_like(p).index_copy(0, order[:n], ps[:n])
        cum = kept.cumsum(0)
        tok = int(((cum > float(s.u[r]) * cum[-1]) & (kept > 0)).int().argmax())
        tokens.append(tok)
        logprobs.append(float(z[tok] - torch.logsumexp(z, 0)))
    # the token is a whole number that the operator's fixed-point weights define: no value of its own in 64 bits
    return None, torch.tensor(logprobs, dtype=torch.float64)
