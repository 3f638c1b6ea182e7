"""Sampling from logits with given random numbers, and acceptance of drafted tokens (host side of csrc/sampling.cu).

The random numbers are inputs: a result can be repeated, and every rank of a
tensor-parallel job that holds the same logits draws the same token.

No reference counterpart: the reference leaves generation to transformers.
"""
from __future__ import annotations

import torch

from . import _lib

MAX_VOCAB = 262144


def _per_row(name: str, v, R: int, dtype: torch.dtype, device, off) -> torch.Tensor | None:
    """A parameter as a tensor of R values (None: off for every row)."""
    if isinstance(v, torch.Tensor):
        if v.dtype != dtype or v.device != device or v.numel() != R or not v.is_contiguous():
            raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor of {R} values on {device}")
        return v
    return None if v is None or v == off else torch.full((R,), v, dtype=dtype, device=device)


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
           min_p=0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """One token per row of logits [..., V] from u [...] (fp32 in [0, 1)) -> (tokens int64 [...], logprobs fp32 [...]).

    In order of (logit descending, index ascending) a row keeps its first
    top_k tokens (<= 0: all), of those the shortest prefix with at least a share
    top_p of their probability (>= 1: all), of those the ones at least min_p
    times as probable as the first (above 1: that one only).  The token is
    where the running sum of the kept probabilities, in index order, passes u.
    temperature <= 0 takes the largest logit (the lowest index among equals).
    Each parameter is a number or a tensor of a value per row.

    logprobs: log softmax(logits / temperature) of the token, before the
    filters (temperature 1 for a greedy row).  NaN logits count as -inf, +inf as
    the largest finite value; a row without any finite logit gives token -1
    and logprob -inf.

    Probabilities are summed as whole multiples of 2^-34 of the row's largest, so
    the result does not depend on the order of the sums.
    """
    dev, shape = logits.device, logits.shape
    if dev.type != "cuda" or u.device != dev:
        _lib.require_cuda(logits, u)
        raise ValueError(f"u must be on {dev}")
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError("logits must be [..., V] with V >= 1")
    code = _lib.DTYPE_CODE.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be float32, bfloat16 or float16")
    lead, V = shape[:-1], shape[-1]
    if V > MAX_VOCAB:
        raise NotImplementedError(f"{V} logits in a row: the kernel takes up to {MAX_VOCAB}")
    if u.shape != lead or u.dtype != torch.float32:
        raise ValueError(f"u must be fp32 of shape {tuple(lead)}")
    x = logits if len(shape) == 2 else logits.reshape(-1, V)
    ld, step = x.stride()
    if step != 1 and V > 1:
        x = x.contiguous()
        ld = V
    R = x.shape[0]
    if not u.is_contiguous():
        u = u.contiguous()
    tokens = torch.empty(lead, dtype=torch.int64, device=dev)
    logprobs = torch.empty(lead, dtype=torch.float32, device=dev)
    if R == 0:
        return tokens, logprobs
    t = _per_row("temperature", temperature, R, torch.float32, dev, 1.0)
    k = _per_row("top_k", top_k, R, torch.int32, dev, 0)
    p = _per_row("top_p", top_p, R, torch.float32, dev, 1.0)
    m = _per_row("min_p", min_p, R, torch.float32, dev, 0.0)
    ptr = _lib.ptr
    _lib.call_on(dev.index, "fp4_sample", x.data_ptr(), code, R, V, ld, u.data_ptr(), ptr(t), ptr(k), ptr(p),
                 ptr(m), tokens.data_ptr(), logprobs.data_ptr())
    return tokens, logprobs


def accept_tree(parents: torch.Tensor, tokens: torch.Tensor, sampled: torch.Tensor,
                counts: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted nodes the sampled tokens accept: parents int32, tokens and sampled int64, all [B, N]
    -> (keep int32 [B, N], n int32 [B], next int64 [B]).

    Node 0 is the last token that is certain; sampled[b, i] is what the model
    says after node i.  From node 0 on, the child (its parent comes before it)
    whose token is what was sampled is accepted -- the lowest of several --
    until there is none.  keep[b, :n[b]] lists the accepted nodes for
    ``PagedNVFP4Cache.compact``; next[b] is the token sampled after the last.
    counts [B] int32: row b has counts[b] nodes.
    """
    _lib.require_cuda(parents, tokens, sampled)
    if parents.dim() != 2 or parents.shape[1] < 1 or tokens.shape != parents.shape or sampled.shape != parents.shape:
        raise ValueError("parents, tokens and sampled must be [B, N]")
    if parents.dtype != torch.int32 or tokens.dtype != torch.int64 or sampled.dtype != torch.int64:
        raise ValueError("parents must be int32, tokens and sampled int64")
    B, N = parents.shape
    dev = parents.device
    if tokens.device != dev or sampled.device != dev:
        raise ValueError(f"tokens and sampled must be on {dev}")
    if counts is not None and (counts.dtype != torch.int32 or counts.shape != (B,) or counts.device != dev):
        raise ValueError(f"counts must be int32 [{B}] on {dev}")
    keep = torch.empty(B, N, dtype=torch.int32, device=dev)
    n = torch.empty(B, dtype=torch.int32, device=dev)
    nxt = torch.empty(B, dtype=torch.int64, device=dev)
    parents, tokens, sampled = parents.contiguous(), tokens.contiguous(), sampled.contiguous()
    counts = None if counts is None else counts.contiguous()
    _lib.call_on(dev.index, "fp4_accept_tree", parents.data_ptr(), tokens.data_ptr(), sampled.data_ptr(),
                 _lib.ptr(counts), B, N, keep.data_ptr(), n.data_ptr(), nxt.data_ptr())
    return keep, n, nxt
