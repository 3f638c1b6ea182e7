"""Paged NVFP4 KV cache and attention of drafted tokens (host side of csrc/paged_cache.cu and csrc/paged_attn.cu).

``PagedNVFP4Cache`` holds sequences of different lengths in pages of 16 to 128
tokens that sequences can share.  Everything that changes from call to call
(lengths, page tables, reference counts) is on the device: appending drafted
tokens, dropping the rejected ones, forking and freeing sequences neither wait
for the GPU nor copy anything to the host, so a serving step can be captured
in a CUDA graph.

``tree_attention`` attends with the last N tokens of each sequence (one new
token, a chunk of a prompt, or a tree of drafted tokens with its mask) over
the whole sequence.

No reference counterpart: the reference attends over the HF cache
(llama_patch.py:212-215).  ``kv_cache.NVFP4KVCache`` keeps the reference's values
for a batch of equal lengths; here V is quantized like K -- per token, blocks
of 16 along head_dim -- since a block that runs along the tokens could be
neither moved nor shared token by token.

Layout (device tensors), H = num_kv_heads, P = page_size:
  k_codes, v_codes    uint8 [num_pages, H, P, D/2]   E2M1 pairs, element 2k in the low nibble
  k_scales, v_scales  uint8 [num_pages, H, P, D/16]  E4M3 block scales along head_dim
  k_g, v_g            fp32  [num_pages, P]           per-token global scale over all heads (row max)
  page_table          int32 [max_seqs, max_pages_per_seq], -1 past a sequence's pages
  lens                int32 [max_seqs]
  refs                int32 [num_pages]              sequences that hold a page; 0 = free

Errors that only the device can see (no free pages, a sequence longer than its
row of the page table, ...) leave the cache as it was and set bits in
``status``; ``check()`` reads them (it waits for the GPU) and raises.

``seqs`` of a call that changes sequences names each of them once (twice is
such an error); ``gather`` and ``tree_attention`` may read one in several rows.

Calls on one cache go to one stream, or are ordered by the caller.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

HEAD_DIM = 128
PAGE_SIZES = (16, 32, 64, 128)
ERRORS = {1: "not enough free pages", 2: "a sequence is longer than its row of the page table",
          4: "a keep list is not increasing or leaves its tail", 8: "a write to a shared page (fork with deep=True)",
          16: "a sequence index out of range, a sequence named twice, or a fork onto a sequence that is not empty"}


class _Struct(ctypes.Structure):  # fp4paged_cache of include/fp4attn.h
    _fields_ = [(n, ctypes.c_void_p) for n in ("k_codes", "k_scales", "k_g", "v_codes", "v_scales", "v_g",
                                               "page_table", "lens", "refs", "status", "work")] + \
               [(n, ctypes.c_int32) for n in ("num_pages", "page_size", "num_kv_heads", "head_dim", "max_seqs",
                                              "max_pages")]


def _int32(name: str, t: torch.Tensor | None, shape: tuple, device) -> int | None:
    """Address of an optional int32 device tensor of a call (None: NULL)."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.device != device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape} on {device}")
    return t.data_ptr()


class PagedNVFP4Cache:
    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, max_seqs: int,
                 max_pages_per_seq: int, device):
        if head_dim != HEAD_DIM:
            raise NotImplementedError(f"head_dim {head_dim}: the kernels implement {HEAD_DIM}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if min(num_pages, num_kv_heads, max_seqs, max_pages_per_seq) <= 0:
            raise ValueError("num_pages, num_kv_heads, max_seqs and max_pages_per_seq must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("fp4_attn_b200 runs on CUDA tensors only (no CPU path)")
        self.num_pages, self.page_size, self.num_kv_heads, self.head_dim = num_pages, page_size, num_kv_heads, head_dim
        self.max_seqs, self.max_pages_per_seq = max_seqs, max_pages_per_seq
        u8 = dict(dtype=torch.uint8, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        pages = (num_pages, num_kv_heads, page_size)
        self.k_codes = torch.zeros(*pages, head_dim // 2, **u8)
        self.k_scales = torch.zeros(*pages, head_dim // 16, **u8)
        self.k_g = torch.zeros(num_pages, page_size, device=device)
        self.v_codes = torch.zeros(*pages, head_dim // 2, **u8)
        self.v_scales = torch.zeros(*pages, head_dim // 16, **u8)
        self.v_g = torch.zeros(num_pages, page_size, device=device)
        self.page_table = torch.full((max_seqs, max_pages_per_seq), -1, **i32)
        self.lens = torch.zeros(max_seqs, **i32)
        self.refs = torch.zeros(num_pages, **i32)
        self.status = torch.zeros(1, **i32)
        self._work = torch.empty(_lib.load().fp4paged_work_size(num_pages, max_seqs), **i32)
        self.device = self.lens.device
        tensors = (self.k_codes, self.k_scales, self.k_g, self.v_codes, self.v_scales, self.v_g, self.page_table,
                   self.lens, self.refs, self.status, self._work)
        self._index = self.device.index
        self._work_bytes = {}  # workspace sizes of tree_attention by shape
        self._spaces = []      # workspaces, the last one in use: older ones stay, as captured graphs may hold them
        self._struct = _Struct(*(t.data_ptr() for t in tensors), num_pages, page_size, num_kv_heads, head_dim,
                               max_seqs, max_pages_per_seq)
        self._ref = ctypes.addressof(self._struct)

    # ------------------------------------------------------------ helpers
    def _call(self, name: str, *args) -> None:
        _lib.call_on(self._index, name, self._ref, *args)

    def _workspace(self, B: int, Hq: int, N: int) -> torch.Tensor:
        need = self._work_bytes.get((B, Hq, N))
        if need is None:
            with torch.cuda.device(self._index):  # the size goes by the device's SMs
                need = _lib.load().fp4paged_attention_workspace_size(B, Hq, self.num_kv_heads, N)
            self._work_bytes[B, Hq, N] = need
        if not self._spaces or self._spaces[-1].numel() < need:
            grown = max(need, 2 * self._spaces[-1].numel()) if self._spaces else need
            self._spaces.append(torch.empty(grown, dtype=torch.uint8, device=self.device))
        return self._spaces[-1]

    def _rows(self, seqs: torch.Tensor | None, B: int) -> int | None:
        if B > self.max_seqs:
            raise ValueError(f"{B} rows, the cache has {self.max_seqs} sequences")
        return None if seqs is None else _int32("seqs", seqs, (B,), self.device)

    def check(self) -> None:
        """Wait for the GPU and raise if a call since the last check could not be carried out."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise RuntimeError("paged cache: " + "; ".join(m for b, m in ERRORS.items() if bits & b))

    # --------------------------------------------------------- operations
    def append(self, k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor | None = None,
               counts: torch.Tensor | None = None) -> None:
        """Quantize T new tokens per row, k and v [B, H, T, D] (post-RoPE K), and store them behind sequence
        seqs[b] (int32 [B], each sequence once; default: b); counts [B] int32: only the first counts[b] tokens of row
        b."""
        shape, device = k.shape, self.device
        if k.device != device or v.device != device:
            _lib.require_cuda(k, v)
            raise ValueError(f"k and v must be on {device}")
        if len(shape) != 4 or shape != v.shape or shape[1] != self.num_kv_heads or shape[3] != self.head_dim:
            raise ValueError(f"k and v must be [B, {self.num_kv_heads}, T, {self.head_dim}]")
        code = _lib.DTYPE_CODE.get(k.dtype)
        if code is None or k.dtype != v.dtype:
            raise ValueError("k and v must both be float32, bfloat16 or float16")
        B, _, T, _ = shape
        if k.stride(3) != 1:
            k = k.contiguous()
        if v.stride(3) != 1:
            v = v.contiguous()
        ks, vs = k.stride(), v.stride()
        self._call("fp4paged_append", k.data_ptr(), v.data_ptr(), code, B, T, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                   self._rows(seqs, B), None if counts is None else _int32("counts", counts, (B,), device))

    def truncate(self, lens: torch.Tensor, seqs: torch.Tensor | None = None) -> None:
        """Row b (sequence seqs[b], each once) keeps its first lens[b] tokens (int32 [B]) if it has more; pages nobody
        holds become free."""
        B = lens.shape[0]
        self._call("fp4paged_truncate", _int32("lens", lens, (B,), self.device), self._rows(seqs, B), B)

    def release(self, seqs: torch.Tensor | None = None) -> None:
        """Empty the sequences seqs (int32, each once; default: all) and free the pages that nobody else holds."""
        B = self.max_seqs if seqs is None else seqs.shape[0]
        self._call("fp4paged_truncate", None, self._rows(seqs, B), B)

    def compact(self, keep: torch.Tensor, counts: torch.Tensor, seqs: torch.Tensor | None = None,
                tails: torch.Tensor | None = None) -> None:
        """Of the last tails[b] tokens (default: N) of row b keep those listed in keep[b, :counts[b]] (int32 [B, N],
        increasing, 0 = the tail's first token), moved together; the rest is dropped.  seqs: each sequence once."""
        if keep.dim() != 2:
            raise ValueError("keep must be [B, N]")
        B, N = keep.shape
        self._call("fp4paged_compact", _int32("keep", keep, (B, N), self.device),
                   _int32("counts", counts, (B,), self.device), _int32("tails", tails, (B,), self.device),
                   self._rows(seqs, B), B, N)

    def fork(self, src: torch.Tensor, dst: torch.Tensor, deep: bool = False) -> None:
        """The empty sequences dst become copies of src (int32 [n] each, dst distinct): full pages are shared, a last
        page that is not full is copied; deep=True copies every page."""
        n = src.shape[0]
        if n > self.max_seqs:
            raise ValueError(f"{n} rows, the cache has {self.max_seqs} sequences")
        self._call("fp4paged_fork", _int32("src", src, (n,), self.device), _int32("dst", dst, (n,), self.device), n,
                   1 if deep else 0)

    def gather(self, T: int, seqs: torch.Tensor | None = None, B: int | None = None,
               dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """Dequantized K and V of the first T tokens, [B, H, T, D] each, 0 past a sequence's end
        (B rows: len(seqs), or the first B sequences, by default all)."""
        if dtype not in _lib.DTYPE_CODE:
            raise ValueError("dtype must be float32, bfloat16 or float16")
        if T < 0:
            raise ValueError("T must not be negative")
        B = seqs.shape[0] if seqs is not None else self.max_seqs if B is None else B
        rows = self._rows(seqs, B)
        shape = (B, self.num_kv_heads, T, self.head_dim)
        k, v = torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device)
        self._call("fp4paged_gather", k.data_ptr(), v.data_ptr(), _lib.DTYPE_CODE[dtype], rows, B, T)
        return k, v


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """Mask of drafted trees for ``tree_attention``: parents [B, N] (a node's parent comes before it, -1: none;
    what is not before it counts as none) -> bool [B, N, N], node i sees itself and its ancestors."""
    N = parents.shape[-1]
    nodes = torch.arange(N, device=parents.device)
    at, seen = nodes.expand(parents.shape), None
    parents = torch.where(parents < nodes, parents, -1).long()
    for _ in range(N):
        hit = at[..., None] == nodes
        seen = hit if seen is None else seen | hit
        at = torch.where(at >= 0, parents.gather(-1, at.clamp(min=0)), at)
    return seen


def tree_attention(q: torch.Tensor, cache: PagedNVFP4Cache, mask: torch.Tensor | None = None,
                   seqs: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                   scaling: float | None = None, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the last N tokens of each sequence over the sequence: q [B, Hq, N, D] (post-RoPE) -> [B, N, Hq, D].

    The N tokens are in the cache already (append first).  Every token before
    them is visible; among them node j is visible to node i where mask[i, j]
    (bool, [N, N] or [B, N, N]) says so -- without a mask, where j <= i.  A row
    that sees nothing is 0.  counts [B] int32: row b has counts[b] <= N nodes;
    the rest of its output is 0.  seqs [B] int32: the sequence of each row.

    q is quantized to NVFP4 as the cache's tokens are (per token over its Hq*D
    channels), QK^T runs on the FP4 tensor cores, softmax in fp32, and P is not
    quantized: blocks of P would run over sibling nodes, so that a token's
    output would depend on what else was drafted.  (As it is, only its last
    places do: how the keys are shared out, and the maximum that weights are
    rounded under, go by all rows of the call.)  The output has q's dtype
    unless out or out_dtype says otherwise.  V tokens whose largest value is
    below 2^-100 count as 0.

    workspace: a device buffer of fp4paged_attention_workspace_size bytes,
    256-byte aligned (default: one that the cache keeps).
    """
    device = q.device
    if device != cache.device:
        _lib.require_cuda(q)
        raise ValueError(f"q must be on {cache.device}")
    if q.dim() != 4:
        raise ValueError("q must be [B, Hq, N, D]")
    B, Hq, N, D = q.shape
    if D != cache.head_dim or Hq % cache.num_kv_heads or Hq == 0:
        raise ValueError(f"q [B, Hq, N, {cache.head_dim}] needs Hq a multiple of {cache.num_kv_heads}")
    in_code = _lib.DTYPE_CODE.get(q.dtype)
    if in_code is None:
        raise ValueError("q must be float32, bfloat16 or float16")
    sB, sH, sN, sD = q.stride()
    if sD != 1:
        q = q.contiguous()
        sB, sH, sN, _ = q.stride()
    if out_dtype is None:
        out_dtype = q.dtype if out is None else out.dtype
    out_code = _lib.DTYPE_CODE.get(out_dtype)
    if out_code is None:
        raise ValueError("the output must be float32, bfloat16 or float16")
    if out is None:
        out = torch.empty((B, N, Hq, D), dtype=out_dtype, device=device)
    elif out.shape != (B, N, Hq, D) or out.dtype != out_dtype or not out.is_contiguous() or out.device != device:
        raise ValueError(f"out must be a contiguous {out_dtype} [B, N, Hq, D] tensor on {device}")
    mp, mB, mI, mJ = None, 0, 0, 0
    if mask is not None:
        if mask.dtype != torch.bool or mask.device != device or mask.shape not in ((N, N), (B, N, N)):
            raise ValueError(f"mask must be bool [N, N] or [B, N, N] on {device}")
        mp, mI, mJ = mask.data_ptr(), mask.stride(-2), mask.stride(-1)
        mB = mask.stride(0) if mask.dim() == 3 else 0
    if B == 0 or N == 0:
        return out
    if workspace is None:
        workspace = cache._workspace(B, Hq, N)
    elif workspace.device != device or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous buffer on {device}")
    cache._call("fp4paged_attention", q.data_ptr(), in_code, B, Hq, N, sB, sH, sN, mp, mB, mI, mJ,
                None if counts is None else _int32("counts", counts, (B,), device), cache._rows(seqs, B),
                D ** -0.5 if scaling is None else float(scaling), out.data_ptr(), out_code, workspace.data_ptr(),
                workspace.numel() * workspace.element_size())
    return out
