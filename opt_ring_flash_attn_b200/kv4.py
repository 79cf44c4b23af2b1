"""Serving what the operators of this package train: a paged K/V cache held in 4 bits, and the attention of new tokens over it.

``kv4_append`` puts tokens into the cache, ``kv4_attn`` lets the last tokens of every sequence attend to all of it (with the
capped and distance-biased scores of :func:`scored_flash_attn`): one token, a few drafted ones, or the next part of a prompt.
``kv4_gather`` reads tokens back.  Each call is asynchronous on the current stream; positions and lengths are read on the device, so
a decoding step can be captured into a CUDA graph and replayed as the sequences grow.

The reference has no serving path; the scores follow its ``alibi_slopes`` arguments (ring_flash_attn.py:385-463).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _native, workspace
from .scored import _check_slopes, _check_softcap, _refuse_tangents

PAGE = 64    # tokens of a page
GROUP = 32   # channels that share a scale and a minimum
HEAD_DIMS = (64, 96, 128, 192, 256)


class KV4Cache:
    """A pool of pages of 64 tokens.  ``codes`` is uint8 ``[n_pages, H_kv, 2, 64, D / 2]`` (K, then V), ``meta`` bf16 or fp16
    ``[n_pages, H_kv, 2, 64, D / 32, 2]``: scale and minimum of every 32 channels; a code u stands for ``u * scale + minimum``
    (5 bits a value, 3.2 times smaller than 16).  The order of the codes inside a row is that of ``rfa_kv4_append`` in the C header.
    Both tensors belong to the caller: which page holds which tokens is said by the block table of each call."""

    def __init__(self, codes: torch.Tensor, meta: torch.Tensor):
        if codes.dim() != 5 or codes.dtype != torch.uint8 or codes.shape[2] != 2 or codes.shape[3] != PAGE:
            raise ValueError(f"codes must be uint8 [n_pages, H_kv, 2, {PAGE}, D / 2], got {codes.dtype} {tuple(codes.shape)}")
        n, H, _, _, half = codes.shape
        if 2 * half not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {2 * half}")
        if n < 1 or H < 1:
            raise ValueError("a cache needs at least one page and one head")
        if meta.dtype not in _native.DTYPE_CODES or meta.shape != (n, H, 2, PAGE, 2 * half // GROUP, 2):
            raise ValueError(f"meta must be bf16 or fp16 {(n, H, 2, PAGE, 2 * half // GROUP, 2)}, got {meta.dtype} {tuple(meta.shape)}")
        if not codes.is_contiguous() or not meta.is_contiguous() or codes.data_ptr() % 16 or meta.data_ptr() % 16:
            raise ValueError("codes and meta must be contiguous and start on 16-byte boundaries")
        if meta.device != codes.device:
            raise ValueError(f"codes are on {codes.device}, meta on {meta.device}")
        self.codes, self.meta = codes, meta
        self.n_pages, self.n_kv_heads, self.head_dim = n, H, 2 * half
        self.dtype, self.device = meta.dtype, codes.device

    @classmethod
    def empty(cls, n_pages: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> "KV4Cache":
        """A pool whose pages hold nothing in particular yet."""
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        return cls(torch.empty(n_pages, n_kv_heads, 2, PAGE, head_dim // 2, dtype=torch.uint8, device=device),
                   torch.empty(n_pages, n_kv_heads, 2, PAGE, head_dim // GROUP, 2, dtype=dtype, device=device))


def _check_ints(x: Optional[torch.Tensor], B: int, device: torch.device, what: str, dims: int = 1) -> Optional[torch.Tensor]:
    if x is None:
        return None
    if x.dtype != torch.int32 or x.dim() != dims or x.shape[0] != B:
        raise ValueError(f"{what} must be int32 [{B}{', n' if dims == 2 else ''}], got {x.dtype} {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{what} is on {x.device}, the cache on {device}")
    return x if x.is_contiguous() else x.contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where the kernels can read it as it lies (whole rows of channels on 16-byte boundaries, any strides
    of the other dimensions), else a copy."""
    st = t.stride()
    if st[3] == 1 and (st[0] | st[1] | st[2]) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_tokens(t: torch.Tensor, cache: KV4Cache, heads: Optional[int], what: str) -> None:
    if t.dim() != 4 or t.shape[3] != cache.head_dim or (heads is not None and t.shape[2] != heads):
        raise ValueError(f"{what} must be [B, T, {heads if heads is not None else 'H'}, {cache.head_dim}], got {tuple(t.shape)}")
    if t.dtype != cache.dtype:
        raise ValueError(f"{what} is {t.dtype}, the cache {cache.dtype}")
    if t.device != cache.device:
        raise ValueError(f"{what} is on {t.device}, the cache on {cache.device}")


def _check_cuda(cache: KV4Cache) -> None:
    if cache.device.type != "cuda":
        raise RuntimeError("the 4-bit cache works on CUDA tensors only (sm_100a kernels; there is no CPU path)")


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, positions: torch.Tensor,
               counts: Optional[torch.Tensor] = None) -> None:
    """Writes new tokens into the cache, in place.

    Args:
      k, v: ``[B, T, H_kv, D]`` in the cache's dtype (any strides with whole rows of channels; slices of a fused projection
          are read as they lie).
      block_table: int32 ``[B, max_pages]``: the page of tokens ``[64 i, 64 i + 64)`` of each sequence.
      positions: int32 ``[B]``: position of each sequence's first new token; token t goes to ``positions[b] + t``.
      counts: int32 ``[B]``: how many of the T tokens count (all of them by default).
    Tokens beyond the table, or on a page that is not in the pool, are left out; no other token of the cache changes.  The
    result is unspecified where two tokens of one call go to the same place.  The cache holds numbers: no gradient flows through it.
    A group with a NaN, an infinity, or values further apart than fp32's largest number reads back as no numbers.
    """
    _check_tokens(k, cache, cache.n_kv_heads, "k")
    _check_tokens(v, cache, cache.n_kv_heads, "v")
    if k.shape != v.shape:
        raise ValueError(f"k and v shapes differ: {tuple(k.shape)} vs {tuple(v.shape)}")
    B = k.shape[0]
    table = _check_ints(block_table, B, cache.device, "block_table", 2)
    positions = _check_ints(positions, B, cache.device, "positions")
    counts = _check_ints(counts, B, cache.device, "counts")
    _check_cuda(cache)
    if k.numel() == 0 or table.shape[1] == 0:
        return
    _native.kv4_append(_rows(k), _rows(v), cache.codes, cache.meta, table, positions, counts)


def kv4_gather(cache: KV4Cache, block_table: torch.Tensor, positions: torch.Tensor, T: int,
               counts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Reads tokens ``positions[b] + t``, t < T, back: ``(k, v)``, each ``[B, T, H_kv, D]`` in the cache's dtype, zero where
    there is no such token (arguments as for :func:`kv4_append`)."""
    if T < 0:
        raise ValueError(f"T must not be negative, got {T}")
    B = block_table.shape[0]
    table = _check_ints(block_table, B, cache.device, "block_table", 2)
    positions = _check_ints(positions, B, cache.device, "positions")
    counts = _check_ints(counts, B, cache.device, "counts")
    _check_cuda(cache)
    shape = (B, T, cache.n_kv_heads, cache.head_dim)
    if B == 0 or T == 0 or table.shape[1] == 0:
        return tuple(torch.zeros(shape, dtype=cache.dtype, device=cache.device) for _ in range(2))
    k, v = (torch.empty(shape, dtype=cache.dtype, device=cache.device) for _ in range(2))
    _native.kv4_gather(k, v, cache.codes, cache.meta, table, positions, counts)
    return k, v


def _attn(q, cache, block_table, lens, softmax_scale, softcap, alibi_slopes, want_lse, tokens_after=None):
    _check_tokens(q, cache, None, "q")
    B, T, Hq, D = q.shape
    if Hq == 0 or Hq % cache.n_kv_heads != 0:
        raise ValueError(f"H_q must be a multiple of the cache's {cache.n_kv_heads} heads, got {Hq}")
    table = _check_ints(block_table, B, cache.device, "block_table", 2)
    lens = _check_ints(lens, B, cache.device, "lens")
    after = _check_ints(tokens_after, B, cache.device, "tokens_after")
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not (scale > 0) or math.isinf(scale):
        raise ValueError("softmax_scale must be positive and finite")
    softcap = _check_softcap(softcap, scale)
    slopes = _check_slopes(alibi_slopes, B, Hq, cache.device)
    if torch.is_grad_enabled() and q.requires_grad:
        raise RuntimeError("kv4_attn has no gradient: call it under torch.no_grad()")
    _refuse_tangents("kv4_attn", q, alibi_slopes)
    _check_cuda(cache)
    if B == 0 or T == 0 or table.shape[1] == 0:
        out = torch.zeros((B, T, Hq, D), dtype=q.dtype, device=q.device)
        return out, torch.full((B, Hq, T), -math.inf, device=q.device) if want_lse else None
    ws = workspace.status_workspace(cache.device)
    workspace.raise_if_failed(ws, "kv4_attn")
    out = torch.empty((B, T, Hq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device) if want_lse else None
    # scratch per call: calls on several streams, or in several captured graphs, do not meet in it
    scratch = torch.empty(_native.kv4_scratch_elems(B, T, Hq, cache.n_kv_heads, D), dtype=torch.float32, device=q.device)
    _native.kv4_attn(_rows(q), cache.codes, cache.meta, table, lens, after, out, lse, scratch, scale, softcap,
                     slopes, ws.status)
    workspace.publish_status(ws, "kv4_attn")
    return out, lse


def kv4_attn(q: torch.Tensor, cache: KV4Cache, block_table: torch.Tensor, lens: torch.Tensor,
             softmax_scale: Optional[float] = None, *, softcap: float = 0.0,
             alibi_slopes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the last T tokens of every sequence over its tokens in the cache (their own included: append first).

    Args:
      q: ``[B, T, H_q, D]`` in the cache's dtype: one token (T = 1), a few drafted ones, or the next part of a prompt.  The
          cache is read once for every 16 rows (8 above head dim 128) of T times the group's heads.
      block_table: int32 ``[B, max_pages]`` as for :func:`kv4_append`.
      lens: int32 ``[B]``: tokens of each sequence in the cache; query t is token ``lens[b] - T + t`` and sees the tokens up to
          itself.  Lengths beyond the table end at it; tokens on a page that is not in the pool do not exist.
      softmax_scale, softcap, alibi_slopes: as in :func:`scored_flash_attn`.

    Returns: out ``[B, T, H_q, D]``; rows that see no token are zero.  What the pages hold behind the last token does not
    matter; the tokens themselves must be finite (of T > 1, a row may take up a NaN of a token behind it), and like q so far from
    the largest numbers that a sequence's sums stay in fp32.  The weights times the scales of V are rounded to 11 bits, relative to
    the largest scale of their 32 channels; what lies 2^-18 or more below it keeps fewer.  The same call gives the same bits; the
    other sequences of a batch decide how the work is split, so another batch may give the last bits differently.
    """
    return _attn(q, cache, block_table, lens, softmax_scale, softcap, alibi_slopes, False)[0]


def kv4_attn_with_lse(q, cache, block_table, lens, softmax_scale=None, *, softcap=0.0, alibi_slopes=None,
                      tokens_after: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """As :func:`kv4_attn`, also returning the log-sum-exp ``[B, H_q, T]`` (fp32, -inf where a row sees no token).

    Where the tokens of a sequence lie in several caches (on several GPUs, say), each in a part of its own, ``tokens_after``
    (int32 ``[B]``) says how many of them lie behind the part in this one: query t is then token
    ``lens[b] + tokens_after[b] - T + t`` of this part, and sees as much of it, at the distances, as it does of the whole.  With
    ``w = exp(lse_part - logsumexp of all lse_part)`` the sum of ``w * out_part`` is the attention over the whole sequence
    (``w = 0`` where a part's lse is -inf).
    """
    return _attn(q, cache, block_table, lens, softmax_scale, softcap, alibi_slopes, True, tokens_after)
