"""Attention with modified scores: ``scored_flash_attn`` caps them by a tanh, adds a bias that falls with the distance
(ALiBi) and takes document and prefix masks, forward and backward, on one GPU or sequence-parallel on a ring.

For query i and key j (positions in the whole sequence)::

    x = softmax_scale * q_i . k_j        y = softcap * tanh(x / softcap)        z = y - slope[h] * |i - j|

and row i is the softmax of z over the keys it sees, times V.  A row that sees nothing is zero, its lse is -inf, and it takes
no part in any gradient.  The schedules of the ring are those of :mod:`.schedule`; a pass hands them a backend whose hops
know which shard of the sequence is visiting.

The reference computes causal and full attention only; its baseline file passes ``alibi_slopes`` on to flash-attn
(ring_flash_attn.py:385-463), which is what the distance bias follows.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native, schedule, workspace
from .api import _deterministic_now, _validate


MAX_SOFTCAP = 1000.0  # here the tanh is off by 5e-4 of a score (fp32)


class DocumentMask:
    """Which keys the queries of a batch see (made by :func:`document_mask`).  It lives on the device; the forward and the
    backward passes of every layer that works on the same batch read it."""

    def __init__(self, buffer, batch: int, seq_len: int, shards: int, causal: bool, has_prefix: bool, typical_keys: int = 0):
        self.buffer = buffer
        self.batch, self.seq_len, self.shards = batch, seq_len, shards
        self.causal, self.has_prefix = causal, has_prefix
        self.typical_keys = typical_keys  # guides the split of long rows over CTAs (0: a row may see everything)

    @property
    def device(self) -> torch.device:
        return self.buffer.device

    def update_(self, cu_seqlens, prefix_lens=None) -> "DocumentMask":
        """Overwrites the mask in stream order with that of other documents (a replayed graph then sees them).  A backward pass
        that is still to come and needs the old one raises, as after any change in place of what autograd saved."""
        if (prefix_lens is not None) != self.has_prefix:
            raise ValueError("update_ takes prefix_lens exactly where the mask was made with them")
        cu, prefix = _borders(cu_seqlens, prefix_lens, self.batch, self.seq_len, self.device)
        if not self.buffer.is_inference():
            torch.autograd.graph.increment_version(self.buffer)
        _native.document_mask(cu, prefix, self.batch, self.seq_len // self.shards, self.shards, self.causal, self.buffer)
        return self


_Ints = Union[torch.Tensor, Sequence]


def _int32(x: _Ints, device: torch.device, what: str) -> torch.Tensor:
    t = x if isinstance(x, torch.Tensor) else torch.tensor(x)
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what} must be int32 or int64, got {t.dtype}")
    if t.is_cuda and t.device != device:
        raise ValueError(f"{what} is on {t.device}, the mask on {device}")
    if t.dtype == torch.int64:  # what int32 cannot hold lies outside every sequence, on the same side as its ends
        t = t.clamp(-1, 2 ** 31 - 1)
    return t.to(device=device, dtype=torch.int32).contiguous()


def _borders(cu_seqlens: _Ints, prefix_lens: Optional[_Ints], batch: int, seq_len: int, device: torch.device):
    on_device = isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.is_cuda
    cu = _int32(cu_seqlens, device, "cu_seqlens")
    if cu.dim() not in (1, 2) or cu.shape[-1] < 2:
        raise ValueError(f"cu_seqlens must be [n + 1] or [B, n + 1] with n >= 1, got {tuple(cu.shape)}")
    if cu.dim() == 2 and cu.shape[0] != batch:
        raise ValueError(f"cu_seqlens has {cu.shape[0]} rows for a batch of {batch}")
    if not on_device:  # borders that came from the host are checked there; those on the device are clamped by the kernel
        host = cu_seqlens if isinstance(cu_seqlens, torch.Tensor) else torch.tensor(cu_seqlens)
        if bool((host < 0).any()) or bool((host > seq_len).any()) or bool((host.diff(dim=-1) < 0).any()):
            raise ValueError(f"cu_seqlens must not decrease and lie in [0, {seq_len}]")
    prefix = None
    if prefix_lens is not None:
        prefix = _int32(prefix_lens, device, "prefix_lens")
        if prefix.shape != (*cu.shape[:-1], cu.shape[-1] - 1):
            raise ValueError(f"prefix_lens must be {(*cu.shape[:-1], cu.shape[-1] - 1)}, got {tuple(prefix.shape)}")
    return cu, prefix


def document_mask(cu_seqlens: _Ints, seq_len: int, *, prefix_lens: Optional[_Ints] = None, causal: bool = True,
                  batch: Optional[int] = None, group=None, device: Optional[torch.device] = None) -> DocumentMask:
    """Mask of packed documents, for :func:`scored_flash_attn`.

    Args:
      cu_seqlens: document borders, int ``[n + 1]`` (the same for every batch row) or ``[B, n + 1]``; document d of a row is
          its tokens ``[cu[d], cu[d + 1])``.  Rows with fewer documents repeat their last border.  Tokens before the first
          and from the last border on are padding: they see nothing, nothing sees them, and they may hold anything.
      seq_len: length of the whole sequence (of all ranks together).
      prefix_lens: ``[n]`` or ``[B, n]``: the first so many tokens of each document are seen by all of it (prefix mask).
      causal: a token sees its document up to itself (and its prefix); otherwise all of its document.
      batch: batch size, needed where ``cu_seqlens`` is ``[n + 1]`` and the batch is not 1.
      group: the process group (or ring) the sequence is sharded over, as in the call of the attention.

    ``cu_seqlens`` and ``prefix_lens`` on the device are read there, without synchronisation: borders outside the sequence
    count as its ends, and borders that decrease give an unspecified (but safe) mask.
    """
    if device is None:
        device = cu_seqlens.device if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.is_cuda else torch.device(
            "cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:  # tensors say which one they are on
        device = torch.device("cuda", torch.cuda.current_device())
    shards, _ = schedule._world(group)
    if seq_len < 1 or seq_len % shards != 0:
        raise ValueError(f"seq_len {seq_len} must be positive and a multiple of the {shards} ranks")
    rows = cu_seqlens if isinstance(cu_seqlens, torch.Tensor) else torch.tensor(cu_seqlens)
    if batch is None:
        batch = rows.shape[0] if rows.dim() == 2 else 1
    if batch < 1:
        raise ValueError("batch must be positive")
    cu, prefix = _borders(cu_seqlens, prefix_lens, batch, seq_len, device)
    if device.type != "cuda":
        raise RuntimeError("document_mask runs on CUDA only (sm_100a kernels; there is no CPU path)")
    buffer = torch.empty(_native.mask_elems(batch, seq_len // shards, shards), dtype=torch.int32, device=device)
    _native.document_mask(cu, prefix, batch, seq_len // shards, shards, causal, buffer)
    return DocumentMask(buffer, batch, seq_len, shards, bool(causal), prefix is not None,
                        _typical_keys(seq_len, cu.shape[-1] - 1))


def _typical_keys(seq_len: int, documents: int) -> int:
    """What a long one of them holds, some twice the mean; their borders stay on the device.  Never 0, which would say: all."""
    return max(1, min(seq_len, 2 * seq_len // documents))


class _Scores:
    """What a pass does to its scores, and the kernel backend that the ring schedules call hop by hop."""

    def __init__(self, softmax_scale: float, softcap: float, slopes, causal: bool, mask_buffer, sees_later: bool,
                 world: int, rank: int, typical_keys: int = 0):
        self.scale, self.softcap, self.slopes, self.causal, self.mask = softmax_scale, softcap, slopes, causal, mask_buffer
        self.sees_later = sees_later  # some key behind a query may be visible: no hop can be left out
        self.world, self.rank, self._step = world, rank, 0
        self.typical_keys = typical_keys  # what a long document holds, as far as the host knows (0: everything)

        self._args = _native.score_args(softmax_scale, softcap, slopes, causal, mask_buffer, world, rank, rank)

    def again(self) -> "_Scores":
        """For another pass: the backward may run on another thread, and more than once."""
        return self if self.world == 1 else _Scores(self.scale, self.softcap, self.slopes, self.causal, self.mask,
                                                    self.sees_later, self.world, self.rank)

    def args(self, k_shard: int) -> _native.ScoreArgs:
        self._args.k_shard = k_shard
        return self._args

    def _next(self) -> _native.ScoreArgs:
        shard = (self.rank - self._step) % self.world  # a schedule runs its hops in the order of the steps
        self._step += 1
        return self.args(shard)

    # ---- the calls of a kernel backend (see _native) ----
    pack_kv = staticmethod(_native.pack_kv)
    bwd_prepare = staticmethod(_native.bwd_prepare)
    dq_finalize = staticmethod(_native.dq_finalize)
    dkdv_accumulate = staticmethod(_native.dkdv_accumulate)
    dkdv_accumulate_to16 = staticmethod(_native.dkdv_accumulate_to16)
    cast_from_f32 = staticmethod(_native.cast_from_f32)

    def fwd_hop(self, q, k, v, acc, m, l, out, lse, softmax_scale, first, last, causal_diag, status):
        _native.scored_fwd_hop(q, k, v, acc, m, l, out, lse, self._next(), first, last, status)

    def bwd_hop(self, q, k, v, dout, lse2, delta, dq_acc, dkdv_prev, dkdv_out, softmax_scale, accumulate_prev, causal_diag,
                status, dq_order=None):
        assert dkdv_prev is None and not accumulate_prev
        _native.scored_bwd_hop(q, k, v, dout, lse2, delta, dq_acc, dkdv_out, self._next(), status, dq_order=dq_order)


def _forward(group, q, k, v, sc: _Scores):
    if sc.world > 1:
        return schedule.ring_forward(group, q, k, v, sc.scale, not sc.sees_later, kernels=sc)
    ws = workspace.status_workspace(q.device)
    workspace.raise_if_failed(ws, "scored_flash_attn forward")
    B, S, Hq, _ = q.shape
    out = torch.empty_like(q)
    lse = torch.empty((B, Hq, _native.padded_seq(S)), dtype=torch.float32, device=q.device)
    n = _native.scored_fwd_scratch_elems(B, S, Hq, q.shape[3], sc.causal, sc.typical_keys)
    scratch = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
    _native.scored_fwd_local(q, k, v, out, lse, scratch, sc.args(0), sc.typical_keys, ws.status)
    workspace.publish_status(ws, "scored_flash_attn forward")
    return out, lse


def _backward(group, dout, q, k, v, out, lse, sc: _Scores, deterministic: bool):
    if sc.world > 1:
        return schedule.ring_backward(group, dout, q, k, v, out, lse, sc.scale, not sc.sees_later, kernels=sc,
                                      deterministic=deterministic)
    # Scratch per call: passes on several streams, or in several captured graphs, do not meet in it.
    ws = workspace.status_workspace(q.device)
    workspace.raise_if_failed(ws, "scored_flash_attn backward")
    B, S, Hq, D = q.shape
    offsets = _native.scored_bwd_scratch(B, S, Hq, k.shape[2], D, deterministic)
    scratch = torch.empty(offsets[5], dtype=torch.float32, device=q.device)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    _native.scored_bwd_local(q, k, v, out, dout, lse, scratch, offsets, dq, dk, dv, sc.args(0), ws.status,
                             deterministic=deterministic)
    workspace.publish_status(ws, "scored_flash_attn backward")
    return dq, dk, dv


def _operand(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, and on the 16-byte boundary that the copies of the kernels start on."""
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _call(q, k, v, sc: _Scores, group):
    """The forward pass on operands as the kernels want them."""
    if q.numel() == 0:
        return torch.empty_like(q), q.new_empty((q.shape[0], q.shape[2], 0), dtype=torch.float32)
    return _forward(group, q, k, v, sc)


class _ScoredFlashAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sc, group):
        q, k, v = _operand(q), _operand(k), _operand(v)
        out, lse = _call(q, k, v, sc, group)
        ctx.sc, ctx.group = sc, group
        ctx.deterministic = _deterministic_now()
        # The scores read the slopes and the mask through their own references; saved as well, a change in place between the
        # passes is found by their versions (which tensors made in inference mode do not have).
        ctx.save_for_backward(q, k, v, out, lse, *(t if t is not None and not t.is_inference() else None
                                                   for t in (sc.slopes, sc.mask)))
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _dlse=None):
        q, k, v, out, lse, _, _ = ctx.saved_tensors
        if dout is None or q.numel() == 0:
            return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), None, None
        dq, dk, dv = _backward(ctx.group, _operand(dout), q, k, v, out, lse, ctx.sc.again(), ctx.deterministic)
        return dq, dk, dv, None, None


def _refuse_tangents(what: str, *tensors) -> None:
    """Forward-mode differentiation: an output without a tangent would read as one of zero."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside of it; asking each tensor takes a microsecond apiece
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative")


def _check_slopes(slopes: Optional[torch.Tensor], B: int, Hq: int, device: torch.device) -> Optional[torch.Tensor]:
    if slopes is None:
        return None
    if slopes.shape not in ((Hq,), (B, Hq)):
        raise ValueError(f"alibi_slopes must be [{Hq}] or [{B}, {Hq}], got {tuple(slopes.shape)}")
    if slopes.dtype != torch.float32:
        raise ValueError(f"alibi_slopes must be float32, got {slopes.dtype}")
    if slopes.device != device:
        raise ValueError(f"alibi_slopes are on {slopes.device}, the queries on {device}")
    if slopes.requires_grad:
        raise ValueError("alibi_slopes are constants: there is no gradient for them (detach them)")
    return slopes.contiguous()


def _check_softcap(softcap: float, softmax_scale: float) -> float:
    softcap = float(softcap or 0.0)
    if not (0.0 <= softcap <= MAX_SOFTCAP):
        raise ValueError(f"softcap must be 0 (none) or a positive number up to {MAX_SOFTCAP:g}, got {softcap}")
    # the kernels work with scale * log2(e) and, for the tanh, 2 * scale * log2(e) / softcap in fp32
    if not (softmax_scale * 1.45 <= 3.4e38):
        raise ValueError(f"softmax_scale {softmax_scale:g} is too large for fp32")
    if softcap > 0 and not (softmax_scale * 2.9 <= 3.4e38 * softcap):
        raise ValueError(f"softcap {softcap:g} is too small for softmax_scale {softmax_scale:g}")
    return softcap


def _apply(q, k, v, softmax_scale, causal, softcap, alibi_slopes, mask, group) -> Tuple[torch.Tensor, torch.Tensor]:
    if q.dim() == 4 and softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    if k.dim() == 4 and k.shape[2] == 0:
        raise ValueError("k and v have no heads")
    _validate(q, k, v, softmax_scale)
    if math.isinf(softmax_scale):
        raise ValueError("softmax_scale must be finite")
    if k.device != q.device or v.device != q.device:
        raise ValueError(f"q, k, v are on different devices: {q.device}, {k.device}, {v.device}")
    _refuse_tangents("scored_flash_attn", q, k, v, alibi_slopes)
    B, S, Hq, _ = q.shape
    softcap = _check_softcap(softcap, softmax_scale)
    slopes = _check_slopes(alibi_slopes, B, Hq, q.device)
    causal = bool(causal)
    world, rank = schedule._world(group)
    if mask is not None:
        if not isinstance(mask, DocumentMask):
            raise ValueError("mask must come from document_mask")
        if mask.causal != causal:
            raise ValueError(f"the mask was made with causal={mask.causal}, the call says causal={causal}")
        if mask.device != q.device:
            raise ValueError(f"the mask is on {mask.device}, the queries on {q.device}")
        if (mask.batch, mask.seq_len, mask.shards) != (B, S * world, world):
            raise ValueError(f"the mask is for a batch of {mask.batch} and {mask.seq_len} tokens on {mask.shards} ranks, "
                             f"the call has {B}, {S * world} and {world}")
    sees_later = not causal or (mask is not None and mask.has_prefix)
    buffer, typical = (None, 0) if mask is None else (mask.buffer, mask.typical_keys)
    sc = _Scores(float(softmax_scale), softcap, slopes, causal, buffer, sees_later, world, rank, typical)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _ScoredFlashAttnFunc.apply(q, k, v, sc, group)
    return _call(_operand(q), _operand(k), _operand(v), sc, group)


def scored_flash_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: Optional[float] = None,
                      causal: bool = False, *, softcap: float = 0.0, alibi_slopes: Optional[torch.Tensor] = None,
                      mask: Optional[DocumentMask] = None, group=None) -> torch.Tensor:
    """Attention with modified scores, sequence-parallel like :func:`ring_flash_attn` (contiguous shards; no zigzag layout).

    Args:
      q, k, v, softmax_scale, causal, group: as in :func:`ring_flash_attn`.
      softcap: scores are capped to ``softcap * tanh(score / softcap)``, softcap up to 1000; 0 leaves them as they are.
      alibi_slopes: fp32 ``[H_q]`` or ``[B, H_q]``; ``slope * |i - j|`` is taken off the (capped) score.  Not differentiable.  Slopes and mask must
          stay as they are until the backward pass.
      mask: documents and prefixes, from :func:`document_mask` with the same ``causal`` and ``group``.

    Returns: out [B, S_local, H_q, D] in q's dtype; rows that see no key are zero.  Outside its padding (see
    :func:`document_mask`) K and V must be finite: an infinity or a NaN reaches rows that do not see it.  (In bf16 without a cap a
    masked key may keep a weight of 2^-125 of the row's largest: V has to stay below 1e30 there.)
    :func:`deterministic` holds here too, at the price of visiting every tile of a masked block.
    """
    return _apply(q, k, v, softmax_scale, causal, softcap, alibi_slopes, mask, group)[0]


def scored_flash_attn_with_lse(q, k, v, softmax_scale=None, causal=False, *, softcap=0.0, alibi_slopes=None, mask=None,
                               group=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """As :func:`scored_flash_attn`, also returning the log-sum-exp ``[B, H_q, S_local]`` of the modified scores (fp32, not
    differentiable; -inf where a row sees no key)."""
    out, lse = _apply(q, k, v, softmax_scale, causal, softcap, alibi_slopes, mask, group)
    return out, lse[:, :, : q.shape[1]]
