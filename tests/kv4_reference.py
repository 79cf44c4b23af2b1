"""Attention over the 4-bit cache from its bytes, in 64 bits, with elementwise bounds of what the kernel may be off by.

A cached value is v = u sc + mn, u in 0..15.  The kernel sums, per query row and group of 32 channels, P sc (rounded to fp16 for
its product with the codes, whatever the cache's type) times u' plus P mn' in fp32, where u' = u, mn' = mn for bf16 caches and u' = u - 8,
mn' = mn + 8 sc for fp16 ones.  With M = sum P (|u'| |sc| + |mn'|) and n keys the result is off by
  2^-11 sum P |u'| |sc|               the rounding of P sc (fp16 has 11 bits),
  2^-25 n Pmax scmax_g                where P sc falls below fp16's smallest normal number: half its smallest step, 2^-25, under a
                                      power of two that brings the group's largest scale so far to 2^4 or more, times 15;
                                      unnormalised weights are relative to a maximum at most the row's, so 1 / sum <= Pmax,
  (n / 8 + 16) 2^-23 M                its sums in fp32, longest chain n / 8,
  sum P e_p (|u'| |sc| + |mn'|)       the weights, e_p = e_s + sum P e_s, e_s the error of a score,
  u_T |out|                           its own rounding (below the type's normal numbers 2^-25 or 2^-134, with n 2^-149 for P mn there).
Scores: products of codes (4 bits) and q (11 bits at most) are exact, sums of 16 are off by 2^-23 of the magnitudes, D / 16
+ 6 of them in turn with the scale, minima and scale of the row; the group sums of q that the minima meet are two 16-bit
parts: off by 2^-17 of the sum for bf16, for fp16 by its smallest half step, 2^-25 2^24 / up with up >= 2^12 / max|q|.  Then
2^-21 of (1 + |z| + max|z|) for the change to log2 units, the subtraction of the maximum and exp2; a cap adds 2^-21 of itself.
"""
import math

import torch


def decoded(cache, table_row, n):
    """(u, sc, mn) of K and of V of the first n tokens of a sequence, in 64 bits: u [n, H, D], sc and mn [n, H, D / 32]."""
    pages = table_row[: (n + 63) // 64].long()
    codes, meta = cache.codes[pages], cache.meta[pages].double()
    D, ng = cache.head_dim, cache.head_dim // 32
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    ch = torch.arange(D, device=codes.device)
    g, r = ch // 32, ch % 32
    at = ((r // 8 * ng + g) * 8 + r % 8, (r // 4 * ng + g) * 4 + r % 4)
    res = []
    for i in range(2):
        u = nib[:, :, i][..., at[i]].double().transpose(1, 2).flatten(0, 1)[:n]
        m = meta[:, :, i].transpose(1, 2).flatten(0, 1)[:n]
        res.append((u, m[..., 0], m[..., 1]))
    return res


def _wide(x):
    return x.repeat_interleave(32, -1)


def reference(q, cache, table, lens, *, scale=None, softcap=0.0, slopes=None, after=None):
    """(out, bound, lse, lse bound).  ``after[b]``: tokens of the sequence that lie behind its part in this cache."""
    B, T, Hq, D = q.shape
    dev = q.device
    half = q.dtype == torch.float16
    uT = torch.finfo(q.dtype).eps / 2
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    bound = torch.zeros_like(out)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=dev)
    lse_bound = torch.full_like(lse, 2.0 ** -20)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        (ku, ksc, kmn), (vu, vsc, vmn) = decoded(cache, table[b], n)
        G = Hq // ku.shape[1]
        ahead = n + (0 if after is None else after[b]) - T + torch.arange(T, device=dev)[:, None] - torch.arange(n, device=dev)[None]
        for h in range(Hq):
            g = h // G
            Q = q[b, :, h].double()
            sc, mn = _wide(ksc[:, g]), _wide(kmn[:, g])
            x = Q @ (ku[:, g] * sc + mn).T * scale
            e = (D / 16 + 6) * 2.0 ** -23 * (Q.abs() @ (ku[:, g] * sc.abs() + mn.abs()).T)
            sums = Q.unflatten(-1, (-1, 32)).sum(-1).abs()
            if half:
                e = e + 2.0 ** -13 * Q.abs().amax(1, keepdim=True) * kmn[:, g].abs().sum(-1)[None]
            else:
                e = e + 2.0 ** -17 * (sums @ kmn[:, g].abs().T)
            e = e * scale
            z = x
            if softcap:
                t = torch.tanh(x / softcap)
                z, e = softcap * t, (1 - t * t) * e + softcap * 2.0 ** -21
            if slopes is not None:
                z = z - (slopes[b, h] if slopes.dim() == 2 else slopes[h]).double() * ahead
            seen = ahead >= 0
            zmax = z.abs().masked_fill(~seen, 0).amax(1, keepdim=True)
            e = e + 2.0 ** -21 * (1 + z.abs() + zmax)
            z = z.masked_fill(~seen, -math.inf)
            lse[b, h] = torch.logsumexp(z, 1)
            P = torch.exp(z - lse[b, h][:, None]).masked_fill(~seen, 0)
            e = e.masked_fill(~seen, 0)
            e_l = (P * e).sum(1, keepdim=True) + 2.0 ** -23 * (n / 8 + 16)
            lse_bound[b, h] += (e_l + 2.0 ** -22 * lse[b, h][:, None].abs().nan_to_num(0, 0, 0))[:, 0]
            sc, mn = _wide(vsc[:, g]), _wide(vmn[:, g])
            u = vu[:, g]
            out[b, :, h] = P @ (u * sc + mn)
            if half:
                u, mn = u - 8, mn + 8 * sc
            A = u.abs() * sc.abs()
            M = A + mn.abs()
            bound[b, :, h] += (2.0 ** -11 * (P @ A) + (P * (e + e_l)) @ M + (n / 8 + 16) * 2.0 ** -23 * (P @ M)
                               + n * P.amax(1, keepdim=True) * 2.0 ** -25 * _wide(vsc[:, g].abs().amax(0))[None]
                               + 1.01 * uT * out[b, :, h].abs() + (2.0 ** -25 if half else 2.0 ** -134 + n * 2.0 ** -149))
    return out, bound, lse, lse_bound


def check(got, lse, ref, channels=slice(None)):
    out, bound, want, lse_bound = ref
    got, out, bound = got[..., channels].double(), out[..., channels], bound[..., channels]
    assert torch.isfinite(got).all(), f"not finite at {(~torch.isfinite(got)).nonzero()[:4].tolist()}"
    over = ((got - out).abs() / bound).nan_to_num(0)  # 0 / 0: a sequence without keys
    assert over.max() <= 1, f"{over.max().item():.2f} of the bound at {(over == over.max()).nonzero()[0].tolist()}"
    if lse is not None:
        inf = torch.isinf(want)
        assert torch.equal(torch.isinf(lse), inf)
        off = ((lse.double() - want).masked_fill(inf, 0).abs() / lse_bound).max()
        assert off <= 1, f"lse: {off.item():.2f} of the bound"
