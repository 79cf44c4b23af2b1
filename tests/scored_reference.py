"""Attention with modified scores from its definition, in 64 bits, with elementwise bounds of what the kernels may be off by.

The bounds count roundings.  With u = finfo(dtype).eps / 2 (half a step of the 16-bit type) and A = P |V|:
  out  the weights are rounded for their product (u A), the result once (u |out|);
  dV   likewise: u P^T |dO| + u |dV|;
  dQ   W = P (1 - tanh^2) and dX are rounded (2 u |dX|), delta = sum(dO o out) is formed from the rounded out, off by
       D_i = |dO_i| . u (A_i + |out_i|), so dX is off by 2 u |dX| + W D; times |K| and the scale, and the result's rounding;
  dK   the same, times |Q|.
Rounding to fp16 is off by u of the value or, below its smallest normal number, by half its smallest step, h = 2^-25 (bf16
reaches down to 2^-133): P adds h sum|V| and h sum|dO|, W adds h |dP - delta|, dX adds h.
EXTRA covers the arithmetic in fp32 between the roundings: exp2 to 2^-22 and the quartic to 2^-17, tanh to 2^-22 of a cap of at
most 50 (1e-5; a larger cap C adds C 2^-22), all relative to P.
The scores themselves: products of 16-bit numbers are exact in fp32, their sum over the head dim is taken in steps of 16, each
off by at most 2^-23 of the magnitudes so far: e_x = (D / 16 + 2) 2^-23 scale |q|.|k|.  Behind the cap that is e_y = (1 -
tanh^2) e_x, which moves a weight by e_y and its row's sum by sum(P e_y), relative to P; 1 - tanh^2 itself moves by 2 e_x / cap
of its value (its derivative is -2 tanh (1 - tanh^2) / cap).  Large scores feel this (|q||k| scale = 1e5: e_x = 0.07), ordinary
ones do not (30: 2e-5).
"""
import math

import torch

EXTRA = 2.0 ** -13  # > 2^-17 + 4e-5 + 1e-5 + 2^-22, relative to the sums of magnitudes


def visible(S, causal, cu=None, prefix=None, device="cpu"):
    vis = torch.zeros(S, S, dtype=torch.bool, device=device)
    cu = [0, S] if cu is None else cu
    for d, (a, e) in enumerate(zip(cu, cu[1:])):
        blk = torch.ones(e - a, e - a, dtype=torch.bool, device=device)
        if causal:
            blk = blk.tril()
            if prefix is not None:
                blk[:, :prefix[d]] = True
        vis[a:e, a:e] = blk
    return vis


def reference(q, k, v, dout, vis, *, causal_pos=None, scale=None, softcap=0.0, slopes=None):
    """``vis``: [S, S], or one per batch row.  Returns {name: (value, bound)} for out, lse, dq, dk, dv."""
    B, S, Hq, D = q.shape
    G = Hq // k.shape[2]
    u = torch.finfo(q.dtype).eps / 2
    h2 = torch.finfo(q.dtype).smallest_normal * u  # half the smallest step
    scale = D ** -0.5 if scale is None else scale
    pos = torch.arange(S, device=q.device, dtype=torch.float64)
    names = ("out", "dq", "dk", "dv")
    like = dict(out=q, dq=q, dk=k, dv=k)
    val = {n: torch.zeros(like[n].shape, dtype=torch.float64, device=q.device) for n in names}
    err = {n: torch.zeros_like(val[n]) for n in names}
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        seen = vis[b] if vis.dim() == 3 else vis
        rows, cols = seen.any(1), seen.any(0)
        for h in range(Hq):
            # padding may hold anything; it takes no part
            Q = q[b, :, h].double().masked_fill(~rows[:, None], 0)
            dO = dout[b, :, h].double().masked_fill(~rows[:, None], 0)
            K = k[b, :, h // G].double().masked_fill(~cols[:, None], 0)
            V = v[b, :, h // G].double().masked_fill(~cols[:, None], 0)
            x = Q @ K.T * scale
            jac, jac_off = torch.ones_like(x), torch.zeros_like(x)
            e_x = (D / 16 + 2) * 2.0 ** -23 * (Q.abs() @ K.abs().T) * scale
            if softcap:
                jac_off = 2 * e_x / softcap
                t = torch.tanh(x / softcap)
                x, jac = softcap * t, 1 - t * t
            if slopes is not None:
                sl = slopes[b, h] if slopes.dim() == 2 else slopes[h]
                x = x - sl.double() * (pos[:, None] - pos[None]).abs()
            x = x.masked_fill(~seen, -math.inf)
            lse[b, h] = torch.logsumexp(x, 1)
            P = torch.exp(x - lse[b, h][:, None]).masked_fill(~seen, 0)
            O, A = P @ V, P @ V.abs()
            e_y = jac * e_x + softcap * 2.0 ** -22
            e_p = EXTRA + e_y + (P * e_y).sum(1, keepdim=True)  # of a weight, relative
            E = (P * e_p + h2 * seen) @ V.abs()
            val["out"][b, :, h] = O
            err["out"][b, :, h] = u * A + E + u * O.abs()
            dP = dO @ V.T
            delta = (dO * O).sum(1)
            W = P * jac
            dX = W * (dP - delta[:, None])
            off = (dO.abs() * (u * (A + O.abs()) + E)).sum(1)
            # fp32 relative errors act on both terms of the difference
            dX_err = h2 * seen * (1 + (dP - delta[:, None]).abs()) + 2 * u * dX.abs() + W * off[:, None] + (e_p + jac_off) * W * ((dO.abs() @ V.abs().T) + delta.abs()[:, None])
            val["dq"][b, :, h] = dX @ K * scale
            err["dq"][b, :, h] = dX_err @ K.abs() * scale
            val["dk"][b, :, h // G] += dX.T @ Q * scale
            err["dk"][b, :, h // G] += dX_err.T @ Q.abs() * scale
            val["dv"][b, :, h // G] += P.T @ dO
            err["dv"][b, :, h // G] += (P * (u + e_p) + h2 * seen).T @ dO.abs()
    for n in ("dq", "dk", "dv"):
        err[n] += u * val[n].abs()
    # 1e-6: fp16 results below its smallest normal number are rounded to multiples of 2^-24
    res = {n: (val[n], 1.01 * err[n] + 1e-6) for n in names}
    res["lse"] = (lse, torch.full_like(lse, 1e-3))
    return res


def check(ref, **got):
    for name, g in got.items():
        value, bound = ref[name]
        g = g.double()
        assert g.shape == value.shape, (name, g.shape, value.shape)
        if name == "lse":
            inf = torch.isinf(value)
            assert torch.equal(torch.isinf(g), inf), name
            g, value = g.masked_fill(inf, 0), value.masked_fill(inf, 0)
        assert torch.isfinite(g).all(), f"{name} is not finite at {(~torch.isfinite(g)).nonzero()[:4].tolist()}"
        over = (g - value).abs() / bound
        assert over.max() <= 1, (f"{name}: {over.max().item():.2f} of the bound at "
                                 f"{(over == over.max()).nonzero()[0].tolist()}, {int((over > 1).sum())} values over it")


def inputs(seed, B, S, Hq, Hkv, D, dtype, device, std=1.0):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    mk = lambda H, s: (torch.randn(B, S, H, D, generator=g, device=device) * s).to(dtype)  # noqa: E731
    return mk(Hq, std), mk(Hkv, std), mk(Hkv, 1.0), mk(Hq, 1.0)
