"""How far the gradients are from the definition, in norm, beside what their roundings to 16 bits give when they are made in 64-bit
arithmetic: dX and the results to the type, W = P (1 - tanh^2) to fp16 (for bf16 under 2^15), delta from the rounded out.
What else the kernels do (fp32 sums, exponentials to 2^-17, P within 2^-13) is a sixteenth of the smallest of these for bf16 and
half of it for fp16, so that in quadrature the norms may be 1 + (1/16)^2 / 2 and 1 + (1/2)^2 / 2 of the emulation's: 1.05 and 1.15 are
asked for, sampling included (10^5 values)."""
import math

import pytest
import torch

from scored_reference import inputs
from test_gpu_scored import BF, DEV, HF, _run

pytestmark = pytest.mark.gpu


def _gradients(q, k, v, dout, cap, rounded):
    """dq, dk of one head each, [S, D], in 64 bits; with the roundings or without."""
    S, D = q.shape[1], q.shape[3]
    T = q.dtype
    r16 = (lambda x: x.to(T).double()) if rounded else (lambda x: x)
    up = 2.0 ** 15 if T == BF else 1.0
    w16 = (lambda x: (x * up).half().double() / up) if rounded else (lambda x: x)
    hidden = torch.ones(S, S, dtype=torch.bool, device=DEV).triu(1)
    dq, dk = [], []
    for h in range(q.shape[2]):
        Q, K, V, dO = (t[0, :, h].double() for t in (q, k, v, dout))
        t = torch.tanh(Q @ K.T * D ** -0.5 / cap) if cap else None
        x = cap * t if cap else Q @ K.T * D ** -0.5
        P = torch.softmax(x.masked_fill(hidden, -math.inf), 1)
        W = w16(P * (1 - t * t) if cap else P)
        dX = r16(W * (dO @ V.T - (dO * r16(P @ V)).sum(1, keepdim=True)))
        dq.append(r16(dX @ K * D ** -0.5))
        dk.append(r16(dX.T @ Q * D ** -0.5))
    return torch.stack(dq, 1)[None], torch.stack(dk, 1)[None]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_gradients(D, dt, cap):
    q, k, v, dout = inputs(70, 1, 1000, 2, 2, D, dt, DEV, std=1.3)
    got = _run(q, k, v, dout, causal=True, softcap=cap)
    exact, coarse = (_gradients(q, k, v, dout, cap, r) for r in (False, True))
    for name, e, c in zip(("dq", "dk"), exact, coarse):
        off, expected = (got[name].double() - e).norm() / e.norm(), (c - e).norm() / e.norm()
        assert off <= (1.05 if dt == BF else 1.15) * expected, f"{name}: {off.item():.2e}, the roundings alone {expected.item():.2e}"


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kind", ["plain", "bias"])
def test_scores_that_lse_cannot_hold(D, kind):
    """Scores of 10^7 to 5 * 10^8: lse keeps no more than their leading digits, so weights come out too large; what flows back stays
    finite.  (Below 2^29 in log2 units neighbouring numbers are 32 apart: maximum and lse are off by 16 each, a weight by 2^32, and
    under 2^15 that is still far inside fp32 and bf16.  From 2^32 on they are 512 apart, and the forward pass itself, plain or not,
    overflows in exp2: there is nothing to hold.)"""
    q, k, v, dout = inputs(71, 1, 300, 2, 2, D, BF, DEV)
    slopes = torch.full((2,), 0.1, device=DEV) if kind == "bias" else None
    for std in (2.0 ** 12, 2.0 ** 13):
        got = _run(q * std * (64 / D) ** 0.25, k * std * (64 / D) ** 0.25, v, dout, causal=True, alibi_slopes=slopes)
        assert all(torch.isfinite(got[n]).all() for n in got)
