"""The operators beside plain ring attention, as they are timed: attention with modified scores (tanh cap, distance bias,
document and prefix masks; forward, or forward and backward) and the K/V cache held in 4 bits (append with read-back,
attention of new tokens over it).

``run`` computes a case in its plain form, with elementary operations in fp32, or through the package (``own``).
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_PAGE = 64    # tokens per cache page
_GROUP = 32   # channels that share a scale and a minimum


def _attn(name, B, S, Hq, Hkv, D, *, dtype="bf16", causal=True, backward=True, softcap=0.0, alibi=False, doc_mean=0,
          prefix=0.0, tail=0.0, layout=1):
    c = dict(kind="attn", B=B, S=S, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, causal=causal, backward=backward, softcap=softcap,
             alibi=alibi, doc_mean=doc_mean, prefix=prefix, tail=tail, layout=layout)
    return c if name is None else dict(c, name=name)


def _decode(name, B, T, Hq, Hkv, D, min_len, max_len, *, dtype="bf16", softcap=0.0, alibi=False, layout=1):
    c = dict(kind="decode", B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, min_len=min_len, max_len=max_len, dtype=dtype,
             softcap=softcap, alibi=alibi, layout=layout)
    return c if name is None else dict(c, name=name)


def _append(name, B, T, Hkv, D, max_len, *, dtype="bf16", layout=1):
    c = dict(kind="append", B=B, T=T, Hkv=Hkv, D=D, max_len=max_len, dtype=dtype, layout=layout)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # The smallest training call: 256 tokens, 8 heads of 64, capped scores.  Launches and gaps.
        _attn("train_s256_d64_cap", 1, 256, 8, 8, 64, softcap=30.0),
        # A prompt whose first part is seen by all of it (prefix mask), forward only, ragged length, GQA.
        _attn("infer_s1000_prefix", 1, 1000, 32, 8, 128, backward=False, prefix=0.4),
        # Training with a distance bias instead of position embeddings, heads of 64, fp16.
        _attn("train_s4096_alibi", 1, 4096, 16, 16, 64, dtype="fp16", alibi=True),
        # Pretraining on packed documents: one long row, documents of some two thousand tokens, GQA.
        _attn("train_s16384_docs", 1, 16384, 32, 8, 128, doc_mean=2048),
        # Fine-tuning on packed conversations whose prompts are seen whole: everything at once, ragged rows with padding at
        # the end, a head dim that needs padding.
        _attn("train_s2100_d96_all", 2, 2100, 16, 4, 96, dtype="fp16", softcap=20.0, alibi=True, doc_mean=400, prefix=0.3,
              tail=0.1),
        # The wide heads that capped scores come with.
        _attn("train_s4096_d256_cap", 1, 4096, 16, 8, 256, softcap=50.0),
        # One user, a short context: latency.
        _decode("decode_b1_s1000", 1, 1, 32, 8, 128, 1000, 1000),
        # A full serving batch of mixed lengths, capped scores.
        _decode("decode_b64_cap", 64, 1, 32, 8, 128, 100, 8192, softcap=30.0),
        # Two users with very long contexts: the work of few rows has to be split along the cache.
        _decode("decode_b2_s131072", 2, 1, 32, 8, 128, 100000, 131072, alibi=True),
        # Four drafted tokens per sequence are verified at once; no head groups, heads of 64, fp16.
        _decode("verify_t4_b16_d64", 16, 4, 16, 16, 64, 300, 5000, dtype="fp16"),
        # A prompt goes into the cache and is read back for the next part of it.
        _append("append_s8192", 1, 8192, 8, 128, 8192),
        # One new token for each sequence of a serving batch.
        _append("append_b64_t1", 64, 1, 8, 128, 8192),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype, layout = rng.choice(["bf16", "bf16", "fp16"]), rng.randrange(1, 1 << 20)
    kind = rng.random()
    while True:
        Hkv = rng.choice([1, 2, 4, 8, 16])
        Hq = Hkv * rng.choice([1, 1, 2, 4, 8])
        if Hq > 32:
            continue
        if kind < 0.55:
            S = spread(64, 16384)
            if rng.random() < 0.5:
                S = max(64, S // 64 * 64)
            docs = rng.random() < 0.6
            c = _attn(None, rng.choice([1, 1, 1, 2, 3]), S, Hq, Hkv, rng.choice([64, 64, 128, 128, 256, 96, 160, 32]),
                      dtype=dtype, causal=rng.random() < 0.8, backward=rng.random() < 0.7,
                      softcap=rng.choice([0.0, 0.0, 20.0, 30.0, 50.0]), alibi=rng.random() < 0.35,
                      doc_mean=spread(16, max(17, S)) if docs else 0, prefix=rng.choice([0.0, 0.0, 0.3, 0.6]),
                      tail=rng.choice([0.0, 0.0, 0.1]) if docs else 0.0, layout=layout)
            if not c["causal"]:
                c["prefix"] = 0.0  # every key of the document is seen anyway
            if c["B"] * Hq * S * S <= 32 * 16384 ** 2 and work(c)["flops"] <= _largest("attn"):
                return c
        elif kind < 0.85:
            hi = spread(16, 131072)
            c = _decode(None, spread(1, 64), rng.choice([1, 1, 1, 2, 4, 5, 8]), Hq, Hkv, rng.choice([64, 128, 128, 256, 96]),
                        rng.choice([0, 1, hi // 8, hi]), hi, dtype=dtype, softcap=rng.choice([0.0, 0.0, 30.0]),
                        alibi=rng.random() < 0.3, layout=layout)
            if c["min_len"] > hi:
                continue
            if c["B"] * hi * Hkv * c["D"] <= 2 * 131072 * 8 * 128 and work(c)["bytes"] <= _largest("decode"):
                return c
        else:
            T = rng.choice([1, 1, 3, spread(2, 8192)])
            c = _append(None, spread(1, 64), T, Hkv, rng.choice([64, 128, 128, 256, 96]), max(T, spread(16, 8192)),
                        dtype=dtype, layout=layout)
            if work(c)["bytes"] <= _largest("append") and c["B"] * c["max_len"] * Hkv * c["D"] <= 64 * 8192 * 8 * 128:
                return c


def _largest(kind):
    key = "flops" if kind == "attn" else "bytes"
    return max(work(c)[key] for c in listed() if c["kind"] == kind)


# ---------------------------------------------------------------------------------------------------------------------
# Layout of a case: what belongs to its sizes and not to the values of its inputs
# ---------------------------------------------------------------------------------------------------------------------

def _documents(case):
    """Per batch row the document borders (the last one is where the padding starts) and the lengths of their prefixes."""
    rng = random.Random(case["layout"])
    S, rows = case["S"], []
    for _ in range(case["B"]):
        end = S - int(S * case["tail"] * rng.random())
        cu = [0]
        while cu[-1] < end:
            n = min(end - cu[-1], max(1, int(rng.expovariate(1 / case["doc_mean"])))) if case["doc_mean"] else end
            cu.append(cu[-1] + n)
        rows.append((cu, [int(case["prefix"] * (b - a)) for a, b in zip(cu, cu[1:])]))
    n = max(len(cu) for cu, _ in rows)
    return [(cu + [cu[-1]] * (n - len(cu)), pre + [0] * (n - 1 - len(pre))) for cu, pre in rows]


def _lengths(case):
    rng = random.Random(case["layout"])
    return [rng.randint(case["min_len"], case["max_len"]) for _ in range(case["B"])]


def _pages(lengths, seed):
    """A block table whose pages lie scattered in the pool, and the number of pages of the pool."""
    counts = [max(1, -(-n // _PAGE)) for n in lengths]
    order = list(range(sum(counts)))
    random.Random(seed).shuffle(order)
    table, at = [], 0
    for c in counts:
        table.append(order[at:at + c] + [0] * (max(counts) - c))
        at += c
    return table, len(order)


def work(case):
    B, D = case["B"], case["D"]
    if case["kind"] == "attn":
        S, Hq, Hkv = case["S"], case["Hq"], case["Hkv"]
        pairs = 0
        for cu, pre in _documents(case):
            for a, b, p in zip(cu, cu[1:], pre):
                n = b - a
                pairs += n * n if not case["causal"] else n * (n + 1) // 2 + p * (p - 1) // 2
        nbytes = 2 * (2 * B * S * Hq * D + 2 * B * S * Hkv * D)
        if case["backward"]:
            nbytes += 2 * (2 * B * S * Hq * D + 2 * B * S * Hkv * D)
        return {"bytes": nbytes, "flops": (14 if case["backward"] else 4) * D * Hq * pairs}
    kv_row = 2 * (D // 2 + D // _GROUP * 4)  # bytes of one token and head in the cache, K and V
    Hkv = case["Hkv"]
    if case["kind"] == "decode":
        keys = sum(_lengths(case))
        return {"bytes": keys * Hkv * kv_row + 2 * 2 * B * case["T"] * case["Hq"] * D,
                "flops": 4 * D * case["Hq"] * case["T"] * keys}
    rows = B * case["T"] * Hkv
    return {"bytes": rows * (2 * 2 * D + kv_row) + rows * (kv_row + 2 * 2 * D), "flops": rows * 2 * D * 8}


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev, dt = torch.device("cuda"), _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * std).to(dt)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    st = {"case": case}
    B, D = case["B"], case["D"]
    if case["kind"] == "attn":
        S, Hq, Hkv = case["S"], case["Hq"], case["Hkv"]
        # with capped scores queries and keys grow until the cap holds them: scores of several units, some near the cap
        std = 1.8 if case["softcap"] else 1.0
        for name, H, s in (("q", Hq, std), ("k", Hkv, std), ("v", Hkv, 1.0)):
            st[name] = normal(B, S, H, D, std=s).requires_grad_(case["backward"])
        if case["backward"]:
            st["dout"] = normal(B, S, Hq, D)
        docs = _documents(case)
        st["cu"], st["prefix"] = ints([cu for cu, _ in docs]), ints([pre for _, pre in docs])
        if own and (case["doc_mean"] or case["prefix"]):
            import opt_ring_flash_attn_b200 as rfa

            st["mask"] = rfa.document_mask(st["cu"], S, prefix_lens=st["prefix"], causal=case["causal"])
    elif case["kind"] == "decode":
        lens = _lengths(case)
        table, n = _pages(lens, seed)
        st["table"], st["lens"] = ints(table), ints(lens)
        st["q"] = normal(B, case["T"], case["Hq"], D)
        st["codes"], st["meta"] = _pack(*_quantize(normal(n, case["Hkv"], 2, _PAGE, D)))
    else:
        rng = random.Random(seed)
        starts = [rng.randint(0, case["max_len"] - case["T"]) for _ in range(B)]
        table, n = _pages([a + case["T"] for a in starts], seed)
        st["table"], st["starts"] = ints(table), ints(starts)
        st["k"], st["v"] = normal(B, case["T"], case["Hkv"], D), normal(B, case["T"], case["Hkv"], D)
        st["codes"] = torch.zeros(n, case["Hkv"], 2, _PAGE, D // 2, dtype=torch.uint8, device=dev)
        st["meta"] = torch.zeros(n, case["Hkv"], 2, _PAGE, D // _GROUP, 2, dtype=dt, device=dev)
    if case.get("alibi"):
        H = case["Hq"]
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device=dev)
    if own and case["kind"] != "attn":
        import opt_ring_flash_attn_b200 as rfa

        st["cache"] = rfa.KV4Cache(st["codes"], st["meta"])
    return st


# ---------------------------------------------------------------------------------------------------------------------
# The 4-bit format in elementary operations
# ---------------------------------------------------------------------------------------------------------------------

def _quantize(x):
    """[..., D] -> codes [..., D] (0..15) and (scale, minimum) [..., D / 32, 2] in x's type."""
    g = x.unflatten(-1, (-1, _GROUP)).float()
    lo, hi = g.amin(-1), g.amax(-1)
    sc = ((hi - lo) / 15).to(x.dtype)
    # the quotient decides at borders between two codes: correctly rounded, in 64 bits
    t = (g.double() - lo[..., None].double()) / sc[..., None].double()
    u = torch.where(sc[..., None] > 0, t.round().clamp(0, 15), torch.zeros_like(t)).to(torch.uint8)
    return u.flatten(-2), torch.stack([sc, lo.to(x.dtype)], -1)


def _pack(u, meta):
    """Codes [n, H, 2, 64, D] (K, V) -> bytes [n, H, 2, 64, D / 2].  Inside a row, K holds the words of 8 channels
    [32 g + 8 c, + 8) at word c * (D / 32) + g, V the half words of 4 channels [32 g + 4 c, + 4) at c * (D / 32) + g; the
    first channel is in the lowest bits."""
    k, v = u[:, :, 0], u[:, :, 1]
    k = k.unflatten(-1, (-1, 4, 8)).transpose(-3, -2).flatten(-3)
    v = v.unflatten(-1, (-1, 8, 4)).transpose(-3, -2).flatten(-3)
    s = torch.stack([k, v], 2)
    return (s[..., 0::2] | (s[..., 1::2] << 4)).contiguous(), meta.contiguous()


def _unpack(codes, meta):
    """Bytes and (scale, minimum) of pages -> values [n, H, 2, 64, D] in fp32."""
    s = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    ng = s.shape[-1] // _GROUP
    k = s[:, :, 0].unflatten(-1, (4, ng, 8)).transpose(-3, -2).flatten(-3)
    v = s[:, :, 1].unflatten(-1, (8, ng, 4)).transpose(-3, -2).flatten(-3)
    u = torch.stack([k, v], 2).unflatten(-1, (ng, _GROUP)).float()
    m = meta.float()
    return (u * m[..., 0:1] + m[..., 1:2]).flatten(-2)


# ---------------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attn": _own_attn, "decode": _own_decode, "append": _own_append}[kind](state)
    return {"attn": _plain_attn, "decode": _plain_decode, "append": _plain_append}[kind](state)


def _own_attn(st):
    import opt_ring_flash_attn_b200 as rfa

    c = st["case"]
    kw = dict(causal=c["causal"], softcap=c["softcap"], alibi_slopes=st.get("slopes"), mask=st.get("mask"))
    q, k, v = st["q"], st["k"], st["v"]
    if not c["backward"]:
        with torch.no_grad():
            return rfa.scored_flash_attn(q, k, v, **kw)
    out = rfa.scored_flash_attn(q, k, v, **kw)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), st["dout"]))


def _own_decode(st):
    import opt_ring_flash_attn_b200 as rfa

    c = st["case"]
    return rfa.kv4_attn(st["q"], st["cache"], st["table"], st["lens"], softcap=c["softcap"], alibi_slopes=st.get("slopes"))


def _own_append(st):
    import opt_ring_flash_attn_b200 as rfa

    rfa.kv4_append(st["cache"], st["k"], st["v"], st["table"], st["starts"])
    return rfa.kv4_gather(st["cache"], st["table"], st["starts"], st["case"]["T"])


def _visible(case, cu, prefix):
    """[S, S] truth values: query i (row) sees key j."""
    S = case["S"]
    pos = torch.arange(S, device=cu.device)
    doc = torch.searchsorted(cu[1:].long().contiguous(), pos, right=True)  # number of documents that end at or before pos
    real = pos < cu[-1]
    doc = doc.clamp(max=len(cu) - 2)
    vis = (doc[:, None] == doc[None]) & real[:, None] & real[None]
    if case["causal"]:
        vis &= (pos[None] <= pos[:, None]) | (pos < cu[doc] + prefix[doc])[None]
    return vis


def _plain_attn(st):
    c = st["case"]
    q, k, v = st["q"].detach(), st["k"].detach(), st["v"].detach()
    B, S, Hq, D = q.shape
    G, cap, scale = Hq // c["Hkv"], c["softcap"], D ** -0.5
    pos = torch.arange(S, device=q.device, dtype=torch.float32)
    out = torch.empty(B, S, Hq, D, device=q.device)
    if c["backward"]:
        dq = torch.empty_like(out)
        dk, dv = torch.zeros_like(k, dtype=torch.float32), torch.zeros_like(v, dtype=torch.float32)
    for b in range(B):
        hidden = ~_visible(c, st["cu"][b], st["prefix"][b])
        empty = hidden.all(1)[:, None]
        for h in range(Hq):
            qh, kh, vh = q[b, :, h].float(), k[b, :, h // G].float(), v[b, :, h // G].float()
            z = (qh @ kh.T) * scale
            if cap:
                t = torch.tanh(z / cap)
                z = t * cap
            if "slopes" in st:
                z = z - st["slopes"][h] * (pos[:, None] - pos[None]).abs()
            z.masked_fill_(hidden, float("-inf"))
            p = torch.exp(z - z.amax(1, keepdim=True))
            p = (p / p.sum(1, keepdim=True)).masked_fill_(empty, 0.0)
            del z
            o = p @ vh
            out[b, :, h] = o
            if c["backward"]:
                do = st["dout"][b, :, h].float()
                dv[b, :, h // G] += p.T @ do
                ds = p * (do @ vh.T - (o * do).sum(1, keepdim=True))
                if cap:
                    ds = ds * (1 - t * t)
                dq[b, :, h] = (ds @ kh) * scale
                dk[b, :, h // G] += (ds.T @ qh) * scale
    if not c["backward"]:
        return out.to(q.dtype)
    return tuple(x.to(q.dtype) for x in (out, dq, dk, dv))


def _plain_decode(st):
    c = st["case"]
    q, lens = st["q"].float(), _lengths(c)
    B, T, Hq, D = q.shape
    G, cap = Hq // c["Hkv"], c["softcap"]
    out = torch.zeros_like(q)
    for b in range(B):
        n = lens[b]
        if n == 0:
            continue
        pages = st["table"][b, :-(-n // _PAGE)].long()
        kv = _unpack(st["codes"][pages], st["meta"][pages])                       # [pages, Hkv, 2, 64, D]
        k, v = (kv[:, :, i].transpose(0, 1).flatten(1, 2)[:, :n] for i in (0, 1))  # [Hkv, n, D]
        qb = q[b].transpose(0, 1).unflatten(0, (c["Hkv"], G))                     # [Hkv, G, T, D]
        z = (qb @ k[:, None].transpose(-1, -2)) * D ** -0.5
        if cap:
            z = torch.tanh(z / cap) * cap
        at = n - T + torch.arange(T, device=q.device)[:, None] - torch.arange(n, device=q.device)[None]
        if "slopes" in st:
            z = z - st["slopes"].view(c["Hkv"], G, 1, 1) * at.float()
        z = z.masked_fill(at < 0, float("-inf"))
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).masked_fill((at < 0).all(1)[:, None], 0.0)
        out[b] = (p @ v[:, None]).flatten(0, 1).transpose(0, 1)
    return out.to(st["q"].dtype)


def _plain_append(st):
    c = st["case"]
    B, T, Hkv, D = st["k"].shape
    x = torch.stack([st["k"], st["v"]], 3)                                        # [B, T, H, 2, D]
    codes, meta = _pack(*(y.permute(0, 2, 3, 1, 4).flatten(0, 1)[:, None] if y.dim() == 5 else
                          y.permute(0, 2, 3, 1, 4, 5).flatten(0, 1)[:, None] for y in _quantize(x)))
    at = st["starts"][:, None].long() + torch.arange(T, device=x.device)
    page, row = st["table"].long().gather(1, at // _PAGE), at % _PAGE              # [B, T]
    codes = codes.view(B, Hkv, 2, T, -1).permute(0, 3, 1, 2, 4)
    meta = meta.view(B, Hkv, 2, T, D // _GROUP, 2).permute(0, 3, 1, 2, 4, 5)
    st["codes"][page, :, :, row] = codes
    st["meta"][page, :, :, row] = meta
    rows = _unpack(st["codes"][page, :, :, row].permute(0, 2, 3, 1, 4).flatten(0, 1)[:, None],
                   st["meta"][page, :, :, row].permute(0, 2, 3, 1, 4, 5).flatten(0, 1)[:, None])
    rows = rows.view(B, Hkv, 2, T, D).permute(2, 0, 3, 1, 4).to(x.dtype)
    return rows[0].contiguous(), rows[1].contiguous()


# ---------------------------------------------------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    with torch.enable_grad():
        return {"attn": _exact_attn, "decode": _exact_decode, "append": _exact_append}[case["kind"]](case, st)


def _log_weights(scores, distance, case, slope):
    """Scores in 64 bits, capped and biased."""
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    return scores if slope is None else scores - slope.double() * distance.double()


def _exact_attn(case, st):
    B, S, Hq, Hkv, D = (case[x] for x in ("B", "S", "Hq", "Hkv", "D"))
    if B * Hq * S * S > 1.2e10 or S > 20000:
        return None
    dev = st["q"].device
    q, k, v = (st[x].detach().double() for x in "qkv")
    i = torch.arange(S, device=dev)
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b, (cu, pre) in enumerate(_documents(case)):
        for a, e, p in zip(cu, cu[1:], pre):  # the documents do not see each other
            if e == a:
                continue
            pos = i[a:e]
            dist = (pos[:, None] - pos[None]).abs()
            seen = torch.ones(e - a, e - a, dtype=torch.bool, device=dev)
            if case["causal"]:
                seen = torch.tril(seen)
                seen[:, :p] = True
            for h in range(Hq):
                x, y, w = (t[b, a:e, g].clone().requires_grad_(case["backward"])
                           for t, g in ((q, h), (k, h // (Hq // Hkv)), (v, h // (Hq // Hkv))))
                z = _log_weights(x @ y.T / math.sqrt(D), dist, case, st["slopes"][h] if "slopes" in st else None)
                o = torch.softmax(z.masked_fill(~seen, -math.inf), dim=1) @ w
                out[b, a:e, h] = o.detach()
                if case["backward"]:
                    gx, gy, gw = torch.autograd.grad(o, (x, y, w), st["dout"][b, a:e, h].double())
                    dq[b, a:e, h] = gx
                    dk[b, a:e, h // (Hq // Hkv)] += gy
                    dv[b, a:e, h // (Hq // Hkv)] += gw
    return (out, dq, dk, dv) if case["backward"] else out


def _nibbles(row):
    """Codes of the bytes of one row, low bits first, as a [.., 2 n] tensor."""
    return torch.cat([(row & 15)[..., None], (row // 16)[..., None]], dim=-1).reshape(*row.shape[:-1], -1)


def _values(codes, meta):
    """K and V [H, tokens, D] in 64 bits of the bytes [H, 2, tokens, D / 2] and their scales: channel by channel."""
    D = codes.shape[-1] * 2
    ng = D // _GROUP
    ch = torch.arange(D, device=codes.device)
    g, r = ch // _GROUP, ch % _GROUP
    k_at = (r // 8 * ng + g) * 8 + r % 8
    v_at = (r // 4 * ng + g) * 4 + r % 4
    u, m = _nibbles(codes).double(), meta.double()
    return tuple(u[:, i][..., at] * m[:, i][..., g, 0] + m[:, i][..., g, 1] for i, at in ((0, k_at), (1, v_at)))


def _exact_decode(case, st):
    if work(case)["bytes"] > 6e8:
        return None
    T, Hq, Hkv, D = (case[x] for x in ("T", "Hq", "Hkv", "D"))
    out = torch.zeros_like(st["q"], dtype=torch.float64)
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        pages = st["table"][b][:(n + _PAGE - 1) // _PAGE].long()
        k, v = _values(st["codes"][pages].permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n],
                       st["meta"][pages].permute(1, 2, 0, 3, 4, 5).flatten(2, 3)[:, :, :n])
        for t in range(T):
            last = n - T + t  # the position of this token
            if last < 0:
                continue
            dist = last - torch.arange(last + 1, device=k.device)
            for h in range(Hq):
                x = st["q"][b, t, h].double()
                z = _log_weights(k[h // (Hq // Hkv), :last + 1] @ x / math.sqrt(D), dist, case,
                                 st["slopes"][h] if "slopes" in st else None)
                out[b, t, h] = torch.softmax(z, 0) @ v[h // (Hq // Hkv), :last + 1]
    return out


def _exact_append(case, st):
    res = []
    for x in (st["k"], st["v"]):
        g = x.double().reshape(*x.shape[:-1], x.shape[-1] // _GROUP, _GROUP)
        lo = g.min(-1, keepdim=True).values
        sc = ((g.max(-1, keepdim=True).values - lo) / 15).to(x.dtype).double()
        u = torch.round((g - lo) / torch.where(sc > 0, sc, torch.ones_like(sc))) * (sc > 0)
        res.append((u.clamp(0, 15) * sc + lo).reshape(x.shape))
    return tuple(res)
