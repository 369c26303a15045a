"""Serving from a paged KV cache: the operators it is made of, and the cases they are timed on.

* ``rope``    rotary positions of query or key heads: half or interleaved pairs,
  all of a head or its first dims, cos/sin tables of any scaling, either direction
  (the inverse rotation is the gradient of the forward one).
* ``append``  new keys and values into the pages of their segments, the keys (and
  the queries that will read them) rotated on the way.
* ``attn``    attention of the new tokens of every segment -- one each, or chunks of
  any lengths -- over the segment's pages, causal, with the score cap, the distance
  bias and the window, document and prefix masks that models put on it.

A page holds ``page`` tokens of every kv head, ``[n_pages, Hkv, page, hd]``; a
segment's row of ``table`` names its pages in order.  New token t of segment b sits
at position ``pos[b] + t``; the tokens of ragged segments lie one after the other,
``cu[b]`` to ``cu[b + 1]``.  Pages that no segment owns, and page rows behind a
segment's last token, hold leftovers of other segments.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases -------------------------------------------------------------------

def _rope(name, T, H, hd, rot, dtype, interleaved=False, inverse=False, scaled=1.0, far=2048):
    """far: positions run up to this; scaled: context extension of the table."""
    return {"name": name, "op": "rope", "T": T, "H": H, "hd": hd, "rot": rot, "dtype": dtype,
            "interleaved": interleaved, "inverse": inverse, "scaled": scaled, "far": far}


def _append(name, B, W, ctx, H, Hkv, hd, page, dtype, ragged=False, rot=16, interleaved=False):
    return {"name": name, "op": "append", "B": B, "W": W, "ctx": ctx, "H": H, "Hkv": Hkv, "hd": hd, "page": page,
            "dtype": dtype, "ragged": ragged, "rot": rot, "interleaved": interleaved}


def _attn(name, B, W, ctx, H, Hkv, hd, page, dtype, ragged=False, softcap=0.0, slopes=False, window=0, docs=0, prefix=0):
    """docs: typical document length inside a segment (0: one document)."""
    return {"name": name, "op": "attn", "B": B, "W": W, "ctx": ctx, "H": H, "Hkv": Hkv, "hd": hd, "page": page,
            "dtype": dtype, "ragged": ragged, "softcap": softcap, "slopes": slopes, "window": window, "docs": docs,
            "prefix": prefix}


def listed():
    return [
        # one decode row of 64 segments: 8 heads of 64 dims, 16 of them rotated
        _rope("rope_rows", 64, 8, 64, 16, "bf16"),
        # chunk scoring of a model that rotates whole heads in interleaved pairs,
        # its table stretched four times for long contexts
        _rope("rope_chunk_scaled", 65536, 16, 128, 128, "fp16", interleaved=True, scaled=4.0, far=131072),
        # the gradient of a rotation in the fp32 compute mode, an odd number of rows
        _rope("rope_inverse_fp32", 9973, 8, 64, 16, "fp32", inverse=True),
        # a decode step of 64 segments puts its row into the cache
        _append("append_rows", 64, 1, 2047, 8, 8, 64, 64, "bf16"),
        # a ragged prefill of 16 grouped-query segments, from nothing to 2048 tokens each
        _append("append_chunks", 16, 2048, 1000, 8, 4, 64, 64, "bf16", ragged=True),
        # one segment decoding: latency
        _attn("decode_b1", 1, 1, 2047, 8, 8, 64, 64, "bf16"),
        # the decode batch of the benchmark
        _attn("decode_b64", 64, 1, 2047, 8, 8, 64, 64, "bf16"),
        # 256 segments at context 4096: the largest cache read
        _attn("decode_b256", 256, 1, 4095, 8, 8, 64, 64, "bf16"),
        # one encode window of the student at the end of its 32768-token buffer
        _attn("window_b1_long", 1, 64, 32704, 8, 4, 64, 64, "bf16"),
        # chunk scoring: whole 2048-token chunks from position 0
        _attn("prefill_b16", 16, 2048, 0, 8, 8, 64, 64, "bf16"),
        # a mixed batch (drafts of up to 9 tokens, idle segments) of a grouped-query
        # model with sliding window, score cap and distance bias, small pages
        _attn("mixed_bias_gqa", 48, 9, 5000, 16, 2, 128, 16, "fp16", ragged=True, softcap=30.0, slopes=True, window=2048),
        # packed documents behind a shared prefix, ragged chunks, capped scores
        _attn("packed_docs", 8, 1500, 600, 8, 8, 128, 32, "bf16", ragged=True, softcap=50.0, docs=300, prefix=100),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attn", "attn", "attn"])
    hd = rng.choice([64, 64, 128])
    if op == "rope":
        H = rng.choice([1, 2, 4, 8, 16, 5])
        return {k: v for k, v in _rope("", _log(rng, 1, (1 << 27) // (H * hd)), H, hd, rng.choice([16, hd // 2, hd, 32, 24]),
                                       rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.5, rng.random() < 0.3,
                                       rng.choice([1.0, 2.0, 8.0]), _log(rng, 64, 131072)).items() if k != "name"}
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * rng.choice([1, 1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        B = _log(rng, 1, 256)
        W = 1 if rng.random() < 0.4 else _log(rng, 2, 32768 // B)
        ctx = _log(rng, 1, min(4096, 65536 // B))
        return {k: v for k, v in _append("", B, W, ctx, H, Hkv, hd, page, rng.choice(["bf16", "fp16", "fp32"]),
                                         W > 1 and rng.random() < 0.6, rng.choice([0, 16, hd // 2, hd, 24]),
                                         rng.random() < 0.4).items() if k != "name"}
    kind = rng.choice(["decode", "decode", "window", "prefill"])
    if kind == "decode":
        B, W = _log(rng, 1, 256), 1
        ctx = _log(rng, 1, min(32768, (256 * 4096 * 8 * 64) // (B * Hkv * hd)))
    elif kind == "window":
        B, W = _log(rng, 1, 64), _log(rng, 2, 128)
        ctx = _log(rng, 1, min(16384, max(1, (64 * 4096 * 8 * 64) // (B * Hkv * hd))))
        W = max(2, min(W, (1 << 28) // (B * H * ctx)))
    else:
        W = _log(rng, 100, min(2048, math.isqrt((4 * 2048 * 2048 * 8 * 64) // (H * hd))))
        B = _log(rng, 1, max(1, min(256, (4 * 2048 * 2048 * 8 * 64) // (W * W * H * hd))))
        ctx = rng.choice([0, _log(rng, 1, 512)])
    biased = rng.random() < 0.4
    return {k: v for k, v in _attn("", B, W, ctx, H, Hkv, hd, page, rng.choice(["bf16", "bf16", "fp16"]),
                                   W > 1 and rng.random() < 0.6,
                                   rng.choice([15.0, 30.0, 50.0]) if biased else 0.0, biased and rng.random() < 0.6,
                                   rng.choice([0, 0, _log(rng, 8, 2048)]),
                                   _log(rng, 20, 1000) if W > 1 and rng.random() < 0.3 else 0,
                                   _log(rng, 1, 200) if W > 1 and rng.random() < 0.3 else 0).items() if k != "name"}


# ---- what a case's program knows on the host -----------------------------------

def _lens(case):
    """New tokens and context of every segment; idle segments among ragged ones."""
    B, W, ctx = case["B"], case["W"], case["ctx"]
    if not case["ragged"]:
        return np.full(B, W), np.full(B, ctx)
    r = np.random.RandomState(B * 7919 + W * 31 + ctx)
    n = r.randint(0, W + 1, B)
    n[r.randint(B)] = W
    c = r.randint(0, ctx + 1, B)
    c[r.randint(B)] = ctx
    return n, c


def _ranges(case):
    """First and last visible key (half open) of every new token, the token's segment and
    position, its document's start and the segments' prefix lengths (None: not used)."""
    n, c = _lens(case)
    seg = np.repeat(np.arange(case["B"]), n)
    p = np.concatenate([np.arange(a, a + m) for a, m in zip(c, n)]) if seg.size else np.zeros(0, np.int64)
    lo, hi = np.zeros_like(p), p + 1
    starts = prefix = None
    if case["docs"]:  # documents begin at multiples of a length of the segment's own; every 97th token
        r = np.random.RandomState(case["docs"])  # is padding between two documents and sees nothing
        size = r.randint(max(2, case["docs"] // 2), case["docs"] * 2, case["B"])[seg]
        starts = p // size * size
        starts[np.arange(p.size) % 97 == 41] = 1 << 20
        lo = np.maximum(lo, starts)
    if case["window"]:
        lo = np.maximum(lo, p - case["window"] + 1)
    if case["prefix"]:
        prefix = np.random.RandomState(case["prefix"]).randint(0, case["prefix"] * 2 + 1, case["B"])
        hi = np.maximum(hi, np.minimum(prefix, c + n)[seg])
    return seg, p, lo, np.maximum(hi, lo), starts, prefix


def work(case):
    size = DTYPE[case["dtype"]].itemsize
    if case["op"] == "rope":
        n = case["T"] * case["H"]
        tab = min(case["T"], case["far"]) * case["rot"] * 4
        return {"bytes": 2 * n * case["hd"] * size + tab + 4 * case["T"], "flops": 3 * n * case["rot"]}
    H, Hkv, hd = case["H"], case["Hkv"], case["hd"]
    if case["op"] == "append":
        n, c = _lens(case)
        T = int(n.sum())
        return {"bytes": T * (2 * H + 4 * Hkv) * hd * size + T * case["rot"] * 4 + 4 * case["B"],
                "flops": 3 * T * (H + Hkv) * case["rot"]}
    seg, p, lo, hi, _, _ = _ranges(case)
    keys = 0
    for b in np.unique(seg):
        m = (seg == b) & (hi > lo)
        if m.any():
            keys += int(hi[m].max() - lo[m].min())
    return {"bytes": 2 * keys * Hkv * hd * size + 2 * len(seg) * H * hd * size, "flops": 4 * int((hi - lo).sum()) * H * hd}


# ---- inputs ------------------------------------------------------------------

def _tables(rows, rot, scaled):
    """cos/sin [rows, rot / 2]: base 10000, stretched as the base of a longer context."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot
    base = 1e4 * scaled ** (rot / max(1, rot - 2))
    a = torch.outer(torch.arange(rows, dtype=torch.float64, device=DEV), base ** -i)
    return a.cos().float(), a.sin().float()


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    dt = DTYPE[case["dtype"]]

    def rows(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dt)

    st = dict(case)
    if case["op"] == "rope":
        T, H, hd = case["T"], case["H"], case["hd"]
        # heads as they come out of a joint projection: each row has as many others behind it
        st["x"] = rows(T, 2 * H, hd)[:, :H]
        st["cos"], st["sin"] = _tables(case["far"], case["rot"], case["scaled"])
        first = torch.randint(0, case["far"], (1,), generator=g, device=DEV)
        st["pos"] = ((first + torch.arange(T, device=DEV)) % case["far"]).to(torch.int32)
        return st
    n, c = _lens(case)
    B, H, Hkv, hd, page = case["B"], case["H"], case["Hkv"], case["hd"], case["page"]
    T, S = int(n.sum()), int((n + c).max())
    width = -(-S // page)
    held = -(-(n + c) // page)
    total = int(held.sum()) + 3  # a few that nobody owns
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = np.full((B, width), -1, np.int64)
    table[np.arange(width)[None] < held[:, None]] = np.arange(int(held.sum()))
    table = _dev(table)
    st["table"] = torch.where(table >= 0, perm[table.clamp_min(0).long()], table)
    st["pos"] = _dev(c)
    st["cu"] = _dev(np.concatenate([[0], np.cumsum(n)])) if case["ragged"] else None
    st["max_len"] = S
    st["k_cache"] = torch.empty(total, Hkv, page, hd, dtype=dt, device=DEV).normal_(generator=g)
    st["v_cache"] = torch.empty(total, Hkv, page, hd, dtype=dt, device=DEV).normal_(generator=g)
    # what a host program that splits a ragged batch itself would keep: each token's segment and position
    seg = np.repeat(np.arange(B), n)
    off = np.arange(T) - np.repeat(np.cumsum(n) - n, n)
    st["seg"], st["tok_pos"], st["tok_off"], st["W"] = _dev(seg, torch.int64), _dev(c[seg] + off, torch.int64), _dev(off, torch.int64), int(n.max())
    if case["op"] == "append":
        qkv = rows(T, (H + 2 * Hkv), hd)
        st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        st["cos"], st["sin"] = _tables(S, case["rot"], 1.0) if case["rot"] else (None, None)
        return st
    st["q"] = rows(T, H, hd, scale=2.0)
    _, _, _, _, starts, prefix = _ranges(case)
    st["starts"] = _dev(starts) if starts is not None else None
    st["prefix"] = _dev(prefix) if prefix is not None else None
    st["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEV, dtype=torch.float32) / H) if case["slopes"] else None
    return st


# ---- one pass ----------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"rope": _plain_rope, "append": _plain_append, "attn": _plain_attn}[state["op"]](state)


def _run_own(s):
    from altxs_amd import ops

    if s["op"] == "rope":
        return ops.rope(s["x"], s["pos"], s["cos"], s["sin"], interleaved=s["interleaved"], inverse=s["inverse"])
    if s["op"] == "append":
        q = ops.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["pos"], cu=s["cu"], q=s["q"],
                             cos=s["cos"], sin=s["sin"], interleaved=s["interleaved"])
        return {"q": q, "k": s["k_cache"], "v": s["v_cache"]}
    return ops.paged_attn(s["q"], s["k_cache"], s["v_cache"], s["table"], s["pos"], cu=s["cu"], max_len=s["max_len"],
                          softcap=s["softcap"], slopes=s["slopes"], window=s["window"], starts=s["starts"],
                          prefix=s["prefix"])


def _rotate(x, cos, sin, interleaved, inverse=False):
    """x [T, H, hd], cos/sin [T, rot / 2]: (a, b) -> (a cos + b sin, b cos - a sin) for each pair."""
    y = x.float()
    half = cos.shape[-1]
    c, s = cos[:, None], -sin[:, None] if inverse else sin[:, None]
    z = y[..., :2 * half]
    a, b = (z[..., 0::2], z[..., 1::2]) if interleaved else (z[..., :half], z[..., half:])
    ra, rb = a * c + b * s, b * c - a * s
    z = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([z, y[..., 2 * half:]], -1).to(x.dtype)


def _plain_rope(s):
    p = s["pos"].long()
    return _rotate(s["x"], s["cos"][p], s["sin"][p], s["interleaved"], s["inverse"])


def _plain_append(s):
    p, page = s["tok_pos"], s["page"]
    k, q = s["k"], s["q"]
    if s["rot"]:
        c, sn = s["cos"][p], s["sin"][p]
        k, q = _rotate(k, c, sn, s["interleaved"]), _rotate(q, c, sn, s["interleaved"])
    at = s["table"][s["seg"], p // page].long()
    s["k_cache"][at, :, p % page] = k
    s["v_cache"][at, :, p % page] = s["v"]
    return {"q": q.contiguous() if s["rot"] else q.clone(), "k": s["k_cache"], "v": s["v_cache"]}


def _gathered(cache, table, S):
    """[B, Hkv, S, hd] fp32 of every segment's pages in order."""
    B, _ = table.shape
    _, Hkv, page, hd = cache.shape
    x = cache[table.clamp_min(0).long()].float()  # [B, width, Hkv, page, hd]
    return x.transpose(1, 2).reshape(B, Hkv, -1, hd)[:, :, :S]


def _plain_attn(s):
    B, H, Hkv, hd, S, W = s["B"], s["H"], s["Hkv"], s["hd"], s["max_len"], s["W"]
    G, dev = H // Hkv, s["q"].device
    T = s["q"].shape[0]
    q = torch.zeros(B, W, H, hd, device=dev)
    q[s["seg"], s["tok_off"]] = s["q"].float()
    q = q.view(B, W, Hkv, G, hd).transpose(1, 2).reshape(B, Hkv, W * G, hd)
    new = (s["cu"][1:] - s["cu"][:-1]).long() if s["cu"] is not None else torch.full((B,), W, device=dev)
    length = s["pos"].long() + new
    key = torch.arange(S, device=dev)
    p = s["pos"].long()[:, None] + torch.arange(W, device=dev)
    hi = p + 1
    if s["prefix"] is not None:
        hi = torch.maximum(hi, torch.minimum(s["prefix"].long(), length)[:, None])
    lo = torch.zeros_like(p)
    if s["window"]:
        lo = torch.maximum(lo, p - s["window"] + 1)
    if s["starts"] is not None:
        st = torch.zeros(B, W, dtype=torch.int64, device=dev)
        st[s["seg"], s["tok_off"]] = s["starts"].long()
        lo = torch.maximum(lo, st)
    seen = (key >= lo[..., None]) & (key < hi[..., None])  # [B, W, S]
    x = torch.matmul(q, _gathered(s["k_cache"], s["table"], S).transpose(-1, -2).contiguous()) * hd ** -0.5
    x = x.view(B, Hkv, W, G, S)
    if s["softcap"]:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    if s["slopes"] is not None:
        x = x - s["slopes"].view(Hkv, 1, G, 1) * (p[..., None] - key).abs().float()[:, None, :, None]
    seen = seen[:, None, :, None]
    x = torch.where(seen, x, x.new_full((), -math.inf))
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    x = x / x.sum(-1, keepdim=True).clamp_min(1e-30)
    v = torch.where((key < length[:, None])[:, None, :, None], _gathered(s["v_cache"], s["table"], S), 0.0)
    y = torch.matmul(x.view(B, Hkv, W * G, S), v).view(B, Hkv, W, G, hd)
    return y.transpose(1, 2).reshape(B, W, H, hd)[s["seg"], s["tok_off"]].to(s["q"].dtype)


# ---- the definition in 64 bits -----------------------------------------------

def _turned(x, pos, cos, sin, interleaved, sign):
    """Each pair of a head as a complex number, turned by its position's angle."""
    y = x.double().clone()
    half = cos.shape[1]
    w = torch.complex(cos.double(), -sign * sin.double())[pos.long()][:, None]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    z = torch.complex(y[..., first], y[..., second]) * w
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _turned(s["x"], s["pos"], s["cos"], s["sin"], case["interleaved"], -1.0 if case["inverse"] else 1.0)
    n, c = _lens(case)
    first = np.cumsum(n) - n
    page, table = case["page"], s["table"].cpu().numpy()
    if case["op"] == "append":
        k, q = s["k"].double(), s["q"].double()
        if case["rot"]:
            p = torch.from_numpy(np.concatenate([np.arange(a, a + m) for a, m in zip(c, n)])).to(DEV)
            k, q = (_turned(x, p, s["cos"], s["sin"], case["interleaved"], 1.0) for x in (k, q))
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for b in range(case["B"]):
            done = 0
            while done < n[b]:  # a page's share at a time
                at = int(c[b]) + done
                m = min(page - at % page, int(n[b]) - done)
                rows = slice(int(first[b]) + done, int(first[b]) + done + m)
                kc[table[b, at // page], :, at % page:at % page + m] = k[rows].transpose(0, 1)
                vc[table[b, at // page], :, at % page:at % page + m] = s["v"][rows].double().transpose(0, 1)
                done += m
        return {"q": q, "k": kc, "v": vc}
    H, Hkv, hd = case["H"], case["Hkv"], case["hd"]
    _, p, lo, hi, _, _ = _ranges(case)
    out = torch.zeros(int(n.sum()), H, hd, dtype=torch.float64, device=DEV)
    for b in np.flatnonzero(n):
        rows = slice(int(first[b]), int(first[b] + n[b]))
        L = int(c[b] + n[b])
        pages = torch.from_numpy(table[b, :-(-L // page)].astype(np.int64)).to(DEV)
        k, v = (s[x][pages].transpose(0, 1).reshape(Hkv, -1, hd)[:, :L].double() for x in ("k_cache", "v_cache"))
        q = s["q"][rows].double().view(-1, Hkv, H // Hkv, hd).permute(1, 2, 0, 3)  # [Hkv, G, n, hd]
        x = (q / math.sqrt(hd)) @ k[:, None].transpose(-1, -2)
        if case["softcap"]:
            x = (x / case["softcap"]).tanh() * case["softcap"]
        key = torch.arange(L, device=DEV)
        if case["slopes"]:
            slope = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEV, dtype=torch.float64) / H)
            x = x - slope.view(Hkv, -1, 1, 1) * (_dev(p[rows], torch.int64)[:, None] - key).abs()
        hidden = (key < _dev(lo[rows], torch.int64)[:, None]) | (key >= _dev(hi[rows], torch.int64)[:, None])
        x = x.masked_fill(hidden, -math.inf).softmax(-1).masked_fill(hidden, 0.0)
        out[rows] = (x @ v[:, None]).permute(2, 0, 1, 3).reshape(-1, H, hd)
    return out
