"""64-bit CPU forms of the paged-cache operators, with the error bounds the tests use."""

from __future__ import annotations

import math

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


def rope_ref(x, pos, cos, sin, interleaved=False, inverse=False):
    """x [T, H, hd] -> float64; rows outside the tables unchanged."""
    y = x.double().cpu().clone()
    c, s = cos.double().cpu(), sin.double().cpu() * (-1.0 if inverse else 1.0)
    half = c.shape[1]
    ia = torch.arange(half) * 2 if interleaved else torch.arange(half)
    ib = ia + 1 if interleaved else ia + half
    for t, p in enumerate(pos.cpu().tolist()):
        if 0 <= p < c.shape[0]:
            a, b = y[t][:, ia].clone(), y[t][:, ib].clone()
            y[t][:, ia] = a * c[p] + b * s[p]
            y[t][:, ib] = b * c[p] - a * s[p]
    return y


def rope_tol(x, cos, sin, dtype):
    """|err| <= u |y| + 2^-23 (|a| + |b|) max(cos, sin): one product and one fma in fp32, one
    rounding; pairs bounded by the head's largest element."""
    big = x.double().cpu().abs().amax(-1, keepdim=True)
    m = max(1.0, float(cos.abs().max()), float(sin.abs().max()))
    return lambda y: UNIT[dtype] * y.abs() * 1.001 + 2.0 ** -23 * 2 * m * big


def key_range(p, length, window=0, start=0, prefix=0):
    hi = max(p + 1, min(prefix, length))
    lo = max(0, start, p - window + 1 if window else 0)
    return (lo, hi) if lo < hi else (0, 0)


def attn_ref(q, k_cache, v_cache, table, pos, cu, *, scale=None, softcap=0.0, slopes=None, window=0, starts=None,
             prefix=None):
    """(y, tol) [T, H, hd] in float64: every row from its own visible keys.  The
    bound of row (t, h), with A = sum p |v| and n keys:
        u |y|             the output's rounding
      + u' A              the weights' rounding (16-bit types; u' = u, else 0)
      + 2 e A             scores off by e each: fp32 sums of hd products, the scale, cap
                          (a tanh of relative error 2^-21) and bias
      + (n + 16) 2^-24 A  fp32 sums over the keys
    """
    q, kc, vc = q.cpu(), k_cache.cpu(), v_cache.cpu()
    table, pos, cu = table.cpu().numpy(), pos.cpu().numpy(), cu.cpu().numpy()
    T, H, hd = q.shape
    Hkv, page = kc.shape[1], kc.shape[2]
    G = H // Hkv
    scale = hd ** -0.5 if scale is None else scale
    u = UNIT[q.dtype]
    up = u if q.dtype != torch.float32 else 0.0
    y, tol = torch.zeros(T, H, hd, dtype=torch.float64), torch.zeros(T, H, hd, dtype=torch.float64)
    for b in range(len(pos)):
        n = int(cu[b + 1] - cu[b])
        length = int(pos[b]) + n
        for i in range(n):
            t, p = int(cu[b]) + i, int(pos[b]) + i
            lo, hi = key_range(p, length, window, int(starts[t]) if starts is not None else 0,
                               int(prefix[b]) if prefix is not None else 0)
            if lo == hi:
                continue
            keys = np.arange(lo, hi)
            pg, sl = torch.from_numpy(table[b, keys // page].astype(np.int64)), torch.from_numpy(keys % page)
            K, V = kc[pg, :, sl].double(), vc[pg, :, sl].double()  # [n, Hkv, hd]
            K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
            qt = q[t].double()
            s = torch.einsum("hd,nhd->hn", qt, K) * scale
            e = (hd + 4) * 2.0 ** -24 * scale * torch.einsum("hd,nhd->hn", qt.abs(), K.abs())
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            e = e + 2.0 ** -21 * (s.abs() + softcap)
            if slopes is not None:
                d = slopes.double().cpu()[:, None] * torch.from_numpy(np.abs(p - keys)).double()
                s = s - d
                e = e + 2.0 ** -22 * d
            w = torch.softmax(s, -1)
            y[t] = torch.einsum("hn,nhd->hd", w, V)
            A = torch.einsum("hn,nhd->hd", w, V.abs())
            # keys of weight below 2^-40 do not matter to the bound of the others
            e = torch.where(w > 2.0 ** -40, e, torch.zeros_like(e)).amax(-1, keepdim=True)
            tol[t] = u * y[t].abs() + A * (up + 2 * e + (hi - lo + 16) * 2.0 ** -24)
    return y, tol * 1.01 + 1e-30


def paged_case(lens, ctx, H, Hkv, hd, page, dtype, seed, *, spare=3, qscale=2.0):
    """Random queries and a cache whose pages lie in random order; leftovers are NaN."""
    g = torch.Generator().manual_seed(seed)
    r = np.random.RandomState(seed)
    B = len(lens)
    total = [a + b for a, b in zip(lens, ctx)]
    held = [-(-t // page) for t in total]
    width = max(1, max(held))
    n_pages = sum(held) + spare
    perm = r.permutation(n_pages)
    table = np.full((B, width), -1, np.int32)
    k = torch.full((n_pages, Hkv, page, hd), float("nan"))
    v = torch.full((n_pages, Hkv, page, hd), float("nan"))
    at = 0
    for b in range(B):
        for i in range(held[b]):
            pg = int(perm[at])
            at += 1
            table[b, i] = pg
            n = min(page, total[b] - i * page)
            k[pg, :, :n] = torch.randn(Hkv, n, hd, generator=g)
            v[pg, :, :n] = torch.randn(Hkv, n, hd, generator=g)
    T = sum(lens)
    q = (torch.randn(T, H, hd, generator=g) * qscale).to(dtype)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    return dict(q=q, k=k.to(dtype), v=v.to(dtype), table=torch.from_numpy(table), pos=torch.tensor(ctx, dtype=torch.int32),
                cu=torch.from_numpy(cu), max_len=max(1, max(total)))


def alibi(H):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / H) for i in range(H)], dtype=torch.float32)


def off(got, want, tol):
    """Largest error over its bound; inf where one is not finite."""
    d = (got.double().cpu() - want).abs()
    if not torch.isfinite(d).all():
        return math.inf
    return float((d / tol).max()) if d.numel() else 0.0
