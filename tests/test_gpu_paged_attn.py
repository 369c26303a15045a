"""altxs_paged_attn on the device against the 64-bit form, row by row.

Cache rows that no segment holds -- other pages, the end of a last page -- are NaN in
every case here, so a kernel that lets one through fails everywhere.
"""

from __future__ import annotations

import pytest
import torch

from tests.paged_ref import alibi, attn_ref, off, paged_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _log(msg: str) -> None:
    print(f"[gpu-case] {msg}", flush=True)


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _run(c, **kw):
    from altxs_amd import ops

    d = {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in {**c, **kw}.items()}
    return ops.paged_attn(d.pop("q"), d.pop("k"), d.pop("v"), d.pop("table"), d.pop("pos"), **d)


def _check(c, **masks):
    want, tol = attn_ref(c["q"], c["k"], c["v"], c["table"], c["pos"], c["cu"], **masks)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = _run(c, err=err, **masks)
    assert int(err) == 0
    worst = off(got, want, tol)
    assert worst <= 1, worst
    return got


SHAPES = [
    # lens, ctx, H, Hkv, hd, page
    ([1], [0], 1, 1, 64, 16),
    ([1], [1], 8, 8, 64, 64),
    ([1, 1, 1, 1], [0, 62, 63, 64], 8, 8, 64, 64),
    ([1, 1, 1], [255, 256, 257], 8, 4, 64, 32),
    ([1, 1], [1100, 511], 16, 2, 128, 16),
    ([1] * 70, [3 * i for i in range(70)], 4, 4, 64, 16),
    ([2, 2, 2], [1, 254, 700], 8, 8, 64, 256),
    ([5, 0, 17, 1, 0], [0, 40, 130, 600, 9], 8, 2, 64, 32),
    ([16, 3], [48, 1000], 8, 8, 128, 128),
    ([64], [1000], 8, 4, 64, 64),
    ([130, 67], [0, 300], 4, 4, 64, 64),
    ([300], [0], 6, 2, 128, 16),
    ([100, 0, 257, 129], [27, 500, 0, 255], 3, 1, 128, 64),
    ([20, 1], [100, 7], 40, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"n{max(s[0])}x{len(s[0])}-H{s[2]}.{s[3]}-{s[4]}-p{s[5]}")
def test_causal(shape, dtype):
    _log(f"paged_attn causal {shape[2:]} {dtype}")
    _check(paged_case(*shape, dtype, seed=sum(shape[0]) + shape[2]))


@pytest.mark.parametrize("B", [65, 300, 5000])
@pytest.mark.parametrize("n", [1, 40])
def test_many_ragged_segments(B, n):
    """Ragged calls search for their segments: the bits of one call per segment, with idle
    segments between, rows behind the last, and another kernel's tiles."""
    from altxs_amd import ops

    _log(f"paged_attn ragged B={B} n={n}")
    g = torch.Generator().manual_seed(B + n)
    H, Hkv, hd, page = 4, 2, 64, 16
    if n > 1 and B > 1000:
        B = 1000
    lens = torch.randint(0, n + 1, (B,), generator=g) if n > 1 else (torch.rand(B, generator=g) < 0.7).int()
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).int().to(DEV)
    T = int(cu[-1]) + 3
    pos = torch.randint(0, 70, (B,), generator=g, dtype=torch.int32).to(DEV)
    table = torch.randint(0, 32, (B, 7), generator=g, dtype=torch.int32).to(DEV)
    kc, vc = (torch.randn(32, Hkv, page, hd, generator=g).to(BF).to(DEV) for _ in range(2))
    q = torch.randn(T, H, hd, generator=g).to(BF).to(DEV)
    out = torch.full_like(q, 7.0)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.paged_attn(q, kc, vc, table, pos, cu=cu, out=out, err=err)
    assert int(err) == 0 and bool((out[T - 3:] == 7).all())
    # the same tokens as segments of one token each, their positions spelt out: no search
    seg = torch.repeat_interleave(torch.arange(B), lens.long()).to(DEV)
    at = torch.arange(T - 3, device=DEV) - cu.long()[seg]
    one = ops.paged_attn(q[:T - 3], kc, vc, table[seg].contiguous(), (pos[seg] + at).int())
    assert torch.equal(_bits(out[:T - 3]), _bits(one))
    # append finds the same places
    k, v = (torch.randn(T, Hkv, hd, generator=g).to(BF).to(DEV) for _ in range(2))
    own = torch.arange(B * 7, dtype=torch.int32, device=DEV).view(B, 7)
    ka, va, kb, vb = (torch.zeros(B * 7, Hkv, page, hd, dtype=BF, device=DEV) for _ in range(4))
    ops.paged_append(k, v, ka, va, own, pos, cu=cu, err=err)
    ops.paged_append(k[:T - 3], v[:T - 3], kb, vb, own[seg].contiguous(), (pos[seg] + at).int(), err=err)
    assert int(err) == 0 and torch.equal(_bits(ka), _bits(kb)) and torch.equal(_bits(va), _bits(vb))
    cu[B // 2] = T + 9  # one bound past the tokens: flagged, wherever in cu it is
    ops.paged_attn(q, kc, vc, table, pos, cu=cu, err=err)
    assert int(err) & 1


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("masks", ["cap", "slopes", "window", "window1", "prefix", "docs", "all"])
@pytest.mark.parametrize("shape", [SHAPES[4], SHAPES[7], SHAPES[10], SHAPES[12]],
                         ids=["decode", "drafts", "chunks", "gqa128"])
def test_masks(shape, masks, dtype):
    _log(f"paged_attn masks={masks} {shape[2:]} {dtype}")
    c = paged_case(*shape, dtype, seed=17)
    lens, ctx, H = shape[:3]
    kw = {}
    if masks in ("cap", "all"):
        kw["softcap"] = 5.0
    if masks in ("slopes", "all"):
        kw["slopes"] = alibi(H)
    if masks == "window" or masks == "all":
        kw["window"] = 70
    if masks == "window1":
        kw["window"] = 1
    if masks in ("prefix", "all"):
        kw["prefix"] = torch.tensor([(37 * i + 5) % 160 for i in range(len(lens))], dtype=torch.int32)
    if masks in ("docs", "all"):  # documents of 45 tokens; some tokens see nothing at all
        p = torch.cat([torch.arange(a, a + n) for a, n in zip(ctx, lens)])
        s = p // 45 * 45
        s[3::11] = 1 << 30
        s[5::13] = -7
        kw["starts"] = s.to(torch.int32)
    got = _check(c, **kw)
    if masks == "docs" and got.shape[0] > 3:
        assert not got[3].any()


def test_scale_and_large_scores():
    c = paged_case([3, 40], [100, 5], 4, 4, 64, 16, BF, seed=2, qscale=1.0)
    _check(c, scale=0.5)
    _check(c, scale=2.0 ** -10)
    big = paged_case([3, 40], [100, 5], 4, 4, 64, 16, FP, seed=3, qscale=60.0)  # scores of hundreds
    _check(big)


def test_rows_behind_the_last_segment_and_idle_segments():
    c = paged_case([3, 0, 50], [10, 20, 0], 4, 4, 64, 16, BF, seed=4)
    want = _run(c)
    q = torch.cat([c["q"], torch.full((6, 4, 64), float("nan"), dtype=BF)])
    out = torch.full((59, 4, 64), 9.0, dtype=BF, device=DEV)
    got = _run({**c, "q": q}, out=out)
    assert got is out and torch.equal(_bits(got[:53]), _bits(want)) and (got[53:] == 9).all()
    none = torch.zeros(4, dtype=torch.int32)
    out.fill_(9.0)
    _run({**c, "q": q}, out=out, cu=none)
    assert (out == 9).all()


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_bits_do_not_depend_on_the_call(dtype, hd):
    """A row decoded alone, in a batch, in a window, in a whole chunk, on other pages, with a looser bound: the same bits."""
    _log(f"paged_attn bits {dtype} hd={hd}")
    n, H, Hkv = 700, 4, 2
    c = paged_case([n], [0], H, Hkv, hd, 64, dtype, seed=8)
    kw = dict(window=333, softcap=9.0, slopes=alibi(H))
    for masks in ({}, kw):
        whole = _run(c, **masks)
        rows = torch.tensor([0, 1, 63, 64, 255, 256, 257, 300, 511, 512, 640, 699])
        # every row decoded alone as a segment of one batch sharing the pages
        one = dict(q=c["q"][rows], k=c["k"], v=c["v"], table=c["table"].expand(len(rows), -1).contiguous(),
                   pos=rows.to(torch.int32))
        assert torch.equal(_bits(_run(one, **masks)), _bits(whole[rows]))
        for r in (0, 256, 699):
            alone = dict(q=c["q"][r:r + 1], k=c["k"], v=c["v"], table=c["table"], pos=torch.tensor([r], dtype=torch.int32))
            assert torch.equal(_bits(_run(alone, max_len=r + 1, **masks)), _bits(whole[r:r + 1]))
        for a, b in ((0, 5), (250, 270), (500, 564), (123, 700)):
            win = dict(q=c["q"][a:b], k=c["k"], v=c["v"], table=c["table"], pos=torch.tensor([a], dtype=torch.int32))
            assert torch.equal(_bits(_run(win, **masks)), _bits(whole[a:b])), (a, b)
        # a bound of 16384 keys: the chunks are shared among workgroups and folded by a second launch
        far = torch.full((1, 256), -1, dtype=torch.int32)
        far[:, :c["table"].shape[1]] = c["table"]
        for a, b in ((0, 1), (699, 700), (250, 253), (100, 700)):
            win = dict(q=c["q"][a:b], k=c["k"], v=c["v"], table=far, pos=torch.tensor([a], dtype=torch.int32))
            assert torch.equal(_bits(_run(win, **masks)), _bits(whole[a:b])), (a, b)
        # many windows in one call: enough work that the keys are not split
        many = dict(q=c["q"][:640], k=c["k"], v=c["v"], table=c["table"].expand(640 // 16, -1).contiguous(),
                    pos=torch.arange(0, 640, 16, dtype=torch.int32))
        assert torch.equal(_bits(_run(many, **masks)), _bits(whole[:640]))
        reps = 300
        wide = dict(q=c["q"][rows].repeat(reps, 1, 1), k=c["k"], v=c["v"],
                    table=c["table"].expand(len(rows) * reps, -1).contiguous(), pos=rows.to(torch.int32).repeat(reps))
        assert torch.equal(_bits(_run(wide, **masks)), _bits(whole[rows].repeat(reps, 1, 1)))
        # the same keys on small pages, token-major
        k2, v2 = (torch.full((n // 16 + 1, 16, Hkv, hd), float("nan"), dtype=dtype) for _ in range(2))
        flat_k = c["k"][c["table"][0].long()].transpose(1, 2).reshape(-1, Hkv, hd)
        flat_v = c["v"][c["table"][0].long()].transpose(1, 2).reshape(-1, Hkv, hd)
        k2.view(-1, Hkv, hd)[:n], v2.view(-1, Hkv, hd)[:n] = flat_k[:n], flat_v[:n]
        small = dict(q=c["q"], k=k2.to(DEV).transpose(1, 2), v=v2.to(DEV).transpose(1, 2),
                     table=torch.arange(n // 16 + 1, dtype=torch.int32)[None], pos=torch.zeros(1, dtype=torch.int32))
        assert torch.equal(_bits(_run(small, **masks)), _bits(whole))


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("n,hd", [(3, 64), (40, 64), (150, 64), (150, 128)])
def test_masked_nonfinite_values_stay_out(n, hd, dtype, poison):
    """Values that a row does not see -- another document's, ones before its window, later tokens' -- may be anything."""
    _log(f"paged_attn poison {poison} n={n} hd={hd} {dtype}")
    c = paged_case([n, n], [50, 200], 4, 2, hd, 32, dtype, seed=9)
    # documents end at position 100 in segment 0, 230 in segment 1; the last key of each first document and
    # the very last token are poisoned, in V and, for other heads, in K
    clean = {**c, "k": c["k"].clone(), "v": c["v"].clone()}
    lens = n
    hit = [(b, p) for b, p in ((0, 99), (1, 229), (0, 50 + n - 1), (1, 200 + n - 1)) if p < (50, 200)[b] + n]
    for b, p in hit:
        g, s = int(c["table"][b, p // 32]), p % 32
        c["v"][g, 0, s, ::3] = poison
        c["k"][g, 1, s, ::5] = poison
    p = torch.cat([torch.arange(50, 50 + lens), torch.arange(200, 200 + lens)])
    seg = torch.tensor([0] * lens + [1] * lens)
    border = torch.where(seg == 0, 100, 230)
    starts = torch.where(p >= border, border, torch.zeros_like(p))
    sees = torch.zeros(2 * n, dtype=torch.bool)
    for b, x in hit:
        sees |= (seg == b) & (starts <= x) & (p >= x)
    want = _run(clean, starts=starts.to(torch.int32))
    got = _run(c, starts=starts.to(torch.int32))
    assert torch.equal(_bits(got[~sees.to(DEV)]), _bits(want[~sees.to(DEV)]))
    # and rows that do see one show it: V's poison in its dims, K's in every dim of the head's group
    if sees.any():
        bad = got[sees.to(DEV)].float()
        assert not torch.isfinite(bad[:, :2, ::3]).any()
        clean_dims = [d for d in range(hd) if d % 3]
        ref = want[sees.to(DEV)].float()
        assert torch.isfinite(bad[:, :2, clean_dims]).all() and torch.isfinite(ref).all()


def test_bad_pages_positions_and_cu():
    from altxs_amd import ops

    _log("paged_attn flags")
    c = paged_case([2, 2, 30, 2], [70, 100, 40, 9], 4, 4, 64, 32, BF, seed=10)
    want = _run(c)
    fine = lambda got, segs: all(torch.equal(_bits(got[int(c["cu"][b]):int(c["cu"][b + 1])]),  # noqa: E731
                                             _bits(want[int(c["cu"][b]):int(c["cu"][b + 1])])) for b in segs)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    t = c["table"].clone()
    t[0, 1], t[2, 0] = c["k"].shape[0], -1
    got = _run({**c, "table": t}, err=err)
    assert int(err) == 8 and fine(got, (1, 3))
    err.zero_()
    p = c["pos"].clone()
    p[1], p[3] = 1 << 20, -4
    got = _run({**c, "pos": p}, err=err)
    assert int(err) == 1 and fine(got, (0, 2))
    assert not got[2:4].any() and not got[34:].any()  # segments left out: zeros
    err.zero_()
    got = _run(c, err=err, max_len=80)
    assert int(err) == 1 and fine(got, (0, 2, 3)) and not got[2:4].any()
    for cu in ([0, 2, 1, 34, 36], [0, 2, 4, 77, 36], [0, -3, 4, 34, 36]):
        err.zero_()
        _run(c, err=err, cu=torch.tensor(cu, dtype=torch.int32))
        assert int(err) & 1
    torch.cuda.synchronize()
    assert ops is not None


def test_strides():
    c = paged_case([9, 40], [30, 3], 4, 2, 64, 32, BF, seed=12)
    want = _run(c)
    qkv = torch.randn(49, 8, 64, device=DEV).to(BF)
    qkv[:, :4] = c["q"].to(DEV)
    out = torch.zeros(49, 12, 64, dtype=BF, device=DEV)
    got = _run({**c, "q": qkv[:, :4]}, out=out[:, 4:8])
    assert torch.equal(_bits(got), _bits(want)) and not out[:, :4].any() and not out[:, 8:].any()
    kv = torch.stack([c["k"], c["v"]], 1).to(DEV)  # K and V of a page side by side
    assert torch.equal(_bits(_run({**c, "k": kv[:, 0], "v": kv[:, 1]})), _bits(want))
    nhd = {n: c[n].transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for n in "kv"}
    assert torch.equal(_bits(_run({**c, **nhd})), _bits(want))
    q = c["q"].to(DEV)
    assert torch.equal(_bits(_run({**c, "q": q}, out=q)), _bits(want))  # in place


@pytest.mark.parametrize("lens", [[1] * 5, [37, 0, 3, 90, 1]])
def test_captured_and_replayed(lens):
    """Two graphs of calls that need workspaces, replayed in turn with eager work between; inputs change between replays."""
    from altxs_amd import ops

    _log(f"paged_attn graphs {lens}")
    ctx = [900, 40, 600, 33, 1500]
    cs = [paged_case(lens, ctx, 8, 4, 64, 64, BF, seed=s) for s in (1, 2, 3, 4)]
    graphs = []
    for c in cs[:2]:
        d = {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
        call = lambda d=d: ops.paged_attn(d["q"], d["k"], d["v"], d["table"], d["pos"], cu=d["cu"], max_len=d["max_len"])  # noqa: E731
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, d, out, call))
    for i in range(4):
        for (g, d, out, call), c in zip(graphs, (cs[i], cs[3 - i])):
            for name in ("q", "k", "v", "table", "pos", "cu"):
                if d[name].shape == c[name].shape:
                    d[name].copy_(c[name])
            g.replay()
        torch.cuda.synchronize()
        for g, d, out, call in graphs:
            assert torch.equal(_bits(out), _bits(call()))
        torch.cuda.synchronize()


def test_another_stream():
    c = paged_case([1] * 9, [100 * i for i in range(9)], 8, 8, 64, 64, BF, seed=6)
    want = _run(c)
    d = {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [_run(d) for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(_bits(x), _bits(want)) for x in got)


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements, read at its far end."""
    _log("paged_attn long pool")
    n_pages, Hkv, page = (1 << 31) // (8 * 64 * 64) + 70, 8, 64
    c = paged_case([1, 30], [500, 260], 8, Hkv, 64, page, BF, seed=13)
    want = _run(c)
    m = c["k"].shape[0]
    k = torch.zeros(n_pages, Hkv, page, 64, dtype=BF, device=DEV)
    v = torch.zeros_like(k)
    k[-m:], v[-m:] = c["k"].to(DEV), c["v"].to(DEV)
    t = torch.where(c["table"] >= 0, c["table"] + (n_pages - m), c["table"])
    assert torch.equal(_bits(_run({**c, "k": k, "v": v, "table": t})), _bits(want))


def test_refuses():
    from altxs_amd import ops

    c = paged_case([2, 2], [3, 40], 4, 2, 64, 16, BF, seed=14)
    d = {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    ok = dict(q=d["q"], k_cache=d["k"], v_cache=d["v"], table=d["table"], pos=d["pos"], cu=d["cu"])
    assert ops.paged_attn(**ok).shape == (4, 4, 64)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    for kw in (dict(q=d["q"].half()), dict(q=d["q"][..., :32]), dict(k_cache=d["k"].float()), dict(v_cache=d["v"][:1]), dict(v_cache=d["v"].transpose(1, 2).contiguous().transpose(1, 2)),
               dict(pos=d["pos"].long()), dict(table=d["table"].long()), dict(cu=d["cu"][:2]), dict(q=d["q"][:3], cu=None),
               dict(starts=i32(3)), dict(starts=i32(4).long()), dict(prefix=i32(4)), dict(slopes=torch.zeros(3, device=DEV)),
               dict(slopes=torch.zeros(4, dtype=torch.float64, device=DEV)), dict(out=d["q"][:, :2]), dict(out=d["q"].half()),
               dict(out=d["q"][:, :1].expand(4, 4, 64)), dict(err=i32(1).long())):
        with pytest.raises(ValueError):
            ops.paged_attn(**{**ok, **kw})
    for kw in (dict(max_len=-1), dict(window=-2), dict(window=1 << 31), dict(max_len=1 << 40), dict(window=(1 << 32) + 1)):
        with pytest.raises(ValueError):
            ops.paged_attn(**{**ok, **kw})
    odd = torch.zeros(4 * 4 * 64 + 1, dtype=BF, device=DEV)[1:].view(4, 4, 64)
    for kw in (dict(max_len=1 << 20), dict(scale=0.0), dict(scale=-1.0), dict(softcap=-1.0), dict(q=d["q"][:, :3]),
               dict(q=odd), dict(out=odd)):
        with pytest.raises(RuntimeError):
            ops.paged_attn(**{**ok, **kw})
    assert ops.paged_attn(**{**ok, "q": d["q"][:0], "cu": i32(3)}).shape == (0, 4, 64)


def test_append_then_attend_together():
    """A decode loop through the cache object: chunks, then single tokens, segments coming and going; each
    row against the 64-bit form on the tokens appended so far, and against the framework's dense attention."""
    from altxs_amd import ops
    from altxs_amd.paged import PagedKVCache

    _log("paged cache run")
    H, Hkv, hd, rot, B = 8, 4, 64, 16, 3
    cos, sin = ops.rope_tables(256, rot)
    cache = PagedKVCache(14, B, 256, num_kv_heads=Hkv, head_dim=hd, page_size=32, device=DEV)
    g = torch.Generator().manual_seed(20)
    pos, hist = [0] * B, [[] for _ in range(B)]
    for step, lens in enumerate([[40, 0, 7], [1, 33, 1], [1, 1, 1], [1, 1, 0], [0, 3, 90], [1, 1, 1]]):
        if step == 4:  # segment 2 ends; its pages go to a new one
            cache.release(2)
            pos[2], hist[2] = 0, []
        T = sum(lens)
        for b in range(B):
            cache.reserve(b, pos[b] + lens[b])
        qkv = torch.randn(T, H + 2 * Hkv, hd, generator=g).to(BF).to(DEV)
        cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
        p = torch.tensor(pos, dtype=torch.int32, device=DEV)
        q = cache.append(qkv[:, H:H + Hkv], qkv[:, H + Hkv:], p, cu=cu, q=qkv[:, :H], rope=(cos, sin))
        y = cache.attend(q, p, cu=cu)
        cache.check_errors()
        want, tol = attn_ref(q, cache.k, cache.v, cache.table, p, cu)
        assert off(y, want, tol) <= 1
        for b in range(B):
            rows = slice(int(cu[b]), int(cu[b + 1]))
            if lens[b]:
                kr = ops.rope(qkv[rows, H:H + Hkv], torch.arange(pos[b], pos[b] + lens[b], dtype=torch.int32, device=DEV), cos, sin)
                hist[b].append((kr, qkv[rows, H + Hkv:]))
                k, v = (torch.cat([h[i] for h in hist[b]]).transpose(0, 1) for i in (0, 1))
                L = k.shape[1]
                dense = [torch.zeros(1, Hkv, 256, hd, dtype=BF, device=DEV) for _ in range(2)]
                dense[0][0, :, :L], dense[1][0, :, :L] = k, v
                d = ops.decode_attn(q[rows].float().contiguous(), *dense, p[b:b + 1].contiguous(), W=lens[b], natural=True)
                assert off(d.view(-1, H, hd), want[rows], tol[rows]) <= 1
            pos[b] += lens[b]
    assert cache.free_pages == 14 - sum(-(-x // 32) for x in pos)
