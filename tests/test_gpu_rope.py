"""altxs_rope and altxs_paged_append on the device against 64-bit forms."""

from __future__ import annotations

import pytest
import torch

from tests.paged_ref import UNIT, off, rope_ref, rope_tol

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _log(msg: str) -> None:
    print(f"[gpu-case] {msg}", flush=True)


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _tables(rows, rot, **kw):
    from altxs_amd import ops

    return ops.rope_tables(rows, rot, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,hd,rot", [(1, 1, 64, 16), (7, 8, 64, 64), (33, 5, 128, 24), (300, 3, 80, 48), (5, 2, 6, 2),
                                        (64, 8, 64, 12), (2, 40, 128, 128), (9, 1, 1024, 1024)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(T, H, hd, rot, dtype, interleaved):
    from altxs_amd import ops

    _log(f"rope T={T} H={H} hd={hd} rot={rot} {dtype} interleaved={interleaved}")
    g = torch.Generator().manual_seed(T * 100 + rot)
    cos, sin = _tables(500, rot, scaling="yarn", factor=4.0, trained_len=100)
    pos = torch.randint(0, 500, (T,), generator=g).to(torch.int32).to(DEV)
    x = torch.randn(T, H, hd, generator=g).to(dtype).to(DEV)
    tol = rope_tol(x, cos, sin, dtype)
    for inverse in (False, True):
        want = rope_ref(x, pos, cos, sin, interleaved, inverse)
        got = ops.rope(x, pos, cos, sin, interleaved=interleaved, inverse=inverse)
        assert off(got, want, tol(want)) <= 1
        assert torch.equal(_bits(got[..., rot:]), _bits(x[..., rot:]))
        y = x.clone()
        assert ops.rope(y, pos, cos, sin, interleaved=interleaved, inverse=inverse, out=y) is y
        assert torch.equal(_bits(y), _bits(got))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strides(dtype, interleaved):
    """Slices of a joint projection, rows at odd offsets, head-major arrays: the bits of the packed call."""
    from altxs_amd import ops

    g = torch.Generator().manual_seed(3)
    T, H, hd, rot = 37, 4, 64, 32
    cos, sin = _tables(64, rot)
    pos = torch.randint(0, 64, (T,), generator=g).to(torch.int32).to(DEV)
    base = torch.randn(T, 3 * H, hd, generator=g).to(dtype).to(DEV)
    x = base[:, H:2 * H]
    want = ops.rope(x.contiguous(), pos, cos, sin, interleaved=interleaved)
    assert torch.equal(_bits(ops.rope(x, pos, cos, sin, interleaved=interleaved)), _bits(want))
    odd = torch.zeros(T * H * hd + 1, dtype=dtype, device=DEV)[1:].view(T, H, hd)
    odd.copy_(x)
    assert torch.equal(_bits(ops.rope(odd, pos, cos, sin, interleaved=interleaved)), _bits(want))
    major = x.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.zeros_like(base)
    got = ops.rope(major, pos, cos, sin, interleaved=interleaved, out=out[:, :H])
    assert torch.equal(_bits(got), _bits(want)) and not out[:, H:].any()
    copy = base.clone()
    ops.rope(copy[:, H:2 * H], pos, cos, sin, interleaved=interleaved, out=copy[:, H:2 * H])
    assert torch.equal(_bits(copy[:, H:2 * H]), _bits(want))
    assert torch.equal(_bits(copy[:, :H]), _bits(base[:, :H])) and torch.equal(_bits(copy[:, 2 * H:]), _bits(base[:, 2 * H:]))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_inverse_is_the_gradient(interleaved):
    from altxs_amd import ops

    g = torch.Generator().manual_seed(4)
    T, H, hd, rot = 6, 2, 64, 32
    cos, sin = _tables(40, rot, scaling="yarn", factor=2.0, trained_len=20)
    pos = torch.randint(0, 40, (T,), generator=g).to(torch.int32).to(DEV)
    x, dy = (torch.randn(T, H, hd, generator=g, dtype=torch.float64) for _ in range(2))
    got = ops.rope(dy.float().to(DEV), pos, cos, sin, interleaved=interleaved, inverse=True)
    # the formula's gradient, by autograd in 64 bits
    xg = x.clone().requires_grad_()
    rows = pos.long().cpu()
    c, s = cos.double().cpu()[rows][:, None], sin.double().cpu()[rows][:, None]
    z = xg[..., :rot]
    a, b = (z[..., 0::2], z[..., 1::2]) if interleaved else (z[..., :rot // 2], z[..., rot // 2:])
    ra, rb = a * c + b * s, b * c - a * s
    y = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    (torch.cat([y, xg[..., rot:]], -1) * dy.float().double()).sum().backward()
    assert off(got, xg.grad, rope_tol(dy.float(), cos, sin, torch.float32)(xg.grad)) <= 1
    # and differences of the kernel's own forward (linear, so a step of 1 has no error of its own)
    f = lambda v: ops.rope(v.float().to(DEV), pos, cos, sin, interleaved=interleaved).double().cpu()  # noqa: E731
    base = f(x)
    for t, h, d in ((0, 0, 0), (1, 1, 17), (5, 0, rot - 1), (3, 1, 63)):
        step = x.float().double().clone()
        step[t, h, d] += 1.0
        diff = float(((f(step) - base) * dy.float().double()).sum())
        # two rows' fp32 roundings of values up to ~8, against |dy| <= 4: 2^-24 * 8 * 2 elements * 4 * 2
        assert abs(diff - float(got[t, h, d])) < 2 ** -24 * 8 * 2 * 4 * 2 * 4


def test_rope_positions_outside():
    from altxs_amd import ops

    cos, sin = _tables(10, 16)
    x = torch.randn(5, 2, 64, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.rope(x, torch.tensor([-1, 3, -(1 << 31), 9, 0], dtype=torch.int32, device=DEV), cos, sin, err=err)
    assert int(err) == 0
    pos = torch.tensor([10, 3, -1, (1 << 31) - 1, 0], dtype=torch.int32, device=DEV)
    got = ops.rope(x, pos, cos, sin, err=err)
    assert int(err) == 1
    want = rope_ref(x, pos, cos, sin)
    assert off(got, want, rope_tol(x, cos, sin, torch.float32)(want)) <= 1
    assert torch.equal(got[0], x[0]) and torch.equal(got[2], x[2]) and torch.equal(got[3], x[3])


def test_rope_far_positions_and_long_arrays():
    """Angles of position 10^6, and more than 2^31 elements."""
    from altxs_amd import ops

    cos, sin = _tables(1 << 20, 8)
    pos = torch.tensor([(1 << 20) - 1], dtype=torch.int32, device=DEV)
    x = torch.randn(1, 1, 64, device=DEV)
    ang = ((1 << 20) - 1) * 1e4 ** -(torch.arange(4, dtype=torch.float64) / 4)
    want = x.double().cpu().clone()
    a, b = x.double().cpu()[..., :4], x.double().cpu()[..., 4:8]
    want[..., :4], want[..., 4:8] = a * ang.cos() + b * ang.sin(), b * ang.cos() - a * ang.sin()
    assert off(ops.rope(x, pos, cos, sin), want, 2.0 ** -22 * (x.double().cpu().abs().max() + 0 * want)) <= 1
    T = (1 << 31) // (16 * 128) + 5
    x = torch.empty(T, 16, 128, dtype=torch.bfloat16, device=DEV)
    x.copy_(torch.arange(16 * 128, device=DEV).view(16, 128) / 100)
    cos, sin = _tables(64, 128)
    pos = (torch.arange(T, device=DEV) % 64).to(torch.int32)
    ops.rope(x, pos, cos, sin, out=x)
    assert torch.equal(x[:64], x[64:128])
    assert torch.equal(x[T - 5 - (T - 5) % 64:], x[:T - (T - 5 - (T - 5) % 64)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_of_arrays_past_the_cache(dtype, interleaved):
    """Arrays of more than 256 MB are loaded and stored otherwise: the bits of its parts."""
    from altxs_amd import ops

    T, H, hd, part = 40001, 16, 128, 9000
    _log(f"rope of a large array {dtype} interleaved={interleaved}")
    cos, sin = _tables(500, 64)
    g = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn(T, H, hd, generator=g, device=DEV, dtype=torch.float32).to(dtype)
    assert 2 * x.numel() * x.element_size() > 256 << 20 > 2 * part * H * hd * x.element_size()
    pos = torch.randint(-1, 500, (T,), generator=g, device=DEV, dtype=torch.int32)
    got = ops.rope(x, pos, cos, sin, interleaved=interleaved)
    for t in range(0, T, part):
        want = ops.rope(x[t:t + part], pos[t:t + part], cos, sin, interleaved=interleaved)
        assert torch.equal(_bits(got[t:t + part]), _bits(want))
    assert ops.rope(x, pos, cos, sin, interleaved=interleaved, out=x) is x and torch.equal(_bits(x), _bits(got))


def test_rope_refuses():
    from altxs_amd import ops

    cos, sin = _tables(8, 16)
    x = torch.zeros(4, 2, 64, device=DEV)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    ok = dict(x=x, pos=pos, cos=cos, sin=sin)
    for kw in (dict(x=x[0]), dict(x=x.double()), dict(x=x[..., ::2]), dict(pos=pos.long()), dict(pos=pos[:3]), dict(pos=pos.cpu()),
               dict(cos=cos.double()), dict(cos=cos[:4]), dict(sin=sin.cpu()), dict(cos=cos[:, :0], sin=sin[:, :0]),
               dict(x=x[..., :8]), dict(out=x.half()), dict(out=x[:3]), dict(out=x[:1].expand(4, 2, 64)),
               dict(err=torch.zeros(1, device=DEV))):
        with pytest.raises(ValueError):
            ops.rope(**{**ok, **kw})
    buf = torch.zeros(5, 2, 64, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.rope(buf[:4], pos, cos, sin, out=buf[1:])
    assert ops.rope(x[:0], pos[:0], cos, sin).shape == (0, 2, 64)
    assert ops.rope(x[:, :0], pos, cos, sin).shape == (4, 0, 64)


# ---- append --------------------------------------------------------------------


def _append_case(lens, ctx, H, Hkv, hd, page, dtype, seed, behind=0):
    g = torch.Generator().manual_seed(seed)
    total = [a + b for a, b in zip(lens, ctx)]
    held = [-(-t // page) for t in total]
    width, n_pages = max(1, max(held)), sum(held) + 2
    perm = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = perm[at:at + h]
        at += h
    T = sum(lens) + behind
    qkv = torch.randn(T, H + 2 * Hkv, hd, generator=g).to(dtype).to(DEV)
    kc = torch.randn(n_pages, Hkv, page, hd, generator=g).to(dtype).to(DEV)
    vc = torch.randn(n_pages, Hkv, page, hd, generator=g).to(dtype).to(DEV)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    return (qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:], kc, vc, table.to(DEV),
            torch.tensor(ctx, dtype=torch.int32, device=DEV), cu)


def _appended(k, v, kc, vc, table, pos, cu, page):
    """The caches as they should be, from keys already rotated (float64)."""
    kc, vc = kc.double().cpu().clone(), vc.double().cpu().clone()
    for b in range(len(pos)):
        for t in range(int(cu[b]), int(cu[b + 1])):
            p = int(pos[b]) + t - int(cu[b])
            g = int(table[b, p // page])
            kc[g, :, p % page], vc[g, :, p % page] = k[t], v.double().cpu()[t]
    return kc, vc


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens,ctx,H,Hkv,hd,page,rot", [
    ([1], [0], 1, 1, 64, 16, 16), ([1, 1, 1], [63, 64, 200], 8, 8, 64, 64, 16), ([5, 0, 33, 1], [0, 7, 15, 300], 8, 2, 64, 32, 64),
    ([130, 0, 0, 70], [1, 0, 9, 64], 4, 1, 128, 128, 24), ([3] * 70, list(range(70)), 2, 2, 64, 16, 0),
    ([17, 2], [1000, 1023], 6, 3, 80, 1024, 40), ([4, 4], [3, 90], 40, 8, 128, 16, 128),
])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(lens, ctx, H, Hkv, hd, page, rot, dtype, interleaved):
    from altxs_amd import ops

    _log(f"append {len(lens)} segments H={H} Hkv={Hkv} hd={hd} page={page} rot={rot} {dtype} interleaved={interleaved}")
    q, k, v, kc, vc, table, pos, cu = _append_case(lens, ctx, H, Hkv, hd, page, dtype, 11, behind=2)
    T = sum(lens)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    p = torch.cat([torch.arange(a, a + n) for a, n in zip(ctx, lens)]).to(torch.int32)
    p = torch.cat([p, torch.tensor([-1, -1], dtype=torch.int32)])
    kw = {}
    kr, qr = k.double().cpu(), q.double().cpu()
    if rot:
        cos, sin = _tables(max(ctx) + max(lens) + 1, rot)
        kr, qr = (rope_ref(x, p, cos, sin, interleaved) for x in (k, q))
        q_out = torch.full_like(q.contiguous(), 7.0)
        kw = dict(q=q, q_out=q_out, cos=cos, sin=sin, interleaved=interleaved)
    wk, wv = _appended(kr, v, kc, vc, table, pos, cu, page)
    before = kc.clone(), vc.clone()
    got = ops.paged_append(k, v, kc, vc, table, pos, cu=cu, err=err, **kw)
    assert int(err) == 0
    assert torch.equal(vc.double().cpu(), wv)
    if rot:
        big = float(k.double().abs().max())
        assert off(kc, wk, UNIT[dtype] * wk.abs() * 1.001 + 2.0 ** -22 * big) <= 1
        assert got is kw["q_out"] and (got[T:] == 7).all()  # behind the last segment
        assert off(got[:T], qr[:T], rope_tol(q, cos, sin, dtype)(qr)[:T]) <= 1
        # the bits of the rotation alone
        alone = ops.rope(q, p.to(DEV), cos, sin, interleaved=interleaved)
        assert torch.equal(_bits(got[:T]), _bits(alone[:T]))
        # in place, and uniform segments without cu
        if len(set(lens)) == 1:
            kc2, vc2 = before[0].clone(), before[1].clone()
            qq = q[:T].clone()
            assert ops.paged_append(k[:T], v[:T], kc2, vc2, table, pos, q=qq, q_out=qq, cos=cos, sin=sin,
                                    interleaved=interleaved) is qq
            assert torch.equal(_bits(qq), _bits(got[:T])) and torch.equal(_bits(kc2), _bits(kc))
    else:
        assert got is None and torch.equal(kc.double().cpu(), wk)
    touched = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for b in range(len(lens)):
        for i in range(lens[b]):
            touched[int(table[b, (ctx[b] + i) // page]), (ctx[b] + i) % page] = True
    keep = ~touched[:, None, :, None].to(DEV).expand_as(kc)
    assert torch.equal(kc[keep], before[0][keep]) and torch.equal(vc[keep], before[1][keep])


def test_append_layouts():
    """Token-major pages and both halves of one array: the bits of the head-major layout."""
    from altxs_amd import ops

    q, k, v, kc, vc, table, pos, cu = _append_case([9, 30], [5, 40], 4, 2, 64, 32, torch.bfloat16, 5)
    cos, sin = _tables(100, 16)
    kc0, vc0 = kc.clone(), vc.clone()
    ops.paged_append(k, v, kc, vc, table, pos, cu=cu, cos=cos, sin=sin)
    nhd = torch.empty(kc.shape[0], 2, 32, 2, 64, dtype=kc.dtype, device=DEV)  # [page, K/V, slot, head, dim]
    k2, v2 = nhd[:, 0].transpose(1, 2), nhd[:, 1].transpose(1, 2)
    k2.copy_(kc0)
    v2.copy_(vc0)
    ops.paged_append(k, v, k2, v2, table, pos, cu=cu, cos=cos, sin=sin)
    assert torch.equal(_bits(k2), _bits(kc)) and torch.equal(_bits(v2), _bits(vc))
    odd = torch.empty(kc.numel() + 1, dtype=kc.dtype, device=DEV)[1:].view(kc.shape)  # rows off 16 bytes
    odd.copy_(kc0)
    ops.paged_append(k, v, odd, vc0, table, pos, cu=cu, cos=cos, sin=sin)
    assert torch.equal(_bits(odd), _bits(kc))


def test_append_in_place_in_a_packed_array():
    """q, k and v as parts of one [T, H + 2 Hkv, hd] array, q rotated where it lies."""
    from altxs_amd import ops

    q, k, v, kc, vc, table, pos, cu = _append_case([2, 5], [0, 30], 4, 2, 64, 16, torch.bfloat16, 8)
    cos, sin = _tables(64, 16)
    kc2, vc2 = kc.clone(), vc.clone()
    want = ops.paged_append(k, v, kc, vc, table, pos, cu=cu, q=q, cos=cos, sin=sin)
    qkv = torch.cat([q, k, v], 1)
    parts = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    got = ops.paged_append(parts[1], parts[2], kc2, vc2, table, pos, cu=cu, q=parts[0], q_out=parts[0], cos=cos, sin=sin)
    assert got.data_ptr() == qkv.data_ptr() and torch.equal(_bits(got), _bits(want))
    assert torch.equal(_bits(kc2), _bits(kc)) and torch.equal(_bits(vc2), _bits(vc))
    assert torch.equal(_bits(parts[1]), _bits(k)) and torch.equal(_bits(parts[2]), _bits(v))


def test_append_flags():
    """Bad pages, positions and cu: flagged, the rest appended, nothing else touched."""
    from altxs_amd import ops

    q, k, v, kc, vc, table, pos, cu = _append_case([4, 4, 4, 4], [0, 30, 10, 60], 2, 2, 64, 16, torch.bfloat16, 6)
    cos, sin = _tables(200, 16)
    want_k, want_v = _appended(rope_ref(k, torch.cat([torch.arange(a, a + 4) for a in (0, 30, 10, 60)]).int(), cos, sin), v, kc,
                               vc, table, pos, cu, 16)
    k0 = kc.double().cpu()
    bad = table.clone()
    bad[0, 0], bad[2, 0] = kc.shape[0], -5
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    p2 = pos.clone()
    p2[3] = 4 * 1000
    ops.paged_append(k, v, kc, vc, bad, p2, cu=cu, cos=cos, sin=sin, err=err)
    assert int(err) == 9
    for b, fine in ((0, False), (1, True), (2, False), (3, False)):
        for i in range(4):
            x = int(pos[b]) + i
            g = int(table[b, x // 16])
            skipped = not fine and not (b == 2 and x >= 16)  # segment 2's good second page is not reached here
            w = k0 if skipped else want_k
            assert (kc.double().cpu()[g, :, x % 16] - w[g, :, x % 16]).abs().max() <= 2 ** -7 * 6
    for c in ([0, 4, 2, 8, 16], [0, 4, 8, 99, 16], [0, -3, 8, 12, 16]):
        err.zero_()
        ops.paged_append(k, v, kc, vc, table, pos, cu=torch.tensor(c, dtype=torch.int32, device=DEV), cos=cos, sin=sin, err=err)
        assert int(err) & 1
    err.zero_()
    ops.paged_append(k, v, kc, vc, table, pos, cu=cu, cos=cos[:50].contiguous(), sin=sin[:50].contiguous(), err=err)
    assert int(err) == 1


def test_append_refuses():
    from altxs_amd import ops

    q, k, v, kc, vc, table, pos, cu = _append_case([2, 2], [0, 30], 4, 2, 64, 16, torch.bfloat16, 7)
    cos, sin = _tables(64, 16)
    ok = dict(k=k, v=v, k_cache=kc, v_cache=vc, table=table, pos=pos, cu=cu, q=q, cos=cos, sin=sin)
    for kw in (dict(v=v[:3]), dict(v=v.half()), dict(k=k.float()), dict(k_cache=kc.half()), dict(k_cache=kc[:, :1]),
               dict(v_cache=vc[:, :, :8]), dict(table=table.long()), dict(table=table[0]), dict(table=table.t()),
               dict(pos=pos.long()), dict(pos=pos[:1]), dict(cu=cu[:2]), dict(cos=None), dict(q=q[:1]), dict(q=q.half()),
               dict(q_out=q[:, :2]), dict(q_out=k[:, :1].expand(4, 4, 64)), dict(cos=None, sin=None, q_out=q),
               dict(q=q[:, :2], q_out=k), dict(q=q[:, :2], q_out=v), dict(q=q[:, :2], q_out=q[:, 1:3]),
               dict(k=k[:3], v=v[:3], q=q[:3], cu=None), dict(pos=pos.cpu())):
        with pytest.raises(ValueError):
            ops.paged_append(**{**ok, **kw})
    with pytest.raises(RuntimeError, match="expanded"):
        ops.paged_append(k, v, kc[:1].expand(*kc.shape), vc[:1].expand(*vc.shape), table, pos, cu=cu)
    with pytest.raises(RuntimeError, match="page_size"):
        ops.paged_append(k, v, kc[:, :, :12], vc[:, :, :12], table, pos, cu=cu)
    before = kc.clone()
    z = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert ops.paged_append(k[:0], v[:0], kc, vc, table, pos, cu=z, q=q[:0], cos=cos, sin=sin).shape == (0, 4, 64)
    assert torch.equal(_bits(kc), _bits(before))
    assert ops.paged_append(k, v, kc, vc, table, pos, cu=z, q=q) is q and torch.equal(_bits(kc), _bits(before))
