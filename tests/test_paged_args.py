"""Refusals of the paged-cache entry points, their layouts, the rope tables and the
page bookkeeping -- everything that runs without a GPU."""

from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from altxs_amd import _lib, ops
from altxs_amd.paged import PagedKVCache

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "altxs.h")
FAKE = 1 << 20


def _rope(**kw):
    a = _lib.RopeArgs(FAKE, FAKE * 2, FAKE, FAKE, FAKE, None, 4, 16, 512, 64, 512, 64, 8, 64, 16, _lib.BF16, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _append(**kw):
    a = _lib.PagedAppendArgs(T=4, n_pages=8, rope_rows=64, B=4, H=8, Hkv=8, head_dim=64, page_size=64, table_width=2, rot=16,
                             dtype=_lib.BF16, kv_page=32768, kv_head=4096, kv_slot=64)
    for n in "k v q q_out k_cache v_cache table pos cos sin".split():
        setattr(a, n, FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _attn(**kw):
    a = _lib.PagedAttnArgs(T=4, n_pages=8, B=4, H=8, Hkv=8, head_dim=64, page_size=64, table_width=2, max_len=128,
                           dtype=_lib.BF16, scale=0.125, q_tok=512, q_head=64, out_tok=512, out_head=64, kv_page=32768,
                           kv_head=4096, kv_slot=64)
    for n in "q k_cache v_cache out table pos".split():
        setattr(a, n, FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(dtype=3), b"dtype"), (dict(flags=4), b"flags"), (dict(rot=15), b"rot"), (dict(rot=66), b"rot"), (dict(rot=0), b"rot"),
    (dict(H=0), b"H="), (dict(T=-1), b"T"), (dict(rows=0), b"rows"), (dict(x=None), b"null"), (dict(cos=None), b"null"),
    (dict(head_dim=0), b"head_dim"), (dict(head_dim=2048), b"head_dim"),
])
def test_rope_refusals(kw, what):
    L = _lib.load()
    assert L.altxs_rope(ctypes.byref(_rope(**kw)), None) == -1
    assert what in L.altxs_last_error() and b"altxs_rope" in L.altxs_last_error()
    assert L.altxs_rope(None, None) == -1


@pytest.mark.parametrize("kw,what", [
    (dict(dtype=7), b"dtype"), (dict(flags=2), b"flags"), (dict(rot=3), b"rot"), (dict(rot=80), b"rot"), (dict(rot=0), b"q without"),
    (dict(Hkv=0), b"Hkv"), (dict(H=0), b"H="), (dict(page_size=48), b"page_size"), (dict(page_size=8), b"page_size"),
    (dict(T=5), b"equal segments"), (dict(k=None), b"null"), (dict(q_out=None), b"null"), (dict(table=None), b"null"),
    (dict(sin=None), b"null"), (dict(rope_rows=0), b"rope_rows"), (dict(B=-1), b"bad T"), (dict(T=1 << 31), b"bad T"),
    (dict(kv_slot=-64), b"stride"), (dict(kv_page=1 << 31), b"stride"), (dict(kv_page=0), b"expanded"), (dict(kv_head=0), b"expanded"),
])
def test_append_refusals(kw, what):
    L = _lib.load()
    assert L.altxs_paged_append(ctypes.byref(_append(**kw)), None) == -1
    assert what in L.altxs_last_error(), L.altxs_last_error()


@pytest.mark.parametrize("kw,what", [
    (dict(dtype=-1), b"dtype"), (dict(head_dim=96), b"head_dim"), (dict(H=12), b"multiple"), (dict(Hkv=0), b"multiple"),
    (dict(page_size=100), b"page_size"), (dict(max_len=129), b"max_len"), (dict(scale=0.0), b"scale"),
    (dict(scale=-1.0), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(softcap=-1.0), b"softcap"),
    (dict(softcap=float("inf")), b"softcap"), (dict(softcap=float("nan")), b"softcap"), (dict(softcap=3e38), b"softcap"),
    (dict(softcap=1e-40), b"softcap"), (dict(scale=3e38), b"scale"), (dict(window=-1), b"window"), (dict(T=5), b"equal segments"),
    (dict(T=1 << 29), b"bad T"), (dict(T=1 << 62), b"bad T"), (dict(table_width=1 << 25, max_len=(1 << 30) + 1), b"max_len"),
    (dict(B=1 << 29, cu=FAKE), b"row tiles"), (dict(B=(1 << 31) - 1, H=4096, Hkv=4096, cu=FAKE), b"row tiles"), (dict(kv_slot=-64), b"stride"), (dict(kv_page=1 << 31), b"stride"), (dict(q=None), b"null"), (dict(pos=None), b"null"),
])
def test_attn_refusals(kw, what):
    L = _lib.load()
    assert L.altxs_paged_attn(ctypes.byref(_attn(**kw)), None) == -1
    assert what in L.altxs_last_error(), L.altxs_last_error()


def test_workspace_of_few_tokens_among_many_idle_segments():
    """Few row tiles share their chunks; hundreds of thousands of idle segments' slots do not multiply by it."""
    L = _lib.load()
    big = dict(table_width=512, max_len=32768, cu=FAKE)
    assert L.altxs_paged_attn_workspace_bytes(ctypes.byref(_attn(B=4, **big))) == 4 * 8 * 128 * (8 + 64 * 4)
    assert L.altxs_paged_attn_workspace_bytes(ctypes.byref(_attn(B=1000, **big))) == 0
    assert L.altxs_paged_attn_workspace_bytes(ctypes.byref(_attn(B=1 << 20, **big))) == 0


def test_nothing_to_do_is_done():
    L = _lib.load()
    assert L.altxs_rope(ctypes.byref(_rope(T=0, x=None, out=None, pos=None)), None) == 0
    assert L.altxs_paged_append(ctypes.byref(_append(T=0, k=None)), None) == 0
    assert L.altxs_paged_append(ctypes.byref(_append(B=0, T=0)), None) == 0
    assert L.altxs_paged_attn(ctypes.byref(_attn(T=0, q=None)), None) == 0
    assert L.altxs_paged_attn_workspace_bytes(ctypes.byref(_attn(T=0))) == 0
    assert L.altxs_paged_attn_workspace_bytes(ctypes.byref(_attn(page_size=1))) == -1


def test_struct_layouts(tmp_path):
    names = {"AltxsRopeArgs": _lib.RopeArgs, "AltxsPagedAppendArgs": _lib.PagedAppendArgs, "AltxsPagedAttnArgs": _lib.PagedAttnArgs}
    body = "".join(f'  printf("%zu\\n", sizeof({c}));\n' + "".join(f'  printf("%zu\\n", offsetof({c}, {f[0]}));\n' for f in py._fields_)
                   for c, py in names.items())
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{\n{body}  return 0;\n}}\n')
    subprocess.run(["gcc", "-std=c99", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    want = [n for py in names.values() for n in [ctypes.sizeof(py)] + [getattr(py, f[0]).offset for f in py._fields_]]
    assert [int(x) for x in out] == want


def test_packed_structures():
    """pack() lays the fields out as the ctypes structure (and so the header) does."""
    for c in (_lib.RopeArgs, _lib.PagedAppendArgs, _lib.PagedAttnArgs):
        values = [i / 4 if t is ctypes.c_float else i * 1000003 + 1 for i, (_, t) in enumerate(c._fields_)]
        got = c.pack(*values)
        assert len(got) == ctypes.sizeof(c) and got == bytes(c(*values))


def test_apart():
    """Which outputs share memory with an input: against the sets of elements."""
    buf = torch.arange(6 * 10 * 4)
    def view(off, T, H, st):
        return buf.as_strided((T, H, 4), (st, 4, 1), off)
    views = [view(o, T, H, st) for o in (0, 4, 8, 16, 40, 60, 120) for T in (1, 3) for H in (1, 2) for st in (8, 12, 40)]
    for t in views:
        for x in views:
            if ops._apart(t, x):
                assert not set(t.flatten().tolist()) & set(x.flatten().tolist())
    packed = buf[:240].view(6, 10, 4)
    q, k, v = packed[:, :6], packed[:, 6:8], packed[:, 8:]
    assert all(ops._apart(a, b) for a in (q, k, v) for b in (q, k, v) if a is not b)
    assert not ops._apart(q, q) and not ops._apart(packed[:, :7], k) and not ops._apart(k, packed[1:, 7:])


def test_host_tensors_are_refused():
    x = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="device tensor"):
        ops.rope(x, torch.zeros(2, dtype=torch.int32), torch.zeros(8, 8), torch.zeros(8, 8))
    with pytest.raises(ValueError, match="device tensor"):
        ops.paged_append(x, x, x, x, x, x)
    with pytest.raises(ValueError, match="device tensor"):
        ops.paged_attn(x, x, x, x, x)


def test_rope_tables():
    cos, sin = ops.rope_tables(100, 16, device="cpu")
    ang = np.arange(100)[:, None] * 1e4 ** -(np.arange(8) / 8)
    assert np.abs(cos.numpy() - np.cos(ang)).max() < 2 ** -24 and np.abs(sin.numpy() - np.sin(ang)).max() < 2 ** -24
    lin, _ = ops.rope_tables(100, 16, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(lin[40], cos[10])
    # the reference's own stretching of the base: rows of its Rotary warmed at the longer context
    from altxs_amd.config import make_config
    from altxs_amd.synth import rope_table

    cfg = make_config("tiny")
    want, _ = rope_table(cfg, 256)  # block_size 64: factor 4
    ntk, _ = ops.rope_tables(256, 16, scaling="ntk", factor=4.0, device="cpu")
    assert (ntk - want).abs().max() < 256 * 2 ** -22  # fp32 angles up to 256 there: frequency and product rounded
    yc, ys = ops.rope_tables(64, 32, scaling="yarn", factor=4.0, trained_len=2048, device="cpu")
    mag = 0.1 * np.log(4.0) + 1.0
    assert abs(float(yc[0, 0]) - mag) < 1e-6
    f = np.arctan2(ys[1].numpy(), yc[1].numpy()) / 1e4 ** -(np.arange(16) / 16)
    assert abs(f[0] - 1) < 1e-5 and abs(f[-1] - 0.25) < 1e-4 and (np.diff(f) < 1e-5).all()
    for bad in (dict(rot=15), dict(rot=0), dict(scaling="x"), dict(factor=0.5), dict(length=0), dict(rot=2, scaling="ntk")):
        with pytest.raises(ValueError):
            ops.rope_tables(**{"length": 8, "rot": 16, "device": "cpu", **bad})


def test_page_bookkeeping():
    c = PagedKVCache(6, 3, 200, num_kv_heads=2, page_size=64, device="cpu")
    assert c.table.shape == (3, 4) and c.free_pages == 6
    c.reserve(0, 1)
    c.reserve(1, 130)
    assert c.capacity(0) == 64 and c.capacity(1) == 192 and c.free_pages == 2
    c.reserve(1, 100)  # what it has stays
    assert c.capacity(1) == 192
    before = c.table.clone()
    with pytest.raises(RuntimeError, match="3 pages needed, 2 free"):
        c.reserve(2, 129)
    assert torch.equal(c.table, before) and c.free_pages == 2
    with pytest.raises(ValueError):
        c.reserve(0, 201)
    used = [int(x) for x in c.table.flatten() if x >= 0]
    assert len(used) == len(set(used)) == 4 and all(0 <= x < 6 for x in used)
    c.release(1)
    assert c.free_pages == 5 and (c.table[1] == -1).all()
    c.reserve(2, 200)
    assert c.capacity(2) == 256 and c.free_pages == 1
    used = [int(x) for x in c.table.flatten() if x >= 0]
    assert len(used) == len(set(used)) == 5
    for bad in (dict(page_size=48), dict(page_size=8), dict(n_pages=0), dict(segments=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{"n_pages": 4, "segments": 1, "max_len": 64, "num_kv_heads": 1, "device": "cpu", **bad})
