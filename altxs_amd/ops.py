"""torch-facing wrappers of the standalone C-ABI entry points.

Each wrapper validates shapes on the host, launches on the current torch
stream and never synchronises.  Names follow the reference call sites they
replace:

* :func:`scale_cum`     <- ``_scale_cum_np(probs, alphabet_size)``
  (src/model/arithmetic_coder_lm.py:49-64), batched over rows;
* :func:`softmax_cdf`   <- ``torch.softmax(logits, -1, out=probs_dev)``
  (src/xsa_ttt/incremental.py:603-605) + ``_scale_cum_np``;
* :func:`dequant`       <- ``dequantize_channels`` (mixed_bit_delta.py:172-229);
* :func:`qgemm`         <- ``gemv_rows(x, w, out)`` (src/xsa_ttt/ac_gemv.py:391-420);
* :func:`decode_attn`   <- ``run_split_attn`` (src/xsa_ttt/split_attn.py:341-425).

Serving from a paged KV cache (:mod:`altxs_amd.paged` holds the cache itself):

* :func:`rope`, :func:`rope_tables` -- rotary positions
  (``apply_rotary_emb`` / ``Rotary``, src/xsa_ttt/model.py:130-206) of any head
  layout, and their tables for long contexts;
* :func:`paged_append` -- new keys and values into their pages, rotated on the way;
* :func:`paged_attn` -- attention of one or more new tokens per segment over the pages.
"""

from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from .codec import PackedTensor


def _s(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(int(torch.cuda.current_stream(t.device).cuda_stream))


def _need(t: torch.Tensor, dtype, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def scale_cum(probs: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """probs fp32 [..., V] -> cum int32 (uint32 values) [..., V+1]."""
    _need(probs, torch.float32, "probs")
    V = probs.shape[-1]
    rows = probs.numel() // V
    if out is None:
        out = torch.empty(probs.shape[:-1] + (V + 1,), dtype=torch.int32, device=probs.device)
    _need(out, torch.int32, "out")
    rc = _lib.load().altxs_scale_cum(probs.data_ptr(), rows, V, out.data_ptr(), _s(probs))
    _lib.check(rc, "altxs_scale_cum")
    return out


def softmax_cdf(logits: torch.Tensor, *, renorm: bool = False, want_probs: bool = True,
                want_cdf: bool = True):
    """Deterministic fp32 softmax (+ renorm) and integer CDF rows."""
    _need(logits, torch.float32, "logits")
    V = logits.shape[-1]
    rows = logits.numel() // V
    probs = torch.empty_like(logits) if want_probs else None
    cum = (torch.empty(logits.shape[:-1] + (V + 1,), dtype=torch.int32, device=logits.device)
           if want_cdf else None)
    rc = _lib.load().altxs_softmax_cdf(
        logits.data_ptr(), rows, V, _lib.CDF_RENORM if renorm else 0,
        probs.data_ptr() if probs is not None else None,
        cum.data_ptr() if cum is not None else None, _s(logits))
    _lib.check(rc, "altxs_softmax_cdf")
    return probs, cum


class DeviceQTensor:
    """A packed tensor uploaded to HBM (keeps its buffers alive)."""

    def __init__(self, p: PackedTensor, device="cuda"):
        self.codes = torch.from_numpy(np.ascontiguousarray(p.tiled)).to(device)
        self.scales = torch.from_numpy(np.ascontiguousarray(p.tiled_scales).view(np.int16)).to(device)
        self.N, self.K = p.shape
        self.bits = p.bits
        self.qt = _lib.QTensor(self.codes.data_ptr(), self.scales.data_ptr(), self.N, self.K,
                               self.bits, 0)


def dequant(w: DeviceQTensor) -> torch.Tensor:
    out = torch.empty(w.N, w.K, dtype=torch.float32, device=w.codes.device)
    rc = _lib.load().altxs_dequant(ctypes.byref(w.qt), out.data_ptr(), _s(out))
    _lib.check(rc, "altxs_dequant")
    return out


_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def qgemm(w: DeviceQTensor, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """y[rows, N] = x[rows, K] . W^T (fp32 out)."""
    if x.dtype not in _DT:
        raise ValueError(f"x dtype {x.dtype} not supported")
    if not x.is_cuda or not x.is_contiguous() or x.shape[-1] != w.K:
        raise ValueError("x must be a contiguous device tensor [..., K]")
    rows = x.numel() // w.K
    if out is None:
        out = torch.empty(x.shape[:-1] + (w.N,), dtype=torch.float32, device=x.device)
    _need(out, torch.float32, "out")
    rc = _lib.load().altxs_qgemm(ctypes.byref(w.qt), x.data_ptr(), _DT[x.dtype], rows,
                                 out.data_ptr(), _s(x))
    _lib.check(rc, "altxs_qgemm")
    return out


def qgemm_stream(codes: torch.Tensor, scales: torch.Tensor, count: int, N: int, K: int, bits: int,
                 codes_stride: int, scales_stride: int, x: torch.Tensor,
                 out: torch.Tensor) -> torch.Tensor:
    """One launch over ``count`` packed tensors at fixed byte strides."""
    qt = _lib.QTensor(codes.data_ptr(), scales.data_ptr(), N, K, bits, 0)
    rows = x.numel() // K
    rc = _lib.load().altxs_qgemm_stream(ctypes.byref(qt), count, codes_stride, scales_stride,
                                        x.data_ptr(), _DT[x.dtype], rows, out.data_ptr(), _s(x))
    _lib.check(rc, "altxs_qgemm_stream")
    return out


def qgemv(w: DeviceQTensor, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """y[rows, N] = x[rows, K] . W^T for 1..4 fp16/bf16 rows, each row on its
    own (VALU dot arithmetic; a row's bits depend on that row alone)."""
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"x dtype {x.dtype} not supported (fp16 or bf16)")
    if not x.is_cuda or not x.is_contiguous() or x.shape[-1] != w.K:
        raise ValueError("x must be a contiguous device tensor [..., K]")
    rows = x.numel() // w.K
    if out is None:
        out = torch.empty(x.shape[:-1] + (w.N,), dtype=torch.float32, device=x.device)
    _need(out, torch.float32, "out")
    rc = _lib.load().altxs_qgemv(ctypes.byref(w.qt), x.data_ptr(), _DT[x.dtype], rows,
                                 out.data_ptr(), _s(x))
    _lib.check(rc, "altxs_qgemv")
    return out


def qgemv_stream(codes: torch.Tensor, scales: torch.Tensor, count: int, N: int, K: int, bits: int,
                 codes_stride: int, scales_stride: int, x: torch.Tensor,
                 out: torch.Tensor) -> torch.Tensor:
    """:func:`qgemv` over ``count`` packed tensors at fixed byte strides."""
    qt = _lib.QTensor(codes.data_ptr(), scales.data_ptr(), N, K, bits, 0)
    rows = x.numel() // K
    rc = _lib.load().altxs_qgemv_stream(ctypes.byref(qt), count, codes_stride, scales_stride,
                                        x.data_ptr(), _DT[x.dtype], rows, out.data_ptr(), _s(x))
    _lib.check(rc, "altxs_qgemv_stream")
    return out


def decode_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, *,
                W: int = 1, gate: torch.Tensor | None = None, use_xsa: bool = False,
                y_bf16: bool = False, ops_bf16: bool = False, tiled: bool = False,
                err: torch.Tensor | None = None, rows: bool = False,
                xcd_rows: bool = False, natural: bool = False, kv_tail_end: int = 0) -> torch.Tensor:
    """q [B*W, H, 64] fp32; k/v [B, Hkv, max_len, 64] (fp32 or bf16); pos [B] int32.

    bf16 k/v are given in natural [key][dim] order and tiled here
    (:func:`altxs_amd.codec.tile_kv`) unless ``tiled`` says they already are.
    ``ops_bf16`` rounds q and the softmax weights to bf16 for the MFMA products
    (the reference's tl.dot arithmetic); otherwise fp32-faithful splits.
    ``rows`` runs windows (W > 1) of a bf16 cache one row per workgroup (the
    decode kernel) instead of the window kernel; the bits are the same.
    ``xcd_rows`` places the one-row kernel's workgroups in 8-row tiles, tile t
    on XCD t % 8 (B*W a multiple of 64; otherwise ignored); the bits are the same.
    ``natural`` keeps bf16 k/v in their natural order (the reference's k_pack
    layout; the MFMA kernel reads them in place, with the tiled layout's bits).  ``kv_tail_end`` (natural
    layouts): window token t's K/V sit in row kv_tail_end - W + t and query t
    attends to rows [0, pos) and then to those rows (the reference's
    StaticKV tail, model.py:259-461).
    """
    from .codec import tile_kv

    _need(q, torch.float32, "q")
    _need(pos, torch.int32, "pos")
    B, Hkv, max_len, hd = k.shape
    if v.shape != k.shape or v.dtype != k.dtype or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("k and v must be contiguous with equal shape/dtype")
    if k.dtype == torch.bfloat16 and not tiled and not natural:
        k = tile_kv(k, "k").contiguous()
        v = tile_kv(v, "v").contiguous()
    H = q.shape[1]
    a = _lib.AttnArgs()
    a.B, a.W, a.H, a.Hkv, a.head_dim, a.max_len = B, W, H, Hkv, hd, max_len
    a.kv_bf16 = (_lib.KV_F32 if k.dtype != torch.bfloat16 else
                 _lib.KV_BF16_NATURAL if natural else _lib.KV_BF16)
    a.kv_tail_end = int(kv_tail_end)
    a.y_bf16 = int(y_bf16)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.kv_seg_stride = Hkv * max_len * hd
    a.pos = pos.data_ptr()
    a.gate = gate.data_ptr() if gate is not None else None
    a.use_xsa = int(use_xsa)
    a.flags = ((_lib.ATTN_OPS_BF16 if ops_bf16 else 0) | (_lib.ATTN_ROWS if rows else 0)
               | (_lib.ATTN_XCD_ROWS if xcd_rows else 0))
    y = torch.empty(B * W, H * hd, dtype=torch.bfloat16 if y_bf16 else torch.float32,
                    device=q.device)
    a.y = y.data_ptr()
    a.err = err.data_ptr() if err is not None else None
    rc = _lib.load().altxs_decode_attn(ctypes.byref(a), _s(q))
    _lib.check(rc, "altxs_decode_attn")
    return y


# ---- serving from a paged KV cache -------------------------------------------


def rope_tables(length: int, rot: int, base: float = 1e4, *, scaling: str | None = None, factor: float = 1.0,
                trained_len: int = 2048, device="cuda"):
    """cos/sin fp32 [length, rot/2] of the rotary angles pos * base^(-2i/rot).

    The angles are formed in float64, so far positions keep theirs (position 10^6
    in fp32 would be off by 0.03 rad).  ``scaling`` stretches them for contexts
    ``factor`` times the ``trained_len`` tokens a model was trained on:

    * ``"linear"``: positions divided by the factor;
    * ``"ntk"``: base * factor^(rot/(rot-2)), the rule of the reference's Rotary
      (src/xsa_ttt/model.py:147-192);
    * ``"yarn"``: dims that turn more than 32 times in ``trained_len`` tokens stay,
      those that turn less than once are divided by the factor, a linear ramp
      between, and cos/sin carry the method's 0.1 ln(factor) + 1 (arXiv 2309.00071).
    """
    if rot < 2 or rot % 2 or length < 1:
        raise ValueError(f"rope_tables: rot={rot} must be even and length={length} positive")
    if scaling not in (None, "linear", "ntk", "yarn") or factor < 1.0:
        raise ValueError(f"rope_tables: scaling={scaling!r} factor={factor}")
    if scaling == "ntk":
        if rot == 2:
            raise ValueError("rope_tables: ntk scaling needs rot > 2")
        base = base * factor ** (rot / (rot - 2))
    freq = base ** -(np.arange(0, rot, 2, dtype=np.float64) / rot)
    mag = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        turns = freq * trained_len / (2 * np.pi)
        keep = np.clip((turns - 1.0) / 31.0, 0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
        mag = 0.1 * np.log(factor) + 1.0
    ang = np.outer(np.arange(length, dtype=np.float64), freq)
    return tuple(torch.from_numpy((mag * f(ang)).astype(np.float32)).to(device) for f in (np.cos, np.sin))


# Host time counts here: a decode step's rotation, append or attention runs a few
# microseconds.  The checks below read each attribute once and pack the argument
# structure in one call; the stream comes as the handle itself (torch's public
# current_stream builds an object for it, 1.9 us against 0.1).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _heads(t: torch.Tensor, name: str, index: int = -1, dtype=None) -> tuple:
    """Strides of a [T, heads, head_dim] device tensor whose heads are contiguous."""
    st = t.stride()
    if len(st) != 3 or st[2] != 1 or not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor [T, heads, head_dim] with contiguous heads")
    if t.dtype not in _DT:
        raise ValueError(f"{name} dtype {t.dtype} not supported")
    if dtype is not None and (t.dtype != dtype or t.get_device() != index):
        raise ValueError(f"{name} must have the dtype and device of the other heads")
    return st


def _span(t: torch.Tensor) -> tuple[int, int]:
    lo = t.data_ptr()
    return lo, lo + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _apart(t: torch.Tensor, x: torch.Tensor) -> bool:
    """Whether two [T, heads, head_dim] tensors share no memory: their spans do not meet, or
    their tokens alternate in one buffer (q, k and v as parts of one array)."""
    lo, hi = _span(t)
    xl, xh = _span(x)
    if hi <= xl or xh <= lo:
        return True
    size, period = t.element_size(), t.stride(0) * t.element_size()
    if x.stride(0) != t.stride(0) or not period:
        return False
    d = (xl - lo) % period
    width, xwidth = (size * (1 + (n[1] - 1) * st[1] + n[2] - 1) for n, st in ((t.shape, t.stride()), (x.shape, x.stride())))
    return d >= width and d + xwidth <= period


def _output(t: torch.Tensor, name: str, like: torch.Tensor, *reads: torch.Tensor) -> tuple:
    """Strides of a caller's output: ``like``'s shape, every element its own, and either ``like``
    itself or apart from it, and apart from the other tensors that are read."""
    st = _heads(t, name, like.get_device(), like.dtype)
    if t.shape != like.shape:
        raise ValueError(f"{name} must have the shape {tuple(like.shape)}")
    if any(n > 1 and s == 0 for n, s in zip(t.shape, st)):
        raise ValueError(f"{name} must not be expanded")
    if t.numel():
        for x in (like, *reads):
            same = x is like and x.data_ptr() == t.data_ptr() and x.stride() == st
            if x.numel() and not same and not _apart(t, x):
                raise ValueError(f"{name} must be the input itself or not overlap what is read")
    return st


def _index(t: torch.Tensor, name: str, n: int, index: int) -> int:
    if t.dtype != torch.int32 or t.get_device() != index or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor [{n}] on device {index}")
    return t.data_ptr()


def _err(err: torch.Tensor | None, index: int):
    if err is None:
        return 0
    if err.dtype != torch.int32 or err.get_device() != index or err.numel() < 1:
        raise ValueError(f"err must be an int32 tensor on device {index}")
    return err.data_ptr()


def _rot_tables(cos: torch.Tensor, sin: torch.Tensor, hd: int, index: int) -> tuple[int, int]:
    """(rows, rot) of a pair of tables [rows, rot/2]."""
    shape = cos.shape
    if (cos.dtype != torch.float32 or sin.dtype != torch.float32 or len(shape) != 2 or sin.shape != shape
            or cos.get_device() != index or sin.get_device() != index or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError(f"cos and sin must be contiguous fp32 tensors [rows, rot/2] on device {index}")
    rows, half = shape
    if not 2 <= 2 * half <= hd or rows < 1:
        raise ValueError(f"tables of {2 * half} dims for heads of {hd}")
    return rows, 2 * half


def _launch(name: str, args: bytes, index: int) -> None:
    """Call ``name`` on the current stream of device ``index`` (which need not be the current one)."""
    f = getattr(_lib.load(), name)
    if index == torch.cuda.current_device():
        rc = f(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def rope(x: torch.Tensor, pos: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *, interleaved: bool = False,
         inverse: bool = False, out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions: x [T, H, hd] (fp32, bf16 or fp16, any token and head
    strides), pos [T] int32, cos/sin fp32 [rows, rot/2].

    The pairs (a, b) of each head's first ``rot`` dims -- (i, i + rot/2), or
    (2i, 2i + 1) with ``interleaved`` -- become (a cos + b sin, b cos - a sin), the
    reference's sign (src/xsa_ttt/model.py:195-206); ``inverse`` turns the other
    way, which is also the gradient.  ``out`` may be ``x``.  Rows whose position is
    outside the tables are copied unrotated and, unless it is negative
    (padding), flagged in ``err`` (int32).
    """
    xs = _heads(x, "x")
    T, H, hd = x.shape
    index = x.get_device()
    rows, rot = _rot_tables(cos, sin, hd, index)
    if out is None:
        out = x.new_empty((T, H, hd))
        os_ = (H * hd, hd)
    else:
        os_ = _output(out, "out", x)
    a = _lib.RopeArgs.pack(x.data_ptr(), out.data_ptr(), _index(pos, "pos", T, index), cos.data_ptr(), sin.data_ptr(),
                      _err(err, index), T, rows, xs[0], xs[1], os_[0], os_[1], H, hd, rot, _DT[x.dtype],
                      (_lib.ROPE_INTERLEAVED if interleaved else 0) | (_lib.ROPE_INVERSE if inverse else 0), 0)
    if H:
        _launch("altxs_rope", a, index)
    return out


def _pages(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, pos: torch.Tensor, cu: torch.Tensor | None,
           T: int, dtype, index: int) -> tuple:
    """Check the cache's arrays; returns (its strides, segments, table width, pos, cu)."""
    st = k_cache.stride()
    if len(st) != 4 or v_cache.shape != k_cache.shape or st[3] != 1 or v_cache.stride() != st:
        raise ValueError("k_cache and v_cache must be [n_pages, Hkv, page_size, head_dim] of equal shape and strides, "
                         "with contiguous rows")
    if (k_cache.dtype != dtype or v_cache.dtype != dtype or k_cache.get_device() != index
            or v_cache.get_device() != index):
        raise ValueError("the caches must have the dtype and device of the heads")
    if table.dim() != 2 or table.dtype != torch.int32 or table.get_device() != index or not table.is_contiguous():
        raise ValueError(f"table must be a contiguous int32 tensor [segments, pages] on device {index}")
    B, width = table.shape
    pp = _index(pos, "pos", B, index)
    if cu is not None:
        return st, B, width, pp, _index(cu, "cu", B + 1, index)
    if B and T % B:
        raise ValueError(f"{T} tokens are not {B} equal segments (give cu)")
    return st, B, width, pp, 0


def paged_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor,
                 pos: torch.Tensor, *, cu: torch.Tensor | None = None, q: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                 interleaved: bool = False, err: torch.Tensor | None = None) -> torch.Tensor | None:
    """Write new keys and values k, v [T, Hkv, hd] into their segments' pages.

    k_cache/v_cache [n_pages, Hkv, page_size, hd] (any strides, the same for both,
    contiguous rows; page_size a power of two, 16 to 1024), table int32 [B, width] (page ids in
    order), pos int32 [B]: new token t of segment b goes to position pos[b] + t.
    ``cu`` int32 [B + 1]: segment b's tokens are rows cu[b] to cu[b+1] (default:
    T / B each); rows from cu[B] on are left alone.  With tables ``cos``/``sin`` the
    keys are rotated by their positions on the way (as :func:`rope`), and so
    is ``q`` [T, H, hd] into ``q_out`` (default: a new tensor; may be ``q``), which
    is returned -- a new one's rows that belong to no segment, or to one that was
    left out (``err``), are not written.  Without tables ``q`` is returned as it is.
    """
    ks = _heads(k, "k")
    T, Hkv, hd = shape = k.shape
    index, dtype = k.get_device(), k.dtype
    vs = _heads(v, "v", index, dtype)
    if v.shape != shape:
        raise ValueError("k and v must have equal shapes")
    kv, B, width, pp, cp = _pages(k_cache, v_cache, table, pos, cu, T, dtype, index)
    n_pages, ch, page, chd = k_cache.shape
    if ch != Hkv or chd != hd or not Hkv:
        raise ValueError(f"caches of {ch} heads of {chd}, keys of {Hkv} of {hd}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    rows = rot = H = 0
    qp = qo = tp = sp = 0
    qs = os_ = (0, 0)
    result = q
    if cos is not None:
        rows, rot = _rot_tables(cos, sin, hd, index)
        tp, sp = cos.data_ptr(), sin.data_ptr()
        if q is not None:
            qs = _heads(q, "q", index, dtype)
            qT, H, qd = q.shape
            if qT != T or qd != hd:
                raise ValueError(f"q must be [{T}, heads, {hd}]")
            if q_out is None:
                result = q.new_empty((T, H, hd))
                os_ = (H * hd, hd)
            else:
                result, os_ = q_out, _output(q_out, "q_out", q, k, v)
            if H:
                qp, qo = q.data_ptr(), result.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without cos and sin")
    a = _lib.PagedAppendArgs.pack(k.data_ptr(), v.data_ptr(), qp, qo, k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(),
                             pp, cp, tp, sp, _err(err, index), T, n_pages, rows, ks[0], ks[1], vs[0], vs[1],
                             qs[0], qs[1], os_[0], os_[1], kv[0], kv[1], kv[2], B, H, Hkv, hd, page, width, rot,
                             _DT[dtype], _lib.ROPE_INTERLEAVED if interleaved and rot else 0, 0)
    _launch("altxs_paged_append", a, index)
    return result


def paged_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, pos: torch.Tensor, *,
               cu: torch.Tensor | None = None, max_len: int | None = None, scale: float | None = None,
               softcap: float = 0.0, slopes: torch.Tensor | None = None, window: int = 0,
               starts: torch.Tensor | None = None, prefix: torch.Tensor | None = None,
               out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new tokens q [T, H, hd] (hd 64 or 128; fp32, bf16 or fp16; rows
    of q and the caches at multiples of 16 bytes) over their segments' pages, in which
    their own keys and values already are (:func:`paged_append` with the same table, pos
    and cu); H a multiple of the cache's heads.

    The token at position p sees the keys [lo, hi): hi = p + 1, or the first
    ``prefix[b]`` keys of the segment if that is more (int32 [B]; a prefix mask);
    lo = max(0, p - window + 1 (``window`` > 0), ``starts[t]`` (int32 [T], the position
    where the token's document begins)).  Scores are scale * q.k (default
    hd^-1/2), then softcap * tanh(. / softcap) if ``softcap`` > 0, then minus
    ``slopes[h]`` (fp32 [H]) * |p - key|.  A token that sees nothing gets zeros; rows
    behind the last segment keep what ``out`` held.

    ``max_len``: the most keys any segment has (at most 2^30; default: what its table can
    hold); it sizes the launch, so give it where it is known.  A row's bits
    depend on the row's own query, keys and masks alone.
    """
    qs = _heads(q, "q")
    T, H, hd = q.shape
    index, dtype = q.get_device(), q.dtype
    kv, B, width, pp, cp = _pages(k_cache, v_cache, table, pos, cu, T, dtype, index)
    n_pages, Hkv, page, chd = k_cache.shape
    if chd != hd:
        raise ValueError(f"caches of heads of {chd}, queries of {hd}")
    if out is None:
        out = q.new_empty((T, H, hd))
        os_ = (H * hd, hd)
    else:
        os_ = _output(out, "out", q)
    max_len = min(width * page, 2**30) if max_len is None else max_len
    if not (0 <= max_len < 2**31 and 0 <= window < 2**31):  # what the structure's fields hold
        raise ValueError(f"max_len={max_len} and window={window} must be 0 to 2^31 - 1")
    if slopes is not None and (slopes.dtype != torch.float32 or slopes.shape != (H,) or slopes.get_device() != index
                               or not slopes.is_contiguous()):
        raise ValueError(f"slopes must be a contiguous fp32 tensor [{H}] on device {index}")
    def args(ws: int, ws_bytes: int) -> bytes:
        return _lib.PagedAttnArgs.pack(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), table.data_ptr(), pp, cp, sp, xp, lp, ep,
            ws, ws_bytes, T, n_pages, qs[0], qs[1], os_[0], os_[1], kv[0], kv[1], kv[2], scale, softcap,
            B, H, Hkv, hd, page, width, max_len, window, _DT[dtype], 0)

    sp = _index(starts, "starts", T, index) if starts is not None else 0
    xp = _index(prefix, "prefix", B, index) if prefix is not None else 0
    lp = slopes.data_ptr() if slopes is not None else 0
    ep = _err(err, index)
    scale = hd ** -0.5 if scale is None else scale
    a = args(0, 0)
    n = _lib.load().altxs_paged_attn_workspace_bytes(a)
    if n:
        if n < 0:
            _lib.check(int(n), "altxs_paged_attn")
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        a = args(ws.data_ptr(), n)
    _launch("altxs_paged_attn", a, index)
    return out
