"""A KV cache in pages for segments of different lengths.

The dense cache of :class:`altxs_amd.model.StaticState` keeps ``max_len`` rows for
every segment (the reference's StaticKV, src/xsa_ttt/model.py:259-461, a whole
32768-row buffer); here segments take pages of ``page_size`` tokens from one pool as they
grow and give them back when they end.  Page bookkeeping is host work; the
device sees the table :func:`altxs_amd.ops.paged_append` and
:func:`altxs_amd.ops.paged_attn` read.
"""

from __future__ import annotations

import torch

from . import _lib, ops


class PagedKVCache:
    """Pool of ``n_pages`` pages shared by up to ``segments`` segments of at most ``max_len`` tokens.

    ``k``/``v``: [n_pages, num_kv_heads, page_size, head_dim]; ``table``: int32 [segments, pages of
    max_len], -1 where no page is held; ``err``: the device error word.
    """

    def __init__(self, n_pages: int, segments: int, max_len: int, *, num_kv_heads: int, head_dim: int = 64,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size={page_size} must be a power of two from 16 to 1024")
        if n_pages < 1 or segments < 1 or max_len < 1 or num_kv_heads < 1:
            raise ValueError("n_pages, segments, max_len and num_kv_heads must be positive")
        self.page_size, self.segments, self.max_len = page_size, segments, max_len
        dev = torch.device(device)
        self.k = torch.zeros(n_pages, num_kv_heads, page_size, head_dim, dtype=dtype, device=dev)
        self.v = torch.zeros_like(self.k)
        self.table = torch.full((segments, -(-max_len // page_size)), -1, dtype=torch.int32, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        self._free = list(range(n_pages - 1, -1, -1))
        self._held: list[list[int]] = [[] for _ in range(segments)]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def capacity(self, segment: int) -> int:
        """Tokens that ``segment``'s pages hold."""
        return len(self._held[segment]) * self.page_size

    def reserve(self, segment: int, length: int) -> None:
        """Give ``segment`` the pages for ``length`` tokens (those it has stay).  Takes
        none if the pool has too few."""
        if not 0 <= length <= self.max_len:
            raise ValueError(f"length {length} of segments of at most {self.max_len}")
        held = self._held[segment]
        more = -(-length // self.page_size) - len(held)
        if more <= 0:
            return
        if more > len(self._free):
            raise RuntimeError(f"{more} pages needed, {len(self._free)} free")
        new = [self._free.pop() for _ in range(more)]
        self.table[segment, len(held):len(held) + more] = torch.tensor(new, dtype=torch.int32, device=self.table.device)
        held.extend(new)

    def release(self, segment: int) -> None:
        """Give ``segment``'s pages back.  Work already enqueued on the stream of
        its calls still reads them; what takes them next must follow on that stream."""
        self._free.extend(reversed(self._held[segment]))
        self._held[segment] = []
        self.table[segment].fill_(-1)

    def append(self, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, *, cu: torch.Tensor | None = None,
               q: torch.Tensor | None = None, rope=None, interleaved: bool = False,
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """:func:`altxs_amd.ops.paged_append` into this cache; ``rope``: (cos, sin) or None."""
        cos, sin = rope if rope is not None else (None, None)
        return ops.paged_append(k, v, self.k, self.v, self.table, pos, cu=cu, q=q, q_out=q_out, cos=cos, sin=sin,
                                interleaved=interleaved, err=self.err)

    def attend(self, q: torch.Tensor, pos: torch.Tensor, *, cu: torch.Tensor | None = None, max_len: int | None = None,
               **masks) -> torch.Tensor:
        """:func:`altxs_amd.ops.paged_attn` over this cache.  ``max_len`` defaults to the
        longest segment's reserved capacity (a graph captured so holds for that
        capacity: give the bound of its replays)."""
        if max_len is None:
            max_len = min(self.max_len, max(len(h) for h in self._held) * self.page_size)
        return ops.paged_attn(q, self.k, self.v, self.table, pos, cu=cu, max_len=max_len, err=self.err, **masks)

    def check_errors(self) -> None:
        e = int(self.err.item())
        if e:
            raise RuntimeError(f"altxs device error flags 0x{e:x} ({_lib.EDEV_POS} = position outside a segment's "
                               f"pages or the rope table, {_lib.EDEV_PAGE} = page id outside the pool)")
