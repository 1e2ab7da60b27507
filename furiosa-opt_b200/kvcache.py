"""Rotary positions and the paged 4-bit key / value cache: what a decoder keeps between the tokens that it
answers with. The operators are `B200.rotary`, `B200.cache_append`, `B200.cache_read` and
`B200.cache_attention`; `workloads.DecoderBlockW8A8.step` runs them in a block.

    rope = Rope.scaled(128, base=500000.0, scaling="by_parts", factor=8.0, original_length=8192)
    cache = PagedCache(be, pages=1024, page_size=64, heads=8)
    step = CacheBatch(be, cache, q_lens=[512, 1], kv_lens=[512, 4097], pages=[[...], [...]])
    be.rotary(q, step.positions, rope, heads=32, out=q)
    be.cache_append(cache, k, v, step.slots, positions=step.positions, rope=rope)
    o = be.cache_attention(q, cache, step.table, step.q_start, step.kv_len, heads=32)
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

import numpy as np

from . import _lib
from ._lib import check

ROPE_LAYOUTS = {"half": 0, "interleaved": 1}
GROUP = 32  # channels that share a step and an offset


class Rope:
    """A rotation plan: the angle per position (radians) of each pair of a head's channels. `layout`
    "half" pairs channel p with p + len(inv_freq), "interleaved" 2 p with 2 p + 1; a head's channels past
    the pairs are not rotated. `magnitude` scales the rotated channels. Belongs to no device."""

    def __init__(self, inv_freq: Sequence[float], layout: str = "half", magnitude: float = 1.0):
        if layout not in ROPE_LAYOUTS:
            raise ValueError(f"Rope: layout {layout!r} is none of {sorted(ROPE_LAYOUTS)}")
        self.inv_freq = [float(f) for f in inv_freq]
        self.layout, self.magnitude = layout, float(magnitude)
        self.rot_dim = 2 * len(self.inv_freq)
        h = C.c_void_p()
        check(_lib.lib().fopt_rope_create((C.c_double * max(len(self.inv_freq), 1))(*self.inv_freq),
                                          len(self.inv_freq), ROPE_LAYOUTS[layout], self.magnitude, C.byref(h)))
        self._h = h

    @classmethod
    def scaled(cls, rot_dim: int, base: float = 10000.0, layout: str = "half", scaling: Optional[str] = None,
               factor: float = 1.0, original_length: int = 0, low: float = 1.0, high: float = 32.0,
               magnitude: float = 1.0) -> "Rope":
        """Frequencies base^(-2 p / rot_dim), stretched for contexts `factor` times as long:
        "linear" divides every frequency by the factor; "ntk" raises the base so that the lowest
        frequency is divided by it and the highest kept; "by_parts" keeps the pairs that turn more than
        `high` times within `original_length` positions, divides those that turn less than `low` times, and
        blends in between by the number of turns."""
        if rot_dim <= 0 or rot_dim % 2:
            raise ValueError("Rope: an even number of rotated channels")
        if scaling not in (None, "linear", "ntk", "by_parts"):
            raise ValueError(f"Rope: unknown scaling {scaling!r}")
        if not factor > 0 or not base > 0:
            raise ValueError("Rope: base and factor must be positive")
        if scaling == "ntk":
            base = base * factor ** (rot_dim / max(rot_dim - 2, 1))
        f = [base ** (-2.0 * p / rot_dim) for p in range(rot_dim // 2)]
        if scaling == "linear":
            f = [x / factor for x in f]
        elif scaling == "by_parts":
            if original_length <= 0 or not high > low:
                raise ValueError("Rope: by_parts needs original_length and high > low")
            keep = [min(max((original_length * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
            f = [x / factor * (1 - k) + x * k for x, k in zip(f, keep)]
        return cls(f, layout, magnitude)

    @property
    def handle(self):
        return self._h

    def __del__(self):
        try:
            if self._h:
                _lib.lib().fopt_rope_free(self._h)
        except Exception:
            pass


class PagedCache:
    """Keys and values of any number of sequences, 4 bits each in groups of 32 channels with a bf16
    (step, offset): `pages` pages of `page_size` slots for `heads` heads of `head_dim` channels. The four
    images are ordinary storages, laid out as `k_map`, `v_map` and `scale_map` say."""

    def __init__(self, be, pages: int, page_size: int, heads: int, head_dim: int = 128):
        from .backend import Mapping, Storage
        if head_dim not in (64, 128, 256):
            raise ValueError("PagedCache: head_dim must be 64, 128 or 256")
        if page_size <= 0 or page_size % 16 or page_size > 65536:
            raise ValueError("PagedCache: page_size must be a multiple of 16, at most 65536")
        if pages <= 0 or heads <= 0 or pages * page_size > 2 ** 31 - 1:
            raise ValueError("PagedCache: empty, or slots past 2^31")
        self.be, self.pages, self.page_size, self.heads, self.head_dim = be, pages, page_size, heads, head_dim
        ax = dict(P=pages, H=heads, S=page_size, D=head_dim, G=head_dim // GROUP, C=2)
        self.k_map = Mapping("[P, H, S, D % 32 / 8, D / 32, D % 8]", ax)
        self.v_map = Mapping("[P, H, S, D % 32 / 4, D / 32, D % 4]", ax)
        self.scale_map = Mapping("[P, H, S, G, C]", ax)
        n = pages * heads * page_size * head_dim
        self.k, self.v = Storage(be, "i4", n), Storage(be, "i4", n)
        self.k_scale, self.v_scale = Storage(be, "bf16", n // GROUP * 2), Storage(be, "bf16", n // GROUP * 2)

        self._images = self.k, self.v, self.k_scale, self.v_scale
        self._desc = _lib.PagedCacheDesc(*(s.addr for s in self._images), pages, page_size, heads, head_dim)
        self.ref = C.byref(self._desc)  # what the entry points take

    @property
    def slots(self) -> int:
        return self.pages * self.page_size

    def _will_write(self) -> None:
        for s in self._images:
            s._will_write()


class CacheBatch:
    """The device arrays of one step over a cache: sequence b brings q_lens[b] new tokens, after which it
    holds kv_lens[b] keys in the pages pages[b]. `tokens` (at least the sum of q_lens) pads the step to
    a fixed size: the rows behind the last sequence are no tokens. `rewrite` puts another step of the same
    shape into the same storages, for a captured graph to replay."""

    def __init__(self, be, cache: PagedCache, q_lens: Sequence[int], kv_lens: Sequence[int],
                 pages: Sequence[Sequence[int]], tokens: Optional[int] = None, table_width: Optional[int] = None):
        from .backend import Storage
        self.be, self.cache = be, cache
        self.batch = len(q_lens)
        self.tokens = int(sum(q_lens)) if tokens is None else int(tokens)
        self.table_width = max([1, *map(len, pages)]) if table_width is None else int(table_width)
        host = self._arrays(q_lens, kv_lens, pages)
        for name, a in host.items():
            setattr(self, name, Storage(be, "i32", a.size))
        self._upload(host)

    def _arrays(self, q_lens, kv_lens, pages):
        c = self.cache
        if not (len(q_lens) == len(kv_lens) == len(pages) == self.batch) or not self.batch:
            raise ValueError("CacheBatch: q_lens, kv_lens and pages name the same sequences, one at least")
        if sum(q_lens) > self.tokens:
            raise ValueError("CacheBatch: more new tokens than the step has rows")
        if self.tokens <= 0:
            raise ValueError("CacheBatch: no tokens")
        positions, slots = np.zeros(self.tokens, np.int32), np.full(self.tokens, -1, np.int32)
        table = np.full((self.batch, self.table_width), -1, np.int32)
        at = 0
        for b, (q, n, p) in enumerate(zip(q_lens, kv_lens, pages)):
            if not 0 <= q <= n:
                raise ValueError("CacheBatch: a sequence's keys count its new tokens")
            if len(p) > self.table_width or n > len(p) * c.page_size:
                raise ValueError("CacheBatch: a sequence's pages do not hold its keys, or exceed the table")
            p = np.asarray(p, np.int64)
            if p.size and (p.min() < 0 or p.max() >= c.pages):
                raise ValueError("CacheBatch: a page number outside the cache")
            table[b, :p.size] = p
            i = np.arange(n - q, n)
            positions[at:at + q] = i
            slots[at:at + q] = p[i // c.page_size] * c.page_size + i % c.page_size if q else 0
            at += q
        live = slots[slots >= 0]
        if np.unique(live).size != live.size:
            raise ValueError("CacheBatch: two new tokens share a slot")
        return dict(positions=positions, slots=slots, table=table.reshape(-1),
                    q_start=np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32),
                    kv_len=np.asarray(kv_lens, np.int32))

    def _upload(self, host):
        for name, a in host.items():
            s = getattr(self, name)
            s._will_write()
            check(_lib.lib().fopt_h2d(self.be.ctx, s.ptr, a.ctypes.data, a.nbytes), self.be.ctx)
        self.be.sync()  # the host arrays go away

    def rewrite(self, q_lens, kv_lens, pages) -> None:
        self._upload(self._arrays(q_lens, kv_lens, pages))
