"""KV4Cache: a paged key/value cache held in 4 bits, and attention over it.

What the target model of a speculative step keeps per request, at 27% of the
size of 16-bit types (136 bytes a token and KV head of width 128, not 512): keys
as e2m1 with a power-of-two scale per 32 channels, values as e2m1 with a float32
scale per token.  ``append`` writes the newest tokens'
keys and values, drafts among them; ``attend`` is the attention of those tokens'
queries, each over everything up to itself; a rejected draft's entries are
simply overwritten by the next ``append``.  No counterpart in the reference.
"""

from __future__ import annotations

import torch

from suffixgpu_amd import _lib
from suffixgpu_amd._lib import (SuffixGPUError, check, count_arg, elsewhere,
                                lib, require_gpu, stream_of)

BLOCK = 32  # tokens


def block_bytes(head_dim: int) -> int:
    """Bytes of 32 tokens of one KV head: 32 (D + D/32 + 4)."""
    return BLOCK * (head_dim + head_dim // 32 + 4)


class KV4Cache:
    """``num_pages`` pages of ``page_size`` tokens (a power of two, 32 to
    65536) for ``num_kv_heads`` heads of width ``head_dim`` (64, 128 or 256),
    for keys, values and queries of type ``dtype`` (bfloat16 or float16).

    ``pages`` [num_pages, num_kv_heads, page_size / 32, block_bytes] uint8 is
    the pool (its layout is in include/suffixgpu_amd.h); an existing one may be
    passed.  Which pages a request holds is the caller's: every call takes
    ``page_table`` [B, W] int32, position p of row b lying in page
    ``page_table[b, p // page_size]``.  Page ids outside [0, num_pages) hold
    nothing: nothing is written there and no query sees them.
    """

    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda",
                 pages: torch.Tensor | None = None):
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if not 32 <= page_size <= 65536 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two in 32..65536")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("dtype must be bfloat16 or float16")
        if num_pages < 0 or not 1 <= num_kv_heads <= 65535:
            raise ValueError("num_pages >= 0 and 1..65535 KV heads")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise SuffixGPUError("KV4Cache needs a ROCm GPU device; there is "
                                 "no CPU path")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.num_pages = int(num_pages)
        self.num_kv_heads = int(num_kv_heads)
        self.head_dim = int(head_dim)
        self.page_size = int(page_size)
        self.dtype = dtype
        shape = (self.num_pages, self.num_kv_heads, self.page_size // BLOCK,
                 block_bytes(self.head_dim))
        if pages is None:
            pages = torch.zeros(shape, dtype=torch.uint8, device=self.device)
        elif (pages.shape != shape or pages.dtype != torch.uint8
              or pages.device != self.device or not pages.is_contiguous()):
            raise ValueError(f"pages must be a contiguous uint8 {list(shape)} "
                             f"tensor on {self.device}")
        elif pages.data_ptr() % 16:
            raise ValueError("pages must be 16-byte aligned")
        self._pages = pages
        # what every call's C view begins with, and workspace bytes by shape
        self._geometry = (pages.data_ptr(), self.num_pages, self.num_kv_heads,
                          self.head_dim, self.page_size,
                          _lib.DTYPE_CODES[dtype])
        self._sizes: dict[tuple, int] = {}

    @property
    def pages(self) -> torch.Tensor:
        """The pool, for as long as the cache lives."""
        return self._pages

    # ------------------------------------------------------------------
    def _view(self, page_table: torch.Tensor, rows: int) -> _lib.SfxKv4:
        if (page_table.dim() != 2 or page_table.dtype is not torch.int32
                or page_table.device != self.device):
            self._refuse_table(page_table, rows)
        n, width = page_table.shape
        s0, s1 = page_table.stride()
        if n != rows or (s1 != 1 and width > 1):
            self._refuse_table(page_table, rows)
        return _lib.SfxKv4(*self._geometry, page_table.data_ptr(), width, s0)

    def _refuse_table(self, page_table, rows):
        require_gpu(page_table)
        raise ValueError(f"page_table must be an int32 [{rows}, W] tensor on "
                         f"{self.device} with contiguous rows")

    def _heads(self, name: str, x: torch.Tensor, heads: int | None = None):
        """The C view of x [B, T, heads, head_dim], and B, T, heads."""
        if x.dim() == 4 and x.dtype is self.dtype and x.device == self.device:
            b, t, h, d = x.shape
            sb, st, sh, sd = x.stride()
            if (d == self.head_dim and sd == 1
                    and (heads is None or h == heads)):
                return _lib.SfxHeads(x.data_ptr(), sb, st, sh), b, t, h
        require_gpu(x)
        raise ValueError(
            f"{name} must be a {self.dtype} [B, T, heads, {self.head_dim}] "
            f"tensor on {self.device}, contiguous along the last dimension"
            + (f", with {heads} heads" if heads is not None else ""))

    def _counts(self, name: str, t: torch.Tensor | None, rows: int,
                optional: bool = False):
        """(tensor to keep, address, is64) of a vector of counts."""
        if t is None and optional:
            return None, None, 0
        if t is None:
            raise ValueError(f"{name} is needed")
        if t.dim() != 1 or t.shape[0] != rows or t.device != self.device:
            require_gpu(t)
            raise ValueError(f"{name} must hold {rows} integers on "
                             f"{self.device}")
        t, is64 = count_arg(t)
        return t, t.data_ptr(), is64

    def append(self, k: torch.Tensor, v: torch.Tensor,
               page_table: torch.Tensor, start: torch.Tensor,
               count: torch.Tensor | None = None) -> None:
        """Write tokens i < ``count[b]`` (all without it) of ``k`` and ``v``
        [B, T, num_kv_heads, head_dim] at positions ``start[b] + i``.

        A page that one row of a call writes must not be written by another
        row of it.  Infinities and NaN make their 32 channels of a key, or
        their token's values, NaN."""
        if elsewhere(self.device):
            with torch.cuda.device(self.device):
                return self.append(k, v, page_table, start, count)
        kh, b, t, _ = self._heads("k", k, self.num_kv_heads)
        vh, vb, vt, _ = self._heads("v", v, self.num_kv_heads)
        if b != vb or t != vt:
            raise ValueError("k and v differ in shape")
        view = self._view(page_table, b)
        keep = (self._counts("start", start, b),
                self._counts("count", count, b, optional=True))
        if b == 0 or t == 0:
            return
        check(lib().sfx_kv4_append(view, kh, vh, b, t, *keep[0][1:],
                                   *keep[1][1:], stream_of(self.device)),
              "KV4Cache.append")

    def read(self, page_table: torch.Tensor, start: torch.Tensor,
             tokens: int, count: torch.Tensor | None = None):
        """The keys and values [B, tokens, num_kv_heads, head_dim] that the
        cache holds at positions ``start[b] + i``, i < ``count[b]``; zeros
        elsewhere."""
        if elsewhere(self.device):
            with torch.cuda.device(self.device):
                return self.read(page_table, start, tokens, count)
        b = page_table.shape[0]
        view = self._view(page_table, b)
        keep = (self._counts("start", start, b),
                self._counts("count", count, b, optional=True))
        shape = (b, int(tokens), self.num_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=self.dtype, device=self.device)
        v = torch.empty(shape, dtype=self.dtype, device=self.device)
        if b == 0 or tokens == 0:
            return k, v
        check(lib().sfx_kv4_read(view, b, int(tokens), *keep[0][1:],
                                 *keep[1][1:], k.data_ptr(), v.data_ptr(),
                                 stream_of(self.device)), "KV4Cache.read")
        return k, v

    def attend(self, q: torch.Tensor, page_table: torch.Tensor,
               kv_len: torch.Tensor, q_len: torch.Tensor | None = None,
               scale: float | None = None) -> torch.Tensor:
        """Attention of the newest tokens' queries ``q`` [B, T, q_heads,
        head_dim] over the cache.

        Row b holds ``kv_len[b]`` tokens (as appended, the new ones included);
        its last ``q_len[b]`` (T without it) are q's tokens 0 .. q_len - 1, and
        query i sees the positions up to its own, kv_len - q_len + i.  Both
        count tokens past the table's end, which no query sees (``append``
        drops them), and q_len may be more than T.  q_heads is a multiple of
        num_kv_heads, consecutive query heads sharing a KV head.  ``scale``
        defaults to head_dim ** -0.5.  Returns [B, T, q_heads, head_dim] in the
        cache's type: zeros for a query that sees nothing and for tokens from
        q_len on.  T = 1 is a decode step, T = k + 1 a verification step, a
        long T a chunk of a prompt."""
        if elsewhere(self.device):
            with torch.cuda.device(self.device):
                return self.attend(q, page_table, kv_len, q_len, scale)
        qh, b, t, heads = self._heads("q", q)
        if heads < 1 or heads % self.num_kv_heads:
            raise ValueError(f"{heads} query heads do not share "
                             f"{self.num_kv_heads} KV heads evenly")
        view = self._view(page_table, b)
        keep = (self._counts("kv_len", kv_len, b),
                self._counts("q_len", q_len, b, optional=True))
        if scale is None:
            scale = self.head_dim ** -0.5
        out = torch.empty(b, t, heads, self.head_dim, dtype=self.dtype,
                          device=self.device)
        if b == 0 or t == 0:
            return out
        L = lib()
        key = (b, t, heads, view.table_width)
        nbytes = self._sizes.get(key)
        if nbytes is None:
            nbytes = self._sizes[key] = L.sfx_kv4_attend_workspace_size(
                view, b, t, heads)
        ws = (torch.empty(nbytes, dtype=torch.uint8, device=self.device)
              if nbytes else None)
        check(L.sfx_kv4_attend(view, qh, b, t, heads, *keep[0][1:],
                               *keep[1][1:], scale, out.data_ptr(),
                               None if ws is None else ws.data_ptr(), nbytes,
                               stream_of(self.device)), "KV4Cache.attend")
        return out
