"""The paged key/value cache in 4 bits, and attention over it.

A serving loop around this package's constraint step checks a block of drafted
tokens per request in one pass of its model: :meth:`PagedKV4.append` rotates
the block's keys (and queries) to their positions and appends keys and values
to the cache, :meth:`PagedKV4.attend` is the block's attention over the cache,
and :meth:`bpdecode_amd.batch.ConstraintBatch.verify` decides on the drafts.
A prompt is a long block, a plain decoding step a block of one token.
:meth:`PagedKV4.attend_shared` is the attention of requests that begin with the
same prompt, read once for all of them.

An element takes 4.25 bits: an e2m1 code, and one power of two for 32
neighbouring channels (the OCP microscaling layout of 4-bit floats, scales
chosen so that the largest channel is never cut by more than a rounding; in
float16 magnitudes past 57,344 are, and kept as 49,152).
``include/bpdecode_hip.h`` states the bytes of a page.  Tensors on the device
run the HIP kernels on torch's current stream, CPU tensors the library's host
entry points.  The cache keeps no lengths: the caller says where each request
stands, so a block whose drafts were refused is overwritten by the next one.
Nothing here has a gradient.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import check, lib, ptr

HEAD_DIMS = (64, 96, 128, 192, 256)
GROUP = 32  # channels that share a scale

_CODES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


def block_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one page of one key/value head."""
    return page_size * (head_dim + 2 * (head_dim // GROUP))


class PagedKV4:
    """A pool of cache pages: uint8 ``pages`` [num_pages, kv_heads,
    ``block_bytes(page_size, head_dim)``], contiguous, for keys and values of
    ``dtype`` (float16 or bfloat16: what goes in and comes out).  ``page_size``
    is a power of two from 16 to 256, ``head_dim`` one of ``HEAD_DIMS``.

    ``block_table`` int32 [requests, blocks] names the pages of each request:
    its token p lies in page ``block_table[b, p // page_size]``.  Positions and
    pages outside their tables are left out (not written, not attended, read
    as zeros) and noted in ``err`` (int32 [1], optional): ``check_errors``
    raises on them."""

    def __init__(self, pages: torch.Tensor, page_size: int, head_dim: int, dtype: torch.dtype,
                 err: torch.Tensor | None = None) -> None:
        code = _CODES.get(dtype)
        if code is None:
            raise RuntimeError(f"the cache takes float16 or bfloat16, got {dtype}")
        if head_dim not in HEAD_DIMS:
            raise RuntimeError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if not 16 <= page_size <= 256 or page_size & (page_size - 1):
            raise RuntimeError(f"page_size must be a power of two from 16 to 256, got {page_size}")
        want = block_bytes(page_size, head_dim)
        if pages.dtype != torch.uint8 or pages.dim() != 3 or pages.shape[2] != want or not pages.is_contiguous():
            raise RuntimeError(f"pages must be contiguous uint8 [num_pages, kv_heads, {want}]")
        if pages.shape[1] < 1:
            raise RuntimeError("the cache needs at least one head")
        _lib.err_ptr(err, pages.device)
        self.pages, self.page_size, self.head_dim, self.dtype, self.err = pages, page_size, head_dim, dtype, err
        self.num_pages, self.kv_heads = pages.shape[0], pages.shape[1]
        self.device = pages.device
        self._on_dev = self.device.type == "cuda"
        self._head = (pages.data_ptr(), self.num_pages, page_size, self.kv_heads, head_dim, code)

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype,
              device) -> PagedKV4:
        """A pool of ``num_pages`` pages, all zeros, with an error word."""
        pages = torch.zeros((num_pages, kv_heads, block_bytes(page_size, head_dim)), dtype=torch.uint8, device=device)
        return cls(pages, page_size, head_dim, dtype, torch.zeros(1, dtype=torch.int32, device=pages.device))

    # --- arguments ---------------------------------------------------------
    def _block(self, x: torch.Tensor, name: str, heads: int | None = None) -> tuple[torch.Tensor, tuple]:
        """``x`` with its channels next to each other, and its address and strides."""
        shape = x.shape
        if len(shape) != 4 or shape[3] != self.head_dim or (heads is not None and shape[2] != heads):
            raise RuntimeError(f"{name} must be [requests, tokens, {heads or 'heads'}, {self.head_dim}], "
                               f"got {list(shape)}")
        if x.dtype is not self.dtype or x.device != self.device:
            raise RuntimeError(f"{name} must be {self.dtype} on {self.device}, got {x.dtype} on {x.device}")
        a, b, c, d = x.stride()
        if d != 1:
            x = x.contiguous()
            a, b, c, d = x.stride()
        return x, (x.data_ptr(), a, b, c)

    def _table(self, block_table: torch.Tensor, rows: int) -> tuple[torch.Tensor, tuple]:
        shape = block_table.shape
        if len(shape) != 2 or shape[0] != rows:
            raise RuntimeError(f"block_table must be [{rows}, blocks], got {list(shape)}")
        if block_table.dtype is not torch.int32 or block_table.device != self.device:
            raise RuntimeError(f"block_table must be int32 on {self.device}")
        n = shape[1]
        ld, unit = block_table.stride()
        if n > 1 and unit != 1 or rows > 1 and ld < n:
            block_table = block_table.contiguous()
            ld = n
        return block_table, (block_table.data_ptr(), ld if rows > 1 else n, n)

    def _per_request(self, x: torch.Tensor | None, name: str, rows: int) -> torch.Tensor | None:
        if x is None:
            return None
        if x.dtype is not torch.int32 or x.dim() != 1 or x.shape[0] != rows or x.device != self.device:
            raise RuntimeError(f"{name} must be int32 [{rows}] on {self.device}")
        return x if rows <= 1 or x.stride(0) == 1 else x.contiguous()

    # --- operators -----------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, starts: torch.Tensor, *,
               counts: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
               interleaved: bool = False, q: torch.Tensor | None = None, positions: torch.Tensor | None = None,
               axes: torch.Tensor | None = None) -> torch.Tensor | None:
        """Append ``k`` and ``v`` [requests, tokens, kv_heads, head_dim]: token
        i < ``counts[b]`` (all without ``counts``) of request b at position
        ``starts[b] + i``, over whatever was there.  With ``cos`` and ``sin``
        (float32 [positions, R / 2], R <= head_dim) the first R channels of
        ``k`` and of ``q`` [requests, tokens, heads, head_dim] are rotated to
        that position first, in float32: channel pairs (j, j + R / 2), or
        (2j, 2j + 1) with ``interleaved``.  Returns the rotated ``q`` (zeros
        past ``counts[b]``), None without ``q``.  Two requests must not append
        to one page in one call.

        With ``positions`` (int32 [axes, requests, tokens], up to 4 axes, or
        [requests, tokens]) the rotation goes by them, not by the place in the
        cache: pair j by the position on axis ``axes[j]`` (int32 [R / 2]; all
        on the first without it), as models place the patches of images and
        video by time, height and width.  A token with a position outside the
        rotation's tables is left out."""
        k, ks = self._block(k, "k", self.kv_heads)
        v, vs = self._block(v, "v", self.kv_heads)
        B, T, _, _ = k.shape
        if v.shape != k.shape:
            raise RuntimeError(f"k and v differ in shape: {list(k.shape)} and {list(v.shape)}")
        block_table, table = self._table(block_table, B)
        starts, counts = self._per_request(starts, "starts", B), self._per_request(counts, "counts", B)
        rotary = rows = 0
        if (cos is None) != (sin is None):
            raise RuntimeError("the rotation needs both cos and sin")
        if cos is not None:
            if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype is not torch.float32 \
                    or sin.dtype is not torch.float32 or cos.device != self.device or sin.device != self.device:
                raise RuntimeError(f"cos and sin must be float32 [positions, R / 2] on {self.device}")
            cos, sin = cos.contiguous(), sin.contiguous()
            rows, rotary = cos.shape
            rotary *= 2
            if rotary > self.head_dim:
                raise RuntimeError(f"{rotary} rotated channels in heads of {self.head_dim}")
        on_axes = ()
        if positions is not None:
            if cos is None:
                raise RuntimeError("positions need the rotation's cos and sin")
            if positions.dim() == 2:
                positions = positions[None]
            if positions.dim() != 3 or positions.shape[1:] != (B, T) or not 1 <= positions.shape[0] <= _lib.MAX_AXES \
                    or positions.dtype is not torch.int32 or positions.device != self.device:
                raise RuntimeError(f"positions must be int32 [1 to {_lib.MAX_AXES} axes, {B}, {T}] on {self.device}")
            if axes is not None:
                if axes.dtype is not torch.int32 or axes.shape != cos.shape[1:] or axes.device != self.device:
                    raise RuntimeError(f"axes must be int32 [{cos.shape[1]}] on {self.device}")
                axes = axes.contiguous()
            elif positions.shape[0] > 1:
                raise RuntimeError("positions on several axes need the axis of each channel pair")
            on_axes = (positions.data_ptr(), *positions.stride(), positions.shape[0], ptr(axes)) if cos.shape[1] else ()
        elif axes is not None:
            raise RuntimeError("axes need positions")
        out, heads, qs = None, 0, (None, 0, 0, 0)
        if q is not None:
            q, qs = self._block(q, "q")
            if q.shape[:2] != k.shape[:2]:
                raise RuntimeError(f"q and k differ in requests or tokens: {list(q.shape)} and {list(k.shape)}")
            heads = q.shape[2]
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        args = (*self._head, *ks, *vs, *qs, heads, ptr(out), B, T, *table, ptr(starts), ptr(counts), ptr(cos), ptr(sin),
                rows, rotary, int(interleaved), *on_axes, ptr(self.err))
        if self._on_dev:
            append = lib().bpd_kv_append_axes if on_axes else lib().bpd_kv_append
            check(append(*args, _lib.stream_of(self.device)))
        else:
            append = lib().bpd_host_kv_append_axes if on_axes else lib().bpd_host_kv_append
            check(append(*args))
        return out

    def read(self, block_table: torch.Tensor, starts: torch.Tensor, tokens: int, *,
             counts: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys (rotated, as appended) and values of tokens ``starts[b] + i``,
        i < ``tokens``, as [requests, tokens, kv_heads, head_dim] each; zeros
        past ``counts[b]``.  Exact: what the cache holds is representable."""
        B = starts.shape[0] if starts.dim() == 1 else -1
        block_table, table = self._table(block_table, B)
        starts, counts = self._per_request(starts, "starts", B), self._per_request(counts, "counts", B)
        k = self.pages.new_empty((B, tokens, self.kv_heads, self.head_dim), dtype=self.dtype)
        v = torch.empty_like(k)
        args = (*self._head, k.data_ptr(), v.data_ptr(), B, tokens, *table, ptr(starts), ptr(counts), ptr(self.err))
        if self._on_dev:
            check(lib().bpd_kv_read(*args, _lib.stream_of(self.device)))
        else:
            check(lib().bpd_host_kv_read(*args))
        return k, v

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *,
               query_lens: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
        """``softmax(scale q k^T) v`` over the cache for a block of queries
        ``q`` [requests, tokens, heads, head_dim] (rotated) whose keys are
        appended: of n = ``query_lens[b]`` (``tokens`` without it) queries,
        query i sees the request's first ``lengths[b] - n + 1 + i`` tokens,
        ``lengths`` counting the block itself.  Query head h reads key head
        ``h // (heads // kv_heads)``; ``scale`` defaults to 1 / sqrt(head_dim).
        Zeros where a query sees nothing and past n."""
        q, qs = self._block(q, "q")
        B, T, H, D = q.shape
        if H < 1 or H % self.kv_heads:
            raise RuntimeError(f"query heads ({H}) must be a multiple of the cache's heads ({self.kv_heads})")
        block_table, table = self._table(block_table, B)
        lengths, query_lens = self._per_request(lengths, "lengths", B), self._per_request(query_lens, "query_lens", B)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        args = (*self._head, *qs, H, out.data_ptr(), B, T, *table, ptr(lengths), ptr(query_lens),
                D ** -0.5 if scale is None else float(scale))
        if self._on_dev:
            need = lib().bpd_kv_attend_workspace_bytes(B, T, H, self.kv_heads, D, table[2] * self.page_size)
            ws = self.pages.new_empty(need) if need else None
            check(lib().bpd_kv_attend(*args, ptr(ws), need, ptr(self.err), _lib.stream_of(self.device)))
        else:
            check(lib().bpd_host_kv_attend(*args, ptr(self.err)))
        return out

    def attend_shared(self, q: torch.Tensor, prefix_table: torch.Tensor, shared: int | torch.Tensor,
                      block_table: torch.Tensor, lengths: torch.Tensor, *, query_lens: torch.Tensor | None = None,
                      scale: float | None = None) -> torch.Tensor:
        """:meth:`attend` for a batch whose requests begin with the same
        ``shared`` tokens (a number, or int32 [1] on the device), which are
        attended to once for all of them.  Those, cut to whole pages, lie in the
        pages of ``prefix_table`` int32 [blocks]; ``block_table`` and ``lengths``
        are those of the whole requests, as :meth:`append` and :meth:`attend`
        take them (a table's entries before the shared pages' end are not
        read).  The result is :meth:`attend`'s with the shared pages first in
        every request's table, and where prompt or batch are small that is the
        faster call: single tokens of 32 heads, 8 of 128 in the cache, gain from
        4 requests behind 8,000 tokens (25 us there, 20 here) and 128 behind
        2,000 (43 and 39; of 128 behind 32,768 508 and 102), and lose behind 500
        (128 requests 21 and 37); blocks of 100 tokens are even behind 8,000."""
        q, qs = self._block(q, "q")
        B, T, H, D = q.shape
        if H < 1 or H % self.kv_heads:
            raise RuntimeError(f"query heads ({H}) must be a multiple of the cache's heads ({self.kv_heads})")
        block_table, table = self._table(block_table, B)
        lengths, query_lens = self._per_request(lengths, "lengths", B), self._per_request(query_lens, "query_lens", B)
        if prefix_table.dim() != 1 or prefix_table.dtype is not torch.int32 or prefix_table.device != self.device:
            raise RuntimeError(f"prefix_table must be int32 [blocks] on {self.device}")
        prefix_table = prefix_table.contiguous()
        blocks, count = prefix_table.shape[0], 0
        if isinstance(shared, torch.Tensor):
            if shared.dtype is not torch.int32 or shared.numel() != 1 or shared.device != self.device:
                raise RuntimeError(f"shared must be a number or int32 [1] on {self.device}")
        else:
            shared, count = None, shared
            if not 0 <= count <= blocks * self.page_size:
                raise RuntimeError(f"{count} shared tokens in a prefix of {blocks} pages of {self.page_size}")
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        args = (*self._head, *qs, H, out.data_ptr(), B, T, ptr(prefix_table), blocks, ptr(shared), count, *table,
                ptr(lengths), ptr(query_lens), D ** -0.5 if scale is None else float(scale))
        if self._on_dev:
            need = lib().bpd_kv_attend_shared_workspace_bytes(B, T, H, self.kv_heads, D, table[2] * self.page_size,
                                                              blocks * self.page_size)
            ws = self.pages.new_empty(need)
            check(lib().bpd_kv_attend_shared(*args, ptr(ws), need, ptr(self.err), _lib.stream_of(self.device)))
        else:
            check(lib().bpd_host_kv_attend_shared(*args, ptr(self.err)))
        return out

    def check_errors(self) -> None:
        """Raise if a call met a position or page outside its tables since the
        last check (synchronises with the device)."""
        if self.err is not None and int(self.err.item()):
            self.err.zero_()
            raise IndexError("a position or page outside the cache, its block table or the rotation's tables")
