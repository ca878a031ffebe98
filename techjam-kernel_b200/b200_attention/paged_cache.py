"""Paged key/value cache on the B200 (``include/b200_paged.h``).

A cache is two pools of pages, ``k_pages`` and ``v_pages``
``[layers, pages, kv_heads, page_size, head_dim]`` (or, for one layer, without the
first dimension), and its bookkeeping in device memory:

* ``page_table`` int32 ``[batch, slots]``: the page in each slot of a sequence, -1
  for none.  Token ``i`` lies in row ``i % page_size`` of slot ``i // page_size``;
* ``seq_lens`` int32 ``[batch]``: committed tokens.  Drafted tokens (one, or a
  tree of them) lie directly behind the committed ones until they are accepted;
* ``page_refs`` int32 ``[pages]``: how many sequences hold a page (0: free).

Pools of uint8 hold the cache in 4 bits (``include/b200_cache4.h``): a row of 48 bytes
(``head_dim`` up to 64) or 80 (up to 128) stands for a vector in four groups, each number
``low + step * code``.  ``b200_cache_append`` rounds vectors into such rows,
``b200_tree_attention`` reads them, ``b200_cache_read`` gives the numbers back, and the page
operations move the rows as they are.

One decode step is ``b200_cache_reserve`` (pages for the tokens to come, copy on
write), for every layer ``b200_cache_append`` and ``b200_tree_attention``, and
``b200_cache_accept`` (keep the accepted path).  ``b200_cache_fork``,
``b200_cache_free`` and ``b200_cache_compact`` share, release and gather pages.
Every call is launched on the current stream, none waits for the host, and all
work in place on the tensors given, so a step can be captured in a CUDA graph.
Results do not depend on execution order: free pages are given out lowest
number first, in (sequence, slot) order.

Inference only: tensors that ask for gradients are refused.
Shapes, types and devices are checked on the host (``ValueError`` / ``TypeError``).
Page numbers, lengths and sequence numbers lie on the device; a bad one skips its
access there and is reported like every device error of this package (the next
launch raises ``DeviceError``).  ``PagedKVCache`` keeps the tensors together.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _native
from .fused_attention import (DeviceError, _attention_op, _describe, _error_word_address,
                              device_error_word)

_ops = None


def _load():
    global _ops
    _attention_op()  # loads the library; raises when it has not been built
    _ops = torch.ops.b200
    return _ops


def _call(name: str, device: torch.device, *args):
    """``torch.ops.b200.<name>`` on the current stream, with this package's exceptions."""
    ops = _ops if _ops is not None else _load()
    try:
        return getattr(ops, name)(*args, _error_word_address(device))
    except RuntimeError as exc:
        if str(exc).startswith("b200 device error"):
            value = int(device_error_word(device)[0])
            raise DeviceError(f"b200_{name} refused to launch: an earlier kernel on {device} "
                              f"reported a {_describe(value)}; its output is undefined "
                              "(clear_device_errors resumes launches)") from None
        raise


def b200_cache_append(k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor,
                      v_pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                      draft_lens: Optional[torch.Tensor] = None) -> None:
    """Write ``k_new``/``v_new`` ``[(layers,) batch, kv_heads, tokens, head_dim]`` (any
    strides, last dimension contiguous) as tokens ``seq_lens[b] + j`` of each
    sequence; with ``draft_lens`` int32 ``[batch]`` only rows ``j < draft_lens[b]``.

    Into a 4-bit cache (uint8 pools) go vectors of bfloat16, float16 or float32: each quarter
    of a vector padded to 64 or 128 has a ``low``, the bfloat16 number at or below its smallest, a
    ``step``, that at or above a fifteenth of the way from it to the largest, and codes
    ``(x - low) / step`` rounded to nearest, ties to even.  A number is off by half a step at
    most; a group that holds an infinity or NaN, or whose numbers lie further apart than the
    largest float32, reads as NaN."""
    _call("cache_append", k_pages.device, k_new, v_new, k_pages, v_pages, page_table, seq_lens,
          draft_lens)


def b200_cache_read(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    starts: torch.Tensor, tokens: int, head_dim: int,
                    dtype: torch.dtype = torch.bfloat16,
                    counts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that a 4-bit cache holds for tokens ``starts[b] + j``, ``j <
    tokens`` (``starts`` int32 ``[batch]``), as ``dtype`` tensors ``[(layers,) batch, kv_heads,
    tokens, head_dim]``, each number rounded once.  With ``counts`` int32 ``[batch]`` only rows
    ``j < counts[b]`` are read, and the others are zero."""
    return _call("cache_read", k_pages.device, k_pages, v_pages, page_table, starts, tokens,
                 head_dim, dtype, counts)


def b200_cache_accept(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                      seq_lens: torch.Tensor, paths: torch.Tensor,
                      counts: torch.Tensor) -> torch.Tensor:
    """Keep ``counts[b]`` drafted tokens of each sequence: drafted token
    ``paths[b, j]`` (int32 ``[batch, width]``, strictly increasing in ``j``) moves to
    token ``seq_lens[b] + j`` in all layers.  Returns the new lengths
    ``seq_lens + counts``; ``seq_lens`` itself is left as it is."""
    return _call("cache_accept", k_pages.device, k_pages, v_pages, page_table, seq_lens, paths,
                 counts)


def b200_cache_reserve(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                       seq_lens: torch.Tensor, page_refs: torch.Tensor,
                       tokens: Union[int, torch.Tensor]) -> torch.Tensor:
    """Give each sequence pages of its own for its next ``tokens`` (one number for
    all, or int32 ``[batch]``; 0 leaves a sequence alone): empty slots get a free
    page, slots whose page is shared too, with the committed rows of such a page
    copied.  All or nothing: returns an int32 ``[1]`` status on the device, 0 when
    done; with ``NO_PAGES`` (too few free pages), ``ROW_FULL`` (a sequence does not
    fit its slots) or ``BAD_ENTRY`` (a page number or length out of range) nothing
    was changed."""
    given = isinstance(tokens, torch.Tensor)
    return _call("cache_reserve", k_pages.device, k_pages, v_pages, page_table, seq_lens,
                 page_refs, tokens if given else None, 0 if given else int(tokens))


def b200_cache_fork(page_table: torch.Tensor, seq_lens: torch.Tensor, page_refs: torch.Tensor,
                    src: torch.Tensor, dst: torch.Tensor, page_size: int) -> None:
    """Sequence ``dst[i]`` lets go of its pages and becomes a copy of ``src[i]`` that
    shares its pages (int32 ``[n]`` each; no ``dst`` is named twice or is a ``src``).
    Rows are copied only when one of the two is written (``b200_cache_reserve``)."""
    _call("cache_fork", page_table.device, page_table, seq_lens, page_refs, src, dst, page_size)


def b200_cache_free(page_table: torch.Tensor, seq_lens: torch.Tensor, page_refs: torch.Tensor,
                    rows: torch.Tensor) -> None:
    """Sequences ``rows`` (int32 ``[n]``) let go of their pages; their length becomes 0."""
    _call("cache_free", page_table.device, page_table, seq_lens, page_refs, rows)


def b200_cache_compact(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                       page_refs: torch.Tensor) -> torch.Tensor:
    """Close the gaps in the pools: with n pages held, the i-th held page at or past
    place n moves to the i-th free place before n, and ``page_table`` and
    ``page_refs`` follow.  Returns n as an int32 ``[1]`` on the device."""
    return _call("cache_compact", k_pages.device, k_pages, v_pages, page_table, page_refs)


def b200_tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                        page_table: torch.Tensor, seq_lens: torch.Tensor,
                        tree_mask: Optional[torch.Tensor] = None,
                        draft_lens: Optional[torch.Tensor] = None,
                        scale: Optional[float] = None, output_bshd: bool = False, *,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of drafted tokens ``q [B, H, T, D]`` over one layer's cache
    (``k_pages``/``v_pages`` ``[pages, kv_heads, page_size, D]``; ``H`` a multiple of
    ``kv_heads``).

    Drafted token ``i`` of a sequence sees every committed token and those drafted
    tokens ``j`` that ``tree_mask`` (bool ``[T, T]``, or ``[B, T, T]``) shows it: for a
    tree, its ancestors and itself.  Without a mask it sees ``j <= i``, so ``T = 1``
    is the ordinary decode step and a longer chain a piece of a prompt.
    ``draft_lens`` int32 ``[B]`` gives each sequence its number of drafted tokens
    (all ``T`` without it).  Rows past it, and rows that see nothing, are zero (the
    attention forward gives NaN for rows that see nothing, as torch's softmax does;
    here such rows are padding).

    bfloat16 and float16 products run on the tensor cores, float32 in fp32.
    Scores, maximum, sum and output sums are fp32 and the output is rounded once; the
    softmax weights of the 16-bit types are rounded to the type for the product with the
    values, and summed as rounded.  A call under graph capture keeps no counters between
    launches, so cut units of few rows are joined by a second kernel there.

    Over a 4-bit cache (uint8 pools ``[pages, kv_heads, page_size, row bytes]``) ``q`` is
    bfloat16 or float16.  Products with the codes are exact in fp32 sums, steps and lows are
    applied in fp32; a weight times the step of its value is rounded to fp16 for the product
    with the codes (relative to the largest such step), the sum of weights is not.  With
    bfloat16 queries and more than 16 rows (``T * H / kv_heads``) keys are rounded to fp16
    relative to the largest of 32, values to bfloat16.  Returns
    ``[B, H, T, D]``, or ``[B, T, H, D]`` with ``output_bshd``; ``out`` may supply it; it
    may be ``q`` itself, and shares no memory with another argument."""
    return _call("tree_attention", q.device, q, k_pages, v_pages, page_table, seq_lens, tree_mask,
                 draft_lens, scale, output_bshd, out)


class PagedKVCache:
    """The tensors of a paged cache, all pages free and all sequences empty, and the
    page operations on them.  With ``bits=4`` the pools hold 4-bit rows, and ``dtype`` is that of
    the vectors that go in and out."""

    NO_PAGES = _native.CACHE_NO_PAGES
    ROW_FULL = _native.CACHE_ROW_FULL
    BAD_ENTRY = _native.CACHE_BAD_ENTRY

    def __init__(self, layers: int, pages: int, kv_heads: int, page_size: int, head_dim: int,
                 batch: int, slots: int, *, dtype: torch.dtype = torch.bfloat16,
                 device: Union[str, torch.device] = "cuda", bits: Optional[int] = None) -> None:
        shape = (layers, pages, kv_heads, page_size, head_dim)
        if min(shape) < 1 or batch < 1 or slots < 1:
            raise ValueError(f"a cache needs positive sizes, got {shape}, batch {batch}, "
                             f"slots {slots}")
        if bits not in (None, 4):
            raise ValueError(f"bits must be 4, or None for pages of {dtype}, got {bits}")
        self.head_dim, self.dtype, stored = head_dim, dtype, dtype
        if bits == 4:
            if head_dim % 8 or head_dim > 128:
                raise ValueError(f"head_dim {head_dim} is outside the kernel envelope of a 4-bit "
                                 "cache (multiples of 8 up to 128)")
            shape, stored = (*shape[:-1], 48 if head_dim <= 64 else 80), torch.uint8
        self.k_pages = torch.zeros(shape, dtype=stored, device=device)
        self.v_pages = torch.zeros(shape, dtype=stored, device=device)
        ints = dict(dtype=torch.int32, device=device)
        self.page_table = torch.full((batch, slots), -1, **ints)
        self.seq_lens = torch.zeros(batch, **ints)
        self.page_refs = torch.zeros(pages, **ints)

    @property
    def page_size(self) -> int:
        return self.k_pages.shape[3]

    def reserve(self, tokens: Union[int, torch.Tensor]) -> torch.Tensor:
        return b200_cache_reserve(self.k_pages, self.v_pages, self.page_table, self.seq_lens,
                                  self.page_refs, tokens)

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor,
               draft_lens: Optional[torch.Tensor] = None) -> None:
        b200_cache_append(k_new, v_new, self.k_pages[layer], self.v_pages[layer], self.page_table,
                          self.seq_lens, draft_lens)

    def attend(self, layer: int, q: torch.Tensor, tree_mask: Optional[torch.Tensor] = None,
               draft_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
               output_bshd: bool = False) -> torch.Tensor:
        return b200_tree_attention(q, self.k_pages[layer], self.v_pages[layer], self.page_table,
                                   self.seq_lens, tree_mask, draft_lens, scale, output_bshd)

    def read(self, layer: int, starts: torch.Tensor, tokens: int,
             counts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``b200_cache_read`` of one layer (4-bit caches)."""
        return b200_cache_read(self.k_pages[layer], self.v_pages[layer], self.page_table, starts,
                               tokens, self.head_dim, self.dtype, counts)

    def accept(self, paths: torch.Tensor, counts: torch.Tensor) -> None:
        self.seq_lens.copy_(b200_cache_accept(self.k_pages, self.v_pages, self.page_table,
                                              self.seq_lens, paths, counts))

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        b200_cache_fork(self.page_table, self.seq_lens, self.page_refs, src, dst, self.page_size)

    def free(self, rows: torch.Tensor) -> None:
        b200_cache_free(self.page_table, self.seq_lens, self.page_refs, rows)

    def compact(self) -> torch.Tensor:
        return b200_cache_compact(self.k_pages, self.v_pages, self.page_table, self.page_refs)
