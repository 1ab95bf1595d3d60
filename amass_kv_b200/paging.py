"""Page bookkeeping of a serving step on the GPU: which blocks a request's new
tokens get, the block table, and the step's start offsets, positions and slot
mapping, all from the new token counts -- no host round trip, capturable in a
CUDA graph.

  BlockPool        owns the free blocks, block table and lengths of up to
                   ``max_reqs`` requests: begin_step (grow), truncate (drop
                   the last tokens: a rejected draft), release (a finished
                   request)
  build_slot_map   positions and slots of a step whose block table and
                   lengths an engine keeps itself

The tensors are the ones the rest of the package reads: ``block_table``,
``seq_lens``, ``query_start_loc`` and ``slot_mapping`` (block * page + offset,
-1 skips).
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import check_i32

MAX_REQS = 4096


class BlockPool(_lib.FixedBuffers):
    """Device-resident block allocator, allocated once.

      free_stack (NB,), free_top (1,)   free blocks, popped from the top
      block_table (R, MP)               blocks of each row, -1 behind them
      seq_lens (R,)                     tokens of each row (0: idle)
      query_start_loc (R + 1,)          set by begin_step for its rows
      positions, slot_mapping (max_tokens,) int64
      status (R,), overflow (1,)        what begin_step refused

    All int32 but the two token maps.  ``status[r]``: 0 granted, 1 too few
    free blocks, 2 longer than ``max_pages`` or past 2^30 tokens in the step;
    a refused row keeps its pages and length and its new tokens get slot -1;
    hand ``status`` to ``attention.paged_chunk_attention``, which cannot see
    from the lengths that the row's tokens are not among them.  ``overflow``
    latches 1 / 2 for such a row and 4 for more new tokens than the step's
    ``n_tokens``; ``check()`` reads it (synchronises) and raises.

    Calls on one pool must run one after the other (one stream, or ordered
    by events)."""

    def __init__(self, device, *, num_blocks: int, max_reqs: int,
                 max_pages: int, max_tokens: int, page: int = 16):
        if num_blocks < 1 or max_pages < 1 or max_tokens < 1 or page < 1:
            raise ValueError("num_blocks, max_pages, max_tokens and page "
                             "must be at least 1")
        if not 1 <= max_reqs <= MAX_REQS:
            raise ValueError(f"max_reqs must be 1 .. {MAX_REQS}, got "
                             f"{max_reqs}")
        if max_pages * page >= 1 << 31:
            raise ValueError("max_pages * page must fit int32")
        dev = _lib.device_of(device)
        self.device, self.NB, self.R = dev, num_blocks, max_reqs
        self.MP, self.max_tokens, self.page = max_pages, max_tokens, page
        kw = dict(dtype=torch.int32, device=dev)
        self.free_stack = torch.arange(num_blocks - 1, -1, -1, **kw)
        self.free_top = torch.full((1,), num_blocks, **kw)
        self.block_table = torch.full((max_reqs, max_pages), -1, **kw)
        self.seq_lens = torch.zeros(max_reqs, **kw)
        self.query_start_loc = torch.zeros(max_reqs + 1, **kw)
        self.status = torch.zeros(max_reqs, **kw)
        self.overflow = torch.zeros(1, **kw)
        self.ticket = torch.zeros(1, **kw)
        self.positions = torch.zeros(max_tokens, dtype=torch.int64,
                                     device=dev)
        self.slot_mapping = torch.full((max_tokens,), -1, dtype=torch.int64,
                                       device=dev)

        self._index = -1 if dev.index is None else dev.index
        # the C side's view of the buffers: fill them in place, they are not
        # to be replaced
        self._pool = _lib.PAGE_POOL.pack(
            *(t.data_ptr() for t in (
                self.block_table, self.seq_lens, self.free_stack,
                self.free_top, self.query_start_loc, self.positions,
                self.slot_mapping, self.status, self.overflow, self.ticket)),
            self.block_table.stride(0), num_blocks, max_reqs, max_pages,
            max_tokens, page, 0)
        self._fixed = True

    def _rows(self, t, name: str) -> int:
        n, = check_i32(self._index, name, t, 1)
        if n > self.R:
            raise ValueError(f"{name} has {n} rows, the pool {self.R}")
        return n

    def begin_step(self, new_tokens, n_tokens: int | None = None) -> None:
        """Rows 0 .. len(new_tokens) - 1 grow by ``new_tokens`` (int32, < 0
        counts as 0), in order: blocks, block table, ``seq_lens``,
        ``query_start_loc``, and ``positions`` / ``slot_mapping`` of the first
        ``n_tokens`` tokens (default ``max_tokens``; 0 / -1 behind the last
        one, so a padded batch writes nothing).  One launch."""
        n = self._rows(new_tokens, "new_tokens")
        nt = self.max_tokens if n_tokens is None else int(n_tokens)
        if not 0 <= nt <= self.max_tokens:
            raise ValueError(f"n_tokens {nt} outside 0 .. {self.max_tokens}")
        _lib.launch(self._index, "amass_pages_begin", self._pool,
                    new_tokens.data_ptr(), n, nt)

    def truncate(self, drop) -> None:
        """Row r loses its last ``drop[r]`` tokens (int32; clipped to what it
        has).  Pages left empty go back to the free stack, last row and last
        page first: dropping all that a ``begin_step`` granted restores the
        stack's order.  A row that the step refused has none of its tokens:
        give it 0, or it loses older ones."""
        n = self._rows(drop, "drop")
        _lib.launch(self._index, "amass_pages_trim", self._pool,
                    drop.data_ptr(), n, 0)

    def release(self, done) -> None:
        """Rows with ``done[r] != 0`` (int32) give back all their pages and
        become idle."""
        n = self._rows(done, "done")
        _lib.launch(self._index, "amass_pages_trim", self._pool,
                    done.data_ptr(), n, 1)

    def check(self) -> None:
        f = int(self.overflow.item())
        if f:
            why = [s for b, s in ((1, "the free blocks ran out"),
                                  (2, "a row outgrew max_pages"),
                                  (4, "more new tokens than n_tokens"))
                   if f & b]
            raise RuntimeError("BlockPool: " + ", ".join(why))


def build_slot_map(block_table, seq_lens, query_start_loc, positions,
                   slot_mapping, *, page: int = 16,
                   n_tokens: int | None = None) -> None:
    """Fill ``positions`` and ``slot_mapping`` (int64) of the step's first
    ``n_tokens`` tokens (default: all of slot_mapping): token t of request r,
    query_start_loc[r] <= t < query_start_loc[r + 1], is one of the last of
    its ``seq_lens[r]``.  Slot -1 for a position without a block (< 0, beyond
    the table's row, block < 0); tokens of no request get 0 and -1."""
    dev = block_table.get_device()
    rows, max_pages = check_i32(dev, "block_table", block_table, 2)
    n, = check_i32(dev, "seq_lens", seq_lens, 1)
    starts, = check_i32(dev, "query_start_loc", query_start_loc, 1)
    if rows < n or max_pages < 1 or starts <= n:
        raise ValueError(f"block_table {(rows, max_pages)} and "
                         f"query_start_loc {tuple(query_start_loc.shape)} do "
                         f"not cover {n} requests")
    if n > MAX_REQS:
        raise ValueError(f"{n} requests > {MAX_REQS}")
    if page < 1 or page * max_pages >= 1 << 31:
        raise ValueError(f"page must be at least 1 and a row's tokens fit "
                         f"int32, got {page} x {max_pages}")
    nt = slot_mapping.shape[0] if n_tokens is None else int(n_tokens)
    for name, t in (("positions", positions), ("slot_mapping", slot_mapping)):
        if t.dtype != torch.int64 or t.get_device() != dev or t.dim() != 1 \
                or not t.is_contiguous() or not 0 <= nt <= t.shape[0]:
            raise ValueError(f"{name} must be a contiguous int64 vector of "
                             f"at least {nt} tokens on GPU {dev}")
    _lib.launch(dev, "amass_slot_map", block_table.data_ptr(),
                block_table.stride(0), seq_lens.data_ptr(),
                query_start_loc.data_ptr(), n, positions.data_ptr(),
                slot_mapping.data_ptr(), nt, max_pages, page)


__all__ = ["BlockPool", "build_slot_map"]
