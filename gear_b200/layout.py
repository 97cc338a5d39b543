"""Where the rows of a batch of unequal sequences go: offsets, pages and slots, built on the GPU.

A batch of requests with `lengths` rows each is laid out either packed (request r owns rows
[offsets[r], offsets[r+1])) or in the pages of a pool (row t of request r lives in slot
block_table[r][t // page] * page + t % page).  paged_layout() makes the tables of both in one call from lengths
that may only be known on the device, such as those of a sampled batch:

    n = handler.segment_lengths(idx, ts, ln, column)
    lay = paged_layout(n, page=16, block_table=table, used=used, free_pages=free, max_tokens=room)
    handler.gather_packed(columns, idx, ts, ln, lay.offsets, pools, block_table=lay.block_table, page=16)

and, with `past`, adds rows to requests that have some already (a decoding step adds one to each).

The reference has no counterpart: its batches are padded (gear/loader/offline_loader.py:178-203).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as N
from ._native import GearError, check, lib
from .core import _Scope, _stream

__all__ = ["PagedLayout", "paged_layout"]

_LAYOUT = lib.gearb_layout_paged


class PagedLayout(NamedTuple):
    offsets: torch.Tensor              # int64 [requests + 1]
    slot_map: Optional[torch.Tensor]   # int64 [max_tokens]; -1 behind the last token and without a page
    block_table: torch.Tensor          # int32 [requests, max_blocks]
    used: torch.Tensor                 # int64 [1]: pages of the free list handed out so far


def _need(t, what: str, dtype, device, numel=None):
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or not t.is_cuda or not t.is_contiguous():
        raise GearError(N.ERR_INVALID, f"paged_layout: {what} must be a contiguous {dtype} CUDA tensor")
    if t.device != device:
        raise GearError(N.ERR_INVALID, f"paged_layout: {what} is on {t.device}, lengths on {device}")
    if numel is not None and t.numel() != numel:
        raise GearError(N.ERR_INVALID, f"paged_layout: {what} must have {numel} entries")
    return t.data_ptr()


def paged_layout(lengths: torch.Tensor, page: int, block_table: torch.Tensor, used: torch.Tensor, *,
                 free_pages: Optional[torch.Tensor] = None, num_pages: Optional[int] = None,
                 past: Optional[torch.Tensor] = None, max_tokens: int = 0, offsets: Optional[torch.Tensor] = None,
                 slot_map: Optional[torch.Tensor] = None, used_out: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None, stream=None) -> PagedLayout:
    """Lay `lengths[r]` new rows of every request out behind the `past[r]` it has (default none).

    lengths, past   int64 [requests]; a request holds at most block_table.shape[1] * page rows, what is
                    beyond is cut (ST_LEN_CLAMPED)
    block_table     int32 [requests, max_blocks]: the new pages are written into it, in place, behind the
                    ceil(past / page) a request has; its other entries are left as they are
    used            int64 [1]: how many pages of the free list were handed out before.  The result's `used` is a
                    new tensor, or `used_out`, which may be `used` itself
    free_pages      int32 [n]: the pool's pages in the order in which they are handed out (None: 0, 1, 2, ...,
                    num_pages of them).  When they run out, entries and slots are -1 (ST_NO_PAGE)
    max_tokens      entries of the slot map (0: none is made): rows in packed order, -1 behind the last one;
                    rows beyond it have their pages but no entry
    offsets, slot_map, used_out   write there instead of allocating; status int32[4] as of the other launches
    """
    if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1:
        raise GearError(N.ERR_INVALID, "paged_layout: lengths must be a one-dimensional int64 CUDA tensor")
    dev, r = lengths.device, lengths.numel()
    at_lengths = _need(lengths, "lengths", torch.int64, dev)
    at_past = 0 if past is None else _need(past, "past", torch.int64, dev, r)
    at_table = _need(block_table, "block_table", torch.int32, dev)
    shape = block_table.shape
    if len(shape) != 2 or shape[0] != r or shape[1] < 1:
        raise GearError(N.ERR_INVALID, f"paged_layout: block_table must be [{r}, max_blocks]")
    at_free = 0 if free_pages is None else _need(free_pages, "free_pages", torch.int32, dev)
    at_used = _need(used, "used", torch.int64, dev, 1)
    if free_pages is None and num_pages is None:
        raise GearError(N.ERR_INVALID, "paged_layout: num_pages is required without free_pages")
    pages = free_pages.numel() if num_pages is None else num_pages
    if free_pages is not None and pages > free_pages.numel():
        raise GearError(N.ERR_INVALID, "paged_layout: num_pages is more than free_pages has")
    page, pages, max_tokens = int(page), int(pages), int(max_tokens)
    if not 1 <= page <= 1 << 31 or not 0 <= pages <= 1 << 31:
        raise GearError(N.ERR_INVALID, "paged_layout: page must be 1 to 2^31, num_pages 0 to 2^31")
    if slot_map is not None:
        _need(slot_map, "slot_map", torch.int64, dev)
        if max_tokens not in (0, slot_map.numel()):
            raise GearError(N.ERR_INVALID, "paged_layout: slot_map must have max_tokens entries")
        max_tokens = slot_map.numel()
    if max_tokens < 0:
        raise GearError(N.ERR_INVALID, "paged_layout: max_tokens must not be negative")
    if offsets is not None:
        _need(offsets, "offsets", torch.int64, dev, r + 1)
    if used_out is not None:
        _need(used_out, "used_out", torch.int64, dev, 1)
    at_status = 0 if status is None else _need(status, "status", torch.int32, dev, N.STATUS_WORDS)
    with _Scope(dev, stream):
        if offsets is None:
            offsets = torch.empty(r + 1, dtype=torch.int64, device=dev)
        if slot_map is None and max_tokens:
            slot_map = torch.empty(max_tokens, dtype=torch.int64, device=dev)
        if used_out is None:
            used_out = torch.empty(1, dtype=torch.int64, device=dev)
        nbytes = lib.gearb_layout_scratch_bytes(r)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        check(_LAYOUT(N.LAYOUT_ARGS.pack(at_lengths, at_past, r, page, shape[1], at_table, at_free, pages, at_used,
                                         used_out.data_ptr(), offsets.data_ptr(),
                                         0 if slot_map is None else slot_map.data_ptr(), max_tokens,
                                         scratch.data_ptr(), nbytes, at_status), _stream()))
    return PagedLayout(offsets, slot_map, block_table, used_out)
