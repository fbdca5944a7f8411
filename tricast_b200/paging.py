"""Page plans of a batch on the GPU: from the lengths of its requests to the block table, slots and offsets that
:class:`PagedKVCache` and :func:`paged_attention` take, and ended requests' pages back. No TriCast counterpart."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N


class PagePlan(NamedTuple):
    """What :func:`plan_pages` returns; all on the GPU, int32 but for the slots."""

    seq_lens: torch.Tensor  # [batch] lengths with the new tokens
    cu_q: torch.Tensor  # [batch + 1] where each sequence's new tokens begin
    slots: torch.Tensor  # int64 [tokens] cache slot of each new token; -1 without a page
    sequence: torch.Tensor  # [tokens] the row of the batch it belongs to; -1 behind the last token
    positions: torch.Tensor  # [tokens] its position in its sequence; -1 behind the last token
    taken: torch.Tensor  # [1] the stack's new top
    missing: torch.Tensor  # [1] pages that were lacking


def _check(t: torch.Tensor, shape, name: str, device, dtype=torch.int32) -> None:
    if t.dtype != dtype or t.device != device or t.shape != shape or (t.ndim and t.numel() > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} tensor of shape {list(shape)} on the block table's device")


def _table(block_table: torch.Tensor, free_pages: torch.Tensor, taken: torch.Tensor) -> tuple:
    if not block_table.is_cuda:
        raise ValueError("the B200 backend requires a CUDA tensor")
    if block_table.ndim != 2 or block_table.dtype != torch.int32:
        raise ValueError("block_table must be an int32 tensor [batch, max_pages]")
    batch, width = block_table.shape
    stride, one = block_table.stride()
    if (one != 1 and width > 1) or (batch > 1 and stride < width):
        raise ValueError("block_table is written in place: its rows must be contiguous and lie apart")
    device = block_table.device
    if free_pages.ndim != 1:
        raise ValueError("free_pages must be a 1-D int32 tensor")
    _check(free_pages, free_pages.shape, "free_pages", device)
    if taken.numel() != 1 or taken.dtype != torch.int32 or taken.device != device:
        raise ValueError("taken must be one int32 number on the block table's device")
    return batch, width, stride, device


def plan_pages(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               taken: torch.Tensor, *, page_size: int, tokens: int) -> PagePlan:
    """Pages and slots of a batch's new tokens, without a word to the host: a decode step can be captured with it.

    ``seq_lens`` (int32 ``[batch]``): the tokens each sequence has in the cache; ``new_lens`` (int32 ``[batch]``): how many
    it gets (0: idle). The new tokens stand one after the other, sequence by sequence; ``tokens`` is the room for them,
    those beyond it are left out (their sequences get fewer), as are those that would make a sequence longer than ``2**31 -
    1``. ``free_pages`` (int32, 1-D) is a stack, of whose entries those from ``taken`` (one int32 number) on are free. Pages
    that a sequence lacks are taken from there in order and written into its row of ``block_table`` (int32 ``[batch,
    max_pages]``), in place; no other entry is touched. Where the stack is empty the entry becomes ``-1``, and pages beyond
    ``max_pages`` are not taken: tokens on them get the slot ``-1`` (:meth:`PagedKVCache.write` skips it) and ``missing``
    counts them.

    Returns a :class:`PagePlan`: its ``slots``, ``seq_lens``, ``cu_q`` go to the cache's ``write`` and
    :func:`paged_attention`; ``seq_lens`` and ``taken`` are the next call's (copy them over where a captured call reads
    them). Inputs other than ``block_table`` are left as they are."""
    batch, width, stride, device = _table(block_table, free_pages, taken)
    _check(seq_lens, (batch,), "seq_lens", device)
    _check(new_lens, (batch,), "new_lens", device)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    if not 1 <= page_size <= 1 << 20:  # the C entry's numbers have 32 bits
        raise ValueError("page_size must be a power of two of at most 2**20")
    ints = torch.empty(2 * tokens + 2 * batch + 3, dtype=torch.int32, device=device)
    sequence, positions, cu, lens, out_taken, missing = ints.split((tokens, tokens, batch + 1, batch, 1, 1))
    slots = torch.empty(tokens, dtype=torch.int64, device=device)
    lib, index = N.lib(), device.index
    with N.on_device(index):
        nbytes = lib.tc_plan_pages_workspace(batch)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        at = ints.data_ptr()
        status = lib.tc_plan_pages(
            seq_lens.data_ptr(), new_lens.data_ptr(), batch, block_table.data_ptr(), stride, width, free_pages.data_ptr(),
            free_pages.shape[0], taken.data_ptr(), page_size, tokens, at + 4 * (2 * tokens + batch + 1), at + 8 * tokens,
            slots.data_ptr(), at, at + 4 * tokens, at + 4 * (2 * tokens + 2 * batch + 1), at + 4 * (2 * tokens + 2 * batch + 2),
            None if ws is None else ws.data_ptr(), nbytes, N.raw_stream(index))
    if status:
        N.check(status, "tc_plan_pages")
    return PagePlan(lens, cu, slots, sequence, positions, out_taken, missing)


def release_pages(block_table: torch.Tensor, ended: torch.Tensor, free_pages: torch.Tensor, taken: torch.Tensor) -> torch.Tensor:
    """Puts the pages of ended sequences (``ended``, bool ``[batch]``) back on the stack of :func:`plan_pages`, in the
    order of sequences and columns, and fills their rows of ``block_table`` with ``-1``; both in place. Returns the stack's
    new top (int32 ``[1]``); their ``seq_lens`` are the caller's to set to 0. A page must stand in one row only: pages that
    sequences share are the caller's to keep apart."""
    batch, width, stride, device = _table(block_table, free_pages, taken)
    _check(ended, (batch,), "ended", device, torch.bool)
    out = torch.empty(1, dtype=torch.int32, device=device)
    lib, index = N.lib(), device.index
    with N.on_device(index):
        nbytes = lib.tc_release_pages_workspace(batch)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        status = lib.tc_release_pages(block_table.data_ptr(), stride, width, ended.data_ptr(), batch, free_pages.data_ptr(),
                                      free_pages.shape[0], taken.data_ptr(), out.data_ptr(),
                                      None if ws is None else ws.data_ptr(), nbytes, N.raw_stream(index))
    if status:
        N.check(status, "tc_release_pages")
    return out


__all__ = ["PagePlan", "plan_pages", "release_pages"]
