"""The plan of a ragged batch: where the tokens of its requests lie, from their lengths.

CPU tensors take the restatement in :mod:`mfq_b200.ops.reference`.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import reference
from .lib import check, elsewhere, lib, ptr, stream_ptr
from .logits import _index, _refuse

MAX_REQUESTS = 1024  # of a batch; kPlanRequests of the kernel
MAX_TABLE_ROWS = 1 << 16  # of a table whose pages are handed out; kPlanRows

_REFUSED = {1: "a request names a row outside the table, a row that another one has too, or a negative length",
            2: "more tokens than the plan has places, or more pages than a row of the table",
            3: "too few free pages"}


@dataclass
class BatchPlan:
    positions: torch.Tensor  # [T] position of each token in its sequence; 0 behind the last token
    slots: torch.Tensor  # [T] page * page_size + place; -1 behind the last token
    tok_seq: torch.Tensor  # [T] request of each token; -1 behind the last token
    q_starts: torch.Tensor  # [b + 1] first token of each request
    seq_lens: torch.Tensor  # [b] tokens of each sequence, the new ones included
    block_table: torch.Tensor  # [b, P] pages of each request in use, then null pages
    info: torch.Tensor  # [2] tokens planned and pages taken; a refused plan: minus its reason, and 0

    def check(self) -> tuple[int, int]:
        """(tokens, pages taken); raises ``ValueError`` with the reason if the plan was refused (synchronizes)."""
        tokens, pages = self.info.tolist()
        if tokens < 0:
            raise ValueError(f"the plan was refused: {_REFUSED[-tokens]}")
        return tokens, pages

    @classmethod
    def joined(cls, plans: list["BatchPlan"]) -> "BatchPlan":
        """The plan of the plans' batches one after the other; every one has exactly as many places as tokens, or is refused."""
        seqs, starts, first, at = [], [], 0, 0
        for p in plans:
            seqs.append(p.tok_seq + first)
            starts.append(p.q_starts[0 if not starts else 1 :] + at)
            first, at = first + p.seq_lens.numel(), at + p.positions.numel()
        cat = lambda name: torch.cat([getattr(p, name) for p in plans])  # noqa: E731
        info = torch.stack([p.info for p in plans])
        refused = info[:, 0].amin().clamp(max=0)
        info = torch.where(refused < 0, torch.stack([refused, torch.zeros_like(refused)]), info.sum(0).to(torch.int32))
        return cls(cat("positions"), cat("slots"), torch.cat(seqs), torch.cat(starts), cat("seq_lens"), cat("block_table"), info)


def plan_batch(block_table: torch.Tensor, rows: torch.Tensor, past: torch.Tensor, counts: torch.Tensor, *, tokens: int, page_size: int = 16,
               pages: torch.Tensor | None = None) -> BatchPlan:
    """Plan a batch in which request ``i`` brings ``counts[i]`` tokens behind ``past[i]`` of the sequence in row ``rows[i]`` of
    ``block_table [R, P]`` (all int32, lengths on the device).  ``tokens``: places of the plan, at least ``counts.sum()``.

    With ``pages`` (int32 ``[n]`` free page ids), the row holds the pages of its past, ``ceil(past / page_size)``; the pages that the new
    tokens need beside them are taken from the front of the list, request by request, and written into ``block_table``.  A row
    may then occur once.

    Lengths that do not fit are found on the device: the plan then is that of a batch without tokens, nothing is written into
    ``block_table``, and :meth:`BatchPlan.check` says why."""
    if block_table.dtype is not torch.int32 or block_table.ndim != 2 or not block_table.is_contiguous() or not block_table.numel():
        _refuse("block_table", "contiguous int32 [R, P] is", block_table)
    b, (r, p), index = rows.numel(), block_table.shape, block_table.get_device()
    _index("rows", rows, None, index)
    _index("past", past, b, index)
    _index("counts", counts, b, index)
    if not 1 <= b <= MAX_REQUESTS:
        raise ValueError(f"a plan takes 1 to {MAX_REQUESTS} requests, got {b}")
    if not 0 <= tokens <= 1 << 30 or page_size < 1 or p * page_size > 2 ** 31 - 1:
        raise ValueError(f"{tokens} tokens, rows of {p} pages of {page_size}")
    if pages is not None:
        _index("pages", pages, None, index)
        if r > MAX_TABLE_ROWS:
            raise ValueError(f"pages are handed out to tables of at most {MAX_TABLE_ROWS} rows, got {r}")
    if index >= 0 and elsewhere(index):
        with torch.cuda.device(index):
            return plan_batch(block_table, rows, past, counts, tokens=tokens, page_size=page_size, pages=pages)
    sizes = [tokens, tokens, tokens, b + 1, b, b * p, 2]
    whole = block_table.new_empty(sum(sizes))  # one allocation; a part's beginning needs no alignment
    parts = list(torch.split_with_sizes(whole, sizes))
    parts[5] = parts[5].view(b, p)
    plan = BatchPlan(*parts)
    if index < 0:
        reference.plan_batch(plan, block_table, rows, past, counts, tokens, page_size, pages)
        return plan
    at = whole.data_ptr()  # (an empty part has no address)
    check(lib().mfq_plan_batch(block_table.data_ptr(), r, p, rows.data_ptr(), past.data_ptr(), counts.data_ptr(), b, ptr(pages), -1 if pages is None else pages.numel(),
                               at, at + 4 * tokens, at + 8 * tokens, tokens, at + 12 * tokens, at + 12 * tokens + 4 * (b + 1), at + 12 * tokens + 8 * b + 4,
                               at + 12 * tokens + 8 * b + 4 + 4 * b * p, page_size, stream_ptr()), "plan_batch")
    return plan
