"""The plan of a ragged batch: where the tokens of its requests lie, from their lengths.

CPU tensors take the restatement in :mod:`mfq_b200.ops.reference`.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import reference
from .lib import check, current_device, lib, ptr, stream_ptr
from .logits import _index

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


def plan_batch(block_table: torch.Tensor, rows: torch.Tensor, past: torch.Tensor, counts: torch.Tensor, *, tokens: int, page_size: int = 16,
               pages: torch.Tensor | None = None) -> BatchPlan:
    """Plan a batch in which request ``i`` brings ``counts[i]`` tokens behind ``past[i]`` of the sequence in row ``rows[i]`` of
    ``block_table [R, P]`` (all int32, lengths on the device).  ``tokens``: places of the plan, at least ``counts.sum()``.

    With ``pages`` (int32 ``[n]`` free page ids), the row holds the pages of its past, ``ceil(past / page_size)``; the pages that the new
    tokens need beside them are taken from the front of the list, request by request, and written into ``block_table``.  A row
    may then occur once.

    Lengths that do not fit are found on the device: the plan then is that of a batch without tokens, nothing is written into
    ``block_table``, and :meth:`BatchPlan.check` says why."""
    dev = block_table.device
    if block_table.dtype != torch.int32 or block_table.ndim != 2 or not block_table.is_contiguous() or block_table.numel() == 0:
        raise ValueError(f"block_table: contiguous int32 [R, P] is wanted, got {block_table.dtype} {tuple(block_table.shape)}")
    b, (r, p) = rows.numel(), block_table.shape
    for name, t in (("rows", rows), ("past", past), ("counts", counts)):
        _index(name, t, b, dev)
    if not 1 <= b <= MAX_REQUESTS:
        raise ValueError(f"a plan takes 1 to {MAX_REQUESTS} requests, got {b}")
    if tokens < 0 or page_size < 1 or p * page_size > 2 ** 31 - 1:
        raise ValueError(f"{tokens} tokens, rows of {p} pages of {page_size}")
    if pages is not None:
        _index("pages", pages, None, dev)
        if r > MAX_TABLE_ROWS:
            raise ValueError(f"pages are handed out to tables of at most {MAX_TABLE_ROWS} rows, got {r}")
    flat = torch.empty(3 * tokens + 2 * b + 3 + b * p, dtype=torch.int32, device=dev)  # one allocation; a part's beginning needs no alignment
    at = 0

    def part(n: int) -> torch.Tensor:
        nonlocal at
        at += n
        return flat[at - n : at]

    plan = BatchPlan(part(tokens), part(tokens), part(tokens), part(b + 1), part(b), part(b * p).view(b, p), part(2))
    if not block_table.is_cuda:
        reference.plan_batch(plan, block_table, rows, past, counts, tokens, page_size, pages)
        return plan
    with current_device(dev):
        check(lib().mfq_plan_batch(ptr(block_table), r, p, ptr(rows), ptr(past), ptr(counts), b, ptr(pages), pages.numel() if pages is not None else -1,
                                   ptr(plan.positions), ptr(plan.slots), ptr(plan.tok_seq), tokens, ptr(plan.q_starts), ptr(plan.seq_lens),
                                   ptr(plan.block_table), ptr(plan.info), page_size, stream_ptr()), "plan_batch")
    return plan
