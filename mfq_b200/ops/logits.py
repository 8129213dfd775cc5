"""Processing of logits between the output projection and the sampler: biases, penalties for repeated tokens, masks.

Every row of the tables (``records``, ``counts``, the biases, ``allowed``) belongs to a request; ``rows`` says which one a row of
logits is processed by, so that a verify window or a mixed batch needs no copies of them.  The penalties go by 16-bit words: the
lower 15 bits count how often the request's answer has the token, the top bit says that its prompt has it.  The repetition penalty
goes by both, presence and frequency by the answer alone.

CPU tensors take the restatements in :mod:`mfq_b200.ops.reference`.
"""

from __future__ import annotations

import torch

from . import reference
from .lib import check, current_device, lib, ptr, stream_ptr

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_BIASES = 1024  # places per row; kMaxBias of the kernel
RECORD_WORDS = 8  # a sampling record: temperature f32, top_k i32, top_p f32, presence f32, frequency f32, repetition f32, seed u64


def _table(name: str, t: torch.Tensor, dtype: torch.dtype, device, rows: int | None = None) -> None:
    if t.dtype != dtype or t.ndim != 2 or t.device != device or (rows is not None and t.shape[0] != rows):
        raise ValueError(f"{name}: a {dtype} table [{'rows' if rows is None else rows}, ...] on {device} is wanted, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _index(name: str, t: torch.Tensor, count: int | None, device) -> None:
    if t.dtype != torch.int32 or t.ndim != 1 or t.device != device or not t.is_contiguous() or (count is not None and t.numel() != count):
        raise ValueError(f"{name}: contiguous int32 [{'n' if count is None else count}] on {device} is wanted, got {t.dtype} {tuple(t.shape)} on {t.device}")


def process_logits(logits: torch.Tensor, records: torch.Tensor, *, counts: torch.Tensor | None = None,
                   bias: tuple[torch.Tensor, torch.Tensor] | None = None, allowed: torch.Tensor | None = None,
                   rows: torch.Tensor | None = None, first: int = 0, fill: float = float("-inf"), out: torch.Tensor | None = None) -> torch.Tensor:
    """``logits [B, V]`` (bf16, fp16 or fp32; the rows may lie apart) with biases, penalties and mask applied in that order, in fp32,
    rounded once.  Returns ``out``: a new tensor, one given, or ``logits`` itself.

    * ``records [R, 8]`` int32: the requests' sampling records; their penalties apply where ``counts`` is given;
    * ``counts [R, V]`` int16 words of :func:`count_tokens` (a column slice of a wider table will do);
    * ``bias`` = (ids ``[R, K]`` int32, values ``[R, K]`` fp32), at most :data:`MAX_BIASES` places a row; negative ids are unused places,
      an id that occurs twice has the sum;
    * ``allowed [R, words]`` int32: bit ``id % 32`` of word ``id // 32``; a token whose bit is not set becomes ``fill``, whatever it was.
      A row that allows nothing is all ``fill``;
    * ``rows [B]`` int32: the tables' row of each row of logits (default: its own number); a row outside the tables passes through;
    * ``first``: vocabulary id of column 0, for a shard of the vocabulary (biases and masks go by ids, ``counts`` by columns)."""
    if logits.ndim != 2 or logits.dtype not in _DTYPES or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"logits: bf16, fp16 or fp32 [B, V] with neighbouring columns are wanted, got {logits.dtype} {tuple(logits.shape)} strides {logits.stride()}")
    b, v = logits.shape
    dev = logits.device
    _table("records", records, torch.int32, dev)
    r = records.shape[0]
    if records.shape[1] != RECORD_WORDS or not records.is_contiguous() or r == 0:
        raise ValueError(f"records: contiguous [R, {RECORD_WORDS}] are wanted, got {tuple(records.shape)}")
    if rows is None:
        if b > r:
            raise ValueError(f"{b} rows of logits, but {r} records")
    else:
        _index("rows", rows, b, dev)
    if first < 0:
        raise ValueError(f"first: {first}")
    if counts is not None:
        _table("counts", counts, torch.int16, dev, r)
        if counts.shape[1] != v or (v > 1 and counts.stride(1) != 1):
            raise ValueError(f"counts: [R, {v}] with neighbouring columns are wanted, got {tuple(counts.shape)}")
    ids = values = None
    k = 0
    if bias is not None:
        ids, values = bias
        _table("bias ids", ids, torch.int32, dev, r)
        _table("bias values", values, torch.float32, dev, r)
        k = ids.shape[1]
        if values.shape != ids.shape or k > MAX_BIASES or not (ids.is_contiguous() and values.is_contiguous()):
            raise ValueError(f"bias: contiguous ids and values of one shape [R, at most {MAX_BIASES}] are wanted, got {tuple(ids.shape)} and {tuple(values.shape)}")
    if allowed is not None:
        _table("allowed", allowed, torch.int32, dev, r)
        if allowed.shape[1] * 32 < first + v or not allowed.is_contiguous():
            raise ValueError(f"allowed: contiguous [R, at least {(first + v + 31) // 32}] are wanted, got {tuple(allowed.shape)}")
    if out is None:
        out = torch.empty((b, v), dtype=logits.dtype, device=dev)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev or (v > 1 and out.stride(1) != 1) or (b > 1 and out.stride(0) < v):
        raise ValueError(f"out: {logits.dtype} {tuple(logits.shape)} on {dev} with neighbouring columns is wanted, got {out.dtype} {tuple(out.shape)} on {out.device}")
    if b == 0 or v == 0:
        return out
    if not logits.is_cuda:
        out.copy_(reference.process_logits(logits, records, counts, bias, allowed, rows, first, fill))
        return out
    with current_device(dev):
        check(lib().mfq_process_logits(ptr(logits), ptr(out), _DTYPES[logits.dtype], b, v, logits.stride(0), out.stride(0), ptr(records), r, ptr(counts),
                                       counts.stride(0) if counts is not None else 0, ptr(ids), ptr(values), k, ptr(allowed),
                                       allowed.shape[1] if allowed is not None else 0, ptr(rows), first, fill, stream_ptr()), "process_logits")
    return out


def count_tokens(counts: torch.Tensor, tokens: torch.Tensor, rows: torch.Tensor, *, prompt: bool = False) -> None:
    """Count ``tokens [n]`` int32 in ``counts[rows [n], token]`` (int16 words ``[R, V]``, see the top of this module): as tokens of an
    answer, whose counts stay at 32767 once there, or with ``prompt`` as tokens that the prompt has.  A pair outside the table is left
    out, so a batch may be padded with negative rows."""
    if counts.dtype != torch.int16 or counts.ndim != 2 or (counts.shape[1] > 1 and counts.stride(1) != 1):
        raise ValueError(f"counts: int16 [R, V] with neighbouring columns are wanted, got {counts.dtype} {tuple(counts.shape)}")
    _index("tokens", tokens, None, counts.device)
    _index("rows", rows, tokens.numel(), counts.device)
    if counts.numel() == 0 or tokens.numel() == 0:
        return
    if not counts.is_cuda:
        reference.count_tokens(counts, tokens, rows, prompt)
        return
    with current_device(counts.device):
        check(lib().mfq_count_tokens(ptr(counts), counts.stride(0), counts.shape[0], counts.shape[1], ptr(tokens), ptr(rows), tokens.numel(), int(prompt),
                                     stream_ptr()), "count_tokens")
