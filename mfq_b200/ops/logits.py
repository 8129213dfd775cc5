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
from .lib import check, elsewhere, lib, ptr, stream_ptr

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_BIASES = 1 << 16  # places per row; kMaxBias of the kernel
MAX_ROWS = 65535  # of logits on a GPU: blocks of a grid in y
RECORD_WORDS = 8  # a sampling record: temperature f32, top_k i32, top_p f32, presence f32, frequency f32, repetition f32, seed u64


def _refuse(name: str, wanted: str, t: torch.Tensor) -> None:
    raise ValueError(f"{name}: {wanted} wanted, got {t.dtype} {tuple(t.shape)}, strides {t.stride()}, on {t.device}")


def _index(name: str, t: torch.Tensor, count: int | None, index: int) -> None:
    n = t.numel()
    if t.dtype is not torch.int32 or t.ndim != 1 or t.get_device() != index or not t.is_contiguous() or n != (min(n, 1 << 30) if count is None else count):
        _refuse(name, f"contiguous int32 [{'n' if count is None else count}] on the device of the others are", t)


def process_logits(logits: torch.Tensor, records: torch.Tensor, *, counts: torch.Tensor | None = None,
                   bias: tuple[torch.Tensor, torch.Tensor] | None = None, allowed: torch.Tensor | None = None,
                   rows: torch.Tensor | None = None, first: int = 0, fill: float = float("-inf"), out: torch.Tensor | None = None) -> torch.Tensor:
    """``logits [B, V]`` (bf16, fp16 or fp32; the rows may lie apart) with biases, penalties and mask applied in that order, in fp32,
    rounded once; at most :data:`MAX_ROWS` rows on a GPU.  Returns ``out``: a new tensor, one given, or ``logits`` itself.

    * ``records [R, 8]`` int32: the requests' sampling records; their penalties apply where ``counts`` is given (16-bit logits on a GPU are multiplied by the
      reciprocal of the repetition penalty, which is infinite for a factor under 2^-128);
    * ``counts [R, V]`` int16 words of :func:`count_tokens` (a column slice of a wider table will do);
    * ``bias`` = (ids ``[R, K]`` int32, values ``[R, K]`` fp32), at most :data:`MAX_BIASES` places a row; negative ids are unused places,
      an id that occurs twice has the sum;
    * ``allowed [R, words]`` int32: bit ``id % 32`` of word ``id // 32``; a token whose bit is not set becomes ``fill``, whatever it was.
      A row that allows nothing is all ``fill``;
    * ``rows [B]`` int32: the tables' row of each row of logits (default: its own number); a row outside the tables passes through;
    * ``first``: vocabulary id of column 0, for a shard of the vocabulary (biases and masks go by ids, ``counts`` by columns)."""
    if logits.ndim != 2 or logits.dtype not in _DTYPES or (logits.shape[1] > 1 and logits.stride(1) != 1):
        _refuse("logits", "bf16, fp16 or fp32 [B, V] with neighbouring columns are", logits)
    b, v = logits.shape
    index = logits.get_device()
    if records.dtype is not torch.int32 or records.ndim != 2 or records.shape[1] != RECORD_WORDS or records.get_device() != index or \
            not records.is_contiguous() or not records.numel():
        _refuse("records", f"contiguous int32 [R, {RECORD_WORDS}] on the logits' device are", records)
    r = records.shape[0]
    if rows is not None:
        _index("rows", rows, b, index)
    elif b > r:
        raise ValueError(f"{b} rows of logits, but {r} records")
    if v > 1 << 30 or not 0 <= first <= 2 ** 31 - 1 - v:
        raise ValueError(f"{v} columns from token {first}")
    if counts is not None and (counts.dtype is not torch.int16 or counts.shape != (r, v) or counts.get_device() != index or (v > 1 and counts.stride(1) != 1)):
        _refuse("counts", f"int16 [{r}, {v}] with neighbouring columns on the logits' device are", counts)
    ids = values = None
    k = 0
    if bias is not None:
        ids, values = bias
        if ids.dtype is not torch.int32 or ids.ndim != 2 or ids.shape[0] != r or ids.get_device() != index or not ids.is_contiguous() or ids.shape[1] > MAX_BIASES:
            _refuse("bias ids", f"contiguous int32 [{r}, at most {MAX_BIASES}] on the logits' device are", ids)
        if values.dtype is not torch.float32 or values.shape != ids.shape or values.get_device() != index or not values.is_contiguous():
            _refuse("bias values", f"contiguous fp32 {tuple(ids.shape)} on the logits' device are", values)
        k = ids.shape[1]
    if allowed is not None and (allowed.dtype is not torch.int32 or allowed.ndim != 2 or allowed.shape[0] != r or allowed.shape[1] * 32 < first + v or
                                allowed.get_device() != index or not allowed.is_contiguous()):
        _refuse("allowed", f"contiguous int32 [{r}, at least {(first + v + 31) // 32}] on the logits' device are", allowed)
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty((b, v))
    elif out.shape != logits.shape or out.dtype is not logits.dtype or out.get_device() != index or (v > 1 and out.stride(1) != 1) or (b > 1 and out.stride(0) < v):
        _refuse("out", f"{logits.dtype} {tuple(logits.shape)} with neighbouring columns on the logits' device is", out)
    if b == 0 or v == 0:
        return out
    if index < 0:
        out.copy_(reference.process_logits(logits, records, counts, bias, allowed, rows, first, fill))
        return out
    if b > MAX_ROWS:
        raise ValueError(f"{b} rows of logits, a call takes {MAX_ROWS}")
    if elsewhere(index):
        with torch.cuda.device(index):
            return process_logits(logits, records, counts=counts, bias=bias, allowed=allowed, rows=rows, first=first, fill=fill, out=out)
    check(lib().mfq_process_logits(logits.data_ptr(), out.data_ptr(), _DTYPES[logits.dtype], b, v, logits.stride(0), out.stride(0), records.data_ptr(), r, ptr(counts),
                                   0 if counts is None else counts.stride(0), ptr(ids), ptr(values), k, ptr(allowed), 0 if allowed is None else allowed.shape[1],
                                   ptr(rows), first, fill, stream_ptr()), "process_logits")
    return out


def count_tokens(counts: torch.Tensor, tokens: torch.Tensor, rows: torch.Tensor, *, prompt: bool = False) -> None:
    """Count ``tokens [n]`` int32 in ``counts[rows [n], token]`` (int16 words ``[R, V]``, see the top of this module): as tokens of an
    answer, whose counts stay at 32767 once there, or with ``prompt`` as tokens that the prompt has.  A pair outside the table is left
    out, so a batch may be padded with negative rows.  Calls that count in the same rows follow one another: two at once could bring a count
    past 32767 between them."""
    if counts.dtype is not torch.int16 or counts.ndim != 2 or (counts.shape[1] > 1 and counts.stride(1) != 1) or (counts.shape[0] > 1 and counts.stride(0) < counts.shape[1]):
        _refuse("counts", "int16 [R, V] with neighbouring columns and rows apart are", counts)
    index = counts.get_device()
    _index("tokens", tokens, None, index)
    _index("rows", rows, tokens.numel(), index)
    if counts.numel() == 0 or tokens.numel() == 0:
        return
    if index < 0:
        reference.count_tokens(counts, tokens, rows, prompt)
        return
    if elsewhere(index):
        with torch.cuda.device(index):
            return count_tokens(counts, tokens, rows, prompt=prompt)
    check(lib().mfq_count_tokens(counts.data_ptr(), counts.stride(0), counts.shape[0], counts.shape[1], tokens.data_ptr(), rows.data_ptr(), tokens.numel(), int(prompt),
                                 stream_ptr()), "count_tokens")
