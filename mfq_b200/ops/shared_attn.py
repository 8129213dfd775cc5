"""Decode attention of sequences that share their first pages in groups (:func:`paged_attn_decode_shared`).

What ``paged_attn_decode`` computes, with every group's prefix read once instead of once per sequence.  CPU tensors take the
restatement in :mod:`mfq_b200.ops.reference`.
"""

from __future__ import annotations

import torch

from . import reference
from .lib import Workspace, check, current_device, lib, ptr, stream_ptr

HEAD_DIMS = (64, 128, 256)
SMS = 148


def _pick_splits(units: int, pages: int, per_sm: int, least: int, most: int = 32) -> int:
    """Splits of ``pages`` for a grid of ``units`` CTAs a split: as many as fit one wave of ``per_sm`` CTAs an SM, each of at least ``least`` pages."""
    return max(1, min(SMS * per_sm // max(1, units), pages // least, most))


def _pick_tile(rows: int, d: int) -> int:
    """Query rows of a prefix CTA for groups of ``rows`` query rows a KV head: 16, 32, 64 on mma.sync, 128 and 256 on tcgen05."""
    for tile in (16, 32, 64):
        if rows <= tile:
            return tile
    return 64 if d > 128 else 128 if rows <= 128 else 256


def paged_attn_decode_shared(q: torch.Tensor, kv, block_table: torch.Tensor, seq_lens: torch.Tensor, group_starts: torch.Tensor,
                             prefix_lens: torch.Tensor, *, sm_scale: float, members: torch.Tensor | None = None, q_len: int = 1,
                             max_group: int | None = None, max_prefix: int | None = None, max_tail: int | None = None,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """``q [B * q_len, Hq, D]`` (bf16) against the paged FP8 cache ``kv`` (a :class:`LayerKV`), ``D`` 64, 128 or 256 and at most 16 query heads
    times ``q_len`` to a KV head; ``block_table [B, P]`` and ``seq_lens [B]`` int32 as for ``paged_attn_decode`` (the lengths count the query tokens too).

    * ``members [B]`` int32: batch rows in the order of the groups (default ``0 .. B - 1``);
    * ``group_starts [n + 1]`` int32, ascending: group ``g`` has the rows ``members[group_starts[g] : group_starts[g + 1]]``; rows behind
      the last group are left as ``out`` has them;
    * ``prefix_lens [n]`` int32: the leading tokens whose pages the group's rows share.  Whole pages of them are read through the first
      row's table, the rest through each row's own; 0 shares nothing.

    All of that may change on the device between replays of a graph.  ``max_group`` (rows of a group), ``max_prefix`` and ``max_tail`` (tokens):
    what the host knows of them; they choose the shape of the launches, a wrong one costs time."""
    if q.ndim != 3 or q.dtype != torch.bfloat16 or not q.is_contiguous() or q.shape[2] not in HEAD_DIMS or q_len < 1 or q.shape[0] % q_len:
        raise ValueError(f"q: contiguous bf16 [B * {q_len}, Hq, 64 | 128 | 256] is wanted, got {q.dtype} {tuple(q.shape)}")
    n, hq, d = q.shape
    b, dev = n // q_len, q.device
    pages, hk = kv.k.shape[:2]
    if kv.page_size != 16 or kv.k.dtype != torch.float8_e4m3fn or kv.k.shape != (pages, hk, d // 64, 16, 64) or kv.v.shape != (pages, hk, d, 16) or \
            any(not t.is_contiguous() or t.device != dev for t in (kv.k, kv.v, kv.k_scale, kv.v_scale)):
        raise ValueError(f"kv: contiguous FP8 pages of 16 tokens and {d}-wide heads on {dev} are wanted, got {kv.k.dtype} {tuple(kv.k.shape)} on {kv.k.device}")
    if hq % hk or hq // hk * q_len > 16:
        raise ValueError(f"{hq} query heads on {hk} KV heads in windows of {q_len}: at most 16 query rows a KV head are taken")
    for name, t, shape in (("block_table", block_table, (b, block_table.shape[-1])), ("seq_lens", seq_lens, (b,)), ("group_starts", group_starts, (prefix_lens.numel() + 1,)),
                           ("prefix_lens", prefix_lens, (prefix_lens.numel(),))) + ((("members", members, (b,)),) if members is not None else ()):
        if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name}: contiguous int32 {shape} on {dev} is wanted, got {t.dtype} {tuple(t.shape)} on {t.device}")
    groups, width = prefix_lens.numel(), block_table.shape[1]
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out: contiguous bf16 {tuple(q.shape)} on {dev} is wanted, got {out.dtype} {tuple(out.shape)} on {out.device}")
    if b == 0 or groups == 0:
        return out
    if groups > b:
        raise ValueError(f"{groups} groups of {b} rows")
    if not q.is_cuda:
        reference.paged_attn_decode_shared(q, kv, block_table, seq_lens, group_starts, prefix_lens, sm_scale, members, q_len, out)
        return out
    max_group = b if max_group is None else max(1, min(b, max_group))
    whole = width if max_prefix is None else min(width, max(0, max_prefix) // 16)
    rows = max_group * (hq // hk) * q_len
    tile = _pick_tile(rows, d)
    prefix_splits = _pick_splits(-(-rows // tile) * hk * groups, whole, 1 if tile >= 128 or d > 128 else 3, 8 if tile >= 128 else 4)
    tail_splits = _pick_splits(b * hk, 8, 4 if d <= 128 else 2, 1, 8)
    slots = prefix_splits * (2 if tile == 128 else 1)
    with current_device(dev):
        scratch = torch.empty(n * hq * slots * (d + 2), dtype=torch.float32, device=dev)  # of this call: a workspace would tie streams and graphs together
        split = n * hq * slots * d
        check(lib().mfq_paged_attn_decode_shared(
            ptr(q), ptr(kv.k), ptr(kv.v), ptr(kv.k_scale), ptr(kv.v_scale), ptr(block_table), ptr(seq_lens), ptr(group_starts), ptr(prefix_lens), ptr(members),
            ptr(out), ptr(scratch), scratch.data_ptr() + 4 * split, b, hq, hk, d, width, pages, groups, q_len, tile, prefix_splits, tail_splits,
            float(sm_scale), ptr(Workspace.get(dev).status), stream_ptr()), "paged_attn_decode_shared", 2)
    return out
