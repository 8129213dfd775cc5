"""Decode attention of sequences that share their first pages in groups (:func:`paged_attn_decode_shared`).

What ``paged_attn_decode`` computes, with every group's prefix read once instead of once per sequence where that is faster (heads of 64 and 128).  CPU tensors take the
restatement in :mod:`mfq_b200.ops.reference`.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import reference
from .lib import Workspace, check, elsewhere, lib, ptr, stream_ptr
from .logits import _index, _refuse

HEAD_DIMS = (64, 128, 256)
MAX_ROWS = 65535  # of a batch: blocks of a grid in y
SMS = 148


@lru_cache(maxsize=4096)
def _shape(b: int, per_seq: int, hk: int, d: int, groups: int, group: int, whole: int, tail: int) -> tuple[int, int, int]:
    """(query rows of a prefix CTA, splits of a prefix, CTAs of a sequence's own pages) for ``b`` sequences of ``per_seq`` query rows a KV head, in groups
    of up to ``group`` with ``whole`` pages of a prefix and ``tail`` of their own.  0 splits of a prefix: every sequence is read whole, which is one kernel, and
    all that heads of 256 have.

    The form that is fastest by a model of the kernels in microseconds: a few numbers fitted to 852 shapes on a B200 (1 to 5 groups of 2 to 64
    sequences, equal and ragged, prefixes of 130 to 24000 tokens, heads of 64 and 128), some twenty forms of each measured.  Of 791 of them the chosen form is among
    these: it takes 3 % longer than the fastest on average, and more than 12 % in 61 (55 % at worst: 16 sequences in 5 groups, 1488 tokens and 612 of their own).  Heads of 256
    were not swept."""
    rows, narrow = group * per_seq, per_seq <= 8
    per_sm = 2 if d > 128 else (4 if narrow else 3) + (d == 64)  # CTAs that read pages by warps
    slots_of_gpu = SMS * per_sm
    bandwidth = 1.2e7 / (16 * (2 * d + 8))  # pages of a head, from memory or L2

    def waves(n: int, slots: int) -> float:
        return 1.0 if n <= slots else 0.3 * n / slots + 0.7 * -(-n // slots)

    def pages_of(pages: int, ranks: int, n: int) -> float:  # of n CTAs, four warps each
        each = (0.70 + 0.10 * min(n / SMS, per_sm) if narrow else 0.77 + 0.25 * min(n / SMS, per_sm)) * (1.0 if d <= 128 else 2.0)
        return max(-(-pages // (4 * ranks)) * each * waves(n, slots_of_gpu), b * hk * pages / bandwidth)

    forms = []
    ranks = [r for r in (1, 2, 4, 8) if r == 1 or b * hk * r <= 2 * slots_of_gpu]
    for r in ranks:
        forms.append((4.9 + pages_of(whole + tail, r, b * hk * r) + 0.6 * (r.bit_length() - 1), 16, 0, r))
    tiles = () if d > 128 or whole == 0 or group == 1 else ((8 if rows <= 8 else 16,) if rows <= 32 else ()) + ((128 if rows <= 128 else 256,) if rows > 8 else ())
    for tile in tiles:
        units, blocks = -(-rows // tile) * hk * groups, -(-whole // 8)
        if tile >= 128:  # blocks of eight pages; as many splits as SMs, each of whole blocks, or a power of two
            most = max(1, min(SMS // units, blocks, 32))
            splits_to_try = {s for s in (1, 2, 4, 8, 16, 32) if s <= blocks} | {-(-blocks // -(-blocks // most))}
        else:
            slots_of_tiles = SMS * ((4 if tile == 8 else 3) + (d == 64 and tile == 16))
            splits_to_try = {s for s in (1, 2, 4, 8, 16, 32) if s <= max(1, whole // 4)} | {max(1, min(slots_of_tiles // units, whole // 4, 32))}
        for splits in splits_to_try:
            ctas = units * splits
            if tile >= 128:  # one an SM, where nothing else fits beside it
                t = 0.9 + (2.0 if tile == 128 else 3.6) * -(-blocks // splits) * max(1, -(-ctas // SMS))
                room = max(0, SMS - ctas) * per_sm
            else:
                t = 2.0 + max(-(-whole // (4 * splits)) * (0.92 if tile == 8 else 1.8), units * whole / bandwidth) * waves(ctas, slots_of_tiles)
                room = max(0, slots_of_gpu - ctas)
            parts = splits * (2 if tile == 128 else 1)
            for r in ranks[: 2 if tile >= 128 else 3]:
                n = b * hk * r  # CTAs of the sequences' own pages: those with room beside the prefixes keep it until these are there, the rest come behind
                rest = max(0, n - room)
                whole_t = max(t, pages_of(tail, r, n - rest) if room else 0.0) + (pages_of(tail, r, rest) + 2.4 if rest else 0.0)
                merge = 6.0 + 0.6 * (r.bit_length() - 1) + 0.64 * -(-parts // 8) * -(-per_seq * d // (512 * r)) * waves(n, slots_of_gpu) + 1.3e-6 * b * per_seq * hk * parts * d
                forms.append((whole_t + merge, tile, splits, r))
    return min(forms)[1:]


def paged_attn_decode_shared(q: torch.Tensor, kv, block_table: torch.Tensor, seq_lens: torch.Tensor, group_starts: torch.Tensor,
                             prefix_lens: torch.Tensor, *, sm_scale: float, members: torch.Tensor | None = None, q_len: int = 1,
                             max_group: int | None = None, max_prefix: int | None = None, max_tail: int | None = None,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """``q [B * q_len, Hq, D]`` (bf16) against the paged FP8 cache ``kv`` (a :class:`LayerKV`), ``D`` 64, 128 or 256 and at most 16 query heads
    times ``q_len`` to a KV head; ``block_table [B, P]`` and ``seq_lens [B]`` int32 as for ``paged_attn_decode`` (the lengths count the query tokens too, and go up to
    ``16 P``); at most :data:`MAX_ROWS` sequences.

    * ``members [B]`` int32: batch rows in the order of the groups, each once (default ``0 .. B - 1``);
    * ``group_starts [n + 1]`` int32, ascending: group ``g`` has the rows ``members[group_starts[g] : group_starts[g + 1]]``; rows behind
      the last group are left as ``out`` has them;
    * ``prefix_lens [n]`` int32: the leading tokens whose pages the group's rows share: their tables name the same pages for them.  Whole pages of
      them are read through the table of the group's first row, or through each row's own where sharing would take longer, the rest through each row's
      own; 0 shares nothing.

    Multipliers of the pages are not negative; ``q``, ``out``, the pages and their multipliers begin on 16 bytes.  A page or a member out of range
    is reported by ``Workspace.check``.

    All of the indices may change on the device between replays of a graph.  ``max_group`` (rows of a group), ``max_prefix`` and ``max_tail`` (tokens):
    what the host knows of them; they choose the shape of the launches, a wrong one costs time."""
    if q.ndim != 3 or q.dtype is not torch.bfloat16 or not q.is_contiguous() or q.shape[2] not in HEAD_DIMS or q_len < 1 or q.shape[0] % q_len:
        _refuse("q", f"contiguous bf16 [B * {q_len}, Hq, 64 | 128 | 256] are", q)
    n, hq, d = q.shape
    b, index = n // q_len, q.get_device()
    k, v = kv.k, kv.v
    pages, hk = k.shape[:2]
    if kv.page_size != 16 or k.dtype is not torch.float8_e4m3fn or v.dtype is not torch.float8_e4m3fn or k.shape != (pages, hk, d // 64, 16, 64) or v.shape != (pages, hk, d, 16):
        _refuse("kv", f"FP8 pages of 16 tokens and {d}-wide heads are", k)
    for t in (kv.k_scale, kv.v_scale):
        if t.dtype is not torch.float32 or t.shape != (pages, hk, 16):
            _refuse("kv multipliers", f"fp32 {(pages, hk, 16)} are", t)
    for t in (k, v, kv.k_scale, kv.v_scale):
        if t.get_device() != index or not t.is_contiguous():
            _refuse("kv", "contiguous pages on the device of q are", t)
    if hk < 1 or pages < 1 or hq % hk or hq // hk * q_len > 16:
        raise ValueError(f"{hq} query heads on {hk} KV heads in windows of {q_len}: at most 16 query rows a KV head are taken")
    if block_table.dtype is not torch.int32 or block_table.ndim != 2 or block_table.shape[0] != b or block_table.get_device() != index or not block_table.is_contiguous():
        _refuse("block_table", f"contiguous int32 [{b}, P] on the device of q is", block_table)
    groups, width = prefix_lens.numel(), block_table.shape[1]
    if not 1 <= width < 1 << 27 or b > MAX_ROWS:
        raise ValueError(f"{b} sequences of up to {width} pages: at most {MAX_ROWS}, of 1 to 2^27 - 1")
    _index("seq_lens", seq_lens, b, index)
    _index("group_starts", group_starts, groups + 1, index)
    _index("prefix_lens", prefix_lens, groups, index)
    if members is not None:
        _index("members", members, b, index)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != index or not out.is_contiguous():
        _refuse("out", f"contiguous bf16 {tuple(q.shape)} on the device of q is", out)
    wide = [t.data_ptr() for t in (q, k, v, kv.k_scale, kv.v_scale, out)]
    if (wide[0] | wide[1] | wide[2] | wide[3] | wide[4] | wide[5]) & 15:
        raise ValueError("q, out, the pages and their multipliers have to begin on 16 bytes")
    if b == 0 or groups == 0:
        return out
    if groups > b:
        raise ValueError(f"{groups} groups of {b} rows")
    if index < 0:
        reference.paged_attn_decode_shared(q, kv, block_table, seq_lens, group_starts, prefix_lens, sm_scale, members, q_len, out)
        return out
    if elsewhere(index):
        with torch.cuda.device(index):
            return paged_attn_decode_shared(q, kv, block_table, seq_lens, group_starts, prefix_lens, sm_scale=sm_scale, members=members, q_len=q_len,
                                            max_group=max_group, max_prefix=max_prefix, max_tail=max_tail, out=out)
    tile, prefix_splits, tail_splits = _shape(b, hq // hk * q_len, hk, d, groups, b if max_group is None else max(1, min(b, max_group)),
                                              width if max_prefix is None else min(width, max(0, max_prefix) // 16),
                                              width if max_tail is None else min(width, max(0, max_tail) // 16 + 1))
    parts = n * hq * prefix_splits * (2 if tile == 128 else 1)
    scratch = torch.empty(parts * (d + 2), dtype=torch.float32, device=q.device) if parts else None  # of this call: a workspace would tie streams and graphs together
    at = scratch.data_ptr() if parts else 0
    check(lib().mfq_paged_attn_decode_shared(
        *wide[:5], block_table.data_ptr(), seq_lens.data_ptr(), group_starts.data_ptr(), prefix_lens.data_ptr(), ptr(members), wide[5], at, at + 4 * parts * d, b, hq, hk, d, width, pages, groups, q_len, tile, prefix_splits, tail_splits,
        sm_scale, Workspace.get(q.device).status.data_ptr(), stream_ptr()), "paged_attn_decode_shared", 2 if prefix_splits else 1)
    return out
