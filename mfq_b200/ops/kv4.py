"""A KV cache held in 4 bits: writing tokens into its pages (:func:`kv4_write`), reading them back (:func:`kv4_gather`), and decode attention over the pages
(:func:`paged_attn_decode_kv4`).  The pool of a layer is a :class:`~mfq_b200.engine.kv_cache.LayerKV4`.

A head's vector is held in groups of 64 values.  A group has a bf16 scale ``s``, a bf16 minimum ``m`` and a code ``c`` of 0 to 15 for each value, which
stands for ``m + s c``: ``m`` is the largest bf16 that is not above the group's values, ``s`` the least one whose 15-fold reaches the largest value,
``c`` the integer nearest to ``(x - m) / s``, ties to even, and 0 where ``s`` is 0.  So a value is off by at most ``s / 2``.  A group with a NaN or a magnitude above
2^126 stands for NaN.  4.5 bits a value, 1.83 times the tokens of the FP8 pages; a value of normally distributed groups is off by 9 % of their deviation.

The reference holds its pages in fp16, bf16 or TurboQuant codes (``cpp_runtime/backends/cuda/kernels/kv_quantization.cu``); this format is this repository's own.

CPU tensors take the restatements in :mod:`mfq_b200.ops.reference`.
"""

from __future__ import annotations

import math
from functools import lru_cache

import numpy as np
import torch

from . import reference
from .lib import Workspace, check, elsewhere, lib, ptr, stream_ptr
from .logits import _DTYPES, _index, _refuse

RECORDS = {18 * 64: 64, 18 * 128: 128, 18 * 256: 256}  # bytes of a page and head: head dim
SMS = 148
LEAST = 4  # pairs of pages of a share: one a warp
MAX_PAGES = 1 << 27  # of a pool, and of a table's row: slots and lengths are int32
MAX_HEADS = 65536
MAX_SEQS = 1 << 30  # of a table: they are counted in 32 bits, as tokens are


def _pool(kv, index: int) -> tuple[int, int, int]:
    """(pages, heads, head dim) of a pool that the kernels take."""
    data = kv.data
    shape = data.shape
    if kv.page_size != 16 or data.dtype is not torch.uint8 or len(shape) != 3 or shape[2] not in RECORDS or not data.is_contiguous() or data.get_device() != index or \
            not 1 <= shape[0] <= MAX_PAGES or not 1 <= shape[1] <= MAX_HEADS:
        _refuse("kv", f"contiguous uint8 [at most {MAX_PAGES} pages of 16 tokens, at most {MAX_HEADS} heads, 18 * (64 | 128 | 256)] on the device of the others are", data)
    if data.data_ptr() & 15:
        raise ValueError("kv: the pool has to begin on 16 bytes")
    return shape[0], shape[1], RECORDS[shape[2]]


def _rows(name: str, t: torch.Tensor, n: int, heads: int, d: int, index: int, *, written: bool = False) -> tuple[int, int]:
    """Strides of tokens and heads of ``t [n, heads, d]``, which is read or written 16 bytes at a time."""
    if t.shape != (n, heads, d) or t.dtype not in _DTYPES or t.get_device() != index or t.stride(2) != 1 or n >= 1 << 31:
        _refuse(name, f"bf16, fp16 or fp32 [{n} below 2^31, {heads}, {d}] with neighbouring dims on the device of the others are", t)
    a, b, _ = t.stride()
    a, b, unit = a if n > 1 else 0, b if heads > 1 else 0, 16 // t.element_size()
    if (a | b) & (unit - 1) or t.data_ptr() & 15:
        raise ValueError(f"{name}: tokens and heads have to begin on 16 bytes, got strides {t.stride()} of {t.dtype}")
    if written:  # heads inside a token or tokens inside a head: no two of them over one another
        (near, count), (far, more) = sorted(((a, n) if n > 1 else (0, 1), (b, heads) if heads > 1 else (0, 1)))
        if (count > 1 and near < d) or (more > 1 and far < (count - 1) * near + d):
            raise ValueError(f"{name}: rows lie over one another, strides {t.stride()}")
    return a, b


def _meet(gap: int, n: int, heads: int, d: int, ks: tuple[int, int], vs: tuple[int, int]) -> bool:
    """Whether a row of ``v_out`` lies over one of ``k_out``: ``[n, heads]`` rows of ``d`` elements each, strides ``vs`` and ``ks``, ``gap`` elements from k's first to v's.
    Rows of one output are known not to lie over one another."""
    if gap >= (n - 1) * ks[0] + (heads - 1) * ks[1] + d or -gap >= (n - 1) * vs[0] + (heads - 1) * vs[1] + d:
        return False
    if ks == vs:  # a row of v is i near strides, j far ones and the gap from one of k
        (near, count), (far, more) = sorted(((ks[0], n), (ks[1], heads)))
        for j in range(-(gap // far) - 2, -(gap // far) + 3) if far else (0,):
            if -more < j < more:
                rest = -gap - j * far
                i = rest // near if near else 0
                if any(-count < e < count and abs(e * near - rest) < d for e in (i, i + 1)):
                    return True
        return False
    at = [(np.arange(n, dtype=np.int64)[:, None] * a + np.arange(heads, dtype=np.int64) * b).ravel() for a, b in (ks, vs)]
    return bool((np.diff(np.sort(np.concatenate([at[0], at[1] + gap]))) < d).any())


def kv4_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, kv) -> None:
    """Quantise ``k`` and ``v [T, heads, D]`` (bf16, fp16 or fp32; slices of a fused projection will do: tokens and heads may lie apart, in steps of 16 bytes)
    into the pages of ``kv`` (a :class:`~mfq_b200.engine.kv_cache.LayerKV4`) at ``slots [T]`` int32: ``page * 16 + place``.  Tokens of negative slots are left out, so a
    batch may be padded; a slot behind the pool is left out and reported by ``Workspace.check``.  A slot that several tokens of a call name holds codes
    and parameters of any of them: a step writes a token once."""
    index = k.get_device()
    pages, heads, d = _pool(kv, index)
    n = k.shape[0] if k.ndim == 3 else 0
    ks, vs = _rows("k", k, n, heads, d, index), _rows("v", v, n, heads, d, index)
    if v.dtype is not k.dtype:
        _refuse("v", f"{k.dtype}, as k is,", v)
    _index("slots", slots, n, index)
    if n == 0:
        return
    if index < 0:
        reference.kv4_write(kv, k, v, slots)
        return
    if elsewhere(index):
        with torch.cuda.device(index):
            return kv4_write(k, v, slots, kv)
    check(lib().mfq_kv4_write(k.data_ptr(), v.data_ptr(), slots.data_ptr(), kv.data.data_ptr(), _DTYPES[k.dtype], n, heads, d, pages, *ks, *vs,
                              Workspace.get(k.device).status.data_ptr(), stream_ptr()), "kv4_write")


@lru_cache(maxsize=4096)
def _shape(units: int, cols: int, d: int, pages: int) -> tuple[int, int]:
    """(CTAs of a unit's cluster, 0) or (0, CTAs that share all pairs of pages) for ``units`` units of ``cols`` columns and up to ``pages`` pages.

    The fastest by a model in microseconds, its numbers fitted on a B200 to 1 to 200 sequences of 48 to 32000 tokens (8 KV heads of 128, 4 columns, bf16), in eight forms each.
    Four warps take four pairs in a round.  With n CTAs an SM a round takes 0.45 + 0.29 n, what is before and behind the rounds 1.4 for each of them, a further wave 1.5; shares need a
    second kernel, 3 for every unit or piece of one, and a sum over a unit's pieces.  Replayed, in single CTAs | in pairs | in 592 shares: 64 rows of 4096 tokens 60 | 66 | 63; of 16384
    218 | 200 | 201; 3 of 2000: 16 | 12 | 14, in clusters of eight 10; 1 of 32000: 188 | 98 | 25, in 296 shares 21, in 148, as is chosen, 23 to 25, in clusters of eight 31.
    Other heads and columns enter by ``work``, types not at all: of 30 shapes with heads of 64 to 256, 2 to 16 rows a head and both types the choice was within 4 % of the fastest
    form in 28; 8 of 8000 with heads of 64 took 16.4 instead of 14.4, and 1 of 32000."""
    each = 2 if d == 256 or cols == 16 else 4  # CTAs that an SM holds
    work = {64: 0.6, 128: 1.0, 256: 2.0}[d] * {4: 1.0, 8: 1.2, 16: 2.0}[cols]
    pairs = max(1, (pages + 1) // 2)

    def rounds(n: float, r: float) -> float:
        waves = math.ceil(n / each)
        n = math.ceil(n) if 2 < n <= each else max(1.0, n)
        return n * (0.29 * work * r + 1.4) + (0.45 * work * r + 1.5) * waves

    forms = [(7.5 + rounds(units * c / SMS, -(-pairs // (4 * c))), c, 0) for c in (1, 2, 4, 8) if c == 1 or 2 * c <= pairs]
    for k in range(1, each + 1):
        ctas = min(SMS * k, units * -(-pairs // LEAST))
        forms.append((13.5 + rounds(ctas / SMS, units * pairs / (4 * ctas)) + 3 * units / ctas + 0.15 * ctas / units, 0, ctas))
    return min(forms)[1:]


def _table(block_table: torch.Tensor, b: int, index: int) -> int:
    shape = block_table.shape
    if block_table.dtype is not torch.int32 or len(shape) != 2 or shape[0] != b or block_table.get_device() != index or not block_table.is_contiguous() or \
            not 1 <= shape[1] < MAX_PAGES or b > MAX_SEQS:
        _refuse("block_table", f"contiguous int32 [{b}, at most {MAX_SEQS}; 1 to {MAX_PAGES - 1} pages] on the device of the others is", block_table)
    return shape[1]


def kv4_gather(kv, block_table: torch.Tensor, starts: torch.Tensor, tokens: int | None = None, *, first: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16, k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cached keys and values of ragged sequences as packed rows ``[tokens, heads, D]`` of ``dtype`` (bf16, fp16 or fp32), for the attention of a prompt's next chunk.

    * ``block_table [B, P]`` int32: the sequences' pages;
    * ``starts [B + 1]`` int32, ascending: rows ``starts[i] : starts[i + 1]`` are sequence ``i``'s; rows in front of the first and behind the last are left as they were;
    * ``first [B]`` int32: the position of each sequence's first row (default 0);
    * ``k_out`` / ``v_out``: where to, both or neither (tokens and heads may lie apart, in steps of 16 bytes, neither's rows over others of it or of the other); they say ``tokens`` and ``dtype`` then.

    A row without a page in the table, or whose page is out of range, is left as it was and reported by ``Workspace.check``."""
    index = block_table.get_device()
    pages, heads, d = _pool(kv, index)
    if k_out is None and v_out is None:
        if tokens is None or not 0 <= tokens < 1 << 31:
            raise ValueError(f"tokens: 0 to 2^31 - 1 rows wanted, got {tokens}")
        if dtype not in _DTYPES:
            raise ValueError(f"dtype: bf16, fp16 or fp32 wanted, got {dtype}")
        n, ks = tokens, (heads * d, d)
        vs = ks
        k_out = torch.empty((n, heads, d), dtype=dtype, device=block_table.device)
        v_out = torch.empty_like(k_out)
    elif k_out is None or v_out is None:
        raise ValueError("k_out and v_out are given together")
    else:
        n = k_out.shape[0] if k_out.ndim == 3 else 0
        if tokens is not None and tokens != n:
            raise ValueError(f"tokens: {tokens}, but k_out has {n} rows")
        ks, vs = _rows("k_out", k_out, n, heads, d, index, written=True), _rows("v_out", v_out, n, heads, d, index, written=True)
        if v_out.dtype is not k_out.dtype:
            _refuse("v_out", f"{k_out.dtype}, as k_out is,", v_out)
        if n and _meet((v_out.data_ptr() - k_out.data_ptr()) // k_out.element_size(), n, heads, d, ks, vs):
            raise ValueError("v_out: lies over k_out")
    b = block_table.shape[0] if block_table.ndim == 2 else -1
    width = _table(block_table, b, index)
    _index("starts", starts, b + 1, index)
    if first is not None:
        _index("first", first, b, index)
    if n == 0 or b == 0:
        return k_out, v_out
    if index < 0:
        reference.kv4_gather(kv, block_table, starts, first, k_out, v_out)
        return k_out, v_out
    if elsewhere(index):
        with torch.cuda.device(index):
            return kv4_gather(kv, block_table, starts, tokens, first=first, k_out=k_out, v_out=v_out)
    check(lib().mfq_kv4_gather(kv.data.data_ptr(), block_table.data_ptr(), starts.data_ptr(), ptr(first), k_out.data_ptr(), v_out.data_ptr(), _DTYPES[k_out.dtype], b, n, heads,
                               d, width, pages, *ks, *vs, Workspace.get(block_table.device).status.data_ptr(), stream_ptr()), "kv4_gather")
    return k_out, v_out


def paged_attn_decode_kv4(q: torch.Tensor, kv, block_table: torch.Tensor, seq_lens: torch.Tensor, *, sm_scale: float, q_len: int = 1,
                          max_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """What ``paged_attn_decode`` computes, over pages held in 4 bits: ``q [B * q_len, Hq, D]`` (bf16 or fp16) against the cache ``kv`` (a
    :class:`~mfq_b200.engine.kv_cache.LayerKV4`); ``block_table [B, P]`` and ``seq_lens [B]`` int32.  The lengths count the query tokens too and go up to ``16 P``; a
    window's query sees no later token of it, and one that sees nothing has zeros.  Any number of query heads to a KV head.

    The tables and lengths may change on the device between replays of a graph.  ``max_len``: what the host knows of the longest sequence; it chooses the shape of the
    launches, a wrong one costs time.  A page out of range that a sequence reads is reported by ``Workspace.check``; ``q`` and ``out`` begin on 16 bytes."""
    index = q.get_device()
    pages, hk, d = _pool(kv, index)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3 or (dtype is not torch.bfloat16 and dtype is not torch.float16) or not q.is_contiguous() or shape[2] != d or q_len < 1 or shape[0] % q_len:
        _refuse("q", f"contiguous bf16 or fp16 [B * {q_len}, Hq, {d}] are", q)
    n, hq, _ = shape
    b = n // q_len
    if hq < 1 or hq % hk:
        raise ValueError(f"{hq} query heads on {hk} KV heads")
    width = _table(block_table, b, index)
    _index("seq_lens", seq_lens, b, index)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != shape or out.dtype is not dtype or out.get_device() != index or not out.is_contiguous():
        _refuse("out", f"contiguous {dtype} {tuple(shape)} on the device of q is", out)
    at, to = q.data_ptr(), out.data_ptr()
    if (at | to) & 15:
        raise ValueError("q and out have to begin on 16 bytes")
    if b == 0:
        return out
    if index < 0:
        out.copy_(reference.paged_attn_decode_kv4(q, kv, block_table, seq_lens, sm_scale, q_len))
        return out
    if elsewhere(index):
        with torch.cuda.device(index):
            return paged_attn_decode_kv4(q, kv, block_table, seq_lens, sm_scale=sm_scale, q_len=q_len, max_len=max_len, out=out)
    rows = hq // hk * q_len
    cols = 4 if rows <= 4 else (8 if rows <= 8 or d == 256 else 16)
    cluster, ctas = _shape(b * hk * -(-rows // cols), cols, d, width if max_len is None else max(1, min(width, (max_len + 15) // 16)))
    scratch = torch.empty(ctas * (4 + 2 * cols * (d + 4)), dtype=torch.float32, device=q.device) if ctas else None  # of this call: a workspace would tie streams and graphs together
    check(lib().mfq_paged_attn_decode_kv4(at, kv.data.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), to, ptr(scratch), int(dtype is torch.float16), b, hq, hk, d, width,
                                          pages, q_len, ctas or cluster, LEAST, sm_scale, Workspace.get(q.device).status.data_ptr(), stream_ptr()), "paged_attn_decode_kv4", 2 if ctas else 1)
    return out
