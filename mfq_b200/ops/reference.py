"""Plain PyTorch (fp32) restatements of every fused kernel: the numerical oracle of the GPU tests and the
CPU execution path of the models."""

from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0
FP8 = torch.float8_e4m3fn


def quant_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    xf = x.float()
    scale = xf.abs().amax(-1).clamp_min(1e-12) / E4M3_MAX
    q = (xf / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(FP8)
    return q, scale


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()
    return y.to(torch.bfloat16)


def rmsnorm_quant(x, w, eps, residual=None):
    if residual is not None:
        x = (x.float() + residual.float()).to(torch.bfloat16)
    y = rmsnorm(x, w, eps)
    q, s = quant_rows(y)
    return q, s, y, x


def silu_mul_quant(gate_up: torch.Tensor):
    i = gate_up.shape[1] // 2
    g, u = gate_up[:, :i].float(), gate_up[:, i:].float()
    h = (g / (1 + torch.exp(-g)) * u).to(torch.bfloat16)
    return quant_rows(h)


def dequant_block(w_q: torch.Tensor, w_scale: torch.Tensor, block: int = 128) -> torch.Tensor:
    n, k = w_q.shape
    s = w_scale.repeat_interleave(block, 0)[:n].repeat_interleave(block, 1)[:, :k]
    return w_q.float() * s


def fp8_gemm(x_q, x_scale, w_q, w_scale, residual=None) -> torch.Tensor:
    y = (x_q.float() * x_scale[:, None]) @ dequant_block(w_q, w_scale).T
    if residual is not None:
        y = y + residual.float()
    return y.to(torch.bfloat16)


def rope(x: torch.Tensor, positions: torch.Tensor, theta: float, rot: int | None = None, scaling=None) -> torch.Tensor:
    """``x [T, H, D]``; rotate-half pairing (i, i + rot/2) over the first ``rot`` dims.  ``scaling``: a
    :class:`~mfq_b200.models.rope_scaling.YarnScaling` (blended frequencies, cos / sin times its attention factor)."""
    d = x.shape[-1]
    rot = rot or d
    half = rot // 2
    if scaling is not None:
        inv, mscale = scaling.inv_freq(rot, theta, x.device), scaling.mscale
    else:
        inv, mscale = torch.exp2(-math.log2(theta) * (2 * torch.arange(half, device=x.device, dtype=torch.float32)) / rot), 1.0
    ang = positions.float()[:, None] * inv[None, :]
    c, s = ang.cos()[:, None, :] * mscale, ang.sin()[:, None, :] * mscale
    xf = x.float()
    a, b = xf[..., :half], xf[..., half:rot]
    out = xf.clone()
    out[..., :half] = a * c - b * s
    out[..., half:rot] = b * c + a * s
    return out.to(torch.bfloat16)


def quant_kv(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``[T, H, D]`` bf16 -> fp8 codes + one multiplier per (token, head)."""
    xf = x.float()
    scale = xf.abs().amax(-1).clamp_min(1e-12) / E4M3_MAX
    return (xf / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(FP8), scale


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sm_scale: float, causal_offset: int | None = None):
    """``q [Tq, Hq, D]``, ``k/v [Tk, Hk, D]`` (float).  Query i sees keys ``<= i + causal_offset``."""
    tq, hq, d = q.shape
    tk, hk, _ = k.shape
    g = hq // hk
    kf = k.float().repeat_interleave(g, 1)
    vf = v.float().repeat_interleave(g, 1)
    s = torch.einsum("qhd,khd->hqk", q.float(), kf) * sm_scale
    if causal_offset is not None:
        qi = torch.arange(tq, device=q.device)[:, None] + causal_offset
        ki = torch.arange(tk, device=q.device)[None, :]
        s = s.masked_fill((ki > qi)[None], float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.einsum("hqk,khd->qhd", p, vf).to(torch.bfloat16)


def gather_paged(kv, block_table_row: torch.Tensor, length: int):
    """Dequantized ``k, v [length, Hk, D]`` of one sequence from a :class:`LayerKV` (physical page layout)."""
    pos = torch.arange(length, device=kv.k.device)
    return gather_slots(kv, block_table_row.long()[pos // kv.page_size] * kv.page_size + pos % kv.page_size)


def gather_slots(kv, slots: torch.Tensor):
    """Dequantized ``k, v [T, Hk, D]`` rows at physical slots (page * page_size + offset)."""
    from ..engine.kv_cache import V_SLOT_OF_TOKEN
    ps = kv.page_size
    pages, off = (slots // ps).long(), (slots % ps).long()
    k = kv.k[pages, :, :, off]  # [T, Hk, D/64, 64]
    k = k.reshape(k.shape[0], k.shape[1], -1).float() * kv.k_scale[pages, :, off][..., None]
    vslot = torch.tensor(V_SLOT_OF_TOKEN, device=slots.device)[off]
    v = kv.v[pages, :, :, vslot].float() * kv.v_scale[pages, :, off][..., None]
    return k, v


def paged_attn_decode(q, kv, block_table, seq_lens, sm_scale, q_len: int = 1):
    outs = []
    b = q.shape[0] // q_len
    for i in range(b):
        n = int(seq_lens[i])
        if n <= 0:  # an unused row of the batch bucket: nothing to attend to (the GPU kernel writes zeros too)
            outs.append(torch.zeros_like(q[i * q_len : (i + 1) * q_len]))
            continue
        k, v = gather_paged(kv, block_table[i], n)
        outs.append(attention(q[i * q_len : (i + 1) * q_len], k, v, sm_scale, causal_offset=n - q_len))
    return torch.cat(outs, 0)


def paged_attn_decode_shared(q, kv, block_table, seq_lens, group_starts, prefix_lens, sm_scale, members, q_len: int, out) -> None:
    starts, width = group_starts.tolist(), block_table.shape[1]
    order = list(range(seq_lens.numel())) if members is None else members.tolist()
    for g, prefix in enumerate(prefix_lens.tolist()):
        rows = order[starts[g] : starts[g + 1]]
        front = min(max(0, prefix) // kv.page_size, width)
        for r in rows:
            table = torch.cat([block_table[rows[0], :front], block_table[r, front:]])
            n = min(int(seq_lens[r]), width * kv.page_size)
            at = slice(r * q_len, (r + 1) * q_len)
            if n <= 0:
                out[at] = 0
                continue
            k, v = gather_paged(kv, table, n)
            o = attention(q[at], k, v, sm_scale, causal_offset=n - q_len)
            if n < q_len:  # a window's queries in front of the sequence's first token see nothing
                o[: q_len - n] = 0
            out[at] = o


def write_kv(kv, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    from ..engine.kv_cache import V_SLOT_OF_TOKEN
    kq, ks = quant_kv(k)
    vq, vs = quant_kv(v)
    ok = slots >= 0
    pages, off = (slots[ok] // kv.page_size).long(), (slots[ok] % kv.page_size).long()
    kq, vq, ks, vs = kq[ok], vq[ok], ks[ok], vs[ok]
    t, hk, d = kq.shape
    kv.k[pages, :, :, off] = kq.reshape(t, hk, d // 64, 64)
    vslot = torch.tensor(V_SLOT_OF_TOKEN, device=slots.device)[off]
    kv.v[pages, :, :, vslot] = vq
    kv.k_scale[pages, :, off] = ks
    kv.v_scale[pages, :, off] = vs


def process_logits(logits, records, counts=None, bias=None, allowed=None, rows=None, first: int = 0, fill: float = float("-inf")) -> torch.Tensor:
    b, v = logits.shape
    rows = torch.arange(b, device=logits.device) if rows is None else rows.long()
    known = (rows >= 0) & (rows < records.shape[0])
    rows = torch.where(known, rows, 0)
    l = logits.float()
    if bias is not None and bias[0].shape[1]:
        ids, values = bias[0][rows].long() - first, bias[1][rows]
        ok = (bias[0][rows] >= 0) & (ids >= 0) & (ids < v)
        l = l + torch.zeros_like(l).scatter_add_(1, ids.clamp(0, v - 1), torch.where(ok, values, torch.zeros_like(values)))
    if counts is not None:
        presence, frequency, repetition = (records[rows, i].view(torch.float32)[:, None] for i in (3, 4, 5))
        on = (presence != 0) | (frequency != 0) | (repetition != 1)
        word = counts[rows].int() & 0xFFFF
        n = (word & 0x7FFF).float()
        l = torch.where(on & (word != 0), torch.where(l > 0, l / repetition, l * repetition), l)
        l = torch.where(on & (n > 0), l - (presence + frequency * n), l)
    if allowed is not None:
        ids = torch.arange(first, first + v, device=logits.device)
        l = torch.where((allowed[rows][:, ids // 32] >> (ids % 32).int()) & 1 != 0, l, torch.full_like(l, fill))
    return torch.where(known[:, None], l.to(logits.dtype), logits)


def count_tokens(counts, tokens, rows, prompt: bool = False) -> None:
    ok = (tokens >= 0) & (tokens < counts.shape[1]) & (rows >= 0) & (rows < counts.shape[0])
    t, r = tokens[ok].long(), rows[ok].long()
    word = counts[r, t].int() & 0xFFFF
    if prompt:
        word = word | 0x8000
    else:
        pair, times = torch.unique(r * counts.shape[1] + t, return_counts=True)
        r, t = pair // counts.shape[1], pair % counts.shape[1]
        word = counts[r, t].int() & 0xFFFF
        word = (word & 0x8000) | ((word & 0x7FFF) + times.int()).clamp(max=0x7FFF)
    counts[r, t] = torch.where(word >= 0x8000, word - 0x10000, word).to(torch.int16)


def plan_batch(plan, block_table, rows, past, counts, tokens: int, page_size: int, pages=None) -> None:
    for t, empty in ((plan.positions, 0), (plan.slots, -1), (plan.tok_seq, -1), (plan.q_starts, 0), (plan.seq_lens, 0), (plan.block_table, 0)):
        t.fill_(empty)
    r, n, c = (t.tolist() for t in (rows, past, counts))
    table_rows, width = block_table.shape

    def whole(x: int) -> int:
        return -(-x // page_size)

    def code() -> int:  # of a refusal: the latest rule that a request breaks, then the sums
        bad = [0]
        for i, (row, a, m) in enumerate(zip(r, n, c)):
            if not 0 <= row < table_rows or a < 0 or m < 0:
                bad.append(1)
            elif a + m > width * page_size:
                bad.append(2)
            elif pages is not None and row in [q for q, x, y in zip(r[:i], n, c) if x >= 0 and y >= 0 and x + y <= width * page_size]:
                bad.append(1)
        if not max(bad) and sum(c) > tokens:
            return 2
        if not max(bad) and pages is not None and sum(whole(a + m) - whole(a) for a, m in zip(n, c)) > pages.numel():
            return 3
        return max(bad)

    refused = code()
    plan.info[0], plan.info[1] = -refused, 0
    if refused:
        return
    at = taken = 0
    for i, (row, a, m) in enumerate(zip(r, n, c)):
        have, need = whole(a), whole(a + m)
        if pages is not None:
            block_table[row, have:need] = pages[taken : taken + max(0, need - have)]
            taken += need - have
        mine = block_table[row, :need]
        pos = torch.arange(a, a + m, dtype=torch.int32)
        plan.positions[at : at + m] = pos
        plan.slots[at : at + m] = mine[(pos // page_size).long()] * page_size + pos % page_size
        plan.tok_seq[at : at + m] = i
        at += m
        plan.q_starts[i + 1], plan.seq_lens[i] = at, a + m
        plan.block_table[i, :need] = mine
    plan.info[0], plan.info[1] = at, taken
