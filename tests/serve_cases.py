"""Logits, counts and plans for the tests of the operators of a served batch, with the definitions in 64 bits."""

import math

import numpy as np
import torch

VALUE = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


def records(penalties, device="cpu"):
    """Sampling records of ``[(presence, frequency, repetition)]``."""
    t = torch.zeros((len(penalties), 8), dtype=torch.float32)
    for i, p in enumerate(penalties):
        t[i, 3:6] = torch.tensor(p)
    t[:, 0], t[:, 2] = 0.7, 0.9
    return t.view(torch.int32).to(device)


def words(mask: np.ndarray, device="cpu"):
    """Bit words of a truth table ``[R, ids]``."""
    r, n = mask.shape
    padded = np.zeros((r, -(-n // 32) * 32), dtype=np.uint8)
    padded[:, :n] = mask
    return torch.from_numpy(np.packbits(padded, axis=1, bitorder="little").view(np.int32).copy()).to(device)


def exact_logits(logits, recs, counts, bias, mask, rows, first, fill):
    """Row by row and id by id, with how large the values were on the way: (values in 64 bits, magnitudes, whether masked)."""
    x = logits.detach().cpu().double().numpy().copy()
    big, masked = np.abs(x), np.zeros(x.shape, dtype=bool)
    penalties = recs.cpu().view(torch.float32).double().numpy()[:, 3:6]
    with np.errstate(all="ignore"):
        for b in range(x.shape[0]):
            r = b if rows is None else int(rows[b])
            if not 0 <= r < penalties.shape[0]:
                continue
            presence, frequency, repetition = penalties[r]
            if bias is not None:
                for i, v in zip(bias[0][r].tolist(), bias[1][r].tolist()):
                    if i >= 0 and first <= i < first + x.shape[1]:
                        x[b, i - first] += v
                        big[b, i - first] += abs(v)
            if counts is not None:
                word = counts[r].cpu().numpy().astype(np.int64) & 0xFFFF
                n = word & 0x7FFF
                x[b] = np.where(word > 0, np.where(x[b] > 0, x[b] / repetition, x[b] * repetition), x[b])
                x[b] = np.where(n > 0, x[b] - (presence + frequency * n), x[b])
                big[b] = big[b] * max(1.0, repetition, 1 / repetition if repetition else 1.0) + abs(presence) + abs(frequency) * n
            if mask is not None:
                masked[b] = ~mask[r, first : first + x.shape[1]]
                x[b, masked[b]] = fill
    return x, big, masked


def assert_logits(got, want, big, masked, fill):
    """At most eight fp32 operations on the way (each off by 2^-24 of what it has), then one rounding to the type of the logits."""
    t = got.dtype
    y = got.detach().cpu().double().numpy()
    assert np.array_equal(y[masked], np.full(int(masked.sum()), float(torch.tensor(fill, dtype=torch.float32).to(t))))
    y, want, big = y[~masked], want[~masked], big[~masked]
    top = float(torch.finfo(t).max)
    odd = ~np.isfinite(want) | (np.abs(want) >= top)
    assert np.array_equal(np.isnan(y), np.isnan(want))
    sure = odd & ~np.isnan(want)
    assert np.array_equal(np.sign(y[sure]), np.sign(want[sure])) and (np.abs(y[sure]) >= top).all()
    y, want, big = y[~odd], want[~odd], big[~odd]
    assert np.isfinite(y).all()
    limit = VALUE[t] * np.abs(want) + (1 + VALUE[t]) * 8 * 2.0 ** -24 * big + torch.finfo(t).smallest_normal * 2 * VALUE[t]
    off = np.abs(y - want) - limit
    assert (off <= 0).all(), f"off by up to {off.max():.3g} more than the roundings explain"


def exact_counts(counts, tokens, rows, prompt):
    out = counts.cpu().numpy().astype(np.int64) & 0xFFFF
    for t, r in zip(tokens.tolist(), rows.tolist()):
        if 0 <= r < out.shape[0] and 0 <= t < out.shape[1]:
            w = int(out[r, t])
            out[r, t] = w | 0x8000 if prompt else (w & 0x8000) | min((w & 0x7FFF) + 1, 0x7FFF)
    return out


def logits_case(seed, b, r, v, dtype, *, first=0, k=0, mask=False, counted=True, mapped=False, odd=False, device="cpu"):
    """A drawn batch: (arguments of ``process_logits``, truth table of the mask)."""
    g = torch.Generator().manual_seed(seed)
    pad = 0 if not odd else 3
    logits = torch.randn((b, v + pad), generator=g).mul_(4).to(dtype)[:, :v]
    recs = records([[(0.0, 0.0, 1.0), (0.6, 0.2, 1.2), (0.0, 0.0, 0.8), (-0.5, 0.1, 1.0)][i % 4] for i in range(r)])
    counts = None
    if counted:
        counts = torch.randint(0, 4, (r, v + pad), generator=g, dtype=torch.int32)
        counts = torch.where(torch.rand(counts.shape, generator=g) < 0.7, 0, counts)
        counts = counts - 32768 * (torch.rand(counts.shape, generator=g) < 0.1).int()
        counts = counts.to(torch.int16)[:, :v]
    bias = None
    if k:
        ids = torch.randint(-1, first + v + 40, (r, k), generator=g, dtype=torch.int32)  # some of other shards, some unused
        if k > 4:
            ids[:, 3] = ids[:, 1]  # an id twice
        bias = (ids, torch.randn((r, k), generator=g).mul_(5))
    table = None
    if mask:
        table = (torch.rand((r, first + v), generator=g) < 0.4).numpy()
        table[0] = False  # nothing allowed
        if r > 1:
            table[1] = True
    rows = None
    if mapped:
        rows = torch.randint(-1, r + 1, (b,), generator=g, dtype=torch.int32)
    args = dict(logits=logits.to(device), records=recs.to(device), counts=None if counts is None else counts.to(device),
                bias=None if bias is None else tuple(x.to(device) for x in bias), allowed=None if table is None else words(table, device),
                rows=None if rows is None else rows.to(device), first=first)
    return args, table


LOGITS = [  # b, r, v, what else
    (1, 1, 1, {}), (1, 1, 7, {"mask": True}), (2, 2, 8, {"k": 1}), (3, 5, 2047, {"mask": True, "k": 9, "mapped": True}), (2, 2, 2048, {"mask": True, "k": 300}),
    (4, 4, 2049, {"odd": True, "mask": True, "k": 40}), (5, 3, 6000, {"mask": True, "k": 1024, "mapped": True}), (2, 2, 4104, {"first": 40, "mask": True, "k": 30}),
    (2, 3, 1001, {"first": 333, "mask": True, "k": 60, "odd": True}), (3, 3, 5000, {"counted": False, "mask": True}), (2, 2, 9, {"k": 3000}), (2, 2, 7000, {"k": 2500}), (2, 2, 128256, {"k": 5})]


def plan_case(seed, b, most, past, rows=None, ps=16, pages=False, wide=None, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    counts = torch.randint(0, most + 1, (b,), generator=g)
    pasts = torch.randint(0, past + 1, (b,), generator=g)
    rows = rows or b + 3
    wide = wide or int(math.ceil((most + past) / ps)) + 1
    table = torch.randperm(rows * wide, generator=g).add_(1).view(rows, wide).to(torch.int32)
    order = torch.randperm(rows, generator=g)[:b] if pages or rows >= b else torch.randint(0, rows, (b,), generator=g)
    free = torch.randperm(b * wide + 5, generator=g).add_(rows * wide + 1).to(torch.int32) if pages else None
    args = [x.to(torch.int32).to(device) for x in (table, order, pasts, counts)]
    return args, dict(tokens=int(counts.sum()), page_size=ps, pages=None if free is None else free.to(device))


def exact_plan(table, rows, past, counts, tokens, page_size, pages):
    """Token by token, on lists: (the plan's seven parts, the table afterwards)."""
    table = [list(x) for x in table.tolist()]
    free = list(pages.tolist()) if pages is not None else None
    pos, slots, seq, starts, lens, mine = [], [], [], [0], [], []
    for i, (r, a, m) in enumerate(zip(rows.tolist(), past.tolist(), counts.tolist())):
        if free is not None:
            for j in range(-(-a // page_size), -(-(a + m) // page_size)):
                table[r][j] = free.pop(0)
        for t in range(a, a + m):
            pos.append(t)
            slots.append(table[r][t // page_size] * page_size + t % page_size)
            seq.append(i)
        starts.append(len(pos))
        lens.append(a + m)
        need = -(-(a + m) // page_size)
        mine.append(table[r][:need] + [0] * (len(table[r]) - need))
    taken = 0 if pages is None else pages.numel() - len(free)
    info = [len(pos), taken]
    rest = tokens - len(pos)
    return [pos + [0] * rest, slots + [-1] * rest, seq + [-1] * rest, starts, lens, mine, info], table


PLANS = [(1, 1, 0, {}), (1, 357, 3001, {}), (3, 40, 100, {}), (7, 33, 17, {"ps": 5}), (64, 1, 4000, {"pages": True}), (5, 100, 64, {"pages": True}),
         (1024, 4, 40, {"pages": True}), (300, 20, 20, {"rows": 9}), (2, 5000, 3, {"pages": True, "ps": 1})]


def plan_parts(p):
    return [p.positions, p.slots, p.tok_seq, p.q_starts, p.seq_lens, p.block_table, p.info]
