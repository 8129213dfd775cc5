"""The operators of one step of a served batch, as cases that can be timed and compared.

Three operators, each through the entry point a program calls:

* ``attend``: ``ops.paged_attn_decode_shared``, decode attention over FP8 pages of sequences that share their first pages in groups;
* ``logits``: ``ops.process_logits``, biases, penalties for repeated tokens and grammar masks (``count``: with ``ops.count_tokens`` before it);
* ``plan``: ``ops.plan_batch``, positions, slots and block tables of a ragged batch from the lengths of its requests.

Where :data:`own` is false the same is computed by elementary torch operations, in 32 bits.
"""

from __future__ import annotations

import math
import zlib

import torch

own = False

PAGE = 16
V_ORDER = (0, 1, 8, 9, 2, 3, 10, 11, 4, 5, 12, 13, 6, 7, 14, 15)  # token of each slot in a page of values
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------------

def _attend(rows, groups, prefix, tail, heads=32, kv_heads=8, dim=128, q_len=1, ragged=False):
    return {"kind": "attend", "rows": rows, "groups": groups, "prefix": prefix, "tail": tail, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "q_len": q_len, "ragged": ragged}


def _logits(rows, vocab, dtype, mask=False, biases=0, tables=0, count=0):
    return {"kind": "logits", "rows": rows, "vocab": vocab, "dtype": dtype, "mask": mask, "biases": biases, "tables": tables or rows, "count": count}


def _plan(singles, portions, most, past, pages=False):
    return {"kind": "plan", "singles": singles, "portions": portions, "most": most, "past": past, "pages": pages}


def listed():
    return [
        {"name": "attend 2 x 48+5", **_attend(2, 1, 48, 5)},  # two samples of a short prompt, just begun: latency counts
        {"name": "attend 6 x 1999+130", **_attend(6, 1, 1999, 130)},  # a few samples of one prompt; it ends inside a page
        {"name": "attend 64 x 8192+512", **_attend(64, 1, 8192, 512)},  # a full batch behind one long system prompt
        {"name": "attend 48 in 5 ragged", **_attend(48, 5, 4100, 700, 16, 8, 64, 1, True)},  # several assistants in one batch, some rows unshared
        {"name": "attend 16 x 3001+90 windows", **_attend(16, 1, 3001, 90, 16, 2, 256, 2)},  # draft/verify windows, heads of 256
        {"name": "attend 64 x 32768+200", **_attend(64, 1, 32768, 200)},  # many questions about one long document
        {"name": "logits 1 x 32000 fp32", **_logits(1, 32000, "fp32")},  # one user's stream with penalties
        {"name": "logits 64 x 128256", **_logits(64, 128256, "bf16", True, 40)},  # a batch with penalties, biases and grammars
        {"name": "logits 37 x 49999 fp16", **_logits(37, 49999, "fp16", True, 300, 50)},  # an odd vocabulary, rows of a wider table
        {"name": "logits 24 x 128256 counted", **_logits(24, 128256, "bf16", False, 0, 0, 4000)},  # replayed requests: histories counted first
        {"name": "plan 357 past 3001", **_plan(0, 1, 357, 3001)},  # the next turn of one conversation
        {"name": "plan 240 + 16 portions", **_plan(240, 16, 512, 8000, True)},  # continuous batching: pages handed out too
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["attend", "attend", "attend", "logits", "logits", "plan"])
        if kind == "plan":
            portions = size(1, 24)
            case = _plan(rng.choice([0, size(1, 256)]), portions, size(1, 2048), size(1, 30000), rng.random() < 0.5)
        elif kind == "logits":
            rows = size(1, 96)
            case = _logits(rows, size(1000, 160000), rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.6, rng.choice([0, size(1, 300)]),
                           rng.choice([0, rows + size(1, 32)]), rng.choice([0, 0, size(1, 6000)]))
        else:
            rows = size(2, 96)
            heads, kv_heads, dim, q_len = rng.choice([(32, 8, 128, 1), (32, 8, 128, 1), (32, 8, 128, 4), (16, 8, 64, 1), (8, 8, 128, 2), (40, 8, 128, 1),
                                                      (16, 2, 256, 1), (16, 2, 256, 2), (14, 2, 64, 1), (16, 1, 128, 1)])
            case = _attend(rows, rng.randint(1, max(1, min(8, rows // 2))), size(17, 33000), size(1, 2000), heads, kv_heads, dim, q_len, rng.random() < 0.5)
        if _cost(case) <= most:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ---- the shape of a case: what the host knows -----------------------------------------------------------------------------

def _groups(case):
    """``[(sequences, prefix tokens)]`` and the tail of every sequence, its query tokens among them."""
    b, n, ql = case["rows"], case["groups"], case["q_len"]
    if not case["ragged"]:
        sizes = [b // n + (i < b % n) for i in range(n)]
        prefixes, tails = [case["prefix"]] * n, [max(ql, case["tail"])] * b
    else:
        sizes = [1 + (b - n) * (2 * i + 1) // (n * n) for i in range(n)]  # from small groups to large ones
        sizes[-1] += b - sum(sizes)
        prefixes = [max(1, case["prefix"] * ((5 * i) % n + 1) // n) for i in range(n)]
        if n > 1:
            prefixes[0] = 0  # these share nothing
        tails = [max(ql, 1 + case["tail"] * ((7 * i) % b) // b) for i in range(b)]
    return list(zip(sizes, prefixes)), tails


def _spans(case):
    """``(tokens in the pages, new tokens)`` of every request of a plan."""
    past, most = case["past"], case["most"]
    spans = [(1 + (past * (i % 17 + 3)) // 20, 1) for i in range(case["singles"])]
    if case["portions"] == 1:
        return spans + [(past, most)]
    return spans + [(past * (i % 5) // 4, max(1, most * (i % 7 + 1) // 7)) for i in range(case["portions"])]


def work(case):
    if case["kind"] == "attend":
        groups, tails = _groups(case)
        d, hk, hq, ql = case["dim"], case["kv_heads"], case["heads"], case["q_len"]
        keys = sum(p for _, p in groups) + sum(tails)
        seen = sum(n * p for n, p in groups) + sum(tails)
        pages = sum(n * (p // PAGE) for n, p in groups) + sum(t // PAGE + 1 for t in tails)
        return {"bytes": keys * hk * (2 * d + 8) + 4 * case["rows"] * ql * hq * d + 4 * pages, "flops": 4 * d * hq * ql * seen}
    if case["kind"] == "logits":
        b, v = case["rows"], case["vocab"]
        el = DTYPES[case["dtype"]].itemsize
        byt = b * v * (2 * el + 2) + b * (v / 8 if case["mask"] else 0) + 8 * b * case["biases"] + 32 * b
        if case["count"]:
            byt += case["tables"] * (v * 2 + case["count"] * 8)
        return {"bytes": byt, "flops": 8 * b * v}
    spans = _spans(case)
    tokens, used = sum(m for _, m in spans), sum((p + m + PAGE - 1) // PAGE for p, m in spans)
    wide = max((p + m + PAGE - 1) // PAGE for p, m in spans) + 3
    return {"bytes": 4 * (3 * len(spans) + used + 3 * tokens + 2 * len(spans) + 1 + len(spans) * wide), "flops": 8 * tokens}


# ---- seeded data: every tensor from the seed and its own name -------------------------------------------------------------

def _generator(seed, name):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(f"{seed}/{name}".encode()))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class _State:
    pass


class _Pages:
    """One layer's pool of FP8 pages, in the layout of the framework's cache."""

    def __init__(self, seed, pages, heads, dim):
        gen = _generator(seed, "pages")

        def codes(*shape):  # a row's largest value (about 4 standard deviations) sits at 448
            return torch.randn(shape, generator=gen, device="cuda").mul_(112.0).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)

        self.k = codes(pages, heads, dim // 64, PAGE, 64)
        self.v = codes(pages, heads, dim, PAGE)
        self.k_scale = torch.rand((pages, heads, PAGE), generator=gen, device="cuda").mul_(0.006).add_(0.006)
        self.v_scale = torch.rand((pages, heads, PAGE), generator=gen, device="cuda").mul_(0.006).add_(0.006)
        self.page_size = PAGE


def _prepare_attend(case, seed):
    s = _State()
    groups, tails = _groups(case)
    b, gen = case["rows"], _generator(seed, "order")
    shared = [p // PAGE for _, p in groups]  # whole pages; the rest of a prefix is every sequence's own copy
    lens, at = [], 0
    for n, p in groups:
        lens += [p + t for t in tails[at : at + n]]
        at += n
    wide = max((n + PAGE - 1) // PAGE for n in lens) + 1
    total = 1 + sum(shared) + sum((n + PAGE - 1) // PAGE for n in lens)  # more than are used
    ids = (torch.randperm(total - 1, generator=gen, device="cuda") + 1).tolist()
    table, at = [[0] * wide for _ in range(b)], 0
    order = torch.randperm(b, generator=gen, device="cuda").tolist()  # batch rows of the sequences, group by group
    seq_lens = [0] * b
    for (n, p), keep in zip(groups, shared):
        front = [ids.pop() for _ in range(keep)]
        for _ in range(n):
            row, length = order[at], lens[at]
            own_pages = [ids.pop() for _ in range((length + PAGE - 1) // PAGE - keep)]
            table[row][: keep + len(own_pages)] = front + own_pages
            seq_lens[row] = length
            at += 1
    s.kv = _Pages(seed, total, case["kv_heads"], case["dim"])
    s.q = torch.randn((b * case["q_len"], case["heads"], case["dim"]), generator=gen, device="cuda").mul_(2.0).to(torch.bfloat16)
    s.block_table, s.seq_lens, s.members = _ints(table), _ints(seq_lens), _ints(order)
    starts = [0]
    for n, _ in groups:
        starts.append(starts[-1] + n)
    s.group_starts, s.prefix_lens = _ints(starts), _ints([p for _, p in groups])
    s.scale = 1.0 / math.sqrt(case["dim"])
    s.most_rows, s.most_prefix, s.most_tail = max(n for n, _ in groups), max(shared) * PAGE, max(n - k * PAGE for n, k in zip(lens, [k for (m, _), k in zip(groups, shared) for _ in range(m)]))
    return s


def _prepare_logits(case, seed):
    s = _State()
    b, v, r = case["rows"], case["vocab"], case["tables"]
    gen = _generator(seed, "logits")
    s.logits = torch.randn((b, v), generator=gen, device="cuda").mul_(3.0).to(DTYPES[case["dtype"]])
    # temperature, top-k, top-p, presence, frequency, repetition, seed: the record a row's sampler reads; every third row has none
    records = torch.zeros((r, 8), dtype=torch.float32, device="cuda")
    draws = torch.rand((r, 3), generator=gen, device="cuda")
    on = (torch.arange(r, device="cuda") % 3 != 2).float() if r > 2 else torch.ones(r, device="cuda")
    records[:, 3], records[:, 4], records[:, 5] = draws[:, 0] * on, draws[:, 1] * 0.5 * on, 1 + draws[:, 2] * 0.3 * on
    s.records = records.view(torch.int32)
    s.rows = torch.randperm(r, generator=gen, device="cuda")[:b].to(torch.int32) if r != b else None
    n = case["count"] or 1500  # tokens of a history: some of them often, most once
    tokens = (torch.rand((r, n), generator=gen, device="cuda").pow(4) * v).long().clamp_(max=v - 1)
    split = n * 2 // 3  # the prompt's
    s.tokens = tokens
    s.prompt, s.prompt_rows = tokens[:, :split].reshape(-1).to(torch.int32), torch.arange(r, device="cuda", dtype=torch.int32).repeat_interleave(split)
    s.answer, s.answer_rows = tokens[:, split:].reshape(-1).to(torch.int32), torch.arange(r, device="cuda", dtype=torch.int32).repeat_interleave(n - split)
    s.counts = _plain_counts(s, r, v)
    k = case["biases"]
    s.bias = None
    if k:
        ids = torch.rand((r, v), generator=gen, device="cuda").topk(k, dim=1).indices.to(torch.int32)
        ids[:, k - k // 4 :] = -1  # unused places
        s.bias = (ids, torch.randn((r, k), generator=gen, device="cuda").mul_(4.0))
    s.allowed = None
    if case["mask"]:  # about half of the words are empty, the others half full: what a grammar leaves
        words = torch.randint(-(1 << 31), 1 << 31, (r, (v + 31) // 32), generator=gen, device="cuda", dtype=torch.int64)
        some = torch.rand(words.shape, generator=gen, device="cuda") < 0.5
        words = torch.where(some, words, 0)
        words[torch.arange(r, device="cuda") % 4 == 1] = -1  # no grammar
        s.allowed = words.to(torch.int32)
    return s


def _prepare_plan(case, seed):
    s = _State()
    spans = _spans(case)
    n, gen = len(spans), _generator(seed, "plan")
    wide = max((p + m + PAGE - 1) // PAGE for p, m in spans) + 3
    rows = n + 5
    s.block_table = torch.randperm(rows * wide, generator=gen, device="cuda").add_(1).view(rows, wide).to(torch.int32)
    s.rows = torch.randperm(rows, generator=gen, device="cuda")[:n].to(torch.int32)
    s.past, s.counts = _ints([p for p, _ in spans]), _ints([m for _, m in spans])
    s.tokens = sum(m for _, m in spans)
    new = sum((p + m + PAGE - 1) // PAGE - (p + PAGE - 1) // PAGE for p, m in spans)
    s.pages = torch.randperm(new + 64, generator=gen, device="cuda").add_(rows * wide + 1).to(torch.int32) if case["pages"] else None
    return s


def prepare(case, seed):
    s = {"attend": _prepare_attend, "logits": _prepare_logits, "plan": _prepare_plan}[case["kind"]](case, seed)
    s.case = case
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(s):
    case = s.case
    if case["kind"] == "attend":
        return _run_attend(s, case)
    return _run_logits(s, case) if case["kind"] == "logits" else _run_plan(s, case)


def _run_attend(s, case):
    if own:
        from mfq_b200 import ops
        return ops.paged_attn_decode_shared(s.q, s.kv, s.block_table, s.seq_lens, s.group_starts, s.prefix_lens, sm_scale=s.scale, members=s.members,
                                            q_len=case["q_len"], max_group=s.most_rows, max_prefix=s.most_prefix, max_tail=s.most_tail)
    return _plain_attend(s, case)


def _run_logits(s, case):
    if own:
        from mfq_b200 import ops
        counts = s.counts
        if case["count"]:
            counts = torch.zeros((case["tables"], case["vocab"]), dtype=torch.int16, device="cuda")
            ops.count_tokens(counts, s.prompt, s.prompt_rows, prompt=True)
            ops.count_tokens(counts, s.answer, s.answer_rows)
        out = ops.process_logits(s.logits, s.records, counts=counts, bias=s.bias, allowed=s.allowed, rows=s.rows)
        return (out, counts) if case["count"] else out
    counts = _plain_counts(s, case["tables"], case["vocab"]) if case["count"] else s.counts
    out = _plain_logits(s, counts)
    return (out, counts) if case["count"] else out


def _run_plan(s, case):
    if own:
        from mfq_b200 import ops
        p = ops.plan_batch(s.block_table, s.rows, s.past, s.counts, tokens=s.tokens, page_size=PAGE, pages=s.pages)
        return [p.positions, p.slots, p.tok_seq, p.q_starts, p.seq_lens, p.block_table, p.info, s.block_table]
    return _plain_plan(s)


# ---- the plain forms ------------------------------------------------------------------------------------------------------

def _token_rows(kv, pages, off):
    """Keys and values ``[..., heads, dim]`` of tokens at ``(page, place in the page)``."""
    k = kv.k.view(torch.uint8)[pages, :, :, off].view(torch.float8_e4m3fn).float().flatten(-2) * kv.k_scale[pages, :, off][..., None]
    place = torch.tensor(V_ORDER, device=pages.device).argsort()[off]
    v = kv.v.view(torch.uint8)[pages, :, :, place].view(torch.float8_e4m3fn).float() * kv.v_scale[pages, :, off][..., None]
    return k, v


def _softmax_part(scores, seen, values):
    """Maximum, sum and weighted values of the keys that are seen; ``scores [..., rows, keys]``, ``values [..., keys, dim]``."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True) if scores.shape[-1] else scores.new_full(scores.shape[:-1] + (1,), -math.inf)
    p = torch.where(seen, torch.exp(scores - torch.where(top == -math.inf, 0.0, top)), 0.0)
    return top, p.sum(-1, keepdim=True), p @ values


def _plain_attend(s, case):
    b, ql, hk, d = case["rows"], case["q_len"], case["kv_heads"], case["dim"]
    g = case["heads"] // hk
    dev = s.q.device
    q = s.q.view(b, ql, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, ql * g, d).float()
    last = (torch.arange(ql, device=dev).repeat_interleave(g) - (ql - 1))[None, None, :, None]  # a window's query sees no later token of it
    member, starts = s.members.long(), s.group_starts.long()
    whole = s.prefix_lens.long() // PAGE * PAGE
    # the prefixes: all sequences of a group against its keys
    place = starts[:-1, None] + torch.arange(s.most_rows, device=dev)
    seq = member[place.clamp(max=b - 1)]
    keys = torch.arange(s.most_prefix, device=dev)
    pages = s.block_table.long()[member[starts[:-1]]][:, keys // PAGE]
    k, v = _token_rows(s.kv, pages, (keys % PAGE).expand_as(pages))
    k, v = k.transpose(1, 2), v.transpose(1, 2)  # [groups, heads, keys, dim]
    qg = q[seq].transpose(1, 2).flatten(2, 3)
    lens = (s.seq_lens.long()[seq][:, :, None] + last[0, 0, :, 0]).flatten(1)  # [groups, sequences x queries]
    seen = (keys < whole[:, None])[:, None, None] & (keys < lens[:, None, :, None])
    parts = [x.unflatten(2, (s.most_rows, ql * g)) for x in _softmax_part(qg @ k.transpose(-1, -2) * s.scale, seen, v)]
    group = (torch.arange(b, device=dev)[:, None] >= starts[1:]).sum(-1)
    at = torch.arange(b, device=dev) - starts[group]
    top_a, sum_a, out_a = (x[group, :, at] for x in parts)
    # the tails: every sequence against its own keys
    pos = whole[group][:, None] + torch.arange(s.most_tail, device=dev)
    pages = s.block_table.long()[member].gather(1, (pos // PAGE).clamp(max=s.block_table.shape[1] - 1))
    k, v = _token_rows(s.kv, pages, pos % PAGE)
    k, v, q = k.transpose(1, 2), v.transpose(1, 2), q[member]
    seen = pos[:, None, None] < s.seq_lens.long()[member][:, None, None, None] + last
    top_b, sum_b, out_b = _softmax_part(q @ k.transpose(-1, -2) * s.scale, seen, v)
    top = torch.maximum(top_a, top_b)
    wa, wb = (torch.where(t == -math.inf, 0.0, torch.exp(t - torch.where(top == -math.inf, 0.0, top))) for t in (top_a, top_b))
    total = sum_a * wa + sum_b * wb
    o = torch.where(total > 0, (out_a * wa + out_b * wb) / total, 0.0)
    out = torch.empty_like(s.q).view(b, ql, hk, g, d)
    out[member] = o.view(b, hk, ql, g, d).permute(0, 2, 1, 3, 4).to(out.dtype)
    return out.view_as(s.q)


def _plain_counts(s, rows, vocab):
    """15 bits of a word count the answer's tokens, the highest says that the prompt has the token."""
    seen = torch.zeros(rows * vocab, dtype=torch.int32, device="cuda")
    seen[s.prompt_rows.long() * vocab + s.prompt.long()] = 1
    times = torch.zeros(rows * vocab, dtype=torch.int32, device="cuda")
    times.scatter_add_(0, s.answer_rows.long() * vocab + s.answer.long(), torch.ones_like(s.answer))
    return (times.clamp(max=32767) - 32768 * seen).to(torch.int16).view(rows, vocab)


def _plain_logits(s, counts):
    rows = torch.arange(s.logits.shape[0], device="cuda") if s.rows is None else s.rows.long()
    l, v = s.logits.float(), s.logits.shape[1]
    if s.bias is not None:
        ids, values = s.bias[0][rows].long(), s.bias[1][rows]
        l = l + torch.zeros_like(l).scatter_add_(1, ids.clamp(min=0), torch.where(ids >= 0, values, 0.0))
    presence, frequency, repetition = (s.records.view(torch.float32)[rows, i, None] for i in (3, 4, 5))
    word = counts[rows].int()
    times = (word & 0x7FFF).float()
    l = torch.where(word != 0, torch.where(l > 0, l / repetition, l * repetition), l)
    l = torch.where(times > 0, l - (presence + frequency * times), l)
    if s.allowed is not None:
        at = torch.arange(v, device="cuda")
        l = torch.where((s.allowed[rows][:, at // 32] >> (at % 32).int()) & 1 != 0, l, -math.inf)
    return l.to(s.logits.dtype)


def _plain_plan(s):
    dev = s.block_table.device
    rows, past, counts = s.rows.long(), s.past.long(), s.counts.long()
    starts = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    lens = past + counts
    have, need = (past + PAGE - 1) // PAGE, (lens + PAGE - 1) // PAGE
    table, taken = s.block_table.clone(), torch.zeros((), dtype=torch.long, device=dev)
    place = torch.arange(table.shape[1], device=dev)
    if s.pages is not None:
        first = (need - have).cumsum(0) - (need - have)
        taken = (need - have).sum()
        at = (first - have)[:, None] + place
        new = s.pages[at.clamp(0, s.pages.numel() - 1)]
        table[rows] = torch.where((place >= have[:, None]) & (place < need[:, None]), new, table[rows])
    mine = torch.where(place < need[:, None], table[rows], 0)
    t = torch.arange(s.tokens, device=dev)
    seq = (t[:, None] >= starts[1:]).sum(-1)
    pos = past[seq] + t - starts[seq]
    slots = mine[seq, pos // PAGE] * PAGE + pos % PAGE
    info = torch.stack([starts[-1], taken])
    return [x.to(torch.int32) for x in (pos, slots, seq, starts, lens, mine, info, table)]


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s = prepare(case, seed)
    return _exact_attend(s, case) if case["kind"] == "attend" else _exact_logits(s, case)


def _exact_attend(s, case):
    """Sequence by sequence: the softmax over all keys that a query sees, through the sequence's own table."""
    ql, hk, hq, d = case["q_len"], case["kv_heads"], case["heads"], case["dim"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    order = torch.tensor(V_ORDER, device="cuda")
    for row, n in enumerate(s.seq_lens.tolist()):
        ids = s.block_table[row, : (n + PAGE - 1) // PAGE].long()
        k = s.kv.k[ids].double() * s.kv.k_scale[ids].double()[:, :, None, :, None]  # [pages, heads, chunks, tokens, 64]
        k = k.permute(1, 0, 3, 2, 4).reshape(hk, -1, d)[:, :n]
        v = torch.empty((ids.numel(), hk, d, PAGE), dtype=torch.float64, device="cuda")
        v[..., order] = s.kv.v[ids].double()
        v = (v * s.kv.v_scale[ids].double()[:, :, None, :]).permute(1, 0, 3, 2).reshape(hk, -1, d)[:, :n]
        for i in range(ql):
            sees = n - (ql - 1 - i)
            if sees <= 0:
                continue
            q = s.q[row * ql + i].double().view(hk, hq // hk, d)
            p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k[:, :sees]) * s.scale, -1)
            out[row * ql + i] = torch.einsum("hgt,htd->hgd", p, v[:, :sees]).reshape(hq, d)
    return out


def _exact_logits(s, case):
    out = s.logits.double()
    r, v = case["tables"], case["vocab"]
    base = torch.arange(r, device="cuda")[:, None] * v
    split = s.tokens.shape[1] * 2 // 3
    seen = torch.bincount((base + s.tokens[:, :split]).reshape(-1), minlength=r * v).view(r, v) > 0
    times = torch.bincount((base + s.tokens[:, split:]).reshape(-1), minlength=r * v).view(r, v)
    record = s.records.view(torch.float32).double()
    for i in range(out.shape[0]):
        row = i if s.rows is None else int(s.rows[i])
        presence, frequency, repetition = record[row, 3], record[row, 4], record[row, 5]
        if s.bias is not None:
            used = s.bias[0][row] >= 0
            out[i].index_add_(0, s.bias[0][row][used].long(), s.bias[1][row][used].double())
        both = seen[row] | (times[row] > 0)
        x = out[i]
        x[both] = torch.where(x[both] > 0, x[both] / repetition, x[both] * repetition)
        x -= torch.where(times[row] > 0, presence + frequency * times[row], 0.0)
        if s.allowed is not None:
            bits = (s.allowed[row].long()[:, None] >> torch.arange(32, device="cuda")) & 1
            x[bits.reshape(-1)[:v] == 0] = -math.inf
    return (out, None) if case["count"] else out
