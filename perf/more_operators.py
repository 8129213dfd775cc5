"""The operators of a cache held in 4 bits, as cases that can be timed and compared.

Three operators, each through the entry point a program calls:

* ``store``: ``ops.kv4_write``, keys and values of new tokens quantised into 4-bit pages, and the same tokens read back by ``ops.kv4_gather``;
* ``gather``: ``ops.kv4_gather``, cached tokens of ragged sequences as packed rows, for the attention of a prompt's next chunk;
* ``attend``: ``ops.paged_attn_decode_kv4``, decode attention over 4-bit pages.

A head's vector is held in groups of 64 values, each with a bf16 scale ``s`` and minimum ``m`` and codes ``c`` of 0 to 15 for the values ``m + s c``.
Where :data:`own` is false the same is computed by elementary torch operations, in 32 bits, the choice of a code in 64.
"""

from __future__ import annotations

import math
import zlib

import torch

own = False

PAGE = 16
GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SHAPES = [(32, 8, 128), (32, 8, 128), (32, 8, 128), (16, 8, 64), (14, 2, 64), (16, 2, 256), (8, 8, 128), (40, 8, 128), (16, 1, 128), (24, 1, 128)]


# ---- cases ------------------------------------------------------------------------------------------------------------

def _store(rows, past, new, heads=8, dim=128, dtype="bf16", ragged=False):
    return {"kind": "store", "rows": rows, "past": past, "new": new, "kv_heads": heads, "dim": dim, "dtype": dtype, "ragged": ragged}


def _gather(rows, length, heads=8, dim=128, dtype="bf16", ragged=False):
    return {"kind": "gather", "rows": rows, "length": length, "kv_heads": heads, "dim": dim, "dtype": dtype, "ragged": ragged}


def _attend(rows, length, heads=32, kv_heads=8, dim=128, q_len=1, dtype="bf16", ragged=False):
    return {"kind": "attend", "rows": rows, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim, "q_len": q_len, "dtype": dtype, "ragged": ragged}


def listed():
    return [
        {"name": "store 64 x 1", **_store(64, 4000, 1)},  # a decode step of a full batch: one new token each
        {"name": "store 1 x 4096", **_store(1, 1000, 4096)},  # a chunk of a prompt, behind a part that ends inside a page
        {"name": "store 11 ragged fp32 256", **_store(11, 500, 2500, 2, 256, "fp32", True)},  # portions of several prompts, unrounded heads of 256
        {"name": "gather 1 x 700", **_gather(1, 700)},  # the past of one short conversation
        {"name": "gather 13 ragged fp16 64", **_gather(13, 9000, 8, 64, "fp16", True)},  # several pasts for one packed chunk
        {"name": "gather 4 x 32768", **_gather(4, 32768)},  # long documents, for their next chunks
        {"name": "attend 1 x 48", **_attend(1, 48)},  # one user's stream, just begun: latency counts
        {"name": "attend 3 x 1999 ragged", **_attend(3, 1999, ragged=True)},  # a few users
        {"name": "attend 64 x 4096", **_attend(64, 4096)},  # a full batch
        {"name": "attend 24 ragged fp16 64", **_attend(24, 16001, 14, 2, 64, 1, "fp16", True)},  # ragged contexts, an odd number of heads a group, unused rows
        {"name": "attend 16 x 3001 windows", **_attend(16, 3001, 16, 2, 256, 4)},  # draft/verify windows: 32 query rows a head
        {"name": "attend 64 x 16384", **_attend(64, 16384)},  # a full batch of long contexts
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["attend", "attend", "attend", "store", "store", "gather", "gather"])
        heads, kv_heads, dim = rng.choice(SHAPES)
        ragged = rng.random() < 0.5
        if kind == "attend":
            case = _attend(size(1, 96), size(1, 66000), heads, kv_heads, dim, rng.choice([1, 1, 1, 2, 3, 4, 5]), rng.choice(["bf16", "bf16", "fp16"]), ragged)
        elif kind == "store":
            case = _store(size(1, 96), size(1, 20000), rng.choice([1, size(1, 9000)]), kv_heads, dim, rng.choice(["bf16", "bf16", "fp16", "fp32"]), ragged)
        else:
            case = _gather(size(1, 64), size(1, 66000), kv_heads, dim, rng.choice(["bf16", "bf16", "fp16", "fp32"]), ragged)
        if _cost(case) <= most and (kind == "attend" or sum(_spans(case)[1]) * kv_heads * dim < 1 << 28):
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ---- the shape of a case: what the host knows -----------------------------------------------------------------------------

def _spans(case):
    """``(tokens before, tokens of the call)`` of every sequence; for ``attend`` the length, the query tokens among them."""
    b = case["rows"]
    if case["kind"] == "store":
        past, new = case["past"], case["new"]
        if not case["ragged"]:
            return [past] * b, [new] * b
        return [past * ((5 * i) % b) // b for i in range(b)], [max(1, new * ((3 * i) % b + 1) // b) for i in range(b)]
    n = max(case["length"], case.get("q_len", 1))
    if not case["ragged"]:
        return [0] * b, [n] * b
    lens = [max(case.get("q_len", 1), n * ((7 * i) % b + 1) // b) for i in range(b)]
    for i in range(4, b, 6):
        lens[i] = 0  # unused rows of the batch
    return [0] * b, lens


def work(case):
    hk, d = case["kv_heads"], case["dim"]
    past, new = _spans(case)
    held = 2 * d // 2 + 2 * (d // GROUP) * 4  # bytes of a token's keys and values of a head
    tokens = sum(new)
    if case["kind"] == "attend":
        rows = case["rows"] * case["q_len"] * case["heads"]
        return {"bytes": tokens * hk * held + 4 * rows * d + 4 * sum(-(-n // PAGE) for n in new), "flops": 4 * d * case["heads"] * case["q_len"] * tokens}
    plain = 2 * tokens * hk * d * DTYPES[case["dtype"]].itemsize
    if case["kind"] == "store":  # in, held, out
        return {"bytes": 2 * plain + tokens * (hk * held + 4), "flops": 16 * tokens * hk * d}
    return {"bytes": plain + tokens * hk * held, "flops": 4 * tokens * hk * d}


# ---- seeded data: every tensor from the seed and its own name -------------------------------------------------------------

def _generator(seed, name):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(f"{seed}/{name}".encode()))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class _State:
    pass


class _Pages:
    """One layer's pool of 4-bit pages: a record of ``18 D`` bytes for each page and head, in this order:

    * codes of the keys ``[D/64 groups][token % 8][4][4][4]`` bytes: byte ``[g][t][c][j][b]`` has token ``t + 8 (b % 2)``, dim ``64 g + 16 j + 2 c + b // 2``
      in its lower half and the dim eight behind it in its upper one;
    * their parameters ``[token % 8][token // 8][groups][scale, minimum]`` in bf16;
    * codes of the values: byte ``[g][i][c][j][b]`` has token ``2 c + b // 2 + 8 (b % 2)``, dims ``64 g + 16 j + i`` and the one eight behind it;
    * their parameters, as those of the keys."""

    def __init__(self, data, dim):
        self.data, self.head_dim, self.page_size = data, dim, PAGE


def _table(case, lens, gen):
    """Pages in no order, with some that nobody has; what is not in use is page 0."""
    counts = [-(-n // PAGE) for n in lens]
    total = sum(counts) + 9
    ids = (torch.randperm(total - 1, generator=gen, device="cuda") + 1).to(torch.int32)
    table = torch.zeros((len(lens), max(1, max(counts)) + 1), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = ids[at : at + n]
        at += n
    return table, total


def _filled(case, lens, table, total, gen):
    """A pool whose tokens hold what quantised heads look like; places that no sequence has are all ones, a NaN in every parameter."""
    hk, d = case["kv_heads"], case["dim"]
    data = torch.full((total, hk, 18 * d), 255, dtype=torch.uint8, device="cuda")
    used = torch.zeros((total, PAGE), dtype=torch.bool, device="cuda")
    place = torch.arange(table.shape[1], device="cuda")[:, None] * PAGE + torch.arange(PAGE, device="cuda")
    for i, n in enumerate(lens):
        k = -(-n // PAGE)
        used[table[i, :k].long()] = place[:k] < n
    used = used.view(total, 1, 2, 8)
    for at in (0, 9 * d):
        # sums of two uniform codes of 0 to 7, a carry among them: few codes at the ends of a group's range, most in its middle
        a = torch.randint(0, 256, (total, hk, 8 * d), dtype=torch.uint8, device="cuda", generator=gen)
        b = torch.randint(0, 256, (total, hk, 8 * d), dtype=torch.uint8, device="cuda", generator=gen)
        data[:, :, at : at + 8 * d] = ((a >> 1) & 0x77) + ((b >> 1) & 0x77) + (a & b & 0x11)
        scale = torch.rand((total, hk, 8, 2, d // GROUP), generator=gen, device="cuda").mul_(0.3).add_(0.15)
        least = -scale * (7.5 + torch.randn(scale.shape, generator=gen, device="cuda"))
        params = torch.stack([scale, least], -1).to(torch.bfloat16)
        params = torch.where(used.transpose(2, 3)[..., None, None], params, math.nan)
        data[:, :, at + 8 * d : at + 9 * d] = params.contiguous().view(torch.uint8).view(total, hk, d)
    return data


def prepare(case, seed):
    s = _State()
    s.case = case
    hk, d, gen = case["kv_heads"], case["dim"], _generator(seed, case["kind"])
    past, new = _spans(case)
    lens = [p + n for p, n in zip(past, new)]
    s.block_table, total = _table(case, lens, gen)
    if case["kind"] == "attend":
        s.kv = _Pages(_filled(case, lens, s.block_table, total, gen), d)
        s.seq_lens, s.most = _ints(lens), max(lens)
        s.q = torch.randn((case["rows"] * case["q_len"], case["heads"], d), generator=gen, device="cuda").mul_(1.5).to(DTYPES[case["dtype"]])
        s.scale = 1.0 / math.sqrt(d)
        return s
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s.tokens, s.starts, s.first = starts[-1], _ints(starts), _ints(past)
    if case["kind"] == "gather":
        s.kv = _Pages(_filled(case, lens, s.block_table, total, gen), d)
        return s
    s.kv = _Pages(torch.full((total, hk, 18 * d), 255, dtype=torch.uint8, device="cuda"), d)
    # rows of a fused projection: queries in front, keys with a few strong channels and values behind them
    wide = torch.randn((s.tokens, 4 * hk, d), generator=gen, device="cuda")
    wide[:, 2 * hk : 3 * hk] *= 1 + 5 * (torch.rand((hk, d), generator=gen, device="cuda") < 0.05)
    wide[:, 2 * hk : 3 * hk] += torch.randn((hk, d), generator=gen, device="cuda")
    s.wide = wide.to(DTYPES[case["dtype"]])
    s.k, s.v = s.wide[:, 2 * hk : 3 * hk], s.wide[:, 3 * hk :]
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
    pos = s.first.long()[seq] + torch.arange(s.tokens, device="cuda") - s.starts.long()[seq]
    s.slots = (s.block_table[seq, pos // PAGE] * PAGE + pos % PAGE).to(torch.int32)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(s):
    case = s.case
    if own:
        from mfq_b200 import ops
        if case["kind"] == "attend":
            return ops.paged_attn_decode_kv4(s.q, s.kv, s.block_table, s.seq_lens, sm_scale=s.scale, q_len=case["q_len"], max_len=s.most)
        if case["kind"] == "store":
            ops.kv4_write(s.k, s.v, s.slots, s.kv)
        return ops.kv4_gather(s.kv, s.block_table, s.starts, s.tokens, first=s.first, dtype=DTYPES[case["dtype"]])
    if case["kind"] == "attend":
        return _plain_attend(s, case)
    if case["kind"] == "store":
        _plain_write(s)
    return _plain_gather(s, case)


# ---- the plain forms ------------------------------------------------------------------------------------------------------

def _unpack(data, d):
    """Records ``[n, heads, 18 D]`` -> keys and values ``[n, heads, 16, D]`` in 32 bits."""
    n, hk, g = data.shape[0], data.shape[1], d // GROUP
    out = []
    for at, order in ((0, (0, 1, 7, 3, 2, 5, 8, 4, 6)), (9 * d, (0, 1, 7, 4, 6, 2, 5, 8, 3))):
        codes = data[:, :, at : at + 8 * d]
        codes = torch.stack([codes & 15, codes >> 4], -1).view(n, hk, g, 8, 4, 4, 2, 2, 2)  # [.., group, t or i, c, j, odd, half, upper]
        codes = codes.permute(order).reshape(n, hk, PAGE, g, GROUP)
        params = data[:, :, at + 8 * d : at + 9 * d].contiguous().view(torch.bfloat16).view(n, hk, 8, 2, g, 2).transpose(2, 3).reshape(n, hk, PAGE, g, 2).float()
        out.append((params[..., 1:] + params[..., :1] * codes.float()).view(n, hk, PAGE, d))
    return out


def _down(x):
    """The largest bf16 that is not above ``x`` (fp32)."""
    near = x.to(torch.bfloat16)
    return torch.where(near.float() > x, torch.nextafter(near, torch.full_like(near, -math.inf)), near)


def _plain_codes(x):
    """``x [T, heads, D]`` -> codes ``[T, heads, D/64, 64]``, scale and minimum ``[T, heads, D/64]`` in bf16."""
    t, hk, d = x.shape
    x = x.float().view(t, hk, d // GROUP, GROUP)
    least = _down(x.amin(-1))
    wide = x.double().amax(-1) - least.double()
    scale = (wide / 15).float().to(torch.bfloat16)
    zero, far = torch.zeros_like(scale), torch.full_like(scale, math.inf)
    lower = torch.nextafter(scale, zero)
    scale = torch.where(scale.double() * 15 < wide, torch.nextafter(scale, far), torch.where(lower.double() * 15 >= wide, lower, scale))
    codes = torch.round((x.double() - least.double()[..., None]) / torch.where(scale > 0, scale, 1.0).double()[..., None])
    bad = ~(x.abs() <= 2.0 ** 126).all(-1)
    codes = torch.where(bad[..., None] | (scale == 0)[..., None], 0.0, codes)
    return codes.to(torch.uint8), torch.where(bad, math.nan, scale), torch.where(bad, math.nan, least)


def _plain_write(s):
    d, dev = s.kv.head_dim, s.slots.device
    data, g = s.kv.data, d // GROUP
    page, tok = s.slots.long() // PAGE, s.slots.long() % PAGE
    group, j, i = torch.meshgrid(torch.arange(g, device=dev), torch.arange(4, device=dev), torch.arange(8, device=dev), indexing="ij")
    t = tok[:, None, None, None]
    for x, at in ((s.k, 0), (s.v, 9 * d)):
        codes, scale, least = _plain_codes(x)
        pair = codes.view(*codes.shape[:3], 4, 2, 8)
        pair = pair[..., 0, :] + 16 * pair[..., 1, :]
        if at == 0:
            place = group * 512 + t % 8 * 64 + i // 2 * 16 + j * 4 + i % 2 * 2 + t // 8
        else:
            place = at + group * 512 + i * 64 + t % 8 // 2 * 16 + j * 4 + t % 2 * 2 + t // 8
        data[page[:, None, None], torch.arange(data.shape[1], device=dev)[:, None], place.flatten(1)[:, None]] = pair.flatten(2)
        params = torch.stack([scale, least], -1).view(torch.uint8).flatten(2)
        place = at + 8 * d + (tok % 8 * 2 + tok // 8)[:, None] * 4 * g + torch.arange(4 * g, device=dev)
        data[page[:, None, None], torch.arange(data.shape[1], device=dev)[:, None], place[:, None]] = params


def _plain_gather(s, case):
    hk, d, dt = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    k, v = (torch.empty((s.tokens, hk, d), dtype=dt, device="cuda") for _ in range(2))
    past, new = _spans(case)
    at = 0
    for i, (p, n) in enumerate(zip(past, new)):
        if n:
            lo, hi = p // PAGE, -(-(p + n) // PAGE)
            for out, x in zip((k, v), _unpack(s.kv.data[s.block_table[i, lo:hi].long()], d)):
                out[at : at + n] = x.transpose(1, 2).reshape(-1, hk, d)[p - lo * PAGE : p - lo * PAGE + n].to(dt)
        at += n
    return k, v


def _plain_attend(s, case):
    hk, d, ql = case["kv_heads"], case["dim"], case["q_len"]
    g = case["heads"] // hk
    lens = _spans(case)[1]
    out = torch.empty_like(s.q)
    last = (torch.arange(ql, device="cuda").repeat_interleave(g) - (ql - 1))[None, None, :, None]  # a window's query sees no later token of it
    q = s.q.float().view(-1, ql, hk, g, d).permute(0, 2, 1, 3, 4).reshape(-1, hk, ql * g, d)
    at = 0
    while at < len(lens):  # as many sequences at once as a few GB hold
        wide = end = 0
        while end < len(lens) - at and (end == 0 or (end + 1) * max(wide, lens[at + end]) * hk * d < 1 << 28):
            wide, end = max(wide, lens[at + end]), end + 1
        rows = slice(at, at + end)
        pages = max(1, -(-max(wide, ql) // PAGE))
        k, v = (x.view(end, pages, hk, PAGE, d).transpose(1, 2).reshape(end, hk, pages * PAGE, d)
                for x in _unpack(s.kv.data[s.block_table[rows, :pages].long().flatten()], d))
        seen = torch.arange(pages * PAGE, device="cuda") < s.seq_lens.long()[rows, None, None, None] + last
        there = seen.any(2)[..., None]  # a NaN in a place that nobody sees stays out
        scores = torch.where(seen, q[rows] @ torch.where(there, k, 0.0).transpose(-1, -2) * s.scale, -math.inf)
        top = scores.amax(-1, keepdim=True)
        p = torch.where(seen, torch.exp(scores - torch.where(top == -math.inf, 0.0, top)), 0.0)
        total = p.sum(-1, keepdim=True)
        o = torch.where(total > 0, p @ torch.where(there, v, 0.0) / total, 0.0)
        out.view(-1, ql, hk, g, d)[rows] = o.view(end, hk, ql, g, d).permute(0, 2, 1, 3, 4).to(out.dtype)
        at += end
    return out


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(s, case)
    if case["kind"] == "store":
        return _exact_values(s.k), _exact_values(s.v)
    rows = [_exact_tokens(s, i, p, p + n) for i, (p, n) in enumerate(zip(*_spans(case)))]
    return torch.cat([k for k, _ in rows]), torch.cat([v for _, v in rows])


def _exact_values(x):
    """Scale and minimum by their places in units of the last of bf16's eight bits; for values of ordinary size."""
    t, hk, d = x.shape
    x = x.double().view(t, hk, d // GROUP, GROUP)

    def unit(y):  # of bf16 around y
        return torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1e-30))) - 7)

    low = x.min(-1, keepdim=True).values
    low = torch.floor(low / unit(low)) * unit(low)
    step = (x.max(-1, keepdim=True).values - low) / 15
    step = torch.ceil(step / unit(step)) * unit(step)
    codes = torch.where(step > 0, torch.round((x - low) / torch.where(step > 0, step, 1.0)), 0.0)
    return (low + step * codes).view(t, hk, d)


def _exact_tokens(s, row, begin, end):
    """Keys and values ``[tokens, heads, D]`` of a sequence, each from the byte that has it."""
    d, dev = s.kv.head_dim, s.kv.data.device
    pos = torch.arange(begin, end, device=dev)
    rec = s.kv.data[s.block_table[row].long()[pos // PAGE]]  # [tokens, heads, 18 D]
    t, dim = (pos % PAGE)[:, None], torch.arange(d, device=dev)
    g, j, upper, i = dim // 64, dim % 64 // 16, dim % 16 // 8, dim % 8
    out = []
    for at, place in ((0, 512 * g + 64 * (t % 8) + 16 * (i // 2) + 4 * j + 2 * (i % 2) + t // 8),
                      (9 * d, 512 * g + 64 * i + 16 * (t % 8 // 2) + 4 * j + 2 * (t % 2) + t // 8)):
        byte = rec.gather(2, (at + place)[:, None].expand(-1, rec.shape[1], -1))
        code = torch.where(upper == 1, byte // 16, byte % 16).double()
        where = at + 8 * d + ((t % 8) * 2 + t // 8) * (d // 16) + 4 * g

        def param(k):
            lo, hi = (rec.gather(2, (where + k + e)[:, None].expand(-1, rec.shape[1], -1)).int() for e in (0, 1))
            return ((lo + 256 * hi) << 16).view(torch.float32).double()

        out.append(param(2) + param(0) * code)
    return out


def _exact_attend(s, case):
    """Sequence by sequence: the softmax over the keys that a query sees."""
    ql, hk, hq, d = case["q_len"], case["kv_heads"], case["heads"], case["dim"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for row, n in enumerate(s.seq_lens.tolist()):
        if n == 0:
            continue
        k, v = (x.transpose(0, 1) for x in _exact_tokens(s, row, 0, n))
        for i in range(ql):
            sees = n - (ql - 1 - i)
            q = s.q[row * ql + i].double().view(hk, hq // hk, d)
            p = torch.softmax(q @ k[:, :sees].transpose(1, 2) * s.scale, dim=-1)
            out[row * ql + i] = (p @ v[:, :sees]).reshape(hq, d)
    return out
