"""Pools held in 4 bits, and batches over them, for the tests of ``ops.kv4_write``, ``ops.kv4_gather`` and ``ops.paged_attn_decode_kv4``.

Every place of a pool that no sequence has is all ones: a NaN in each parameter."""

import math
from types import SimpleNamespace

import torch

from mfq_b200.engine.kv_cache import LayerKV4


def place(is_v, t, dim):
    """Byte and shift of the code of token ``t``, dim ``dim`` in a record's K or V codes (relative to them)."""
    g, j, upper, i = dim // 64, dim % 64 // 16, dim % 16 // 8, dim % 8
    if is_v:
        return 512 * g + 64 * i + 16 * (t % 8 // 2) + 4 * j + 2 * (t % 2) + t // 8, 4 * upper
    return 512 * g + 64 * (t % 8) + 16 * (i // 2) + 4 * j + 2 * (i % 2) + t // 8, 4 * upper


_MAPS = {}


def _maps(d):
    if d not in _MAPS:
        where = torch.tensor([[[place(v, t, x)[0] + 9 * d * v for x in range(d)] for t in range(16)] for v in (0, 1)])
        shift = torch.tensor([place(0, 0, x)[1] for x in range(d)])
        _MAPS[d] = where, shift
    return _MAPS[d]


def unpack(data):
    """``[pages, heads, 18 D]`` -> codes ``[2 (K, V), pages, heads, 16, D]``, scales and minima ``[2, pages, heads, 16, D / 64]`` in 64 bits."""
    data = data.cpu()
    n, hk, d = data.shape[0], data.shape[1], data.shape[2] // 18
    where, shift = _maps(d)
    codes = torch.stack([data[:, :, w] >> shift & 15 for w in where.to(torch.long)])
    out = []
    for at in (8 * d, 17 * d):
        x = data[:, :, at : at + d].contiguous().view(torch.bfloat16).double().view(n, hk, 8, 2, d // 64, 2)
        out.append(x.transpose(2, 3).reshape(n, hk, 16, d // 64, 2))
    out = torch.stack(out)
    return codes, out[..., 0], out[..., 1]


def values(data):
    codes, s, m = unpack(data)
    return (m[..., None] + s[..., None] * codes.double().unflatten(-1, (-1, 64))).flatten(-2)


def pool(seed, pages, hk, d, used=None, spread=1.0):
    """A pool with something in the places ``used [pages, 16]`` (default: all)."""
    g = torch.Generator().manual_seed(seed)
    used = torch.ones((pages, 16), dtype=torch.bool) if used is None else used
    data = torch.randint(0, 256, (pages, hk, 18 * d), generator=g, dtype=torch.uint8)
    for at in (8 * d, 17 * d):
        s = torch.rand((pages, hk, 16, d // 64), generator=g).mul_(0.25).add_(0.1)
        if spread != 1.0:
            s *= torch.exp2(torch.rand(s.shape, generator=g).sub_(0.5).mul_(2 * math.log2(spread)).round())
        m = -s * (7.5 + torch.randn(s.shape, generator=g))
        both = torch.where(used[:, None, :, None, None], torch.stack([s, m], -1), math.nan).to(torch.bfloat16)
        both = both.unflatten(2, (2, 8)).transpose(2, 3).contiguous()
        data[:, :, at : at + d] = both.view(torch.uint8).view(pages, hk, d)
    return data


def batch(seed, lens, *, hq=8, hk=2, d=128, q_len=1, dtype=torch.bfloat16, device="cpu", spread=1.0, q_std=1.5):
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    width = max(1, max(-(-n // 16) for n in lens)) + 2
    counts = [-(-n // 16) for n in lens]
    pages = 3 + sum(counts)
    ids = (torch.randperm(pages - 1, generator=g) + 1).tolist()
    table = torch.full((b, width), 2 ** 30, dtype=torch.int32)  # what is not in use names no page
    used = torch.zeros((pages, 16), dtype=torch.bool)
    for i, n in enumerate(lens):
        mine = [ids.pop() for _ in range(counts[i])]
        table[i, : len(mine)] = torch.tensor(mine, dtype=torch.int32)
        for j, p in enumerate(mine):
            used[p, : max(0, min(16, n - 16 * j))] = True
    data = pool(seed, pages, hk, d, used, spread)
    q = torch.randn((b * q_len, hq, d), generator=g).mul_(q_std).to(dtype)
    return SimpleNamespace(q=q.to(device), kv=LayerKV4(data.to(device), d, 16), table=table.to(device), lens=list(lens),
                           seq_lens=torch.tensor(lens, dtype=torch.int32, device=device), scale=1 / math.sqrt(d), q_len=q_len, d=d, hq=hq, hk=hk)


def call(ops, s, **how):
    return ops.paged_attn_decode_kv4(s.q, s.kv, s.table, s.seq_lens, sm_scale=s.scale, q_len=s.q_len, **how)


def exact(s):
    """Per query row: (o, sum p (|m| + s c), bound of what a score is the sum of, keys, largest |m| + 15 s)."""
    out, q, g = {}, s.q.cpu().double(), s.hq // s.hk
    codes, sc, mi = unpack(s.kv.data)
    parts = mi[..., None].abs() + sc[..., None] * codes.double().unflatten(-1, (-1, 64))
    vals = (mi[..., None] + sc[..., None] * codes.double().unflatten(-1, (-1, 64))).flatten(-2)
    parts = parts.flatten(-2)
    for i, n in enumerate(s.lens):
        n = min(n, 16 * s.table.shape[1])
        ids = s.table[i, : -(-n // 16)].cpu().long()
        k, v, ka, va = (x[e][ids].transpose(0, 1).flatten(1, 2)[:, :n] for x, e in ((vals, 0), (vals, 1), (parts, 0), (parts, 1)))
        for j in range(s.q_len):
            sees = max(0, n - (s.q_len - 1 - j))
            x = q[i * s.q_len + j].view(s.hk, g, s.d)
            if sees == 0:
                zero = torch.zeros(s.hk, g, s.d, dtype=torch.float64)
                out[i * s.q_len + j] = (zero, zero, zero[..., :1], 0, 0.0)
                continue
            p = torch.softmax(x @ k[:, :sees].transpose(1, 2) * s.scale, -1)
            size = (x.abs() @ ka[:, :sees].transpose(1, 2)).amax(-1, keepdim=True) * abs(s.scale)
            out[i * s.q_len + j] = (p @ v[:, :sees], p @ va[:, :sees], size, sees, float(va[:, :sees].max()))
    return out


def assert_attends(s, got, want):
    """Roundings on the way to ``o = sum p (m + s c) / l``: a score is a sum of ``d`` products and a few more, on tensor cores, whose additions may cut off
    (2^-23 each of at most ``size``, and a query's values 2^-31 of its largest one); a score off by e puts p off by e, and l too; p times the scale to fp16 (2^-11
    each for bf16 queries, 2^-22 for fp16 ones, or 2^-25 where the largest is 2^7 at least, times up to 15); exponentials and sums over the keys in fp32 (a key in eight counts as one addition); and the result to its type."""
    last = torch.finfo(s.q.dtype).eps / 2
    each = 2.0 ** -11 if s.q.dtype is torch.bfloat16 else 2.0 ** -22
    got = got.cpu().double().view(-1, s.hk, s.hq // s.hk, s.d)
    for r, (o, weight, size, n, top) in want.items():
        score = (s.d + 16) * 2.0 ** -23 * size
        limit = last * o.abs() + (1 + last) * (weight * (each + 2 * score + (16 + n / 8) * 2.0 ** -23) + n * 2.0 ** -32 * top) + 1e-37
        if s.q.dtype is torch.float16:
            limit = limit + 2.0 ** -25
        off = (got[r] - o).abs() - limit
        assert torch.isfinite(got[r]).all() and (off <= 0).all(), f"query row {r} of {n} keys: off by up to {off.max():.3g} more than {limit.max():.3g}"


HALF = torch.float16
BATCHES = [  # lengths, what else
    ([1], {}),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 64, 65], {}),
    ([48], {"hq": 32, "hk": 8}),
    ([700, 0, 1999, 5], {"hq": 32, "hk": 8}),
    ([100, 101, 117, 400], {"d": 64}),
    ([333, 1, 0, 90], {"d": 64, "hq": 14, "hk": 2, "dtype": HALF}),
    ([333, 40], {"hq": 3, "hk": 3}),
    ([513, 514, 20], {"hq": 8, "hk": 1}),
    ([600, 77], {"hq": 9, "hk": 1, "dtype": HALF}),
    ([600, 77, 16], {"hq": 16, "hk": 1}),
    ([610, 18], {"hq": 17, "hk": 1}),
    ([256, 300, 259, 4, 3, 1, 0], {"q_len": 4, "hq": 8, "hk": 2}),
    ([64, 66, 3, 2, 65, 80], {"q_len": 3, "hq": 5, "hk": 1}),
    ([90, 31], {"q_len": 5, "hq": 24, "hk": 2}),
    ([200, 233, 7], {"d": 256, "hq": 8, "hk": 1, "q_len": 2}),
    ([96, 120, 1], {"d": 256, "hq": 4, "hk": 1, "dtype": HALF}),
    ([301, 64], {"d": 256, "hq": 16, "hk": 2, "q_len": 4}),
    ([2049, 1500], {"spread": 1e4}),
    ([5000, 4999, 130], {"hq": 4, "hk": 1}),
]
