"""Batches whose sequences share prefixes, for the tests of ``ops.paged_attn_decode_shared``, with the softmax in 64 bits.

Every place of the pool that no sequence has holds NaN codes under NaN multipliers."""

import math
from types import SimpleNamespace

import torch

from mfq_b200.engine.kv_cache import V_SLOT_OF_TOKEN, V_TOKEN_ORDER, LayerKV


def batch(seed, groups, *, hq=8, hk=2, d=128, q_len=1, behind=0, shuffle=True, device="cpu", v_spread=1.0, q_std=2.0):
    """``groups``: ``[(prefix tokens, [lengths of its sequences])]``; ``behind``: rows in no group."""
    g = torch.Generator().manual_seed(seed)
    lens = [n for _, ns in groups for n in ns] + [40] * behind
    b = len(lens)
    width = max(1, max(-(-n // 16) for n in lens)) + 2
    fronts = [min(p, max(ns, default=0)) // 16 for p, ns in groups]
    pages = 1 + sum(fronts) + sum(-(-n // 16) + 1 for n in lens)
    ids = (torch.randperm(pages - 1, generator=g) + 1).tolist()
    order = torch.randperm(b, generator=g).tolist() if shuffle else list(range(b))
    table = torch.full((b, width), 2 ** 30, dtype=torch.int32)  # what is not in use names no page
    seq_lens = torch.zeros(b, dtype=torch.int32)
    used = torch.zeros((pages, 16), dtype=torch.bool)
    starts, at = [0], 0
    for (prefix, ns), front in zip(groups, fronts):
        shared = [ids.pop() for _ in range(front)]
        for n in ns:
            row, mine = order[at], shared[: prefix // 16]
            keep = len(mine)
            own = [ids.pop() for _ in range(max(0, -(-n // 16) - keep))]
            have = mine + own
            table[row, : len(have)] = torch.tensor(have, dtype=torch.int32)
            seq_lens[row] = n
            for j, p in enumerate(have):
                used[p, : max(0, min(16, n - 16 * j))] = True
            at += 1
        starts.append(at)
    for i in range(behind):
        seq_lens[order[at + i]] = 40
    k = torch.full((pages, hk, d // 64, 16, 64), 0x7F, dtype=torch.uint8)
    v = torch.full((pages, hk, d, 16), 0x7F, dtype=torch.uint8)
    ks, vs = torch.full((pages, hk, 16), math.nan), torch.full((pages, hk, 16), math.nan)
    codes = lambda *s: torch.randn(s, generator=g).mul_(112).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)  # noqa: E731
    k = torch.where(used[:, None, None, :, None], codes(*k.shape), k)
    v = torch.where(used[:, list(V_TOKEN_ORDER)][:, None, None, :], codes(*v.shape), v)
    ks = torch.where(used[:, None, :], torch.rand(ks.shape, generator=g).mul_(0.006).add_(0.006), ks)
    spread = torch.exp2(torch.rand(vs.shape, generator=g).sub_(0.5).mul_(2 * math.log2(v_spread))) if v_spread != 1.0 else 1.0
    vs = torch.where(used[:, None, :], torch.rand(vs.shape, generator=g).mul_(0.006).add_(0.006) * spread, vs)
    f8 = torch.float8_e4m3fn
    kv = LayerKV(k.view(f8).to(device), v.view(f8).to(device), ks.to(device), vs.to(device), 16)
    q = torch.randn((b * q_len, hq, d), generator=g).mul_(q_std).to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return SimpleNamespace(q=q.to(device), kv=kv, table=table.to(device), seq_lens=seq_lens.to(device), starts=i32(starts), prefixes=i32([p for p, _ in groups]),
                           members=i32(order) if shuffle else None, scale=1 / math.sqrt(d), q_len=q_len, grouped=order[:at], d=d, hq=hq, hk=hk)


def call(ops, s, **how):
    return ops.paged_attn_decode_shared(s.q, s.kv, s.table, s.seq_lens, s.starts, s.prefixes, sm_scale=s.scale, members=s.members, q_len=s.q_len, **how)


def exact(s):
    """Per row: (o, sum p |v|, how far scores may be off, keys, largest |v|)."""
    out = {}
    kc, vc = s.kv.k.cpu().float().double(), s.kv.v.cpu().float().double()
    ks, vs = s.kv.k_scale.cpu().double(), s.kv.v_scale.cpu().double()
    slot = list(V_SLOT_OF_TOKEN)
    q, g = s.q.cpu().double(), s.hq // s.hk
    for row in s.grouped:
        n = int(s.seq_lens[row])
        ids = s.table[row, : -(-n // 16)].cpu().long()
        k = (kc[ids].permute(0, 1, 3, 2, 4).flatten(3) * ks[ids][..., None]).transpose(0, 1).flatten(1, 2)[:, :n]
        v = (vc[ids][..., slot].transpose(2, 3) * vs[ids][..., None]).transpose(0, 1).flatten(1, 2)[:, :n]
        for i in range(s.q_len):
            sees = max(0, n - (s.q_len - 1 - i))
            x = q[row * s.q_len + i].view(s.hk, g, s.d)
            if sees == 0:
                zero = torch.zeros(s.hk, g, s.d, dtype=torch.float64)
                out[row * s.q_len + i] = (zero, zero, zero[..., :1], 0, 0.0)
                continue
            p = torch.softmax(x @ k[:, :sees].transpose(1, 2) * s.scale, -1)
            size = (x.abs() @ k[:, :sees].abs().transpose(1, 2)).amax(-1, keepdim=True) * s.scale
            out[row * s.q_len + i] = (p @ v[:, :sees], p @ v[:, :sees].abs(), size, sees, float(v[:, :sees].abs().max()))
    return out


def assert_attends(s, got, want):
    """Roundings on the way to ``o = sum p v / l``: P times the V multiplier to fp16 (2^-11 each, or 2^-25 of 2^4 where it is that small), the scores'
    fp32 sums (``d`` and a few operations on at most ``size``, twice 2^-24 each; a score off by e puts p off by e, and l too), exponentials and
    sums over the keys in fp32 (a key in eight counts as one addition), and the result to bf16 (2^-8)."""
    got = got.cpu().double().view(-1, s.hk, s.hq // s.hk, s.d)
    for r, (o, weight, size, n, top) in want.items():
        score = 2 * (s.d + 8) * 2.0 ** -24 * size
        limit = 2.0 ** -8 * o.abs() + (1 + 2.0 ** -8) * (weight * (2.0 ** -11 + 2 * score + (16 + n / 8) * 2.0 ** -23) + n * 2.0 ** -29 * top) + 1e-37
        off = (got[r] - o).abs() - limit
        assert torch.isfinite(got[r]).all() and (off <= 0).all(), f"query row {r} of {n} keys: off by up to {off.max():.3g} more than {limit.max():.3g}"


BATCHES = [  # groups, what else
    ([(16, [17, 18])], {}),
    ([(0, [1, 5, 16, 17])], {}),
    ([(48, [53, 53])], {"hq": 32, "hk": 8}),
    ([(100, [100, 101, 117, 400])], {"d": 64}),  # the prefix ends inside a page
    ([(33, [1, 0, 16, 33, 34, 700])], {"hq": 4, "hk": 4}),  # rows shorter than the prefix, one without a token
    ([(640, [641 + 7 * i for i in range(9)])], {"hq": 8, "hk": 1}),  # 72 query rows
    ([(320, [330] * 5), (0, [12]), (1000, [1001, 1500]), (15, [40] * 3)], {"hq": 14, "hk": 2, "d": 64, "behind": 3}),
    ([(512, [513 + i for i in range(40)])], {"hq": 8, "hk": 2, "shuffle": False}),
    ([(256, [260, 300, 256 + 3])], {"q_len": 4, "hq": 8, "hk": 2}),
    ([(64, [67, 66, 3, 2, 65, 80])], {"q_len": 3, "hq": 4, "hk": 2, "behind": 1}),  # windows that begin in front of the sequence, or inside the prefix
    ([(200, [230] * 4), (16, [90])], {"d": 256, "hq": 8, "hk": 1, "q_len": 2}),
    ([(96, [120] * 7)], {"d": 256, "hq": 4, "hk": 1}),
    ([(2048, [2049 + 50 * i for i in range(6)])], {"v_spread": 1e4}),
    ([(1000, [1500] * 3)], {"hq": 16, "hk": 1}),
]
