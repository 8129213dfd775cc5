"""How far attention over 4-bit pages is off on the average, beside what rounding its outputs takes; and pools whose averages cancel.

A bound for each output has to allow for the worst case in every score, which hides most mistakes.  Errors of many outputs add up as squares: what the
rounding of the outputs leaves is known from the exact outputs themselves, and all else has to be small beside it."""

import torch

from kv4_cases import unpack


def skewed(s, seed=5):
    """V with codes that are mostly small and minima that make up for them: values of mean zero in groups that are not symmetric."""
    d, data = s.d, s.kv.data
    g = torch.Generator().manual_seed(seed)
    shape = (data.shape[0], data.shape[1], 8 * d)
    a, b = (torch.randint(0, 256, shape, generator=g, dtype=torch.uint8) for _ in range(2))
    data[:, :, 9 * d : 17 * d] = (torch.minimum(a & 15, b & 15) | torch.minimum(a & 240, b & 240)).to(data.device)  # 4.84 on the average
    x = data[:, :, 17 * d :].cpu().contiguous().view(torch.bfloat16).view(*shape[:2], -1, 2).float()
    x[..., 1] = -x[..., 0] * (4.84 + 0.3 * torch.randn(x[..., 0].shape, generator=g))
    data[:, :, 17 * d :] = x.to(torch.bfloat16).view(torch.uint8).view(*shape[:2], d).to(data.device)
    return s


def exact_and_weights(s):
    """Per query row that sees something: the outputs in 64 bits, ``sum p s c`` and ``sqrt(sum (p s c)^2)``, each ``[hk, g, D]``."""
    codes, sc, mi = unpack(s.kv.data)
    grown = (sc[..., None] * codes.double().unflatten(-1, (-1, 64))).flatten(-2)
    low = mi[..., None].expand(*mi.shape, 64).flatten(-2)
    out, q, g = {}, s.q.cpu().double(), s.hq // s.hk
    for i, n in enumerate(s.lens):
        n = min(n, 16 * s.table.shape[1])
        ids = s.table[i, : -(-n // 16)].cpu().long()
        gk, gv, lk, lv = (x[e][ids].transpose(0, 1).flatten(1, 2)[:, :n] for x, e in ((grown, 0), (grown, 1), (low, 0), (low, 1)))
        for j in range(s.q_len):
            sees = n - (s.q_len - 1 - j)
            if sees <= 0:
                continue
            x = q[i * s.q_len + j].view(s.hk, g, s.d)
            p = torch.softmax(x @ (lk + gk)[:, :sees].transpose(1, 2) * s.scale, -1)
            out[i * s.q_len + j] = (p @ (lv + gv)[:, :sees], p @ gv[:, :sees], (p.square() @ gv[:, :sees].square()).sqrt())
    return out


def assert_close_on_average(s, got, want, *, products=None, rounded=None):
    """Root mean squares over all outputs, each row and head in units of its own outputs' size.  What may be added, as squares, to the outputs' rounding:

    * V's sums on tensor cores: an addition cuts off less than 2^-23 of the sum so far, so between two meetings of V's sums (4 pairs of pages for fp16 queries, 32 for
      bf16 ones: ``products`` is 16 or 64 additions) less than ``products * 2^-23`` of half of ``sum p s c``, and so of all of it;
    * ``p s`` to fp16 (``rounded`` is 2^-11 of the term, or 2^-22 where it is two numbers), a uniform error on a logarithmic scale: 0.41 of the bound;
    * scores: products and sums in fp32, 2^-24 each; the sum of 30 of them as squares moves p by 2^-20 of ``sqrt(sum (p s c)^2)``;
    and 2 % for the number of samples (some thousand outputs at least)."""
    half = s.q.dtype is torch.float16
    products = products or (16 if half else 64)
    rounded = rounded or (2.0 ** -22 if half else 2.0 ** -11)
    got = got.cpu().double().view(-1, s.hk, s.hq // s.hk, s.d)
    mean = lambda x: x.square().mean(-1, keepdim=True)  # noqa: E731
    off, by = [], []
    for r, (o, weight, spread) in want.items():
        size = mean(o).clamp_min(1e-300)
        off.append(mean(got[r] - o) / size)
        by.append((mean(o.to(s.q.dtype).double() - o) + mean(weight * products * 2.0 ** -24) + mean(spread * (0.41 * rounded + 2.0 ** -20))) / size)
    off, by = torch.cat([x.flatten() for x in off]).mean().sqrt().item(), torch.cat([x.flatten() for x in by]).mean().sqrt().item()
    assert off <= 1.02 * by, f"off by {off:.3g} on the average, {off / by:.2f} times what rounding leaves"
