"""What the criterion of averages lets pass and what it does not: attention in 64 bits with one step of it done in fewer bits, or a key left out."""

import pytest
import torch

from mfq_b200 import ops
from kv4_cases import BATCHES, assert_attends, batch, call, exact, unpack
from kv4_rms import assert_close_on_average, exact_and_weights, skewed

CASES = [x for x in BATCHES if sum(x[0]) > 700 and "spread" not in x[1]]
HALF, BF16 = torch.float16, torch.bfloat16


def emulated(s, *, weights=None, terms=None, scores=None, drop=False):
    """``weights``: the type of p, ``terms``: of p s, ``scores``: of the scores; ``drop``: a key in the middle of each row counts as none."""
    codes, sc, mi = unpack(s.kv.data)
    codes, as_type = codes.double(), lambda x, t: x if t is None else x.to(t).double()  # noqa: E731
    out, g, groups = torch.zeros_like(s.q), s.hq // s.hk, s.d // 64
    for i, n in enumerate(s.lens):
        n = min(n, 16 * s.table.shape[1])
        ids = s.table[i, : -(-n // 16)].long()
        ck, cv, sk, sv, mk, mv = (x[e][ids].transpose(0, 1).flatten(1, 2)[:, :n] for x in (codes, sc, mi) for e in (0, 1))
        k = mk.repeat_interleave(64, -1) + sk.repeat_interleave(64, -1) * ck
        for j in range(s.q_len):
            sees = n - (s.q_len - 1 - j)
            if sees <= 0:
                continue
            x = as_type(s.q[i * s.q_len + j].double().view(s.hk, g, s.d) @ k[:, :sees].transpose(1, 2) * s.scale, scores)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            if drop:
                p[..., sees // 2] = 0
            p = as_type(p, weights)
            ps = as_type(p[..., None] * sv[:, None, :sees] * 64, terms) / 64
            o = torch.einsum("hgtn,htnc->hgnc", ps, cv[:, :sees].unflatten(-1, (groups, 64))) + torch.einsum("hgt,htn->hgn", p, mv[:, :sees])[..., None]
            out[i * s.q_len + j] = (o.flatten(-2) / p.sum(-1, keepdim=True)).reshape(s.hq, s.d).to(s.q.dtype)
    return out


@pytest.mark.parametrize("lens,how", CASES)
def test_what_passes_and_what_does_not(lens, how):
    for dtype in (HALF, BF16):
        s = batch(len(lens), lens, **{**how, "dtype": dtype})
        want = exact_and_weights(s)
        assert_close_on_average(s, emulated(s), want)
        assert_close_on_average(s, call(ops, s), want)
        if dtype is BF16:
            assert_close_on_average(s, emulated(s, terms=HALF), want)
        for wrong in ({"weights": BF16}, {"scores": HALF}, {"drop": True}, {"terms": BF16}) + (({"terms": HALF},) if dtype is HALF else ()):
            with pytest.raises(AssertionError, match="on the average"):
                assert_close_on_average(s, emulated(s, **wrong), want)


def test_skewed_values_have_no_mean():
    s = skewed(batch(1, [6000], hq=8, hk=2, q_std=0.1, dtype=HALF))
    want = exact_and_weights(s)
    assert all(o.abs().max() < 0.05 * weight.min() for o, weight, _ in want.values())
    assert_close_on_average(s, emulated(s), want)
    assert_attends(s, emulated(s), exact(s))
