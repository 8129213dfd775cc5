"""Calls of the cache held in 4 bits that its documentation allows or refuses and that are easily got wrong, on CPU tensors."""

import math

import pytest
import torch

from mfq_b200 import ops
from kv4_cases import batch, call


@pytest.mark.parametrize("hq,d", [(2, 128), (4, 128), (8, 64), (4, 256)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_a_later_token_of_a_window_is_not_seen_through_its_nan(what, hq, d):
    s = batch(2, [64, 90, 33], hq=hq, hk=2, d=d, q_len=4)
    clean = call(ops, s)
    assert torch.isfinite(clean).all()
    k, v = torch.randn(1, 2, d), torch.randn(1, 2, d)
    (k if what == "k" else v)[:] = math.nan
    for row, n in enumerate((64, 90, 33)):
        ops.kv4_write(k, v, (s.table[row, (n - 1) // 16 : (n - 1) // 16 + 1] * 16 + (n - 1) % 16).int(), s.kv)
    out = call(ops, s).view(3, 4, hq, d)
    assert torch.equal(out[:, :3], clean.view(3, 4, hq, d)[:, :3]) and out[:, 3].isnan().all()
