"""Calls of the cache held in 4 bits that its documentation allows or refuses and that are easily got wrong, on CPU tensors."""

import math

import pytest
import torch

from mfq_b200 import ops
from mfq_b200.engine.kv_cache import LayerKV4
from kv4_cases import batch, call, pool


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


def outputs(device="cpu"):
    """Pairs of outputs ``[25, 2, 64]`` that share memory: whether they lie over one another, and the pair."""
    flat = lambda n: torch.zeros(n, device=device)  # noqa: E731
    same, wide, rows = flat(25 * 2 * 64).view(25, 2, 64), flat(25 * 6 * 64).view(25, 6, 64), flat(60 * 2 * 64).view(60, 2, 64)
    heads, three = flat(4 * 25 * 64).view(4, 25, 64), flat(25 * 4 * 80).view(25, 4, 80)
    return [(True, same, same), (True, same, same.clone().set_(same)), (True, wide[:, :2], wide[:, 1:3]), (True, wide[:, 1:3], wide[:, :2]), (True, rows[:25], rows[24:49]),
            (True, rows[24:49], rows[:25]), (True, wide[:, :2], wide[:, 0:4:2]), (True, wide[:, 0:4:2], wide[:, 2:6:2]), (True, wide[:, 0:2], wide.flatten(1)[:, 32 : 32 + 128].unflatten(1, (2, 64))),
            (True, heads[:2].transpose(0, 1), heads[1:3].transpose(0, 1)), (True, same, same.flatten().view(2, 25, 64).transpose(0, 1)), (True, rows[0:50:2], rows[2:52:2]),
            (True, three[:, :2, :64], three.flatten(1)[:, 76 : 76 + 160].unflatten(1, (2, 80))[..., :64]),
            (False, wide[:, :2], wide[:, 2:4]), (False, wide[:, 4:], wide[:, :2]), (False, wide[:, 0:4:2], wide[:, 1:5:2]), (False, rows[:25], rows[25:50]), (False, rows[0:50:2], rows[1:51:2]),
            (False, heads[:2].transpose(0, 1), heads[2:].transpose(0, 1)), (False, wide[:, :2], wide[:, 2:6:2]), (False, three[:, :2, :64], three[:, 2:, :64]), (False, same, same.clone())]


@pytest.mark.parametrize("case", range(len(outputs())))
def test_keys_read_back_over_values_are_refused(case):
    over, k_out, v_out = outputs()[case]
    kv = LayerKV4(pool(1, 4, 2, 64), 64, 16)
    table, starts = torch.tensor([[1, 2], [3, 0]], dtype=torch.int32), torch.tensor([0, 20, 25], dtype=torch.int32)
    if over:
        with pytest.raises(ValueError, match="v_out: lies over k_out"):
            ops.kv4_gather(kv, table, starts, k_out=k_out, v_out=v_out)
        assert (k_out == 0).all() and (v_out == 0).all()
    else:
        k, v = ops.kv4_gather(kv, table, starts, 25, dtype=torch.float32)
        ops.kv4_gather(kv, table, starts, k_out=k_out, v_out=v_out)
        assert torch.equal(k, k_out) and torch.equal(v, v_out)


def test_one_row_of_neighbouring_outputs():
    kv = LayerKV4(pool(1, 4, 2, 64), 64, 16)
    row, i32 = torch.zeros(1, 4, 64), lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    ops.kv4_gather(kv, i32(1)[None], i32(0, 1), k_out=row[:, :2], v_out=row[:, 2:])
    assert (row != 0).any(-1).all()
    with pytest.raises(ValueError, match="lies over"):
        ops.kv4_gather(kv, i32(1)[None], i32(0, 1), k_out=row[:, :2], v_out=row[:, 1:3])


def test_more_than_32_bits_count_is_refused():
    """Memory that is asked for and never touched; a token's row may be one for all."""
    kv, n = LayerKV4(pool(1, 2, 1, 64), 64, 16), 2 ** 32 + 3
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="below 2\\^31"):
        ops.kv4_write(torch.zeros(1, 1, 64).expand(n, 1, 64), torch.zeros(1, 1, 64).expand(n, 1, 64), i32[:1].expand(n), kv)
    with pytest.raises(ValueError, match="block_table: .*at most 1073741824"):
        ops.kv4_gather(kv, torch.empty(2 ** 30 + 1, 1, dtype=torch.int32, device="meta"), i32, 1)
