"""The operators of a served batch on CPU tensors, and what they refuse."""

import numpy as np
import pytest
import torch

from mfq_b200 import ops
from serve_cases import LOGITS, PLANS, assert_logits, exact_counts, exact_logits, exact_plan, logits_case, plan_case, plan_parts, records, words
from served_batch import serve


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,r,v,how", LOGITS)
def test_process_logits(b, r, v, how, dtype):
    args, table = logits_case(v + b, b, r, v, dtype, **how)
    want, big, masked = exact_logits(args["logits"], args["records"], args["counts"], args["bias"], table, args["rows"], args["first"], -np.inf)
    assert_logits(ops.process_logits(**args), want, big, masked, float("-inf"))
    assert_logits(ops.process_logits(**args, fill=-1e30), *exact_logits(args["logits"], args["records"], args["counts"], args["bias"], table, args["rows"],
                                                                      args["first"], float(torch.tensor(-1e30).to(dtype))), -1e30)


def test_process_logits_in_place_and_unusual_values():
    logits = torch.tensor([[float("nan"), float("inf"), -float("inf"), 1.0, -2.0, torch.finfo(torch.float32).min]])
    counts = torch.tensor([[0, 1, 2, -32768, -32766, 0]], dtype=torch.int16)
    got = ops.process_logits(logits, records([(0.5, 0.25, 2.0)]), counts=counts, allowed=words(np.array([[False, True, True, True, True, False]])), out=logits)
    assert got is logits
    assert got[0].tolist() == [-float("inf"), float("inf"), -float("inf"), 0.5, -5.0, -float("inf")]


@pytest.mark.parametrize("prompt", [False, True])
def test_count_tokens(prompt):
    g = torch.Generator().manual_seed(3)
    counts = torch.randint(-32768, 32767, (3, 50), generator=g).to(torch.int16)
    counts[0, :10] = 32766
    tokens, rows = torch.randint(-3, 55, (400,), generator=g, dtype=torch.int32), torch.randint(-1, 4, (400,), generator=g, dtype=torch.int32)
    want = exact_counts(counts, tokens, rows, prompt)
    ops.count_tokens(counts, tokens, rows, prompt=prompt)
    assert np.array_equal(counts.numpy().astype(np.int64) & 0xFFFF, want)


@pytest.mark.parametrize("b,most,past,how", PLANS)
def test_plan_batch(b, most, past, how):
    (table, rows, pasts, counts), kw = plan_case(b + most, b, most, past, **how)
    for spare in (0, 5):
        kw["tokens"] += spare
        want, after = exact_plan(table, rows, pasts, counts, **kw)
        mine = table.clone()
        plan = ops.plan_batch(mine, rows, pasts, counts, **kw)
        assert [x.tolist() for x in plan_parts(plan)] == want and mine.tolist() == after
        assert plan.check() == tuple(want[-1])


BAD_PLANS = [("row", "outside the table"), ("negative row", "outside"), ("past", "negative"), ("count", "negative"), ("long", "more pages than a row"),
             ("places", "more tokens than"), ("twice", "another one has"), ("free", "too few free pages"), ("none free", "too few free pages")]


def spoilt_plan(what, device="cpu"):
    (table, rows, past, counts), kw = plan_case(4, 6, 60, 50, pages=True, device=device)
    past, counts = past.clone(), counts.clone()
    counts[2:5] = 40
    kw["tokens"] = int(counts.sum())
    if what == "row":
        rows[3] = table.shape[0]
    elif what == "negative row":
        rows[0] = -1
    elif what == "past":
        past[1] = -1
    elif what == "count":
        counts[5] = -7
    elif what == "long":
        past[4] = 2 ** 31 - 20
    elif what == "places":
        kw["tokens"] -= 1
    elif what == "twice":
        rows[5] = rows[1]
    elif what == "free":
        kw["pages"] = kw["pages"][:2].contiguous()
    else:
        kw["pages"] = kw["pages"][:0]
    return (table, rows, past, counts), kw


@pytest.mark.parametrize("what,why", BAD_PLANS)
def test_plan_batch_refuses_on_the_device(what, why):
    args, kw = spoilt_plan(what)
    before = args[0].clone()
    plan = ops.plan_batch(*args, **kw)
    with pytest.raises(ValueError, match=why):
        plan.check()
    assert torch.equal(args[0], before)
    assert not plan.block_table.any() and not plan.q_starts.any() and not plan.seq_lens.any() and (plan.slots == -1).all() and (plan.tok_seq == -1).all()


def test_refusals():
    x, rec = torch.zeros(2, 40), records([(0, 0, 1)] * 2)
    i32 = torch.int32
    for bad in (dict(logits=torch.zeros(40)), dict(logits=torch.zeros(2, 40).double()), dict(logits=torch.zeros(40, 2).t()), dict(records=rec.float()),
                dict(records=rec[:, :6]), dict(records=rec[:1]), dict(records=rec[:0], rows=torch.zeros(2, dtype=i32)), dict(rows=torch.zeros(3, dtype=i32)), dict(rows=torch.zeros(2)),
                dict(counts=torch.zeros(2, 40)), dict(counts=torch.zeros((2, 39), dtype=torch.int16)), dict(counts=torch.zeros((1, 40), dtype=torch.int16)),
                dict(bias=(torch.zeros((2, 3), dtype=i32), torch.zeros(2, 4))), dict(bias=(torch.zeros((2, 3)), torch.zeros(2, 3))),
                dict(bias=(torch.zeros((2, 65537), dtype=i32), torch.zeros(2, 65537))), dict(allowed=torch.zeros((2, 1), dtype=i32)), dict(allowed=torch.zeros((2, 2))),
                dict(first=-1), dict(first=25, allowed=torch.zeros((2, 2), dtype=i32)), dict(out=torch.zeros(2, 41)), dict(out=torch.zeros(2, 40, dtype=torch.bfloat16)),
                dict(out=torch.zeros(1, 40).expand(2, 40))):
        with pytest.raises(ValueError):
            ops.process_logits(**{"logits": x, "records": rec, **bad})
    counts = torch.zeros((2, 9), dtype=torch.int16)
    one = torch.zeros(1, dtype=i32)
    for bad in ((counts.int(), one, one), (counts[0], one, one), (counts, one.long(), one), (counts, one, torch.zeros(2, dtype=i32)), (counts.t(), one, one)):
        with pytest.raises(ValueError):
            ops.count_tokens(*bad)
    table = torch.zeros((3, 4), dtype=i32)
    for bad, kw in (((table.long(), one, one, one), {}), ((table[:, ::2], one, one, one), {}), ((table, one, one.repeat(2), one), {}), ((table, one[:0], one[:0], one[:0]), {}),
                    ((table, one, one, one), {"tokens": -1}), ((table, one, one, one), {"page_size": 0}), ((table, one, one, one), {"page_size": 2 ** 30}),
                    ((table, one, one, one), {"pages": one.long()}), ((table, *[torch.zeros(1025, dtype=i32)] * 3), {}),
                    ((torch.zeros((65537, 1), dtype=i32), one, one, one), {"pages": one})):
        with pytest.raises(ValueError):
            ops.plan_batch(*bad, **{"tokens": 4, **kw})


def test_empty_calls():
    assert ops.process_logits(torch.zeros(0, 5), records([(0, 0, 1)])).shape == (0, 5)
    assert ops.process_logits(torch.zeros(1, 0), records([(0, 0, 1)])).shape == (1, 0)
    counts, none = torch.zeros((2, 9), dtype=torch.int16), torch.zeros(0, dtype=torch.int32)
    ops.count_tokens(counts, none, none)
    assert not counts.any()
    plan = ops.plan_batch(torch.ones((1, 1), dtype=torch.int32), *[torch.zeros(1, dtype=torch.int32)] * 3, tokens=0)
    assert plan.check() == (0, 0) and not plan.block_table.any()


def test_plans_of_too_many_places_are_refused():
    """Places are counted in 32 bits on the device."""
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="tokens"):
        ops.plan_batch(torch.ones((1, 4), dtype=torch.int32), one, one, one, tokens=(1 << 30) + 1)


def test_a_served_batch():
    serve("cpu")


def test_the_c_entry_refuses_short_masks_of_the_last_tokens():
    """Ids up to 2^31 - 2: the mask's words are counted without passing 31 bits (refused before anything is launched)."""
    from mfq_b200.ops.lib import LIB_PATH, lib
    if not LIB_PATH.exists():
        pytest.skip("the CUDA library is not built")
    for first, v in ((2 ** 31 - 2, 1), (2 ** 31 - 41, 40), (64, 33)):
        assert lib().mfq_process_logits(16, 16, 0, 1, v, v, v, 16, 1, None, 0, None, None, 0, 16, (first + v + 31) // 32 - 1, None, first, 0.0, None) == -1


def test_rows_of_counts_that_lie_over_one_another_are_refused():
    """A token of one row would be another's of the next."""
    buffer, one = torch.zeros(40, dtype=torch.int16), torch.zeros(1, dtype=torch.int32)
    for bad in (buffer[:9].expand(3, 9), buffer.as_strided((3, 9), (5, 1))):
        with pytest.raises(ValueError, match="counts"):
            ops.count_tokens(bad, one, one)
    ops.count_tokens(buffer[:9].expand(1, 9), one, one)
    assert buffer[0] == 1
