"""The kernels of a served batch's operators against their definitions in 64 bits."""

import numpy as np
import pytest
import torch

from mfq_b200 import ops
from gpu_common import check_status, require_gpu_lib
from serve_cases import LOGITS, PLANS, assert_logits, exact_counts, exact_logits, exact_plan, logits_case, plan_case, plan_parts, records, words
from served_batch import serve
from test_serve_ops_cpu import BAD_PLANS, spoilt_plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,r,v,how", LOGITS)
def test_process_logits(b, r, v, how, dtype):
    require_gpu_lib()
    args, table = logits_case(v + b, b, r, v, dtype, device="cuda", **how)
    want = exact_logits(args["logits"], args["records"], args["counts"], args["bias"], table, args["rows"], args["first"], -np.inf)
    got = ops.process_logits(**args)
    assert_logits(got, *want, float("-inf"))
    assert torch.equal(got, ops.process_logits(**args, out=args["logits"].clone() if how.get("odd") else None)), "the same inputs, the same bits"
    held = args["logits"]
    assert_logits(ops.process_logits(**args, out=held), *want, float("-inf"))  # in place


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,r,v,how", [(60, 60, 30104, {"k": 40}), (240, 50, 30104, {"mapped": True}), (240, 50, 30100, {"mapped": True, "k": 9, "first": 17}), (240, 240, 30104, {"odd": True})])
def test_process_logits_of_large_batches(b, r, v, how, dtype):
    """Large enough for a thread to have two sets of eight, in wide accesses and value by value."""
    require_gpu_lib()
    args, table = logits_case(v + b, b, r, v, dtype, device="cuda", mask=True, **how)
    want = exact_logits(args["logits"], args["records"], args["counts"], args["bias"], table, args["rows"], args["first"], -np.inf)
    assert_logits(ops.process_logits(**args), *want, float("-inf"))


def test_rows_of_nothing_and_unusual_values():
    require_gpu_lib()
    v = 4096
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        low = torch.finfo(dtype).min
        logits = torch.tensor([float("nan"), float("inf"), -float("inf"), low, -low, 0.0, -0.0, 1.0]).to(dtype).repeat(3, v // 8).cuda()
        mask = np.zeros((3, v), dtype=bool)
        mask[1, 5::8] = True
        mask[2] = True
        rec = records([(0.5, 0.25, 2.0)] * 3, "cuda")
        counts = torch.tensor([1, 1, -32768, 2, 2, 3, -32768, 32767], dtype=torch.int16).repeat(3, v // 8).cuda()
        bias = (torch.tensor([[7, 7, -1]] * 3, dtype=torch.int32, device="cuda"), torch.tensor([[100.0, 0.5, 9.0]] * 3, device="cuda"))
        got = ops.process_logits(logits, rec, counts=counts, bias=bias, allowed=words(mask, "cuda"))
        want = exact_logits(logits, rec, counts, bias, mask, None, 0, -np.inf)
        assert_logits(got, *want, float("-inf"))
        assert (got[0] == -float("inf")).all()


def test_rows_behind_4_gigabytes():
    require_gpu_lib()
    args, table = logits_case(12, 4, 3, 128256, torch.bfloat16, mask=True, k=30, device="cuda")
    args["rows"] = torch.tensor([2, 0, 1, 2], dtype=torch.int32, device="cuda")
    want = ops.process_logits(**args)
    b = 2 ** 32 // (2 * 128256) + 20
    logits = torch.zeros((b, 128256), dtype=torch.bfloat16, device="cuda")
    logits[-4:].copy_(args["logits"])
    rows = torch.full((b,), -1, dtype=torch.int32, device="cuda")
    rows[-4:].copy_(args["rows"])
    got = ops.process_logits(**{**args, "logits": logits, "rows": rows}, out=logits)
    assert torch.equal(got[-4:], want) and not got[: b - 4].any()


def test_records_that_begin_on_4_bytes():
    require_gpu_lib()
    args, table = logits_case(11, 3, 3, 5000, torch.bfloat16, mask=True, device="cuda")
    buffer = torch.zeros(3 * 8 + 1, dtype=torch.int32, device="cuda")
    part = buffer[1:].view(3, 8)
    part.copy_(args["records"])
    args["records"] = part
    assert_logits(ops.process_logits(**args), *exact_logits(args["logits"], part, args["counts"], None, table, None, 0, -np.inf), float("-inf"))


def test_process_logits_by_another_stream_in_a_graph_and_in_bands():
    """A captured call reads what its tensors hold at the replay; rows of a wider buffer leave what lies between them alone."""
    require_gpu_lib()
    args, table = logits_case(5, 4, 4, 3000, torch.bfloat16, mask=True, k=20, device="cuda")
    wide = torch.full((4, 3100), 7.0, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.process_logits(**args, out=wide[:, 50:3050])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.count_tokens(args["counts"], torch.arange(4, device="cuda", dtype=torch.int32), torch.arange(4, device="cuda", dtype=torch.int32))
        ops.process_logits(**args, out=wide[:, 50:3050])
    for _ in range(2):
        args["logits"].copy_(torch.randn(4, 3000, device="cuda"))
        counts = args["counts"].clone()
        graph.replay()
        torch.cuda.synchronize()
        want_counts = exact_counts(counts, torch.arange(4), torch.arange(4), False)
        assert np.array_equal(args["counts"].cpu().numpy().astype(np.int64) & 0xFFFF, want_counts)
        assert_logits(wide[:, 50:3050], *exact_logits(args["logits"], args["records"], args["counts"], args["bias"], table, None, 0, -np.inf), float("-inf"))
        assert (wide[:, :50] == 7).all() and (wide[:, 3050:] == 7).all()


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("v,n", [(50, 4000), (1, 700), (128256, 90000), (333, 31)])
def test_count_tokens(v, n, prompt):
    require_gpu_lib()
    g = torch.Generator().manual_seed(n)
    wide = torch.randint(-32768, 32767, (3, v + 5), generator=g).to(torch.int16)
    wide[0, :10] = 32760
    held = wide.cuda()
    tokens, rows = torch.randint(-3, v + 3, (n,), generator=g, dtype=torch.int32), torch.randint(-1, 4, (n,), generator=g, dtype=torch.int32)
    tokens[: n // 3] = min(5, v - 1)  # one token very often
    want = exact_counts(wide[:, 3 : 3 + v], tokens, rows, prompt)
    ops.count_tokens(held[:, 3 : 3 + v], tokens.cuda(), rows.cuda(), prompt=prompt)
    got = held.cpu()
    assert np.array_equal(got[:, 3 : 3 + v].numpy().astype(np.int64) & 0xFFFF, want)
    assert torch.equal(got[:, :3], wide[:, :3]) and torch.equal(got[:, 3 + v :], wide[:, 3 + v :])


@pytest.mark.parametrize("b,most,past,how", PLANS)
def test_plan_batch(b, most, past, how):
    require_gpu_lib()
    (table, rows, pasts, counts), kw = plan_case(b + most, b, most, past, device="cuda", **how)
    for spare in (0, 1000):
        kw["tokens"] += spare
        want, after = exact_plan(table, rows, pasts, counts, **kw)
        mine = table.clone()
        plan = ops.plan_batch(mine, rows, pasts, counts, **kw)
        for got, w in zip(plan_parts(plan), want):
            assert got.tolist() == w
        assert mine.tolist() == after and plan.check() == tuple(want[-1])


@pytest.mark.parametrize("what,why", BAD_PLANS)
def test_plan_batch_refuses_on_the_device(what, why):
    require_gpu_lib()
    args, kw = spoilt_plan(what, "cuda")
    before = args[0].clone()
    plan = ops.plan_batch(*args, **kw)
    with pytest.raises(ValueError, match=why):
        plan.check()
    assert torch.equal(args[0], before)
    assert not plan.block_table.any() and not plan.q_starts.any() and not plan.seq_lens.any() and (plan.slots == -1).all() and (plan.tok_seq == -1).all()


def test_plan_batch_in_a_graph():
    """Lengths are read at the replay; the places behind the last token are marked."""
    require_gpu_lib()
    (table, rows, pasts, counts), kw = plan_case(9, 8, 30, 60, device="cuda")
    kw["tokens"] = 8 * 30
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = ops.plan_batch(table, rows, pasts, counts, **kw)
    for seed in (1, 2):
        (_, _, p2, c2), _ = plan_case(seed, 8, 30, 60)
        pasts.copy_(p2)
        counts.copy_(c2)
        graph.replay()
        want, _ = exact_plan(table, rows, pasts, counts, **kw)
        for got, w in zip(plan_parts(plan), want):
            assert got.tolist() == w


def test_a_served_batch_and_its_captured_step():
    require_gpu_lib()
    assert serve("cuda") == serve("cuda", graphed=True), "the same kernels on the same inputs"
    check_status()


@pytest.mark.parametrize("ps,past,count", [(2 ** 31 - 1, 5, 3), (2 ** 31 - 1, 0, 1), (2 ** 30 + 3, 2 ** 30 + 2, 1), (2 ** 30, 1, 7)])
def test_plans_of_pages_of_nearly_2_to_the_31_tokens(ps, past, count):
    """Lengths and the size of a page together pass 31 bits; a page of the past is none to hand out again."""
    require_gpu_lib()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = i32([[0], [0]]), i32([1]), i32([past]), i32([count])
    for pages in (None, i32([0, 0])):
        kw = dict(tokens=count + 2, page_size=ps, pages=pages)
        want, after = exact_plan(*args, **kw)
        mine = args[0].clone()
        plan = ops.plan_batch(mine, *args[1:], **kw)
        for got, w in zip(plan_parts(plan), want):
            assert got.tolist() == w
        assert mine.tolist() == after and plan.check() == tuple(want[-1])


def test_more_rows_of_logits_than_a_grid_are_refused():
    require_gpu_lib()
    logits = torch.zeros((65536, 8), device="cuda")
    rows = torch.zeros(65536, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="65535"):
        ops.process_logits(logits, records([(0.0, 0.0, 1.0)], "cuda"), rows=rows)
    ops.process_logits(logits[:65535], records([(0.0, 0.0, 1.0)], "cuda"), rows=rows[:65535])
