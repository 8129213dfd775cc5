"""The operators of a served batch, one after the other as a server runs them, each checked against its definition at every step.

A model of one layer: a token's row of a table is its q, k and v, and the attention's output times a matrix its logits.  Two groups of
requests share their first pages.  Their prompts are planned as ragged batches that take pages from a free list; then every request answers
token by token: plan, KV write, attention over the shared prefixes, counting, processing, arg-max."""

from types import SimpleNamespace

import numpy as np
import torch

from mfq_b200 import ops
from mfq_b200.engine.kv_cache import PagedKVCache
from mfq_b200.ops import reference
from serve_cases import assert_logits, exact_counts, exact_logits, exact_plan, plan_parts, records, words
from shared_attn_cases import assert_attends, exact

HQ, HK, D, VOCAB, THETA, FILL = 8, 2, 128, 1003, 1e4, -1e30


def write(cache, qkv, positions, slots):
    kv = cache.layer(0)
    if qkv.is_cuda:
        return ops.rope_kv_write(qkv, positions, slots, kv, n_q=HQ, n_kv=HK, head_dim=D, theta=THETA)
    x = qkv.view(-1, HQ + 2 * HK, D)
    reference.write_kv(kv, reference.rope(x[:, HQ : HQ + HK], positions, THETA), x[:, HQ + HK :], slots)
    return reference.rope(x[:, :HQ], positions, THETA)


def serve(device, *, steps=20, graphed=False):
    g = torch.Generator().manual_seed(3)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    embedding = torch.randn((VOCAB, (HQ + 2 * HK) * D), generator=g).to(torch.bfloat16).to(device)
    output = torch.randn((HQ * D, VOCAB), generator=g).mul_(0.3).to(device)
    groups = [(50, [7, 1, 30, 14]), (35, [2, 20, 5])]  # tokens of the common prompt, of each request's own
    b = sum(len(own) for _, own in groups)
    cache = PagedKVCache(layers=1, kv_heads=HK, head_dim=D, num_pages=120, max_seqs=b + 2, max_pages_per_seq=9, device=device)
    cache.block_table.zero_()
    row_of = [4, 0, 6, 2, 8, 3, 5]  # table rows of the requests
    free = (torch.randperm(119, generator=g) + 1).to(torch.int32).to(device)
    past, lens, prompts = [0] * b, [], []
    for shared, own in groups:
        common = torch.randint(0, VOCAB, (shared,), generator=g).tolist()
        for n in own:
            prompts.append(common + torch.randint(0, VOCAB, (n,), generator=g).tolist())
            lens.append(shared + n)

    def read(requests, upto):  # their prompts up to a token, as one ragged batch
        nonlocal free
        counts = [upto[i] - past[i] for i in requests]
        args = (i32([row_of[i] for i in requests]), i32([past[i] for i in requests]), i32(counts))
        want, _ = exact_plan(cache.block_table, *args, sum(counts), 16, free)
        plan = ops.plan_batch(cache.block_table, *args, tokens=sum(counts), pages=free)
        for got, w in zip(plan_parts(plan), want):
            assert got.tolist() == w
        free = free[plan.check()[1] :].contiguous()
        ids = i32([t for i in requests for t in prompts[i][past[i] : upto[i]]])
        write(cache, embedding[ids.long()], plan.positions, plan.slots)
        for i in requests:
            past[i] = upto[i]

    first, members = 0, []
    for shared, own in groups:  # the first of a group reads the common pages, the others' rows get them
        whole = shared // 16 * 16
        read([first], {first: whole})
        for i in range(first + 1, first + len(own)):
            cache.block_table[row_of[i], : whole // 16] = cache.block_table[row_of[first], : whole // 16]
            past[i] = whole
        members += range(first, first + len(own))
        first += len(own)
    read(members, dict(enumerate(lens)))

    starts, prefixes = i32([0, 4, 7]), i32([50 // 16 * 16, 35 // 16 * 16])
    recs = records([(0.0, 0.0, 1.0), (0.5, 0.1, 1.3), (0.0, 0.0, 1.5), (1.0, 0.0, 1.0), (0.0, 0.4, 0.9), (0.0, 0.0, 1.0), (0.2, 0.2, 1.1)], device)
    counts = torch.zeros((b, VOCAB), dtype=torch.int16, device=device)
    own_row = torch.arange(b, dtype=torch.int32, device=device)
    for i, p in enumerate(prompts):
        ops.count_tokens(counts, i32(p), i32([i] * len(p)), prompt=True)
    bias = (torch.randint(-1, VOCAB, (b, 6), generator=g, dtype=torch.int32).to(device), torch.randn((b, 6), generator=g).mul_(3).to(device))
    mask = (torch.rand((b, VOCAB), generator=g) < 0.5).numpy()
    mask[:2] = True
    allowed = words(mask, device)
    rows, pasts, ones = i32(row_of), i32(past), i32([1] * b)
    ids = i32([p[-1] for p in prompts])  # fed once more, as the first tokens of the answers
    pool = torch.zeros(b, dtype=torch.int32, device=device)

    def step():
        plan = ops.plan_batch(cache.block_table, rows, pasts, ones, tokens=b, pages=pool)
        q = write(cache, embedding[ids.long()], plan.positions, plan.slots)
        o = ops.paged_attn_decode_shared(q, cache.layer(0), plan.block_table, plan.seq_lens, starts, prefixes, sm_scale=D ** -0.5, max_group=4, max_prefix=48)
        ops.count_tokens(counts, ids, own_row)
        raw = (o.float().view(b, -1) @ output).to(torch.bfloat16)
        logits = ops.process_logits(raw, recs, counts=counts, bias=bias, allowed=allowed, fill=FILL)
        return plan, q, o, raw, logits

    def checked(held, seen, table):
        plan, q, o, raw, logits = held
        want, after = exact_plan(table, rows, pasts, ones, b, 16, pool)
        for got, w in zip(plan_parts(plan), want):
            assert got.tolist() == w
        assert cache.block_table.tolist() == after
        s = SimpleNamespace(q=q, kv=cache.layer(0), table=plan.block_table, seq_lens=plan.seq_lens, scale=D ** -0.5, q_len=1, grouped=list(range(b)), d=D, hq=HQ, hk=HK)
        assert_attends(s, o, exact(s))
        assert np.array_equal(counts.cpu().numpy().astype(np.int64) & 0xFFFF, exact_counts(seen, ids, own_row, False))
        assert_logits(logits, *exact_logits(raw, recs, counts, bias, mask, None, 0, FILL), FILL)
        return plan.check()[1]

    graph = None
    if graphed:  # the words of the captured calls are those of the replays: what a warm-up would count is taken back
        before = counts.clone(), cache.block_table.clone()
        pool.copy_(free[:b])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        counts.copy_(before[0])
        cache.block_table.copy_(before[1])
    answers = []
    for _ in range(steps):
        pool.copy_(free[:b])
        seen, table = counts.clone(), cache.block_table.clone()
        if graph is not None:
            graph.replay()
        else:
            held = step()
        free = free[checked(held, seen, table) :].contiguous()
        ids.copy_(held[4].argmax(-1))
        pasts += 1
        answers.append(ids.tolist())
    assert all(mask[i, t] for a in answers for i, t in enumerate(a))
    return answers
