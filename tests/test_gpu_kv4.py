"""The kernels of the cache held in 4 bits against the definition in 64 bits, and bytes against the restatement."""

import math

import pytest
import torch

from mfq_b200 import ops
from mfq_b200.engine.kv_cache import LayerKV4
from mfq_b200.ops import kv4, reference
from gpu_common import check_status, require_gpu_lib
from kv4_cases import BATCHES, assert_attends, batch, call, exact, pool, values
from test_kv4_cpu import groups

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def empty_pool(pages, hk, d, device="cuda"):
    return LayerKV4(torch.full((pages, hk, 18 * d), 255, dtype=torch.uint8, device=device), d, 16)


def write_both(k, v, slots, kv):
    """On the GPU, and the bytes that the restatement leaves."""
    want = LayerKV4(kv.data.cpu(), kv.head_dim, 16)
    ops.kv4_write(k, v, slots, kv)
    check_status()
    ops.kv4_write(k.cpu(), v.cpu(), slots.cpu(), want)
    return want.data


def assert_bytes(got, want):
    got = got.cpu()
    if not torch.equal(got, want):
        a, b = values(got), values(want)
        at = ((a != b) & ~(a.isnan() & b.isnan())).nonzero()
        assert False, f"{(got != want).sum()} bytes, {len(at)} values differ; the first (K or V, page, head, token, dim): " + "; ".join(
            f"{tuple(i.tolist())}: {a[tuple(i)].item():.9g}, not {b[tuple(i)].item():.9g}" for i in at[:4])


SLOTS = {  # pages, slots of the tokens in order
    "one": (3, [37]),
    "a page": (3, list(range(16, 32))),
    "from inside a page": (6, list(range(21, 21 + 70))),
    "single tokens of many": (40, [16 * i + (5 * i) % 16 for i in range(40)]),
    "no order": (9, torch.randperm(144, generator=torch.Generator().manual_seed(1)).tolist()),
    "backwards": (4, list(range(63, -1, -1))),
    "pages in no order": (7, [16 * p + t for p in (5, 2, 6, 0, 3) for t in range(16)][3:-2]),
    "padded": (4, [-1, -1, 3, 4, -1, 5, 6, 16, 17, -5, 18, 47, -1, 48] + list(range(32, 47)) + [-1] * 9),
    "neighbours that are two runs": (4, [14, 15, 16, 17, 17 + 3, 21, 22, 47, 48, 0, 1]),
    "evens": (4, list(range(0, 64, 2))),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hk", [(64, 3), (128, 2), (256, 1)])
@pytest.mark.parametrize("name", list(SLOTS))
def test_written_bytes(name, d, hk, dtype):
    require_gpu_lib()
    pages, slots = SLOTS[name]
    n = len(slots)
    wide = torch.randn(n, 2 * hk + 1, d).mul_(3).add_(torch.randn(2 * hk + 1, d)).to(dtype).cuda()
    kv = empty_pool(pages, hk, d)
    at = torch.tensor(slots, dtype=torch.int32, device="cuda")
    want = write_both(wide[:, 1 : hk + 1], wide[:, hk + 1 :], at, kv)
    assert_bytes(kv.data, want)
    kv = empty_pool(pages, hk, d)
    ops.kv4_write(wide[:, 1 : hk + 1].transpose(0, 1).contiguous().transpose(0, 1), wide[:, hk + 1 :].contiguous(), at, kv)  # heads outside, tokens outside
    check_status()
    assert_bytes(kv.data, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_groups_that_are_close_calls(dtype):
    """Ties, steps of 2^-133, values of 2^126, groups of one value, and groups that are none."""
    require_gpu_lib()
    x = groups()
    g = torch.Generator().manual_seed(9)
    more = torch.randn(4000, 64, generator=g) * torch.exp2(torch.randint(-30, 30, (4000, 1), generator=g).float())
    more[::3] = (more[::3] * 16 / more[::3].abs().amax(-1, keepdim=True)).round() / 2  # many halves of steps
    more[1::5] += 1000 * torch.randn(800, 1, generator=g)
    x = torch.cat([x, more, torch.randn(6, 64, generator=g)]).to(dtype)
    for i, bad in enumerate((math.nan, math.inf, -math.inf, 3e38, -math.nan)):
        x[-1 - i, 7 * i] = bad
    x = torch.cat([x, x[: -x.shape[0] % 34 or 34]])[: x.shape[0] // 34 * 34 + 34].view(-1, 17, 2 * 64).cuda()
    kv = empty_pool(x.shape[0] // 16 + 2, 17, 128)
    at = torch.arange(5, x.shape[0] + 5, dtype=torch.int32, device="cuda")
    want = write_both(x, -x, at, kv)
    assert_bytes(kv.data, want)
    one = empty_pool(x.shape[0] // 16 + 2, 17, 128)  # tokens by themselves
    for i in (0, 1, 30, x.shape[0] - 1):
        ops.kv4_write(x[i : i + 1], -x[i : i + 1], at[i : i + 1], one)
        t = int(at[i])
        a, b = values(one.data.cpu()[t // 16 : t // 16 + 1])[:, 0, :, t % 16], values(want[t // 16 : t // 16 + 1])[:, 0, :, t % 16]
        assert torch.equal(a.nan_to_num(123.0), b.nan_to_num(123.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hk", [(64, 3), (128, 2), (256, 1)])
@pytest.mark.parametrize("lens,first", [([1], [0]), ([16], [0]), ([33], [15]), ([0, 5, 33, 16, 1, 0, 0, 50], [3, 0, 17, 16, 31, 0, 9, 7]), ([1] * 40, list(range(40))),
                                        ([0, 0], [1, 2]), ([300, 1, 17], [4, 9, 16])])
def test_read_back(lens, first, d, hk, dtype):
    require_gpu_lib()
    width = max(f + n for f, n in zip(first, lens)) // 16 + 2
    b = len(lens)
    pages = b * width + 3
    data = pool(len(lens), pages, hk, d)
    table = torch.randperm(pages)[: b * width].view(b, width).int()
    starts = [3]
    for n in lens:
        starts.append(starts[-1] + n)
    rows = starts[-1] + 5
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    outs = []
    for device in ("cpu", "cuda"):
        k_out = torch.full((rows, hk + 1, d), 7.0, dtype=dtype, device=device)
        v_out = torch.full((hk, rows, d), 7.0, dtype=dtype, device=device).transpose(0, 1)
        kv = LayerKV4(data.to(device), d, 16)
        ops.kv4_gather(kv, table.to(device), i32(starts).to(device), first=i32(first).to(device), k_out=k_out[:, 1:], v_out=v_out)
        outs.append((k_out.cpu(), v_out.cpu()))
    check_status()
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    if starts[-1] > 3:
        k, _ = ops.kv4_gather(kv, table.cuda(), i32([0] + [s - 3 for s in starts[1:]]).cuda(), starts[-1] - 3, dtype=dtype, first=i32(first).cuda())
        assert torch.equal(k.cpu(), outs[0][0][3 : starts[-1], 1:])


def run(s, want, **how):
    out = torch.full_like(s.q, 3.0)
    assert call(ops, s, out=out, **how) is out
    check_status()
    assert_attends(s, out, want)
    return out


@pytest.mark.parametrize("lens,how", BATCHES)
def test_attention_against_the_definition(lens, how):
    require_gpu_lib()
    s = batch(len(lens), lens, device="cuda", **how)
    want = exact(s)
    one = run(s, want)
    assert torch.equal(one, run(s, want)), "the same inputs, the same bits"
    for most in (0, 1, max(lens), 10 ** 6):  # a wrong one is only slower
        run(s, want, max_len=most)


@pytest.mark.parametrize("form", [(1, 0), (2, 0), (4, 0), (8, 0), (0, 1), (0, 3), (0, 50), (0, 592)])
@pytest.mark.parametrize("lens,how", BATCHES + [([40 * (i % 9) for i in range(150)], {"hq": 4, "hk": 2})])
def test_every_form_takes_every_batch(lens, how, form, monkeypatch):
    """Clusters of a unit and shares of all units differ in time alone."""
    require_gpu_lib()
    monkeypatch.setattr(kv4, "_shape", lambda *a: form)
    s = batch(len(lens), lens, device="cuda", **how)
    want = exact(s)
    one = run(s, want)
    assert torch.equal(one, run(s, want)), "the same inputs, the same bits"


@pytest.mark.parametrize("hq,hk,d,q_len", [(32, 8, 128, 1), (16, 8, 64, 1), (32, 8, 128, 4), (16, 2, 256, 2), (8, 8, 128, 1), (16, 1, 128, 1), (40, 8, 128, 1), (14, 2, 64, 2),
                                           (24, 1, 128, 3)])
@pytest.mark.parametrize("rows,length", [(1, 9001), (3, 2500), (17, 777), (70, 140)])
def test_attention_of_longer_batches(hq, hk, d, q_len, rows, length):
    require_gpu_lib()
    s = batch(rows, [max(q_len, length - (37 * i) % length) for i in range(rows)], hq=hq, hk=hk, d=d, q_len=q_len, device="cuda")
    run(s, exact(s), max_len=length)


def test_attention_of_large_and_small_values():
    """Rows of q from 2^-60 to 2^60, scores that differ by thousands, scales of V from 2^-30 to 2^30, all of V near 2^-100 and 2^100."""
    require_gpu_lib()
    s = batch(3, [700, 640, 62, 900], device="cuda")
    s.q *= torch.exp2(torch.linspace(-60, 4, s.q.shape[0] * s.q.shape[1], device="cuda").round()).view(*s.q.shape[:2], 1).to(torch.bfloat16)
    run(s, exact(s))
    s = batch(4, [700, 640, 62, 900], spread=2.0 ** 30, device="cuda")
    s.scale *= 2.0 ** -28
    run(s, exact(s))
    s = batch(5, [700, 640, 62, 900], q_std=2.0 ** 60, device="cuda")
    s.scale *= 2.0 ** -60
    run(s, exact(s))
    for e in (-100, 100):
        s = batch(6, [700, 64], device="cuda")
        both = s.kv.data[:, :, 17 * 128 :].contiguous().view(torch.bfloat16)
        s.kv.data[:, :, 17 * 128 :] = (both.float() * 2.0 ** e).to(torch.bfloat16).view(torch.uint8)
        run(s, exact(s))


def test_attention_with_a_negative_and_a_zero_scale():
    require_gpu_lib()
    for scale in (-0.2, 0.0):
        s = batch(3, [700, 64, 1], device="cuda")
        s.scale = scale
        run(s, exact(s))


def test_a_run_as_it_is_used():
    """Two prompts by chunks (written, read back, attended), then decode steps: against one attention in 64 bits over what the pages hold."""
    require_gpu_lib()
    from mfq_b200.engine.kv_cache import PagedKV4Cache
    hq, hk, d, chunk, lens, steps = 8, 2, 128, 70, [150, 200], 20
    cache = PagedKV4Cache(layers=1, kv_heads=hk, head_dim=d, num_pages=40, max_seqs=2, max_pages_per_seq=16, device="cuda")
    kv, scale = cache.layer(0), 1 / math.sqrt(d)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    qkv = [torch.randn(n + steps, hq + 2 * hk, d, device="cuda").to(torch.bfloat16) for n in lens]
    got = [torch.zeros(n + steps, hq, d, device="cuda", dtype=torch.bfloat16) for n in lens]
    for i, n in enumerate(lens):
        for a in range(0, n, chunk):
            b = min(n, a + chunk)
            cache.assign(i, i, b)
            rows = qkv[i][a:b]
            ops.kv4_write(rows[:, hq : hq + hk], rows[:, hq + hk :], cache.slots(i, a, b - a).cuda(), kv)
            k, v = ops.kv4_gather(kv, cache.block_table[i : i + 1], i32([0, b]), b)
            got[i][a:b] = ops.kernels.attn_prefill_bf16(rows[:, :hq].contiguous(), k, v, scale)
    pos = list(lens)
    for _ in range(steps):
        rows = torch.stack([qkv[i][p] for i, p in enumerate(pos)])
        for i in range(2):
            cache.assign(i, i, pos[i] + 1)
        ops.kv4_write(rows[:, hq : hq + hk], rows[:, hq + hk :], torch.cat([cache.slots(i, p, 1) for i, p in enumerate(pos)]).cuda(), kv)
        pos = [p + 1 for p in pos]
        o = ops.paged_attn_decode_kv4(rows[:, :hq].contiguous(), kv, cache.block_table, i32(pos), sm_scale=scale, max_len=256)
        for i in range(2):
            got[i][pos[i] - 1] = o[i]
    check_status()
    held = values(kv.data)
    for i, n in enumerate(pos):
        ids = torch.tensor(cache.allocator.owned[i])
        k, v = (x[ids].transpose(0, 1).flatten(1, 2)[:, :n] for x in held)
        q = qkv[i][:, :hq].cpu().double().view(n, hk, hq // hk, d)
        p = torch.einsum("qhgd,hkd->hgqk", q, k) * scale
        p = torch.softmax(p.masked_fill(torch.arange(n) > torch.arange(n)[:, None], -math.inf), -1)
        want, weight = torch.einsum("hgqk,hkd->qhgd", p, v), torch.einsum("hgqk,hkd->qhgd", p, v.abs())
        # a chunk's keys and values are rounded to bf16 on the way (2^-8 each; a key's moves a score by at most that times the largest |q| |k|), p to bf16, the result to bf16
        size = (q.abs().amax(0).max() * k.abs().sum(-1).max() * scale).item()
        off = (got[i].cpu().double().view(n, hk, hq // hk, d) - want).abs() / weight
        assert off[lens[i] :].max() < 2.0 ** -8 + 2.0 ** -9, "decode steps read what the pages hold"
        assert off.max() < 3 * 2.0 ** -8 + 2 * 2.0 ** -8 * size / math.sqrt(d)


def test_another_stream_and_a_graph_whose_batch_changes():
    require_gpu_lib()
    s, other = batch(7, [400, 350, 0, 17], device="cuda"), batch(7, [17, 0, 400, 350], device="cuda")
    want = exact(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = call(ops, s)
    torch.cuda.current_stream().wait_stream(side)
    assert_attends(s, out, want)
    k = torch.randn(4, 2, 128, device="cuda").to(torch.bfloat16)
    slots = torch.tensor([-1, -1, -1, -1], dtype=torch.int32, device="cuda")
    starts, first = torch.tensor([0, 4, 4, 4, 4], dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    k_out, v_out = torch.zeros_like(k), torch.zeros_like(k)

    def step():
        ops.kv4_write(k, k, slots, s.kv)
        ops.kv4_gather(s.kv, s.table, starts, first=first, k_out=k_out, v_out=v_out)
        call(ops, s, out=out, max_len=400)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    s.kv.data.copy_(other.kv.data)
    for name in ("q", "table", "seq_lens"):
        getattr(s, name).copy_(getattr(other, name))
    s.lens = other.lens
    slots.copy_(other.table[2, :1] * 16 + torch.arange(4, device="cuda"))  # the first tokens of the third sequence
    starts.copy_(torch.tensor([0, 0, 0, 3, 4], device="cuda"))
    graph.replay()
    check_status()
    assert_attends(s, out, exact(s))
    assert not torch.equal(s.kv.data, other.kv.data)
    held = values(s.kv.data[s.table[2, :1].long()])[0, 0].transpose(0, 1).float().to(torch.bfloat16)
    assert torch.equal(k_out[:3].cpu(), held[:3])


def test_calls_and_graphs_at_once():
    """Calls on two streams keep their sums apart, and so do two graphs."""
    require_gpu_lib()
    cases = [batch(i, [5000, 4100, 300], hq=32, hk=8, device="cuda") for i in (1, 2)]
    wants = [exact(s) for s in cases]
    streams, graphs, outs = [torch.cuda.Stream() for _ in cases], [], [[], []]
    torch.cuda.synchronize()
    for _ in range(8):
        for i, s in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                outs[i].append(call(ops, s, max_len=5000))
    torch.cuda.synchronize()
    captured = []
    for s in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            captured.append(call(ops, s, max_len=5000))
    for _ in range(8):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    check_status()
    for s, want, got, last in zip(cases, wants, outs, captured):
        assert_attends(s, got[0], want)
        assert all(torch.equal(got[0], x) for x in got + [last])


def test_pages_and_rows_behind_4_gigabytes():
    require_gpu_lib()
    s = batch(5, [430, 410, 50], hq=32, hk=8)
    want = exact(s)
    used, most = s.kv.data.shape[0], 2 ** 32 // (8 * 18 * 128) + 1000
    small = s.kv.data.cuda()
    s.kv = LayerKV4(torch.zeros((most, *small.shape[1:]), dtype=torch.uint8, device="cuda"), 128, 16)
    s.kv.data[most - used :].copy_(small)
    for name in ("q", "table", "seq_lens"):
        setattr(s, name, getattr(s, name).cuda())
    s.table += most - used
    run(s, want)
    k = torch.randn(20, 8, 128, device="cuda")
    slots = torch.arange(20, dtype=torch.int32, device="cuda") + 16 * (most - 2) + 7
    few = LayerKV4(s.kv.data[-4:].clone(), 128, 16)
    ops.kv4_write(k, k, slots, s.kv)
    ops.kv4_write(k, k, slots - 16 * (most - 4), few)
    assert torch.equal(s.kv.data[-4:], few.data)
    apart = torch.zeros(2 ** 31 + 2 ** 28, dtype=torch.bfloat16, device="cuda").as_strided((540, 8, 128), (1 << 22, 128, 1))
    starts = torch.tensor([0, 430, 540], dtype=torch.int32, device="cuda")
    k_out, v_out = ops.kv4_gather(s.kv, s.table[:2], starts, k_out=apart, v_out=torch.zeros_like(apart, memory_format=torch.contiguous_format))
    a, b = ops.kv4_gather(s.kv, s.table[:2], starts, 540)
    check_status()
    assert torch.equal(k_out, a) and torch.equal(v_out, b)
    ops.kv4_write(apart[500:], apart[500:], torch.arange(40, dtype=torch.int32, device="cuda"), s.kv)
    ops.kv4_write(a[500:], a[500:], torch.arange(48, 88, dtype=torch.int32, device="cuda"), s.kv)
    check_status()
    assert torch.equal(s.kv.data[:2], s.kv.data[3:5])


def test_what_is_out_of_range_is_reported_and_left_out():
    require_gpu_lib()
    s = batch(2, [64, 90], device="cuda")
    table, pages = s.table.clone(), s.kv.data.shape[0]
    for bad in (pages, -1, 2 ** 30):
        s.table[1, 2] = bad
        call(ops, s)
        with pytest.raises(RuntimeError, match="status code 5"):
            check_status()
        out = [torch.full((90, 2, 128), 7.0, device="cuda") for _ in range(2)]
        ops.kv4_gather(s.kv, s.table[1:].contiguous(), torch.tensor([0, 90], dtype=torch.int32, device="cuda"), k_out=out[0], v_out=out[1])
        with pytest.raises(RuntimeError, match="status code 5"):
            check_status()
        for x in out:
            assert (x[32:48] == 7).all() and (x[:32] != 7).any(-1).all() and (x[48:] != 7).any(-1).all()
    s.table.copy_(table)
    short = s.table[:, :2].contiguous()
    for first in (-3, 2 ** 31 - 9, 20):
        out = [torch.full((20, 2, 128), 7.0, device="cuda") for _ in range(2)]
        ops.kv4_gather(s.kv, short, torch.tensor([0, 20, 20], dtype=torch.int32, device="cuda"), first=torch.tensor([first, 0], dtype=torch.int32, device="cuda"),
                       k_out=out[0], v_out=out[1])
        with pytest.raises(RuntimeError, match="status code 5"):
            check_status()
        there = [0 <= first + i < 32 for i in range(20)]
        for x in out:
            assert [bool((row != 7).any()) for row in x] == there
    before = s.kv.data.clone()
    k = torch.randn(3, 2, 128, device="cuda")
    ops.kv4_write(k, k, torch.tensor([pages * 16, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32, device="cuda"), s.kv)
    with pytest.raises(RuntimeError, match="status code 5"):
        check_status()
    assert torch.equal(before, s.kv.data)


def test_lengths_of_nearly_2_to_the_31_see_all_of_their_table():
    require_gpu_lib()
    s = batch(3, [96, 96, 96], device="cuda")
    want = exact(s)
    s.table = s.table[:, :6].contiguous()
    s.seq_lens.fill_(2 ** 31 - 1)
    run(s, want)
    run(s, want, max_len=2 ** 31 - 1)
    s.seq_lens.fill_(-5)
    out = torch.full_like(s.q, 3.0)
    call(ops, s, out=out)
    assert (out == 0).all()


def test_a_group_of_nan_is_seen_by_those_who_see_it():
    """A NaN among a sequence's own values makes its head's rows NaN from there on, and nobody else's."""
    require_gpu_lib()
    s = batch(2, [64, 90], hq=4, hk=2, device="cuda")
    page = int(s.table[1, 1])
    clean = call(ops, s)
    assert torch.isfinite(clean).all()
    k = torch.randn(1, 2, 128, device="cuda")
    k[0, 1, 3] = math.nan
    ops.kv4_write(k, torch.randn_like(k), torch.tensor([page * 16 + 3], dtype=torch.int32, device="cuda"), s.kv)
    out = call(ops, s)
    assert torch.equal(out[0], clean[0]) and out[1, 2:].isnan().all() and torch.isfinite(out[1, :2]).all()


@pytest.mark.parametrize("d,hk,dtype", [(64, 3, torch.bfloat16), (128, 2, torch.float32), (256, 2, torch.float16)])
def test_many_tokens_in_runs_of_every_kind(d, hk, dtype):
    """Enough of them that a warp has windows of 8 or 16 tokens: whole pages, parts, single tokens and padding beside one another."""
    require_gpu_lib()
    g = torch.Generator().manual_seed(d)
    pages, parts = 3000, []
    for page in torch.randperm(pages, generator=g).tolist():
        kind = int(torch.randint(0, 6, (1,), generator=g))
        lo = int(torch.randint(0, 16, (1,), generator=g))
        hi = int(torch.randint(lo, 17, (1,), generator=g))
        at = list(range(16 * page, 16 * page + 16))
        parts += [at, at, at[lo:hi], at[hi:] + [-1] * 3 + at[:lo], at[::-1], at[lo : lo + 1]][kind]
    slots = torch.tensor(parts, dtype=torch.int32, device="cuda")
    assert 2 * len(parts) * hk > 148 * 64 * 8
    wide = torch.randn((len(parts), 2 * hk, d), generator=g).mul_(2).to(dtype).cuda()
    kv = empty_pool(pages, hk, d)
    want = write_both(wide[:, :hk], wide[:, hk:], slots, kv)
    assert_bytes(kv.data, want)


@pytest.mark.parametrize("d,hk,dtype", [(64, 3, torch.bfloat16), (128, 2, torch.float32), (256, 2, torch.float16)])
def test_many_sequences_read_back(d, hk, dtype):
    require_gpu_lib()
    g = torch.Generator().manual_seed(d)
    b, width, pages = 1500, 12, 700
    lens = (torch.rand(b, generator=g) * 90).int() * (torch.rand(b, generator=g) < 0.7)
    first = (torch.rand(b, generator=g) * 90).int()
    table = torch.randint(0, pages, (b, width), generator=g, dtype=torch.int32)
    starts = torch.cat([torch.zeros(1, dtype=torch.int32), lens.cumsum(0).int()])
    data, n = pool(d, pages, hk, d), int(starts[-1])
    want = ops.kv4_gather(LayerKV4(data, d, 16), table, starts, n, first=first, dtype=dtype)
    got = ops.kv4_gather(LayerKV4(data.cuda(), d, 16), table.cuda(), starts.cuda(), n, first=first.cuda(), dtype=dtype)
    check_status()
    for x, y in zip(got, want):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("form", [(1, 0), (0, 592)])
def test_more_sequences_than_a_grid_has_rows(form, monkeypatch):
    """70000 sequences of one or two tokens; of one token the output is its value."""
    require_gpu_lib()
    monkeypatch.setattr(kv4, "_shape", lambda *a: form)
    b = 70000
    data = pool(1, b + 1, 1, 64)
    kv = LayerKV4(data.cuda(), 64, 16)
    table = (torch.randperm(b) + 1).int().view(b, 1).cuda()
    lens = torch.ones(b, dtype=torch.int32, device="cuda")
    lens[::7] = 0
    q = torch.randn(b, 4, 64, device="cuda").to(torch.bfloat16)
    out = ops.paged_attn_decode_kv4(q, kv, table, lens, sm_scale=0.1)
    check_status()
    _, v = ops.kv4_gather(kv, table, torch.arange(b + 1, dtype=torch.int32, device="cuda"), b, dtype=torch.float32)
    assert (out[::7] == 0).all()
    some = lens.bool()
    off = (out[some].float() - v[some]).abs() - (2.0 ** -8 * v[some].abs() + 2.0 ** -10 * 15 * 0.36)  # the output's rounding, and p s to fp16 of up to 15 scales
    assert (off <= 0).all()


@pytest.mark.parametrize("hq,hk,d,q_len,dtype", [(64, 1, 128, 3, torch.bfloat16), (128, 2, 64, 2, torch.float16), (48, 1, 256, 2, torch.bfloat16), (8, 8, 128, 40, torch.bfloat16)])
def test_many_query_rows(hq, hk, d, q_len, dtype):
    require_gpu_lib()
    s = batch(4, [100, 30, 700], hq=hq, hk=hk, d=d, q_len=q_len, dtype=dtype, device="cuda")
    run(s, exact(s))


@pytest.mark.parametrize("hq,d", [(2, 128), (4, 128), (8, 128), (2, 64), (4, 256)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_a_later_token_of_a_window_is_not_seen_through_its_nan(what, hq, d):
    require_gpu_lib()
    s = batch(2, [64, 90, 33], hq=hq, hk=2, d=d, q_len=4, device="cuda")
    clean = call(ops, s)
    assert torch.isfinite(clean).all()
    k, v = torch.randn(1, 2, d, device="cuda"), torch.randn(1, 2, d, device="cuda")
    (k if what == "k" else v)[:] = math.nan
    for n in (64, 90, 33):
        row, last = (64, 90, 33).index(n), n - 1
        ops.kv4_write(k, v, (s.table[row, last // 16 : last // 16 + 1] * 16 + last % 16).int(), s.kv)
    out = call(ops, s).view(3, 4, hq, d)
    assert torch.equal(out[:, :3], clean.view(3, 4, hq, d)[:, :3]) and out[:, 3].isnan().all()


def test_the_self_check():
    require_gpu_lib()
    from mfq_b200 import diagnostics
    report = diagnostics.run(["kv4-cache"])
    assert report["ok"] and report["checks"]["kv4-cache"]["same_bits"], report
