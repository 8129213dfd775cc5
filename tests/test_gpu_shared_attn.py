"""The kernels of ``ops.paged_attn_decode_shared`` against the softmax in 64 bits."""

import pytest
import torch

from mfq_b200 import ops
from mfq_b200.ops import shared_attn
from gpu_common import assert_close, check_status, require_gpu_lib
from shared_attn_cases import BATCHES, assert_attends, batch, call, exact

pytestmark = pytest.mark.gpu


def run(s, want, **how):
    out = torch.full_like(s.q, 3.0)
    assert call(ops, s, out=out, **how) is out
    check_status()
    assert_attends(s, out, want)
    rest = [r * s.q_len + i for r in range(s.seq_lens.numel()) if r not in s.grouped for i in range(s.q_len)]
    assert (out[rest] == 3).all()
    return out


@pytest.mark.parametrize("groups,how", BATCHES)
def test_against_the_definition(groups, how):
    require_gpu_lib()
    s = batch(len(groups), groups, device="cuda", **how)
    want = exact(s)
    one = run(s, want)
    assert torch.equal(one, run(s, want)), "the same inputs, the same bits"
    run(s, want, max_group=1, max_prefix=10 ** 6, max_tail=10 ** 6)  # wrong in each direction: only slower
    run(s, want, max_group=max(len(n) for _, n in groups), max_prefix=max(p for p, _ in groups), max_tail=0)


FORMS = [(16, 0, 1), (16, 0, 8), (8, 1, 2), (8, 5, 1), (16, 1, 1), (16, 7, 4), (128, 1, 1), (128, 3, 2), (128, 32, 8), (256, 1, 4), (256, 5, 1), (256, 64, 3)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("groups,how", [x for x in BATCHES if x[1].get("d", 128) <= 128])
def test_every_form_takes_every_batch(groups, how, form, monkeypatch):
    """The forms (query rows of a prefix CTA, splits of a prefix, CTAs of a tail) differ in time alone."""
    require_gpu_lib()
    monkeypatch.setattr(shared_attn, "_shape", lambda *a: form)
    s = batch(len(groups), groups, device="cuda", **how)
    want = exact(s)
    one = run(s, want)
    assert torch.equal(one, run(s, want)), "the same inputs, the same bits"


@pytest.mark.parametrize("form", FORMS)
def test_every_form_with_large_and_small_rows(form, monkeypatch):
    """Rows of q from 2^-60 to 2^4, scores that differ by thousands, multipliers of V from 2^-30 to 2^30."""
    require_gpu_lib()
    monkeypatch.setattr(shared_attn, "_shape", lambda *a: form)
    s = batch(3, [(600, [700, 640, 620, 900, 610, 601])], device="cuda")
    s.q *= torch.exp2(torch.linspace(-60, 4, s.q.shape[0] * s.q.shape[1], device="cuda").round()).view(*s.q.shape[:2], 1).to(torch.bfloat16)
    run(s, exact(s))
    s = batch(4, [(1200, [1300, 1240, 1220, 1500])], v_spread=2.0 ** 30, device="cuda")
    run(s, exact(s))
    s = batch(5, [(600, [700, 640, 620, 900])], q_std=2.0 ** 60, device="cuda")
    s.scale *= 2.0 ** -60
    run(s, exact(s))


@pytest.mark.parametrize("hq,hk,d,q_len", [(32, 8, 128, 1), (16, 8, 64, 1), (32, 8, 128, 4), (16, 2, 256, 2), (8, 8, 128, 1), (16, 1, 128, 1), (40, 8, 128, 1), (14, 2, 64, 2)])
@pytest.mark.parametrize("rows,prefix", [(2, 4000), (5, 1111), (17, 777), (33, 2500), (64, 400)])
def test_one_long_prefix(hq, hk, d, q_len, rows, prefix):
    require_gpu_lib()
    s = batch(rows, [(prefix, [prefix + q_len + (37 * i) % 200 for i in range(rows)])], hq=hq, hk=hk, d=d, q_len=q_len, device="cuda")
    run(s, exact(s), max_group=rows, max_prefix=prefix, max_tail=220)


def test_values_with_large_and_small_rows():
    """Rows of q from 2^-60 to 2^60, scores that differ by thousands, multipliers of V from 2^-30 to 2^30."""
    require_gpu_lib()
    s = batch(3, [(600, [700, 640, 620, 900])], device="cuda")
    s.q *= torch.exp2(torch.linspace(-60, 4, s.q.shape[0] * s.q.shape[1], device="cuda").round()).view(*s.q.shape[:2], 1).to(torch.bfloat16)
    run(s, exact(s))
    s = batch(4, [(600, [700, 640, 620, 900])], v_spread=2.0 ** 30, device="cuda")
    run(s, exact(s))
    s = batch(5, [(600, [700, 640, 620, 900])], q_std=2.0 ** 60, device="cuda")
    s.scale *= 2.0 ** -60
    run(s, exact(s))


def test_another_stream_and_a_graph_whose_groups_change():
    require_gpu_lib()
    s = batch(7, [(320, [400, 350, 330]), (160, [200, 161])], device="cuda")
    other = batch(8, [(160, [170]), (320, [400, 350, 330, 360])], device="cuda")
    want, want_other = exact(s), exact(other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = call(ops, s)
    torch.cuda.current_stream().wait_stream(side)
    assert_attends(s, out, want)
    pages, width = max(s.kv.k.shape[0], other.kv.k.shape[0]), max(s.table.shape[1], other.table.shape[1])

    def grown(t, n, dim=0):
        shape = list(t.shape)
        shape[dim] = n
        out = torch.zeros(shape, dtype=t.dtype, device=t.device)
        out.narrow(dim, 0, t.shape[dim]).copy_(t)
        return out

    for x in (s, other):
        for name in ("k", "v", "k_scale", "v_scale"):
            setattr(x.kv, name, grown(getattr(x.kv, name), pages))
        x.table = grown(x.table, width, 1)
    out = torch.empty_like(s.q)
    call(ops, s, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(ops, s, out=out)
    for name in ("q", "table", "seq_lens", "starts", "prefixes", "members"):
        getattr(s, name).copy_(getattr(other, name))
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(s.kv, name).copy_(getattr(other.kv, name))
    graph.replay()
    check_status()
    assert_attends(other, out, want_other)


def test_two_calls_at_once():
    """Calls on two streams keep their sums apart."""
    require_gpu_lib()
    cases = [batch(i, [(2000, [2100] * 12)], hq=32, hk=8, device="cuda") for i in (1, 2)]
    wants = [exact(s) for s in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, s in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                outs[i].append(call(ops, s))
    torch.cuda.synchronize()
    for s, want, got in zip(cases, wants, outs):
        assert_attends(s, got[0], want)
        assert all(torch.equal(got[0], x) for x in got)


def test_two_graphs_replayed_at_once():
    """Every captured call has partials of its own."""
    require_gpu_lib()
    cases = [batch(i, [(2000, [2100] * 12)], hq=32, hk=8, device="cuda") for i in (3, 4)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for s in cases:
        call(ops, s)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(ops, s))
    for _ in range(8):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    check_status()
    for s, out in zip(cases, outs):
        assert_attends(s, out, exact(s))


@pytest.mark.parametrize("form", [(16, 0, 2), (16, 3, 1), (128, 2, 1), (256, 2, 1)])
def test_pages_behind_4_gigabytes(form, monkeypatch):
    require_gpu_lib()
    monkeypatch.setattr(shared_attn, "_shape", lambda *a: form)
    s = batch(5, [(400, [430, 410, 500, 401, 460])], hq=32, hk=8)
    want = exact(s)
    used, most = s.kv.k.shape[0], 2 ** 32 // (8 * 16 * 128) + 1000
    for name in ("k", "v", "k_scale", "v_scale"):
        small = getattr(s.kv, name).cuda()
        large = torch.zeros((most, *small.shape[1:]), dtype=small.dtype, device="cuda")
        large[most - used :].copy_(small)
        setattr(s.kv, name, large)
    for name in ("q", "table", "seq_lens", "starts", "prefixes", "members"):
        setattr(s, name, getattr(s, name).cuda())
    s.table += most - used
    run(s, want)


def test_a_page_outside_the_pool_is_reported():
    require_gpu_lib()
    s = batch(2, [(64, [80, 90])], device="cuda")
    s.table[s.members[0].long(), 2] = s.kv.k.shape[0]
    call(ops, s)
    with pytest.raises(RuntimeError, match="status code 5"):
        check_status()


@pytest.mark.parametrize("form", [(16, 0, 1), (8, 1, 2), (128, 1, 1), (256, 1, 1)])
def test_a_member_that_is_no_row_is_reported(form, monkeypatch):
    """Kernels leave such a place out (and read nothing through it)."""
    require_gpu_lib()
    monkeypatch.setattr(shared_attn, "_shape", lambda *a: form)
    for bad in (-1, 3):
        s = batch(2, [(64, [80, 90, 70])], device="cuda")
        s.members[1] = bad
        call(ops, s)
        with pytest.raises(RuntimeError, match="status code 5"):
            check_status()


def test_equals_the_attention_of_unshared_rows():
    require_gpu_lib()
    s = batch(9, [(1000, [1100 + 9 * i for i in range(20)])], hq=32, hk=8, device="cuda")
    s.table.clamp_(max=s.kv.k.shape[0] - 1)
    for t in (s.kv.k, s.kv.v):
        u = t.view(torch.uint8)
        u[(u & 0x7F) == 0x7F] = 0
    for t in (s.kv.k_scale, s.kv.v_scale):
        t.nan_to_num_(0.0)
    want = ops.paged_attn_decode(s.q, s.kv, s.table, s.seq_lens, sm_scale=s.scale, splits=4)
    assert_close(call(ops, s), want, rel=1e-2, what="shared against unshared")


def test_lengths_of_nearly_2_to_the_31_see_all_of_their_table():
    """A length behind the table's end sees what the table has, whatever is added to it on the way."""
    require_gpu_lib()
    s = batch(3, [(64, [96, 96, 96])], device="cuda")
    want = exact(s)
    s.table = s.table[:, :6].contiguous()
    s.seq_lens.fill_(2 ** 31 - 1)
    out = call(ops, s)
    check_status()
    assert_attends(s, out, want)
