"""``ops.paged_attn_decode_shared`` on CPU tensors, and what it refuses."""

import pytest
import torch

from mfq_b200 import ops
from shared_attn_cases import BATCHES, assert_attends, batch, call, exact


@pytest.mark.parametrize("groups,how", BATCHES)
def test_against_the_definition(groups, how):
    s = batch(len(groups), groups, **how)
    out = torch.full_like(s.q, 3.0)
    assert call(ops, s, out=out) is out
    assert_attends(s, out, exact(s))
    rest = [r * s.q_len + i for r in range(s.seq_lens.numel()) if r not in s.grouped for i in range(s.q_len)]
    assert (out[rest] == 3).all()


def test_refusals():
    s = batch(1, [(16, [20, 30])])
    long = lambda t: t.long()  # noqa: E731
    for name, make in (("q", lambda t: t.float()), ("q", lambda t: t[:, :7]), ("q", lambda t: t[:, :, :96].contiguous()), ("q", lambda t: t.transpose(0, 1)),
                       ("table", long), ("table", lambda t: t[:1]), ("table", lambda t: t[:, ::2]), ("seq_lens", long), ("seq_lens", lambda t: t[:1]), ("starts", long),
                       ("starts", lambda t: t[:1]), ("prefixes", long), ("members", long), ("members", lambda t: t[:1])):
        held = getattr(s, name)
        setattr(s, name, make(held))
        with pytest.raises(ValueError):
            call(ops, s)
        setattr(s, name, held)
    with pytest.raises(ValueError, match="16 query rows"):
        call(ops, batch(1, [(16, [20, 30])], hq=24, hk=1))
    s.q_len = 3
    with pytest.raises(ValueError):
        call(ops, s)
    s.q_len = 1
    with pytest.raises(ValueError, match="out"):
        call(ops, s, out=torch.zeros_like(s.q, dtype=torch.float32))
    s.kv.page_size = 32
    with pytest.raises(ValueError, match="16 tokens"):
        call(ops, s)
    s.kv.page_size = 16
    s.starts, s.prefixes = torch.tensor([0, 1, 2, 2], dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="3 groups of 2 rows"):
        call(ops, s)


def test_no_groups():
    s = batch(1, [(16, [20, 30])])
    s.starts, s.prefixes = s.starts[:1].contiguous(), s.prefixes[:0].contiguous()
    out = torch.full_like(s.q, 3.0)
    assert (call(ops, s, out=out) == 3).all()


@pytest.mark.parametrize("name", ["q", "out", "k", "v", "k_scale", "v_scale"])
def test_tensors_that_begin_between_16_bytes_are_refused(name):
    """The kernels read and write them 16 bytes at a time; a slice of a buffer may begin anywhere."""
    s = batch(1, [(16, [20, 30])])
    out = torch.zeros_like(s.q)

    def shifted(t):
        buffer = torch.zeros(t.numel() + 16, dtype=t.dtype)
        part = buffer[4 // t.element_size():][:t.numel()].view(t.shape)
        assert part.data_ptr() % 16 == 4
        return part.copy_(t)

    if name == "q":
        s.q = shifted(s.q)
    elif name != "out":
        setattr(s.kv, name, shifted(getattr(s.kv, name)))
    with pytest.raises(ValueError, match="16 bytes"):
        call(ops, s, out=shifted(out) if name == "out" else out)


@pytest.mark.parametrize("name", ["k_scale", "v_scale"])
@pytest.mark.parametrize("make", [lambda t: t[:-1], lambda t: t.double(), lambda t: t[:, :, :8].contiguous()])
def test_multipliers_of_another_pool_are_refused(name, make):
    s = batch(1, [(16, [20, 30])])
    setattr(s.kv, name, make(getattr(s.kv, name)))
    with pytest.raises(ValueError, match="multipliers"):
        call(ops, s)


def test_chosen_forms_are_forms_that_the_kernels_have():
    """Whatever the sizes: tiles, partials of a query row and CTAs of a cluster within the limits of the C entry."""
    from mfq_b200.ops.shared_attn import _shape
    g = torch.Generator().manual_seed(1)
    pick = lambda *x: x[int(torch.randint(0, len(x), (1,), generator=g))]  # noqa: E731
    for _ in range(1500):
        b, per_seq, hk, d = pick(1, 2, 5, 31, 64, 700, 65535), pick(1, 2, 4, 7, 8, 9, 16), pick(1, 2, 8, 40), pick(64, 128, 256)
        groups, whole, tail = min(b, pick(1, 2, 9, 300)), pick(0, 1, 3, 4, 40, 1000, 70000), pick(0, 1, 2, 30, 900, 70000)
        tile, splits, ranks = _shape(b, per_seq, hk, d, groups, pick(1, max(1, b // groups), b), whole, tail)
        assert tile in (8, 16, 128, 256) and ranks in (1, 2, 4, 8) and 0 <= splits * (2 if tile == 128 else 1) <= 64
        assert splits == 0 or (d <= 128 and splits <= max(1, whole)) and (tile != 8 or per_seq <= 8)


def test_pools_without_heads_and_tables_without_pages_are_refused():
    s = batch(1, [(16, [20, 30])])
    table = s.table
    s.table = table[:, :0].contiguous()
    with pytest.raises(ValueError, match="pages"):
        call(ops, s)
    s.table = table
    for name in ("k", "v", "k_scale", "v_scale"):
        setattr(s.kv, name, getattr(s.kv, name)[:, :0].contiguous())
    with pytest.raises(ValueError, match="KV heads"):
        call(ops, s)


def test_batches_of_more_sequences_than_a_grid_are_refused():
    n = 65536
    s = batch(1, [(16, [20])], hq=1, hk=1, d=64)
    i32 = torch.int32
    s.q, s.table, s.seq_lens = s.q.expand(n, 1, 64).contiguous(), s.table.expand(n, -1).contiguous(), s.seq_lens.expand(n).contiguous()
    s.starts, s.members = torch.tensor([0, n], dtype=i32), None
    with pytest.raises(ValueError, match="65535"):
        call(ops, s)
