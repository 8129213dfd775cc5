"""The cache held in 4 bits on CPU tensors: its format against exact arithmetic, the operators against the definition, and what they refuse."""

import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from mfq_b200 import ops
from mfq_b200.engine.kv_cache import LayerKV4, PagedKV4Cache, PagedKVCache
from mfq_b200.ops import reference
from kv4_cases import BATCHES, assert_attends, batch, call, exact, pool, unpack, values


def groups():
    """``[n, 64]`` fp32: ordinary groups and those where the choice of scale or code is close."""
    g = torch.Generator().manual_seed(5)
    rows = [torch.randn(64, generator=g) * 10.0 ** e for e in (-38, -20, -3, 0, 0, 2, 20, 36)]
    rows += [torch.randn(64, generator=g).to(torch.bfloat16).float() for _ in range(6)]
    rows += [torch.zeros(64), torch.full((64,), 3.7), torch.full((64,), -1.0), torch.cat([torch.zeros(63), torch.tensor([1e-44])])]
    ties = torch.arange(64) % 31 * 0.5 * 0.75  # halves of a step of 0.75 between 0 and 15 steps
    ties[62], ties[63] = 0.0, 15 * 0.75
    rows += [ties, ties - 4.0, -ties, torch.nextafter(ties, torch.tensor(9.0)), torch.nextafter(ties, torch.tensor(-9.0)).clamp_(min=0)]
    rows += [torch.cat([torch.tensor([-15.0, 0.0]), torch.linspace(-1e-9, 1e-9, 62)]), torch.cat([torch.tensor([-1.5, 13.5]), torch.linspace(-3e-8, 3e-8, 62)])]
    rows += [torch.cat([torch.tensor([2.0 ** 126, -(2.0 ** 126)]), torch.randn(62, generator=g)]), 100 + torch.randn(64, generator=g) * 1e-3]
    return torch.stack(rows)


def _bf16_next(x, up):
    t = torch.tensor(x).to(torch.bfloat16)
    return Fraction(float(torch.nextafter(t, torch.full_like(t, math.inf if up else -math.inf))))


def test_scale_minimum_and_codes_are_what_the_format_says():
    x = groups()
    codes, s, m = reference.kv4_quantise(x[:, None])
    for row, c, scale, least in zip(x, codes[:, 0], s[:, 0, 0].tolist(), m[:, 0, 0].tolist()):
        v = [Fraction(float(y)) for y in row]
        fs, fm = Fraction(scale), Fraction(least)
        assert float(torch.tensor(scale).to(torch.bfloat16)) == scale and float(torch.tensor(least).to(torch.bfloat16)) == least
        assert fm <= min(v) < _bf16_next(least, True)
        assert 15 * fs >= max(v) - fm and (fs == 0 or 15 * _bf16_next(scale, False) < max(v) - fm)
        for y, code in zip(v, c.tolist()):
            if fs == 0:
                assert code == 0
                continue
            q = (y - fm) / fs
            assert code == round(q) and 0 <= code <= 15  # of fractions: to the nearest, ties to even
            assert abs(y - (fm + code * fs)) <= fs / 2


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 1.5 * 2.0 ** 126, -3e38])
def test_a_group_with_a_value_that_is_none_stands_for_nan(bad):
    x = torch.randn(3, 2, 128)
    x[1, 0, 70] = bad
    kv = LayerKV4(torch.zeros((2, 2, 18 * 128), dtype=torch.uint8), 128, 16)
    ops.kv4_write(x, x, torch.tensor([16, 17, 31], dtype=torch.int32), kv)
    k, v = ops.kv4_gather(kv, torch.tensor([[1]], dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32), 2, dtype=torch.float32)
    for y in (k, v):
        assert y[1, 0, 64:].isnan().all() and y[1, 0, :64].isfinite().all() and y[0].isfinite().all() and y[1, 1].isfinite().all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_layout_of_a_record(d):
    """Every code and parameter has its place, a byte has the codes of one token alone, and together they are the whole record."""
    kv = LayerKV4(torch.full((3, 2, 18 * d), 255, dtype=torch.uint8), d, 16)
    k, v = torch.randn(16, 2, d), torch.randn(16, 2, d)
    slots = torch.randperm(16).int() + 16
    touched = torch.zeros((2, 18 * d), dtype=torch.int32)
    for i in range(16):
        before = kv.data.clone()
        kv.data[1] = 0x55
        one = kv.data.clone()
        ops.kv4_write(k[i : i + 1], v[i : i + 1], slots[i : i + 1], kv)
        a = kv.data[1] != one[1]
        one[1] = 0xAA
        kv.data[1] = 0xAA
        ops.kv4_write(k[i : i + 1], v[i : i + 1], slots[i : i + 1], kv)
        touched += a | (kv.data[1] != 0xAA)
        kv.data.copy_(before)
        ops.kv4_write(k[i : i + 1], v[i : i + 1], slots[i : i + 1], kv)
    assert (touched == 1).all()
    assert (kv.data[[0, 2]] == 255).all()
    held = values(kv.data)[:, 1].transpose(1, 2)[:, slots.long() - 16]  # [2, token, head, D]
    _, s, _ = unpack(kv.data)
    step = s[:, 1].transpose(1, 2)[:, slots.long() - 16].repeat_interleave(64, -1)
    for x, y, e in ((k, held[0], step[0]), (v, held[1], step[1])):
        assert ((x.double() - y).abs() <= e / 2 * (1 + 1e-12)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,hk", [(64, 3), (128, 2), (256, 1)])
def test_written_and_read_back(dtype, d, hk):
    lens, first = [0, 5, 33, 16, 1], [3, 0, 17, 16, 31]
    starts = [2]
    for n in lens:
        starts.append(starts[-1] + n)
    table = torch.randperm(24)[:20].view(5, 4).int()
    kv = LayerKV4(torch.full((24, hk, 18 * d), 255, dtype=torch.uint8), d, 16)
    wide = torch.randn(starts[-1] - 2, 2 * hk, d).to(dtype)
    slots = torch.cat([torch.stack([table[i, p // 16] * 16 + p % 16 for p in range(f, f + n)]) if n else torch.zeros(0, dtype=torch.int32)
                       for i, (f, n) in enumerate(zip(first, lens))]).int()
    ops.kv4_write(wide[:, :hk], wide[:, hk:], slots, kv)
    k_out, v_out = torch.full((starts[-1] + 3, hk, d), 7.0, dtype=dtype), torch.full((hk, starts[-1] + 3, d), 7.0, dtype=dtype).transpose(0, 1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    ops.kv4_gather(kv, table, i32(starts), first=i32(first), k_out=k_out, v_out=v_out)
    mine = slice(2, starts[-1])
    held = values(kv.data)
    for e, (x, y) in enumerate(((wide[:, :hk], k_out), (wide[:, hk:], v_out))):
        want = held[e].transpose(1, 2)[slots.long() // 16, slots.long() % 16].float()  # the fp32 sum, then the type: as it is computed
        assert torch.equal(y[mine], want.to(dtype))
        assert (y[:2] == 7).all() and (y[starts[-1] :] == 7).all()
        assert (x.float() - want).abs().max() <= x.float().abs().max() / 15 * 1.1


@pytest.mark.parametrize("lens,how", BATCHES)
def test_attention_against_the_definition(lens, how):
    s = batch(len(lens), lens, **how)
    out = torch.full_like(s.q, 3.0)
    assert call(ops, s, out=out) is out
    assert_attends(s, out, exact(s))


def test_lengths_behind_the_table_see_what_it_has():
    s = batch(3, [96, 96])
    want = exact(s)
    s.table = s.table[:, :6].contiguous()
    s.seq_lens.fill_(2 ** 31 - 1)
    assert_attends(s, call(ops, s), want)


def test_refused_writes():
    kv = LayerKV4(torch.zeros((2, 2, 18 * 64), dtype=torch.uint8), 64, 16)
    k, slots = torch.randn(4, 2, 64), torch.arange(4, dtype=torch.int32)
    ops.kv4_write(k, k, slots, kv)
    wide = torch.randn(4, 2, 80)
    odd = torch.randn(4 * 2 * 64 + 3)
    for bad in (k.double(), k[:, :1], k[..., :32], k.transpose(0, 1), torch.randn(4, 64, 2).transpose(1, 2), k[0], wide[..., 1:65], odd[1 : 4 * 2 * 64 + 1].view(4, 2, 64),
                torch.randn(4, 2 * 64 + 2)[:, : 2 * 64].unflatten(1, (2, 64)), torch.randn(4, 2 * 66).unflatten(1, (2, 66))[..., :64]):
        for a, b in ((bad, k), (k, bad)):
            with pytest.raises(ValueError):
                ops.kv4_write(a, b, slots, kv)
    with pytest.raises(ValueError, match="as k is"):
        ops.kv4_write(k, k.to(torch.bfloat16), slots, kv)
    for bad in (slots.long(), slots[:3], slots[None], torch.arange(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="slots"):
            ops.kv4_write(k, k, bad, kv)
    with pytest.raises(ValueError, match="behind the pool"):
        ops.kv4_write(k, k, slots + 30, kv)
    before = kv.data.clone()
    ops.kv4_write(k, k, torch.full((4,), -1, dtype=torch.int32), kv)
    ops.kv4_write(k[:0], k[:0], slots[:0], kv)
    assert torch.equal(before, kv.data)


POOLS = [torch.zeros((2, 2, 18 * 64), dtype=torch.int8), torch.zeros((2, 18 * 64), dtype=torch.uint8), torch.zeros((2, 2, 18 * 96), dtype=torch.uint8),
         torch.zeros((2, 2, 20 * 64), dtype=torch.uint8)[..., : 18 * 64], torch.zeros((0, 2, 18 * 64), dtype=torch.uint8), torch.zeros((2, 0, 18 * 64), dtype=torch.uint8),
         torch.zeros(2 * 2 * 18 * 64 + 1, dtype=torch.uint8)[1:].view(2, 2, 18 * 64)]


@pytest.mark.parametrize("data", POOLS)
def test_refused_pools(data):
    kv, i32 = LayerKV4(data, 64, 16), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="kv"):
        ops.kv4_write(torch.randn(1, 2, 64), torch.randn(1, 2, 64), i32, kv)
    with pytest.raises(ValueError, match="kv"):
        ops.kv4_gather(kv, i32[None], torch.zeros(2, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="kv"):
        ops.paged_attn_decode_kv4(torch.randn(1, 4, 64).to(torch.bfloat16), kv, i32[None], i32, sm_scale=1.0)
    with pytest.raises(ValueError, match="kv"):
        ops.paged_attn_decode_kv4(torch.randn(1, 4, 64).to(torch.bfloat16), LayerKV4(pool(0, 2, 2, 64), 64, 32), i32[None], i32, sm_scale=1.0)


def test_refused_gathers():
    kv = LayerKV4(pool(1, 4, 2, 64), 64, 16)
    table, starts = torch.tensor([[1, 2], [3, 0]], dtype=torch.int32), torch.tensor([0, 20, 25], dtype=torch.int32)
    ops.kv4_gather(kv, table, starts, 25)
    out = lambda *s, t=torch.float32: torch.zeros(s, dtype=t)  # noqa: E731
    good = out(25, 2, 64)
    for how in ({}, {"tokens": -1}, {"tokens": 1 << 31}, {"tokens": 25, "dtype": torch.float64}, {"k_out": good}, {"v_out": good}, {"tokens": 24, "k_out": good, "v_out": good},
                {"k_out": good, "v_out": out(24, 2, 64)}, {"k_out": good, "v_out": out(25, 2, 64, t=torch.bfloat16)}, {"k_out": good, "v_out": out(25, 1, 64).expand(25, 2, 64)},
                {"k_out": out(1, 2, 64).expand(25, 2, 64), "v_out": good}, {"k_out": out(25, 2, 128)[..., ::2], "v_out": good}, {"k_out": out(25, 2, 65)[..., :64], "v_out": good},
                {"k_out": torch.zeros(25 * 64 + 64).as_strided((25, 2, 64), (64, 64, 1)), "v_out": good},
                {"tokens": 25, "first": torch.zeros(2)}, {"tokens": 25, "first": torch.zeros(3, dtype=torch.int32)}):
        with pytest.raises(ValueError):
            ops.kv4_gather(kv, table, starts, **how)
    for bad in (table.long(), table[0], table[:, :0], table.t()):
        with pytest.raises(ValueError):
            ops.kv4_gather(kv, bad, starts, 25)
    for bad in (starts.long(), starts[:2], torch.zeros(4, dtype=torch.int32)):
        with pytest.raises(ValueError, match="starts"):
            ops.kv4_gather(kv, table, bad, 25)
    with pytest.raises(ValueError, match="positions"):
        ops.kv4_gather(kv, table, torch.tensor([0, 33, 40], dtype=torch.int32), 40)
    with pytest.raises(ValueError, match="page"):
        ops.kv4_gather(kv, table + 2, starts, 25)
    k, v = ops.kv4_gather(kv, table[:0], starts[:1], 3)
    assert k.shape == v.shape == (3, 2, 64)
    assert ops.kv4_gather(kv, table, starts, 0)[0].shape == (0, 2, 64)


def test_refused_attention():
    s = batch(1, [20, 30])
    for name, make in (("q", lambda t: t.float()), ("q", lambda t: t[:, :7]), ("q", lambda t: t[:, :, :96].contiguous()), ("q", lambda t: t.transpose(0, 1)), ("q", lambda t: t[:, :0]),
                       ("table", lambda t: t.long()), ("table", lambda t: t[:1]), ("table", lambda t: t[:, ::2]), ("table", lambda t: t[:, :0]), ("seq_lens", lambda t: t.long()),
                       ("seq_lens", lambda t: t[:1])):
        held = getattr(s, name)
        setattr(s, name, make(held))
        with pytest.raises(ValueError):
            call(ops, s)
        setattr(s, name, held)
    for q_len in (3, 0, -1):
        s.q_len = q_len
        with pytest.raises(ValueError):
            call(ops, s)
    s.q_len = 1
    for bad in (torch.zeros_like(s.q, dtype=torch.float32), torch.zeros_like(s.q)[:1], torch.zeros_like(s.q).transpose(1, 2)):
        with pytest.raises(ValueError, match="out"):
            call(ops, s, out=bad)
    flat = torch.zeros(s.q.numel() + 1, dtype=s.q.dtype)
    with pytest.raises(ValueError, match="16 bytes"):
        call(ops, s, out=flat[1:].view(s.q.shape))
    s.table[0, 1] = s.kv.data.shape[0]
    with pytest.raises(ValueError, match="page"):
        call(ops, s)
    s = batch(1, [20])
    s.q, s.table, s.seq_lens = s.q[:0], s.table[:0], s.seq_lens[:0]
    assert call(ops, s).shape == (0, 8, 128)


def test_a_cache_of_several_layers():
    """Pages by the cache's own tables, exported and brought back into others; half of the FP8 cache's bytes and a little more."""
    cache = PagedKV4Cache(layers=2, kv_heads=2, head_dim=64, num_pages=9, max_seqs=2, max_pages_per_seq=4, device="cpu")
    fp8 = PagedKVCache(layers=2, kv_heads=2, head_dim=64, num_pages=9, max_seqs=2, max_pages_per_seq=4, device="cpu")
    assert cache.bytes_per_token() * 16 * 9 == cache.data.numel() and cache.bytes_per_token() / fp8.bytes_per_token() < 0.53
    cache.assign(0, 7, 40)
    k, v = torch.randn(2, 40, 2, 64), torch.randn(2, 40, 2, 64)
    for i in range(2):
        ops.kv4_write(k[i], v[i], cache.slots(7, 0, 40), cache.layer(i))
    pages = cache.allocator.owned[7]
    blob = cache.export_pages(pages)
    assert blob.nbytes == cache.page_blob_bytes(3) and blob.dtype == np.uint8
    cache.assign(1, 8, 40)
    cache.import_pages(cache.allocator.owned[8], blob)
    starts = torch.tensor([0, 40, 80], dtype=torch.int32)
    for i in range(2):
        a, b = ops.kv4_gather(cache.layer(i), cache.block_table, starts, 80, dtype=torch.float32)
        assert torch.equal(a[:40], a[40:]) and torch.equal(b[:40], b[40:]) and (a[:40] - k[i]).abs().max() < 0.4
    for how in ({"page_size": 32}, {"head_dim": 96}):
        with pytest.raises(ValueError):
            PagedKV4Cache(**{**dict(layers=1, kv_heads=1, head_dim=64, num_pages=2, max_seqs=1, max_pages_per_seq=1, device="cpu"), **how})
