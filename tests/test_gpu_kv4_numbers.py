"""Attention over 4-bit pages where its sums are hard to hold: scales far apart, long contexts, averages that cancel."""

import math

import pytest
import torch

from mfq_b200 import ops
from mfq_b200.engine.kv_cache import LayerKV4
from mfq_b200.ops import kv4
from gpu_common import check_status, require_gpu_lib
from kv4_cases import BATCHES, assert_attends, batch, call, exact
from kv4_rms import assert_close_on_average, exact_and_weights, skewed

pytestmark = pytest.mark.gpu
FORMS = [None, (1, 0), (2, 0), (8, 0), (0, 1), (0, 3), (0, 50)]


def run(s, want, **how):
    out = call(ops, s, out=torch.full_like(s.q, 3.0), **how)
    check_status()
    assert_attends(s, out, want)
    return out


def value_params(s):
    """Scales and minima of V, ``[pages, heads, 8, 2, groups, 2]`` in bf16, and a way to put them back."""
    d, data = s.d, s.kv.data
    x = data[:, :, 17 * d :].contiguous().view(torch.bfloat16).view(data.shape[0], data.shape[1], 8, 2, d // 64, 2)
    return x, lambda y: data[:, :, 17 * d :].copy_(y.contiguous().view(torch.uint8).view(data.shape[0], data.shape[1], d))


def by_pages(s, power):
    """V's page ``i`` of a sequence times ``2^power(i)``."""
    x, put = value_params(s)
    x = x.float()
    for row, n in enumerate(s.lens):
        for i in range(-(-n // 16)):
            x[int(s.table[row, i])] *= 2.0 ** power(i)
    put(x.to(torch.bfloat16))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("how", [{}, {"d": 64, "dtype": torch.float16}, {"hq": 14}, {"hq": 24, "dtype": torch.float16}, {"d": 256, "hq": 6}])
def test_scales_of_values_that_are_far_apart(form, how, monkeypatch):
    """2^-64 and 2^64: what the rows have in front of the large values keeps its part of the softmax, wherever the border is."""
    require_gpu_lib()
    if form is not None:
        monkeypatch.setattr(kv4, "_shape", lambda *a: form)
    for power in (lambda i: -64 if i < 20 else 64, lambda i: 64 if i < 20 else -64, lambda i: 64 if i // 2 % 4 == 1 else -64, lambda i: (-64, 0, 64)[i // 2 % 3], lambda i: 64 if i == 30 else -64):
        s = batch(3, [640, 900, 40, 333], device="cuda", **how)
        half = how.get("dtype") is torch.float16  # outputs of 2^64 are none of its numbers
        by_pages(s, (lambda i: {-64: -98, 0: -40, 64: 8}[power(i)]) if half else power)
        want = exact(s)
        assert torch.equal(run(s, want), run(s, want))


@pytest.mark.parametrize("form", FORMS)
def test_a_group_of_one_large_value_beside_tiny_ones(form, monkeypatch):
    """Scale 0 and a minimum of 2^20 in one group, scales of 2^-98 in the other."""
    require_gpu_lib()
    if form is not None:
        monkeypatch.setattr(kv4, "_shape", lambda *a: form)
    s = batch(3, [640, 900, 40, 333], device="cuda")
    x, put = value_params(s)
    x = x.float() * 2.0 ** -96
    real = ~x[..., 0, 0].isnan()
    x[..., 0, 0] = torch.where(real, 0.0, x[..., 0, 0])
    x[..., 0, 1] = torch.where(real, 2.0 ** 20, x[..., 0, 1])
    put(x.to(torch.bfloat16))
    out = run(s, exact(s))
    seen = out.view(4, -1, 128)
    assert (seen[..., :64] == 2.0 ** 20).all()


@pytest.mark.parametrize("form", [None, (1, 0), (8, 0), (0, 3), (0, 50)])
def test_many_keys_above_the_first_ones_and_tiny_values(form, monkeypatch):
    """The first keys' scores lie 5.9 powers of two below all others: a reference that lags.  2^19 keys, values near 2^-100."""
    require_gpu_lib()
    if form is not None:
        monkeypatch.setattr(kv4, "_shape", lambda *a: form)
    n, d = 1 << 19, 64
    kv = LayerKV4(torch.full((n // 16 + 1, 1, 18 * d), 255, dtype=torch.uint8, device="cuda"), d, 16)
    k = torch.ones(n, 1, d, device="cuda")
    per = -(-n // 50 // 32) * 32  # the shares' pairs and the clusters' begin here or there: more low keys than one beginning has
    for at in {0, n // 8, n // 4, 3 * n // 8, n // 2, 5 * n // 8, 3 * n // 4, 7 * n // 8, *range(0, n, per), *(n * i // 3 // 32 * 32 for i in range(3))}:
        k[max(0, at - 256) : at + 256] = 0.0
    g = torch.Generator(device="cuda").manual_seed(2)
    v = (torch.randn(n, 1, d, generator=g, device="cuda") + 1) * 2.0 ** -99
    ops.kv4_write(k, v, torch.arange(16, 16 + n, dtype=torch.int32, device="cuda"), kv)
    table = torch.arange(1, n // 16 + 1, dtype=torch.int32, device="cuda")[None]
    q = torch.full((1, 4, d), 1.0, dtype=torch.bfloat16, device="cuda")
    scale = 5.9 * math.log(2) / d
    out = ops.paged_attn_decode_kv4(q, kv, table, torch.tensor([n], dtype=torch.int32, device="cuda"), sm_scale=scale)
    check_status()
    kept_k, kept_v = ops.kv4_gather(kv, table, torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, dtype=torch.float32)
    assert torch.equal(kept_k, k)
    p = torch.softmax(kept_k[:, 0].double().sum(-1) * scale, 0)
    want, size = p @ kept_v[:, 0].double(), p @ kept_v[:, 0].double().abs()
    # the output's rounding; p s to fp16 of up to 15 scales, of which the groups have 7.5 on average and |v| 2.7 or more: 2^-11 * 15 / 2.7
    assert ((out[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * size).all(), (out[0, 0, :4], want[:4])


LONG = [  # lengths, form, what else: chains of thousands of tokens a warp in every kind of columns
    ([16384, 12345], (1, 0), {}),
    ([16384, 12345], (0, 1), {"hq": 32, "hk": 2}),
    ([16384, 9000], (1, 0), {"hq": 16, "hk": 2}),
    ([16384, 12345], (1, 0), {"hq": 4, "hk": 1, "q_len": 3}),
    ([16384], (1, 0), {"hq": 8, "hk": 2, "d": 64}),
    ([16384, 700], (1, 0), {"hq": 32, "hk": 2, "d": 64}),
    ([9000, 16384], (1, 0), {"hq": 8, "hk": 1, "d": 256}),
    ([60000], (1, 0), {"hq": 8, "hk": 1}),
    ([60000], (8, 0), {"hq": 16, "hk": 1}),
    ([60000, 300, 16384], None, {"hq": 32, "hk": 2}),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["even", "skewed"])
@pytest.mark.parametrize("lens,form,how", LONG)
def test_averages_over_long_contexts_keep_their_precision(lens, form, how, kind, dtype, monkeypatch):
    """Queries that see all keys nearly alike: outputs a hundredth of the values, and of what is added up for them."""
    require_gpu_lib()
    if form is not None:
        monkeypatch.setattr(kv4, "_shape", lambda *a: form)
    s = batch(len(lens), lens, dtype=dtype, device="cuda", q_std=0.15, **how)
    if kind == "skewed":
        skewed(s)
    out = call(ops, s)
    check_status()
    assert_close_on_average(s, out, exact_and_weights(s))


@pytest.mark.parametrize("lens,how", [x for x in BATCHES if sum(x[0]) > 700 and "spread" not in x[1]])
def test_batches_are_off_by_little_more_than_their_rounding(lens, how):
    require_gpu_lib()
    for dtype in (torch.float16, torch.bfloat16):
        s = batch(len(lens), lens, device="cuda", **{**how, "dtype": dtype})
        out = call(ops, s)
        check_status()
        assert_close_on_average(s, out, exact_and_weights(s))
