"""What requests bring in biases, masks and penalties, and what neighbours and later requests see of it, on CPU engines."""

import pytest
import torch

from mfq_b200 import ops
from mfq_b200.engine.constraints import LogitTables
from mfq_b200.engine.llm_engine import LLMEngine
from mfq_b200.engine.scheduler import ContinuousBatchScheduler, Request
from mfq_b200.models.llama import LlamaConfig, LlamaModel, LlamaWeights
from penalty_cases import PROMPTS, params
from ragged_stub import ragged_engine


@pytest.fixture(scope="module")
def model():
    cfg = LlamaConfig.tiny()
    return LlamaModel(cfg, LlamaWeights.random_init(cfg, "cpu", seed=7))


def serve(engine, requests, **how):
    sched = ContinuousBatchScheduler(engine, max_queue=16, **how)
    for r in requests:
        sched.submit(r)
    for _ in range(400):
        if not sched.step() and sched.idle:
            break
    return sched, [list(r.generated) for r in requests]


def both_engines(model):
    """Engines that run a prompt at once, and that read it in portions beside other rows; with a scheduler's settings and prompts."""
    return ((lambda: LLMEngine(model, max_batch=4, max_seq_len=160, device="cpu"), {}, PROMPTS),
            (ragged_engine, {"mixed_tokens": 8}, [[t % 97 for t in p] for p in PROMPTS]))


OUTSIDE = [{2 ** 31: 1.0}, {-1: 5.0, 2 ** 40: -3.0, -2 ** 33: 1.0}, {2 ** 31 - 1: 4.0, 10 ** 30: 1.0}]


@pytest.mark.parametrize("bias", OUTSIDE)
def test_biases_of_ids_outside_the_vocabulary_are_none(model, bias):
    for make, how, prompts in both_engines(model):
        _, plain = serve(make(), [Request(list(p), params()) for p in prompts], **how)
        requests = [Request(list(p), params(logit_bias=dict(bias) if i == 1 else None)) for i, p in enumerate(prompts)]
        sched, got = serve(make(), requests, **how)
        assert sched.healthy and all(r.error is None for r in requests) and got == plain
        inside = {plain[0][0]: -100}
        one, other = (serve(make(), [Request(list(prompts[0]), params(logit_bias=b))], **how)[1][0] for b in (inside, {**bias, **inside}))
        assert one == other and plain[0][0] not in one


def test_more_biases_than_a_table_holds():
    """As many as there are tokens, in any engine; the last ones and the ones at the tables' edges count like the first."""
    vocab = 2 * ops.MAX_BIASES + 500
    left = (3, ops.MAX_BIASES - 1, ops.MAX_BIASES, 2 * ops.MAX_BIASES, vocab - 1)
    banned = {t: -100.0 for t in range(vocab) if t not in left}
    make = lambda: ragged_engine(vocab, max_batch=3)  # noqa: E731
    prompts = [list(range(5, 25)), [7, 9, 7, 7, 30, 2], [11] * 20]
    _, plain = serve(make(), [Request(list(p), params()) for p in prompts], mixed_tokens=8)
    eng = make()
    requests = [Request(list(prompts[0]), params(logit_bias=banned)), Request(list(prompts[1]), params()),
                Request(list(prompts[2]), params(presence_penalty=1e4, logit_bias=banned))]
    sched, got = serve(eng, requests, mixed_tokens=8)
    assert sched.healthy and all(r.error is None for r in requests)
    at = prompts[0][-1]
    for token in got[0]:  # the arg-max of what is left
        row = eng.model.table[at % 97]
        assert token == max(left, key=lambda t: row[t])
        at = token
    assert got[1] == plain[1]
    assert set(got[2][:5]) == set(left) and len(set(got[2])) == len(got[2])
    assert serve(eng, [Request(list(prompts[0]), params(presence_penalty=1e-9))], mixed_tokens=8)[1][0] == plain[0]  # no biases any more


class Broken:
    """A constraint of which one half cannot be written."""

    def __init__(self, words, table):
        self.held = words, table

    def words(self, width):
        if isinstance(self.held[0], Exception):
            raise self.held[0]
        return self.held[0]

    def biases(self, width):
        return self.held[1]


@pytest.mark.parametrize("words,table", [(torch.zeros(2, dtype=torch.int32), {5: 1.0, 6: "no number"}), (torch.zeros(7, dtype=torch.int32), {5: 1.0}),
                                         (RuntimeError("no words"), {5: 1.0})])
def test_limits_that_fail_leave_nothing_behind(words, table):
    """The row's next request has the tables as if they were new, and a request that had the row keeps nothing of what failed."""
    for before in (None, Broken(torch.full((2,), 12, dtype=torch.int32), {1: 2.0})):
        t = LogitTables(3, 64, torch.device("cpu"))
        t.limit(1, before)
        with pytest.raises(Exception):
            t.limit(1, Broken(words, table))
        t.limit(1, None)
        assert (t.allowed == -1).all() and (t.bias_ids == -1).all()
        t.limit(1, Broken(torch.full((2,), 9, dtype=torch.int32), {7: 3.0}))
        assert t.allowed[1].tolist() == [9, 9] and t.bias_ids[1, 0] == 7 and t.biases[0][1][1, 0] == 3.0 and (t.bias_ids[1, 1:] == -1).all()


def test_places_of_a_large_request_go_with_it():
    """Every row's kernel goes over all places, so that one request with very many biases must not leave them to all later ones."""
    vocab = ops.MAX_BIASES + 4000
    eng = ragged_engine(vocab, max_batch=3)
    many = {t: -1.0 for t in range(vocab - 9)}
    assert serve(eng, [Request([5, 6, 7], params(logit_bias=many))], mixed_tokens=8)[0].healthy
    assert sum(ids.shape[1] for ids, _ in eng.logit_tables.biases) >= len(many)
    two = {9: 100.0, 10: 99.0}
    got = serve(eng, [Request([5, 6, 7], params(logit_bias=two, presence_penalty=3.0)), Request([8, 9], params(presence_penalty=1.0))], mixed_tokens=8)[1]
    assert sum(ids.shape[1] for ids, _ in eng.logit_tables.biases) == 8 and set(got[0]) <= set(two)
    t = LogitTables(2, 2000, torch.device("cpu"))
    assert t.make_room(1500) and not t.make_room(600) and t.make_room(500)  # not back and forth between requests of like sizes
    assert t.make_room(1000) and not t.make_room(0)  # few enough to stay
