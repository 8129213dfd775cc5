"""Penalties for repeated tokens end to end on the CPU engine."""

import pytest

from mfq_b200.engine.llm_engine import LLMEngine
from mfq_b200.models.llama import LlamaConfig, LlamaModel, LlamaWeights
from mfq_b200.ops import MAX_BIASES
from penalty_cases import PROMPTS, check, params, run
from mfq_b200.engine.scheduler import Request


@pytest.fixture(scope="module")
def model():
    cfg = LlamaConfig.tiny()
    return LlamaModel(cfg, LlamaWeights.random_init(cfg, "cpu", seed=7))


def test_penalties(model):
    check(lambda: LLMEngine(model, max_batch=4, max_seq_len=160, device="cpu"))


def test_many_biases_and_their_end(model):
    eng = LLMEngine(model, max_batch=2, max_seq_len=160, device="cpu")
    first = run(eng, [Request(list(PROMPTS[0]), params())])[0]
    banned = {t: -100 for t in range(1024) if t not in (3, 4)}
    assert set(run(eng, [Request(list(PROMPTS[0]), params(logit_bias=banned))])[0]) <= {3, 4}
    assert eng.logit_tables.bias_ids.shape[1] == 1024
    assert run(eng, [Request(list(PROMPTS[0]), params(presence_penalty=1e-9))])[0] == first  # the row has no biases any more
    with pytest.raises(ValueError, match="biases"):
        eng.logit_tables.make_places(MAX_BIASES + 1)


def test_penalties_that_are_none(model):
    """No numbers and no factors are as no penalty; infinities are as very large ones."""
    make = lambda: LLMEngine(model, max_batch=2, max_seq_len=160, device="cpu")  # noqa: E731
    one = lambda **how: run(make(), [Request(list(PROMPTS[1]), params(**how))])[0]  # noqa: E731
    plain = one()
    nan, inf = float("nan"), float("inf")
    for how in ({"repetition_penalty": 0.0}, {"repetition_penalty": -2.0}, {"repetition_penalty": nan}, {"presence_penalty": nan, "frequency_penalty": nan}):
        eng = make()
        assert run(eng, [Request(list(PROMPTS[1]), params(**how))])[0] == plain and eng.logit_tables is None
    for how in ({"repetition_penalty": inf}, {"presence_penalty": inf}, {"frequency_penalty": 1e300}):
        answer = one(**how)
        assert len(set(answer)) == len(answer)
