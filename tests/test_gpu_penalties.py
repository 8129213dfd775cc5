"""Penalties for repeated tokens and ragged batches planned on the device, end to end on the GPU engine."""

import dataclasses

import pytest
import torch

import tepetar_cases as cases
from gpu_common import check_status, require_gpu_lib
from mfq_b200.engine.llm_engine import LLMEngine
from mfq_b200.engine.scheduler import Request
from mfq_b200.models.llama import LlamaConfig, LlamaModel, LlamaWeights
from mfq_b200.ops import MAX_BIASES
from penalty_cases import PROMPTS, check, params, run
from test_gpu_tepetar import engine_of
from test_logit_limits_cpu import decoded, words_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [False, True])
def test_penalties(graphs):
    require_gpu_lib()
    cfg = LlamaConfig.tiny()
    w = LlamaWeights.random_init(cfg, "cuda", seed=7)
    check(lambda: LLMEngine(LlamaModel(cfg, w), max_batch=4, max_seq_len=160, use_graphs=graphs), replay=False)
    check_status()


def test_a_captured_step_draws_what_an_eager_one_does():
    """Counts are those of the tokens that were fed, not of the passes that warmed a graph up; biases that outgrow their places drop the graphs."""
    require_gpu_lib()
    cfg = LlamaConfig.tiny()
    w = LlamaWeights.random_init(cfg, "cuda", seed=3)
    made = []
    for graphs in (False, True):
        eng = LLMEngine(LlamaModel(cfg, w), max_batch=4, max_seq_len=160, use_graphs=graphs)
        few = params(presence_penalty=0.4, frequency_penalty=0.3, repetition_penalty=1.2, logit_bias={5: 4.0})
        many = params(frequency_penalty=0.6, temperature=0.7, seed=5, logit_bias={t: -3.0 for t in range(0, 1000, 7)})
        first = run(eng, [Request(list(PROMPTS[0]), few), Request(list(PROMPTS[1]), params())])
        made.append((first, run(eng, [Request(list(PROMPTS[2]), many), Request(list(PROMPTS[3]), few)])))
    assert made[0] == made[1]


def test_mixed_batches_count_what_they_feed(tmp_path):
    require_gpu_lib()
    cfg = cases.uneven()
    eng = engine_of(tmp_path, cfg, cases.weights(cfg), max_batch=4, max_seq_len=256)
    assert eng.mixed_batches
    prompts = [cases.tokens(cfg, n, seed=n) for n in (40, 3, 90, 17)]
    for g in run(eng, [Request([int(t) for t in p], params(presence_penalty=1e4)) for p in prompts], mixed_tokens=32):
        assert len(set(g)) == len(g)


def test_more_biases_than_a_table_holds_and_their_end():
    """Several tables inside captured steps, and graphs that are made again when the tables shrink."""
    require_gpu_lib()
    cfg = dataclasses.replace(LlamaConfig.tiny(), vocab_size=2 * MAX_BIASES + 1024)
    w = LlamaWeights.random_init(cfg, "cuda", seed=7)
    left = (3, MAX_BIASES - 1, MAX_BIASES, 2 * MAX_BIASES, cfg.vocab_size - 1)
    banned = {t: -100.0 for t in range(cfg.vocab_size) if t not in left}
    banned[2 ** 40] = 100.0
    made = []
    for graphs in (False, True):
        eng = LLMEngine(LlamaModel(cfg, w), max_batch=4, max_seq_len=160, use_graphs=graphs)
        plain = run(eng, [Request(list(p), params()) for p in PROMPTS[:2]])
        both = run(eng, [Request(list(PROMPTS[0]), params(logit_bias=banned)), Request(list(PROMPTS[1]), params()),
                         Request(list(PROMPTS[2]), params(presence_penalty=1e4, logit_bias=banned))])
        assert set(both[0]) <= set(left) and both[1] == plain[1] and set(both[2][: len(left)]) == set(left) and len(set(both[2])) == len(both[2])
        after = run(eng, [Request(list(PROMPTS[0]), params(presence_penalty=1e-9, logit_bias={7: -1.0})), Request(list(PROMPTS[1]), params())])
        assert after[1] == plain[1] and sum(ids.shape[1] for ids, _ in eng.logit_tables.biases) == 8
        made.append((plain, both, after))
    assert made[0] == made[1]
    check_status()


@pytest.mark.parametrize("graphs", [False, True])
def test_penalties_on_a_row_whose_prompt_was_read_without(graphs):
    require_gpu_lib()
    cfg = LlamaConfig.tiny()
    eng = LLMEngine(LlamaModel(cfg, LlamaWeights.random_init(cfg, "cuda", seed=7)), max_batch=2, max_seq_len=160, use_graphs=graphs)
    strong = params(presence_penalty=1e4)
    for _ in range(2):  # the second time the tables have the counts of the first
        answer = [eng.prefill(0, PROMPTS[0])] + decoded(eng, 0, 4)
        for on in (True, False, True):
            eng.set_sampling(0, strong if on else None)
            if on:
                assert words_of(eng, 0, PROMPTS[0], answer[:-1])
            more = decoded(eng, 0, 4)
            assert not on or (not set(more) & set(answer) and len(set(more)) == len(more))
            answer += more
        assert words_of(eng, 0, PROMPTS[0], answer[:-1])
        eng.release(0)
    check_status()
