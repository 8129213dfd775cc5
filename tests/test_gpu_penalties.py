"""Penalties for repeated tokens and ragged batches planned on the device, end to end on the GPU engine."""

import pytest
import torch

import tepetar_cases as cases
from gpu_common import check_status, require_gpu_lib
from mfq_b200.engine.llm_engine import LLMEngine
from mfq_b200.engine.scheduler import Request
from mfq_b200.models.llama import LlamaConfig, LlamaModel, LlamaWeights
from penalty_cases import PROMPTS, check, params, run
from test_gpu_tepetar import engine_of

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
