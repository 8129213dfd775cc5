"""A ragged model without layers for CPU engines: the logits of a token are a row of a table."""

from types import SimpleNamespace

import torch

from mfq_b200.engine.kv_cache import PlainPagedKVCache
from mfq_b200.engine.llm_engine import LLMEngine


class TableModel:
    ragged, tp, hk = True, 1, 1

    def __init__(self, vocab: int, seed: int = 1) -> None:
        self.table = torch.randn((min(vocab, 97), vocab), generator=torch.Generator().manual_seed(seed))
        self.cfg = SimpleNamespace(num_layers=0, head_dim=64, num_heads=1, num_kv_heads=1)
        self.w = SimpleNamespace(embed=torch.zeros(1), mtp=None, tp_rank=0)

    def make_cache(self, **pool):
        return PlainPagedKVCache([], torch.float32, **pool)

    def forward(self, step, cache, prefill, logits_rows=None, gather_logits=True):
        ids = step.input_ids if logits_rows is None else step.input_ids[logits_rows.long()]
        return self.table[ids.long() % self.table.shape[0]]

    def sample_greedy(self, logits, out=None):
        top = logits.argmax(-1).to(torch.int32)
        return top if out is None else out.copy_(top)


def ragged_engine(vocab: int = 97, **how):
    return LLMEngine(TableModel(vocab), **{"max_batch": 4, "max_seq_len": 160, "device": "cpu", **how})
