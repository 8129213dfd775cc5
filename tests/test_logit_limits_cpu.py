"""What requests bring in biases, masks and penalties, and what neighbours and later requests see of it, on CPU engines."""

import pytest
import torch

from mfq_b200 import ops
from mfq_b200.engine.constraints import LogitTables
from mfq_b200.engine.llm_engine import LLMEngine
from mfq_b200.engine.scheduler import ContinuousBatchScheduler, Request
from mfq_b200.models.llama import LlamaConfig, LlamaModel, LlamaWeights
from mfq_b200.parallel.local_collective import LocalGroup
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


def words_of(engine, row, prompt, answer):
    """What the counts of a row have to be."""
    want = torch.zeros(engine.logit_tables.width, dtype=torch.int32)
    for t in answer:
        want[t] += 1
    want[torch.tensor(prompt, dtype=torch.long)] |= 0x8000
    return torch.equal(engine.logit_tables.counts[row].cpu().int() & 0xFFFF, want)


def decoded(engine, row, steps):
    out = []
    for _ in range(steps):
        assert engine.can_grow(row)
        t = engine.decode([row])[row]
        out += t if isinstance(t, list) else [t]
    return out


def test_penalties_on_a_row_whose_prompt_was_read_without(model):
    """They go by this sequence's tokens, whoever had the row before, from the first step on and after an interval without."""
    strong = params(presence_penalty=1e4)
    for occupied in (False, True):
        eng = LLMEngine(model, max_batch=2, max_seq_len=160, device="cpu")
        if occupied:
            eng.prefill(0, list(range(100, 159)), strong)
            decoded(eng, 0, 3)
            eng.release(0)
        prompt = PROMPTS[0]
        answer = [eng.prefill(0, prompt)] + decoded(eng, 0, 4)
        plain = LLMEngine(model, max_batch=2, max_seq_len=160, device="cpu")
        assert answer == [plain.prefill(0, prompt)] + decoded(plain, 0, 4)
        eng.set_sampling(0, strong)
        assert words_of(eng, 0, prompt, answer[:-1])
        more = decoded(eng, 0, 6)
        assert not set(more) & set(answer) and len(set(more)) == len(more)
        answer += more
        assert words_of(eng, 0, prompt, answer[:-1])
        eng.set_sampling(0, None)
        answer += decoded(eng, 0, 3)
        eng.set_sampling(0, params(repetition_penalty=1e6))
        assert words_of(eng, 0, prompt, answer[:-1])
        more = decoded(eng, 0, 4)
        assert not set(more) & (set(answer) | set(prompt))


def test_penalties_after_draft_and_verify_cycles():
    cfg = LlamaConfig.tiny()
    model = LlamaModel(cfg, LlamaWeights.random_init(cfg, "cpu", seed=5, std=0.05, mtp=True))
    eng = LLMEngine(model, max_batch=2, max_seq_len=160, device="cpu", mtp_draft_tokens=2)
    prompt = PROMPTS[0]
    answer = [eng.prefill(0, prompt)] + decoded(eng, 0, 5)
    eng.set_sampling(0, params(presence_penalty=1e4))
    assert words_of(eng, 0, prompt, answer[:-1])
    more = decoded(eng, 0, 4)
    assert not set(more) & set(answer) and len(set(more)) == len(more)


def test_penalties_on_rows_that_were_extended():
    """Given tokens count as a prompt's; in mixed batches, and for a row that was opened with penalties, too."""
    eng = ragged_engine()
    eng.open_row(2, params(presence_penalty=1e4))
    eng.extend([(2, [5, 6, 7])])
    eng.extend([(2, torch.tensor([8]))], [[0]])
    eng.sampled[2] = 30  # what the caller drew from the logits
    eng.row_drawn[2].append(30)
    answer = [30] + decoded(eng, 2, 5)
    assert words_of(eng, 2, [5, 6, 7, 8], answer[:-1]) and len(set(answer)) == len(answer)
    eng.open_row(0)
    eng.extend([(0, [9, 9])], [[1]])
    eng.set_sampling(0, params(presence_penalty=2.0))
    assert words_of(eng, 0, [9], [])
    eng.begin_prompt(1, [3, 4, 5])
    assert eng.can_grow(2)
    answer.append(eng.mixed_step([2], [(1, 3)])[2])
    assert words_of(eng, 2, [5, 6, 7, 8], answer[:-1]) and len(set(answer)) == len(answer)
    eng.set_sampling(1, params(frequency_penalty=1.0))
    assert words_of(eng, 1, [3, 4, 5], [])


def test_penalties_that_have_nothing_to_go_by_are_refused(model):
    eng = LLMEngine(model, max_batch=2, max_seq_len=160, device="cpu")
    eng.prefill(0, PROMPTS[0], params(temperature=0.5))
    eng.grow(0, 60)
    eng.decode_step(1)
    kept = eng.sample_rows[0].clone()
    with pytest.raises(ValueError, match="penalties"):
        eng.set_sampling(0, params(presence_penalty=1.0))
    assert torch.equal(eng.sample_rows[0], kept) and 0 not in eng.row_penalized
    eng.set_sampling(0, params())
    eng.prefill(0, PROMPTS[0], params(presence_penalty=1.0))  # another sequence
    assert words_of(eng, 0, PROMPTS[0], [])
    empty = LLMEngine(model, max_batch=2, max_seq_len=160, device="cpu")
    empty.open_row(0, params(presence_penalty=1.0))
    empty.grow(0, 16)
    with pytest.raises(RuntimeError, match="penalties"):
        empty.decode([0])


class Misses:
    """Stands for layers whose experts are missing in the first attempts of a step."""

    optimistic = False

    def __init__(self, engine, attempts):
        self.engine, self.attempts, self.run = engine, attempts, 0

    def enable_optimistic(self, count):
        self.count = count

    def settle(self):
        return "uploaded" if self.run < 9 else "fallback"


@pytest.mark.parametrize("attempts", [1, 2, 9])
def test_a_step_that_is_run_again_for_its_experts_counts_once(attempts):
    """What it had counted is taken back word by word, not by a copy of the table."""
    eng = ragged_engine()
    misses = Misses(eng, attempts)
    eng.model.residencies = lambda: [misses]
    forward = eng.model.forward

    def missing(step, cache, prefill, **how):
        if misses.optimistic:
            misses.count.fill_(int(misses.run < attempts))
            misses.run += 1
        return forward(step, cache, prefill, **how)

    strong = params(presence_penalty=1e4)
    eng.model.forward = missing
    for row, prompt in enumerate(([5, 6, 7], [9, 8])):
        eng.begin_prompt(row, prompt, strong if row else None)
    answer = [eng.mixed_step([], [(0, 3), (1, 2)])[1]]
    assert eng.enable_expert_residency_graphs()
    counts = eng.logit_tables.counts

    def whole(*_):
        raise AssertionError("a copy of all counts")

    counts.clone = whole
    for _ in range(4):
        misses.run = 0
        assert eng.can_grow(0) and eng.can_grow(1)
        answer.append(eng.decode([0, 1])[1])
        assert words_of(eng, 1, [9, 8], answer[:-1])
    assert len(set(answer)) == len(answer) and eng.logit_tables.counts is counts


def test_steps_of_more_portions_than_a_plan_takes():
    """A batch may have as many rows as the engine."""
    rows = 2 * ops.batch.MAX_REQUESTS + 3
    eng = ragged_engine(max_batch=rows, max_seq_len=32)
    held = []
    forward = eng.model.forward

    def seen(step, cache, prefill, **how):
        held.append(step)
        return forward(step, cache, prefill, **how)

    eng.model.forward = seen
    portions = [(r, [r % 97] * (1 + r % 3)) for r in range(rows)]
    for r in range(rows):
        eng.open_row(r)
    for _ in range(2):
        before = list(eng.row_len[r] for r in range(rows))
        got = eng.extend(portions, [[len(t) - 1] for _, t in portions])
        assert torch.equal(got, eng.model.table[torch.arange(rows) % 97])
        step = held.pop()
        at = 0
        for i, r in enumerate(sorted(range(rows), key=lambda r: len(portions[r][1]) != 1)):
            m, past = len(portions[r][1]), before[r]
            assert step.positions[at : at + m].tolist() == list(range(past, past + m)) and step.tok_seq[at : at + m].tolist() == [i] * m
            assert step.slots[at : at + m].tolist() == eng.cache.slots(eng.row_seq[r], past, m).tolist()
            assert int(step.q_starts[i]) == at and int(step.seq_lens[i]) == past + m
            assert step.block_table[i].tolist() == eng.cache.block_table[r].tolist()
            at += m
        assert int(step.q_starts[rows]) == at == step.positions.numel()


def test_joined_plans_keep_a_refusal():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    table = torch.arange(1, 9, dtype=torch.int32).view(2, 4)
    good, bad = ops.plan_batch(table, i32(0), i32(3), i32(20), tokens=20), ops.plan_batch(table, i32(1), i32(60), i32(5), tokens=5)
    assert ops.BatchPlan.joined([good, good]).check() == (40, 0)
    for plans in ([good, bad], [bad, good]):
        with pytest.raises(ValueError, match="more pages than a row"):
            ops.BatchPlan.joined(plans).check()


def test_penalties_biases_and_masks_over_vocabulary_shards():
    """Every rank processes its columns by its slice of the counts and by vocabulary ids: the shards together are what one rank makes of all columns, and a
    request's answer is penalized, biased and the same on all ranks."""
    cfg = LlamaConfig.tiny()
    g = torch.Generator().manual_seed(1)
    whole = torch.randn((2, cfg.vocab_size), generator=g)
    words = torch.randint(-2 ** 31, 2 ** 31, (-(-cfg.vocab_size // 32),), generator=g).to(torch.int32)
    bias = {3: 2.0, cfg.vocab_size // 2: 30.0, cfg.vocab_size - 1: -5.0}
    forced = cfg.vocab_size - 7

    def body(rank, collective, world):
        how = {"tp_rank": rank, "tp_size": world} if world > 1 else {}
        weights = LlamaWeights.random_init(cfg, "cpu", seed=7, **how)
        eng = LLMEngine(LlamaModel(cfg, weights, collective=collective) if world > 1 else LlamaModel(cfg, weights), max_batch=2, max_seq_len=160, device="cpu")
        for row, how in enumerate((params(presence_penalty=0.4, repetition_penalty=1.5, logit_bias=bias), params(frequency_penalty=0.7))):
            eng.prefill(row, PROMPTS[row], how)
            eng._write_limits([row], cfg.vocab_size)
        eng.logit_tables.allowed[1].copy_(words)
        v = cfg.vocab_size // world
        shard = eng._process(whole[:, rank * v : (rank + 1) * v].clone())
        eng.logit_tables.allowed[1].fill_(-1)
        answer = [eng.prefill(0, PROMPTS[0], params(presence_penalty=1e4, logit_bias={forced: 100.0}))] + decoded(eng, 0, 6)
        return shard, answer, eng.logit_tables.counts[0].tolist()

    shard, answer, counts = body(0, None, 1)
    assert shard.shape == whole.shape and not torch.equal(shard, whole)
    ranks = LocalGroup(2).run(lambda rank, collective: body(rank, collective, 2))
    assert torch.equal(torch.cat([s for s, _, _ in ranks], 1), shard)
    for _, a, c in ranks:
        assert a == ranks[0][1] and c == ranks[0][2] and a[0] == forced and len(set(a)) == len(a)
        assert sum(x & 0x7FFF for x in c) == len(a) - 1


def test_a_refused_set_sampling_leaves_the_row_as_it_was(model):
    eng = LLMEngine(model, max_batch=2, max_seq_len=160, device="cpu")
    eng.prefill(0, PROMPTS[0], params(presence_penalty=1.0))
    eng.grow(0, 60)
    eng.decode_step(1, constrained=True)
    kept, counts = eng.sample_rows[0].clone(), eng.logit_tables.counts.clone()
    with pytest.raises(ValueError, match="penalties"):
        eng.set_sampling(0, params(presence_penalty=2.0))
    assert torch.equal(eng.sample_rows[0], kept) and 0 in eng.row_penalized and torch.equal(eng.logit_tables.counts, counts)
