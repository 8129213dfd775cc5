"""Requests with penalties through an engine, for the CPU and the GPU tests."""

from mfq_b200.engine.scheduler import ContinuousBatchScheduler, Request, SamplingParams

PROMPTS = [list(range(5, 40)), [7, 9, 7, 7, 300, 2], [11] * 20, list(range(900, 930))]


def run(engine, requests, steps=400, **how):
    sched = ContinuousBatchScheduler(engine, max_queue=16, **how)
    for r in requests:
        sched.submit(r)
    for _ in range(steps):
        if not sched.step() and sched.idle:
            break
    assert all(r.error is None for r in requests)
    return [list(r.generated) for r in requests]


def params(**how):
    return SamplingParams(max_tokens=16, **how)


def check(make, replay=True):
    """``make()``: an engine.  What penalties promise of a greedy answer, beside rows without any.  ``replay``: whether a prompt's pass gives
    the bits of decoding, so that a request that is read again goes on as it did."""
    plain = run(make(), [Request(list(p), params()) for p in PROMPTS])
    free = run(make(), [Request(list(p), params()) for p in PROMPTS])
    assert plain == free
    assert any(len(set(g)) < len(g) for g in plain), "the model has to repeat itself for this to say something"
    # no token of the answer twice; tokens of the prompt are free to come
    eng = make()
    mixed = run(eng, [Request(list(p), params(presence_penalty=1e4) if i % 2 == 0 else params()) for i, p in enumerate(PROMPTS)])
    for i, g in enumerate(mixed):
        assert g == plain[i] if i % 2 else len(set(g)) == len(g) and g[0] == plain[i][0]
    assert not eng.row_penalized  # released with the rows
    # once and no more for a frequency that outweighs everything, however the rows are drawn
    for g in run(make(), [Request(list(p), params(frequency_penalty=1e4, temperature=0.8, seed=i + 1)) for i, p in enumerate(PROMPTS)]):
        assert len(set(g)) == len(g)
    # neither the prompt's tokens nor the answer's: an answer's positive logits are divided away, its negative ones pushed down
    for p, g in zip(PROMPTS, run(make(), [Request(list(p), params(repetition_penalty=1e6)) for p in PROMPTS])):
        assert len(set(g)) == len(g) and not set(g) & set(p)
    # a bias beside penalties
    one = params(presence_penalty=3.0, frequency_penalty=0.5, repetition_penalty=1.3, logit_bias={plain[0][0]: -100})
    whole = run(make(), [Request(list(PROMPTS[0]), one)])[0]
    assert plain[0][0] not in whole
    if not replay:
        return
    again = Request(list(PROMPTS[0]), one)
    again.generated = whole[:7]
    assert run(make(), [again])[0] == whole
