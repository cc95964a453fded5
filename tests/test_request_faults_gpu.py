"""Requests whose masks and biases leave no token, on the GPU's sampling paths."""
import math

import pytest
import torch

from test_requests_gpu import make

pytestmark = pytest.mark.gpu
INF = math.inf


@pytest.mark.parametrize("vocab", [300, 40000])
@pytest.mark.parametrize("options", [dict(temperature=0.0), dict(temperature=0.8, top_k=50), dict(temperature=0.8, top_k=0), dict(temperature=0.8, top_k=5000),
                                     dict(temperature=0.0, repetition_penalty=1.3)])
def test_rows_that_no_token_is_left_to_are_known_by_what_they_draw(vocab, options):
    from ninfer_amd import Sampler, SamplingParams
    from ninfer_amd.kernels import load_ops
    from ninfer_amd.sampling import SampleRow
    from ninfer_amd.sampling.sampler import History, allowed_words
    sampler = Sampler(load_ops(), torch.device("cuda"))
    ids = [7, vocab - 2]
    make_row = lambda i, bias, allowed: SampleRow(SamplingParams(logit_bias=bias, **options), History([7, 8]), i, 0, 5, allowed_words(allowed, vocab))
    rows = [make_row(0, {t: -INF for t in ids}, ids), make_row(1, None, None), make_row(2, {ids[0]: -INF}, ids), make_row(3, {t: -INF for t in range(vocab)}, None)]
    logits = torch.randn(4, vocab, generator=torch.Generator("cuda").manual_seed(vocab), device="cuda")
    tokens = sampler.sample(logits, rows)
    assert all(0 <= t < vocab for t in tokens) and tokens[2] == ids[1]
    assert [r.bars(t) for r, t in zip(rows, tokens)] == [True, False, False, True]


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_requests_that_no_token_is_left_to(model_dirs, temperature):
    from ninfer_amd import Request, SamplingParams, Scheduler
    eng = make(model_dirs, "A", "float32")
    sched = Scheduler(eng.runner, eng.sampler)
    draw = lambda **kw: SamplingParams(temperature=temperature, seed=3, max_new_tokens=4, **kw)
    reqs = [Request("a", [1, 2], draw(logit_bias={9: -INF}), allow=lambda out: [9]), Request("b", [1, 2], draw()),
            Request("c", [1, 2], draw(logit_bias={t: -INF for t in range(256)}))]
    for r in reqs:
        sched.add(r)
    sched.run()
    assert [(r.status, len(r.output)) for r in reqs] == [("failed", 0), ("finished", 4), ("failed", 0)]
    assert all("no token is left" in reqs[i].error for i in (0, 2))
    eng.close()
