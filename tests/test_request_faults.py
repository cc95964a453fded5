"""Requests whose options, or whose steps, fail: what they are told, and what is left behind them (on the CPU, with plain twins of the kernels)."""
import math

import pytest

from test_requests import adapters_of, engine, greedy, tiny  # noqa: F401

INF, NAN = math.inf, math.nan


@pytest.mark.parametrize("options,what", [
    (dict(logit_bias={5: None}), "logit_bias of token 5"), (dict(logit_bias={5: "1"}), "logit_bias of token 5"), (dict(logit_bias={None: 1.0}), "names token None"),
    (dict(logit_bias={"x": 1.0}), "names token 'x'"), (dict(logit_bias={INF: 1.0}), "names token inf"), (dict(logit_bias={NAN: 1.0}), "names token nan"),
    (dict(logit_bias=[1.0, 2.0]), "logit_bias must"), (dict(logit_bias=3), "logit_bias must"), (dict(presence_penalty=None), "finite"),
    (dict(frequency_penalty="1"), "finite"), (dict(presence_penalty=10 ** 400), "finite"), (dict(logprobs="5"), "logprobs"), (dict(logprobs=2.5), "logprobs"),
    (dict(logprobs=[1]), "logprobs")])
def test_options_that_are_no_numbers_fail_their_own_request(tiny, options, what):  # noqa: F811
    from ninfer_amd import Request, Scheduler
    eng = engine(tiny[0])
    sched = Scheduler(eng.runner, eng.sampler)
    bad, fine = Request("bad", [1], greedy(2, **options)), Request("fine", [1, 2], greedy(2))
    sched.add(bad)
    sched.add(fine)
    sched.run()
    assert (bad.status, fine.status) == ("failed", "finished") and what in bad.error
    with pytest.raises(RuntimeError, match="request 0"):
        eng.generate([[1]], greedy(2, **options), [])
