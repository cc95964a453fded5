"""Requests whose options, or whose steps, fail: what they are told, and what is left behind them (on the CPU, with plain twins of the kernels)."""
import ctypes
import math

import pytest

from test_requests import adapters_of, engine, greedy, lib, refuses, tiny  # noqa: F401

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


def test_a_call_that_raises_leaves_nothing_held(tiny, tmp_path, monkeypatch):  # noqa: F811
    """Slots, pages and adapters of requests that wait or run come back, whatever ends the call that made them."""
    folder, cfg, _ = tiny
    eng = engine(folder, max_adapters=1, num_sequences=2, num_pages=14)
    path = adapters_of(tmp_path, cfg)["all"][0]
    free = [g.allocator.free_pages for g in eng.runner.cache.groups]

    def stops(out):
        if len(out) == 2:
            raise KeyboardInterrupt
        return None

    def no_rows(logits, rows):
        raise ArithmeticError("rows")

    for prompts, error, allow, sample in (
            ([[1, 2], [9999], [3], [4]], ValueError, None, None),          # a step that refuses its tokens
            ([[1, 2], [None, 3]], TypeError, None, None),                  # a prompt that is none
            ([[1, 2], [5] * 30, [3], [4]], KeyboardInterrupt, [stops] * 4, None),
            ([[1, 2], [5], [3]], ArithmeticError, None, no_rows)):
        eng.load_adapter("all", path)
        with monkeypatch.context() as m:
            if sample is not None:
                m.setattr(eng.sampler, "sample", sample)
            with pytest.raises(error):
                eng.generate(prompts, greedy(6), [], ["all"] * len(prompts), allow)
        assert eng.runner.cache.free_slots == 2
        assert [g.allocator.free_pages for g in eng.runner.cache.groups] == free
        eng.remove_adapter("all")     # (refused while a request has it)
    eng.runner.cache.check()
    assert len(eng.generate([[1, 2], [3]], greedy(3), [])) == 2


def test_a_scheduler_that_is_given_up(tiny, tmp_path):  # noqa: F811
    from ninfer_amd import Request, Scheduler
    folder, cfg, _ = tiny
    eng = engine(folder, num_sequences=2)
    eng.load_adapter("all", adapters_of(tmp_path, cfg)["all"][0])
    sched = Scheduler(eng.runner, eng.sampler)
    reqs = [Request(str(i), [1 + i, 2, 3], greedy(5), [], "all") for i in range(4)]
    for r in reqs:
        sched.add(r)
    sched.step()
    with pytest.raises(TypeError):
        sched.add(Request("none", [None], greedy(5), [], "all"))
    assert sched.abort("enough") == reqs and not sched.has_work()
    assert [(r.status, r.error, r.slot) for r in reqs] == [("failed", "enough", None)] * 4 and sched.finished == reqs
    assert eng.runner.cache.free_slots == 2 and sched.abort() == []
    eng.remove_adapter("all")


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_a_request_that_no_token_is_left_to_ends_itself(tiny, temperature):  # noqa: F811
    """Masks and biases that together (or biases that alone) bar every token: no barred token comes."""
    from ninfer_amd import Request, Scheduler
    eng = engine(tiny[0])
    every = {t: -INF for t in range(256)}
    sched = Scheduler(eng.runner, eng.sampler)
    draw = lambda **kw: greedy(4, temperature=temperature, seed=3, **kw)
    reqs = [Request("a", [1, 2], draw(logit_bias={9: -INF}), allow=lambda out: [9]),
            Request("b", [1, 2], draw(logit_bias={9: -INF, 8: 1.0}), allow=lambda out: [9, 8] if len(out) < 2 else [9]),
            Request("c", [1, 2], draw(logit_bias=every)), Request("d", [1, 2], draw()),
            Request("e", [1, 2], draw(logit_bias={str(t): -INF for t in range(256)})),
            Request("f", [1, 2], draw(logit_bias={t: v for t, v in every.items() if t != 77}))]
    for r in reqs:
        sched.add(r)
    sched.run()
    assert [r.status for r in reqs] == ["failed", "failed", "failed", "finished", "failed", "finished"]
    assert all("no token is left" in r.error for r in reqs if r.status == "failed")
    assert [r.output for r in reqs[:3]] == [[], [8, 8], []] and reqs[4].output == [] and reqs[5].output == [77] * 4
    assert eng.runner.cache.free_slots == 4
    import numpy as np
    row = np.zeros(256, np.float32)
    for kw in (dict(allowed=[9, 3], logit_bias={9: -INF, 3: -INF}), dict(logit_bias=every)):
        with pytest.raises(ValueError, match="no token is left"):
            eng.sample(row, temperature, **kw)
    assert eng.sample(row, temperature, allowed=[9, 3], logit_bias={9: -INF}) == 3
    low = np.full(256, -INF, np.float32)
    low[5] = 1.0
    with pytest.raises(ValueError, match="no token is left"):   # (the model's own logits leave none of it)
        eng.sample(low, temperature, allowed=[9, 200])


def test_adapter_options_that_are_not_known_are_refused(tiny, tmp_path):  # noqa: F811
    import request_ops as ro
    from ninfer_amd import WeightError
    folder, cfg, _ = tiny
    eng = engine(folder)
    factors = ro.random_factors(ro.attention_shapes(cfg, [0], "q"), 4, 1)
    for i, options in enumerate((dict(alora_invocation_tokens=[5, 6]), dict(some_new_option=True), dict(some_new_option="x"), dict(some_new_option=0.5),
                                 dict(target_parameters=["mlp.experts.down_proj"]), dict(arrow_config={"top_k": 2}), dict(use_rslora="false"))):
        with pytest.raises(WeightError, match=f"{next(iter(options))} ="):
            eng.load_adapter("bad", ro.write_adapter(tmp_path / f"bad{i}", factors, 4, 4, **options))
    assert eng.adapters() == []
    # what training libraries write beside the options that count, and options that are off
    usual = dict(alora_invocation_tokens=None, alpha_pattern={}, arrow_config=None, auto_mapping=None, base_model_name_or_path="some/model", corda_config=None,
                 ensure_weight_tying=False, eva_config=None, exclude_modules=["lm_head"], fan_in_fan_out=False, inference_mode=True, init_lora_weights=True,
                 layer_replication=None, layers_pattern=None, layers_to_transform=None, loftq_config={}, lora_bias=False, lora_dropout=0.05,
                 megatron_config=None, megatron_core="megatron.core", modules_to_save=None, peft_version="0.18.0", qalora_group_size=16, rank_pattern={},
                 revision=None, runtime_config={"ephemeral_gpu_offload": False}, target_modules=["q_proj"], target_parameters=None, task_type="CAUSAL_LM",
                 trainable_token_indices=None, use_qalora=False, use_rslora=False, some_new_option=None, another=False, a_third=[], a_fourth={})
    eng.load_adapter("fine", ro.write_adapter(tmp_path / "fine", factors, 4, 4, **usual))
    assert eng.adapters() == ["fine"]


def test_a_place_changes_only_after_the_steps_that_read_it(tiny, tmp_path, monkeypatch):  # noqa: F811
    """Loading and removing wait for the device before they write, and loading after that too (tables that say they are on a GPU; the waits
    are counted and see what has been written)."""
    import torch

    class OnGpu(torch.Tensor):
        is_cuda = True

    folder, cfg, _ = tiny
    eng = engine(folder, max_adapters=1)
    made = adapters_of(tmp_path, cfg)
    held = eng.runner.adapters
    held._scale = torch.Tensor._make_subclass(OnGpu, held._scale)
    numbers = lambda: [t.clone() for s in held.spots for t in (s.tables.a, s.tables.b, s.tables.ranks)] + [held._scale.clone()]
    same = lambda x, y: all(torch.equal(a, b) for a, b in zip(x, y))
    waits = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: waits.append(numbers()))
    for name in ("all", "o"):
        before = numbers()
        eng.load_adapter(name, made[name][0])
        assert len(waits) == 2 and same(waits[0], before) and same(waits[1], numbers()) and not same(before, numbers())
        waits.clear()
        before = numbers()
        eng.remove_adapter(name)
        assert len(waits) == 1 and same(waits[0], before) and not same(before, numbers())
        waits.clear()


def test_rows_too_long_to_count_past_their_end_are_refused(lib):  # noqa: F811
    """The last turn over a row, and its last part, are counted past the row's end in 32 bits."""
    from ninfer_amd.kernels.ops import _ADAPTER_ARGS, _ADJUST_ARGS, _LOGPROB_ARGS
    p, most = 1 << 20, 2 ** 31 - 1
    for v in (most, most - 4095):
        refuses(lib, lambda: lib.ninfer_token_logprobs(_LOGPROB_ARGS.pack(p, p, p, p, p, p, 0, 0, 0, most, 1, v, 1, 0), ctypes.c_void_p(p), None), "too long")
        refuses(lib, lambda: lib.ninfer_adjust_logits(_ADJUST_ARGS.pack(p, p, *[0] * 12, most, most, 1, v, 0, 0, 0, 0), None), "too long")
    for k in (most, most - 127):
        refuses(lib, lambda: lib.ninfer_adapter_add(_ADAPTER_ARGS.pack(p, p, p, p, p, p, p, p, p, most, 64, 64, 1, k, 8, 1, 1, 64, 0, 64, 64, 64, 64, 1, 0), None),
                "too long")


def test_truth_values_are_no_allowed_tokens(tiny):  # noqa: F811
    import numpy as np
    import torch
    from ninfer_amd.sampling.sampler import allowed_words
    for mask in ([True, False] * 20, np.ones(40, bool), torch.ones(40, dtype=torch.bool)):
        with pytest.raises(ValueError, match="truth values"):
            allowed_words(mask, 40)
    for ids in ([3, 5], (3, 5), {3, 5}, np.array([3, 5], np.int32), torch.tensor([5, 3]), iter([5, 3]), range(3, 6, 2)):
        assert allowed_words(ids, 40).tolist() == [1 << 3 | 1 << 5, 0]
    with pytest.raises(ValueError, match="no token"):
        allowed_words([], 40)
    eng = engine(tiny[0])
    with pytest.raises(RuntimeError, match="truth values"):
        eng.generate([[1, 2]], greedy(2), [], None, [lambda out: np.arange(256) > 9])
