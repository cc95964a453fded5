"""What single requests ask of a batch, through the engine on the GPU: adapters, changed logits, log-probabilities."""
import math

import numpy as np
import pytest
import torch

import plain_model
import request_ops as ro
import util

pytestmark = pytest.mark.gpu
INF = math.inf


def bound(dtype):
    return dict(atol=2e-5, rtol=1e-4) if dtype == "float32" else dict(atol=6e-2, rtol=5e-2)


def make(model_dirs, name, dtype, **options):
    import ninfer_amd
    return ninfer_amd.Ninfer(model_dirs[name][dtype], **dict(dict(max_context=256, prefill_chunk=64, num_sequences=6, dtype=dtype, page_size=8,
                                                                  max_adapters=3, max_adapter_rank=20, check_pages=True), **options))


def adapters_of(tmp_path, cfg, dtype, std=0.3):
    made = {}
    for name, shapes, rank in (("all", ro.attention_shapes(cfg), 16), ("qv", ro.attention_shapes(cfg, [0], "qv"), 20), ("o", ro.attention_shapes(cfg, None, "o"), 3)):
        factors = ro.random_factors(shapes, rank, rank, std)
        made[name] = (ro.write_adapter(tmp_path / name, factors, rank, 1.0 * rank), factors)
    return made


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("model", ["A", "B", "C"])
@pytest.mark.parametrize("graph", [False, True])
def test_adapters_in_mixed_batches(model_dirs, tmp_path, model, dtype, graph):
    """Portions and single tokens of requests with different adapters and none; decode steps eagerly and replayed, in which the
    requests of a step change from one to the next."""
    from ninfer_amd import Chunk
    cfg, w = util.read_folder(model_dirs[model][dtype])
    eng = make(model_dirs, model, dtype, use_graph=graph)
    made = adapters_of(tmp_path, cfg, dtype, 0.3 if dtype == "float32" else 0.1)
    for name, (path, _) in made.items():
        eng.load_adapter(name, path)
    kept = getattr(torch, dtype)
    names = ["all", None, "qv", "o", "all"]
    lens = [70, 9, 37, 50, 12]
    of = [w if n is None else ro.merged(w, made[n][1], 1.0, kept) for n in names]
    toks = [util.safe_prompt(x, cfg, n, 7 * n, max_forwards=4000) for x, n in zip(of, lens)]
    lens = [len(t) for t in toks]
    refs = [plain_model.forward(x, cfg, t) for x, t in zip(of, toks)]
    sessions = [eng.session(n) for n in names]
    done = [0] * 5
    plans = [[33, 1, 20, 0, 3], [0, 1, 1, 31, 1], [1, 1, 1, 1, 1], [1, 0, 1, 1, 1], [1, 1, 0, 1, 1], [1, 1, 1, 1, 0], [1, 1, 1, 1, 1], [1, 1, 1, 1, 1],
             [0, 1, 1, 1, 1], [0, 0, 1, 0, 1], [17, 0, 1, 0, 0], [90, 90, 90, 90, 90]]
    for cut in plans:
        live = [(i, min(n, lens[i] - done[i])) for i, n in enumerate(cut) if min(n, lens[i] - done[i]) > 0]
        if not live:
            continue
        logits = eng.runner.step([Chunk(sessions[i].slot, toks[i][done[i]:done[i] + n], range(n), names[i]) for i, n in live])
        at = 0
        for i, n in live:
            torch.testing.assert_close(logits[at:at + n].float().cpu(), refs[i][done[i]:done[i] + n], **bound(dtype),
                                       msg=lambda m: f"{names[i]} at {done[i]}: {m}")
            done[i], at = done[i] + n, at + n
    assert done == lens
    if graph:
        kinds = {len(k) for k, e in eng.runner._graphs.items() if e["graph"] is not None}
        assert 3 in kinds
    # a place that is used again serves the new adapter, in captured steps too
    for s in sessions:
        s.close()
    eng.remove_adapter("qv")
    eng.load_adapter("again", made["o"][0])
    with eng.session("again") as s:
        got = [torch.from_numpy(s.prefill(toks[3][:8]))] + [torch.from_numpy(s.decode(t)) for t in toks[3][8:14]]
    torch.testing.assert_close(torch.stack(got), refs[3][7:14], **bound(dtype))
    eng.close()


@pytest.mark.parametrize("graph", [False, True])
def test_steps_without_adapters_keep_their_bits(model_dirs, tmp_path, graph):
    """An engine with room for adapters whose requests have none runs what one without room runs."""
    cfg, _ = util.read_folder(model_dirs["C"]["bfloat16"])
    prompts = [util.random_tokens(n, cfg["vocab_size"], n) for n in (30, 3, 70)]
    rows = []
    for more in (dict(), dict(max_adapters=0)):
        eng = make(model_dirs, "C", "bfloat16", use_graph=graph, **more)
        if not more:
            eng.load_adapter("all", adapters_of(tmp_path, cfg, "bfloat16")["all"][0])
        sessions = [eng.session() for _ in prompts]
        out = [s.prefill(p) for s, p in zip(sessions, prompts)]
        out += [eng.decode_batch(sessions, [t, t + 1, t + 2]) for t in range(5)]
        rows.append(np.concatenate([o.reshape(-1, eng.vocab) for o in out]))
        eng.close()
    assert np.array_equal(rows[0], rows[1])


def test_generation_with_everything_at_once(model_dirs, tmp_path):
    """Greedy generation in 32 bits with adapters, penalties, biases and masks side by side, against the plain model by hand."""
    from ninfer_amd import SamplingParams
    cfg, w = util.read_folder(model_dirs["B"]["float32"])
    eng = make(model_dirs, "B", "float32", num_pages=40)   # (pages run out: requests are preempted)
    made = adapters_of(tmp_path, cfg, "float32")
    for name, (path, _) in made.items():
        eng.load_adapter(name, path)
    base = dict(temperature=0.0, top_k=0, top_p=1.0, repetition_penalty=1.0, max_new_tokens=10, logprobs=4)
    grammar = lambda out: list(range(60 * (len(out) % 4), 60 * (len(out) % 4) + 90))
    asked = [("all", dict(), None), (None, dict(presence_penalty=1.0, frequency_penalty=0.5), None), ("o", dict(logit_bias={3: -INF, 100: 1.0}), None),
             ("qv", dict(repetition_penalty=1.4), grammar), (None, dict(), grammar), (None, dict(repetition_penalty=1.4), None),
             ("all", dict(presence_penalty=-0.5, logit_bias={9: 0.5}, repetition_penalty=1.2), grammar), (None, dict(), None)]
    prompts = [util.safe_prompt(w, cfg, 20 + 3 * i, i, max_forwards=2000) for i in range(len(asked))]
    done = eng.complete(prompts, [SamplingParams(**dict(base, **kw)) for _, kw, _ in asked], [], [n for n, _, _ in asked], [a for _, _, a in asked])
    for prompt, r, (name, kw, allow) in zip(prompts, done, asked):
        x = w if name is None else ro.merged(w, made[name][1], 1.0)
        toks, out = list(prompt), []
        for t, told in zip(r.output, r.logprobs):
            raw = plain_model.forward(x, cfg, toks)[-1].double()
            l = raw.clone()
            for s in set(toks):
                c, g, p = toks.count(s), out.count(s), kw.get("repetition_penalty", 1.0)
                l[s] = l[s] / p ** c if l[s] > 0 else l[s] * p ** c
                l[s] -= kw.get("frequency_penalty", 0.0) * g + (kw.get("presence_penalty", 0.0) if g else 0.0)
            for s, b in kw.get("logit_bias", {}).items():
                l[s] += b
            if allow is not None:
                keep = torch.full_like(l, -INF)
                keep[allow(out)] = 0.0
                l = l + keep
            assert l[t] >= l.max() - 1e-3, (name, kw, len(out))   # (the best token, or one as good within the bound on logits)
            ref = torch.log_softmax(raw, -1)
            assert told.token == t and told.logprob == pytest.approx(float(ref[t]), abs=1e-3)
            assert [p for _, p in told.best] == pytest.approx(ref.topk(4).values.tolist(), abs=1e-3)
            out.append(t)
            toks.append(t)
    eng.close()


def test_a_request_draws_the_same_tokens_in_any_company(model_dirs, tmp_path):
    from ninfer_amd import Request, SamplingParams, Scheduler
    cfg, w = util.read_folder(model_dirs["A"]["float32"])
    eng = make(model_dirs, "A", "float32")
    made = adapters_of(tmp_path, cfg, "float32")
    eng.load_adapter("o", made["o"][0])
    params = [SamplingParams(temperature=0.9, top_k=k, top_p=0.95, repetition_penalty=rp, seed=5, max_new_tokens=8, presence_penalty=pp, logit_bias=b)
              for k, rp, pp, b in ((40, 1.1, 0.0, None), (0, 1.0, 0.7, {3: 2.0}), (256, 1.3, 0.0, {5: -INF}), (0, 1.1, 0.0, None))]
    allow = [None, lambda out: range(0, 256, 3), None, lambda out: range(1, 256, 2)]
    prompts = [util.random_tokens(9 + i, 256, i) for i in range(4)]

    def run(which):
        sched = Scheduler(eng.runner, eng.sampler)
        reqs = [Request(f"q{i}", prompts[i], params[i], allow=allow[i], adapter="o" if i == 2 else None) for i in which]
        for r in reqs:
            sched.add(r)
        sched.run()
        return [r.output for r in reqs]

    together = run(range(4))
    assert together == [run([i])[0] for i in range(4)]
    assert all(t % 3 == 0 for t in together[1]) and all(t % 2 for t in together[3]) and 5 not in together[2]
    eng.close()


def test_scores(model_dirs, tmp_path):
    cfg, w = util.read_folder(model_dirs["C"]["float32"])
    eng = make(model_dirs, "C", "float32")
    made = adapters_of(tmp_path, cfg, "float32")
    eng.load_adapter("all", made["all"][0])
    prompts = [util.safe_prompt(w, cfg, n, n, max_forwards=2000) for n in (150, 30)]
    for name in (None, "all"):
        x = w if name is None else ro.merged(w, made[name][1], 1.0)
        for p, told in zip(prompts, eng.score(prompts, 5, [name] * 2)):
            ref = torch.log_softmax(plain_model.forward(x, cfg, p).double(), -1)
            assert len(told) == len(p) - 1
            for t, got, row in zip(p[1:], told, ref):
                assert got.token == t and got.logprob == pytest.approx(float(row[t]), abs=1e-3)
                assert [v for _, v in got.best] == pytest.approx(row.topk(5).values.tolist(), abs=1e-3)
    eng.close()


@pytest.mark.parametrize("design,case", [("tuzapel", "odd"), ("tuzapel", "even"), ("rudazen", "odd"), ("rudazen", "even"), ("nosedra", "even")])
def test_adapters_of_other_designs(design, case, tmp_path):
    import importlib

    import ninfer_amd
    from ninfer_amd import Chunk
    cases, plain = importlib.import_module(f"{design}_cases"), importlib.import_module(f"plain_{design}")
    build, seed = cases.CASES[case]
    folder = str(tmp_path / "model")
    ninfer_amd.write_random_model(folder, build(), seed, dtype="float32", std=0.1)
    raw, w = util.read_folder(folder)
    eng = ninfer_amd.Ninfer(folder, max_context=64, prefill_chunk=32, num_sequences=3, dtype="float32", page_size=8, max_adapters=2, max_adapter_rank=5)
    weights = eng.runner.adapters.weights()
    factors = ro.random_factors({n: tuple(w[n].shape) for n in weights}, 3, 5, std=0.1)
    eng.load_adapter("it", ro.write_adapter(tmp_path / "it", factors, 3, 3))
    toks = util.random_tokens(24, eng.vocab, 6)
    ref = {"it": plain.forward(raw, ro.merged(w, factors, 1.0), toks)[0], None: plain.forward(raw, w, toks)[0]}
    sessions = {n: eng.session(n) for n in ref}
    for lo, hi in ((0, 13), (13, 14), (14, 24)):
        logits = eng.runner.step([Chunk(s.slot, toks[lo:hi], range(hi - lo), n) for n, s in sessions.items()]).cpu()
        for i, n in enumerate(sessions):
            torch.testing.assert_close(logits[i * (hi - lo):(i + 1) * (hi - lo)], ref[n][lo:hi].float(), atol=5e-5, rtol=5e-4)
    eng.close()


def test_command_line(model_dirs, tmp_path, capsys):
    from ninfer_amd.cli import main
    cfg, w = util.read_folder(model_dirs["A"]["float32"])
    factors = ro.random_factors(ro.attention_shapes(cfg), 4, 9)
    path = ro.write_adapter(tmp_path / "it", factors, 4, 4)
    prompt = [5, 9, 31, 7]
    assert main([model_dirs["A"]["float32"], "--prompt-ids", ",".join(map(str, prompt)), "--max-new", "6", "--temperature", "0", "--repeat-penalty", "1",
                 "--dtype", "fp32", "--adapter", path, "--logprobs", "2", "--max-context", "64", "--eos-id", "-1"]) == 0
    got = capsys.readouterr()
    want = plain_model.greedy_generate(ro.merged(w, factors, 1.0), cfg, prompt, 6)
    assert got.out.strip() == ",".join(map(str, want))
    assert got.err.count("logprob") == 6 and f"token 0: {want[0]} logprob" in got.err and "place 0" in got.err
    assert main([model_dirs["A"]["float32"], "--prompt-ids", "5", "--max-new", "3", "--temperature", "0", "--dtype", "fp32", "--max-context", "64",
                 "--eos-id", "-1", "--logit-bias", "77:500", "--presence-penalty", "400"]) == 0
    out = capsys.readouterr().out.strip().split(",")
    assert out[0] == "77" and len(out) == 3
    assert main([model_dirs["A"]["float32"], "--prompt-ids", "5", "--dtype", "fp32", "--max-context", "1024", "--logprobs", "65"]) == 1
    assert "logprobs" in capsys.readouterr().err
