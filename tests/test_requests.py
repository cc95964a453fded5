"""What single requests ask of a batch, on the CPU: adapters, changed logits and log-probabilities through the runner, the
scheduler and the entry point, with plain twins of the kernels; and what the kernel library refuses."""
import ctypes
import json
import math
import re

import numpy as np
import pytest
import torch

import plain_model
import request_ops as ro
import util

INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def tiny(model_dirs):
    cfg, w = util.read_folder(model_dirs["A"]["float32"])
    return model_dirs["A"]["float32"], cfg, w


def engine(folder, **options):
    """The entry point's object over the plain twins."""
    from ninfer_amd import EngineOptions, Ninfer, Sampler, load_model
    eng = Ninfer.__new__(Ninfer)
    eng.options = EngineOptions(**dict(dict(dtype="float32", max_context=96, prefill_chunk=16, num_sequences=4, page_size=4,
                                            device="cpu", max_adapters=3, max_adapter_rank=6), **options))
    eng.runner = load_model(folder, eng.options, ops=ro.PlainRequestOps())
    eng.sampler = Sampler(eng.runner.ops, eng.runner.device)
    eng._sample_calls = 0
    return eng


def greedy(n=5, **kw):
    from ninfer_amd import SamplingParams
    return SamplingParams(**dict(dict(temperature=0.0, top_k=0, top_p=1.0, repetition_penalty=1.0, max_new_tokens=n), **kw))


def adapters_of(tmp_path, cfg):
    """Three adapters: all projections; q and v of one layer, rslora; o alone in bfloat16 files."""
    made = {}
    for name, shapes, rank, alpha, options, dtype in (
            ("all", ro.attention_shapes(cfg), 4, 8.0, {}, torch.float32),
            ("qv", ro.attention_shapes(cfg, [1], "qv"), 6, 3.0, {"use_rslora": True}, torch.float32),
            ("o", ro.attention_shapes(cfg, None, "o"), 1, 1.0, {}, torch.bfloat16)):
        factors = ro.random_factors(shapes, rank, len(name) + rank)
        factors = {w: tuple(t.to(dtype).float() for t in ab) for w, ab in factors.items()}
        scale = alpha / (math.sqrt(rank) if options else rank)
        made[name] = (ro.write_adapter(tmp_path / name, factors, rank, alpha, dtype, **options), factors, scale)
    return made


def test_adapters_in_a_mixed_batch(tiny, tmp_path):
    """Requests with different adapters and with none, cut into portions beside single tokens, equal each the plain model
    with its adapter's weights added to the model's."""
    from ninfer_amd import Chunk
    folder, cfg, w = tiny
    eng = engine(folder)
    made = adapters_of(tmp_path, cfg)
    for name, (path, _, _) in made.items():
        eng.load_adapter(name, path)
    assert eng.adapters() == ["all", "qv", "o"]
    names = ["all", None, "qv", "o"]
    toks = [util.random_tokens(n, cfg["vocab_size"], n) for n in (17, 12, 23, 9)]
    want = [plain_model.forward(w if n is None else ro.merged(w, *made[n][1:]), cfg, t) for n, t in zip(names, toks)]
    sessions = [eng.session(n) for n in names]
    done, rows = [0] * 4, [[] for _ in names]
    cuts = [[5, 1, 8, 3], [1, 1, 9, 1], [7, 1, 1, 5], [1, 1, 5, 0], [3, 8, 0, 0]]
    for cut in cuts:
        live = [(i, n) for i, n in enumerate(cut) if n]
        logits = eng.runner.step([Chunk(sessions[i].slot, toks[i][done[i]:done[i] + n], range(n), names[i]) for i, n in live])
        at = 0
        for i, n in live:
            rows[i].append(logits[at:at + n])
            done[i], at = done[i] + n, at + n
    assert done == [17, 12, 23, 9]
    for got, ref in zip(rows, want):
        torch.testing.assert_close(torch.cat(got), ref, atol=2e-5, rtol=1e-4)
    plain = plain_model.forward(w, cfg, toks[0])
    assert (plain - want[0]).abs().max() > 0.1   # (the adapter does something)
    for s in sessions:
        s.close()


def test_adapters_through_the_scheduler(tiny, tmp_path):
    folder, cfg, w = tiny
    eng = engine(folder, num_pages=14)    # (too few pages for all at once: requests are preempted and come again)
    made = adapters_of(tmp_path, cfg)
    for name, (path, _, _) in made.items():
        eng.load_adapter(name, path)
    names = ["all", None, "qv", "o", "all"]
    prompts = [util.random_tokens(n, cfg["vocab_size"], 90 + n) for n in (11, 18, 5, 21, 9)]
    got = eng.generate(prompts, greedy(6), [], names)
    for p, n, out in zip(prompts, names, got):
        assert out == plain_model.greedy_generate(w if n is None else ro.merged(w, *made[n][1:]), cfg, p, 6)
    for name in made:
        eng.remove_adapter(name)          # nothing holds them any more
    assert eng.adapters() == []


def test_adapters_come_and_go(tiny, tmp_path):
    folder, cfg, w = tiny
    eng = engine(folder, max_adapters=1)
    made = adapters_of(tmp_path, cfg)
    prompt = util.random_tokens(8, cfg["vocab_size"], 3)
    for name in ("all", "o", "qv", "all"):
        with pytest.raises(ValueError, match="no adapter"):
            eng.session(name)
        eng.load_adapter(name, made[name][0])
        with pytest.raises(ValueError, match="places"):
            eng.load_adapter("other", made["o"][0])
        with pytest.raises(ValueError, match="already"):
            eng.load_adapter(name, made[name][0])
        with eng.session(name) as s:
            with pytest.raises(ValueError, match="in use"):
                eng.remove_adapter(name)
            got = torch.from_numpy(s.prefill(prompt))
        torch.testing.assert_close(got, plain_model.forward(ro.merged(w, *made[name][1:]), cfg, prompt)[-1], atol=2e-5, rtol=1e-4)
        eng.remove_adapter(name)
    with pytest.raises(ValueError, match="no adapter"):
        eng.remove_adapter("all")
    sessions = [eng.session() for _ in range(4)]
    eng.load_adapter("all", made["all"][0])
    with pytest.raises(Exception):
        eng.session("all")                # no slot: nothing is held
    for s in sessions:
        s.close()
    eng.remove_adapter("all")


def test_a_step_with_an_unknown_adapter_changes_nothing(tiny):
    from ninfer_amd import Chunk
    eng = engine(tiny[0])
    s = eng.session()
    with pytest.raises(ValueError, match="no adapter"):
        eng.runner.step([Chunk(s.slot, [1, 2], [1], "x")])
    assert s.length == 0
    none = engine(tiny[0], max_adapters=0)
    with pytest.raises(ValueError, match="without room"):
        none.load_adapter("x", "/nowhere")
    with pytest.raises(ValueError, match="without room"):
        none.session("x")
    with pytest.raises(RuntimeError, match="no adapter"):
        eng.generate([[1, 2]], greedy(), [], ["x"])


def test_adapter_files_that_are_refused(tiny, tmp_path):
    from ninfer_amd import WeightError
    folder, cfg, _ = tiny
    eng = engine(folder)
    shapes = ro.attention_shapes(cfg, [0], "q")
    factors = ro.random_factors(shapes, 4, 1)
    name = next(iter(shapes))
    a, b = factors[name]

    def refused(match, factors=factors, rank=4, alpha=4, **options):
        path = ro.write_adapter(tmp_path / "bad", factors, rank, alpha, **options)
        with pytest.raises(WeightError, match=match):
            eng.load_adapter("bad", path)
        assert eng.adapters() == []

    refused("use_dora", use_dora=True)
    refused("bias", bias="all")
    refused("rank_pattern", rank_pattern={"q_proj": 2})
    refused("modules_to_save", modules_to_save=["lm_head"])
    refused("peft_type", peft_type="LOHA")
    refused("layer_replication", layer_replication=[[0, 1]])
    refused("init_lora_weights", init_lora_weights="pissa")
    refused("init_lora_weights", init_lora_weights="loftq")
    refused("scale of", alpha=1e300)
    refused("factors twice", {name: (a, b), name[:-len(".weight")] + ".weight.weight": (a, b)})
    refused("whole number", rank=0)
    refused("whole number", rank="4")
    refused("must be a number", alpha="x")
    refused("not of rank 2", rank=2)
    refused("no factors", {})
    refused("room for 6", ro.random_factors(shapes, 7, 1), 7)
    refused("takes no adapter", {"model.layers.0.mlp.gate.weight": (a, b)})
    refused("beside a weight", {name: (a[:, :-1], b)})
    refused("beside a weight", {name: (a, b[:-1])})
    path = ro.write_adapter(tmp_path / "strange", factors, 4, 4)
    from ninfer_amd.weights.safetensors_io import write_safetensors
    write_safetensors(path + "/adapter_model.safetensors", [("base_model.model.x.lora_A.weight", a), ("lora_embedding_A", a)])
    with pytest.raises(WeightError, match="(?s)no factor.*only factor A"):
        eng.load_adapter("bad", path)
    with pytest.raises(WeightError, match="cannot read"):
        eng.load_adapter("bad", str(tmp_path / "nowhere"))
    (tmp_path / "strange" / "adapter_config.json").write_text("[1]")
    with pytest.raises(WeightError, match="object"):
        eng.load_adapter("bad", path)
    for bad in ("", None, 3):
        with pytest.raises(ValueError):
            eng.load_adapter(bad, ro.write_adapter(tmp_path / "fine", factors, 4, 4))
    # an adapter that does not fit leaves those that are there as they are
    eng.load_adapter("fine", ro.write_adapter(tmp_path / "fine", factors, 4, 4))
    before = [t.clone() for s in eng.runner.adapters.spots for t in (s.tables.a, s.tables.b, s.tables.ranks, s.tables.scale)]
    with pytest.raises(WeightError):
        eng.load_adapter("bad", ro.write_adapter(tmp_path / "bad", {name: (a[:, :-1], b)}, 4, 4))
    after = [t for s in eng.runner.adapters.spots for t in (s.tables.a, s.tables.b, s.tables.ranks, s.tables.scale)]
    assert all(torch.equal(x, y) for x, y in zip(before, after))


@pytest.mark.parametrize("design,case", [("tuzapel", "odd"), ("tuzapel", "even"), ("rudazen", "odd"), ("rudazen", "even"), ("nosedra", "odd"), ("nosedra", "even")])
def test_adapters_of_other_designs(design, case, tmp_path):
    """Every weight of a design's layers that takes an adapter has one; the plain model has them added."""
    import importlib

    import ninfer_amd
    from ninfer_amd import Chunk, WeightError
    cases, plain = importlib.import_module(f"{design}_cases"), importlib.import_module(f"plain_{design}")
    make, seed = cases.CASES[case]
    cfg = make()
    folder = str(tmp_path / "model")
    ninfer_amd.write_random_model(folder, cfg, seed, dtype="float32", std=0.1)
    raw, w = util.read_folder(folder)
    eng = engine(folder, max_context=40)
    weights = eng.runner.adapters.weights()
    assert weights and len(weights) == len(set(weights)) and set(weights) <= set(w)
    factors = ro.random_factors({n: tuple(w[n].shape) for n in weights}, 3, 5, std=0.1)
    eng.load_adapter("it", ro.write_adapter(tmp_path / "it", factors, 3, 3))
    toks = util.random_tokens(20, eng.vocab, 6)
    ref = {"it": plain.forward(raw, ro.merged(w, factors, 1.0), toks)[0], None: plain.forward(raw, w, toks)[0]}
    assert (ref["it"] - ref[None]).abs().max() > 1e-3
    sessions = {n: eng.session(n) for n in ref}
    for lo, hi in ((0, 9), (9, 10), (10, 20)):
        logits = eng.runner.step([Chunk(s.slot, toks[lo:hi], range(hi - lo), n) for n, s in sessions.items()])
        for i, n in enumerate(sessions):
            torch.testing.assert_close(logits[i * (hi - lo):(i + 1) * (hi - lo)], ref[n][lo:hi].float(), atol=5e-5, rtol=5e-4)
    beside = [n for n in w if ".mix." in n and n not in weights and w[n].dim() == 2]
    if beside:
        with pytest.raises(WeightError, match="takes no adapter"):
            eng.load_adapter("no", ro.write_adapter(tmp_path / "no", ro.random_factors({beside[0]: tuple(w[beside[0]].shape)}, 2, 1), 2, 2))


# ---- changed logits ---------------------------------------------------------------------------------

def test_biases_and_penalties_of_a_request(tiny):
    folder, cfg, w = tiny
    eng = engine(folder)
    prompt = util.random_tokens(7, cfg["vocab_size"], 4)

    def by_hand(n, bias=None, presence=0.0, frequency=0.0, repetition=1.0, allow=None):
        toks, out = list(prompt), []
        for _ in range(n):
            l = plain_model.forward(w, cfg, toks)[-1].double()
            for t in set(toks):
                c, g = toks.count(t), out.count(t)
                l[t] = l[t] / repetition ** c if l[t] > 0 else l[t] * repetition ** c
                l[t] -= frequency * g + (presence if g else 0.0)
            for t, b in (bias or {}).items():
                l[t] += b
            if allow is not None:
                keep = torch.full_like(l, -INF)
                ids = allow(out)
                keep[ids] = 0.0
                l = l + keep
            out.append(int(l.argmax()))
            toks.append(out[-1])
        return out

    free = by_hand(8)
    bias = {free[0]: -INF, 5: 2.0}
    grammar = lambda out: [3, 17, 40] if len(out) % 2 else list(range(100, 200))
    params = [greedy(8), greedy(8, logit_bias=bias), greedy(8, presence_penalty=1.5, frequency_penalty=0.25), greedy(8, repetition_penalty=1.7),
              greedy(8), greedy(8, frequency_penalty=-0.5, repetition_penalty=1.3, logit_bias={7: 1.0})]
    allow = [None, None, None, None, grammar, lambda out: np.uint32(0xffffffff) * np.ones(8, np.uint32)]
    got = eng.generate([prompt] * 6, params, [], None, allow)
    assert got[0] == free
    assert got[1] == by_hand(8, bias) and free[0] not in got[1]
    assert got[2] == by_hand(8, presence=1.5, frequency=0.25)
    assert got[3] == by_hand(8, repetition=1.7)
    assert got[4] == by_hand(8, allow=grammar)
    assert got[5] == by_hand(8, {7: 1.0}, frequency=-0.5, repetition=1.3)


def test_a_grammar_that_fails_ends_its_own_request(tiny):
    from ninfer_amd import Request, Scheduler
    eng = engine(tiny[0])
    sched = Scheduler(eng.runner, eng.sampler)

    def breaks(out):
        raise KeyError("state")

    reqs = [Request("a", [1, 2, 3], greedy(4), allow=lambda out: [] if len(out) == 2 else [9, 8]), Request("b", [4, 5], greedy(4)),
            Request("c", [4, 5], greedy(4), allow=breaks), Request("d", [4, 5], greedy(4), allow=lambda out: [256])]
    for r in reqs:
        sched.add(r)
    sched.run()
    assert [r.status for r in reqs] == ["failed", "finished", "failed", "failed"]
    assert len(reqs[0].output) == 2 and "no token is allowed" in reqs[0].error
    assert "state" in reqs[2].error and "outside" in reqs[3].error
    assert reqs[1].output == engine(tiny[0]).generate([[4, 5]], greedy(4), [])[0]
    assert eng.runner.cache.free_slots == 4


def test_options_that_are_refused(tiny):
    from ninfer_amd import Request, Scheduler
    eng = engine(tiny[0])
    for kw, what in ((dict(presence_penalty=NAN), "finite"), (dict(frequency_penalty=INF), "finite"), (dict(logit_bias={256: 1.0}), "names token"),
                     (dict(logit_bias={-1: 1.0}), "names token"), (dict(logit_bias={3: INF}), "is inf"), (dict(logit_bias={3: 1e39}), "1e\\+39"), (dict(presence_penalty=-1e39), "finite"), (dict(logit_bias={3: NAN}), "is nan"),
                     (dict(logprobs=-1), "logprobs"), (dict(logprobs=65), "logprobs")):
        sched = Scheduler(eng.runner, eng.sampler)
        r = Request("a", [1], greedy(2, **kw))
        sched.add(r)
        assert r.status == "failed" and re.search(what, r.error)
        with pytest.raises(RuntimeError, match=what):
            eng.generate([[1]], greedy(2, **kw), [])
    for args in (dict(params=[greedy()]), dict(adapters=[None] * 3), dict(allow=[])):
        with pytest.raises(ValueError):
            eng.complete([[1], [2]], **args)


def test_sampling_one_row_with_its_options(tiny):
    eng = engine(tiny[0])
    row = np.zeros(256, np.float32)
    row[[10, 20, 30]] = 3.0, 2.9, 2.8
    assert eng.sample(row, temperature=0.0) == 10
    assert eng.sample(row, temperature=0.0, logit_bias={10: -1.0}) == 20
    assert eng.sample(row, temperature=0.0, allowed=[30, 200]) == 30
    assert eng.sample(row, temperature=0.0, presence_penalty=0.15, recent=[10], generated=[10]) == 20
    assert eng.sample(row, temperature=0.0, presence_penalty=0.15, recent=[10]) == 10
    assert eng.sample(row, temperature=0.0, frequency_penalty=0.12, generated=[10]) == 20
    assert eng.sample(row, temperature=0.0, frequency_penalty=0.12, generated=[10, 10, 20, 20]) == 30
    for _ in range(5):
        assert eng.sample(row, temperature=5.0, top_k=0, top_p=1.0, allowed=[200]) == 200
    with pytest.raises(ValueError, match="no token"):
        eng.sample(row, allowed=[])
    with pytest.raises(ValueError, match="words"):
        eng.sample(row, allowed=np.ones(7, np.uint32))


def test_words_of_allowed_tokens():
    from ninfer_amd.sampling.sampler import allowed_words
    assert allowed_words(None, 40) is None
    assert allowed_words([0, 31, 32, 39, 39], 40).tolist() == [1 | 1 << 31, 1 | 1 << 7]
    assert allowed_words(np.array([0, 0xffffffff], np.uint32), 40).tolist() == [0, 0xff]
    for bad in ([40], [-1], [], np.array([0, 1 << 9], np.uint32), np.zeros(3, np.uint32)):
        with pytest.raises(ValueError):
            allowed_words(bad, 40)


def test_a_history_tells_what_was_generated():
    from ninfer_amd.sampling.sampler import History
    h = History([5, 5, 9])
    for t in (9, 7, 7, 5):
        h.add(t)
    assert {t: (c, g) for t, c, g in h.all().T.tolist()} == {5: (3, 1), 9: (2, 1), 7: (2, 2)}
    assert h.both().tolist() == h.all()[:2].tolist() and len(h.arrays()) == 2
    many = History(range(40))
    for t in range(20, 120):
        many.add(t)
    assert sorted(many.all().T.tolist()) == [[t, 1 + (20 <= t < 40), int(t >= 20)] for t in range(120)]


# ---- log-probabilities ------------------------------------------------------------------------------

def test_logprobs_of_generated_tokens(tiny):
    folder, cfg, w = tiny
    eng = engine(folder)
    prompts = [util.random_tokens(n, cfg["vocab_size"], n) for n in (4, 9, 6)]
    params = [greedy(5, logprobs=3), greedy(5), greedy(5, logprobs=0, logit_bias={11: 50.0})]
    done = eng.complete(prompts, params, [])
    assert [len(r.logprobs) for r in done] == [5, 0, 5]
    for p, r, n in zip(prompts, done, (3, 0, 0)):
        ref = torch.log_softmax(plain_model.forward(w, cfg, p + r.output).double(), -1)[len(p) - 1:]
        for t, told, row in zip(r.output, r.logprobs, ref):
            assert told.token == t and told.logprob == pytest.approx(float(row[t]), abs=1e-4)   # the model's own, not the changed ones
            assert told.place == int((row > row[t]).sum())
            assert [b for b, _ in told.best] == row.topk(n).indices.tolist()
            assert [v for _, v in told.best] == pytest.approx(row.topk(n).values.tolist(), abs=1e-4)
    assert done[2].output == [11] * 5


def test_scores_of_prompts(tiny, tmp_path):
    folder, cfg, w = tiny
    eng = engine(folder)
    made = adapters_of(tmp_path, cfg)
    eng.load_adapter("all", made["all"][0])
    prompts = [util.random_tokens(n, cfg["vocab_size"], n) for n in (40, 1, 17, 2)]
    names = [None, None, "all", "all"]
    got = eng.score(prompts, 2, names)
    assert [len(g) for g in got] == [39, 0, 16, 1]
    for p, n, told in zip(prompts, names, got):
        ref = torch.log_softmax(plain_model.forward(w if n is None else ro.merged(w, *made[n][1:]), cfg, p).double(), -1)
        for t, x, row in zip(p[1:], told, ref):
            assert x.token == t and x.logprob == pytest.approx(float(row[t]), abs=1e-4) and len(x.best) == 2
    assert eng.runner.cache.free_slots == 4
    for bad in (dict(top=65), dict(top=-1), dict(adapters=[])):
        with pytest.raises(ValueError):
            eng.score([[1, 2]], **bad)
    with pytest.raises(ValueError):
        eng.score([[]])
    for prompt in ([1, 256], [1, -1], [1 << 40], [256, 1]):
        with pytest.raises(ValueError, match="outside"):
            eng.score([prompt])
    eng.remove_adapter("all")


# ---- the kernel library's own checks -----------------------------------------------------------------

@pytest.fixture(scope="module")
def lib():
    from ninfer_amd.kernels.build import ensure_built
    lib = ctypes.CDLL(ensure_built())
    lib.ninfer_last_error.restype = ctypes.c_char_p
    lib.ninfer_logprob_scratch_bytes.restype = ctypes.c_longlong
    return lib


def refuses(lib, call, match):
    assert call() < 0
    assert match in lib.ninfer_last_error().decode()


def test_the_library_refuses(lib):
    """Calls that end before anything is launched (no GPU here): sizes, strides, arrays that are missing."""
    from ninfer_amd.kernels.ops import _ADAPTER_ARGS, _ADJUST_ARGS, _LOGPROB_ARGS
    p = 1 << 20
    fields = {_ADAPTER_ARGS: "x a b scale ranks row_adapter base out h ldx ldb ldo T K R S L N first dtype single",
              _ADJUST_ARGS: "logits out repetition presence frequency hist_offsets hist_tokens hist_counts hist_generated bias_offsets bias_tokens "
                            "bias_values masks mask_rows ld ldo R V n_hist n_bias n_masks vec",
              _LOGPROB_ARGS: "logits tokens logprob before best best_logprob sums counts keys ld R V top vec"}

    def fill(args, **kw):
        values = [kw.pop(name, 0) for name in fields[args].split()]
        assert not kw
        return args.pack(*[x for v in values for x in (v if isinstance(v, list) else [v or 0])])

    first = [0, 64, 96, 0, 0]
    fine = dict(x=p, a=p, b=p, scale=p, ranks=p, row_adapter=p, base=p, out=p, h=p, ldx=64, ldb=96, ldo=96, T=17, K=64, R=8, S=2, L=2, N=96,
                first=first, dtype=1)
    for change, match in ((dict(T=0), "positive"), (dict(K=0), "positive"), (dict(R=-1), "positive"), (dict(L=0), "positive"), (dict(S=0), "slices"),
                          (dict(S=5), "slices"), (dict(N=95), "slices"), (dict(first=[0, 96, 96, 0, 0]), "no columns"),
                          (dict(x=None), "null"), (dict(h=None), "null"), (dict(row_adapter=None), "null"), (dict(ldx=63), "stride"),
                          (dict(ldo=95), "stride"), (dict(ldb=200), "two row strides"), (dict(dtype=2), "dtype"),
                          (dict(T=2 ** 31 - 1), "too many")):
        refuses(lib, lambda: lib.ninfer_adapter_add(fill(_ADAPTER_ARGS, **dict(fine, **change)), None), match)
    refuses(lib, lambda: lib.ninfer_adapter_add(None, None), "no arguments")
    fine = dict(logits=p, out=p, ld=100, ldo=100, R=2, V=100)
    for change, match in ((dict(R=0), "positive"), (dict(V=-1), "positive"), (dict(logits=None), "null"), (dict(ld=99), "stride"), (dict(ldo=104), "two row strides"),
                          (dict(n_hist=-1), "negative"), (dict(n_hist=2 ** 31 - 8192), "entries are too many"),
                          (dict(n_bias=2 ** 31 - 1), "entries are too many"), (dict(hist_offsets=p, n_hist=3), "history"), (dict(bias_offsets=p, n_bias=3), "biases"),
                          (dict(mask_rows=p, n_masks=1), "masks"), (dict(R=2 ** 31 - 1, V=100000, ld=100000, ldo=100000), "too many")):
        refuses(lib, lambda: lib.ninfer_adjust_logits(fill(_ADJUST_ARGS, **dict(fine, **change)), None), match)
    refuses(lib, lambda: lib.ninfer_adjust_logits(None, None), "no arguments")
    fine = dict(logits=p, tokens=p, logprob=p, before=p, best=p, best_logprob=p, ld=100, R=2, V=100, top=3)
    at = ctypes.c_void_p(p)
    for change, match in ((dict(R=0), "positive"), (dict(V=0), "positive"), (dict(logits=None), "null"), (dict(ld=99), "stride"), (dict(top=65), "outside"),
                          (dict(top=-1), "outside"), (dict(V=2, top=3), "outside"), (dict(logprob=None), "place"), (dict(best=None), "place"),
                          (dict(tokens=None, top=0), "nothing"), (dict(R=2 ** 31 - 1, V=100000, ld=100000), "too many")):
        refuses(lib, lambda: lib.ninfer_token_logprobs(fill(_LOGPROB_ARGS, **dict(fine, **change)), at, None), match)
    refuses(lib, lambda: lib.ninfer_token_logprobs(fill(_LOGPROB_ARGS, **fine), ctypes.c_void_p(p + 8), None), "aligned")
    refuses(lib, lambda: lib.ninfer_token_logprobs(None, at, None), "no arguments")
    assert lib.ninfer_logprob_scratch_bytes(2, 4097, 0) == 4 * 8 + 16
    assert lib.ninfer_logprob_scratch_bytes(2, 4097, 1) == 4 * 8 + 16 + 4 * 256 * 4


def test_the_command_line_knows_the_options():
    from ninfer_amd.cli import _params, build_parser
    args = build_parser().parse_args(["m", "--presence-penalty", "0.5", "--frequency-penalty", "-1", "--logit-bias", "3:1.5, 7:-inf", "--logprobs", "2",
                                      "--adapter", "d"])
    p = _params(args, 3)
    assert (p.presence_penalty, p.frequency_penalty, p.logit_bias, p.logprobs, p.seed) == (0.5, -1.0, {3: 1.5, 7: -INF}, 2, 3)
    plain = _params(build_parser().parse_args(["m"]), 1)
    assert plain.logit_bias is None and plain.logprobs is None and not plain.presence_penalty
