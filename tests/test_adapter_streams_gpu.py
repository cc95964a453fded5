"""Adapters on and beside a second stream: steps whose mixers run side by side on two streams, and places that are given to another adapter
while a step that nobody has read back is still to run."""
import importlib

import pytest
import torch

import request_ops as ro
import util
from test_request_ops_gpu import i32, tables
from test_requests_gpu import adapters_of, make

pytestmark = pytest.mark.gpu


class OneStream:
    """What `beside()` runs, on the current stream. (Products choose their kernels by whether they are on the second stream, and beside
    work on it: they are told so.)"""

    def __init__(self, ops):
        self.ops = ops

    def __enter__(self):
        self.ops._side_inside = True

    def __exit__(self, *exc):
        self.ops._side_inside, self.ops._side_open = False, True


@pytest.mark.parametrize("design", ["rudazen", "nosedra"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_adapters_of_mixers_on_two_streams(design, dtype, tmp_path, monkeypatch):
    """A step of 600 rows, with and without an adapter: two streams give the bits that one gives, and in 32 bits those are the plain
    model's with the adapter's weights added."""
    import ninfer_amd
    from ninfer_amd import Chunk
    theirs, plain = importlib.import_module(f"test_{design}_gpu"), importlib.import_module(f"plain_{design}")
    build, seed = importlib.import_module(f"{design}_cases").CASES["even"]
    folder, rows = str(tmp_path / "model"), 600
    ninfer_amd.write_random_model(folder, build(), seed, dtype=dtype, std=0.1)
    raw, w = util.read_folder(folder)
    eng = ninfer_amd.Ninfer(folder, max_context=640, prefill_chunk=608, num_sequences=3, dtype=dtype, page_size=16, max_adapters=2, max_adapter_rank=5)
    factors = ro.random_factors({n: tuple(w[n].shape) for n in eng.runner.adapters.weights()}, 3, 5, std=0.1)
    eng.load_adapter("it", ro.write_adapter(tmp_path / "it", factors, 3, 3))
    ops, blocks = eng.runner.ops, []
    toks = util.random_tokens(rows, eng.vocab, 6)

    def run():
        out = {}
        for name in ("it", None):
            with eng.session(name) as s, eng.session("it") as beside:   # (a single row of another request before them)
                out[name] = eng.runner.step([Chunk(s.slot, toks, range(rows), name), Chunk(beside.slot, [3], [0], "it")]).cpu()
        return out

    inner = ops.beside
    monkeypatch.setattr(ops, "beside", lambda: (blocks.append(1), inner())[1])
    two = [run() for _ in range(3)]
    assert blocks and ops._side is not None and not ops._side_open
    monkeypatch.setattr(ops, "beside", lambda: OneStream(ops))
    monkeypatch.setattr(ops, "_on_side", lambda: ops._side_inside)
    one = run()
    for got in two:
        for name, logits in got.items():
            assert torch.equal(logits, one[name])
    assert not torch.equal(one["it"], one[None])
    if dtype == "float32":
        for name in ("it", None):
            x = ro.merged(w, factors, 1.0) if name else w
            ref = plain.forward(raw, x, toks)[0]
            noise = theirs.noise_of(raw, x, toks, ref)
            theirs.check_logits({"name": design, "ref": {dtype: {"r": ref}}, "noise": {dtype: {"r": noise}}}, dtype, {"r": one[name][:rows]}, str(name))
    eng.close()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [3, 40, 700])
def test_adapters_on_the_second_stream(dtype, t):
    from ninfer_amd.kernels import load_ops
    ops = load_ops()
    widths, r, count = (96, 64), 8, 5
    x, a, b, scale, base = tables(count, 128, widths, r, dtype, t, t)
    rows, ranks = i32([i * 3 % 6 - 1 for i in range(t)]), i32([8, 3, 8, 0, 5])
    want = torch.empty_like(base)
    ops.adapter_add(x, a, b, scale, ranks, widths, rows, want, base=base)
    here, there = base.clone(), base.clone()
    for _ in range(4):
        here.copy_(base)
        there.copy_(base)
        with ops.beside():
            ops.adapter_add(x, a, b, scale, ranks, widths, rows, there)
        ops.adapter_add(x, a, b, scale, ranks, widths, rows, here)
        ops.join()
        assert torch.equal(here, want) and torch.equal(there, want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_place_is_given_away_behind_a_step_that_is_still_to_run(model_dirs, tmp_path, dtype):
    from ninfer_amd import Chunk
    cfg, _ = util.read_folder(model_dirs["A"][dtype])
    eng = make(model_dirs, "A", dtype, max_adapters=1)
    made = adapters_of(tmp_path, cfg, dtype)
    toks = util.random_tokens(40, cfg["vocab_size"], 4)
    stream = torch.cuda.Stream()

    def step(name, late):
        session = eng.session(name)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            if late:
                torch.cuda._sleep(20_000_000)
            logits = eng.runner.step([Chunk(session.slot, toks, range(len(toks)), name)])
        session.close()
        return logits

    eng.load_adapter("all", made["all"][0])
    want = step("all", False).cpu()
    logits = step("all", True)
    eng.remove_adapter("all")
    eng.load_adapter("o", made["o"][0])
    other = step("o", False)
    torch.cuda.synchronize()
    assert torch.equal(logits.cpu(), want) and not torch.equal(other.cpu(), want)
    eng.close()
