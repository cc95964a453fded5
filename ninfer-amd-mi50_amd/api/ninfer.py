"""Python entry point in the manner of the reference's ctypes binding
(tools/ninfer_ctypes.py:48-247): a `Ninfer` engine object and `Session`s with
`prefill`, `decode`, `reset`, `close`, `slot`, `length`; `decode_batch` and
`sample` on the engine; the same names and meanings of options where the
reference has them (`max_context`, `prefill_chunk`, `num_sequences`). Logits
come back as numpy arrays. Added for what the reference leaves to an outside
scheduler: `step` (a mixed batch), `generate` and `complete` (the scheduler), `score` (log-probabilities
of given tokens), and low-rank adapters that sessions and requests name (`load_adapter`).
Return-code conventions of the C API (src/api/ninfer_c_api.cpp:191,226,235)
become exceptions here.
"""
from __future__ import annotations

from typing import Callable, Dict, List, Optional, Sequence, Union

import numpy as np

from ..config.options import EngineOptions
from ..engine.runner import Chunk
from ..engine.scheduler import Request, Scheduler
from ..loading import load_model, random_model
from ..sampling.params import SamplingParams
from ..sampling.sampler import History, SampleRow, Sampler, TokenLogprob, allowed_words, fresh_seed


class Session:
    """One request's place in the cache (reference tools/ninfer_ctypes.py:48-90)."""

    def __init__(self, engine: "Ninfer", adapter: Optional[str] = None):
        engine.runner.hold_adapter(adapter)
        self._engine = engine
        self.adapter = adapter   # the name of the low-rank adapter that all its tokens run with
        self._slot: Optional[int] = None
        try:
            self._slot = engine.runner.open()
        except BaseException:
            engine.runner.let_go_adapter(adapter)
            raise

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def slot(self) -> int:
        return self._slot

    @property
    def length(self) -> int:
        return self._engine.runner.cache.length(self._slot)

    def reset(self) -> None:
        self._engine.runner.close(self._slot)
        self._slot = self._engine.runner.open()

    def prefill(self, tokens: Sequence[int]) -> np.ndarray:
        """Feed tokens in portions of `prefill_chunk`; logits of the last one
        (reference src/api/ninfer_c_api.cpp:171-198)."""
        if len(tokens) == 0:
            raise ValueError("prefill needs at least one token")
        chunk = self._engine.options.prefill_chunk
        logits = None
        for i in range(0, len(tokens), chunk):
            part = list(tokens[i:i + chunk])
            last = i + chunk >= len(tokens)
            logits = self._engine.runner.step(
                [Chunk(self._slot, part, [len(part) - 1] if last else [], self.adapter)])
        return logits[0].float().cpu().numpy()

    def decode(self, token: int) -> np.ndarray:
        logits = self._engine.runner.step([Chunk(self._slot, [int(token)], [0], self.adapter)])
        return logits[0].float().cpu().numpy()

    def close(self) -> None:
        if self._slot is not None:
            self._engine.runner.close(self._slot)
            self._engine.runner.let_go_adapter(self.adapter)
            self._slot = None


class Ninfer:
    def __init__(self, model_dir: Optional[str] = None, max_context: Optional[int] = 32768,
                 prefill_chunk: int = 512, num_sequences: int = 1, dtype: str = "bfloat16",
                 page_size: int = 16, num_pages: Optional[int] = None, use_graph: bool = False,
                 random_config: Optional[dict] = None, random_seed: int = 0,
                 random_weights_dtype: Optional[str] = None, kv_bytes: Optional[int] = None,
                 check_pages: bool = False, max_adapters: int = 0, max_adapter_rank: int = 64):
        if max_context is None:
            # as many positions as the model's parts allow (a table of learned positions has
            # so many rows), and no more than the reference's default
            from ..config.base import read_config_json
            from ..loading import build_spec
            raw = random_config if model_dir is None else read_config_json(model_dir)
            limit = build_spec(raw)[1].max_positions() if raw is not None else None
            max_context = 32768 if limit is None else min(32768, limit)
        self.options = EngineOptions(dtype=dtype, max_context=max_context,
                                     prefill_chunk=prefill_chunk, num_sequences=num_sequences,
                                     page_size=page_size, num_pages=num_pages,
                                     use_graph=use_graph, kv_bytes=kv_bytes,
                                     check_pages=check_pages, max_adapters=max_adapters,
                                     max_adapter_rank=max_adapter_rank)
        if model_dir is not None:
            self.runner = load_model(model_dir, self.options)
        elif random_config is not None:
            self.runner = random_model(random_config, random_seed, self.options,
                                       weights_dtype=random_weights_dtype)
        else:
            raise ValueError("give a model folder or a configuration for random weights")
        self.sampler = Sampler(self.runner.ops, self.runner.device)
        self._sample_calls = 0

    # ---- introspection (reference src/api/ninfer_c_api.h:38-52) --------------------
    @property
    def vocab(self) -> int:
        return self.runner.vocab_size

    @property
    def max_context(self) -> int:
        return self.options.max_context

    @property
    def num_sequences(self) -> int:
        return self.options.num_sequences

    @property
    def devices(self) -> int:
        """GPUs the engine runs on (reference tools/ninfer_ctypes.py:177): always one."""
        return 1

    @property
    def kv_bytes_per_token(self) -> int:
        return self.runner.cache.kv_bytes_per_token(2 if self.options.dtype == "bfloat16" else 4)

    @property
    def state_bytes_per_request(self) -> int:
        """Fixed-size state of a request, apart from its pages (0 for this architecture)."""
        return self.runner.cache.state_bytes_per_request()

    @property
    def kv_total_bytes(self) -> int:
        c = self.runner.cache
        return sum(t.numel() * t.element_size() for pools in c.pools.values()
                   for t in pools.values())

    def kv_pages(self) -> Dict[str, int]:
        c = self.runner.cache
        return {"total": sum(g.allocator.num_pages for g in c.groups),
                "free": sum(g.allocator.free_pages for g in c.groups),
                "reused": c.pages_reused()}

    def tensor_names(self) -> List[str]:
        return self.runner.tensor_names()

    def tensor_read(self, name: str, offset: int = 0, count: Optional[int] = None) -> np.ndarray:
        """`count` numbers (all by default) from flat index `offset` of the checkpoint tensor
        `name` as the engine holds it now, as 32-bit floats: what an outside check needs to
        know of a model whose weights were generated on the device."""
        flat = self.runner.tensor(name).reshape(-1)
        end = flat.numel() if count is None else offset + count
        if not 0 <= offset <= end <= flat.numel():
            raise ValueError(f"{name}: [{offset}, {end}) is outside its {flat.numel()} numbers")
        return flat[offset:end].float().cpu().numpy()

    # ---- adapters -------------------------------------------------------------------
    def load_adapter(self, name: str, folder: str) -> None:
        """Read a low-rank adapter (adapter_config.json and adapter_model.safetensors) and hold it under `name`, for sessions
        and requests that ask for it. The engine has room for `max_adapters` of rank `max_adapter_rank`."""
        self.runner.load_adapter(name, folder)

    def remove_adapter(self, name: str) -> None:
        """Make its place free. Refused while a session or request that has it is open."""
        self.runner.remove_adapter(name)

    def adapters(self) -> List[str]:
        return [] if self.runner.adapters is None else self.runner.adapters.names()

    # ---- sessions -------------------------------------------------------------------
    def session(self, adapter: Optional[str] = None) -> Session:
        return Session(self, adapter)

    def decode_batch(self, sessions: Sequence[Session], tokens: Sequence[int]) -> np.ndarray:
        """One token for each of several sessions in one step; logits [n, vocab]
        (reference src/api/ninfer_c_api.cpp:219-246)."""
        if len(sessions) != len(tokens):
            raise ValueError("one token per session")
        logits = self.runner.step([Chunk(s.slot, [int(t)], [0], s.adapter)
                                   for s, t in zip(sessions, tokens)])
        return logits.float().cpu().numpy()

    def step(self, entries: Sequence[tuple]) -> Optional[np.ndarray]:
        """A mixed batch: entries of (session, tokens, wanted rows); logits of the
        wanted rows in order, or None."""
        logits = self.runner.step([Chunk(s.slot, list(t), list(w), s.adapter) for s, t, w in entries])
        return None if logits is None else logits.float().cpu().numpy()

    def sample(self, logits, temperature: float = 0.7, top_k: int = 50, top_p: float = 0.95,
               repetition_penalty: float = 1.0, seed: int = 0,
               recent: Sequence[int] = (), presence_penalty: float = 0.0, frequency_penalty: float = 0.0,
               logit_bias: Optional[Dict[int, float]] = None, allowed=None, generated: Sequence[int] = ()) -> int:
        """Stateless sampling of one row (reference src/api/ninfer_c_api.cpp:248-260;
        there the history is empty, here `recent` may carry it, and `generated` the tokens behind it that were
        generated, to which alone the presence and frequency penalties apply). `allowed`: what may come, token ids or
        the words of a mask (None: every token). ValueError where biases leave none of it."""
        import torch
        row = torch.as_tensor(np.asarray(logits, dtype=np.float32)).reshape(1, -1).to(
            self.runner.device)
        params = SamplingParams(temperature, top_k, top_p, repetition_penalty, seed, 1, presence_penalty,
                                frequency_penalty, logit_bias)
        params.check(row.shape[1], 0)
        history = History(recent)
        for t in generated:
            history.add(int(t))
        self._sample_calls += 1
        r = SampleRow(params, history, 0, 0 if seed else self._sample_calls,
                      seed or fresh_seed(), allowed_words(allowed, row.shape[1]))
        token = self.sampler.sample(row, [r])[0]
        if r.changes and r.bars(token):
            raise ValueError("no token is left that may come")
        return token

    def close(self) -> None:
        """Give the model, its cache, its captured graphs and the kernels' workspaces back to
        the device (reference tools/ninfer_ctypes.py:238-241: ninfer_free); the object cannot
        be used afterwards. After it another engine may take this one's place in memory."""
        import gc
        import torch
        if self.runner is not None:
            self.runner.release()
        self.runner = None
        self.sampler = None
        gc.collect()
        if torch.cuda.is_available():
            torch.cuda.synchronize()
            torch.cuda.empty_cache()

    # ---- generation -----------------------------------------------------------------
    def generate(self, prompts: Sequence[Sequence[int]],
                 params: Union[SamplingParams, Sequence[SamplingParams], None] = None,
                 stop_ids: Optional[Sequence[int]] = None, adapters: Optional[Sequence[Optional[str]]] = None,
                 allow: Optional[Sequence[Optional[Callable]]] = None) -> List[List[int]]:
        """Generated token ids for each prompt, through the scheduler."""
        return [r.output for r in self.complete(prompts, params, stop_ids, adapters, allow)]

    def complete(self, prompts: Sequence[Sequence[int]],
                 params: Union[SamplingParams, Sequence[SamplingParams], None] = None,
                 stop_ids: Optional[Sequence[int]] = None, adapters: Optional[Sequence[Optional[str]]] = None,
                 allow: Optional[Sequence[Optional[Callable]]] = None) -> List[Request]:
        """The finished requests of the prompts (`output`, `logprobs`), through the scheduler. `params`: one for all of
        them or one for each; `adapters`: the name of each one's adapter or None; `allow`: each one's `Request.allow`."""
        n = len(prompts)
        if params is None or isinstance(params, SamplingParams):
            params = [params or SamplingParams()] * n
        adapters = [None] * n if adapters is None else list(adapters)
        allow = [None] * n if allow is None else list(allow)
        if not len(params) == len(adapters) == len(allow) == n:
            raise ValueError(f"{n} prompts, {len(params)} params, {len(adapters)} adapters, {len(allow)} allow")
        if stop_ids is None:
            stop_ids = list(self.runner.spec.eos_token_ids)
        sched = Scheduler(self.runner, self.sampler)
        reqs = [Request(str(i), list(p), q, stop_ids, a, f) for i, (p, q, a, f) in enumerate(zip(prompts, params, adapters, allow))]
        try:
            for r in reqs:
                sched.add(r)
            sched.run()
        except BaseException as e:   # (the scheduler ends with this call: nothing may stay held by its requests)
            sched.abort(str(e) or type(e).__name__)
            raise
        for r in reqs:
            if r.status == "failed":
                raise RuntimeError(f"request {r.id}: {r.error}")
        return reqs

    def score(self, prompts: Sequence[Sequence[int]], top: int = 0,
              adapters: Optional[Sequence[Optional[str]]] = None) -> List[List[TokenLogprob]]:
        """How likely the model takes each prompt's tokens to be: for every token but the first its log-probability behind the
        tokens before it, its place in the order, and the `top` best tokens in its place. Prompts run one after the
        other, in portions of `prefill_chunk`."""
        adapters = [None] * len(prompts) if adapters is None else list(adapters)
        if len(adapters) != len(prompts):
            raise ValueError(f"{len(prompts)} prompts, {len(adapters)} adapters")
        most = min(getattr(self.runner.ops, "LISTED_TOKENS", 0), self.vocab)
        if not 0 <= top <= most:
            raise ValueError(f"top must be in [0, {most}], is {top}")
        out: List[List[TokenLogprob]] = []
        for prompt, adapter in zip(prompts, adapters):
            if len(prompt) == 0:
                raise ValueError("a prompt to score needs at least one token")
            if not 0 <= min(prompt) <= max(prompt) < self.vocab:   # (the last token is in no step)
                raise ValueError(f"token id outside [0, {self.vocab})")
            told: List[TokenLogprob] = []
            with self.session(adapter) as s:
                for i in range(0, len(prompt) - 1, self.options.prefill_chunk):
                    part = list(prompt[i:min(i + self.options.prefill_chunk, len(prompt) - 1)])
                    logits = self.runner.step([Chunk(s.slot, part, range(len(part)), adapter)])
                    told += self.sampler.logprobs(logits, prompt[i + 1:i + 1 + len(part)], top)
            out.append(told)
        return out
