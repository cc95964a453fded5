"""What single requests ask of a batch they share, as calls that can be timed and compared.

Three operators, each over all rows of a step at once: low-rank adapters beside a shared projection
(every row with its request's own, or none), the changes that requests ask of their rows of logits
before a token is drawn (penalties for repeated tokens, biases, masks of a grammar), and the
log-probabilities that requests want to read of those rows. A case is one call. Sizes are those of
the engine's steps: hidden sizes and heads of the benchmark's models, their vocabulary of 151,936
tokens, up to 64 requests that decode, prompt portions of 512 to 2,048 rows.

`run` computes in plain torch operations in 32 bits, or, where `own` is set, calls the kernels.
"""
from __future__ import annotations

import math
import random
from typing import List, Optional

import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
NONE = -math.inf


# ---- cases -------------------------------------------------------------------------------------

def listed() -> List[dict]:
    return [
        # the output projection of a step in which one request decodes
        adapter("adapters_one_row", rows=1, k=2048, widths="2048", table=16, adapters=4, requests=1),
        # q, k and v of 64 decoding requests that spread over eight adapters, some with none
        adapter("adapters_64_rows_qkv", rows=64, k=2048, widths="2048,2048,2048", table=64, adapters=8, requests=64),
        # ... of prompt portions beside single rows, grouped heads
        adapter("adapters_portions_qkv", rows=2055, k=3584, widths="3584,512,512", table=64, adapters=8, requests=12),
        # the 32-bit path, sizes that no tile divides
        adapter("adapters_odd_32bit", rows=131, k=1001, widths="1043,77,77", table=20, adapters=5, requests=9,
                dtype="float32"),
        # one request whose penalties see a history of some thousand tokens
        adjust("adjust_one_row", rows=1, vocab=151936, history=2000, biases=0, masks=False),
        # a decode step: penalties, biases and, for half of the rows, a grammar's mask
        adjust("adjust_64_rows", rows=64, vocab=151936, history=2500, biases=40, masks=True),
        # masks alone, a vocabulary that ends inside a word and inside a vector
        adjust("adjust_masks_odd_vocab", rows=8, vocab=32001, history=0, biases=0, masks=True),
        # the most rows a step decodes in earnest
        adjust("adjust_256_rows", rows=256, vocab=151936, history=6000, biases=300, masks=True),
        # the token that one request has drawn and the five best beside it
        logprobs("logprobs_one_row", rows=1, vocab=151936, top=5),
        # ... of 64 requests, the twenty best
        logprobs("logprobs_64_rows", rows=64, vocab=151936, top=20),
        # a portion of a prompt that is scored: its own tokens only
        logprobs("logprobs_prompt_512", rows=512, vocab=151936, top=0),
        # logits of 16 bits, of which many are equal
        logprobs("logprobs_ties_odd_vocab", rows=33, vocab=32001, top=8, coarse=True),
    ]


def adapter(name, rows, k, widths, table, adapters, requests, dtype="bfloat16") -> dict:
    return dict(name=name, kind="adapters", rows=rows, k=k, widths=widths, table=table, adapters=adapters,
                requests=requests, dtype=dtype)


def adjust(name, rows, vocab, history, biases, masks) -> dict:
    return dict(name=name, kind="adjust", rows=rows, vocab=vocab, history=history, biases=biases, masks=masks)


def logprobs(name, rows, vocab, top, coarse=False) -> dict:
    return dict(name=name, kind="logprobs", rows=rows, vocab=vocab, top=top, coarse=coarse)


def _log(rng: random.Random, low: int, high: int) -> int:
    """A whole number of [low, high], spread evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("adapters", "adjust", "logprobs"))
    if kind == "adapters":
        rows, k = _log(rng, 1, 2055), _log(rng, 64, 3584)
        if rng.random() < 0.6:   # sizes of models are multiples of 64 more often than not
            k = max(64, k // 64 * 64)
        step = rng.choice((1, 8, 64))
        widths = [max(step, _log(rng, 64, 1536) // step * step) for _ in range(rng.choice((1, 1, 2, 3)))]
        case = adapter("", rows, k, ",".join(map(str, widths)), rng.choice((4, 8, 16, 20, 32, 64)), rng.randint(1, 8),
                       rng.randint(1, rows) if rows <= 64 else rng.randint(1, 64),
                       rng.choice(("bfloat16", "bfloat16", "float32")))
    elif kind == "adjust":
        case = adjust("", _log(rng, 1, 256), _log(rng, 500, 151936), rng.choice((0, _log(rng, 1, 6000))),
                      rng.choice((0, _log(rng, 1, 300))), rng.random() < 0.5)
    else:
        case = logprobs("", _log(rng, 1, 512), _log(rng, 500, 151936), rng.choice((0, 1, 5, 8, 20, 32)),
                        rng.random() < 0.3)
    del case["name"]
    return case


def _widths(case: dict) -> List[int]:
    return [int(w) for w in case["widths"].split(",")]


def _plan(case: dict):
    """The rows' adapters and the adapters' ranks, which are the same for every seed: (a list of one number a row, -1
    for none, and a list of ranks)."""
    rng = random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    ranks = [rng.choice((case["table"], max(1, case["table"] // 2), max(1, case["table"] // 4), rng.randint(1, case["table"])))
             for _ in range(case["adapters"])]
    requests = min(case["requests"], case["rows"])
    of_request = [rng.choice([-1] + list(range(case["adapters"])) * 2) for _ in range(requests)]
    of_request[0] = rng.randrange(case["adapters"])
    # single rows first, as the engine's steps have them; the rest is cut into portions
    if requests == case["rows"]:
        cuts = list(range(requests + 1))
    else:
        single = requests // 2
        cuts = list(range(single + 1)) + sorted(rng.sample(range(single + 1, case["rows"]), requests - single - 1)) \
            + [case["rows"]]
    return [a for a, x, y in zip(of_request, cuts, cuts[1:]) for _ in range(y - x)], ranks


def work(case: dict) -> dict:
    if case["kind"] == "adapters":
        size = _TYPES[case["dtype"]].itemsize
        widths = _widths(case)
        of_row, ranks = _plan(case)
        n, s, k, live = sum(widths), len(widths), case["k"], [a for a in of_row if a >= 0]
        tables = sum(ranks[a] * (s * k + n) for a in set(live))
        return {"bytes": size * (tables + len(live) * k + 2 * case["rows"] * n),
                "flops": sum(2 * ranks[a] * (s * k + n) for a in live)}
    cells = case["rows"] * case["vocab"]
    if case["kind"] == "adjust":
        lists = case["rows"] * (12 * case["history"] + 8 * case["biases"])
        return {"bytes": 8 * cells + lists + (cells // 16 if case["masks"] else 0), "flops": 2 * cells}
    return {"bytes": 4 * cells + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * cells}


# ---- inputs ------------------------------------------------------------------------------------

def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (std * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)

    def whole(high, n):
        return torch.randint(0, high, (n,), generator=gen, device="cuda", dtype=torch.int32)

    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    state = {"case": case}
    if case["kind"] == "adapters":
        t, widths, table, count = _TYPES[case["dtype"]], _widths(case), case["table"], case["adapters"]
        of_row, ranks = _plan(case)
        state.update(x=normal(case["rows"], case["k"], dtype=t), base=normal(case["rows"], sum(widths), dtype=t),
                     a=normal(count, len(widths) * table, case["k"], std=case["k"] ** -0.5, dtype=t),
                     b=normal(count, sum(widths), table, std=0.3, dtype=t),
                     scale=torch.rand(count, generator=gen, device="cuda") + 0.5, ranks=i32(ranks),
                     row_adapter=i32(of_row), widths=tuple(widths))
        return state
    rows, vocab = case["rows"], case["vocab"]
    logits = normal(rows, vocab, std=3.0)
    if case["kind"] == "logprobs":
        if case["coarse"]:
            logits = logits.to(torch.bfloat16).float()
        state.update(logits=logits, tokens=whole(vocab, rows))
        return state
    state.update(logits=logits, repetition=1 + 0.3 * torch.rand(rows, generator=gen, device="cuda"),
                 presence=normal(rows), frequency=normal(rows, std=0.3))

    def lists(most):
        """Between a half and all of `most` tokens for every row, each once: offsets and tokens."""
        rng = random.Random(seed + most)
        sizes = [min(vocab, rng.randint((most + 1) // 2, most)) for _ in range(rows)]
        offsets = [0]
        for n in sizes:
            offsets.append(offsets[-1] + n)
        # (a stride that shares no factor with the vocabulary walks through distinct tokens)
        first = whole(vocab, rows).long()
        step = next(p for p in (7919, 7907, 7901) if vocab % p)
        of = torch.repeat_interleave(torch.arange(rows, device="cuda"), torch.tensor(sizes, device="cuda"))
        at = torch.arange(offsets[-1], device="cuda") - torch.tensor(offsets, device="cuda")[of]
        return i32(offsets), ((first[of] + at * step) % vocab).int()

    if case["history"]:
        state["hist_offsets"], state["hist_tokens"] = lists(case["history"])
        n = state["hist_tokens"].shape[0]
        # most tokens of a text stand in it once or twice
        counts = 1 + (torch.rand(n, generator=gen, device="cuda") ** 6 * 12).int()
        state["hist_counts"] = counts
        state["hist_generated"] = (torch.rand(n, generator=gen, device="cuda") * (counts + 1)).int()
    if case["biases"]:
        state["bias_offsets"], state["bias_tokens"] = lists(case["biases"])
        state["bias_values"] = normal(state["bias_tokens"].shape[0], std=4.0)
    if case["masks"]:
        sets = max(1, rows // 4)
        state["masks"] = torch.randint(-2 ** 31, 2 ** 31, (sets, -(-vocab // 32)), generator=gen, device="cuda").int()
        of = whole(sets, rows)
        if rows > 1:
            of[::2] = -1
        state["mask_rows"] = of
    return state


_OPTIONS = ("hist_offsets", "hist_tokens", "hist_counts", "hist_generated", "bias_offsets", "bias_tokens", "bias_values",
            "masks", "mask_rows")


# ---- one pass ------------------------------------------------------------------------------------

def run(s: dict):
    kind = s["case"]["kind"]
    if own:
        from ninfer_amd.kernels import load_ops
        ops = load_ops()
        if kind == "adapters":
            out = torch.empty_like(s["base"])
            ops.adapter_add(s["x"], s["a"], s["b"], s["scale"], s["ranks"], s["widths"], s["row_adapter"], out,
                            base=s["base"])
            return out
        if kind == "adjust":
            out = torch.empty_like(s["logits"])
            ops.adjust_logits(s["logits"], out, repetition=s["repetition"], presence=s["presence"],
                              frequency=s["frequency"], **{k: s[k] for k in _OPTIONS if k in s})
            return out
        return ops.token_logprobs(s["logits"], s["tokens"], s["case"]["top"])
    return {"adapters": _adapters, "adjust": _adjust, "logprobs": _logprobs}[kind](s)


def _adapters(s: dict):
    """out[t] = base[t] + scale[g] B_g (A_g x[t]) for row t's adapter g, slice of columns by slice."""
    x, out, table = s["x"].float(), s["base"].float().clone(), s["b"].shape[2]
    of_row = s["row_adapter"]
    live = torch.arange(table, device=x.device)
    for g in range(s["a"].shape[0]):
        rows = torch.nonzero(of_row == g)[:, 0]
        keep = live < s["ranks"][g]
        at = 0
        for i, w in enumerate(s["widths"]):
            h = x[rows] @ s["a"][g, i * table:(i + 1) * table].float().t()
            h = torch.where(keep, h, 0.0)
            out[rows, at:at + w] += s["scale"][g] * (h @ s["b"][g, at:at + w].float().t())
            at += w
    return out.to(s["x"].dtype)


def _dense(offsets, tokens, values, rows, vocab):
    """Lists of (token, value) of every row as a table [rows, vocab], 0 where nothing stands."""
    of = torch.repeat_interleave(torch.arange(rows, device=tokens.device), (offsets[1:] - offsets[:-1]).long(),
                                 output_size=tokens.shape[0])
    table = torch.zeros(rows * vocab, dtype=values.dtype, device=tokens.device)
    table.index_add_(0, of * vocab + tokens, values)
    return table.view(rows, vocab)


def _adjust(s: dict):
    v = s["logits"]
    rows, vocab = v.shape
    if "hist_tokens" in s:
        seen, made = (_dense(s["hist_offsets"], s["hist_tokens"], s[k].float(), rows, vocab)
                      for k in ("hist_counts", "hist_generated"))
        factor = s["repetition"][:, None] ** seen
        v = torch.where(v > 0, v / factor, v * factor)
        v = v - s["frequency"][:, None] * made - s["presence"][:, None] * (made > 0)
    if "bias_tokens" in s:
        v = v + _dense(s["bias_offsets"], s["bias_tokens"], s["bias_values"], rows, vocab)
    if "masks" in s:
        bits = (s["masks"][:, :, None] >> torch.arange(32, device=v.device)) & 1
        allowed = bits.view(bits.shape[0], -1)[:, :vocab] != 0
        of = s["mask_rows"].long()
        v = torch.where(allowed[of.clamp(min=0)] | (of < 0)[:, None], v, NONE)
    return v.clone() if v is s["logits"] else v


def _logprobs(s: dict):
    """(the tokens' log-probabilities, how many tokens stand before them, the best tokens, their log-probabilities)."""
    x, tokens, top = s["logits"], s["tokens"].long()[:, None], s["case"]["top"]
    vocab = x.shape[1]
    m = x.max(dim=1, keepdim=True).values
    lse = torch.log(torch.exp(x - m).sum(dim=1, keepdim=True))
    at = torch.arange(vocab, device=x.device)
    mine = torch.gather(x, 1, tokens)
    before = ((x > mine) | ((x == mine) & (at < tokens))).sum(dim=1)
    if not top:
        best = torch.empty(x.shape[0], 0, dtype=torch.int32, device=x.device)
        return (mine - m - lse)[:, 0], before.int(), best, best.float()
    # one number per token that orders by value, then by the lower index
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -2 ** 31 - bits, bits) * 2 ** 24 + (vocab - 1 - at)
    best = torch.topk(key, top, dim=1).indices
    return (mine - m - lse)[:, 0], before.int(), best.int(), torch.gather(x, 1, best) - m - lse


# ---- the definition in 64 bits ------------------------------------------------------------------

def exact(case: dict, seed: int) -> Optional[object]:
    s = prepare(case, seed)
    if case["kind"] == "adapters":
        out = s["base"].double()
        edges = [0]
        for w in s["widths"]:
            edges.append(edges[-1] + w)
        ranks, table = s["ranks"].tolist(), s["b"].shape[2]
        for g in set(s["row_adapter"].tolist()) - {-1}:
            rows, r = (s["row_adapter"] == g).nonzero().flatten(), ranks[g]
            for i in range(len(s["widths"])):
                c = slice(edges[i], edges[i + 1])
                # both factors as one matrix of the full width
                delta = s["b"][g, c, :r].double() @ s["a"][g, i * table:i * table + r].double()
                out[rows, c] += s["scale"][g].double() * (s["x"][rows].double() @ delta.t().contiguous())
        return out
    if case["kind"] == "adjust":
        v = s["logits"].double()
        for r in range(case["rows"]):
            if case["history"]:
                e = slice(int(s["hist_offsets"][r]), int(s["hist_offsets"][r + 1]))
                t, c, g = s["hist_tokens"][e].long(), s["hist_counts"][e].double(), s["hist_generated"][e].double()
                x, p = v[r, t], s["repetition"][r].double()
                x = torch.where(x > 0, x * p ** -c, x * p ** c)
                v[r, t] = x - g * s["frequency"][r].double() - (g >= 1).double() * s["presence"][r].double()
            if case["biases"]:
                e = slice(int(s["bias_offsets"][r]), int(s["bias_offsets"][r + 1]))
                v[r, s["bias_tokens"][e].long()] += s["bias_values"][e].double()
            if case["masks"] and int(s["mask_rows"][r]) >= 0:
                words = s["masks"][int(s["mask_rows"][r])].long()
                t = torch.arange(case["vocab"], device=v.device)
                v[r, (words[t // 32] >> (t % 32)) % 2 == 0] = NONE
        return v
    x, top = s["logits"].double(), case["top"]
    logp = x - torch.logsumexp(x, dim=1, keepdim=True)
    chosen = logp.gather(1, s["tokens"].long()[:, None])[:, 0]
    before, best = [], []
    for r, t in enumerate(s["tokens"].tolist()):
        row = x[r]
        before.append(int((row > row[t]).sum()) + int((row[:t] == row[t]).sum()))
        best.append(torch.sort(row, descending=True, stable=True).indices[:top] if top else row[:0].long())
    best = torch.stack(best)
    return chosen, torch.tensor(before, dtype=torch.int32), best.int(), logp.gather(1, best)
