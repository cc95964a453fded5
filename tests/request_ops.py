"""Plain twins of the kernels for what single requests ask of a batch, beside those of tests/plain_ops.py, and adapters
as files with the weights that they stand for."""
import json
import os

import torch

import request_cases as rc
from plain_ops import PlainOps


class PlainRequestOps(PlainOps):
    LISTED_TOKENS = 64

    def adapter_add(self, x, a, b, scale, ranks, widths, row_adapter, out, base=None, single_rows=0):
        want, _ = rc.adapters(x, a, b, scale, ranks.tolist(), widths, row_adapter, out if base is None else base)
        out.copy_(want)

    def adjust_logits(self, logits, out=None, *, repetition=None, presence=None, frequency=None, hist_offsets=None, hist_tokens=None,
                      hist_counts=None, hist_generated=None, bias_offsets=None, bias_tokens=None, bias_values=None, masks=None,
                      mask_rows=None):
        rows, vocab = logits.shape
        cut = lambda offsets, *cols: [list(zip(*(c[i:j].tolist() for c in cols))) for i, j in zip(offsets.tolist(), offsets.tolist()[1:])]
        histories = None if hist_offsets is None else cut(hist_offsets, hist_tokens, hist_counts, hist_generated)
        biases = None if bias_offsets is None else cut(bias_offsets, bias_tokens, bias_values)
        allowed = None if masks is None else [[bool(m[t // 32] >> (t % 32) & 1) for t in range(vocab)] for m in masks.tolist()]
        want, _ = rc.adjusted(logits, repetition, presence, frequency, histories, biases, allowed, mask_rows)
        (logits if out is None else out).copy_(want)

    def token_logprobs(self, logits, tokens=None, top=0):
        (p, before, best, bp), _ = rc.logprobs(logits, tokens, top)
        return p.float(), before.int(), best.int(), bp.float()


def random_factors(shapes, rank, seed, std=0.3):
    """weight -> (A [rank, in], B [out, rank]) for weights of the given [out, in]."""
    gen = torch.Generator().manual_seed(seed)
    return {w: (torch.randn(rank, i, generator=gen) * i ** -0.5, torch.randn(o, rank, generator=gen) * std) for w, (o, i) in shapes.items()}


def write_adapter(folder, factors, rank, alpha, dtype=torch.float32, **options):
    from ninfer_amd.weights.safetensors_io import write_safetensors
    os.makedirs(folder, exist_ok=True)
    with open(os.path.join(folder, "adapter_config.json"), "w") as f:
        json.dump(dict({"peft_type": "LORA", "r": rank, "lora_alpha": alpha, "bias": "none", "use_dora": False}, **options), f)
    write_safetensors(os.path.join(folder, "adapter_model.safetensors"),
                      [(f"base_model.model.{w.removesuffix('.weight')}.lora_{x}.weight", t.to(dtype))
                       for w, ab in factors.items() for x, t in zip("AB", ab)])
    return str(folder)


def merged(w, factors, scale, dtype=torch.float32):
    """The model's weights with an adapter's added (factors as an engine of `dtype` holds them)."""
    out = dict(w)
    for name, (a, b) in factors.items():
        out[name] = (w[name].double() + scale * (b.to(dtype).double() @ a.to(dtype).double())).float()
    return out


def attention_shapes(cfg, layers=None, which="qkvo"):
    """[out, in] of a Qwen2-MoE model's projections by weight."""
    d, h = cfg["head_dim"], cfg["hidden_size"]
    nq, nk = cfg["num_attention_heads"] * d, cfg["num_key_value_heads"] * d
    size = {"q": (nq, h), "k": (nk, h), "v": (nk, h), "o": (h, nq)}
    return {f"model.layers.{i}.self_attn.{p}_proj.weight": size[p]
            for i in (range(cfg["num_hidden_layers"]) if layers is None else layers) for p in which}
