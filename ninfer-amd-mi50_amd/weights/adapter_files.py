"""Low-rank adapters as files: a folder with `adapter_config.json` and `adapter_model.safetensors`, in the layout that
adapter-training libraries write. Of the configuration are read `r`, `lora_alpha` and `use_rslora` (the factor is
alpha / r, or alpha / sqrt(r)); tensors are `[base_model.model.]<module>.lora_A.weight` [r, in] and `.lora_B.weight` [out, r],
beside the checkpoint's weight `<module>.weight`, or `<module>` where names end without `.weight`. Options that change the formula beyond that are refused by name, and so is every option that is not known here, unless
it is off (false, empty or absent)."""
from __future__ import annotations

import json
import math
import os
import re
from dataclasses import dataclass
from typing import Dict, Tuple

import torch

from .safetensors_io import SafeTensorsFile, WeightError, kept_dtype

_NAME = re.compile(r"^(?:base_model\.model\.)?(.+)\.lora_([AB])\.weight$")
# options under which the files mean something else, unless they have this value (or are absent)
_PLAIN = {"use_dora": (False,), "bias": ("none",), "fan_in_fan_out": (False,), "rank_pattern": ({}, None),
          "alpha_pattern": ({}, None), "modules_to_save": ([], None), "layers_to_transform": ([], None), "lora_bias": (False,),
          "use_qalora": (False,), "trainable_token_indices": ([], {}, None), "peft_type": ("LORA",), "layer_replication": ([], None),
          "alora_invocation_tokens": ([], None), "target_parameters": ([], None), "arrow_config": ({}, None), "use_rslora": (True, False, None),
          # (other starts change the weights beside which the factors lie, and files of such adapters may count on that)
          "init_lora_weights": (True, False, None, "gaussian", "orthogonal", "eva")}
# options that say how an adapter was trained or found, or beside which modules its factors lie (which the tensors' names say too)
_ASIDE = {"r", "lora_alpha", "auto_mapping", "base_model_name_or_path", "corda_config", "ensure_weight_tying", "eva_config", "exclude_modules",
          "inference_mode", "layers_pattern", "loftq_config", "lora_dropout", "megatron_config", "megatron_core", "peft_version",
          "qalora_group_size", "revision", "runtime_config", "target_modules", "task_type"}


@dataclass
class AdapterWeights:
    """`scale` B (A x) beside the weight of every module named: its (A [rank, in], B [out, rank])."""
    rank: int
    scale: float
    factors: Dict[str, Tuple[torch.Tensor, torch.Tensor]]


def read_adapter(folder: str) -> AdapterWeights:
    path = os.path.join(folder, "adapter_config.json")
    try:
        with open(path, encoding="utf-8") as f:
            cfg = json.load(f)
    except (OSError, ValueError) as e:
        raise WeightError(f"cannot read {path}: {e}") from None
    if not isinstance(cfg, dict):
        raise WeightError(f"{path} must hold a JSON object")
    for key, fine in _PLAIN.items():
        if key in cfg and cfg[key] not in fine:
            raise WeightError(f"{path}: {key} = {cfg[key]!r} is not built")
    for key in sorted(set(cfg) - set(_PLAIN) - _ASIDE):
        if cfg[key]:
            raise WeightError(f"{path}: the option {key} = {cfg[key]!r} is not known")
    rank, alpha = cfg.get("r"), cfg.get("lora_alpha", cfg.get("r"))
    if not isinstance(rank, int) or isinstance(rank, bool) or rank < 1:
        raise WeightError(f"{path}: r must be a whole number of at least 1, is {rank!r}")
    if not isinstance(alpha, (int, float)) or isinstance(alpha, bool) or not math.isfinite(alpha):
        raise WeightError(f"{path}: lora_alpha must be a number, is {alpha!r}")
    scale = alpha / math.sqrt(rank) if cfg.get("use_rslora") else alpha / rank
    f = SafeTensorsFile(os.path.join(folder, "adapter_model.safetensors"))
    try:
        pairs: Dict[str, Dict[str, torch.Tensor]] = {}
        strange = []
        for name in sorted(f.tensors):
            m = _NAME.match(name)
            if m is None:
                strange.append(name)
                continue
            tensor = f.read(name).to(kept_dtype(f.tensors[name].dtype)).clone()
            pairs.setdefault(m.group(1), {})[m.group(2)] = tensor
    finally:
        f.close()
    problems = [f"'{n}' is no factor of an adapter" for n in strange]
    for module, p in pairs.items():
        if set(p) != {"A", "B"}:
            problems.append(f"{module}: only factor {'/'.join(p)}")
        elif p["A"].dim() != 2 or p["B"].dim() != 2 or p["A"].shape[0] != rank or p["B"].shape[1] != rank:
            problems.append(f"{module}: factors {list(p['A'].shape)} and {list(p['B'].shape)} are not of rank {rank}")
    if not pairs:
        problems.append("no factors")
    if problems:
        raise WeightError(f"{folder}: " + "; ".join(problems))
    return AdapterWeights(rank, float(scale), {m: (p["A"], p["B"]) for m, p in pairs.items()})
