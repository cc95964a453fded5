"""The low-rank adapters that a model holds: for every product of its parts that takes adapters
(`Part.adapter_spots`) room for `count` adapters of up to `rank`, laid out once, so that captured steps
keep their addresses. An adapter is loaded into a free number by name and taken out again; a step
names each row's number."""
from __future__ import annotations

from typing import Dict, List, Optional

import torch

from ..parts.base import AdapterSpot, AdapterTables
from ..weights import WeightError
from ..weights.adapter_files import AdapterWeights


class AdapterSet:
    def __init__(self, spec, count: int, rank: int, device: torch.device, act_dtype: torch.dtype):
        self.count, self.rank = count, rank
        self.spots: List[AdapterSpot] = []
        for part in spec.parts():
            self.spots += [s for s in part.all_adapter_spots() if not any(s is t for t in self.spots)]
        if not self.spots:
            raise ValueError("no part of this model takes adapters")
        self._names: List[Optional[str]] = [None] * count
        self._holds = [0] * count
        self._scale = torch.zeros(count, dtype=torch.float32, device=device)
        for s in self.spots:
            widths = tuple(n for _, n in s.weights)
            s.tables = AdapterTables(torch.zeros(count, len(widths) * rank, s.width, dtype=act_dtype, device=device),
                                     torch.zeros(count, sum(widths), rank, dtype=act_dtype, device=device), self._scale,
                                     torch.zeros(count, dtype=torch.int32, device=device), widths)

    def names(self) -> List[str]:
        return [n for n in self._names if n is not None]

    def weights(self) -> List[str]:
        """The checkpoint weights beside which adapters may lie."""
        return [name for s in self.spots for name, _ in s.weights]

    def number(self, name: str) -> int:
        if name not in self._names or name is None:
            raise ValueError(f"no adapter named {name!r} is loaded")
        return self._names.index(name)

    def load(self, name: str, weights: AdapterWeights) -> int:
        """Into the first free number. Nothing is changed unless all of it fits."""
        if not name or not isinstance(name, str):
            raise ValueError("an adapter needs a name")
        if name in self._names:
            raise ValueError(f"an adapter named {name!r} is loaded already")
        if None not in self._names:
            raise ValueError(f"all {self.count} places for adapters are taken")
        if weights.rank > self.rank:
            raise WeightError(f"adapter {name!r} has rank {weights.rank}, there is room for {self.rank}")
        if not abs(weights.scale) <= torch.finfo(torch.float32).max:
            raise WeightError(f"adapter {name!r} has a scale of {weights.scale}")
        problems, known = [], {}
        for s in self.spots:
            for weight, columns in s.weights:
                known[weight] = (columns, s.width)
        factors = {}
        for module, (a, b) in weights.factors.items():
            weight = module + ".weight" if module + ".weight" in known else module
            if weight in factors:
                problems.append(f"{weight} has factors twice")
            factors[weight] = (a, b)
            if weight not in known:
                problems.append(f"{module} takes no adapter here")
            elif (tuple(a.shape), tuple(b.shape)) != ((weights.rank, known[weight][1]), (known[weight][0], weights.rank)):
                problems.append(f"{weight}: factors {list(a.shape)} and {list(b.shape)} beside a weight {list(known[weight])}")
        if problems:
            raise WeightError(f"adapter {name!r}: " + "; ".join(problems))
        g, r = self._names.index(None), weights.rank
        self._wait()
        for s in self.spots:
            t, at, here = s.tables, 0, False
            t.a[g].zero_()
            t.b[g].zero_()
            for i, (weight, columns) in enumerate(s.weights):
                if weight in factors:
                    a, b = factors[weight]
                    t.a[g, i * self.rank:i * self.rank + r].copy_(a)
                    t.b[g, at:at + columns, :r].copy_(b)
                    here = True
                at += columns
            t.ranks[g] = r if here else 0
        self._scale[g] = weights.scale
        self._wait()   # (steps on any stream find it)
        self._names[g], self._holds[g] = name, 0
        return g

    def remove(self, name: str) -> None:
        """Its number is free again. Refused while a request or session that has it is open."""
        g = self.number(name)
        if self._holds[g]:
            raise ValueError(f"adapter {name!r} is in use ({self._holds[g]} open requests or sessions)")
        self._wait()
        for s in self.spots:
            s.tables.ranks[g] = 0
        self._names[g] = None

    def _wait(self) -> None:
        """Before a place's numbers change: a step that nobody has read back may still read them, on whatever stream."""
        if self._scale.is_cuda:
            torch.cuda.synchronize(self._scale.device)

    def hold(self, name: str) -> None:
        self._holds[self.number(name)] += 1

    def let_go(self, name: str) -> None:
        self._holds[self.number(name)] -= 1

    def drop(self) -> None:
        for s in self.spots:
            s.tables = None
