"""A model assembled from a plan: embedding, layers in their run order, final norm
and output head.  Nothing here is specific to an architecture."""

from __future__ import annotations

from typing import Dict, List, Mapping, Optional, Set, Tuple

import torch

from ..parts.base import (
    BLOCKS, Block, CacheSpec, Embedding, FeedForward, Head, LayerCall, Mixer, ModelPlan, Norm, Part, Runtime, TensorSpec, is_absolute,
)


class Model:
    def __init__(self, plan: ModelPlan, cache_bits: Optional[int] = None) -> None:
        """`cache_bits`: 4 or 8 for keys and values cached in so many bits; a mixer that cannot refuses."""
        self.plan = plan
        self.cache_bits = cache_bits
        self.vocab_size = plan.vocab_size
        self.dim = plan.dim
        self.blocks: List[Block] = []
        for layer in plan.layers:
            if layer.block not in BLOCKS:
                raise KeyError(f"no block arrangement named {layer.block!r}; registered: {', '.join(sorted(BLOCKS))}")
            built = {role: slot.build() for role, slot in layer.parts.items()}
            names = {role: slot.prefix for role, slot in layer.parts.items()}
            self.blocks.append(BLOCKS[layer.block](names=names, **built))
        if cache_bits is not None:
            for block in self.blocks:
                for mixer in block.mixers():
                    mixer.set_cache_bits(cache_bits)
        self.embedding: Embedding = plan.embedding.build()  # type: ignore[assignment]
        self.final_norm: Norm = plan.final_norm.build()  # type: ignore[assignment]
        self.head: Head = plan.head.build()  # type: ignore[assignment]
        # the model's own parts with the prefixes of their tensors in the folder
        self._ends: List[Tuple[str, str, Part]] = [
            ("embedding", plan.embedding.prefix, self.embedding),
            ("final_norm", plan.final_norm.prefix, self.final_norm),
            ("head", plan.head.prefix, self.head),
        ]
        # run order: entry i runs block `layer` on the cache slots `cache_slots[i]`, one for each of the block's mixers
        self.run_order: List[LayerCall] = list(plan.run_order)
        self.cache_slots: List[Tuple[int, ...]] = []
        self.writes_cache: List[object] = []  # a boolean an entry, or one a mixer where only some read another entry's cache
        self.cache_specs: List[CacheSpec] = []
        owner_slots: Dict[int, Tuple[int, ...]] = {}
        for i, call in enumerate(self.run_order):
            if not 0 <= call.layer < len(self.blocks):
                raise ValueError(f"run order entry {i} names layer {call.layer}, the model has {len(self.blocks)}")
            specs = [mixer.cache_spec() for mixer in self.blocks[call.layer].mixers()]
            if call.cache_of is None:
                if call.shared_mixers is not None:
                    raise ValueError(f"run order entry {i} names shared mixers and no entry whose cache they read")
                owner_slots[i] = tuple(range(len(self.cache_specs), len(self.cache_specs) + len(specs)))
                self.cache_specs.extend(specs)
                self.cache_slots.append(owner_slots[i])
                self.writes_cache.append(True)
            elif call.shared_mixers is not None:
                if call.cache_of not in owner_slots:
                    raise ValueError(
                        f"run order entry {i} reads the cache of entry {call.cache_of}, "
                        "which is not an earlier entry with a cache of its own"
                    )
                theirs = owner_slots[call.cache_of]
                slots, writes = [], []
                for m, spec in enumerate(specs):
                    if m in call.shared_mixers:
                        if m >= len(theirs) or self.cache_specs[theirs[m]] != spec:
                            raise ValueError(f"run order entry {i}: mixer {m} cannot read a cache of another shape (entry {call.cache_of})")
                        slots.append(theirs[m])
                        writes.append(False)
                    else:
                        slots.append(len(self.cache_specs))
                        self.cache_specs.append(spec)
                        writes.append(True)
                if any(not 0 <= m < len(specs) for m in call.shared_mixers):
                    raise ValueError(f"run order entry {i} shares mixers {call.shared_mixers}, its block has {len(specs)}")
                self.cache_slots.append(tuple(slots))
                self.writes_cache.append(tuple(writes))
            else:
                if call.cache_of not in owner_slots:
                    raise ValueError(
                        f"run order entry {i} reads the cache of entry {call.cache_of}, "
                        "which is not an earlier entry with a cache of its own"
                    )
                slots = owner_slots[call.cache_of]
                if [self.cache_specs[slot] for slot in slots] != specs:
                    raise ValueError(f"run order entry {i} cannot read a cache of another shape (entry {call.cache_of})")
                self.cache_slots.append(slots)
                self.writes_cache.append(False)
        self.runtime: Optional[Runtime] = None

    @property
    def cache_slot(self) -> List[Optional[int]]:
        """For each entry of the run order the cache slot of its block's mixer (the first one's if it has
        several, None if it has none)."""
        return [slots[0] if slots else None for slots in self.cache_slots]

    # ---- tensors ---------------------------------------------------------------- #
    def tensor_specs(self) -> Dict[str, TensorSpec]:
        """Every tensor of the model folder by its full name.  Two parts may name one tensor (a head on the
        embedding's table): they must agree on what it is."""
        specs: Dict[str, TensorSpec] = {}

        def add(name: str, spec: TensorSpec) -> None:
            if name in specs and specs[name] != spec:
                raise ValueError(f"tensor {name!r} is named by two parts that disagree: {specs[name]} and {spec}")
            specs[name] = spec

        for role, prefix, part in self._ends:
            if role == "final_norm":
                continue
            for name, spec in part.tensor_specs().items():
                add(prefix + name, spec)
        for layer, block in zip(self.plan.layers, self.blocks):
            for name, spec in block.tensor_specs().items():
                add(name[1:] if is_absolute(name) else layer.prefix + name, spec)
        for name, spec in self.final_norm.tensor_specs().items():
            add(self.plan.final_norm.prefix + name, spec)
        return specs

    def tensor_names(self, role: str) -> Set[str]:
        """Full names of the tensors of the model's own part `role`: "embedding", "final_norm" or "head"."""
        for r, prefix, part in self._ends:
            if r == role:
                return {prefix + name for name in part.tensor_specs()}
        raise KeyError(f"the model's own parts are embedding, final_norm and head, not {role!r}")

    def _check_weight_bits(self, bits: int) -> None:
        if bits != 8:
            raise ValueError(f"matrices are held in 8 bits or in the activations' type, not in {bits} bits")
        for block in self.blocks:
            parts = getattr(block, "parts", None)
            if parts is None:
                raise ValueError(f"{type(block).__name__} keeps its parts itself: which of them would hold their matrices in {bits} bits is not known")
            for part in parts.values():
                if isinstance(part, (Mixer, FeedForward)) and not part.takes_weight_bits:
                    raise ValueError(f"{type(part).__name__} holds its matrices in the activations' type only, not in {bits} bits")

    def bind(self, tensors: Mapping[str, torch.Tensor], runtime: Runtime) -> None:
        if runtime.weight_bits is not None:
            self._check_weight_bits(runtime.weight_bits)
        self.runtime = runtime
        several: Dict[str, torch.Tensor] = {}  # tensors that several parts may name, asked for once

        def shared(name: str) -> torch.Tensor:
            if name not in several:
                several[name] = tensors[name]
            return several[name]

        for layer, block in zip(self.plan.layers, self.blocks):
            prefix = layer.prefix
            # a layer's tensors are asked for here and held no longer than the layer itself holds them (`TensorsOnDemand`)
            own = {n[len(prefix):]: tensors[n] for n in tensors if n.startswith(prefix)}
            own.update({n: shared(n[1:]) for n in block.tensor_specs() if is_absolute(n)})
            block.bind(own, runtime)
            del own
        for _role, prefix, part in self._ends:
            names = part.tensor_specs()
            part.bind({name: shared(prefix + name) for name in names}, runtime)

    @property
    def replayable(self) -> bool:
        """Whether a decode step may be captured once and replayed: every part says so (`Part.replayable`)."""
        return all(block.replayable for block in self.blocks) and all(part.replayable for _r, _p, part in self._ends)

    # ---- one step ------------------------------------------------------------------ #
    def forward(self, batch, cache) -> Optional[torch.Tensor]:
        """Run the batch's tokens through every layer, writing the cache, and return
        float32 logits [R, V] at `batch.logit_rows` (None if no row is wanted).

        Order as cwm/fastgen/forward.py:543-821: embedding, layers, final norm on
        the wanted rows, output projection, float32 logits.
        """
        h = self.embedding.forward(batch)
        delta = None
        for call, slots, writes in zip(self.run_order, self.cache_slots, self.writes_cache):
            views = tuple(cache.view(slot, batch) for slot in slots)
            view = views[0] if len(views) == 1 else (views or None)
            delta = self.blocks[call.layer].forward(h, delta, batch, view, writes)
        if batch.n_logit_rows == 0:
            return None
        x = self.final_norm.forward(h, delta, rows=batch.logit_rows)
        return self.head.forward(x)
