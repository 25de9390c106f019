"""Low-rank adapters of many requests beside one shared projection.

A ``LoraPool`` holds the adapters of one projection (several fine-tunes of one base
weight) in slots on the device; a ``LoraBatch`` says which slot each sequence of a batch
uses; ``pool.add(y, x, batch)`` adds each sequence's low-rank product to the shared
projection's output ``y = x W^T``::

    out[r] = y[r] + scale * B (A x[r])        A [rank, in], B [out, rank] of the row's slot

``LoraAdapters`` holds the pools of a whole model whose attention is patched.
One call serves every adapter of the batch (two launches of ``libspx``), for prompts and
for single tokens.  A projection whose output is several weights side by side (a packed
q|k|v projection) has several ``parts``, each with its own A and B.  float16 and bfloat16;
no gradients.
"""
from __future__ import annotations

import math
from typing import Dict, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _native as N


class LoraBatch:
    """The adapter slot of each sequence of a batch (-1: none), as host integers.  The rows
    are grouped by slot once, on first use for a number of tokens per sequence (the host does
    not wait for the GPU), and kept on ``device``; ``prepare`` the batch before capturing a CUDA
    graph that uses it and keep it as long as the graph is replayed."""

    def __init__(self, slots: Sequence[int], device="cuda"):
        self.slots: Tuple[int, ...] = tuple(int(s) for s in slots)
        if any(s < -1 for s in self.slots):
            raise ValueError(f"a slot is -1 (none) or a pool's slot number, got {min(self.slots)}")
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._front = N.front().Batch(self.slots, self.device)
        self.highest = self._front.highest
        self._elsewhere: Dict[torch.device, "LoraBatch"] = {}

    def on(self, device: torch.device) -> "LoraBatch":
        """This batch on ``device``: itself, or one with the same slots that is kept with it."""
        if device == self.device:
            return self
        if device not in self._elsewhere:
            self._elsewhere[device] = LoraBatch(self.slots, device)
        return self._elsewhere[device]

    def __len__(self) -> int:
        return len(self.slots)

    def prepare(self, tokens: int = 1) -> "LoraBatch":
        """Group the rows of ``tokens`` tokens per sequence now, and wait until the grouping is on
        the device."""
        self._front.prepare(tokens)
        for other in self._elsewhere.values():
            other.prepare(tokens)
        return self

    @staticmethod
    def tiles_of(slots: Sequence[int], tokens: int, blocks: bool = False):
        """Host arrays ``(tile_rows, tiles [n, 4], order)``: rows sorted by slot, cut into tiles of
        one slot: 16 rows of any sequences, or 32 where a slot has more; or ``blocks`` of up to 128
        tokens of one sequence, which name their first row themselves (``order`` is empty)."""
        tile_rows, n, held = N.front().group_rows(list(slots), tokens, blocks)
        held = np.asarray(held, dtype=np.int32)
        return tile_rows, held[:4 * n].reshape(n, 4), held[4 * n:]


class LoraPool:
    """Adapters of one projection ``in_features -> out_features`` (an int, or the widths of
    its parts).  ``max_rank`` (up to 128) bounds the rank of an adapter; widths and
    ``in_features`` are multiples of 8."""

    def __init__(self, in_features: int, out_features: Union[int, Sequence[int]], max_rank: int = 16, slots: int = 8,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        widths = (out_features,) if isinstance(out_features, int) else tuple(int(w) for w in out_features)
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"adapters are float16 or bfloat16, got {dtype}")
        if not 1 <= len(widths) <= N.LORA_MAX_PARTS:
            raise ValueError(f"1 to {N.LORA_MAX_PARTS} parts, got {len(widths)}")
        if in_features < 8 or in_features % 8 or any(w < 8 or w % 8 for w in widths):
            raise ValueError(f"in_features {in_features} and widths {widths} must be multiples of 8")
        if not 1 <= max_rank <= N.LORA_MAX_RANK or slots < 1:
            raise ValueError(f"max_rank 1..{N.LORA_MAX_RANK} and at least one slot, got {max_rank} and {slots}")
        self.in_features, self.widths, self.out_features = in_features, widths, sum(widths)
        self.max_rank, self.slots, self.dtype = max_rank, slots, dtype
        self._rank = (max_rank + 15) // 16 * 16    # stored rank
        parts = len(widths)
        self.a = torch.zeros(slots, parts, self._rank, in_features, dtype=dtype, device=device)
        self.b = torch.zeros(slots, self.out_features, self._rank, dtype=dtype, device=device)
        self.ranks = torch.zeros(slots, parts, dtype=torch.int32, device=device)
        self.scales = torch.zeros(slots, parts, dtype=torch.float32, device=device)
        self.device = self.a.device
        self._add = N.front().Pool(self.a, self.b, self.ranks, self.scales, list(widths)).add

    def _slot(self, slot: int, part: int):
        if not 0 <= slot < self.slots or not 0 <= part < len(self.widths):
            raise IndexError(f"slot {slot}, part {part} of a pool of {self.slots} slots, {len(self.widths)} parts")

    def _fits(self, slot: int, A: torch.Tensor, B: torch.Tensor, scale: float, part: int) -> Tuple[int, int]:
        """The width of a part and the rank of an adapter that is to go there; raises when it cannot."""
        self._slot(slot, part)
        w, r = self.widths[part], A.shape[0] if A.dim() == 2 else 0
        if A.shape != (r, self.in_features) or B.shape != (w, r) or not 1 <= r <= self.max_rank:
            raise ValueError(f"A must be [rank, {self.in_features}] and B [{w}, rank] with rank 1..{self.max_rank}, "
                             f"got {tuple(A.shape)} and {tuple(B.shape)}")
        if not math.isfinite(N.f32(scale)):
            raise ValueError(f"scale must be finite, got {scale}")
        return w, r

    def load(self, slot: int, A: torch.Tensor, B: torch.Tensor, scale: float = 1.0, part: int = 0):
        """Put an adapter's ``A [rank, in_features]``, ``B [width, rank]`` and scale
        (alpha / rank) into a slot; its other parts keep what they hold (nothing at first:
        the shared projection alone)."""
        w, r = self._fits(slot, A, B, scale, part)
        at = sum(self.widths[:part])
        with torch.no_grad():
            # what lies in the pool itself is read before its place is cleared
            A, B = (t.clone() if t.untyped_storage().data_ptr() == held.untyped_storage().data_ptr() else t
                    for t, held in ((A, self.a), (B, self.b)))
            self.a[slot, part].zero_()
            self.a[slot, part, :r].copy_(A)
            self.b[slot, at:at + w].zero_()
            self.b[slot, at:at + w, :r].copy_(B)
            self.ranks[slot, part] = r
            self.scales[slot, part] = float(scale)

    def unload(self, slot: int):
        """Empty a slot: its sequences get the shared projection alone."""
        self._slot(slot, 0)
        self.ranks[slot].zero_()

    def add(self, y: torch.Tensor, x: torch.Tensor, batch: LoraBatch, out=None) -> torch.Tensor:
        """``y + scale * B (A x)`` of each sequence's slot.  ``x [B, T, in]`` (or ``[B, in]``:
        one token each) and ``y [B, T, out]`` in the pool's dtype, rows on 16 bytes and evenly
        spaced; ``out`` may be ``y`` itself (in place) or lie beside it, without it a new tensor is
        returned.  The call does not wait for the GPU: should a copy inside a kernel fail to arrive
        within 2 s, the rows that it was for come out as NaN."""
        return self._add(y, x, batch._front, out)


def adapted(module, name: str, y: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """``y``, the output of projection ``name`` of ``module`` on ``x``, with the adapters of the batch
    in use added in place when a ``LoraAdapters`` covers it."""
    lora = getattr(module, "spx_lora", None)
    if lora is None:
        return y
    owner, pools = lora
    pool = pools.get(name)
    if pool is None or owner.batch is None:
        return y
    if y.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("the adapters' products have no gradients: run the forward under torch.no_grad()")
    return pool.add(y, x, owner.batch.on(pool.device), out=y)


def _projection(where: str, module, model_dtype):
    """``(in, out, dtype, device)`` of a projection.  A packed weight (4 bits a value, say) shows
    neither its sizes nor the type of the products: the module's ``in_features`` and
    ``out_features`` do, and the model's ``dtype`` or else the module's ``compute_dtype``."""
    w = module.weight
    if w.dim() == 2 and w.dtype.is_floating_point:
        n_out, n_in = w.shape
    else:
        n_in, n_out = getattr(module, "in_features", None), getattr(module, "out_features", None)
    types = (torch.float16, torch.bfloat16)
    held = (w.dtype,) if w.dtype.is_floating_point and w.dtype.itemsize > 1 else (
        model_dtype, getattr(module, "compute_dtype", None))
    dtype = next((t for t in held if t in types), None)
    if dtype is None or n_in is None or n_out is None:
        raise TypeError(f"{where} takes no adapters: its weight is {w.dtype} {tuple(w.shape)}, and float16 or bfloat16 "
                        f"products of known sizes are expected")
    return n_in, n_out, dtype, w.device


class LoraAdapters:
    """The adapters of a model: a ``LoraPool`` for every projection of its layers named in
    ``targets``.  ``model`` is a ``SpectralLlama`` or any model that ``patch_unsloth_attention``
    takes (of the latter the attention projections only: their MLPs run their own code)::

        adapters = LoraAdapters(model, max_rank=16, slots=8)
        adapters.load(0, {(layer, "q_proj"): (A, B), ...}, scale=alpha / rank)
        model.generate(ids, 64, adapters=adapters, adapter_slots=[0, -1, 3, 0])

    ``use(slots)`` names the slot of each sequence for the forwards that follow, ``use(None)``
    switches the adapters off.  An attention module or an MLP takes the adapters of one set at a
    time; ``detach()`` takes a set off its model."""

    ATTENTION = ("q_proj", "k_proj", "v_proj", "o_proj")
    MLP = ("gate_proj", "up_proj", "down_proj")

    def __init__(self, model, max_rank: int = 16, slots: int = 8, targets: Sequence[str] = ATTENTION + MLP):
        unknown = set(targets) - set(self.ATTENTION + self.MLP)
        if unknown:
            raise ValueError(f"unknown projections {sorted(unknown)}; expected some of {self.ATTENTION + self.MLP}")
        self.batch: Optional[LoraBatch] = None
        self.slots, self.targets = slots, tuple(targets)
        self._pools: Dict[Tuple[int, str], Tuple[LoraPool, int]] = {}
        model_dtype = getattr(model, "dtype", None)
        layers = model.model.layers
        covered = []           # (module, its pools), attached when all of them are there
        for i, layer in enumerate(layers):
            attn, mlp = layer.self_attn, getattr(layer, "mlp", None)
            if set(targets) & set(self.MLP) and not hasattr(mlp, "spx_lora"):
                raise ValueError(f"layer {i}: {type(mlp).__name__} takes no adapters; leave {self.MLP} out of targets")
            for module, names in ((attn, self.ATTENTION), (mlp, self.MLP)):
                if set(targets) & set(names) and getattr(module, "spx_lora", None) is not None:
                    raise ValueError(f"layer {i}: {type(module).__name__} has the adapters of another LoraAdapters; "
                                     f"detach() that first")
            shape = {n: _projection(f"layer {i}: {n}", getattr(module, n), model_dtype)
                     for module, names in ((attn, self.ATTENTION), (mlp, self.MLP)) for n in names if n in targets}

            def make(name, out=None):
                n_in, n_out, dtype, device = shape[name]
                return LoraPool(n_in, n_out if out is None else out, max_rank, slots, dtype, device)

            held = {}
            qkv = [n for n in self.ATTENTION[:3] if n in targets]
            if qkv and getattr(attn, "spx_qkv_weight", None) is not None:
                held["qkv"] = make(qkv[0], [getattr(attn, n).weight.shape[0] for n in self.ATTENTION[:3]])
                for n in qkv:
                    self._pools[i, n] = held["qkv"], self.ATTENTION.index(n)
            else:
                for n in qkv:
                    held[n] = make(n)
                    self._pools[i, n] = held[n], 0
            if "o_proj" in targets:
                held["o_proj"] = make("o_proj")
                self._pools[i, "o_proj"] = held["o_proj"], 0
            covered.append((attn, held))
            held = {}
            for n in self.MLP:
                if n in targets:
                    held[n] = make(n)
                    self._pools[i, n] = held[n], 0
            covered.append((mlp, held))
        self.device = layers[0].self_attn.o_proj.weight.device
        self._modules = [module for module, held in covered if held]
        for module, held in covered:
            if held:
                module.spx_lora = (self, held)

    def detach(self):
        """Take the set off its model, whose modules run their shared weights alone again and can
        take another set."""
        self.batch = None
        for module in self._modules or ():
            if self._holds(module):
                module.spx_lora = None
        self._modules = None

    def covers(self, model) -> bool:
        """Whether ``model`` is the one that this set is on: each of its modules, and no set since
        detached."""
        there = {id(m) for layer in model.model.layers for m in (layer.self_attn, getattr(layer, "mlp", None))}
        return self._modules is not None and all(id(m) in there and self._holds(m) for m in self._modules)

    def _holds(self, module) -> bool:
        return module.spx_lora is not None and module.spx_lora[0] is self

    def load(self, slot: int, weights: Dict[Tuple[int, str], Tuple[torch.Tensor, torch.Tensor]], scale: float = 1.0):
        """Put an adapter into a slot, in place of what it held: ``{(layer, projection): (A, B)}``
        with ``A [rank, in]``, ``B [out, rank]``; projections left out keep the shared weight alone."""
        for key in weights:
            if key not in self._pools:
                raise KeyError(f"no adapted projection {key}; targets are {self.targets}")
        for (layer, name), (A, B) in weights.items():     # all of it fits, or the slot keeps what it holds
            pool, part = self._pools[layer, name]
            pool._fits(slot, A, B, scale, part)
        self.unload(slot)
        try:
            for key, (A, B) in weights.items():
                pool, part = self._pools[key]
                pool.load(slot, A, B, scale, part)
        except Exception:
            self.unload(slot)     # not half an adapter
            raise

    def unload(self, slot: int):
        """Empty a slot."""
        for pool in {id(p): p for p, _ in self._pools.values()}.values():
            pool.unload(slot)

    def use(self, slots: Optional[Sequence[int]]):
        """The slot of each sequence of the batch that the next forwards run (-1: none), or None."""
        if slots is None:
            self.batch = None
            return
        if self._modules is None:
            raise RuntimeError("these adapters are detached from their model")
        batch = LoraBatch(slots, self.device)
        if batch.highest >= self.slots:
            raise IndexError(f"slot {batch.highest} of {self.slots}")
        for pool, _ in self._pools.values():
            batch.on(pool.device)      # of a model that lies on several devices
        self.batch = batch
