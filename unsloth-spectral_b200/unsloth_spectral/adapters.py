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

import torch

from . import _native as N


class LoraBatch:
    """The adapter slot of each sequence of a batch (-1: none), as host integers.  The rows
    are grouped by slot once, on first use for a number of tokens per sequence, and kept on
    ``device``; build the batch before capturing a CUDA graph that uses it (``prepare``)."""

    def __init__(self, slots: Sequence[int], device="cuda"):
        self.slots: Tuple[int, ...] = tuple(int(s) for s in slots)
        if any(s < -1 for s in self.slots):
            raise ValueError(f"a slot is -1 (none) or a pool's slot number, got {min(self.slots)}")
        self.highest = max(self.slots, default=-1)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._plans: Dict[Tuple[int, bool], tuple] = {}

    def __len__(self) -> int:
        return len(self.slots)

    def prepare(self, tokens: int = 1) -> "LoraBatch":
        """Group the rows of ``tokens`` tokens per sequence now."""
        for blocks in (False, True)[:1 + (tokens >= 64)]:
            self._plan(tokens, blocks)
        return self

    @staticmethod
    def tiles_of(slots: Sequence[int], tokens: int, blocks: bool = False):
        """Host lists ``(tile_rows, tiles, order)``: rows sorted by slot, cut into tiles of one
        slot: 16 rows of any sequences, or 32 where a slot has more, which reads the adapter's
        weights half as often; or ``blocks`` of up to 128 tokens of one sequence."""
        groups: Dict[int, list] = {}
        for i, s in enumerate(slots):
            groups.setdefault(s, []).append(i)
        most = max((len(g) for g in groups.values()), default=0) * tokens
        rows = 128 if blocks else 16 if most <= 16 else 32
        order = torch.empty(len(slots) * tokens, dtype=torch.int32)
        tiles, at = [], 0
        for s in sorted(groups):
            seqs = torch.tensor(groups[s], dtype=torch.int32)
            n = len(groups[s]) * tokens
            order[at:at + n] = (seqs[:, None] * tokens + torch.arange(tokens, dtype=torch.int32)[None]).reshape(-1)
            if rows == 128:
                tiles += [(s, at + q * tokens + i, min(rows, tokens - i), 0) for q in range(len(groups[s]))
                          for i in range(0, tokens, rows)]
            else:
                tiles += [(s, at + i, min(rows, n - i), 0) for i in range(0, n, rows)]
            at += n
        return rows, tiles, order

    def _plan(self, tokens: int, blocks: bool):
        p = self._plans.get((tokens, blocks))
        if p is None:
            if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"call LoraBatch.prepare({tokens}) before capturing a graph that uses the batch")
            rows, tiles, order = self.tiles_of(self.slots, tokens, blocks)
            t = torch.tensor(tiles, dtype=torch.int32).reshape(-1, 4)
            p = (rows, len(tiles), len(order), t.to(self.device), order.to(self.device))
            self._plans[tokens, blocks] = p
        return p


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
        self._index = self.a.get_device()
        # what of spx_lora_args does not change from call to call
        self._pool_args = (in_features, parts, *widths, *(0,) * (N.LORA_MAX_PARTS - parts), self._rank, slots,
                           N.dtype_code(dtype))
        self._pool_ptrs = (self.a.data_ptr(), self.b.data_ptr(), self.ranks.data_ptr(), self.scales.data_ptr())

    def _slot(self, slot: int, part: int):
        if not 0 <= slot < self.slots or not 0 <= part < len(self.widths):
            raise IndexError(f"slot {slot}, part {part} of a pool of {self.slots} slots, {len(self.widths)} parts")

    def load(self, slot: int, A: torch.Tensor, B: torch.Tensor, scale: float = 1.0, part: int = 0):
        """Put an adapter's ``A [rank, in_features]``, ``B [width, rank]`` and scale
        (alpha / rank) into a slot; its other parts keep what they hold (nothing at first:
        the shared projection alone)."""
        self._slot(slot, part)
        w = self.widths[part]
        r = A.shape[0]
        if A.shape != (r, self.in_features) or B.shape != (w, r) or not 1 <= r <= self.max_rank:
            raise ValueError(f"A must be [rank, {self.in_features}] and B [{w}, rank] with rank 1..{self.max_rank}, "
                             f"got {tuple(A.shape)} and {tuple(B.shape)}")
        if not math.isfinite(scale):
            raise ValueError(f"scale must be finite, got {scale}")
        at = sum(self.widths[:part])
        with torch.no_grad():
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
        spaced; ``out`` may be ``y`` itself (in place), else a new tensor is returned."""
        dev, dt = self._index, self.dtype
        xs, ys = x.shape, y.shape
        tokens = xs[1] if len(xs) == 3 else 1
        if len(xs) not in (2, 3) or len(ys) != len(xs) or xs[-1] != self.in_features or ys[-1] != self.out_features \
                or ys[:-1] != xs[:-1] or xs[0] != len(batch.slots):
            raise ValueError(f"x [B, T, {self.in_features}] and y [B, T, {self.out_features}] of {len(batch)} sequences "
                             f"expected, got {tuple(xs)} and {tuple(ys)}")
        if batch.highest >= self.slots:
            raise IndexError(f"the batch names slot {batch.highest}, the pool has {self.slots}")
        if out is None:
            out = x.new_empty(ys)
        elif out.shape != ys:
            raise ValueError(f"out {tuple(out.shape)} must have the shape of y {tuple(ys)}")
        if not (x.dtype == dt and y.dtype == dt and out.dtype == dt and x.get_device() == dev and y.get_device() == dev
                and out.get_device() == dev):
            raise ValueError(f"x, y and out must be {dt} on {self.device}")
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the pool on {self.device}")
        if dev < 0:
            N.lib_for(self.device)
        if tokens == 0 or not batch.slots:
            return out
        # Prompts take the kernels for blocks of adjacent rows: 8 x 4096 tokens on q|k|v at rank 16
        # 209 us against 410; below about 8M values of x and y their longer start shows
        # (5 x 77 tokens on 4096 -> 14336 22 us against 14)
        blocks = tokens >= 64 and len(batch.slots) * tokens * (self.in_features + self.out_features) >= 1 << 23
        rows, n_tiles, n, tiles, order = batch._plan(tokens, blocks)
        # the inner products, a buffer of each call's own: two streams or two captured graphs
        # never share one (the caching allocator hands it out in stream order)
        size = n * len(self.widths) * self._rank + 4
        ws = self.scales.new_empty(size)
        N.launch_packed("spx_lora_add", dev, N.LORA_PACK.pack(
            n_tiles, rows, n, *self._pool_args, x.data_ptr(), y.data_ptr(), out.data_ptr(), _row_stride(x),
            _row_stride(y), _row_stride(out), *self._pool_ptrs, tiles.data_ptr(), order.data_ptr(), ws.data_ptr(),
            4 * size))
        return out


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
    return pool.add(y, x, owner.batch, out=y)


class LoraAdapters:
    """The adapters of a model: a ``LoraPool`` for every projection of its layers named in
    ``targets``.  ``model`` is a ``SpectralLlama`` or any model that ``patch_unsloth_attention``
    takes (of the latter the attention projections only: their MLPs run their own code)::

        adapters = LoraAdapters(model, max_rank=16, slots=8)
        adapters.load(0, {(layer, "q_proj"): (A, B), ...}, scale=alpha / rank)
        model.generate(ids, 64, adapters=adapters, adapter_slots=[0, -1, 3, 0])

    ``use(slots)`` names the slot of each sequence for the forwards that follow, ``use(None)``
    switches the adapters off."""

    ATTENTION = ("q_proj", "k_proj", "v_proj", "o_proj")
    MLP = ("gate_proj", "up_proj", "down_proj")

    def __init__(self, model, max_rank: int = 16, slots: int = 8, targets: Sequence[str] = ATTENTION + MLP):
        unknown = set(targets) - set(self.ATTENTION + self.MLP)
        if unknown:
            raise ValueError(f"unknown projections {sorted(unknown)}; expected some of {self.ATTENTION + self.MLP}")
        self.batch: Optional[LoraBatch] = None
        self.slots, self.targets = slots, tuple(targets)
        self._pools: Dict[Tuple[int, str], Tuple[LoraPool, int]] = {}
        make = lambda w, out: LoraPool(w.shape[1], out, max_rank, slots, w.dtype, w.device)  # noqa: E731
        layers = model.model.layers
        for i, layer in enumerate(layers):
            attn, mlp = layer.self_attn, layer.mlp
            if set(targets) & set(self.MLP) and not hasattr(mlp, "spx_lora"):
                raise ValueError(f"layer {i}: {type(mlp).__name__} takes no adapters; leave {self.MLP} out of targets")
            held = {}
            qkv = [n for n in self.ATTENTION[:3] if n in targets]
            if qkv and getattr(attn, "spx_qkv_weight", None) is not None:
                widths = [getattr(attn, n).weight.shape[0] for n in self.ATTENTION[:3]]
                held["qkv"] = make(attn.spx_qkv_weight, widths)
                for n in qkv:
                    self._pools[i, n] = held["qkv"], self.ATTENTION.index(n)
            else:
                for n in qkv:
                    held[n] = make(getattr(attn, n).weight, getattr(attn, n).weight.shape[0])
                    self._pools[i, n] = held[n], 0
            if "o_proj" in targets:
                held["o_proj"] = make(attn.o_proj.weight, attn.o_proj.weight.shape[0])
                self._pools[i, "o_proj"] = held["o_proj"], 0
            attn.spx_lora = (self, held)
            held = {}
            for n in self.MLP:
                if n in targets:
                    held[n] = make(getattr(mlp, n).weight, getattr(mlp, n).weight.shape[0])
                    self._pools[i, n] = held[n], 0
            if held:
                mlp.spx_lora = (self, held)
        self.device = layers[0].self_attn.o_proj.weight.device

    def load(self, slot: int, weights: Dict[Tuple[int, str], Tuple[torch.Tensor, torch.Tensor]], scale: float = 1.0):
        """Put an adapter into a slot, in place of what it held: ``{(layer, projection): (A, B)}``
        with ``A [rank, in]``, ``B [out, rank]``; projections left out keep the shared weight alone."""
        for key in weights:
            if key not in self._pools:
                raise KeyError(f"no adapted projection {key}; targets are {self.targets}")
        self.unload(slot)
        for key, (A, B) in weights.items():
            pool, part = self._pools[key]
            pool.load(slot, A, B, scale, part)

    def unload(self, slot: int):
        """Empty a slot."""
        for pool in {id(p): p for p, _ in self._pools.values()}.values():
            pool.unload(slot)

    def use(self, slots: Optional[Sequence[int]]):
        """The slot of each sequence of the batch that the next forwards run (-1: none), or None."""
        if slots is None:
            self.batch = None
            return
        batch = LoraBatch(slots, self.device)
        if batch.highest >= self.slots:
            raise IndexError(f"slot {batch.highest} of {self.slots}")
        self.batch = batch


def _row_stride(t: torch.Tensor) -> int:
    """The distance between the rows of ``t [.., n]``, which must be even."""
    shape, stride = t.shape, t.stride()
    if stride[-1] != 1:
        raise ValueError(f"the last dimension must be contiguous, got strides {stride}")
    if len(shape) == 2 or shape[1] == 1:
        return stride[0] if shape[0] > 1 else max(stride[0], shape[-1])
    if shape[0] > 1 and stride[0] != shape[1] * stride[1]:
        raise ValueError(f"rows must be evenly spaced, got strides {stride} of {tuple(shape)}")
    return stride[1]
