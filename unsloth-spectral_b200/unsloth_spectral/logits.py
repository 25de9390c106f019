"""Rules on the logits of a decode step: penalties for repeated tokens, biases, a grammar's
allowed tokens, and the greedy choice under them.

``LogitsRules`` holds a batch's settings and its history (which tokens were in the prompt,
how often each was put out) on the device; ``apply`` gives the processed logits and the
best token, ``pick`` the token alone -- one launch of ``libspx`` each.
"""
from __future__ import annotations

import math
from typing import Dict, Optional, Sequence, Tuple, Union

import torch

from . import _native as N

Setting = Union[float, Sequence[float]]


def allow_words(vocab: int) -> int:
    """int32 words of one row of an ``allow`` mask."""
    return (vocab + 31) // 32


class LogitsRules:
    """Settings (one number for all requests, or one each) and history of ``batch`` requests.

    In this order, in float32, for token t of a request:

    * ``repetition_penalty`` p > 0: a token seen in the prompt or put out has a positive
      logit divided by p, any other multiplied;
    * ``frequency_penalty`` f and ``presence_penalty`` q, of the tokens put out:
      ``l - f * count - q``;
    * ``logit_bias``: ``{token: value}`` (for all, or a list of one dict each), added;
    * ``allow`` (per call): int32 words ``[batch, ceil(vocab / 32)]`` (or one row), bit
      ``t % 32`` of word ``t // 32`` set for an allowed token; any other is -inf.

    The chosen token is the largest of these float32 values, the lowest index among equals;
    a NaN counts as largest; a request whose every token is at -inf gets token 0.

    The calls on one object share its history: make them on one stream, or order them.
    """

    def __init__(self, batch: int, vocab: int, device="cuda", *, repetition_penalty: Setting = 1.0,
                 frequency_penalty: Setting = 0.0, presence_penalty: Setting = 0.0,
                 logit_bias: Union[None, Dict[int, float], Sequence[Optional[Dict[int, float]]]] = None):
        if batch < 1 or batch > 65535 or not 1 <= vocab <= 1 << 30:
            raise ValueError(f"batch 1..65535 and vocab 1..2^30 expected, got {batch} and {vocab}")
        self.batch, self.vocab = batch, vocab
        words = allow_words(vocab)
        rep = _setting("repetition_penalty", repetition_penalty, batch)
        if any(v <= 0 for v in rep):
            raise ValueError("repetition_penalty must be positive, in float32 too")
        freq = _setting("frequency_penalty", frequency_penalty, batch)
        pres = _setting("presence_penalty", presence_penalty, batch)
        rows, toks, vals = _biases(logit_bias, batch, vocab)
        self.seen_bits = torch.zeros(batch, words, dtype=torch.int32, device=device)
        self.counts = torch.zeros(batch, vocab, dtype=torch.int32, device=device)
        dev = self.device = self.counts.device
        put = lambda v, neutral: torch.tensor(v, dtype=torch.float32, device=dev) if any(  # noqa: E731
            x != neutral for x in v) else None
        self._rep, self._freq, self._pres = put(rep, 1.0), put(freq, 0.0), put(pres, 0.0)
        self._bias = None
        if toks:
            t = torch.tensor(toks, dtype=torch.int64)
            word = torch.tensor(rows, dtype=torch.int64) * words + t // 32
            bits = torch.zeros(batch * words, dtype=torch.int64)
            # one bit of a word for each distinct token: a sum sets them
            bits.scatter_add_(0, word, torch.ones_like(t) << (t % 32))
            bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
            n = torch.bincount(word, minlength=batch * words)
            first = (n.cumsum(0) - n).to(torch.int32)
            self._bias = (bits.view(batch, words).to(dev), first.view(batch, words).to(dev),
                          torch.tensor(vals, dtype=torch.float32, device=dev))
        b = self._bias or (None,) * 3
        # the tokens that a rule touches: seen ones and, where there are any, biased ones
        self._touched = self.seen_bits if b[0] is None else b[0].clone()
        self._front = N.front().Rules(batch, vocab, self._rep, self._freq, self._pres, self.seen_bits, self._touched,
                                      self.counts, *b)

    def reset(self):
        """Forget the history (a new generation with the same settings)."""
        self.seen_bits.zero_()
        self.counts.zero_()
        if self._bias is not None:
            self._touched.copy_(self._bias[0])

    def observe_prompt(self, tokens: torch.Tensor):
        """Add the prompt's tokens ``[batch, n]`` (int64; negative ones are padding)."""
        self._observe(tokens, None)

    def observe(self, tokens: torch.Tensor):
        """Add tokens put out, ``[batch]`` or ``[batch, n]`` (int64; negative ones are padding)."""
        self._observe(tokens, self.counts)

    def _observe(self, tokens, counts):
        t = tokens[:, None] if tokens.dim() == 1 else tokens
        if t.dim() != 2 or t.shape[0] != self.batch or t.dtype != torch.int64 or t.device != self.device:
            raise ValueError(f"tokens must be int64 [{self.batch}, n] on {self.device}, got {tokens.dtype} "
                             f"{tuple(tokens.shape)} on {tokens.device}")
        lib = N.lib_for(self.device)
        if t.shape[1] > 1 and t.stride(1) != 1 or t.stride(0) < 0:
            t = t.contiguous()
        N.check(lib, N.on_device(self.device, lib.spx_logits_observe, N.ptr(t), t.stride(0), self.batch, t.shape[1],
                                 self.vocab, N.ptr(self.seen_bits), N.ptr(self._touched), N.ptr(counts),
                                 N.stream_handle(self.device)),
                "spx_logits_observe")

    def apply(self, logits: torch.Tensor, allow: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(processed logits, token)`` of ``logits [batch, vocab]``: float32, float16 or
        bfloat16; the processed ones are rounded to that dtype, into ``out`` when given
        (``out`` may be ``logits``).  The history is left as it is."""
        return self._front.apply(logits, allow, out)

    def pick(self, logits: torch.Tensor, allow: Optional[torch.Tensor] = None, record: bool = False) -> torch.Tensor:
        """The token ``[batch]`` (int64) alone; ``record`` adds it to the history."""
        return self._front.run(logits, allow, None, record)


def _setting(name: str, v: Setting, batch: int):
    vals = [N.f32(v)] * batch if isinstance(v, (int, float)) else [N.f32(x) for x in v]
    if len(vals) != batch or not all(math.isfinite(x) for x in vals):
        raise ValueError(f"{name} must be one finite number or {batch} of them, got {v!r}")
    return vals


def _biases(bias, batch: int, vocab: int):
    """(rows, tokens, values) of the biases as host lists, by row and then by token."""
    each = [bias] * batch if bias is None or isinstance(bias, dict) else list(bias)
    if len(each) != batch:
        raise ValueError(f"logit_bias must be one dict or {batch} of them, got {len(each)}")
    rows, toks, vals = [], [], []
    for b, d in enumerate(each):
        for t in sorted(d or {}):
            v = N.f32(d[t])
            if not isinstance(t, int) or not 0 <= t < vocab or math.isnan(v) or v == math.inf:
                raise ValueError(f"logit_bias {{{t!r}: {d[t]!r}}}: a token 0..{vocab - 1} and a number (or -inf) expected")
            rows.append(b)
            toks.append(t)
            vals.append(v)
    return rows, toks, vals
