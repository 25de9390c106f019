"""The graphed decode loop on the host: which stream each of its operations is issued on, with
fake streams (no GPU)."""
import contextlib
from types import SimpleNamespace

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from unsloth_spectral.llama_loop import SpectralLlama


class _Streams(TorchDispatchMode):
    """Notes every tensor operation with the stream that is current, and every wait."""

    def __init__(self, monkeypatch):
        super().__init__()
        self.log, log = [], []
        self.log = log
        make = lambda name: SimpleNamespace(  # noqa: E731
            name=name, wait_stream=lambda other: log.append(("wait", name, other.name)))
        self.main, self.side = make("main"), make("side")
        self.current = self.main

        @contextlib.contextmanager
        def use(stream):
            before, self.current = self.current, stream
            yield
            self.current = before

        monkeypatch.setattr(torch.cuda, "Stream", lambda device=None: self.side)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.current)
        monkeypatch.setattr(torch.cuda, "stream", use)

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.log.append(("op", self.current.name, str(func)))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("n", [1, 2, 4])
def test_what_the_side_stream_reads_was_issued_before_it_waits(monkeypatch, n):
    """The side stream follows the main one from its wait on: what is issued on the main stream
    after that wait (the copy of the first token) may run beside the first step that reads it."""
    streams = _Streams(monkeypatch)
    tiers = SimpleNamespace(num_blocks=0, hot_len=0)
    caches = [SimpleNamespace(tiers=tiers, block_size=512)]
    model = SimpleNamespace(decode_step=lambda tok, pos, caches: torch.nn.functional.one_hot(tok + 1, 50).float())
    tok, pos, out = torch.tensor([3, 7]), torch.zeros(1, 1, dtype=torch.long), torch.zeros(2, n, dtype=torch.long)
    with streams:
        SpectralLlama._decode_graphed(model, tok, pos, caches, out, lambda logits: logits.argmax(-1))
    assert torch.equal(out, torch.tensor([[3], [7]]) + torch.arange(n))
    assert torch.equal(tok, torch.tensor([3, 7]))          # the caller's token stays
    log = streams.log
    start, end = log.index(("wait", "side", "main")), log.index(("wait", "main", "side"))
    assert start < end
    assert [e for e in log[start:end] if e[:2] == ("op", "main")] == []
    assert [e for e in log[:start] + log[end:] if e[:2] == ("op", "side")] == []


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("n", [0, 1, 3])
def test_as_many_tokens_are_recorded_as_are_returned(n, graphs, monkeypatch):
    _Streams(monkeypatch)
    picked = []

    def pick(logits, allow, record):
        assert record
        picked.append(logits.argmax(-1))
        return picked[-1]

    rules = SimpleNamespace(reset=picked.clear, observe_prompt=lambda ids: None, pick=pick)
    caches = [SimpleNamespace(tiers=SimpleNamespace(num_blocks=0, hot_len=0), block_size=512)]
    step = lambda tok: torch.nn.functional.one_hot(tok + 1, 50).float()  # noqa: E731
    model = SimpleNamespace(prefill=lambda ids: (step(ids[:, -1]), caches), decode_step=lambda tok, pos, caches: step(tok))
    model._decode_graphed = lambda *a: SpectralLlama._decode_graphed(model, *a)
    out = SpectralLlama.generate(model, torch.tensor([[1, 4], [2, 9]]), n, cuda_graphs=graphs, rules=rules)
    assert out.shape == (2, n) and len(picked) == n
    assert torch.equal(out, torch.stack(picked, 1) if n else out)


def test_layers_patched_for_dense_attention_decode_eagerly(monkeypatch):
    """Dense attention takes the context's length from the host at every step: no step is captured."""
    from unsloth_spectral.llama_loop import LlamaShape
    _Streams(monkeypatch)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: pytest.fail("a step was captured"))
    real = SpectralLlama(LlamaShape(layers=1, hidden=64, heads=4, kv_heads=2, head_dim=16, ffn=96, vocab=50), device="cpu")
    real.patch(block_size=512, use_spectral_attention=False)
    caches = [SimpleNamespace(tiers=SimpleNamespace(num_blocks=1, hot_len=0), block_size=512)]
    real.decode_step = lambda tok, pos, caches: torch.nn.functional.one_hot(tok + 1, 50).float()
    out = torch.zeros(1, 8, dtype=torch.long)
    real._decode_graphed(torch.tensor([3]), torch.zeros(1, 1, dtype=torch.long), caches, out, lambda logits: logits.argmax(-1))
    assert out.tolist() == [list(range(3, 11))]


def test_layers_without_the_patchs_mark_are_taken_for_spectral_ones(monkeypatch):
    """A single-token forward put on the layers by hand: the loop asks only whether dense attention was
    asked for."""
    _Streams(monkeypatch)
    captured = []
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: captured.append(1) or pytest.skip("reached the capture"))
    import unsloth_spectral.llama_loop as L
    monkeypatch.setattr(L, "rope_tables_for", lambda *a: None)
    tiers = SimpleNamespace(num_blocks=1, hot_len=0, hot_bound=None, ensure_hot=lambda n: None, hot_len_device=lambda: None)
    caches = [SimpleNamespace(tiers=tiers, block_size=512, total_tokens=512)]
    model = SimpleNamespace(model=SimpleNamespace(layers=[SimpleNamespace(self_attn=SimpleNamespace())]),
                            decode_step=lambda tok, pos, caches: torch.nn.functional.one_hot(tok + 1, 50).float())
    try:
        SpectralLlama._decode_graphed(model, torch.tensor([3]), torch.zeros(1, 1, dtype=torch.long), caches,
                                      torch.zeros(1, 8, dtype=torch.long), lambda logits: logits.argmax(-1))
    except pytest.skip.Exception:
        pass
    assert captured == [1]
