"""LoraAdapters on the host: which modules a set holds, and what it refuses (no GPU)."""
from types import SimpleNamespace

import pytest
import torch

from unsloth_spectral import LoraAdapters, LoraPool
from unsloth_spectral.adapters import adapted
from unsloth_spectral.llama_loop import LlamaShape, SpectralLlama

SHAPE = LlamaShape(layers=2, hidden=64, heads=4, kv_heads=2, head_dim=16, ffn=96, vocab=50)


def _model(seed=0):
    return SpectralLlama(SHAPE, device="cpu", dtype=torch.bfloat16, seed=seed)


def _held(model):
    return [getattr(m, "spx_lora", None) for layer in model.model.layers for m in (layer.self_attn, layer.mlp)]


@pytest.mark.parametrize("first,second", [
    (LoraAdapters.ATTENTION + LoraAdapters.MLP, ("q_proj",)), (("q_proj",), ("o_proj",)), (("up_proj",), ("down_proj",)),
    (LoraAdapters.ATTENTION + LoraAdapters.MLP, LoraAdapters.ATTENTION), (("v_proj", "up_proj"), LoraAdapters.MLP)])
def test_a_second_set_on_a_module_is_refused_until_the_first_is_detached(first, second):
    model = _model()
    a = LoraAdapters(model, max_rank=4, slots=2, targets=first)
    held = _held(model)
    with pytest.raises(ValueError, match="detach"):
        LoraAdapters(model, max_rank=8, slots=3, targets=second)
    assert all(x is y for x, y in zip(_held(model), held))       # the refused set left nothing behind
    a.use([0, 1])
    a.detach()
    assert _held(model) == [None] * 4 and a.batch is None
    b = LoraAdapters(model, max_rank=8, slots=3, targets=second)
    with pytest.raises(RuntimeError, match="detached"):
        a.use([0, 1])
    a.use(None)
    a.detach()                                                   # again: nothing left to take off
    assert [x[0] for x in _held(model) if x is not None] == [b] * sum(x is not None for x in _held(model))


def test_sets_on_different_modules_stand_beside_each_other():
    model = _model()
    a = LoraAdapters(model, max_rank=4, slots=2, targets=("q_proj", "o_proj"))
    b = LoraAdapters(model, max_rank=4, slots=2, targets=("down_proj",))
    assert [x[0] for x in _held(model)] == [a, b, a, b]
    b.detach()
    assert [x and x[0] for x in _held(model)] == [a, None, a, None]
    y = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    a.use([0, 1])
    assert adapted(model.model.layers[0].mlp, "down_proj", y, y) is y
    with pytest.raises(RuntimeError):                            # reaches the pool (on a CPU tensor)
        adapted(model.model.layers[0].self_attn, "o_proj", y, y)


def test_a_refused_set_leaves_the_model_as_it_was():
    model = _model()
    model.model.layers[1].mlp = torch.nn.Identity()
    with pytest.raises(ValueError, match="layer 1"):
        LoraAdapters(model, max_rank=4, slots=2)
    assert _held(model) == [None] * 4


def test_generate_refuses_a_set_that_is_not_this_models():
    model, other = _model(), _model(1)
    ids = torch.zeros(2, 3, dtype=torch.long)
    foreign = LoraAdapters(other, max_rank=4, slots=2)
    gone = LoraAdapters(model, max_rank=4, slots=2)
    gone.detach()
    mine = LoraAdapters(model, max_rank=4, slots=2, targets=("q_proj", "down_proj"))
    for bad in (foreign, gone):
        with pytest.raises(ValueError, match="not .* of this model"):
            model.generate(ids, 1, adapters=bad, adapter_slots=[0, 1])
        assert bad.batch is None
    with pytest.raises(RuntimeError):                            # accepted, then refused for the device
        model.generate(ids, 1, adapters=mine, adapter_slots=[0, 1])
    model.model.layers[1] = other.model.layers[1]                # half of the set is no longer in the model
    with pytest.raises(ValueError, match="not .* of this model"):
        model.generate(ids, 1, adapters=mine, adapter_slots=[0, 1])


def test_a_generation_that_fails_to_start_leaves_the_adapters_as_they_were():
    model = _model()
    ad = LoraAdapters(model, max_rank=4, slots=2)
    ad.use([1])
    before = ad.batch
    with pytest.raises(RuntimeError):                            # the rows cannot be grouped on the CPU
        model.generate(torch.zeros(2, 3, dtype=torch.long), 1, adapters=ad, adapter_slots=[0, 1])
    assert ad.batch is before


class _Packed(torch.nn.Module):
    """A projection whose weight is packed: its sizes and type do not show in it."""

    def __init__(self, linear, compute_dtype=None, **sizes):
        super().__init__()
        n = linear.weight.numel()
        self.weight = torch.nn.Parameter(torch.zeros(n // 2, 1, dtype=torch.uint8), requires_grad=False)
        self.in_features, self.out_features = linear.weight.shape[1], linear.weight.shape[0]
        if compute_dtype is not None:
            self.compute_dtype = compute_dtype


def _pack(model, dtype):
    for layer in model.model.layers:
        layer.self_attn.spx_qkv_weight = None
        for m, names in ((layer.self_attn, LoraAdapters.ATTENTION), (layer.mlp, LoraAdapters.MLP)):
            for n in names:
                setattr(m, n, _Packed(getattr(m, n), dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_packed_projections_take_adapters(dtype):
    model = _model()
    want = {n: tuple(getattr(m, n).weight.shape) for m, names in
            ((model.model.layers[0].self_attn, LoraAdapters.ATTENTION), (model.model.layers[0].mlp, LoraAdapters.MLP))
            for n in names}
    _pack(model, dtype)
    ad = LoraAdapters(model, max_rank=4, slots=2)
    assert len(ad._pools) == 2 * len(want)
    for (i, n), (pool, part) in ad._pools.items():
        assert (pool.out_features, pool.in_features) == want[n] and pool.dtype == dtype and part == 0
    ad.load(1, {(1, "down_proj"): (torch.ones(2, 96), torch.ones(64, 2))})
    assert ad._pools[1, "down_proj"][0].ranks[1, 0] == 2


def test_the_type_of_packed_projections():
    """The model's own type comes before the one that a projection computes in: outputs come in the
    type of the inputs."""
    model = _model()
    _pack(model, torch.float16)
    model.dtype = torch.bfloat16
    assert LoraAdapters(model, max_rank=4, slots=2)._pools[0, "q_proj"][0].dtype == torch.bfloat16
    for dtype in (None, torch.float32):
        model = _model()
        _pack(model, dtype)
        with pytest.raises(TypeError, match="layer 0: q_proj"):
            LoraAdapters(model, max_rank=4, slots=2)
        assert _held(model) == [None] * 4
    model = SpectralLlama(SHAPE, device="cpu", dtype=torch.float32)
    with pytest.raises(TypeError, match="layer 0: q_proj"):
        LoraAdapters(model, max_rank=4, slots=2)


def test_a_model_on_two_devices_has_a_batch_on_each():
    """The second layer's pool on another device (here one that takes the call down): it gets the
    batch there, kept with the one that is in use."""
    model, far, calls = _model(), torch.device("meta"), []
    ad = LoraAdapters(model, max_rank=4, slots=2, targets=("o_proj",))
    pool = SimpleNamespace(device=far, add=lambda y, x, batch, out: calls.append(batch) or out)
    model.model.layers[1].self_attn.spx_lora[1]["o_proj"] = pool
    ad._pools[1, "o_proj"] = (pool, 0)
    ad.use([1, -1])
    assert ad.batch.device == ad.device == torch.device("cpu") and ad.batch.slots == (1, -1)
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    for _ in range(2):
        assert adapted(model.model.layers[1].self_attn, "o_proj", x, x) is x
    assert calls[0] is calls[1] and calls[0].device == far and calls[0].slots == (1, -1)
    assert ad.batch.on(torch.device("cpu")) is ad.batch and ad.batch.on(far) is calls[0]
    with pytest.raises(RuntimeError):                            # the first layer's: reaches the pool on the CPU
        adapted(model.model.layers[0].self_attn, "o_proj", x, x)


def test_an_adapter_made_from_a_slots_own_storage():
    """A slot's own rows and columns, scaled or cut to a smaller rank, put back into it."""
    pool = LoraPool(16, (24, 8), max_rank=4, slots=2, device="cpu")
    A, B = torch.randn(4, 16), torch.randn(24, 4)
    pool.load(1, A, B, 2.0)
    a, b = pool.a.clone(), pool.b.clone()
    pool.load(1, pool.a[1, 0, :4], pool.b[1, :24, :4], 1.0)
    assert torch.equal(pool.a, a) and torch.equal(pool.b, b) and pool.scales[1, 0] == 1.0
    pool.load(1, pool.a[1, 0, 1:4], pool.b[1, :24, 1:4], 0.5)    # rows that overlap their new places
    assert torch.equal(pool.a[1, 0, :3], a[1, 0, 1:4]) and torch.equal(pool.b[1, :24, :3], b[1, :24, 1:4])
    assert not pool.a[1, 0, 3:].any() and not pool.b[1, :24, 3:].any() and pool.ranks[1, 0] == 3


@pytest.mark.parametrize("bad", [(torch.ones(2, 64), torch.ones(63, 2)), (torch.ones(9, 64), torch.ones(64, 9)),
                                 (torch.ones(2, 63), torch.ones(64, 2)), (torch.ones(64), torch.ones(64, 2))])
def test_a_refused_adapter_leaves_the_one_in_the_slot(bad):
    model = _model()
    ad = LoraAdapters(model, max_rank=4, slots=2)
    good = {(i, "q_proj"): (torch.full((3, 64), i + 1.0), torch.ones(64, 3)) for i in range(2)}
    ad.load(1, good, scale=2.0)
    pools = [ad._pools[i, "q_proj"][0] for i in range(2)]
    before = [(p.a.clone(), p.b.clone(), p.ranks.clone(), p.scales.clone()) for p in pools]
    for weights, scale in (({(0, "q_proj"): good[0, "q_proj"], (1, "o_proj"): bad}, 1.0), (good, float("nan"))):
        with pytest.raises(ValueError):
            ad.load(1, weights, scale)
        for p, held in zip(pools, before):
            assert all(torch.equal(u, v) for u, v in zip((p.a, p.b, p.ranks, p.scales), held))
    for slot in (-1, 2):
        with pytest.raises(IndexError):
            ad.load(slot, good)


def test_a_module_whose_adapters_were_taken_off_by_hand_is_not_covered():
    model = _model()
    ad = LoraAdapters(model, max_rank=4, slots=2, targets=("q_proj",))
    assert ad.covers(model) and not ad.covers(_model(1))
    model.model.layers[1].self_attn.spx_lora = None
    assert not ad.covers(model)
    other = LoraAdapters(_model(2), max_rank=4, slots=2, targets=("q_proj",))
    model.model.layers[1].self_attn.spx_lora = (other, {})
    ad.detach()
    assert model.model.layers[0].self_attn.spx_lora is None
    assert model.model.layers[1].self_attn.spx_lora[0] is other      # what another set holds stays
