"""The serving operators together, as the model loop uses them: heads with q/k norms, each
request's adapters on every projection, rules on the logits, eager and from CUDA graphs."""
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

NAMES = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


def _model(dtype, seed=3, layers=2):
    from unsloth_spectral.llama_loop import LlamaShape, SpectralLlama
    shape = LlamaShape(layers=layers, hidden=512, heads=8, kv_heads=2, head_dim=128, ffn=1024, vocab=1000, qk_norm=True)
    model = SpectralLlama(shape, device="cuda", dtype=dtype, std=0.05, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for layer in model.model.layers:
        for norm in (layer.self_attn.q_norm, layer.self_attn.k_norm):
            norm.weight.data.copy_(1 + 0.3 * torch.randn(128, generator=g, device="cuda"))
    model.patch(block_size=512, k_rank_keys=16, k_rank_values=16)
    return model, shape, g


def _weights(model, g, rank, dtype):
    out = {}
    for i, layer in enumerate(model.model.layers):
        for n in NAMES:
            w = getattr(layer.self_attn if n[0] in "qkvo" else layer.mlp, n).weight
            A = torch.randn(rank, w.shape[1], generator=g, device="cuda") / w.shape[1] ** 0.5
            B = torch.randn(w.shape[0], rank, generator=g, device="cuda") * 0.15
            out[i, n] = (A.to(dtype), B.to(dtype))
    return out


def _plain_logits(model, shape, ids, adapter, scale):
    """Last-position logits of one sequence in float64, every weight merged with its adapter."""
    W = lambda i, m, n: (getattr(m, n).weight.double()  # noqa: E731
                         + (scale * adapter[i, n][1].double() @ adapter[i, n][0].double() if adapter else 0))
    norm = lambda x, w, eps: x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()  # noqa: E731
    T, D = len(ids), shape.head_dim
    inv = shape.rope_theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    f = torch.outer(torch.arange(T, dtype=torch.float64, device="cuda"), inv)
    c, s = f.cos(), f.sin()

    def rope(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    h = model.model.embed_tokens.weight.double()[ids]
    for i, layer in enumerate(model.model.layers):
        at, x = layer.self_attn, norm(h, layer.input_layernorm.weight, shape.eps)
        split = lambda y, n: y.view(T, n, D).transpose(0, 1)  # noqa: E731
        q = rope(norm(split(x @ W(i, at, "q_proj").T, shape.heads), at.q_norm.weight, shape.eps))
        k = rope(norm(split(x @ W(i, at, "k_proj").T, shape.kv_heads), at.k_norm.weight, shape.eps))
        v = split(x @ W(i, at, "v_proj").T, shape.kv_heads)
        r = shape.heads // shape.kv_heads
        k, v = k.repeat_interleave(r, 0), v.repeat_interleave(r, 0)
        sc = (q @ k.transpose(1, 2) / D ** 0.5).masked_fill(torch.ones(T, T, device="cuda").triu(1).bool(), -torch.inf)
        a = (sc.softmax(-1) @ v).transpose(0, 1).reshape(T, -1)
        h = h + a @ W(i, at, "o_proj").T
        x, mlp = norm(h, layer.post_attention_layernorm.weight, shape.eps), layer.mlp
        gate = x @ W(i, mlp, "gate_proj").T
        h = h + (gate * torch.sigmoid(gate) * (x @ W(i, mlp, "up_proj").T)) @ W(i, mlp, "down_proj").T
    return norm(h[-1], model.model.norm.weight, shape.eps) @ model.lm_head.weight.double().T


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [9, 150])
def test_prompt_and_decode_logits_against_merged_weights(dtype, T):
    """Each layer rounds about 14 times to the type on a path (norms, projections, adapters,
    attention, residuals), each by at most half a step relative to the vector's size; two
    layers, the last norm and the head: 30 half steps, doubled for the norms' and the
    softmax's amplification: 30 * eps of the reference's size."""
    from unsloth_spectral import LoraAdapters
    model, shape, g = _model(dtype)
    ad = LoraAdapters(model, max_rank=8, slots=3)
    held = {0: _weights(model, g, 8, dtype), 2: _weights(model, g, 5, dtype)}
    for slot, w in held.items():
        ad.load(slot, w, scale=1.5)
    slots = [2, -1, 0, 2, 1]
    ids = torch.randint(0, shape.vocab, (5, T), generator=g, device="cuda")
    ad.use(slots)
    with torch.no_grad():
        got, caches = model.prefill(ids)
        nxt = torch.randint(0, shape.vocab, (5,), generator=g, device="cuda")
        step = model.decode_step(nxt, torch.full((1, 1), T, dtype=torch.long, device="cuda"), caches)
    ad.use(None)
    with torch.no_grad():
        bare, _ = model.prefill(ids)
    tol = 30 * torch.finfo(dtype).eps
    for b, s in enumerate(slots):
        ref = _plain_logits(model, shape, ids[b], held.get(s), 1.5).detach()
        ref2 = _plain_logits(model, shape, torch.cat([ids[b], nxt[b:b + 1]]), held.get(s), 1.5).detach()
        assert float((got[b].double() - ref).norm() / ref.norm()) <= tol
        assert float((step[b].double() - ref2).norm() / ref2.norm()) <= tol
        off = float((bare[b].double() - ref).norm() / ref.norm())
        assert off > 0.3 if s in held else off <= tol      # the adapters matter, and only where they are


def test_generate_with_everything_graphed_and_eager():
    from unsloth_spectral import LogitsRules, LoraAdapters
    model, shape, g = _model(torch.float16, seed=8)
    ad = LoraAdapters(model, max_rank=16, slots=2)
    ad.load(0, _weights(model, g, 16, torch.float16), scale=1.0)
    B, T, NEW, V = 3, 490, 60, shape.vocab
    prompt = torch.randint(0, V, (B, T), generator=g, device="cuda")
    ok = torch.rand(B, V, generator=g, device="cuda") < 0.5
    ok[:, 992:] = False
    words = torch.zeros(B, (V + 31) // 32 * 32, dtype=torch.int64, device="cuda")
    words[:, :V] = ok
    words = (words.view(B, -1, 32) << torch.arange(32, device="cuda")).sum(-1)
    allow = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    forced = int(ok[2].nonzero()[7])
    rules = LogitsRules(B, V, presence_penalty=[1000.0, 0.0, 0.0], frequency_penalty=[0.0, 0.3, 0.0],
                        repetition_penalty=[1.0, 1.2, 1.0], logit_bias=[None, None, {forced: 500.0}])
    runs = []
    for graphs in (False, True):
        torch.manual_seed(5)       # the cache's sketch
        runs.append(model.generate(prompt, NEW, cuda_graphs=graphs, rules=rules, allow=allow, adapters=ad,
                                   adapter_slots=[0, -1, 0]))
        counts = torch.zeros(B, V, dtype=torch.int32, device="cuda")
        counts.scatter_add_(1, runs[-1], torch.ones_like(runs[-1], dtype=torch.int32))
        assert torch.equal(rules.counts, counts)           # every token chosen is in the history once
    assert torch.equal(runs[0], runs[1])
    toks = runs[0]
    assert bool(ok.gather(1, toks).all())
    assert len(set(toks[0].tolist())) == NEW               # a penalty past every logit: nothing twice
    assert (toks[2] == forced).all()
    assert ad.batch is None
    torch.manual_seed(5)
    plain = model.generate(prompt, 4)
    torch.manual_seed(5)
    none = model.generate(prompt, 4, rules=LogitsRules(B, V))
    assert torch.equal(plain, none)                        # rules without a rule: the argmax


def test_a_modules_own_norms():
    """Attention modules whose norms are not the usual per-head RMS norm run their own code
    (here: a norm of whole rows, and one with 1 + weight), the others the kernel; both agree with
    the formula on the keys that the cache holds."""
    class RowNorm(torch.nn.Module):
        def __init__(self, n, plus):
            super().__init__()
            self.weight = torch.nn.Parameter(torch.linspace(0.5, 1.5, n, device="cuda").half())
            self.plus, self.eps = plus, 1e-6

        def forward(self, x):
            y = x.float()
            return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.eps) * (self.weight.float() + self.plus)).half()

    class HeadNorm(RowNorm):       # names its epsilon as the usual per-head norms do: the kernel
        def __init__(self, n):
            super().__init__(n, 0)
            self.variance_epsilon = 1e-6

    model, shape, g = _model(torch.float16, seed=4, layers=1)
    at = model.model.layers[0].self_attn
    ids = torch.randint(0, shape.vocab, (2, 20), generator=g, device="cuda")
    for qn, kn, wide in ((RowNorm(1024, 0), RowNorm(256, 0), True), (RowNorm(128, 1), RowNorm(128, 1), False),
                         (HeadNorm(128), HeadNorm(128), False)):
        at.q_norm, at.k_norm = qn, kn
        at._spectral_cache = None
        with torch.no_grad():
            _, caches = model.prefill(ids)
            x = model.model.layers[0].input_layernorm(model.model.embed_tokens(ids))
            kp = at.k_proj(x)
            want = (kn(kp) if wide else kn(kp.view(2, 20, 2, 128))).view(2, 20, 2, 128).transpose(1, 2)
            # half steps: the projection by another kernel or batch (one), the norm's result (one each way)
            assert float((caches[0].hot_K.float() - want.float()).norm() / want.float().norm()) <= 4 * 2 ** -11
            out = model.decode_step(ids[:, 0], torch.full((1, 1), 20, dtype=torch.long, device="cuda"), caches)
        assert torch.isfinite(out.float()).all()


def test_decode_step_with_adapters_has_no_host_sync():
    from unsloth_spectral import LogitsRules, LoraAdapters
    model, shape, g = _model(torch.float16, seed=5)
    ad = LoraAdapters(model, max_rank=8, slots=2)
    ad.load(1, _weights(model, g, 8, torch.float16))
    rules = LogitsRules(2, shape.vocab, presence_penalty=1.0)
    prompt = torch.randint(0, shape.vocab, (2, 560), generator=g, device="cuda")
    ad.use([1, -1])
    with torch.no_grad():
        logits, caches = model.prefill(prompt)
        pos = torch.full((1, 1), 560, dtype=torch.long, device="cuda")
        tok = rules.pick(model.decode_step(rules.pick(logits, record=True), pos, caches), record=True)
        pos += 1
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            tok = rules.pick(model.decode_step(tok, pos, caches), record=True)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        torch.cuda.synchronize()
    assert int(tok.min()) >= 0


def test_refusals():
    from unsloth_spectral import LogitsRules, LoraAdapters
    model, shape, g = _model(torch.float16, layers=1)
    ids = torch.zeros(2, 4, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError):
        LoraAdapters(model, targets=("q_proj", "lm_head"))
    ad = LoraAdapters(model, max_rank=4, slots=2, targets=("q_proj", "o_proj"))
    with pytest.raises(KeyError):
        ad.load(0, {(0, "up_proj"): (torch.zeros(1, 512), torch.zeros(1024, 1))})
    with pytest.raises(IndexError):
        ad.use([0, 2])
    for kw in (dict(adapters=ad), dict(adapters=ad, adapter_slots=[0]), dict(adapter_slots=[0, 0]),
               dict(allow=torch.zeros(2, 32, dtype=torch.int32, device="cuda")), dict(rules=LogitsRules(3, shape.vocab)),
               dict(rules=LogitsRules(2, 999))):
        with pytest.raises(ValueError):
            model.generate(ids, 2, **kw)
    ad.use([0, 1])
    with pytest.raises(RuntimeError):        # no gradients through the adapters
        at = model.model.layers[0].self_attn
        at.forward(torch.zeros(2, 4, 512, device="cuda", dtype=torch.float16), use_cache=True)
    ad.use(None)
