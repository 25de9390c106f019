"""Patched forwards of attention modules with q_norm / k_norm on the GPU: which path their norms take,
and its results, gradients and positions."""
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

B, T, HQ, H, D = 2, 6, 4, 2, 64


class Norm(torch.nn.Module):
    """The usual norm of each head under another name, and the same with the mean taken off."""

    def __init__(self, dtype, centered=False):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.linspace(0.5, 1.5, D, device="cuda").to(dtype))
        self.variance_epsilon, self.centered = 1e-6, centered

    def forward(self, x):
        y = x.float()
        if self.centered:
            y = y - y.mean(-1, keepdim=True)
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.variance_epsilon)
        return y.to(x.dtype) * self.weight


class Module:
    def __init__(self, dtype, centered=False):
        self.q_norm, self.k_norm = Norm(dtype, centered), Norm(dtype, centered)


def _tables(n, dtype=torch.float32):
    f = torch.outer(torch.arange(n, dtype=torch.float64), 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    f = torch.cat([f, f], -1).cuda()
    return f.cos().to(dtype), f.sin().to(dtype)


def _formula(x, w, heads, cos, sin, pos, eps, centered, turn):
    """In 64 bits, of ``x`` [B, T, heads * D]; differentiable."""
    y = x.double().view(B, T, heads, D)
    if centered:
        y = y - y.mean(-1, keepdim=True)
    y = (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()).transpose(1, 2)
    if not turn:
        return y
    c, s = (t.double()[pos][:, None, :, :D // 2] for t in (cos, sin))
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _inputs(dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(B, T, n * D, generator=g, device="cuda").to(dtype) for n in (HQ, H)]


def _spy(monkeypatch):
    from unsloth_spectral import integration as I
    real, calls = I.qk_norm_rope, []
    monkeypatch.setattr(I, "qk_norm_rope", lambda *a, **kw: calls.append(1) or real(*a, **kw))
    return I, calls


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("centered", [False, True])
@pytest.mark.parametrize("tables", [torch.float32, torch.bfloat16])
def test_results_whichever_path_a_norm_takes(monkeypatch, dtype, centered, tables):
    """Own norms round up to three times (after the norm, the weight, the rotation, whose two terms
    are each off by the first two), half a step each, of values up to the pair's length:
    3 * eps / 2 * sqrt(2) of it, and float32 sums (2^-20)."""
    I, calls = _spy(monkeypatch)
    mod, (q, k) = Module(dtype, centered), _inputs(dtype)
    cos, sin = _tables(40, tables)
    for pos in (torch.arange(5, 5 + T, device="cuda")[None], torch.randint(0, 40, (B, T), device="cuda"), 5):
        for kind in (torch.int64, torch.int32):
            at = pos.to(kind) if isinstance(pos, torch.Tensor) else pos
            idx = pos if isinstance(pos, torch.Tensor) else torch.arange(5, 5 + T, device="cuda")[None]
            with torch.no_grad():
                qo, ko = I._normed_qk(mod, q, k, HQ, H, D, cos, sin, at)
                refs = [_formula(x, n.weight, h, cos, sin, idx, 1e-6, centered, turn) for x, n, h, turn in
                        ((q, mod.q_norm, HQ, True), (k, mod.k_norm, H, False))]
            for got, ref in zip((qo, ko), refs):
                a, b = ref[..., :D // 2], ref[..., D // 2:]
                size = torch.sqrt(a * a + b * b).repeat(1, 1, 1, 2)
                tol = (1.5 * torch.finfo(dtype).eps + 2.0 ** -20) * 2 ** 0.5 * size + torch.finfo(dtype).tiny
                assert got.dtype == dtype and got.shape == ref.shape
                assert ((got.double() - ref).abs() <= tol).all()
    assert len(calls) == (0 if centered else 6)


def test_gradients_against_the_formulas_and_differences(monkeypatch):
    """float32 on the GPU against autograd of the 64-bit formula (float32 sums of D terms, a few
    operations each: 64 * 2^-24 of the gradient's size), and that against central differences in
    64 bits (step 1e-5: h^2 and 1e-16 / h, under 1e-8 of values near 1, a thousand terms)."""
    I, calls = _spy(monkeypatch)
    mod, (q, k) = Module(torch.float32), _inputs(torch.float32, 1)
    cos, sin = _tables(40)
    pos = torch.randint(0, 40, (B, T), device="cuda")
    q.requires_grad_(), k.requires_grad_()
    g = torch.Generator(device="cuda").manual_seed(2)
    ups = [torch.randn(B, h, T, D, generator=g, device="cuda") for h in (HQ, H)]
    outs = I._normed_qk(mod, q, k, HQ, H, D, cos, sin, pos)
    assert not calls
    leaves = (q, k, mod.q_norm.weight, mod.k_norm.weight)
    got = torch.autograd.grad(outs, leaves, ups)
    q64, k64, wq, wk = (t.detach().double().requires_grad_() for t in leaves)
    refs = lambda: (_formula(q64, wq, HQ, cos, sin, pos, 1e-6, False, True),  # noqa: E731
                    _formula(k64, wk, H, cos, sin, pos, 1e-6, False, False))
    want = torch.autograd.grad(refs(), (q64, k64, wq, wk), [u.double() for u in ups])
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) <= 64 * 2.0 ** -24
    with torch.no_grad():
        for leaf, grad in zip((q64, k64, wq, wk), want):
            way = torch.randn(leaf.shape, generator=g, device="cuda", dtype=torch.float64)
            sides = []
            for h in (1e-5, -1e-5):
                leaf.add_(way, alpha=h)
                sides.append(sum((r * u.double()).sum() for r, u in zip(refs(), ups)))
                leaf.add_(way, alpha=-h)
            assert abs(float((sides[0] - sides[1]) / 2e-5 - (grad * way).sum())) <= 1e-5


def test_a_norm_that_was_never_asked_is_captured_with_its_own_code(monkeypatch):
    I, calls = _spy(monkeypatch)
    mod, (q, k) = Module(torch.float16), _inputs(torch.float16, 3)
    cos, sin = _tables(40)
    pos = torch.arange(T, device="cuda")[None]
    with torch.no_grad():
        mod.q_norm(q.view(B, T, HQ, D))       # the allocator and the module's kernels are there
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            own = I._normed_qk(mod, q, k, HQ, H, D, cos, sin, pos)
        assert not calls
        graph.replay()
        fused = I._normed_qk(mod, q, k, HQ, H, D, cos, sin, pos)
        assert calls
        torch.cuda.synchronize()
        for a, b in zip(own, fused):          # three roundings against one, each half a step of values up to 3 * 8
            assert float((a.float() - b.float()).abs().max()) <= 4 * 2.0 ** -11 * float(b.float().abs().max()) * 2 ** 0.5


def test_forwards_with_gradients_on_and_with_other_positions(monkeypatch):
    """A prompt and a token through both patched forwards: with autograd on (own norms) as with it off
    (the kernel), with int32 positions as with int64 ones.  Own norms round twice more, two half
    steps of queries and keys each: scores (up to sqrt(128) * 1.5^2 = 25) off by 4 * 2^-11 * 25 =
    0.05, so the weights of a softmax by up to 5 % each way, and the outputs by 0.1 of their size."""
    from unsloth_spectral.llama_loop import LlamaShape, SpectralLlama
    shape = LlamaShape(layers=1, hidden=256, heads=4, kv_heads=2, head_dim=128, ffn=256, vocab=100, qk_norm=True)
    model = SpectralLlama(shape, device="cuda", dtype=torch.float16, std=0.1, seed=1)
    model.patch(block_size=512, k_rank_keys=16, k_rank_values=16)
    at = model.model.layers[0].self_attn
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(2, 30, 256, generator=g, device="cuda").half()
    one = torch.randn(2, 1, 256, generator=g, device="cuda").half()
    mask = torch.full((30, 30), float("-inf"), device="cuda", dtype=torch.float16).triu_(1)[None, None]
    runs = {}
    for grad in (False, True):
        for kind in (torch.int64, torch.int32):
            pos = torch.arange(30, device="cuda")[None].to(kind)
            at._spectral_cache = None
            with torch.set_grad_enabled(grad):
                a, _, cache = at.forward(x, attention_mask=mask, position_ids=pos, use_cache=True)
                b, _ = at._spx_inference(one, cache, torch.full((1, 1), 30, device="cuda", dtype=kind))
            runs[grad, kind] = (a.detach().float(), b.detach().float())
    at._spectral_cache = None
    for grad in (False, True):
        for u, v in zip(runs[grad, torch.int64], runs[grad, torch.int32]):
            assert torch.equal(u, v)
    for u, v in zip(runs[False, torch.int64], runs[True, torch.int64]):
        assert float((u - v).norm() / v.norm()) <= 0.1
