"""Which q_norm / k_norm modules the patched forwards hand to the fused kernel, and how they run
the others (no GPU)."""
from types import SimpleNamespace

import pytest
import torch

from unsloth_spectral import integration as I
from unsloth_spectral.llama_loop import RMSNorm

D = 16


class Norm(torch.nn.Module):
    """A norm of head vectors that names its epsilon as the usual one does."""

    def __init__(self, dtype=torch.float32, dim=D, eps=1e-6, fill=None):
        super().__init__()
        w = torch.linspace(0.5, 1.5, dim) if fill is None else torch.full((dim,), fill)
        self.weight = torch.nn.Parameter(w.to(dtype))
        self.variance_epsilon = eps

    def scaled(self, y):
        return y.to(self.weight.dtype) * self.weight

    def forward(self, x):
        y = x.float()
        return self.scaled(y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.variance_epsilon))


class RoundedOnce(Norm):
    def scaled(self, y):
        return (y * self.weight.float()).to(self.weight.dtype)


class Centered(Norm):          # a layer norm
    def forward(self, x):
        y = x.float()
        y = y - y.mean(-1, keepdim=True)
        return self.scaled(y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.variance_epsilon))


class Plus(Norm):
    def scaled(self, y):
        return (y * (1 + self.weight.float())).to(self.weight.dtype)


class Biased(Norm):
    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        self.bias = torch.nn.Parameter(torch.zeros_like(self.weight))

    def scaled(self, y):
        return super().scaled(y) + self.bias


class NoEpsilon(Norm):
    def forward(self, x):
        y = x.float()
        return self.scaled(y * torch.rsqrt(y.square().mean(-1, keepdim=True)))


class Outside(Norm):           # epsilon beside the root
    def forward(self, x):
        y = x.float()
        return self.scaled(y / (y.square().mean(-1, keepdim=True).sqrt() + self.variance_epsilon))


class L2(Norm):                # of the length, not of the mean
    def forward(self, x):
        y = x.float()
        return self.scaled(y * torch.rsqrt(y.square().sum(-1, keepdim=True) + self.variance_epsilon))


class Refuses(Norm):
    def forward(self, x):
        raise RuntimeError("not with these shapes")


def _of(q, k, dtype=torch.float32):
    return I._head_norms(SimpleNamespace(q_norm=q, k_norm=k), D, torch.zeros(1, 1, 2 * D, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("eps", [1e-6, 1e-5, 1e-12])
@pytest.mark.parametrize("kind", [Norm, RoundedOnce])
def test_the_usual_norm_is_recognised(dtype, eps, kind):
    q, k = kind(dtype, eps=eps), kind(dtype, eps=eps, fill=0.25)
    for _ in range(2):
        got = _of(q, k, dtype)
        assert got[0] is q.weight and got[1] is k.weight and got[2] == eps
    q, k = (RMSNorm(D, eps, "cpu", dtype) for _ in range(2))
    assert _of(q, k, dtype) == (q.weight, k.weight, eps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fill", [None, 0.0, 1.0])
@pytest.mark.parametrize("kind", [Centered, Plus, Biased, NoEpsilon, Outside, L2, Refuses])
def test_other_norms_run_their_own_code(dtype, fill, kind):
    if fill == 0.0 and kind is not Plus and kind is not Biased and kind is not Refuses:
        pytest.skip("every value is zero, as with the usual norm")
    usual, other = Norm(dtype), kind(dtype, fill=fill)
    for _ in range(2):
        assert _of(usual, other, dtype) is None and _of(other, usual, dtype) is None


def test_a_changed_norm_is_asked_again():
    q, k = Norm(), Norm()
    assert _of(q, k) is not None
    q.variance_epsilon = k.variance_epsilon = 1e-5
    assert _of(q, k)[2] == 1e-5
    k.__class__ = Centered
    assert _of(q, k) is None
    k.__class__ = Norm
    assert _of(q, k) is not None
    k.forward = Centered.forward.__get__(k)      # a forward of the instance's own
    assert _of(q, k) is None


def test_hooks_on_a_norm_are_called():
    for register in ("register_forward_hook", "register_forward_pre_hook"):
        q, k = Norm(), Norm()
        handle = getattr(k, register)(lambda *a: None)
        assert _of(q, k) is None
        handle.remove()
        assert _of(q, k) is not None


class _HeadsOwn(torch.nn.Module):
    """A norm of each head with weights of each head's own, [heads, head_dim]."""

    def __init__(self, heads):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.linspace(0.5, 2.0, heads * D).view(heads, D))

    def forward(self, x):
        return torch.nn.functional.layer_norm(x, (D,)) * self.weight


class _Rows(torch.nn.Module):
    """A norm of whole projection rows."""

    def __init__(self, n):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.linspace(0.5, 2.0, n))

    def forward(self, x):
        assert x.shape[-1] == len(self.weight)
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * self.weight


@pytest.mark.parametrize("heads", [1, 3])
def test_own_norms_of_heads_and_of_rows(heads):
    x = torch.randn(2, 5, heads * D, generator=torch.Generator().manual_seed(heads))
    split = lambda y: y.view(2, 5, heads, D).transpose(1, 2)  # noqa: E731
    for norm, want in ((_HeadsOwn(heads), lambda n: split(n(x.view(2, 5, heads, D)))), (_Rows(heads * D), lambda n: split(n(x))),
                       (Norm(), lambda n: split(n(x.view(2, 5, heads, D)))),
                       (torch.nn.LayerNorm((heads, D)), lambda n: split(n(x.view(2, 5, heads, D))))):
        got = I._own_norm(norm, x, heads, D)
        assert got.shape == (2, heads, 5, D) and torch.equal(got, want(norm))


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on the GPU: for the choice of a path, not for a launch."""

    is_cuda = property(lambda self: True)


def _choice(monkeypatch, positions, prepare=lambda q, k: (q, k), norms=None):
    """What ``_normed_qk`` does with a query and a key of two heads each: the arguments that it hands
    to the fused kernel (None: the modules' own norms), and its results."""
    seen = []
    monkeypatch.setattr(I, "qk_norm_rope", lambda *a, **kw: seen.append((a, kw)) or ("q", "k"))
    g = torch.Generator().manual_seed(0)
    q, k = prepare(torch.randn(2, 3, 2 * D, generator=g), torch.randn(2, 3, 2 * D, generator=g))
    mod = SimpleNamespace(q_norm=(norms or [Norm()])[0], k_norm=(norms or [Norm()])[-1])
    tab = torch.linspace(0, 1, 20 * D).view(20, D)
    out = I._normed_qk(mod, q.as_subclass(_Cuda), k.as_subclass(_Cuda), 2, 2, D, tab.cos(), tab.sin(), positions)
    return (seen[0] if seen else None), out


def test_gradients_take_the_modules_own_norms(monkeypatch):
    pos = torch.arange(3)[None]
    frozen = [Norm().requires_grad_(False) for _ in range(2)]
    with torch.no_grad():
        for q, k in ((False, False), (True, True)):
            assert _choice(monkeypatch, pos, lambda x, y: (x.requires_grad_(q), y.requires_grad_(k)))[0] is not None
    assert _choice(monkeypatch, pos, norms=frozen)[0] is not None
    for q, k in ((True, False), (False, True)):
        used, (qo, ko) = _choice(monkeypatch, pos, lambda x, y: (x.requires_grad_(q), y.requires_grad_(k)), frozen)
        assert used is None and qo.requires_grad == q and ko.requires_grad == k
    used, (qo, ko) = _choice(monkeypatch, pos)             # of the norms' weights alone
    assert used is None and qo.requires_grad and ko.requires_grad


@pytest.mark.parametrize("dtype", [torch.int32, torch.int16, torch.int64])
@pytest.mark.parametrize("rows", [1, 2])
def test_positions_of_any_whole_type_are_taken(monkeypatch, dtype, rows):
    pos = torch.arange(4, 4 + 3 * rows).view(rows, 3)
    with torch.no_grad():
        (args, _), _ = _choice(monkeypatch, pos.to(dtype))
        assert args[6].dtype == torch.int64 and torch.equal(args[6], pos)
        want = _choice(monkeypatch, pos, norms=[Centered(), Centered()])[1]
        got = _choice(monkeypatch, pos.to(dtype), norms=[Centered(), Centered()])[1]
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        (args, _), _ = _choice(monkeypatch, 4)
        assert args[6] == 4


@pytest.mark.parametrize("dtype,dim", [(torch.float64, D), (torch.float32, 1026)])
def test_what_the_fused_kernel_does_not_take_runs_the_modules_norms(monkeypatch, dtype, dim):
    monkeypatch.setattr(I, "qk_norm_rope", lambda *a, **kw: pytest.fail("handed to the kernel"))
    norm, x = Norm(dtype, dim), torch.linspace(-1, 1, 2 * 2 * dim, dtype=dtype).view(1, 2, 2 * dim)
    tab = torch.zeros(4, dim)
    with torch.no_grad():
        q, k = I._normed_qk(SimpleNamespace(q_norm=norm, k_norm=norm), x.as_subclass(_Cuda), x.as_subclass(_Cuda), 2, 2, dim,
                            tab.cos(), tab.sin(), 0)
        want = norm(x.view(1, 2, 2, dim)).transpose(1, 2)
    assert k.dtype == dtype and torch.equal(k.as_subclass(torch.Tensor), want)
    assert torch.equal(q.as_subclass(torch.Tensor), want.float().to(dtype))      # cos 1, sin 0; rotated in float32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("positions", [7, torch.tensor([[4, 0, 9]]), torch.tensor([[4, 5, 6], [19, 2, 40]])])
def test_only_the_rows_in_use_of_tables_in_another_type_are_converted(monkeypatch, dtype, positions):
    """A rotary module's tables in the model's type: thousands of rows, of which a step needs a few."""
    seen = []
    monkeypatch.setattr(I, "qk_norm_rope", lambda *a, **kw: seen.append(a))
    x = torch.zeros(2, 3, 2 * D).as_subclass(_Cuda)
    ang = torch.outer(torch.arange(20.0), torch.linspace(0.1, 1, D))
    cos, sin = ang.cos().to(dtype), ang.sin().to(dtype)
    with torch.no_grad():
        I._normed_qk(SimpleNamespace(q_norm=Norm(), k_norm=Norm()), x, x, 2, 2, D, cos, sin, positions)
    c, s, at = (v.as_subclass(torch.Tensor) for v in seen[0][4:7])
    idx = torch.arange(7, 10)[None] if isinstance(positions, int) else positions.clamp(max=19)     # clamped to the tables
    assert c.dtype == s.dtype == torch.float32 and len(c) == len(s) == idx.numel() and at.dtype == torch.int64
    assert c.is_contiguous() and s.is_contiguous() and at.shape == idx.shape
    assert torch.equal(c[at], cos[idx].float()) and torch.equal(s[at], sin[idx].float())


@pytest.mark.parametrize("before", [0.0, float("nan")])
def test_weights_that_say_nothing_are_not_an_answer(before):
    """Asked before its weights are there, a norm runs its own code, and is asked again."""
    q, k = Centered(fill=before), Centered(fill=before)
    assert _of(q, k) is None
    for norm in (q, k):
        norm.weight.data.fill_(1.0)
    assert _of(q, k) is None
    q, k = Norm(fill=before), Norm(fill=before)
    assert _of(q, k) is None
    for norm in (q, k):
        norm.weight.data.fill_(1.0)
    assert _of(q, k) is not None
