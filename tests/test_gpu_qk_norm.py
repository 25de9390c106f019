"""spx_qk_norm_rope against the formula in 64 bits.

Tolerance, per value: half a step of the output type, eps/2 * |ref| (plus half the smallest
float16 step, 2^-25, below its normal range), and what float32 inside may add.  A lane adds
at most 32 squares one after another and five more sums meet over the lanes (37 roundings,
halved by the square root); rsqrtf is within 2 ulp = 4 u (u = 2^-24), the mean and the sum
with eps 2 u (halved), the two products to y 2 u, the rotation's product and sum 2 u:
19 + 4 + 1 + 2 + 2 < 32 u, of |y1| + |y2|."""
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

DT = [torch.float32, torch.float16, torch.bfloat16]


def _tables(n, D, dev="cuda"):
    inv = 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
    f = torch.outer(torch.arange(n, dtype=torch.float64, device=dev), inv)
    f = torch.cat([f, f], -1)
    return f.cos().float(), f.sin().float()


def _ref(x, w, cos, sin, pos, eps, turn):
    """(value, |y1| + |y2|) in 64 bits, head-major."""
    B, T, n = x.shape
    D = w.shape[0]
    h = D // 2
    y = x.double().view(B, T, n // D, D)
    y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / D + eps) * w.double()
    y = y.transpose(1, 2)
    a, b = y[..., :h], y[..., h:]
    mag = torch.cat([a.abs() + b.abs()] * 2, -1)
    if turn:
        c = cos.double()[pos][:, None, :, :h]
        s = sin.double()[pos][:, None, :, :h]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return y, mag


def _check(got, ref, mag, dt):
    tol = torch.finfo(dt).eps / 2 * ref.abs() + 32 * 2.0 ** -24 * mag + (2.0 ** -25 if dt == torch.float16 else 0.0)
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.double() - ref).abs() - tol).max()))


SHAPES = [(1, 1, 32, 8, 128), (3, 1, 32, 8, 128), (64, 1, 5, 1, 64), (2, 37, 9, 3, 80), (1, 700, 4, 4, 96), (2, 5, 2, 1, 256),
          (1, 3, 7, 2, 512), (2, 3, 3, 1, 1024), (2, 9, 3, 2, 2), (1, 4, 5, 5, 6), (2, 3, 4, 2, 16), (1, 11, 6, 2, 48),
          (1, 2, 1, 1, 32), (300, 9, 3, 1, 128), (1, 33, 5, 2, 144), (3, 11, 4, 2, 160), (2, 301, 3, 1, 112),
          (8, 2049, 5, 2, 80), (3, 4001, 3, 1, 96), (2, 2400, 13, 3, 64)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
def test_against_the_formula(dtype, B, T, Hq, H, D):
    from unsloth_spectral import qk_norm_rope
    g = torch.Generator(device="cuda").manual_seed(B * 1000 + T * 10 + D)
    packed = (torch.randn(B, T, (Hq + 2 * H) * D, generator=g, device="cuda") * 2).to(dtype)
    q, k = packed[..., :Hq * D], packed[..., Hq * D:(Hq + H) * D]
    qw = torch.randn(D, generator=g, device="cuda").to(dtype)
    kw = torch.randn(D, generator=g, device="cuda").to(dtype)
    cos, sin = _tables(2 * T + 50, D)
    for eps, turn, pos in ((1e-6, False, torch.arange(T, device="cuda")[None] + 7),
                           (1e-2, True, torch.randint(0, 2 * T + 50, (B, T), generator=g, device="cuda"))):
        qo, ko = qk_norm_rope(q, k, qw, kw, cos, sin, pos, eps=eps, rotate_keys=turn)
        assert qo.shape == (B, Hq, T, D) and ko.shape == (B, H, T, D) and qo.dtype == ko.dtype == dtype
        _check(qo, *_ref(q, qw, cos, sin, pos.expand(B, T), eps, True), dtype)
        _check(ko, *_ref(k, kw, cos, sin, pos.expand(B, T), eps, turn), dtype)


@pytest.mark.parametrize("dtype", DT)
def test_layouts_and_positions(dtype):
    """Misaligned and strided inputs, queries alone, every form of positions, positions past
    the table (clamped), empty batches."""
    from unsloth_spectral import qk_norm_rope
    g = torch.Generator(device="cuda").manual_seed(2)
    B, T, Hq, H, D = 2, 6, 4, 2, 64
    cos, sin = _tables(40, D)
    w = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dtype)
    flat = torch.randn(B * T * Hq * D + 8, generator=g, device="cuda").to(dtype)
    odd = flat[1:1 + B * T * Hq * D].view(B, T, Hq * D)                     # off 16 bytes
    apart = torch.randn(T, B, Hq * D, 2, generator=g, device="cuda").to(dtype)[..., 0].transpose(0, 1)
    swapped = torch.randn(T, B, Hq * D, generator=g, device="cuda").to(dtype).transpose(0, 1)
    ar = torch.arange(T, device="cuda")
    wide = torch.arange(B * 3 * T, device="cuda").view(B, 3 * T)[:, ::3] % 40
    for q in (odd, apart, swapped):
        for pos, at in ((5, (ar + 5)[None]), (ar + 3, (ar + 3)[None]), (wide, wide), (wide[:1], wide[:1]),
                        (ar + 36, (ar + 36).clamp(max=39)[None]), (ar - 2, (ar - 2).clamp(min=0)[None]),
                        (38, (ar + 38).clamp(max=39)[None])):
            qo, ko = qk_norm_rope(q, None, w, None, cos, sin, pos)
            assert ko is None
            _check(qo, *_ref(q, w, cos, sin, at.expand(B, T), 1e-6, True), dtype)
    odd_w = torch.cat([w[:1], w])[1:]
    k = flat[8:8 + B * T * H * D].view(B, T, H * D)
    qo, ko = qk_norm_rope(swapped, k, odd_w, w, cos, sin, 0)
    _check(qo, *_ref(swapped, w, cos, sin, ar[None].expand(B, T), 1e-6, True), dtype)
    _check(ko, *_ref(k, w, cos, sin, None, 1e-6, False), dtype)
    for b, t in ((0, 3), (3, 0)):
        e = torch.empty(b, t, Hq * D, dtype=dtype, device="cuda")
        qo, ko = qk_norm_rope(e, e, w, w, cos, sin, 0)
        assert qo.shape == (b, Hq, t, D) and ko.shape == (b, Hq, t, D)
    with pytest.raises(ValueError):
        qk_norm_rope(swapped, None, w, None, cos, sin, ar.int())
    with pytest.raises(ValueError):
        qk_norm_rope(swapped, None, w, None, cos, sin, ar[:-1])
    with pytest.raises(ValueError):
        qk_norm_rope(swapped, None, w, None, cos[:, :32], sin[:, :32], ar)
    with pytest.raises(ValueError):
        qk_norm_rope(swapped, k.cpu(), w, w, cos, sin, ar)


def test_values_out_of_the_ordinary_stay_in_their_head():
    from unsloth_spectral import qk_norm_rope
    B, T, Hq, D = 1, 2, 6, 128
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(B, T, Hq * D, generator=g, device="cuda").to(torch.bfloat16)
    clean = x.clone()
    x[0, 0, 3] = float("inf")
    x[0, 0, 2 * D + 70] = float("nan")
    x[0, 1, 4 * D:5 * D] = 0
    w = torch.ones(D, device="cuda", dtype=torch.bfloat16)
    cos, sin = _tables(8, D)
    a, _ = qk_norm_rope(x, None, w, None, cos, sin, 1)
    b, _ = qk_norm_rope(clean, None, w, None, cos, sin, 1)
    assert a[0, 2, 0].isnan().all() and a[0, 0, 0].isnan().any()
    assert not a[0, 4, 1].any()
    keep = torch.ones(Hq, T, dtype=torch.bool)
    keep[0, 0] = keep[2, 0] = keep[4, 1] = False
    assert torch.equal(a[0][keep.cuda()], b[0][keep.cuda()])


def test_streams_and_graphs():
    """Work goes to the current stream; a captured call replays on new inputs."""
    from unsloth_spectral import qk_norm_rope
    g = torch.Generator(device="cuda").manual_seed(4)
    B, T, Hq, H, D = 4, 1, 8, 2, 128
    q = torch.randn(B, T, Hq * D, generator=g, device="cuda").half()
    k = torch.randn(B, T, H * D, generator=g, device="cuda").half()
    w = torch.randn(D, generator=g, device="cuda").half()
    pos = torch.randint(0, 30, (B, T), generator=g, device="cuda")
    cos, sin = _tables(32, D)
    want = qk_norm_rope(q, k, w, w, cos, sin, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = qk_norm_rope(q, k, w, w, cos, sin, pos)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qk_norm_rope(q, k, w, w, cos, sin, pos)
    q.copy_(q.flip(0))
    pos.copy_(pos.flip(0))
    graph.replay()
    assert torch.equal(out[0], want[0].flip(0)) and not torch.equal(out[1], want[1].flip(0))
