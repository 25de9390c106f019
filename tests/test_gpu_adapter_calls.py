"""Calls of the adapters that their documentation allows and that differ in form, not in what they
compute: results are those of the plain call."""
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]


def _pool(g, K=256, W=136, dtype=torch.bfloat16, slots=2, rank=16):
    from unsloth_spectral import LoraPool
    pool = LoraPool(K, W, max_rank=rank, slots=slots, dtype=dtype)
    for s in range(slots):
        pool.load(s, torch.randn(rank, K, generator=g, device="cuda") / K ** 0.5,
                  torch.randn(W, rank, generator=g, device="cuda") * 0.1, 0.5 + s)
    return pool


@pytest.mark.parametrize("T", [1, 70])
@pytest.mark.parametrize("waited", [False, True])
def test_a_batch_is_prepared_again_inside_a_capture(T, waited):
    """Grouped before the capture (and waited for, or not yet): preparing it again there is no work."""
    from unsloth_spectral import LoraBatch
    g = torch.Generator(device="cuda").manual_seed(T)
    pool = _pool(g)
    x, y = (torch.randn(2, T, n, generator=g, device="cuda").bfloat16() for n in (256, 136))
    want = pool.add(y, x, LoraBatch([1, 0]))
    batch = LoraBatch([1, 0])
    for _ in range(2 if waited else 1):
        batch.prepare(T) if waited else pool.add(y, x, batch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if T == 1 or waited:       # all that prepare() groups for T tokens is there
            batch.prepare(T)
        out = pool.add(y, x, batch)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_one_row_of_wider_rows_off_16_bytes():
    """One row has no distance to another: views of rows whose width is no multiple of 8."""
    from unsloth_spectral import LoraBatch
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = _pool(g)
    x, y = (torch.randn(1, 1, n, generator=g, device="cuda").bfloat16() for n in (256, 136))
    want = pool.add(y, x, LoraBatch([1]))
    for shape in ((1, 1, 303), (1, 303)):
        n = len(shape)
        xw, yw, ow = (torch.full(shape, 2.0, dtype=torch.bfloat16, device="cuda") for _ in range(3))
        xv, yv, ov = xw[..., :256], yw[..., 8:144], ow[..., 16:152]
        xv.copy_(x.view(xv.shape)), yv.copy_(y.view(yv.shape))
        got = pool.add(yv, xv, LoraBatch([1]), out=ov)
        assert got.dim() == n and torch.equal(got.flatten(), want.flatten())
        assert (ow[..., :16] == 2).all() and (ow[..., 152:] == 2).all()
        assert torch.equal(pool.add(yv, xv, LoraBatch([1])).flatten(), want.flatten())
