"""LoraPool.add against ``y + scale * B (A x)`` in 64 bits.

Tolerance, per value of out: half a step of the type on the result, eps/2 * |ref| (plus
2^-25 below float16's normal range).  The inner product t is summed in float32 by matrix
instructions of 16 products: each may drop what lies under 2^-23 of the largest term or
partial sum, itself at most S = sum |a x|, for each of the (K + 31) / 32 * 2 instructions and
the 24 sums over warps and CTAs: dt <= (K / 16 + 26) * 2^-23 * S.  t is then held in two values of the type,
within (eps/2)^2 of it (float16: of the row's largest, which the scaling makes normal), and
the second product and the sum with y round like the first:
scale * (sum |B| (dt + (eps/2)^2 |t|max) + (rank / 8 + 4) * 2^-23 * sum |B| |t|) + 2^-23 |y|."""
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]


def _adapters(g, slots, K, widths, ranks, dt):
    """ranks[slot]: one rank or one for each part (0: nothing loaded)."""
    from unsloth_spectral import LoraPool
    top = max(max(r) if isinstance(r, tuple) else r for r in ranks)
    pool = LoraPool(K, widths, max_rank=max(top, 1), slots=slots, dtype=dt)
    held = {}
    for s in range(slots):
        for p, w in enumerate(widths):
            r = ranks[s][p] if isinstance(ranks[s], tuple) else ranks[s]
            if r:
                A = (torch.randn(r, K, generator=g, device="cuda") / K ** 0.5).to(dt)
                B = (torch.randn(w, r, generator=g, device="cuda") * 0.1).to(dt)
                held[s, p] = (A, B, 0.5 + s)
                pool.load(s, A, B, 0.5 + s, p)
    return pool, held


def _ref(y, x, held, ids, widths):
    ref, tol = y.double(), y.double().abs() * 2.0 ** -23
    eps = torch.finfo(y.dtype).eps
    K = x.shape[-1]
    for b, s in enumerate(ids):
        at = 0
        for p, w in enumerate(widths):
            if (s, p) in held:
                A, B, sc = held[s, p]
                A, B, xb = A.double(), B.double(), x[b].double()
                t = xb @ A.T
                dt = (K / 16 + 26) * 2.0 ** -23 * (xb.abs() @ A.abs().T) + (eps / 2) ** 2 * t.abs().amax(-1, keepdim=True)
                ref[b, ..., at:at + w] += sc * (t @ B.T)
                tol[b, ..., at:at + w] += sc * (dt @ B.abs().T + (A.shape[0] / 8 + 4) * 2.0 ** -23 * (t.abs() @ B.abs().T))
            at += w
    tol += eps / 2 * ref.abs() + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    return ref, tol


def _check(got, ref, tol):
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.double() - ref).abs() / tol).max()))


CASES = [
    # B, T, K, widths, ranks by slot, slots of the sequences
    (1, 1, 4096, (4096, 1024, 1024), [16], [0]),
    (1, 1, 8, (8,), [1], [0]),
    (5, 1, 264, (72, 40), [(3, 16), (16, 0), 5], [2, 0, -1, 1, 0]),
    (33, 1, 1000, (520,), [8, 64, 33], [i % 3 for i in range(33)]),
    (40, 1, 512, (136,), [16], [0] * 40),
    (64, 1, 14336, (256,), [64, 7, 0, 20], [i % 5 - 1 for i in range(64)]),
    (3, 7, 96, (64, 8, 16, 200), [(1, 2, 3, 4), 4], [1, 0, 1]),
    (2, 45, 2056, (1032,), [96, 128], [1, 0]),
    (2, 33, 512, (320, 64), [80, 70], [0, 1]),
    (4, 100, 256, (512,), [40, 48], [-1, 1, 1, 0]),
    (2, 300, 4096, (520, 128, 128), [64, 32], [1, 0]),
    (1, 515, 40, (24,), [24], [0]),
    # blocks of adjacent rows: ragged tiles and parts, every stored rank
    (3, 3137, 2056, (1520, 128, 136), [16, (5, 0, 16)], [1, 0, -1]),
    (2, 4500, 1048, (1000,), [32, 20], [0, 1]),
    (1, 6100, 64, (2056, 8), [48], [0]),
    (2, 1100, 4096, (264, 64, 64), [64, 33], [1, 0]),
    (5, 700, 1024, (1400,), [128, 80, 3], [2, 1, 0, -1, 1]),
    (64, 64, 4104, (4136,), [16, 9], [i % 3 - 1 for i in range(64)]),
    (2, 530, 14336, (18000,), [7, 16], [0, 1]),
    (160, 64, 4104, (4136,), [16, 9], [i % 3 - 1 for i in range(160)]),
    (50, 120, 6000, (640,), [16, 9], [i % 3 - 1 for i in range(50)]),
    (100, 128, 2056, (1000,), [16, 9], [i % 3 - 1 for i in range(100)]),
    (30, 127, 4096, (136, 128, 72), [64, 50], [i % 3 - 1 for i in range(30)]),
    (2, 128, 8192, (1032,), [64, 30], [0, 1]),
    (19, 200, 1912, (1520, 128, 136), [64, (5, 0, 64), 9], [i % 4 - 1 for i in range(19)]),
    (4, 112, 14152, (488, 40, 1000), [24, 9], [1, 0, -1, 0]),
    (3, 1, 8200, (264, 16), [24, (16, 0)], [1, 0, -1]),
    (40, 1, 4608, (1000,), [16], [0] * 40),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_formula(dtype, case):
    from unsloth_spectral import LoraBatch
    B, T, K, widths, ranks, ids = CASES[case]
    g = torch.Generator(device="cuda").manual_seed(case)
    pool, held = _adapters(g, len(ranks), K, widths, ranks, dtype)
    x = torch.randn(B, T, K, generator=g, device="cuda").to(dtype)
    y = torch.randn(B, T, sum(widths), generator=g, device="cuda").to(dtype)
    keep = y.clone()
    batch = LoraBatch(ids)
    out = pool.add(y, x, batch)
    assert torch.equal(y, keep) and out.shape == y.shape
    ref, tol = _ref(y, x, held, ids, widths)
    _check(out, ref, tol)
    for b, s in enumerate(ids):
        if not any((s, p) in held for p in range(len(widths))):
            assert torch.equal(out[b], y[b])
    assert torch.equal(pool.add(y, x, batch), out)                # the same every time
    assert pool.add(y, x, batch, out=y) is y and torch.equal(y, out)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_strided_rows_and_what_lies_between_them(dtype):
    """x a column range of wider rows, out a column range whose neighbours stay as they are."""
    from unsloth_spectral import LoraBatch
    g = torch.Generator(device="cuda").manual_seed(7)
    pool, held = _adapters(g, 2, 128, (64,), [16, 16], dtype)
    wide = torch.randn(3, 5, 128 + 40, generator=g, device="cuda").to(dtype)
    x = wide[..., 16:144]
    y = torch.randn(3, 5, 64, generator=g, device="cuda").to(dtype)
    room = torch.full((3, 5, 64 + 24), 3.0, dtype=dtype, device="cuda")
    out = room[..., 8:72]
    ids = [1, -1, 0]
    pool.add(y, x, LoraBatch(ids), out=out)
    _check(out, *_ref(y, x, held, ids, (64,)))
    assert (room[..., :8] == 3).all() and (room[..., 72:] == 3).all()
    one = pool.add(y[:, 0], x[:, 0], LoraBatch(ids))               # [B, n]: one token each, rows far apart
    _check(one[:, None], *_ref(y[:, :1], x[:, :1], held, ids, (64,)))
    empty = pool.add(y[:0], x[:0], LoraBatch([]))
    assert empty.shape == (0, 5, 64)
    from unsloth_spectral import _native as N
    with pytest.raises(N.SpxError):                                # rows off 16 bytes
        pool.add(y, wide[..., 1:129], LoraBatch(ids))
    flat = torch.zeros(3 * 5 * 64 + 8, dtype=dtype, device="cuda")
    with pytest.raises(RuntimeError):                              # out a shifted view of y
        pool.add(flat[:-8].view(3, 5, 64), x, LoraBatch(ids), out=flat[8:].view(3, 5, 64))
    with pytest.raises(N.SpxError):                                # out the same row for every sequence
        pool.add(y[:, :1], x[:, :1], LoraBatch(ids), out=room[:1, :1, 8:72].expand(3, 1, 64))
    with pytest.raises(ValueError):                                # rows not evenly spaced
        pool.add(y[:, :3], wide[:, :3, 16:144], LoraBatch(ids))


@pytest.mark.parametrize("B,T,K,W,parts", [(67, 386, 1576, 8000, 1), (40, 400, 1032, 1160, 3), (12, 1500, 520, 2440, 2)])
def test_blocks_with_and_without_adapters_in_turn(B, T, K, W, parts):
    """Blocks of rows where requests without an adapter, with one on some parts only and with
    one everywhere follow one another, over odd numbers of column chunks: rows without are
    copied, the others equal the kernels for few rows (whose order of sums differs: each within
    the tolerance of the formula), and every run gives the same."""
    from unsloth_spectral import LoraBatch
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(W)
    widths = (W,) * parts
    ranks = [tuple((8 if (s + p) % 3 else 0) for p in range(parts)) for s in range(6)]
    pool, held = _adapters(g, 6, K, widths, ranks, dt)
    ids = [i % 7 - 1 for i in range(B)]
    assert (T / (-(-T // 128) * 128)) ** 3 * B * T * (K + W) * parts * 16 >= 1.5e8     # taken as blocks
    x = torch.randn(B, T, K, generator=g, device="cuda").to(dt)
    y = torch.randn(B, T, W * parts, generator=g, device="cuda").to(dt)
    batch = LoraBatch(ids)
    first = pool.add(y, x, batch)
    for _ in range(8):
        assert torch.equal(pool.add(y, x, batch), first)
    for b in range(B):
        at = 0
        for p, w in enumerate(widths):
            if (ids[b], p) not in held:
                assert torch.equal(first[b, :, at:at + w], y[b, :, at:at + w])
            at += w
    for b in (0, 1, 2, B // 2, B - 1):
        ref, tol = _ref(y[b:b + 1], x[b:b + 1], held, ids[b:b + 1], widths)
        _check(first[b:b + 1], ref, tol)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_and_small_values(dtype):
    """Inner products past float16's range and rows of tiny values keep their precision; an
    infinity stays in its row."""
    from unsloth_spectral import LoraBatch, LoraPool
    g = torch.Generator(device="cuda").manual_seed(8)
    K, W = 256, 48
    pool = LoraPool(K, W, max_rank=4, slots=1, dtype=dtype)
    A = torch.randn(4, K, generator=g, device="cuda").to(dtype)
    B = (torch.randn(W, 4, generator=g, device="cuda") * 2 ** -10).to(dtype)
    pool.load(0, A, B, 1.0)
    held = {(0, 0): (A, B, 1.0)}
    x = torch.randn(1, 4, K, generator=g, device="cuda")
    x[0, 0] *= 4000                    # t about 6e4
    x[0, 2] *= 2 ** -12
    x = x.to(dtype)
    y = torch.randn(1, 4, W, generator=g, device="cuda").to(dtype)
    y[0, 2] = 0
    ref, tol = _ref(y, x, held, [0], (W,))
    out = pool.add(y, x, LoraBatch([0]))
    _check(out, ref, tol)
    x2 = x.clone()
    x2[0, 1, 5] = float("inf")
    out2 = pool.add(y, x2, LoraBatch([0]))
    assert torch.equal(out2[0, [0, 2, 3]], out[0, [0, 2, 3]]) and not out2[0, 1].isfinite().any()


def test_streams_graphs_and_reloading():
    """Two graphs captured on one stream, replayed on two at once; a slot reloaded between
    replays is used by the next one."""
    from unsloth_spectral import LoraBatch
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(10)
    pool, held = _adapters(g, 3, 512, (256,), [16, 8, 4], dt)
    xs = [torch.randn(6, 1, 512, generator=g, device="cuda").to(dt) for _ in range(2)]
    ys = [torch.randn(6, 1, 256, generator=g, device="cuda").to(dt) for _ in range(2)]
    ids = [0, 1, 2, -1, 0, 1]
    batch = LoraBatch(ids).prepare(1)
    graphs, outs = [], []
    for x, y in zip(xs, ys):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(pool.add(y, x, batch))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for x, y, o in zip(xs, ys, outs):
        _check(o, *_ref(y, x, held, ids, (256,)))
    A, B, _ = held[1, 0]
    pool.load(0, A, B, 3.0)
    held[0, 0] = (A, B, 3.0)
    graphs[0].replay()
    _check(outs[0], *_ref(ys[0], xs[0], held, ids, (256,)))
    fresh = LoraBatch(ids)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError):
            pool.add(ys[0], xs[0], fresh)


def test_a_batch_dropped_while_another_stream_still_reads_it():
    """Its grouping of rows is not handed out again before that stream is done."""
    from unsloth_spectral import LoraBatch
    g = torch.Generator(device="cuda").manual_seed(11)
    pool, held = _adapters(g, 2, 128, (64,), [16, 16], torch.bfloat16)
    x = torch.randn(3, 1, 128, generator=g, device="cuda").bfloat16()
    y = torch.randn(3, 1, 64, generator=g, device="cuda").bfloat16()
    ids = [1, -1, 0]
    batch = LoraBatch(ids).prepare(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)            # about 10 ms
        out = pool.add(y, x, batch)
    del batch
    taken = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in range(1, 40)]
    torch.cuda.synchronize()
    _check(out, *_ref(y, x, held, ids, (64,)))
    assert len(taken) == 39


def test_a_new_batch_does_not_wait_for_the_gpu_and_is_there_for_streams_and_graphs():
    from unsloth_spectral import LoraBatch
    g = torch.Generator(device="cuda").manual_seed(12)
    pool, held = _adapters(g, 2, 128, (64,), [16, 16], torch.float16)
    x = torch.randn(3, 1, 128, generator=g, device="cuda").half()
    y = torch.randn(3, 1, 64, generator=g, device="cuda").half()
    ids = [1, -1, 0]
    pool.add(y, x, LoraBatch(ids))               # the host memory of its copy is there from now on
    torch.cuda.synchronize()
    first, side = LoraBatch(ids), torch.cuda.Stream()
    busy = torch.cuda.Event()
    torch.cuda._sleep(100_000_000)               # about 50 ms
    busy.record()
    outs = [pool.add(y, x, first)]
    assert not busy.query()
    with torch.cuda.stream(side):                # x and y have been there since before the sleep
        outs.append(pool.add(y, x, first))
    second = LoraBatch(ids)
    outs.append(pool.add(y, x, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs.append(pool.add(y, x, second))
    graph.replay()
    torch.cuda.synchronize()
    ref = _ref(y, x, held, ids, (64,))
    for o in outs:
        _check(o, *ref)
