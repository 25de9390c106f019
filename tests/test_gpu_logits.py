"""LogitsRules against the rules in 64 bits, and its tokens against the float32 expression.

Each rule is one or two float32 operations, rounded on its own: a processed value is within
u = 2^-24 of every intermediate value, here at most five of them of size at most
m = |x| max(p, 1/p) + |f c| + |q| + |bias|: 5 u m, and half a step of the output type.  The
token is the argmax of exactly those float32 values, so it equals that of the same
expression evaluated by torch in float32 on the CPU."""
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]


def _expr(x, seen, counts, rep, freq, pres, bias, allow, wide):
    ft = torch.float64 if wide else torch.float32
    x, n = x.cpu().to(ft), counts.to(ft)
    rep, freq, pres = (torch.tensor(v, dtype=torch.float32).to(ft)[:, None] for v in (rep, freq, pres))
    m = x.abs() * torch.maximum(rep, 1 / rep) + (freq * n).abs() + pres.abs()
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - freq * n
    x = torch.where(n > 0, x - pres, x)
    for b, d in enumerate(bias):
        for t, v in (d or {}).items():
            x[b, t] += v
            m[b, t] += abs(v)
    if allow is not None:
        x = torch.where(allow, x, torch.full_like(x, -torch.inf))
    return x, m


def _pack(allow, V):
    B, W = allow.shape[0], (V + 31) // 32
    full = torch.zeros(B, W * 32, dtype=torch.int64)
    full[:, :V] = allow
    words = (full.view(B, W, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _first_max(x):
    """Lowest index of the largest value of each row, NaN largest."""
    x = torch.where(x.isnan(), torch.full_like(x, torch.inf), x) if not x.isnan().any() else x
    out = []
    for r in x:
        nan = r.isnan().nonzero()
        out.append(int(nan[0]) if len(nan) else int((r == r.max()).nonzero()[0]))
    return torch.tensor(out)


CASES = [(1, 32768, 16, True), (8, 32768, 3, True), (3, 1000, 2, True), (5, 50021, 40, True), (2, 7, 1, True), (1, 1, 0, False),
         (4, 31, 0, True), (2, 33, 2, False), (300, 513, 1, True), (2, 131077, 300, False), (7, 4104, 0, True),
         (700, 9001, 2, True), (3, 20000, 9, False), (90, 40003, 3, True),
         (2, 131075, 300, True), (20, 70001, 40, False), (25, 65536, 0, True)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,V,nbias,masked", CASES)
def test_against_the_rules(dtype, B, V, nbias, masked):
    from unsloth_spectral import LogitsRules
    g = torch.Generator().manual_seed(B + V)
    rnd = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    x = (torch.randn(B, V, generator=g) * 3).to(dtype).cuda()
    rep, freq, pres = (1 + rnd(B)).tolist(), (rnd(B) - 0.2).tolist(), (rnd(B) - 0.5).tolist()
    rep[0] = 0.8
    bias = [{int(t): float(v) for t, v in zip(torch.randperm(V, generator=g)[:nbias], torch.randn(nbias, generator=g) * 4)}
            for _ in range(B)]
    allow = rnd(B, V) < 0.5 if masked else None
    if masked and B > 1:
        allow[1] = False
    prompt = (rnd(B, 40) * V).long()
    output = (rnd(B, 60) ** 2 * V).long()
    prompt[:, 30:] = -1                                             # padding
    rules = LogitsRules(B, V, repetition_penalty=rep, frequency_penalty=freq, presence_penalty=pres, logit_bias=bias)
    rules.observe_prompt(prompt.cuda())
    rules.observe(output[:, :59].cuda())
    rules.observe(output[:, 59].cuda())
    counts = torch.zeros(B, V, dtype=torch.int32).scatter_add_(1, output, torch.ones_like(output, dtype=torch.int32))
    assert torch.equal(rules.counts.cpu(), counts)
    seen = (counts > 0).scatter(1, prompt[:, :30], True)
    keep = x.clone()
    mask = _pack(allow, V).cuda() if masked else None
    got, token = rules.apply(x, allow=mask)
    assert torch.equal(x, keep) and torch.equal(rules.counts.cpu(), counts) and got.dtype == dtype
    ref, m = _expr(x, seen, counts, rep, freq, pres, bias, allow, True)
    f32, _ = _expr(x, seen, counts, rep, freq, pres, bias, allow, False)
    fin = ref.isfinite()
    assert torch.equal(got.cpu() == -torch.inf, ~fin)
    err = (got.cpu().double() - ref).abs()[fin]
    tol = (torch.finfo(dtype).eps / 2 * ref.abs() + 5 * 2.0 ** -24 * m)[fin] + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert (err <= tol).all(), float((err - tol).max())
    assert torch.equal(token.cpu(), _first_max(f32))
    assert torch.equal(rules.pick(x, allow=mask), token)
    same, _ = rules.apply(x, allow=mask, out=x)                      # in place
    assert same is x and torch.equal(x, got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1000, 1003, 40000])
def test_ties_nan_and_empty_rows(dtype, V):
    from unsloth_spectral import LogitsRules
    x = torch.zeros(6, V, dtype=dtype)
    x[0, [V - 1, 17, 400]] = 5.0                 # the lowest of equals
    x[1] = -torch.inf                            # nothing: token 0
    x[2, 900], x[2, 30], x[2, 31] = torch.inf, torch.nan, torch.nan
    x[3, 5:] = -0.0                              # equal to 0
    x[3, :5] = -1.0
    x[4], x[4, V - 1] = -torch.inf, -3.0
    x[5, 7] = torch.nan                          # in a masked place
    allow = torch.ones(6, V, dtype=torch.bool)
    allow[5, 7] = False
    x = x.cuda()
    rules = LogitsRules(6, V)
    out, tok = rules.apply(x, allow=_pack(allow, V).cuda())
    assert tok.tolist() == [17, 0, 30, 5, V - 1, 0]
    assert out[5, 7] == -torch.inf and out[2, 30].isnan() and out[2, 900] == torch.inf
    none = torch.zeros(1, (V + 31) // 32, dtype=torch.int32, device="cuda")
    out, tok = rules.apply(x, allow=none)        # one row for all, nothing allowed
    assert tok.tolist() == [0] * 6 and (out == -torch.inf).all()
    biased = LogitsRules(6, V, logit_bias={3: -float("inf"), V - 1: 9.0})
    assert biased.pick(torch.zeros_like(x)).tolist() == [V - 1] * 6


@pytest.mark.parametrize("V", [1000, 1003])
def test_touched_tokens_at_minus_infinity(V):
    """Seen and biased tokens that end at -inf (their logit, their bias, their mask) are chosen as
    little as any other: token 0 when nothing is left, the only finite one when one is."""
    from unsloth_spectral import LogitsRules
    rules = LogitsRules(3, V, repetition_penalty=1.3, frequency_penalty=0.5,
                        logit_bias=[{77: -float("inf")}, {77: -float("inf"), 500: 1.0}, {V - 1: -float("inf")}])
    rules.observe(torch.tensor([[5, 900], [77, 900], [900, 900]], device="cuda"))
    x = torch.full((3, V), -float("inf"), device="cuda")
    x[:, 77] = 3.0
    x[2, 900], x[2, 77] = -2.0, -float("inf")
    allow = torch.zeros(3, V, dtype=torch.bool)
    allow[:, [5, 77, 500, 900, V - 1]] = True
    for mask in (None, _pack(allow, V).cuda()):
        out, tok = rules.apply(x, allow=mask)
        assert tok.tolist() == [0, 0, 900]
        assert (out[:2] == -float("inf")).all() and int(out[2].isfinite().sum()) == 1
        assert rules.pick(x, allow=mask).tolist() == [0, 0, 900]


def test_record_counts_the_choice_and_reset_forgets():
    from unsloth_spectral import LogitsRules
    V = 97
    rules = LogitsRules(2, V, frequency_penalty=[1.0, 0.0], presence_penalty=[0.0, 2.0], repetition_penalty=1.5)
    x = torch.zeros(2, V)
    x[:, 5], x[:, 90] = 4.0, 3.5
    x = x.cuda()
    seq = [rules.pick(x, record=True).tolist() for _ in range(5)]
    # row 0: 4 -> 4/1.5 - n, against 3.5 -> 3.5/1.5 - n, others 0: worked out by hand
    hist, want = [torch.zeros(V, dtype=torch.int32) for _ in range(2)], []
    for _ in range(5):
        step = []
        for b in range(2):
            n = hist[b][None]
            r, _ = _expr(x[b:b + 1], n > 0, n, [1.5], [[1.0, 0.0][b]], [[0.0, 2.0][b]], [None], None, False)
            t = int(_first_max(r))
            hist[b][t] += 1
            step.append(t)
        want.append(step)
    assert seq == want
    assert torch.equal(rules.counts.cpu(), torch.stack(hist))
    rules.reset()
    assert not rules.counts.any() and rules.pick(x).tolist() == [5, 5]


def test_strides_streams_and_graphs():
    from unsloth_spectral import LogitsRules
    B, V = 3, 2051
    g = torch.Generator(device="cuda").manual_seed(1)
    room = torch.randn(B, V + 13, generator=g, device="cuda")
    x = room[:, 5:5 + V]                                             # rows off 16 bytes, not adjacent
    rules = LogitsRules(B, V, presence_penalty=0.5)
    out = torch.full((B, V + 3), 7.0, device="cuda")
    _, tok = rules.apply(x, out=out[:, 2:2 + V])
    assert torch.equal(out[:, 2:2 + V], x) and (out[:, :2] == 7).all() and (out[:, -1] == 7).all()
    assert torch.equal(tok, x.argmax(-1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tok2 = rules.pick(x)
    side.synchronize()
    assert torch.equal(tok2, tok)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = rules.pick(x, record=True)
    steps = []
    for _ in range(4):
        graph.replay()
        steps.append(t.clone())
    other = LogitsRules(B, V, presence_penalty=0.5)
    assert torch.equal(torch.stack(steps), torch.stack([other.pick(x, record=True) for _ in range(4)]))
    assert torch.equal(rules.counts, other.counts) and torch.equal(rules.seen_bits, other.seen_bits)
    one = torch.randn(1, 1, device="cuda")
    assert LogitsRules(1, 1).pick(one).tolist() == [0]
