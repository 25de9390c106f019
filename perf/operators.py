"""The serving operators of the model loop as measured cases: per-head query/key norms with the
rotation (``qk``), low-rank adapters of many requests beside a shared projection (``lora``), and the
rules on logits with the greedy choice (``logits``).

``run`` with ``own`` false computes them with elementary torch operations in float32, rounded
once at the end; with ``own`` true it makes the package's calls on the same inputs.
"""
import os
import random
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6


def _package():
    os.environ.setdefault("UNSLOTH_SPECTRAL_QUIET", "1")
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unsloth-spectral_b200")
    if root not in sys.path:
        sys.path.insert(1, root)
    import unsloth_spectral
    return unsloth_spectral


def listed():
    return [
        # one request decoding: the smallest call of every layer, the 32/8-head shape of the loop
        dict(name="qk decode 1", op="qk", batch=1, tokens=1, heads=32, kv_heads=8, dim=128, dtype="bf16",
             rotate_keys=False, per_row=False),
        # a serving batch decoding, every request at its own position
        dict(name="qk decode 64", op="qk", batch=64, tokens=1, heads=32, kv_heads=8, dim=128, dtype="bf16",
             rotate_keys=False, per_row=True),
        # the loop's prompt: 8 requests of 4096 tokens
        dict(name="qk prompt 8x4096", op="qk", batch=8, tokens=4096, heads=32, kv_heads=8, dim=128, dtype="bf16",
             rotate_keys=False, per_row=False),
        # a ragged prompt of a small model with short heads, keys for a cache that holds them rotated
        dict(name="qk prompt 3x1037 d80", op="qk", batch=3, tokens=1037, heads=9, kv_heads=3, dim=80, dtype="f16",
             rotate_keys=True, per_row=True),
        # one request decoding through its adapter on the packed q|k|v projection
        dict(name="lora decode 1 qkv", op="lora", batch=1, tokens=1, inner=4096, out=4096, kv=1024, rank=16, slots=4,
             without=False, dtype="bf16"),
        # a serving batch on the down projection, 24 fine-tunes of mixed ranks, some requests without
        dict(name="lora decode 64 down", op="lora", batch=64, tokens=1, inner=14336, out=4096, kv=0, rank=64,
             slots=24, without=True, dtype="bf16"),
        # the loop's prompt through the packed q|k|v projection, a fine-tune for each request
        dict(name="lora prompt 8x4096 qkv", op="lora", batch=8, tokens=4096, inner=4096, out=4096, kv=1024, rank=16,
             slots=8, without=False, dtype="bf16"),
        # ragged chunks of odd lengths, higher rank, the up projection
        dict(name="lora chunk 5x77 up", op="lora", batch=5, tokens=77, inner=4096, out=14336, kv=0, rank=32, slots=3,
             without=True, dtype="f16"),
        # one request choosing its token under penalties, the loop's vocabulary
        dict(name="logits pick 1", op="logits", batch=1, vocab=32768, prompt=4096, output=200, biases=16, allow=False,
             write=False, dtype="bf16"),
        # the loop's batch of 8, processed logits kept for a sampler
        dict(name="logits apply 8", op="logits", batch=8, vocab=32768, prompt=4096, output=512, biases=50, allow=True,
             write=True, dtype="bf16"),
        # a large serving batch with a large vocabulary, float32 logits
        dict(name="logits apply 128 large", op="logits", batch=128, vocab=131072, prompt=2000, output=1000, biases=300,
             allow=True, write=True, dtype="f32"),
        # a vocabulary whose rows are not aligned (tokens added by hand)
        dict(name="logits apply 33 odd", op="logits", batch=33, vocab=50021, prompt=700, output=90, biases=5,
             allow=True, write=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number, spread over the logarithm of lo..hi."""
    import math
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk", "lora", "logits"])
    if op == "qk":
        kv = rng.choice([1, 2, 3, 4, 8])
        c = dict(op=op, batch=_log(rng, 1, 64), tokens=1 if rng.random() < 0.4 else _log(rng, 2, 4096),
                 heads=kv * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv, dim=rng.choice([64, 80, 96, 128, 192, 256]),
                 dtype=rng.choice(["bf16", "f16", "f32"]), rotate_keys=rng.random() < 0.5, per_row=rng.random() < 0.5)
        most = 8 * 4096 * 40 * 128 * 2
        while c["batch"] * c["tokens"] * (c["heads"] + kv) * c["dim"] * _SIZE[c["dtype"]] > most:
            c["tokens"] = max(1, c["tokens"] // 2)
            c["batch"] = max(1, c["batch"] - 1)
        return c
    if op == "lora":
        c = dict(op=op, batch=_log(rng, 1, 128), tokens=1 if rng.random() < 0.5 else _log(rng, 2, 4096),
                 inner=8 * _log(rng, 32, 1792), out=8 * _log(rng, 32, 1792), kv=rng.choice([0, 0, 256, 1000, 1024]),
                 rank=rng.choice([4, 8, 16, 24, 32, 64]), slots=_log(rng, 1, 32), without=rng.random() < 0.5,
                 dtype=rng.choice(["bf16", "f16"]))
        while c["batch"] * c["tokens"] * (c["inner"] + 2 * c["out"] + 4 * c["kv"]) > 8 * 4096 * (4096 + 2 * 6144):
            c["tokens"] = max(1, c["tokens"] // 2)
        return c
    c = dict(op=op, batch=_log(rng, 1, 128), vocab=_log(rng, 1000, 131072), prompt=_log(rng, 1, 8192),
             output=_log(rng, 1, 2000), biases=rng.choice([0, 1, 40, 300]), allow=rng.random() < 0.6,
             write=rng.random() < 0.7, dtype=rng.choice(["bf16", "f16", "f32"]))
    return c


# ------------------------------------------------------------------------------- inputs

def _outs(c):
    return [c["out"]] + ([c["kv"], c["kv"]] if c["kv"] else [])


def _rank_of(c, slot):
    """The rank of the adapter in a slot: users bring different ones."""
    return max(1, (c["rank"], (c["rank"] + 1) // 2, c["rank"])[slot % 3])


def _ids_in_order(c):
    """The slots in use, before the seed spreads them over the batch."""
    return [-1 if c["without"] and i % 5 == 4 else i % c["slots"] for i in range(c["batch"])]


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _qk_inputs(c, g):
    B, T, Hq, H, D, dt = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], _DT[c["dtype"]]
    packed = (_randn(g, B, T, (Hq + 2 * H) * D) * 1.5).to(dt)           # a q|k|v projection
    start = 777 + int(torch.randint(0, 2000, (1,), generator=g, device="cuda"))
    if c["per_row"]:
        first = torch.randint(0, start, (B, 1), generator=g, device="cuda")
        pos = first + torch.arange(T, device="cuda")[None]
    else:
        pos = (start + torch.arange(T, device="cuda"))[None]
    n = start + T + 1
    inv = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    f = torch.outer(torch.arange(n, dtype=torch.float64, device="cuda"), inv)
    f = torch.cat([f, f], -1)
    return dict(packed=packed, pos=pos, cos=f.cos().float(), sin=f.sin().float(),
                qw=(1 + 0.2 * _randn(g, D)).to(dt), kw=(1 + 0.2 * _randn(g, D)).to(dt))


def _lora_inputs(c, g, seed):
    dt, K, R, n = _DT[c["dtype"]], c["inner"], c["rank"], c["slots"]
    ids = _ids_in_order(c)
    random.Random(seed).shuffle(ids)
    x = _randn(g, c["batch"], c["tokens"], K).to(dt)
    y = _randn(g, c["batch"], c["tokens"], sum(_outs(c))).to(dt)
    A, Bw = [], []
    for s in range(n):
        r = _rank_of(c, s)
        A.append([(_randn(g, r, K) / K ** 0.5).to(dt) for _ in _outs(c)])
        Bw.append([(_randn(g, o, r) * 0.05).to(dt) for o in _outs(c)])
    return dict(x=x, y=y, A=A, B=Bw, ids=ids, scale=[2.0 if s % 2 else 1.0 for s in range(n)])


def _logits_inputs(c, g, seed):
    B, V = c["batch"], c["vocab"]
    rng = random.Random(seed)
    some = lambda n: (torch.rand(B, n, generator=g, device="cuda", dtype=torch.float64) ** 3 * V).long().clamp_(0, V - 1)  # noqa: E731
    prompt, output = some(c["prompt"]), some(c["output"])
    logits = (_randn(g, B, V) * 3).to(_DT[c["dtype"]])
    rep = [1.0 + 0.05 * rng.randint(0, 8) for _ in range(B)]
    freq = [0.1 * rng.randint(0, 8) for _ in range(B)]
    pres = [0.1 * rng.randint(-3, 9) for _ in range(B)]
    bias = []
    for _ in range(B):
        toks = rng.sample(range(V), min(c["biases"], V))
        bias.append({t: rng.choice([-100.0, -2.5, 1.25, 4.0]) for t in toks})
    allow = None
    if c["allow"]:   # a grammar's bit words, bit t % 32 of word t // 32: half of the words leave a few tokens only
        W = (V + 31) // 32
        allow = torch.randint(-2 ** 31, 2 ** 31, (B, W), generator=g, device="cuda").to(torch.int32)
        few = torch.randint(0, 2, (B, W), generator=g, device="cuda", dtype=torch.int32)
        allow = torch.where(few == 1, allow & 0x00010001, allow)
        if B > 2:
            allow[B - 1] = 0   # a grammar that leaves nothing
    return dict(logits=logits, prompt=prompt, output=output, rep=rep, freq=freq, pres=pres, bias=bias, allow=allow)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c)
    if c["op"] == "qk":
        s.update(_qk_inputs(c, g))
        nq, nk = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
        s["q"], s["k"] = s["packed"][..., :nq], s["packed"][..., nq:nq + nk]
        if own:
            s["call"] = _package().qk_norm_rope
    elif c["op"] == "lora":
        s.update(_lora_inputs(c, g, seed))
        if own:
            P = _package()
            outs = _outs(c)
            pool = P.LoraPool(c["inner"], outs, max_rank=c["rank"], slots=c["slots"], dtype=s["x"].dtype,
                              device=s["x"].device)
            for a in range(c["slots"]):
                for i in range(len(outs)):
                    pool.load(a, s["A"][a][i], s["B"][a][i], scale=s["scale"][a], part=i)
            s["pool"], s["batch"] = pool, P.LoraBatch(s["ids"], device=s["x"].device)
        else:
            s["groups"] = [(a, torch.tensor([i for i, k in enumerate(s["ids"]) if k == a], device="cuda"))
                           for a in sorted(set(s["ids"]) - {-1})]
    else:
        s.update(_logits_inputs(c, g, seed))
        B, V = c["batch"], c["vocab"]
        if own:
            rules = _package().LogitsRules(B, V, device=s["logits"].device, repetition_penalty=s["rep"],
                                           frequency_penalty=s["freq"], presence_penalty=s["pres"],
                                           logit_bias=s["bias"])
            rules.observe_prompt(s["prompt"])
            rules.observe(s["output"])
            s["rules"] = rules
        else:
            ones = torch.ones_like(s["output"], dtype=torch.int32)
            s["counts"] = torch.zeros(B, V, dtype=torch.int32, device="cuda").scatter_add_(1, s["output"], ones)
            s["seen"] = (s["counts"] > 0).scatter_(1, s["prompt"], True)
            rows = [b for b in range(B) for _ in s["bias"][b]]
            s["bias_row"] = torch.tensor(rows, dtype=torch.long, device="cuda")
            s["bias_tok"] = torch.tensor([t for d in s["bias"] for t in d], dtype=torch.long, device="cuda")
            s["bias_val"] = torch.tensor([v for d in s["bias"] for v in d.values()], device="cuda")
            for k in ("rep", "freq", "pres"):
                s[k + "_t"] = torch.tensor(s[k], device="cuda")[:, None]
    return s


# ------------------------------------------------------------------------------- one pass

def _head_norm(x, w, heads):
    B, T, _ = x.shape
    x = x.float().view(B, T, heads, -1).transpose(1, 2)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * w.float()


def _rotate(x, c, s):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    c, s = c[:, None, :, :h], s[:, None, :, :h]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _run_qk(s):
    c = s["case"]
    if own:
        return s["call"](s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"], eps=_EPS,
                         rotate_keys=c["rotate_keys"])
    q, k = _head_norm(s["q"], s["qw"], c["heads"]), _head_norm(s["k"], s["kw"], c["kv_heads"])
    cos, sin = s["cos"][s["pos"]], s["sin"][s["pos"]]
    q = _rotate(q, cos, sin)
    if c["rotate_keys"]:
        k = _rotate(k, cos, sin)
    return q.to(s["q"].dtype), k.to(s["k"].dtype)


def _run_lora(s):
    if own:
        return s["pool"].add(s["y"], s["x"], s["batch"])
    x, y = s["x"], s["y"].float()
    for a, rows in s["groups"]:
        xa = x[rows].float()
        delta = [(xa @ A.float().T) @ Bw.float().T for A, Bw in zip(s["A"][a], s["B"][a])]
        y[rows] += s["scale"][a] * torch.cat(delta, -1)
    return y.to(x.dtype)


def _run_logits(s):
    c = s["case"]
    if own:
        if c["write"]:
            return s["rules"].apply(s["logits"], allow=s["allow"])
        return s["rules"].pick(s["logits"], allow=s["allow"])
    x = s["logits"].float()
    x = torch.where(s["seen"], torch.where(x > 0, x / s["rep_t"], x * s["rep_t"]), x)
    x = x - s["freq_t"] * s["counts"].float()
    x = x - s["pres_t"] * (s["counts"] > 0).float()
    x[s["bias_row"], s["bias_tok"]] += s["bias_val"]
    if s["allow"] is not None:
        bits = (s["allow"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = x.masked_fill(bits.view(x.shape[0], -1)[:, :x.shape[1]] == 0, float("-inf"))
    token = x.argmax(-1)
    return (x.to(s["logits"].dtype), token) if c["write"] else token


def run(state):
    return {"qk": _run_qk, "lora": _run_lora, "logits": _run_logits}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------- floors

def work(case):
    c = case
    e = _SIZE[c["dtype"]]
    if c["op"] == "qk":
        rows, per = c["batch"] * c["tokens"], (c["heads"] + c["kv_heads"]) * c["dim"]
        angles = rows if c["per_row"] else c["tokens"]
        return {"bytes": 2 * rows * per * e + angles * (c["dim"] * 4 + 8) + 2 * c["dim"] * e, "flops": 8 * rows * per}
    if c["op"] == "lora":
        rows, ids, outs = c["batch"] * c["tokens"], _ids_in_order(c), _outs(c)
        weights = sum(_rank_of(c, a) * (len(outs) * c["inner"] + sum(outs)) for a in set(ids) - {-1})
        flops = sum(2 * c["tokens"] * _rank_of(c, a) * (len(outs) * c["inner"] + sum(outs)) for a in ids if a >= 0)
        with_one = sum(a >= 0 for a in ids) * c["tokens"]
        return {"bytes": e * (with_one * c["inner"] + 2 * rows * sum(outs) + weights), "flops": flops}
    B, V = c["batch"], c["vocab"]
    words = (V + 31) // 32 * 4
    read = B * (V * e + words * (2 + bool(c["allow"])) + 4 * min(c["output"], V) + 8 * c["biases"])
    return {"bytes": read + B * 8 + (B * V * e if c["write"] else 0), "flops": 4 * B * V}


# ------------------------------------------------------------------------------- in 64 bits

def _exact_qk(c, g):
    i = _qk_inputs(c, g)
    D, h = c["dim"], c["dim"] // 2
    heads, kv = c["heads"], c["kv_heads"]
    p = i["packed"].double().view(c["batch"], c["tokens"], heads + 2 * kv, D)
    ang_c = i["cos"].double()[i["pos"]][:, :, None, :h]
    ang_s = i["sin"].double()[i["pos"]][:, :, None, :h]

    def part(v, w, turn):
        v = v / torch.sqrt((v * v).sum(-1, keepdim=True) / D + _EPS) * w.double()
        if turn:
            z = torch.complex(v[..., :h].contiguous(), v[..., h:].contiguous()) * torch.complex(ang_c, ang_s)
            v = torch.cat([z.real, z.imag], -1)
        return v.permute(0, 2, 1, 3).contiguous()

    return part(p[:, :, :heads], i["qw"], True), part(p[:, :, heads:heads + kv], i["kw"], c["rotate_keys"])


def _exact_lora(c, g, seed):
    i = _lora_inputs(c, g, seed)
    out = i["y"].double()
    for b, a in enumerate(i["ids"]):
        if a < 0:
            continue
        at = 0
        for A, Bw in zip(i["A"][a], i["B"][a]):
            t = torch.einsum("tk,rk->tr", i["x"][b].double(), A.double())
            out[b, :, at:at + Bw.shape[0]] += i["scale"][a] * torch.einsum("tr,or->to", t, Bw.double())
            at += Bw.shape[0]
    return out


def _exact_logits(c, g, seed):
    i = _logits_inputs(c, g, seed)
    B, V = c["batch"], c["vocab"]
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731  the parameters are float32 inputs
    rows, toks = [], []
    for b in range(B):
        v = i["logits"][b].double()
        n = torch.bincount(i["output"][b], minlength=V)
        seen = (n + torch.bincount(i["prompt"][b], minlength=V)) > 0
        p = f32(i["rep"][b])
        v[seen] = torch.where(v[seen] > 0, v[seen] / p, v[seen] * p)
        v = v - f32(i["freq"][b]) * n.double() - f32(i["pres"][b]) * (n > 0).double()
        if i["bias"][b]:
            t = torch.tensor(list(i["bias"][b]), device=v.device)
            v[t] = v[t] + torch.tensor(list(i["bias"][b].values()), device=v.device, dtype=torch.float64)
        if i["allow"] is not None:
            t = torch.arange(V, device=v.device)
            v = torch.where((i["allow"][b][t // 32].long() >> (t % 32)) & 1 == 1, v, torch.full_like(v, -torch.inf))
        rows.append(v)
        toks.append(v.argmax())
    tokens = torch.stack(toks)
    return (torch.stack(rows), tokens) if c["write"] else tokens


def exact(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "qk":
        return _exact_qk(case, g)
    if case["op"] == "lora":
        return _exact_lora(case, g, seed)
    return _exact_logits(case, g, seed)
