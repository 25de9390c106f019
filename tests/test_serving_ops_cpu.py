"""The serving operators (per-head q/k norm with rotation, adapters, logits rules) without a
GPU: struct layouts against include/spx.h, refusals of the C entry points and of the Python
calls before any launch, and the host-side grouping of rows by adapter."""
import ctypes as C
import json
import os
import subprocess
import tempfile

import pytest
import torch

from conftest import REPO
from unsloth_spectral import LogitsRules, LoraBatch, LoraPool, qk_norm_rope
from unsloth_spectral import _native as N

HEADER = os.path.join(REPO, "include", "spx.h")


def test_struct_layouts_match_header():
    structs = {"spx_qk_norm_args": N.QkNormArgs, "spx_lora_args": N.LoraArgs, "spx_logits_args": N.LogitsArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', 'int main(void){', 'printf("{\\"x\\":0");']
    for cname, py in structs.items():
        for f, _ in py._fields_:
            lines.append(f'printf(",\\"{cname}.{f}\\":%zu", offsetof({cname}, {f}));')
        lines.append(f'printf(",\\"{cname}\\":%zu", sizeof({cname}));')
    lines += [f'printf(",\\"parts\\":%d,\\"rank\\":%d}}", SPX_LORA_MAX_PARTS, SPX_LORA_MAX_RANK);', 'return 0;}']
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        open(src, "w").write("\n".join(lines))
        subprocess.run(["gcc", "-std=c11", src, "-o", exe], check=True)
        got = json.loads(subprocess.run([exe], capture_output=True, text=True, check=True).stdout)
    for cname, py in structs.items():
        for f, _ in py._fields_:
            assert got[f"{cname}.{f}"] == getattr(py, f).offset, (cname, f)
        assert got[cname] == C.sizeof(py), cname
    assert (got["parts"], got["rank"]) == (N.LORA_MAX_PARTS, N.LORA_MAX_RANK)


def _qk(**kw):
    a = N.QkNormArgs(batch=1, tokens=1, num_q_heads=4, num_kv_heads=2, head_dim=64, dtype=N.SPX_BF16, rope_len=8, eps=1e-6,
                     q=256, k=256, q_weight=256, k_weight=256, cos_table=256, sin_table=256, q_out=256, k_out=256)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("status,kw", [
    (0, dict(batch=0)), (0, dict(tokens=0)), (1, dict(q=None)), (1, dict(k=None)), (1, dict(k_out=None)),
    (1, dict(cos_table=None)), (2, dict(head_dim=63)), (2, dict(head_dim=2048)), (2, dict(num_q_heads=0)),
    (2, dict(rope_len=0)), (2, dict(eps=-1.0)), (2, dict(q_stride_t=-1)), (2, dict(batch=-1)), (3, dict(dtype=5))])
def test_qk_norm_c_refusals(status, kw):
    assert N.load().spx_qk_norm_rope(_qk(**kw), None) == status


def test_null_args_are_refused():
    lib = N.load()
    assert lib.spx_qk_norm_rope(None, None) == 1
    assert lib.spx_lora_add(None, None) == 1 and lib.spx_lora_workspace_size(None) == 0
    assert lib.spx_logits_rules(None, None) == 1


def _lora(**kw):
    a = N.LoraArgs(num_tiles=2, tile_rows=16, num_rows=20, in_features=64, parts=2,
                   part_width=(C.c_int32 * 4)(64, 32, 0, 0), max_rank=16, slots=2, dtype=N.SPX_F16, x=256, y=256, out=256,
                   x_stride=64, y_stride=96, out_stride=96, a=256, b=256, ranks=256, scales=256, tiles=256, order=256,
                   workspace=256, workspace_bytes=20 * 32 * 4 + 16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("status,kw", [
    (0, dict(num_tiles=0, x=None)), (1, dict(x=None)), (1, dict(tiles=None)), (2, dict(in_features=60)),
    (2, dict(parts=0)), (2, dict(parts=5)), (2, dict(parts=3)), (2, dict(max_rank=24)), (2, dict(max_rank=144)),
    (2, dict(tile_rows=8)), (2, dict(slots=1 << 25)), (2, dict(x_stride=56)), (2, dict(y_stride=88)), (3, dict(dtype=N.SPX_F32)), (4, dict(x=264)),
    (4, dict(out_stride=100)), (5, dict(workspace=None)), (5, dict(workspace_bytes=20 * 32 * 4 + 15))])
def test_lora_c_refusals(status, kw):
    lib = N.load()
    assert lib.spx_lora_add(_lora(**kw), None) == status
    assert lib.spx_lora_workspace_size(_lora()) == 20 * 32 * 4 + 16


def _logits(**kw):
    a = N.LogitsArgs(batch=2, vocab=100, dtype=N.SPX_F32, logits=256, logits_stride=100, token=256, repetition=256,
                     seen_bits=256, touched_bits=256, counts=256)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("status,kw", [
    (0, dict(batch=0)), (1, dict(logits=None)), (1, dict(token=None)), (1, dict(seen_bits=None)), (1, dict(touched_bits=None)),
    (1, dict(counts=None)), (1, dict(bias_bits=256)), (1, dict(repetition=None, record=1, seen_bits=None)),
    (2, dict(vocab=0)), (2, dict(batch=-1)), (2, dict(logits_stride=99)), (2, dict(out=256, out_stride=99)),
    (2, dict(allow=256, allow_stride=3)), (3, dict(dtype=9))])
def test_logits_c_refusals(status, kw):
    assert N.load().spx_logits_rules(_logits(**kw), None) == status


def test_observe_c_refusals():
    lib = N.load()
    assert lib.spx_logits_observe(None, 1, 2, 3, 100, 256, 256, 256, None) == 1
    assert lib.spx_logits_observe(256, 1, 2, 3, 100, None, 256, 256, None) == 1
    assert lib.spx_logits_observe(256, 1, 2, 3, 100, 256, None, 256, None) == 1
    assert lib.spx_logits_observe(256, 1, 2, -3, 100, 256, 256, 256, None) == 2
    assert lib.spx_logits_observe(256, -1, 2, 3, 100, 256, 256, 256, None) == 2
    assert lib.spx_logits_observe(256, 1, 2, 3, 0, 256, 256, 256, None) == 2
    assert lib.spx_logits_observe(None, 1, 2, 0, 100, 256, 256, None, None) == 0


def test_qk_norm_python_refusals():
    q, k = torch.randn(2, 3, 32), torch.randn(2, 3, 16)
    w = torch.ones(8)
    tab = torch.zeros(10, 8)
    pos = torch.arange(3)
    with pytest.raises(N.SpxUnavailable):   # everything fits, but these are CPU tensors
        qk_norm_rope(q, k, w, w, tab, tab, pos)
    for bad in (dict(q=q[0]), dict(q=q[..., :30]), dict(k=k[:, :2]), dict(k=k[..., :12]), dict(k=k.half()),
                dict(k_weight=None), dict(k_weight=torch.ones(4)), dict(q_weight=w.half()), dict(eps=-1.0),
                dict(q_weight=torch.ones(7), k_weight=torch.ones(7))):
        a = dict(q=q, k=k, q_weight=w, k_weight=w, eps=1e-6)
        a.update(bad)
        with pytest.raises(ValueError):
            qk_norm_rope(a["q"], a["k"], a["q_weight"], a["k_weight"], tab, tab, pos, eps=a["eps"])
    with pytest.raises(TypeError):
        qk_norm_rope(q.double(), None, w.double(), None, tab, tab, pos)


def test_lora_batch_groups_rows_by_slot():
    for slots, tokens, blocks in (([2, -1, 2, 0], 1, False), ([0] * 17, 1, False), ([1, 0, 1], 33, False),
                                  ([1, -1, 1], 300, True), ([0, 0], 64, True), ([0, 0], 64, False), ([], 4, False),
                                  ([5], 0, False), ([-1], 2, False), ([], 64, True), ([3, 1, 3, 0], 128, True)):
        rows, tiles, order = LoraBatch.tiles_of(slots, tokens, blocks)
        assert (rows == 128) == blocks and tiles.dtype == order.dtype == "int32"
        taken, at = [], 0
        for slot, first, n, row0 in tiles.tolist():
            assert 1 <= n <= rows and rows in (16, 32, 128) and first == at
            mine = list(range(row0, row0 + n)) if blocks else order[first:first + n].tolist()
            assert all(slots[r // tokens] == slot for r in mine)
            taken, at = taken + mine, at + n
        assert sorted(taken) == list(range(len(slots) * tokens))
    assert LoraBatch.tiles_of([0] * 16, 1)[0] == 16 and LoraBatch.tiles_of([0] * 17, 1)[0] == 32


def test_lora_python_refusals():
    for bad in (dict(in_features=20), dict(out_features=12), dict(out_features=[16] * 5), dict(max_rank=0),
                dict(max_rank=129), dict(slots=0)):
        with pytest.raises(ValueError):
            LoraPool(**{**dict(in_features=16, out_features=24, device="cpu"), **bad})
    with pytest.raises(TypeError):
        LoraPool(16, 24, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError):
        LoraBatch([0, -2], device="cpu")
    pool = LoraPool(16, (24, 8), max_rank=4, slots=2, device="cpu")
    A, B = torch.randn(4, 16), torch.randn(24, 4)
    pool.load(1, A, B, 2.0)
    assert pool.ranks.tolist() == [[0, 0], [4, 0]] and pool.scales[1, 0] == 2.0
    assert torch.equal(pool.a[1, 0, :4], A.bfloat16()) and torch.equal(pool.b[1, :24, :4], B.bfloat16())
    pool.load(1, A[:2], B[:, :2], 1.0)     # a smaller one leaves nothing of the last behind
    assert not pool.a[1, 0, 2:].any() and not pool.b[1, :24, 2:].any() and pool.ranks[1, 0] == 2
    for call in (lambda: pool.load(0, A, B[:8]), lambda: pool.load(0, A[:, :8], B), lambda: pool.load(0, A, B, float("inf")),
                 lambda: pool.load(0, torch.randn(5, 16), torch.randn(24, 5))):
        with pytest.raises(ValueError):
            call()
    for slot, part in ((2, 0), (-1, 0), (0, 2)):
        with pytest.raises(IndexError):
            pool.load(slot, A, B, 1.0, part)
    pool.unload(1)
    assert not pool.ranks.any()
    x, y = torch.zeros(2, 3, 16, dtype=torch.bfloat16), torch.zeros(2, 3, 32, dtype=torch.bfloat16)
    b = LoraBatch([0, -1], device="cpu")
    for a in ((y[:1], x, b), (y, x[..., :8], b), (y, x, LoraBatch([0], device="cpu")), (y.float(), x, b), (y[0], x, b)):
        with pytest.raises(ValueError):
            pool.add(*a)
    with pytest.raises(IndexError):
        pool.add(y, x, LoraBatch([0, 2], device="cpu"))
    with pytest.raises(N.SpxUnavailable):
        pool.add(y, x, b)


def test_logits_python_refusals():
    for bad in (dict(batch=0), dict(vocab=0), dict(repetition_penalty=0.0), dict(repetition_penalty=[1.0]),
                dict(frequency_penalty=float("nan")), dict(presence_penalty=[0.0] * 3), dict(logit_bias={50: 1.0}),
                dict(logit_bias={-1: 1.0}), dict(logit_bias=[{}]), dict(logit_bias={3: float("nan")}),
                dict(logit_bias={3: float("inf")})):
        with pytest.raises(ValueError):
            LogitsRules(**{**dict(batch=2, vocab=50, device="cpu"), **bad})
    r = LogitsRules(2, 50, device="cpu", logit_bias=[{31: 1.0, 0: 2.0, 49: 3.0}, None])
    assert r._bias[0].tolist() == [[1 - (1 << 31), 1 << 17], [0, 0]]
    assert r._bias[1].tolist() == [[0, 2], [3, 3]] and r._bias[2].tolist() == [2.0, 1.0, 3.0]
    x = torch.zeros(2, 50)
    for call in (lambda: r.pick(x[:1]), lambda: r.pick(x.t()), lambda: r.apply(x, out=x.half()),
                 lambda: r.pick(x, allow=torch.zeros(2, 1, dtype=torch.int32)),
                 lambda: r.pick(x, allow=torch.zeros(2, 2, dtype=torch.int64)),
                 lambda: r.pick(x, allow=torch.zeros(3, 2, dtype=torch.int32)),
                 lambda: r.observe(torch.zeros(3, dtype=torch.int64)), lambda: r.observe(torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        r.pick(x.double())
    with pytest.raises(N.SpxUnavailable):
        r.pick(x)


def test_out_over_another_place_of_the_input_is_refused():
    """Rows of an out tensor that lie on the input's, but not on the same ones; rows side by side pass
    (and are then refused for the device)."""
    pool, b = LoraPool(16, 32, max_rank=4, slots=2, device="cpu"), LoraBatch([0, -1], device="cpu")
    x = torch.zeros(2, 3, 16, dtype=torch.bfloat16)
    wide = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    flat = torch.zeros(12 * 32, dtype=torch.bfloat16)
    rules = LogitsRules(4, 10, device="cpu")
    room, line = torch.zeros(4, 24), torch.zeros(80)
    cases = [(pool.add, wide[..., :32], dict(x=x, batch=b), wide[..., 8:40]),
             (pool.add, flat[:192].view(2, 3, 32), dict(x=x, batch=b), flat[32:224].view(2, 3, 32)),
             (pool.add, wide[..., :32], dict(x=x, batch=b), wide.view(-1)[:192].view(2, 3, 32)),
             (pool.add, wide[:, :1, :32], dict(x=x[:, :1], batch=b), wide[:, :1, 24:56]),
             (rules.apply, room[:, :10], {}, room[:, 9:19]),
             (rules.apply, line[:40].view(4, 10), {}, line[10:50].view(4, 10)),
             (rules.apply, room[:, 5:15], {}, room.view(-1)[:40].view(4, 10))]
    for call, y, more, out in cases:
        with pytest.raises(RuntimeError, match="overlaps"):
            call(y, **more, out=out)
    for call, y, more, out in ((pool.add, wide[..., :32], dict(x=x, batch=b), wide[..., 32:]),
                               (pool.add, wide[..., :32], dict(x=x, batch=b), wide[..., :32]),
                               (rules.apply, room[:, :10], {}, room[:, 10:20]), (rules.apply, room[:, :10], {}, room[:, :10])):
        with pytest.raises(N.SpxUnavailable):
            call(y, **more, out=out)


def test_settings_past_float32_are_refused():
    """The kernels hold them in float32: 1e39 is an infinity there, 1e-46 zero."""
    for bad in (dict(repetition_penalty=1e39), dict(repetition_penalty=1e-46), dict(frequency_penalty=[0.0, 1e39]),
                dict(presence_penalty=-1e39), dict(logit_bias={3: 1e39})):
        with pytest.raises(ValueError):
            LogitsRules(**{**dict(batch=2, vocab=50, device="cpu"), **bad})
    r = LogitsRules(2, 50, device="cpu", repetition_penalty=1e-38, presence_penalty=3e38,
                    logit_bias={3: -1e39, 4: 3e38, 5: float("-inf")})
    assert r._bias[2].tolist()[:3] == [float("-inf"), pytest.approx(3e38), float("-inf")]
    pool = LoraPool(16, 24, max_rank=4, slots=2, device="cpu")
    for scale in (1e39, -1e39):
        with pytest.raises(ValueError):
            pool.load(0, torch.ones(2, 16), torch.ones(24, 2), scale)
    assert not pool.ranks.any()
