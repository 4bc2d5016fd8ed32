"""Four-bit pages and matrices without a GPU: what the bindings refuse, and that they refuse before anything is launched."""
import math

import pytest
import torch

import dekinex_cases
import helpers
import sagalorn_cases
import tekilix_cases
import zakusun_cases
from glassbox_amd import ops

BF, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8


def pages(p=3, g=2, page=16, d=64):
    return torch.zeros(ops.fp4_pages_shape(p, g, page, d), dtype=U8)


def store(**change):
    a = dict(qkv=torch.zeros(5, 512, dtype=BF), cos=torch.zeros(5, 32), sin=torch.zeros(5, 32), slots=torch.zeros(5, dtype=I32), k=pages(), v=pages(),
             H=4, G=2, D=64, q=None)
    a.update(change)
    ops.fp4_store(a["qkv"], a["cos"], a["sin"], a["slots"], a["k"], a["v"], a["H"], a["G"], a["D"], q=a["q"])


def attention(**change):
    a = dict(q=torch.zeros(5, 256, dtype=BF), out=torch.zeros(5, 256, dtype=BF), q_start=torch.zeros(2, dtype=I32), q_len=torch.zeros(2, dtype=I32),
             pos0=torch.zeros(2, dtype=I32), tables=torch.zeros(2, 4, dtype=I32), k=pages(), v=pages(), H=4, scale=0.1, most=3, longest=50, window=0,
             ws=None)
    a.update(change)
    ops.fp4_attention(a["q"], a["out"], a["q_start"], a["q_len"], a["pos0"], a["tables"], a["k"], a["v"], a["H"], a["scale"], a["most"], a["longest"],
                      window=a["window"], workspace=a["ws"])


def gemm(**change):
    a = dict(a=torch.zeros(3, 64, dtype=BF), w=ops.Fp4Matrix(torch.zeros(10, 32, dtype=U8), torch.zeros(10, 16, dtype=U8)),
             out=torch.zeros(3, 10, dtype=BF), accumulate=False, silu_mul=False,
             emit=None, rms_parts=None)
    a.update(change)
    ops.fp4_gemm(a["a"], a["w"], a["out"], accumulate=a["accumulate"], silu_mul=a["silu_mul"], emit=a["emit"], rms_parts=a["rms_parts"])


ROWS = torch.zeros(5, 512, dtype=BF)
ADDS = dict(out=torch.zeros(3, 10), accumulate=True)
ADDS8 = dict(out=torch.zeros(3, 16), accumulate=True, w=ops.Fp4Matrix(torch.zeros(16, 32, dtype=U8), torch.zeros(16, 16, dtype=U8)))
EMIT = (torch.ones(16), torch.zeros(3, 16, dtype=BF), torch.zeros(8, 8))
REFUSED = [
    (store, dict(D=48), "multiple of 32"), (store, dict(G=3), "do not hold"), (store, dict(qkv=torch.zeros(5, 511, dtype=BF)), "do not hold"),
    (store, dict(k=pages(d=128)), "alike"), (store, dict(k=pages(g=1), v=pages(g=1)), "kv heads"), (store, dict(k=pages().view(torch.int8)), "uint8"),
    (store, dict(k=pages(page=24), v=pages(page=24)), "16 slots"), (store, dict(k=None), "four-bit pages"),
    (store, dict(k=pages(p=6)[::2], v=pages(p=6)[::2]), "contiguous"), (store, dict(slots=torch.zeros(4, dtype=I32)), "slots"),
    (store, dict(slots=torch.zeros(5, dtype=torch.int64)), "slots"), (store, dict(sin=None), "go together"), (store, dict(cos=torch.zeros(5, 64)), "cos/sin"),
    (store, dict(cos=torch.zeros(4, 32)), "cos/sin"), (store, dict(q=torch.zeros(5, 256)), "type"), (store, dict(q=torch.zeros(5, 128, dtype=BF)), "q must be"),
    (store, dict(qkv=ROWS, q=ROWS[:, 64:320]), "other columns"), (store, dict(qkv=torch.zeros(5, 512, dtype=torch.float16)), "element type"),
    (store, dict(qkv=torch.zeros(512, 5, dtype=BF).t()), "dense rows"), (store, {}, "current GPU"),
    (attention, dict(out=torch.zeros(5, 256)), "one type"), (attention, dict(out=torch.zeros(4, 256, dtype=BF)), "must be"),
    (attention, dict(q=torch.zeros(5, 192, dtype=BF), out=torch.zeros(5, 192, dtype=BF)), "must be"),
    (attention, dict(q=torch.zeros(5, 192, dtype=BF), out=torch.zeros(5, 192, dtype=BF), H=3), "multiple of the kv heads"),
    (attention, dict(q=torch.zeros(5, 640, dtype=BF), out=torch.zeros(5, 640, dtype=BF), k=pages(d=160), v=pages(d=160)), "heads of"),
    (attention, dict(scale=0.0), "positive"), (attention, dict(scale=-1.0), "positive"), (attention, dict(scale=math.nan), "positive"),
    (attention, dict(scale=math.inf), "positive"), (attention, dict(scale=1e-40), "positive"), (attention, dict(pos0=torch.zeros(1, dtype=I32)), "pos0"),
    (attention, dict(q_start=torch.zeros(2)), "q_start"), (attention, dict(tables=torch.zeros(1, 4, dtype=I32)), "tables"),
    (attention, dict(tables=torch.zeros(2, 0, dtype=I32)), "tables"), (attention, dict(tables=torch.zeros(4, 2, dtype=I32).t()), "tables"),
    (attention, dict(window=-1), "below 0"), (attention, dict(most=-1), "below 0"), (attention, dict(ws=torch.zeros(8, dtype=BF)), "workspace"),
    (attention, dict(ws=torch.zeros(9)[1:]), "workspace"), (attention, dict(v=pages(p=4)), "alike"),
    (attention, dict(q=ROWS[:, :256], out=ROWS[:, 128:384]), "other rows"), (attention, {}, "current GPU"),
    (gemm, dict(a=torch.zeros(3, 32, dtype=BF)), "do not match"), (gemm, dict(out=torch.zeros(3, 9, dtype=BF)), "do not match"),
    (gemm, dict(out=torch.zeros(3, 10, dtype=BF), accumulate=True), "32-bit"), (gemm, dict(out=torch.zeros(3, 10, dtype=BF), silu_mul=True), "do not match"),
    (gemm, dict(out=torch.zeros(3, 5), silu_mul=True, accumulate=True), "accumulate"),
    (gemm, dict(w=ops.Fp4Matrix(torch.zeros(10, 32, dtype=U8), torch.zeros(10, 2, dtype=U8))), "multiple of 16"),
    (gemm, dict(w=ops.Fp4Matrix(torch.zeros(10, 24, dtype=U8), torch.zeros(10, 16, dtype=U8))), "columns / 2"),
    (gemm, dict(w=ops.Fp4Matrix(torch.zeros(10, 64, dtype=U8)[:, ::2], torch.zeros(10, 16, dtype=U8))), "contiguous"),
    (gemm, dict(w=ops.Fp4Matrix(torch.zeros(0, 32, dtype=U8), torch.zeros(0, 16, dtype=U8)), out=torch.zeros(3, 0, dtype=BF)), "four-bit matrix"),
    (gemm, dict(a=torch.zeros(3, 64, dtype=torch.float16)), "element type"), (gemm, dict(a=torch.zeros(64, 3, dtype=BF).t()), "dense rows"),
    (gemm, dict(a=ROWS[:3, :64], out=ROWS[:3, 60:70]), "share memory"), (gemm, {}, "current GPU"),
    (gemm, dict(ADDS, emit=(torch.ones(10), torch.zeros(3, 10, dtype=BF), torch.zeros(8, 8))), "emit needs"),           # 10 columns
    (gemm, dict(ADDS8, accumulate=False, emit=EMIT), "emit needs"), (gemm, dict(ADDS8, a=torch.zeros(3, 64), emit=EMIT), "emit needs"),
    (gemm, dict(ADDS8, emit=(torch.ones(15), *EMIT[1:])), "emit needs"), (gemm, dict(ADDS8, emit=(EMIT[0], torch.zeros(3, 16), EMIT[2])), "emit needs"),
    (gemm, dict(ADDS8, emit=(*EMIT[:2], 1e-5)), "emit needs"),                                                          # the whole norm of 3 rows
    (gemm, dict(ADDS8, emit=(*EMIT[:2], torch.zeros(8, 8, dtype=BF))), "emit needs"), (gemm, dict(ADDS8, emit=EMIT), "current GPU"),
    (gemm, dict(ADDS8, a=torch.zeros(9, 64, dtype=BF), out=torch.zeros(9, 16), emit=(EMIT[0], torch.zeros(9, 16, dtype=BF), torch.zeros(8, 64))), "emit needs"),
    (gemm, dict(ADDS8, a=ROWS[:3, :64], emit=(EMIT[0], ROWS[:3, 60:76], EMIT[2])), "share memory"),
    (gemm, dict(rms_parts=(torch.zeros(2, 8), 3, 1e-5)), "partial sums"), (gemm, dict(rms_parts=(torch.zeros(17)[1:].view(2, 8), 2, 1e-5)), "partial sums"), (gemm, dict(rms_parts=(torch.zeros(2, 8), 0, 1e-5)), "partial sums"),
    (gemm, dict(ADDS8, rms_parts=(torch.zeros(2, 8), 2, 1e-5)), "partial sums"), (gemm, dict(a=torch.zeros(3, 64), rms_parts=(torch.zeros(2, 8), 2, 1e-5)), "partial"),
    (gemm, dict(a=torch.zeros(9, 64, dtype=BF), out=torch.zeros(9, 10, dtype=BF), rms_parts=(torch.zeros(2, 64), 2, 1e-5)), "partial sums"),
    (gemm, dict(rms_parts=(torch.zeros(2, 8), 2, 1e-5)), "current GPU"),
    (lambda **k: ops.fp4_quantize(**k), dict(w=torch.zeros(4, 40)), "multiple of 32"), (lambda **k: ops.fp4_quantize(**k), dict(w=torch.zeros(4, 0)), "multiple"),
    (lambda **k: ops.fp4_quantize(**k), dict(w=torch.zeros(4, 32, dtype=torch.float16)), "element type"),
    (lambda **k: ops.fp4_quantize(**k), dict(w=torch.zeros(4, 32)), "current GPU"),
    (lambda **k: ops.fp4_expand(ops.Fp4Matrix(torch.zeros(10, 32, dtype=U8), torch.zeros(10, 16, dtype=U8)), **k), dict(out=torch.zeros(10, 32)), "out must be"),
    (lambda **k: ops.fp4_load(torch.zeros(4, dtype=I32), pages(), pages(), **k), dict(k=torch.zeros(4, 128), v=torch.zeros(4, 64)), "must be"),
    (lambda **k: ops.fp4_load(torch.zeros(4, dtype=I32), pages(), pages(), **k), dict(k=ROWS[:4, :128], v=ROWS[:4, 64:192]), "share memory"),
]


@pytest.mark.parametrize("call,change,why", REFUSED)
def test_refusals(call, change, why):
    with pytest.raises(ops.KernelError, match=why):
        call(**change)


def test_sizes():
    assert ops.fp4_pages_shape(7, 3, 32, 128) == (7, 3, 4, 17, 32)
    assert [ops.fp4_scale_bytes(k) for k in (32, 512, 544, 4096)] == [16, 16, 32, 128]
    assert ops.Fp4Matrix(torch.zeros(10, 32, dtype=U8), torch.zeros(10, 16, dtype=U8)).shape == (10, 64)


def model_of(config):
    from glassbox_amd.config import config_from_dict
    from glassbox_amd.weights import build_model
    return build_model(config_from_dict(config))


@pytest.mark.parametrize("config,kv_cache,weights,why", [
    (helpers.TINY_E, "fp4", None, "cache layer 0: four-bit pages are for plain attention with heads of 32"),     # heads of 16
    (helpers.TINY_E, None, "fp4", "width: 72 is not a multiple of 32"), (helpers.TINY_E, None, "fp4", "intermediate: 120 is not a multiple"),
    (helpers.TINY_A, None, "fp4", "intermediate: 176"), (helpers.TINY_B, "fp8", None, "kv_cache='fp8'"), (helpers.TINY_B, None, "int4", "weights='int4'"),
    (zakusun_cases.CASES["A"], "fp4", None, "four-bit pages"), (zakusun_cases.CASES["A"], None, "fp4", "has no products with four-bit"),
    (tekilix_cases.CASES["A"], "fp4", None, "four-bit pages"), (tekilix_cases.CASES["A"], None, "fp4", "has no products with four-bit"),
    (dekinex_cases.CASES["A"], None, "fp4", "has no products with four-bit"), (sagalorn_cases.CASES["P"], None, "fp4", "has no products with four-bit"),
])
def test_models_that_cannot(config, kv_cache, weights, why):
    from glassbox_amd.engine.engine import EngineError, check_four_bits
    model = model_of(config)
    with pytest.raises(EngineError, match=why):
        check_four_bits(model, kv_cache, weights)
    check_four_bits(model, None, None)


@pytest.mark.parametrize("config", [helpers.TINY_B, helpers.WIDE_W, helpers.MID_M])
def test_models_that_can(config):
    from glassbox_amd.engine.engine import check_four_bits
    check_four_bits(model_of(config), "fp4", "fp4")
