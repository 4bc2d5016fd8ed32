"""Engines whose cache or matrices, or both, are of four-bit numbers.  What the pages hold is compared with the keys and values that the plain
implementation makes (a number is the nearest of its block's, so it lies within half a step of them), and the logits with the plain
implementation's over the keys and values that the pages hold and the matrices rounded as the engine rounds them: what then differs is
arithmetic alone, and the bounds are those of any other engine."""
import functools
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import fp4_plain
import helpers
from plain import llama as plain

pytestmark = pytest.mark.gpu


@functools.lru_cache(maxsize=None)
def held_weights(folder, dtype, packed):
    """The checkpoint's tensors as an engine holds them"""
    cfg, w = helpers._load_rounded(folder) if dtype == "bfloat16" else helpers._load(folder)
    inner = lambda name, t: packed and t.dim() == 2 and name.startswith("model.layers.")
    return cfg, {name: (fp4_plain.rounded(t) if inner(name, t) else t).double() for name, t in w.items()}


def cached(eng, request, layer, n):
    """The keys and values of a request's first n tokens that four-bit pages hold, [n, kv heads, head size]"""
    lc = eng.layers[layer]
    k_pages, v_pages = lc.k_pages.cpu(), lc.v_pages.cpu()
    sid = eng._ids[request]
    k, v = zip(*(fp4_plain.get(k_pages, v_pages, eng.cache.slot(sid, t, lc.group)) for t in range(n)))
    return torch.stack(k), torch.stack(v)


def nearest(held, want, tol):
    """Whether the held numbers are the nearest of their blocks to numbers that are off from the wanted ones by ``tol`` of the block's largest:
    within half a step, and that.  The unit is the power of two that brings the block's largest into (3.5, 7]; steps are 1/2 of it up to 2
    units, 1 up to 4, 2 up to 6, and a largest of up to 7 reads as 6."""
    h, w = held.unflatten(-1, (-1, 32)), want.unflatten(-1, (-1, 32))
    top = w.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top * (1 + tol))          # (near a border of two units the larger, whose steps are nowhere the smaller ones)
    unit = torch.pow(2.0, (e - 3 + (2 * m > 1.75).int()).double())
    x = w.abs() / unit
    half = torch.where(x <= 2, 0.25, torch.where(x <= 4, 0.5, 1.0)) * unit
    return (h - w).abs() <= half + tol * top


def check(eng, folder, dtype, packed, request, tokens, got, bound):
    cfg, w = held_weights(folder, dtype, packed)
    nh, nkv, hd, T = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"], len(tokens)
    x = w["model.embed_tokens.weight"][torch.tensor(tokens)]
    for li in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{li}."
        h = plain.rms_norm(x, w[p + "input_layernorm.weight"], cfg["rms_norm_eps"])
        q, k, v = ((h @ w[p + f"self_attn.{n}_proj.weight"].T).reshape(T, -1, hd) for n in "qkv")
        q, k = (plain.rope(t, range(T), cfg["rope_theta"]) for t in (q, k))
        if eng.kv_cache:
            held = cached(eng, request, li, T)
            for what, mine, exact in zip(("keys", "values"), held, (k, v)):
                # 32 bits: 96 to 160 products, each off by 2^-24, and what the layers before add.  bfloat16: a row's numbers are off by 2^-8
                # each, which brings a sum of 96 of them up to 2^-8 times 6.3 / 2.3 of the block's largest (the sum of its terms' sizes
                # against the largest of 32 normal numbers), and the layers before are off by a few times 2^-8 themselves
                ok = nearest(mine, exact, 1e-4 if dtype == "float32" else 0.05)
                assert ok.all(), (request, li, what, torch.nonzero(~ok)[:4].tolist())
            k, v = held
        x = x + plain.attention(q, k, v).reshape(T, nh * hd) @ w[p + "self_attn.o_proj.weight"].T
        h = plain.rms_norm(x, w[p + "post_attention_layernorm.weight"], cfg["rms_norm_eps"])
        x = x + plain.swiglu(h, *(w[p + f"mlp.{n}_proj.weight"] for n in ("gate", "up", "down")))
    hs = plain.rms_norm(x, w["model.norm.weight"], cfg["rms_norm_eps"])
    head = w["lm_head.weight"] if ("lm_head.weight" in w and not cfg["tie_word_embeddings"]) else w["model.embed_tokens.weight"]
    bad = helpers.first_bad(np.asarray(got), (hs @ head.T).numpy(), bound)
    assert bad is None, f"request {request}: position {bad[0]} off by {bad[1]:.3e} (bound {bound:.3e})"


def run(eng, plan, got):
    """Steps of {request: tokens}; every position's logits are kept."""
    for step in plan:
        logits = eng.step([(r, t, list(range(len(t)))) for r, t in step.items()]).float().cpu().numpy()
        for r, t in step.items():
            got.setdefault(r, []).extend(logits[:len(t)])
            logits = logits[len(t):]


def mixed(requests):
    """A portion, portions beside single tokens, several portions of odd sizes, then single tokens of both."""
    a, b = requests["a"], requests["b"]
    plan = [{"a": a[:17]}, {"a": a[17:18], "b": b[:5]}, {"a": a[18:31], "b": b[5:6]}, {"b": b[6:22], "a": a[31:33]}]
    i, j = 33, 22
    while i < len(a) or j < len(b):
        plan.append({r: t for r, t in (("a", a[i:i + 1]), ("b", b[j:j + 1])) if t})
        i, j = i + 1, j + 1
    return plan


CASES = [(name, dtype, kv, packed) for name, kinds in (("B", ((1, 0), (0, 1), (1, 1))), ("D", ((1, 0),)), ("W", ((1, 1),)))
         for dtype in (("bfloat16",) if name == "W" else ("float32", "bfloat16")) for kv, packed in kinds]


@pytest.mark.parametrize("name,dtype,kv,packed", CASES)
@pytest.mark.parametrize("tapes,graphs", [(True, None), (False, False)])
def test_logits(model_dirs, bf16_bound, name, dtype, kv, packed, tapes, graphs):
    from glassbox_amd.engine import Engine
    folder = model_dirs.get(name, sharp=8.0 if dtype == "float32" else 1.0)
    vocab = helpers.TINY[name]["vocab_size"]
    requests = {"a": helpers.random_tokens(vocab, 45, 1), "b": helpers.random_tokens(vocab, 30, 2)}
    bound = helpers.TOL_F32 if dtype == "float32" else bf16_bound.get(folder, requests)
    eng = Engine(folder, dtype=dtype, max_tokens=256, max_seqs=4, layer_tapes=tapes, graph_decode=graphs, kv_cache="fp4" if kv else None,
                 weights="fp4" if packed else None)
    assert all((lc.k_pages.dtype == torch.uint8) == bool(kv) for lc in eng.layers) and eng.model.quantized == bool(packed)
    got = {}
    run(eng, mixed(requests), got)
    for r, tokens in requests.items():
        check(eng, folder, dtype, bool(packed), r, tokens, got[r], bound)
    if graphs is None and dtype == "bfloat16":
        assert eng.decode_graphs.replays > 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_shared_pages(model_dirs, bf16_bound, dtype):
    """A request that finds its beginning in the cache, and one that goes on from another's half-full page by itself."""
    from glassbox_amd.engine import Engine
    folder = model_dirs.get("B", sharp=8.0 if dtype == "float32" else 1.0)
    first = helpers.random_tokens(384, 40, 3)
    second, third = first[:35] + helpers.random_tokens(384, 6, 4), first + helpers.random_tokens(384, 5, 5)
    requests = {"first": first + [7, 8, 9], "second": second, "third": third}
    bound = helpers.TOL_F32 if dtype == "float32" else bf16_bound.get(folder, requests)
    eng = Engine(folder, dtype=dtype, max_tokens=256, max_seqs=4, prefix_caching=True, kv_cache="fp4", weights="fp4")
    got = {}
    eng.add_request("first", first)
    run(eng, [{"first": first}], got)
    reused = eng.add_request("second", second)
    assert reused == 32
    got["second"] = list(got["first"][:32])
    run(eng, [{"second": second[32:]}], got)
    eng.fork_request("first", "third")          # 40 tokens: the third page is half full and shared
    got["third"] = list(got["first"])
    run(eng, [{"third": third[40:41], "first": [7]}, {"first": [8], "third": third[41:]}, {"first": [9]}], got)
    for r, tokens in requests.items():
        check(eng, folder, dtype, True, r, tokens, got[r], bound)


def test_memory_and_reloading(model_dirs):
    """4.25 bits a number in the pages and the layers' matrices, and a model whose weights are loaded again is held as before."""
    from glassbox_amd.engine import Engine
    folder = model_dirs.get("W")
    whole, packed = (Engine(folder, max_tokens=512, max_seqs=2, kv_cache=k, weights=k) for k in (None, "fp4"))
    size = lambda eng: sum(t.numel() * t.element_size() for lc in eng.layers for t in (lc.k_pages, lc.v_pages))
    assert size(packed) * 16 == size(whole) * 4.25
    head = packed.model.embedding.vocab * packed.model.width * 2
    assert (packed.model.weight_bytes() - head) * 16 == (whole.model.weight_bytes() - head) * 4.25
    tokens = helpers.random_tokens(1000, 9, 6)
    before = packed.step([("r", tokens, list(range(9)))]).clone()
    from glassbox_amd.weights import load_weights
    load_weights(packed.model, folder + "/model.safetensors", packed.dtype, packed.device)
    packed.end_request("r")
    assert packed.model.blocks[0].mixer.wqkv.dtype == torch.uint8
    assert torch.equal(packed.step([("r", tokens, list(range(9)))]), before)


def test_the_command_line(model_dirs):
    from glassbox_amd.engine import Engine, greedy
    folder, root = model_dirs.get("B"), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "bin", "glassbox"), "generate", "--model", folder, "--prompt", "5,17,3,300,41", "-n",
                        "8", "--dtype", "float32", "--kv-cache", "fp4", "--weights", "fp4"], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr
    eng = Engine(folder, dtype="float32", max_tokens=64, max_seqs=1, kv_cache="fp4", weights="fp4")
    assert [int(t) for t in r.stdout.split()] == greedy(eng, [5, 17, 3, 300, 41], 8)


@pytest.mark.parametrize("packed", [False, True])
def test_a_window_and_a_layer_that_reads_another_ones_cache(packed):
    """Three layers: all keys; the last twenty, whose pages are given back on the way; the first layer's cache, read alone."""
    from glassbox_amd.config import config_from_dict
    from glassbox_amd.engine import Engine
    from glassbox_amd.parts.attention import PagedAttention
    from glassbox_amd.parts.block import PreNormBlock
    from glassbox_amd.parts.embedding import Embedding, LMHead
    from glassbox_amd.parts.mlp import SwiGLU
    from glassbox_amd.parts.model import DecoderModel, LayerCall
    from glassbox_amd.parts.norm import RMSNorm
    from glassbox_amd.parts.rotary import Rotary
    from glassbox_amd.weights.loader import random_tensors
    d, H, G, D, vocab, eps, theta, window = 96, 6, 2, 64, 90, 1e-5, 10000.0, 20
    rotary = Rotary(D, theta)
    layer = lambda **how: PreNormBlock(RMSNorm(d, eps), PagedAttention(d, H, G, D, rotary, **how), RMSNorm(d, eps), SwiGLU(d, 160))
    embedding = Embedding(vocab, d)
    cfg = config_from_dict(dict(helpers.TINY_B, hidden_size=d, intermediate_size=160, num_hidden_layers=3, num_attention_heads=H,
                                num_key_value_heads=G, head_dim=D, vocab_size=vocab, rope_theta=theta, rms_norm_eps=eps, tie_word_embeddings=True))
    model = DecoderModel(cfg, embedding, [layer(), layer(window=window), layer(shares_kv=True)],
                         [LayerCall(0, cache=0), LayerCall(1, cache=1), LayerCall(2, reads=0)], RMSNorm(d, eps), LMHead(vocab, d, tied_to=embedding))
    tensors = random_tensors(model, 7, 0.1, "uniform", torch.float32, "cuda:0")
    model.load_tree(tensors)
    w = {n: t.cpu() for n, t in tensors.items()}
    w = {n: (fp4_plain.rounded(t) if packed and n.startswith("model.layers.") and t.dim() == 2 else t).double() for n, t in w.items()}
    eng = Engine(model, dtype="float32", max_tokens=256, max_seqs=2, kv_cache="fp4", weights="fp4" if packed else None)
    assert len(eng.group_keys) == 2
    tokens, held, got, at = helpers.random_tokens(vocab, 70, 8), {0: [], 1: []}, [], 0
    for n in (16, 13, 1, 16, 9) + (1,) * 15:
        got.extend(eng.step([("r", tokens[at:at + n], list(range(n)))]).cpu().numpy())
        at += n
        for c, kept in held.items():      # (what this step brought: the window's pages go back later)
            lc, sid = eng.layers[c], eng._ids["r"]
            k_pages, v_pages = lc.k_pages.cpu(), lc.v_pages.cpu()
            kept += [fp4_plain.get(k_pages, v_pages, eng.cache.slot(sid, t, lc.group)) for t in range(at - n, at)]
    assert at == 70 and eng.cache.table(eng._ids["r"], 1)[:2] == [-1, -1]
    x = w["model.embed_tokens.weight"][torch.tensor(tokens)]
    for li, (source, seen) in enumerate(((0, 0), (1, window), (0, 0))):
        p = f"model.layers.{li}."
        h = plain.rms_norm(x, w[p + "input_layernorm.weight"], eps)
        k, v = (torch.stack(t) for t in zip(*held[source]))
        if li < 2:
            made_k, made_v = ((h @ w[p + f"self_attn.{n}_proj.weight"].T).reshape(70, G, D) for n in "kv")
            assert nearest(k, plain.rope(made_k, range(70), theta), 1e-4).all() and nearest(v, made_v, 1e-4).all()
        q = plain.rope((h @ w[p + "self_attn.q_proj.weight"].T).reshape(70, H, D), range(70), theta)
        x = x + plain.attention(q, k, v, seen).reshape(70, H * D) @ w[p + "self_attn.o_proj.weight"].T
        h = plain.rms_norm(x, w[p + "post_attention_layernorm.weight"], eps)
        x = x + plain.swiglu(h, *(w[p + f"mlp.{n}_proj.weight"] for n in ("gate", "up", "down")))
    want = (plain.rms_norm(x, w["model.norm.weight"], eps) @ w["model.embed_tokens.weight"].T).numpy()
    bad = helpers.first_bad(np.asarray(got), want, helpers.TOL_F32)
    assert bad is None, f"position {bad[0]} off by {bad[1]:.3e}"


def test_norms_that_the_products_do_are_those_of_their_own_launch(monkeypatch):
    """Rows whose squares' sums are exact, so that their order does not matter: the first layer adds nothing to an embedding of halves."""
    from glassbox_amd import ops
    from glassbox_amd.config import config_from_dict
    from glassbox_amd.engine import Engine
    from glassbox_amd.weights import build_model
    from glassbox_amd.weights.loader import random_tensors
    d, inter, vocab = 1056, 8224, 90
    cfg = config_from_dict(dict(helpers.TINY_B, hidden_size=d, intermediate_size=inter, num_hidden_layers=2, num_attention_heads=4,
                                num_key_value_heads=2, head_dim=64, vocab_size=vocab))
    model = build_model(cfg)
    tensors = random_tensors(model, 7, 0.1, "uniform", torch.bfloat16, "cuda:0")
    for name in ("self_attn.o_proj", "mlp.down_proj"):
        tensors[f"model.layers.0.{name}.weight"].zero_()
    tensors["model.embed_tokens.weight"].copy_(torch.randint(-3, 4, (vocab, d), generator=torch.Generator().manual_seed(3)) * 0.5)
    model.load_tree(tensors)
    asked, mode = [], ops.fp4_gemm_emit_mode
    got = []
    for on in (True, False):
        monkeypatch.setattr(ops, "fp4_gemm_emit_mode", lambda m, n, k: (asked.append((m, mode(m, n, k))), mode(m, n, k))[1] if on else 0)
        eng = Engine(model, dtype="bfloat16", max_tokens=1024, max_seqs=48, kv_cache="fp4", weights="fp4")
        first = eng.step([("r", helpers.random_tokens(vocab, 33, 1), list(range(33)))]).clone()
        got.append([first] + [eng.step([((m, i), [3 * i % vocab], [0]) for i in range(m)])[:m].clone() for m in (12, 32)])
        del eng
    assert {(33, 2), (32, 2)} <= set(asked)
    for mine, apart in zip(*got):
        assert mine.isfinite().all() and torch.equal(mine[:, :vocab], apart[:, :vocab])
