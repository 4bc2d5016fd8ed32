"""Engines with four-bit pages whose position encodings do their own work: a learned table, and turns that are stretched."""
import numpy as np
import pytest
import torch

import fp4_plain
import helpers
from fp4_positions import LearnedInPlace, model_of
from plain import llama as plain
from test_fp4_engine_gpu import nearest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [False, True])
def test_the_cached_keys_and_the_logits(packed):
    """What the pages hold is the nearest to the encoded keys, and the logits are the plain model's over what the pages hold."""
    from glassbox_amd.engine import Engine
    from glassbox_amd.parts.rotary import Rotary
    from glassbox_amd.weights.loader import random_tensors
    H, G, D, d, eps, n = 6, 2, 64, 96, 1e-5, 40
    stretched = Rotary(D, 10000.0, (4.0, 16.0, 8.0, 1.0))
    assert stretched.magnitude != 1.0
    model = model_of([LearnedInPlace(D, 64), stretched])
    tensors = random_tensors(model, 7, 0.1, "uniform", torch.float32, "cuda:0")
    model.load_tree(tensors)
    w = {name: t.cpu() for name, t in tensors.items()}
    w = {name: (fp4_plain.rounded(t) if packed and name.startswith("model.layers.") and name.endswith("proj.weight") else t).double() for name, t in w.items()}
    eng = Engine(model, dtype="float32", max_tokens=64, max_seqs=2, kv_cache="fp4", weights="fp4" if packed else None)
    tokens, got, at = helpers.random_tokens(90, n, 8), [], 0
    for rows in (17, 1, 12) + (1,) * 10:
        got.extend(eng.step([("r", tokens[at:at + rows], list(range(rows)))]).cpu().numpy())
        at += rows
    x = w["model.embed_tokens.weight"][torch.tensor(tokens)]

    def turned(t):
        angle = torch.arange(n)[:, None].float() * torch.from_numpy(stretched.inv_host)      # (32-bit angles, as everywhere)
        c, s = angle.double().cos()[:, None], angle.double().sin()[:, None]
        lo, hi = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)

    for li, encoded in enumerate((lambda t: t + w["model.layers.0.self_attn.position_table"][:n, None], turned)):
        p = f"model.layers.{li}."
        h = plain.rms_norm(x, w[p + "input_layernorm.weight"], eps)
        q, made_k, made_v = ((h @ w[p + f"self_attn.{m}_proj.weight"].T).reshape(n, -1, D) for m in "qkv")
        lc, sid = eng.layers[li], eng._ids["r"]
        k_pages, v_pages = lc.k_pages.cpu(), lc.v_pages.cpu()
        k, v = (torch.stack(t) for t in zip(*(fp4_plain.get(k_pages, v_pages, eng.cache.slot(sid, t, lc.group)) for t in range(n))))
        assert nearest(k, encoded(made_k), 1e-4).all() and nearest(v, made_v, 1e-4).all(), li
        x = x + plain.attention(encoded(q), k, v).reshape(n, H * D) @ w[p + "self_attn.o_proj.weight"].T
        h = plain.rms_norm(x, w[p + "post_attention_layernorm.weight"], eps)
        x = x + plain.swiglu(h, *(w[p + f"mlp.{m}_proj.weight"] for m in ("gate", "up", "down")))
    want = (plain.rms_norm(x, w["model.norm.weight"], eps) @ w["model.embed_tokens.weight"].T).numpy()
    bad = helpers.first_bad(np.asarray(got), want, helpers.TOL_F32)
    assert bad is None, f"position {bad[0]} off by {bad[1]:.3e}"
