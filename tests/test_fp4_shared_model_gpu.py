"""One loaded model and engines that hold its matrices in different types."""
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu


def test_engines_of_both_kinds_of_one_model():
    from glassbox_amd.config import config_from_dict
    from glassbox_amd.engine import Engine
    from glassbox_amd.engine.engine import EngineError
    from glassbox_amd.weights import build_model
    from glassbox_amd.weights.loader import random_tensors
    model = build_model(config_from_dict(helpers.TINY_B))
    model.load_tree(random_tensors(model, 7, 0.1, "uniform", torch.bfloat16, "cuda:0"))
    tokens = helpers.random_tokens(helpers.TINY_B["vocab_size"], 9, 1)
    whole = Engine(model, max_tokens=64, max_seqs=2)
    before = whole.step([("a", tokens, list(range(9)))]).clone()
    with pytest.raises(EngineError, match="another engine"):
        Engine(model, max_tokens=64, max_seqs=2, weights="fp4")
    whole.end_request("a")
    assert whole.weights is None and torch.equal(whole.step([("a", tokens, list(range(9)))]), before)
    pages = Engine(model, max_tokens=64, max_seqs=2, kv_cache="fp4")        # (its cache is its own)
    del whole, pages
    packed = Engine(model, max_tokens=64, max_seqs=2, weights="fp4")
    assert packed.weights == "fp4" and model.quantized
    with pytest.raises(EngineError, match="weights=None"):
        Engine(model, max_tokens=64, max_seqs=2)
    again = Engine(model, max_tokens=64, max_seqs=2, weights="fp4")
    assert torch.equal(again.step([("a", tokens, [8])]), packed.step([("a", tokens, [8])]))


@pytest.mark.parametrize("wrong", [dict(kernels="fast"), dict(prefix_caching=True)])
def test_a_call_that_is_refused_leaves_the_model_as_it_was(wrong):
    from glassbox_amd.engine import Engine
    from glassbox_amd.engine.engine import EngineError
    from fp4_positions import model_of
    from glassbox_amd.parts.attention import PagedAttention
    from glassbox_amd.parts.rotary import Rotary
    from glassbox_amd.weights.loader import random_tensors
    model = model_of([Rotary(64, 10000.0)])
    block = model.blocks[0]
    block.mixer = PagedAttention(96, 6, 2, 64, Rotary(64, 10000.0), window=20)      # (whose pages cannot be shared)
    model.load_tree(random_tensors(model, 7, 0.1, "uniform", torch.bfloat16, "cuda:0"))
    with pytest.raises(EngineError):
        Engine(model, max_tokens=64, max_seqs=2, kv_cache="fp4", weights="fp4", **wrong)
    assert not model.quantized and block.mixer.wqkv.dtype == torch.bfloat16
    Engine(model, max_tokens=64, max_seqs=2)
