"""One loaded model and engines that hold its matrices in different types, without a GPU: what is refused."""
import pytest

import helpers
from test_fp4 import model_of


class Holder:
    """In the place of an engine that runs the model"""


def test_a_quantized_model_is_not_run_as_if_it_were_none():
    from glassbox_amd.engine.engine import EngineError, check_four_bits
    model = model_of(helpers.TINY_B)
    model.quantized = True
    for kv_cache in (None, "fp4"):
        with pytest.raises(EngineError, match="weights=None: .* four bits already"):
            check_four_bits(model, kv_cache, None)
        check_four_bits(model, kv_cache, "fp4")


def test_a_model_that_an_engine_runs_is_not_quantized_under_it():
    from glassbox_amd.engine.engine import EngineError, check_four_bits
    model = model_of(helpers.TINY_B)
    engine = Holder()
    model.engines.add(engine)
    with pytest.raises(EngineError, match="weights='fp4': .* another engine"):
        check_four_bits(model, None, "fp4")
    with pytest.raises(RuntimeError, match="an engine runs"):
        model.quantize()
    assert not model.quantized
    check_four_bits(model, "fp4", None)         # (pages are an engine's own)
    del engine
    check_four_bits(model, None, "fp4")
