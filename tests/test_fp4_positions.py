"""Four-bit pages and position encodings that do their own work, without a GPU."""
import pytest

from fp4_positions import Learned, LearnedInPlace, model_of
from glassbox_amd.parts.rotary import NoPosition, Rotary


def test_an_encoding_that_encodes_keys_only_on_their_way_into_pages_is_refused():
    from glassbox_amd.engine.engine import EngineError, check_four_bits
    model = model_of([Rotary(64, 10000.0), Learned(64, 128)])
    with pytest.raises(EngineError, match="cache layer 1: .*position encoding"):
        check_four_bits(model, "fp4", None)
    check_four_bits(model, None, "fp4")


def test_encodings_that_work_in_place_or_by_tables_are_taken():
    from glassbox_amd.engine.engine import check_four_bits
    check_four_bits(model_of([Rotary(64, 10000.0), LearnedInPlace(64, 128), NoPosition(), Rotary(64, 10000.0, (4.0, 64.0, 32.0, 1.0))]), "fp4", "fp4")
