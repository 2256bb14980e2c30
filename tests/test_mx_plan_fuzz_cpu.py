"""Random programs of microscaled and plain steps: the two-stream plan orders every conflicting pair
(tests/plan_hazards.py), and is the list schedule that its rule describes."""
import pytest

from synaptik_amd.native import program_plan, validate_program_image
from tests import plan_hazards as H
from tests.conftest import needs_two_streams
from tests.mx_programs import random_program


@pytest.mark.parametrize("seed", range(80))
def test_random_microscaled_programs_have_no_races(seed):
    image = random_program(seed)[0].image()
    validate_program_image(image)
    streams, waits, folded = program_plan(image)
    hazards = H.check_plan(H.decode(image), streams, waits, folded)
    assert not hazards, "; ".join(map(str, hazards))


@needs_two_streams
def test_the_plan_uses_both_streams():
    """Somewhere in the programs each microscaled step runs on the side stream."""
    beside = set()
    for seed in range(80):
        image = random_program(seed)[0].image()
        streams, _, _ = program_plan(image)
        beside |= {st.opcode for st, s in zip(H.decode(image), streams) if s == 1}
    assert {17, 18, 19, 20, 21} <= beside
