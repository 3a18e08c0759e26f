"""The operators of long contexts through the extension module and through ctypes: the same arguments taken and refused (no GPU needed)."""
import pytest

import effect_torch_b200 as et
from tests import test_calls as calls

PARAMETERS = {"logprobs_into": "ppwwwpppwpp", "rotary_into": "pppwwwpwwwwpwww", "paged_append_into": "ppwppwwpp", "pool_rows_into": "ppwwpwp"}


@pytest.mark.parametrize("make", [calls.module, et._ThroughCtypes])
@pytest.mark.parametrize("name", sorted(PARAMETERS))
def test_operators_take_and_refuse_the_same_arguments(make, name, monkeypatch):
    monkeypatch.setitem(calls.PARAMETERS, name, PARAMETERS[name])
    calls.test_operators_take_and_refuse_the_same_arguments(make, name)


@pytest.mark.parametrize("name", sorted(PARAMETERS))
def test_the_stand_in_hands_over_what_the_arguments_stand_for(name, monkeypatch):
    monkeypatch.setitem(calls.PARAMETERS, name, PARAMETERS[name])
    calls.test_the_stand_in_hands_over_what_the_arguments_stand_for(name, monkeypatch)
