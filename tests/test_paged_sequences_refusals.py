"""Refused calls of PagedSequences leave nothing behind."""
import importlib

import pytest


def test_negative_numbers_of_tokens(abq):
    att = importlib.import_module("abq_llm_b200.attention")
    p = att.PagedSequences(4, 16)
    with pytest.raises(ValueError):
        p.add(-1)
    with pytest.raises(KeyError):
        p.length(0)  # no sequence came of it
    a = p.add(3)
    with pytest.raises(ValueError):
        p.slots(a, -1)
    assert p.slots(a, 0) == [] and len(p.slots(a, 3)) == 3
