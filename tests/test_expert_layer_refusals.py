"""Argument errors of the expert layer's types with EXPERT_HIDDEN_F32 are reported before any device call (no GPU)."""
import ctypes as C

import pytest

from helpers import pkg
from test_serving_refusals import FAKE, error, layer_option


@pytest.mark.parametrize("change,text", [
    (dict(dataType=3 | 0x100), "type"), (dict(dataType=2 | 0x200), "type"), (dict(dataType=-1), "type"),
    (dict(routerType=1 | 0x100), "type"), (dict(dataType=1 | 0x100, strideX=63), "strides")])
def test_types(change, text):
    args = (FAKE,) * 2 + (None,) + (FAKE,) * 4 + (FAKE + (1 << 20), 4, None)
    assert text in error("launchExpertLayer", C.byref(layer_option(**change)), *args)


def test_nothing_to_do():
    for t in range(3):
        o = layer_option(dataType=t | pkg().EXPERT_HIDDEN_F32)
        assert error("launchExpertLayer", C.byref(o), *[None] * 8, 0, None) == ""
