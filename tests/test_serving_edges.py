"""Serving operators' host parts that test_serving.py leaves out, without a GPU."""
import ctypes as C

import pytest

import krafla_b200 as kb
from test_serving import cache


@pytest.fixture(scope="module", autouse=True)
def _built(built):
    return built


def test_workspace_size_needs_a_place():
    assert kb.lib().kc_paged_attend_ws(C.byref(cache()), 4, None) == kb.E_SHAPE
    assert "bytes" in kb.what_detail()
