"""What the key/value cache operators refuse, without a GPU (the C entries get addresses that nothing reads: every call below
ends before it touches a device)."""
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import pingala8_llm_b200 as p8  # noqa: E402
from test_cache_ops import ARG  # noqa: E402


@pytest.mark.parametrize("ns", [-1, 1 << 32, -(1 << 62)])
def test_a_wait_limit_out_of_range(ns):
    assert p8.lib().p8_cache_wait_limit(ns) == ARG
