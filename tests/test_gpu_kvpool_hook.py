"""A serving step's slot plan as the hook's slot list."""
from __future__ import annotations

import pytest

import mp_workers
from test_hook import run_ranks

pytestmark = pytest.mark.gpu


def test_padded_plan_is_protected_and_recovered():
    for _rank, ok in run_ranks(mp_workers.hook_plan, 2, "gloo", timeout=300):
        assert ok is True
