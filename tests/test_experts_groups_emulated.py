"""Grouping of so many places that their workgroups' counts are summed by a launch of its own, on the CPU SIMT emulation."""
import pytest

from dimo_amd import experts as ex
from tests import expert_cases as cases
from tests import expert_emulation


@pytest.mark.parametrize("T,k,E,skew", [(20491, 8, 1000, False), (83977, 2, 1024, True)])
def test_group(monkeypatch, T, k, E, skew):
    expert_emulation.use(monkeypatch, ex)
    cases.check_group(ex, "cpu", T, k, E, seed=T, skew=skew)
