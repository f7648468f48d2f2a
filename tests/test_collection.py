"""What the collection does to the suite (tests/conftest.py), from whatever directory a run starts.  Nothing is run."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SHOW = """
import sys, pytest

class Show:
    def pytest_collection_finish(self, session):
        for item in session.items:
            print("ITEM", item.path.name, item.name, int(item.get_closest_marker("skip") is not None))

sys.exit(pytest.main(["--collect-only", "-q", "-p", "no:cacheprovider"] + sys.argv[1:], plugins=[Show()]))
"""


def _collected(cwd, *paths):
    out = subprocess.run([sys.executable, "-c", SHOW, *paths], cwd=cwd, capture_output=True, text=True, timeout=240)
    assert out.returncode == 0, out.stdout + out.stderr
    return [line.split()[1:] for line in out.stdout.splitlines() if line.startswith("ITEM")]


@pytest.mark.parametrize("cwd,prefix", [(os.path.dirname(HERE), "tests/"), (HERE, ""), (os.path.dirname(os.path.dirname(HERE)), None)])
def test_the_case_that_faulted_is_skipped(cwd, prefix):
    path = os.path.join(HERE, "test_gpu_ops.py") if prefix is None else prefix + "test_gpu_ops.py"
    skipped = [name for file, name, skip in _collected(cwd, path) if skip == "1"]
    assert skipped == ["test_ssim_against_torch_conv[shape2]"]


def test_the_expert_tests_come_last():
    files = [file for file, _, _ in _collected(HERE, "-m", "gpu", "test_gpu_experts.py", "test_gpu_experts_slope.py", "test_gpu_mx4.py",
                                               "test_gpu_ops.py", "test_gpu_ssim_host_reference.py")]
    expert = [f.startswith(("test_gpu_experts", "test_gpu_mx4")) for f in files]
    assert any(expert) and expert == sorted(expert)
