"""conftest.py's rule for machines that refuse to register existing host memory with the GPU."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

SUITE = '''
import pytest

pytestmark = pytest.mark.gpu

def test_first_job():
    raise AssertionError("rank 0 ... esgd: hipHostRegister(seg, sizeof(Segment), hipHostRegisterMapped) failed: "
                         "invalid argument (dataplane.cpp:374)")

@pytest.mark.parametrize("world", [1, 2])
def test_job(world):
    open(f"ran_{world}", "w").close()

def test_job_that_fails_by_itself():
    raise AssertionError("rank 1: wrong sum")
'''
SOUND_FIRST = SUITE.replace("def test_first_job", "def test_other_first():\n    raise AssertionError('invalid argument')\n\ndef test_first_job")


def _suite(tmp_path, text, ranks):
    (tmp_path / "test_jobs.py").write_text(text)
    env = {k: v for k, v in os.environ.items() if k not in ("ESGD_TEST_RANKS", "PYTEST_ADDOPTS")}
    env["PYTHONPATH"] = os.path.join(ROOT, "tests")
    if ranks is not None:
        env["ESGD_TEST_RANKS"] = ranks
    r = subprocess.run([sys.executable, "-m", "pytest", "-p", "conftest", "-p", "no:cacheprovider", "-q", "-rs", "-m", "gpu",
                        "test_jobs.py"], cwd=tmp_path, env=env, capture_output=True, text=True, timeout=120)
    ran = sorted(p.name for p in tmp_path.glob("ran_*"))
    return r.stdout.splitlines()[-1], ran, r.stdout


@pytest.mark.parametrize("ranks,last,ran", [
    (None, "1 passed, 3 skipped", ["ran_1"]),             # seen in the first job: that and what needs the same
    ("0", "1 passed, 3 skipped", ["ran_1"]),              # known beforehand: no job is started
    ("1", "2 failed, 2 passed", ["ran_1", "ran_2"]),      # asked for: a refusal is a failure
])
def test_refused_registration_skips_the_jobs_of_several_ranks(tmp_path, ranks, last, ran):
    got, did, out = _suite(tmp_path, SUITE, ranks)
    assert got.startswith(last) and did == ran, out
    assert ("hipHostRegister" in out) and ("jobs of several ranks" in out) == (ranks != "1"), out


def test_other_failures_stay_failures(tmp_path):
    got, did, out = _suite(tmp_path, SOUND_FIRST, None)
    assert got.startswith("1 failed, 1 passed, 3 skipped") and did == ["ran_1"], out
