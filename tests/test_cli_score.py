"""lssm_cli --score on the CPU: its flag errors (nothing here touches a GPU)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLI = os.path.join(ROOT, "lite_ssm_amd", "lssm_cli")

pytestmark = pytest.mark.skipif(not os.path.exists(CLI), reason="lssm_cli not built")


@pytest.mark.parametrize("args,msg", [
    (["--score", "--input-ids", "5"], "--score needs at least two ids"),
    (["--top-logprobs", "3", "--input-ids", "5,6"], "--top-logprobs needs --score"),
    (["--score", "--top-logprobs", "65", "--input-ids", "5,6"], "--top-logprobs: at most 64"),
    (["--score", "--top-logprobs"], "--top-logprobs expects an argument"),
    (["--score"], "provide a prompt text positionally"),
])
def test_flag_errors(args, msg):
    r = subprocess.run([CLI, *args], capture_output=True, text=True, timeout=60)
    assert r.returncode == 2, r
    assert f"lite-ssm: {msg}" in r.stderr


def test_help_names_it():
    r = subprocess.run([CLI, "--help"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "--score" in r.stderr and "--top-logprobs" in r.stderr


def test_python_front_end_hands_the_flags_on():
    from lite_ssm_amd.cli import split_args
    flags, words, _, _ = split_args(["--score", "--top-logprobs", "4", "a", "b"])
    assert flags == ["--score", "--top-logprobs", "4"] and words == ["a", "b"]
