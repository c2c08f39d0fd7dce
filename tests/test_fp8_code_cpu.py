"""The norm's branch-free FP8 activation code equals the official rule's on every float."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_short_code_is_the_rule_on_every_float(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fopenmp", "-ffp-contract=off", "-I", os.path.join(ROOT, "objeta_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "fp8_code_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, check=True, timeout=600).stdout
    assert out.strip() == "0"
