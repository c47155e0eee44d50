"""Which memory the matrix products of the loss read: tests/c_abi/feed_check.cpp, host arithmetic only, and the one
instruction that makes the loads."""
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
BINARY = os.path.join(HERE, "c_abi", "feed_check.out")
SOURCE = os.path.join(os.path.dirname(HERE), "butterfly_amd", "csrc", "matmul.hpp")


def test_loads_stay_inside_their_operands():
    if not os.path.isfile(BINARY):
        recipe = os.path.join(HERE, "c_abi", "build.py")
        subprocess.run([sys.executable, "-c", f"import runpy; runpy.run_path({recipe!r})['build_feed']()"], check=True, timeout=300)
    run = subprocess.run([BINARY], capture_output=True, text=True, timeout=110)
    assert run.returncode == 0 and run.stdout.strip() == "all loads ok", (run.returncode, run.stdout)


def test_range_check_sees_the_whole_offset():
    # (the operand in front of `offen` would be added behind the check)
    with open(SOURCE) as f:
        loads = re.findall(r"buffer_load_dwordx4 (.*?) offen lds", f.read())
    assert loads and all(operands.split(",")[-1].strip() == "0" for operands in loads), loads
