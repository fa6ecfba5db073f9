"""The waits of the block-FP8 products' kernels, lane by lane on host threads (linear_waits_emulation.cpp)."""
import os
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
LINEAR = os.path.join(os.path.dirname(HERE), "unimonomoe_b200", "csrc", "linear")


@pytest.fixture(scope="module")
def emulation(tmp_path_factory):
    d = tmp_path_factory.mktemp("waits")
    text = open(os.path.join(LINEAR, "waits.cuh")).read()
    (d / "waits.cuh").write_text(text.replace('#include "barriers.cuh"\n', ""))
    exe = str(d / "waits")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-w", f'-DSOURCE="{d}/waits.cuh"', os.path.join(HERE, "linear_waits_emulation.cpp"), "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("case", ["lanes", "limit", "sent"])
def test_lanes_come_through_together_and_in_time(emulation, case):
    r = subprocess.run([emulation, case], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, f"{r.returncode}: {r.stdout}"


@pytest.mark.parametrize("kernel", ["few", "many"])
def test_what_the_ctas_of_a_cluster_send_is_waited_for_in_any_case(kernel):
    """Read from the source: the barrier that counts it is waited for by no wait that another's giving up ends."""
    text = "".join(re.sub(r"//.*", "", line) for line in open(os.path.join(LINEAR, f"linear_{kernel}.cu")))
    assert re.findall(r"(\w+)\(&C\.joined, 0\)", text) == ["wait_sent"]
