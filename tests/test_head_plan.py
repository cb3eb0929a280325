"""How the streaming kernels over rows of logits share out a block and talk to one
another, walked through on the host (head_plan_check.cpp)."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "hexatrain_b200", "csrc")


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "head_plan_check")
    subprocess.run(["g++", "-std=c++17", "-O2", "-x", "c++", f"-I{CSRC}", os.path.join(HERE, "head_plan_check.cpp"), "-o",
                    exe], check=True)

    def run(what):
        r = subprocess.run([exe, what], capture_output=True, text=True)
        assert r.returncode == 0, r.stdout + r.stderr

    return run


def test_every_top_logits_call_can_finish(check):
    """Every element size, vocabulary, alignment and record length: the block's memory
    holds the plan, and consumers, row warps and the ring's producer never wait for one
    another in a circle, however many rows a block takes."""
    check("top")


def test_exchange_of_a_cluster_in_every_order(check):
    """Three CTAs, four exchanges, every order in which sends arrive: each CTA reads
    what was sent for its exchange (with one barrier for all exchanges it may not)."""
    check("exchange")
