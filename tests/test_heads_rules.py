"""Rules of the embedding heads' kernels that no GPU run may break on purpose, checked without one: how a role's
waiting ends (csrc/wait_rules.h run on the host), and that the kernels' source keeps to it."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import ROOT

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(ROOT, "robot-agent_b200", "csrc")


def _code(name):
    """A source file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def test_long_wait_ends(tmp_path):
    """A wait for a whole tile ends when the tile does, when any role of the pair has given up, or at its limit."""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path / "pair_wait")
    subprocess.run([cxx, "-O1", "-std=c++17", "-o", exe, os.path.join(HERE, "pair_wait_check.cpp")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


def test_failure_reaches_both_ctas_of_a_pair():
    """Every role that gives up does so through pr_fail, which marks the other CTA too."""
    s = _code("k_prod.cuh")
    kernel = s[s.index("__global__"):]
    assert not re.search(r"(\*\s*failed|sh_fail)\s*=\s*1", kernel)
    assert kernel.count("pr_fail<PAIR>(failed)") >= 7         # loads, MMAs, scales twice, relay, results, tensor memory
    fail = s[s.index("DEV void pr_fail"):]
    assert "st.relaxed.cluster.shared::cluster" in fail[:fail.index("\n}")]
    assert "while (!ag_wait" not in s                         # no wait without a limit of its own


def test_arrivals_cross_a_pair_with_release_and_acquire():
    """What one CTA of a pair reports to the other's barriers (landed stages, scales, zeros, read accumulators) is released
    and acquired at cluster scope, wherever the leader waits for it."""
    s, tc = _code("k_prod.cuh"), _code("tc_util.cuh")
    assert s.count("mbarrier.arrive.relaxed.cluster.shared::cluster") == 1
    arrive = s[s.index("DEV void pr_arrive_leader"):]
    assert re.search(r"fence\.release\.sync_restrict::shared::cta\.cluster;.*mapa.*mbarrier\.arrive\.relaxed\.cluster", arrive, re.S)
    assert not re.search(r"mbarrier\.arrive\.shared::cluster", s)               # no arrival there without the fence
    assert "mbarrier.try_wait.parity.relaxed.cluster" in tc and "mbarrier.test_wait.parity.relaxed.cluster" in s
    assert re.search(r"ag_wait<PAIR>.*pr_acquire_pair", s, re.S) and "fence.acquire.sync_restrict::shared::cluster.cluster" in s
    barriers = set(re.findall(r"pr_arrive_leader\(&(\w+)\[", s))
    assert barriers == {"cpeer", "fixed", "tempty"}
    assert re.search(r"wait_pair\(&cpeer\[", s) and re.search(r"wait_pair\(&tempty\[", s) and re.search(r"RELAY \? wait_pair\(&landed\[", s)
    assert re.search(r"pr_test<PAIR>\(&landed", s) and re.search(r"else if \(PAIR\) \{\s*pr_acquire_pair\(\)", s)


@pytest.mark.parametrize("name", ["k_mx.cuh", "k_norm.cuh", "k_few.cuh", "k_prod.cuh"])
def test_no_read_only_loads_under_programmatic_launch(name):
    """A kernel that starts before the one that writes its inputs has ended must not read them by the non-coherent path, which
    is for memory that nobody writes while the kernel runs (weights and gains too: a training step writes them)."""
    s = _code(name)
    assert "__ldg" not in s and "ld.global.nc" not in s and "__restrict__" not in s
