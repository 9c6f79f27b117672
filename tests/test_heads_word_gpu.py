"""The device's error word, made by a process's first product: inside a stream capture, in inference mode, on a side
stream.  Each case is a process of its own."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT, has_gpu

pytestmark = pytest.mark.gpu

START = """
import sys, torch
sys.path[:0] = [%r, %r]
from scenemap_b200 import products as P
torch.manual_seed(1)
x, w = torch.randn(40, 64, device="cuda").bfloat16(), torch.randn(2, 16, 64, device="cuda").bfloat16()
off, bad = (torch.tensor(o, dtype=torch.int32, device="cuda") for o in ([0, 7, 40], [0, 50, 40]))
torch.cuda.synchronize()
""" % (os.path.join(ROOT, "robot-agent_b200"), os.path.join(ROOT, "tests"))

CASES = {
    # the first product is captured: the capture holds, and the word is set by its replays and by nothing else
    "capture": """
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = P.grouped(x, w, off)
    P.grouped(x, w, bad)
assert P.error() == 0
g.replay()
assert P.error() == P.BAD_OFFSETS
assert torch.equal(y, P.grouped(x, w, off))
P.clear_error()
assert P.error() == 0
g.replay()
assert P.error() == P.BAD_OFFSETS
""",
    # the word made in inference mode is used outside of it
    "inference": """
with torch.inference_mode():
    P.grouped(x, w, bad)
assert P.error() == P.BAD_OFFSETS
P.clear_error()
assert P.error() == 0
with torch.inference_mode():
    P.clear_error()
P.grouped(x, w, off)
assert P.error() == 0
""",
    "side stream": """
s = torch.cuda.Stream()
with torch.cuda.stream(s):
    P.grouped(x, w, bad)
    assert P.error() == P.BAD_OFFSETS
P.clear_error()
assert P.error() == 0
""",
}


@pytest.mark.parametrize("case", list(CASES))
def test_first_product(case):
    if not has_gpu():
        pytest.skip("no GPU")
    r = subprocess.run([sys.executable, "-c", START + CASES[case] + "\nprint('done')"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout[-500:] + r.stderr[-1500:]
