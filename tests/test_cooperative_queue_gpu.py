"""GPU: who takes the device's cooperative queue, and what a refusal of it lasts.

One process at a time can have the queue, to its end.  A decoder asks for it before its first persistent step: not at
creation, not for steps that are no persistent ones, and not when the library is asked for what it knows."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CFG = (256, 768, 2, 4, 2, 1024, 128)
HEAD = f"""
import sys
sys.path.insert(0, {REPO!r})
from __graft_entry__ import _pkg
_pkg()
from hip_llama_cpp_amd import thallama as tl
tl.check(tl.lib().thallama_set_device(0))
m = tl.DeviceModel(tl.Config.make(*{CFG}), 0, seed=5)
keep = []
def decode(batch):
    s = tl.DeviceState(tl.Config.make(*{CFG}), batch)
    d = tl.Decoder(m, s)
    keep.extend([s, d])
    d.set(tl.OPT_USE_GRAPH, 1)
    t, got = [1] * batch, []
    for i in range(8):
        t = d.greedy(t, [i] * batch, 1)[0].tolist()
        got.append(t[0])
    print("tokens", batch, int(d.persistent()), tl.lib().thallama_persistent_cooperative(), *got, flush=True)
"""


def start(code):
    return subprocess.Popen([sys.executable, "-u", "-c", HEAD + code], stdin=subprocess.PIPE, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)


def line(p):
    got = p.stdout.readline().split()
    assert got[:1] == ["tokens"], p.stderr.read()[-3000:]
    return [int(x) for x in got[1:]]


def end(p):
    out, err = p.communicate("\n", timeout=60)
    assert p.returncode == 0, err[-3000:]
    return [[int(x) for x in y.split()[1:]] for y in out.splitlines() if y.startswith("tokens")]


def test_a_refusal_ends_with_the_holder(gpu, oracle):
    """A decoder that is refused the queue launches plainly; the next one gets it when the holder has gone."""
    want = oracle.Model(CFG, 0, seed=5).greedy(1, 0, 8)
    p = start("decode(1)\nsys.stdin.readline()\n")
    free = line(p)[2]
    if not free:
        end(p)
        pytest.skip("this process has the cooperative queue, or another one does")
    q = start("decode(1)\nsys.stdin.readline()\ndecode(1)\n")
    assert line(q) == [1, 1, 0] + want
    end(p)
    assert end(q) == [[1, 1, 1] + want]


def test_steps_that_are_not_persistent_leave_the_queue(gpu, oracle):
    """While another process has the queue: six sequences, whose steps are several launches by default, do not ask for
    it (it would be refused, and reported); one sequence does."""
    dec_state = gpu.DeviceState(gpu.Config.make(*CFG), 1)
    model = gpu.DeviceModel(gpu.Config.make(*CFG), 0, seed=5)
    dec = gpu.Decoder(model, dec_state)
    want = oracle.Model(CFG, 0, seed=5).greedy(1, 0, 8)
    assert dec.greedy([1], [0], 8)[:, 0].tolist() == want  # this process has it from here on, or another one does
    if not gpu.lib().thallama_persistent_cooperative():
        pytest.skip("another process has the cooperative queue")
    p = start("print('tokens', 0, 0, tl.lib().thallama_persistent_cooperative(), flush=True)\ndecode(6)\ndecode(1)\n")
    assert end(p) == [[0, 0, 1], [6, 0, 1] + want, [1, 1, 0] + want]
    dec.close()
