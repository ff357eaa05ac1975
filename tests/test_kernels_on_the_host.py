"""The kernels of the many-class loss and of the 8-bit checkpoints executed lane by lane on the CPU (tests/host_kernels), every buffer between unmapped pages: an access
outside an operand or the workspace ends the child process, which has printed its case.  Random shapes of every form, both alignments, workspaces of zeros and of NaNs, results against the
definition in 64 bits.  Each run is a process of its own."""
import os
import subprocess
import sys

import pytest

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_kernels")
sys.path.insert(0, HERE)
import build  # noqa: E402

pytestmark = pytest.mark.skipif(not os.path.exists(build.CLANG), reason="needs the host compiler of the ROCm toolchain")
ENV = dict(os.environ, OMP_NUM_THREADS="2", OPENBLAS_NUM_THREADS="2")


def child(args):
    return subprocess.run([sys.executable] + args, cwd=HERE, env=ENV, capture_output=True, text=True, timeout=900)


@pytest.mark.parametrize("which,seed,count", [("class_ce", 3, 120), ("class_ce", 1, 60), ("class_ce_pieces", 2, 80), ("logit_ce", 1, 100), ("act8", 1, 60)])
def test_every_access_is_inside_its_buffer(which, seed, count):
    r = child(["sweep.py", which, str(seed), str(count)])
    assert r.returncode == 0 and r.stdout.endswith("done\n"), (r.returncode, r.stdout[-400:], r.stderr[-800:])


def test_an_access_outside_ends_the_child():
    """What the runs above rest on: a plane told one element longer than its buffer, in front of the page and behind it."""
    code = ("import guarded as g, build, numpy as np\nlib = build.load()\nc = g.Call('%s')\nx = c.put(np.ones((1, 1, %d), np.float32)); q = c.block(8192); s = c.block(64)\n"
            "print(lib.ms_act8_pack(g.p(x), None, g.p(q), g.p(s), 1, 1, %d, None), flush=True)")
    assert child(["-c", code % ("end", 1024, 1024)]).stdout == "0\n"
    assert child(["-c", code % ("end", 1024, 1025)]).returncode == -11


@pytest.mark.parametrize("form", ["wide", "narrow"])
def test_gradients_of_rows_and_classes_of_any_size(form):
    r = child(["scales.py", form])
    assert r.returncode == 0 and r.stdout.endswith("done\n"), "\n".join(l for l in r.stdout.splitlines() if "FAIL" in l) + r.stderr[-800:]
