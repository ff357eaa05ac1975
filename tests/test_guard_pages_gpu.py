"""The op-level and whole-call GPU tests once more with GUARD PAGES behind (and in front of) every tensor the package allocates (tests/guard_pages.py): any kernel access
past the end of an operand ends the test process.  Round 6 found one such read by accident - the Winograd appendix of a layer with an odd
number of 16-channel blocks, harmless until the weights ended their memory segment - this run looks for them on purpose."""
import os
import subprocess

import pytest
import torch

import guard_pages

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def test_guarded_tensors_lie_at_the_edge_of_their_block():
    """The placement that the runs below rest on, read from the addresses alone: at most 15 bytes lie between a tensor's end (`end`) and its block's, none between the
    block's start and the tensor's (`start`); blocks are whole multiples of 2 MiB, so that the page behind (in front of) them belongs to no tensor."""
    for shape, dtype in (((16,), torch.float32), ((3, 5, 7), torch.bfloat16), ((1,), torch.int8), ((1 << 20,), torch.float32), (((1 << 19) + 1,), torch.float32)):
        for mode in ("end", "start"):
            t = guard_pages.guarded_empty(shape, dtype, torch.device("cuda:0"), mode)
            block = t.untyped_storage()
            front = t.data_ptr() - block.data_ptr()
            behind = block.nbytes() - front - t.numel() * t.element_size()
            assert block.nbytes() % (2 << 20) == 0 and t.is_contiguous() and tuple(t.shape) == shape and t.data_ptr() % 16 == 0
            assert (0 <= behind <= 15) if mode == "end" else (front == 0 and behind >= 0)


@pytest.mark.parametrize("mode", ["end", "start"])
def test_kernels_stay_inside_their_operands(mode):
    """Every convolution form (Winograd tiles / blocks / flat list with channel tails and odd block counts, second-generation narrow-row / streaming / stride-2 kernels, the
    random-shape sweep), the MaxStyle kernels, and one whole inner step at config 2 and config 4 (tests/test_round6_gpu.py::test_calls_are_bit_reproducible: every engine
    buffer, packed weight and table in its own guarded block) - one pytest process per file, each must finish."""
    files = ["tests/test_wino_gpu.py", "tests/test_conv_gpu.py", "tests/test_k3n_gpu.py", "tests/test_k1s_gpu.py", "tests/test_s2pro_gpu.py", "tests/test_gen2_random_gpu.py",
             "tests/test_maxstyle_gpu.py", "tests/test_round6_gpu.py"]
    if mode == "start":      # (the page in FRONT of a block: the Winograd family and the whole calls; `bash tools/guard_run.sh start` runs every file - clean at the end of round 6)
        files = ["tests/test_wino_gpu.py", "tests/test_k3n_gpu.py", "tests/test_round6_gpu.py"]
    r = subprocess.run(["bash", os.path.join(ROOT, "tools", "guard_run.sh"), mode] + files, cwd=ROOT, env=dict(os.environ, GRAFT_REPO_ROOT=ROOT), capture_output=True, text=True,
                       timeout=3000)
    lines = [l for l in r.stdout.splitlines() if l.startswith("guard=")]
    assert len(lines) == len(files), r.stdout[-2000:] + r.stderr[-500:]
    bad = [l for l in r.stdout.splitlines() if "EXIT CODE" in l or "failed" in l or "Memory access fault" in l]
    assert not bad, r.stdout[-3000:]
