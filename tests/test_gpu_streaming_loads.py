"""The residual norm's kernels for calls larger than the last-level cache, which read past it: instantiations of their
own.  LBN_STREAM_LOADS=1, read once per process, sends calls of any size to them, so a child process runs small
shapes of every team and every combination of parts through the comparisons of tests/test_gpu_stream_operators.py."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# rows (multiples of eight: others never take these kernels) by team: sixteen lanes with one and two units, single
# waves, several waves, the widest teams, forward with two units a lane; columns; padding and offset of the buffers
SHAPES = [(8, 40, 0, 0), (72, 150, 3, 1), (200, 60, 0, 0), (512, 40, 0, 0), (640, 70, 0, 0), (1024, 66, 5, 3), (4096, 12, 0, 0), (4104, 9, 8, 8),
          (8192, 6, 0, 0), (12288, 6, 0, 0)]
MORE_KINDS = [("none", "layer", 0, 0.9, True), ("layer", "rms", 0, 1.0, True)]  # biases without a gate
RANGES = [(4104, 620, ("layer", "rms", 4, 0.9, True)), (8192, 520, ("none", "rms", 20, 1.0, True)),
          (1024, 2200, ("none", "rms", 22, 1.0, False)), (4096, 600, ("rms", "rms", 600, 1.0, False)),
          (504, 1200, ("rms", "layer", 0, 1.0, False)), (128, 3000, ("none", "layer", 100, 1.0, True))]


def run():
    from lbann_amd import layers as L
    from tests import test_gpu_stream_operators as T
    assert os.environ["LBN_STREAM_LOADS"] == "1"
    done = 0

    def case(test, *args):
        nonlocal done
        print(test.__name__, *args, flush=True)
        test(L, *args)
        done += 1

    for dtype in T.TYPES:
        for kinds in T.KINDS + MORE_KINDS:
            for n, t, pad, shift in SHAPES:
                case(T.test_residual_norm, n, t, pad, shift, kinds, dtype)
        for n, t, kinds in RANGES:
            case(T.test_residual_norm_over_many_ranges, n, t, kinds, dtype)
    for dtype in ("f32", "bf16"):
        for n, t in ((72, 40), (1024, 9), (4096, 12), (8192, 5)):
            case(T.test_residual_norm_in_place, n, t, dtype)
    for n, t, gates in ((256, 4100, 2), (8192, 300, 300)):
        case(T.test_residual_norm_is_reproducible_and_reads_nothing_else, n, t, gates)
    case(T.test_residual_norm_not_finite_in_partly_filled_teams, 1000)
    print("cases passed:", done, flush=True)


@pytest.mark.gpu
def test_streamed_kernels():
    child = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], env={**os.environ, "LBN_STREAM_LOADS": "1"},
                           cwd=ROOT, text=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=110)
    assert child.returncode == 0, child.stdout[-4000:]
    assert child.stdout.splitlines()[-1] == f"cases passed: {3 * (11 * len(SHAPES) + len(RANGES)) + 11}", child.stdout[-2000:]


if __name__ == "__main__":
    sys.path.insert(0, ROOT)
    run()
