"""CPU tier: the GPU tests of the model operators, run against hccl_amd/csrc/model_ops built for the host.

tests/emu/build_model_ops.py compiles entry points and kernels against a stand-in HIP runtime in which every lane is a fiber
(tests/emu/lanes): cross-lane operations have their meaning, and stop the process if lanes of a wavefront meet at different
ones; between two barriers the wavefronts run one after the other, in an order that keeps changing, so that a missing barrier
shows in the results; LDS starts with anything.  AddressSanitizer and the undefined-behaviour checks watch every access, to
global memory and to LDS.  It says nothing about timing or about what the GPU compiler makes of the code."""
import glob
import os
import subprocess
import sys

from test_emulated_kernels import ROOT, emu_env
import build_model_ops

# Left out: streams and graphs, and what is larger than 32 bits of elements.
DESELECT = ["test_calls_can_be_captured_into_a_graph_and_replayed", "test_logits_beyond_32_bits_of_elements",
            "test_tensors_beyond_32_bits_of_elements", "test_more_rows_than_a_launch_of_the_gradient_takes"]


def environment(log):
    base, lib = build_model_ops.build()
    env = emu_env(base, log)
    env["ASAN_OPTIONS"] += ":detect_stack_use_after_return=0"      # would map and unmap a stack of its own for every lane
    env["HCCL_AMD_TEST_EMU_MODEL_OPS_LIB"] = lib
    env["PYTHONPATH"] = os.pathsep.join([ROOT, os.path.join(ROOT, "tests"), os.path.join(ROOT, "tests", "emu"),
                                         env.get("PYTHONPATH", "")])
    return env


def reports(log):
    return "".join(open(f).read()[:3000] for f in sorted(glob.glob(log + "*"))[:2])


def test_gpu_tests_pass_on_the_emulation_and_touch_no_byte_outside_their_buffers(tmp_path):
    log = str(tmp_path / "asan")
    cmd = [sys.executable, "-m", "pytest", "-m", "gpu", "-q", "-x", "-p", "no:cacheprovider", "-p", "host_tensors", "-n",
           str(max(2, min(8, os.cpu_count() or 2))), "--timeout", "900", "tests/test_gpu_model_ops.py"]
    for name in DESELECT:
        cmd += ["--deselect", "tests/test_gpu_model_ops.py::" + name]
    proc = subprocess.run(cmd, cwd=ROOT, env=environment(log), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert proc.returncode == 0 and not reports(log), proc.stdout[-6000:] + reports(log)


OVERRUN = """
import torch, host_tensors
host_tensors.pytest_configure(None)
import hccl_amd
from hccl_amd import HcclDataType as DT, model_ops
comm = hccl_amd.comm_init_all(1)[0]
x = torch.zeros(2 * 1000 - %d)
out = torch.zeros(2)
model_ops.token_log_probs(comm, x, 2, 0, 1000, torch.zeros(2, dtype=torch.int64), out, data_type=DT.FP32, row_stride=1000,
                          stream=host_tensors.Stream())
print("result", out.tolist())
"""


def test_the_run_does_catch_a_kernel_that_leaves_its_buffer(tmp_path):
    """The check checks: rows in memory that is one element too short end the process with a report, others do not."""
    for short in (0, 1):
        log = str(tmp_path / ("asan%d" % short))
        boot = ("import ctypes, os, hccl_amd; hccl_amd._lib = hccl_amd._bind(ctypes.CDLL(os.environ['HCCL_AMD_TEST_EMU_LIB']))")
        proc = subprocess.run([sys.executable, "-c", boot + OVERRUN % short], cwd=ROOT, env=environment(log),
                              stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        if short:
            assert proc.returncode != 0 and "result" not in proc.stdout, proc.stdout[-2000:]
            assert "heap-buffer-overflow" in reports(log), reports(log)
        else:
            assert proc.returncode == 0 and "result" in proc.stdout and not reports(log), proc.stdout[-2000:] + reports(log)
