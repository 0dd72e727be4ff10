"""A pytest plugin for the emulation run of the model operators' GPU tests (tests/test_emulated_model_ops.py): tensors "on the
GPU" are host tensors, and the Python mirror calls the emulation library.  Only that test process loads it."""
import ctypes
import os

import torch
from torch.overrides import TorchFunctionMode


class HostTensors(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        kwargs = dict(kwargs or {})
        if func is torch.Tensor.cuda:
            return args[0].clone()
        if str(kwargs.get("device")).startswith("cuda"):
            kwargs["device"] = "cpu"
        return func(*args, **kwargs)


class Stream:
    """Every launch runs to completion: any handle but null is as good as another."""

    cuda_stream = 0x1000

    def synchronize(self):
        pass


def pytest_configure(config):
    from hccl_amd import model_ops
    model_ops._lib = model_ops._bind(ctypes.CDLL(os.environ["HCCL_AMD_TEST_EMU_MODEL_OPS_LIB"]))
    torch.cuda.synchronize = lambda *a: None
    torch.cuda.empty_cache = lambda: None
    torch.cuda.Stream = Stream
    torch.set_num_threads(1)
    HostTensors().__enter__()
