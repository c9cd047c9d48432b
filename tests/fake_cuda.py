"""Runs a function of a test module in a process of its own on the stand-in CUDA runtime (fake_cudart.cpp): the
library's host code without a GPU. Kernels do nothing there, and device memory is host memory."""

from __future__ import annotations

import ctypes
import os
import subprocess
import sys
from pathlib import Path

import numpy as np

HERE = Path(__file__).resolve().parent


def build(folder: Path) -> Path:
    """The stand-in runtime, compiled into `folder`."""
    out = folder / "libfake_cudart.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-I/usr/local/cuda/include",
                    str(HERE / "fake_cudart.cpp"), "-o", str(out)], check=True)
    return out


def run(fake: Path, module: str, function: str, *args):
    """Calls module.function(*args) (texts and numbers) there; its failure is the caller's."""
    code = f"import importlib; importlib.import_module({module!r}).{function}(*{args!r})"
    p = subprocess.run([sys.executable, "-c", code], cwd=HERE.parent, env=dict(os.environ, LD_PRELOAD=str(fake)),
                       capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stdout + p.stderr


class Runtime:
    """The test's side of the stand-in runtime, inside that process."""

    def __init__(self):
        self.lib = ctypes.CDLL(os.environ["LD_PRELOAD"])
        self.lib.fake_calls.restype = ctypes.c_size_t
        self.lib.fake_calls.argtypes = [ctypes.c_char_p, ctypes.c_size_t]
        self.lib.fake_fail.argtypes = [ctypes.c_char_p, ctypes.c_int]
        self.lib.cudaMalloc.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t]

    def fail(self, name: str, at: int):
        """The call `name` fails, after `at` of them that do not."""
        self.lib.fake_fail(name.encode(), at)

    def clear(self):
        self.lib.fake_clear()

    def in_flight(self) -> int:
        """Copies from pageable memory and memsets of the legacy stream that nothing has waited for."""
        return self.lib.fake_in_flight()

    def raced(self) -> int:
        """Work that was given to another stream meanwhile."""
        return self.lib.fake_raced()

    def calls(self) -> list[str]:
        """The calls since the last clear(); a launch as "launch" and the kernel's name."""
        buf = ctypes.create_string_buffer(1 << 20)
        n = self.lib.fake_calls(buf, len(buf))
        return buf.raw[:n].decode().split("\n")[:-1]

    def launches(self) -> list[str]:
        return [c for c in self.calls() if c.startswith("launch ")]

    def malloc(self, n: int) -> int:
        p = ctypes.c_void_p()
        assert self.lib.cudaMalloc(ctypes.byref(p), n) == 0
        return p.value


class Tensor:
    """A tensor of the stand-in device, as far as the operators' wrappers look at one."""

    def __init__(self, rt: Runtime, shape, dtype, strides=None):
        self.shape, self.dtype = tuple(shape), f"torch.{dtype}"
        dense = np.cumprod((1,) + self.shape[:0:-1])[::-1].tolist() if self.shape else []
        self.strides = tuple(strides) if strides is not None else tuple(int(x) for x in dense)
        self.dense = self.strides == tuple(dense)
        size = np.dtype("uint8" if dtype == "bool" else dtype.replace("bfloat16", "float16")).itemsize
        last = sum((n - 1) * s for n, s in zip(self.shape, self.strides)) + 1
        self.p = rt.malloc(max(1, last) * size)

    def data_ptr(self):
        return self.p

    def stride(self, i=None):
        return self.strides if i is None else self.strides[i]

    def dim(self):
        return len(self.shape)

    def numel(self):
        return int(np.prod(self.shape))

    def is_contiguous(self):
        return self.dense
