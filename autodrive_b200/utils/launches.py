"""Count of this library's own kernel launches issued from Python wrappers.

The Python entry points of the native kernels (tensor-core GEMM, fused
LayerNorm, GAE, fused Adam, peer all-reduce) add the number of kernels each
call launches; benchmarks read the count around a timed region. The operators
whose autograd is in C++ (RMS norm, 8-bit products, token log-probabilities)
count theirs in the extension. Simulator kernels are launched from C++ methods
and are counted by their callers.
"""
from __future__ import annotations

import sys

_COUNT = [0]


def add(n: int = 1) -> None:
    _COUNT[0] += n


def read() -> int:
    ext = sys.modules.get("autodrive_b200._C")
    return _COUNT[0] + (ext.native_launches() if ext is not None else 0)
