"""ingot_amd — MI355X (gfx950) backend for ingot's dense-contraction hot path.

The product is the C-ABI library ``libingot_rocm.so`` (include/ingot_rocm.h):
hand-written HIP kernels for Gemm / MatMul with fused epilogues, the bf16
GEMM and decode GEMV, and int8 MatMulInteger + DequantizeLinear, behind the
reference's op interface, and the operators between a decoder layer's
projections (rotary positions, attention of drafted tokens over a paged cache,
the operations on its pages). This package holds its sources (``csrc/``), its
build (``build.py``) and a thin Python host wrapper (``host.py``) over the
C ABI for tests and benchmarks.
"""
from ._lib import IngotError, load  # noqa: F401
from .host import DeviceTensor, Graph, Heads, KvCache, KvTable, Op, Session, Weight  # noqa: F401

__all__ = ["IngotError", "load", "Session", "Weight", "DeviceTensor", "Op", "Graph",
           "Heads", "KvCache", "KvTable"]
