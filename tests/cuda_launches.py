"""Which kernels a call launches: their names, grids and clusters, read from
the nodes of a captured graph through the driver's API."""
from __future__ import annotations

import ctypes
from typing import Callable, NamedTuple

import torch


class Launch(NamedTuple):
    name: str  # mangled
    grid: int  # CTAs
    cluster: int  # CTAs of a cluster


class _KernelNode(ctypes.Structure):  # CUDA_KERNEL_NODE_PARAMS_v2
    _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3),
                ("shared", ctypes.c_uint), ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p),
                ("kernel", ctypes.c_void_p), ("context", ctypes.c_void_p)]


_KERNEL_NODE = 0  # CU_GRAPH_NODE_TYPE_KERNEL
_CLUSTER_DIMENSION = 4  # CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION


def launches(call: Callable[[], object]) -> list[Launch]:
    """The kernels of one call, which is captured and not run."""
    cuda = ctypes.CDLL("libcuda.so.1")

    def ask(name: str, *args) -> None:
        status = getattr(cuda, name)(*args)
        assert status == 0, f"{name}: {status}"

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        held = call()  # outputs live in the graph's memory
    raw = ctypes.c_void_p(graph.raw_cuda_graph())
    count = ctypes.c_size_t(0)
    ask("cuGraphGetNodes", raw, None, ctypes.byref(count))
    nodes = (ctypes.c_void_p * count.value)()
    ask("cuGraphGetNodes", raw, nodes, ctypes.byref(count))
    found = []
    for node in (ctypes.c_void_p(n) for n in nodes):
        kind = ctypes.c_int(-1)
        ask("cuGraphNodeGetType", node, ctypes.byref(kind))
        if kind.value != _KERNEL_NODE:
            continue
        at, name, value = _KernelNode(), ctypes.c_char_p(), (ctypes.c_uint * 16)()
        ask("cuGraphKernelNodeGetParams_v2", node, ctypes.byref(at))
        if at.func:
            ask("cuFuncGetName", ctypes.byref(name), ctypes.c_void_p(at.func))
        else:
            ask("cuKernelGetName", ctypes.byref(name), ctypes.c_void_p(at.kernel))
        ask("cuGraphKernelNodeGetAttribute", node, _CLUSTER_DIMENSION, value)
        found.append(Launch(name.value.decode(), at.grid[0] * at.grid[1] * at.grid[2],
                            max(1, value[0] * value[1] * value[2])))
    del held
    return found
