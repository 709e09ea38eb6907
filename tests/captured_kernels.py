"""What the driver says of the kernels that a call launches, read from a graph the call is captured in."""
import ctypes

import torch

LOCAL_BYTES, REGISTERS, MOST_DYNAMIC_SHARED = 3, 4, 8  # CU_FUNC_ATTRIBUTE_LOCAL_SIZE_BYTES, _NUM_REGS, _MAX_DYNAMIC_SHARED_SIZE_BYTES


class _KernelNode(ctypes.Structure):  # CUDA_KERNEL_NODE_PARAMS_v2
    _fields_ = [("func", ctypes.c_void_p)] + [(n, ctypes.c_uint) for n in ("gx", "gy", "gz", "bx", "by", "bz", "shared_bytes")] + \
        [(n, ctypes.c_void_p) for n in ("params", "extra", "kern", "ctx")]


class Kernel:
    def __init__(self, driver, func, shared_bytes):
        self._driver, self._func, self.shared_bytes = driver, func, shared_bytes

    def attribute(self, which):
        """As it is now, not as it was at the capture."""
        value = ctypes.c_int()
        assert self._driver.cuFuncGetAttribute(ctypes.byref(value), which, self._func) == 0
        return value.value


def captured_kernels(call):
    """The kernels of a call, in the order the driver lists them. The call runs once before; the graph is not replayed."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        kept = call()
    driver = ctypes.CDLL("libcuda.so.1")
    raw, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert driver.cuGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert driver.cuGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    kernels = []
    for node in nodes:
        kind = ctypes.c_int()
        assert driver.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value != 0:  # CU_GRAPH_NODE_TYPE_KERNEL
            continue
        p = _KernelNode()
        assert driver.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(p)) == 0
        func = ctypes.c_void_p(p.func)
        if not p.func:
            assert driver.cuKernelGetFunction(ctypes.byref(func), ctypes.c_void_p(p.kern)) == 0
        kernels.append(Kernel(driver, func, p.shared_bytes))
    del kept
    return kernels
