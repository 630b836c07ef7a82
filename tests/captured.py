"""The kernels that calls launch, read from a capture of them: nothing runs."""
import ctypes as C
import re

import torch


def kernels_of(ops, path, calls):
    """Names of the kernels that calls() launches on a stream of its own, one behind the other; `path`: a file for the graph's text."""
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph(keep_graph=True)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ops.stream(stream.cuda_stream)
        try:
            calls()
        finally:
            ops.stream()
    assert C.CDLL("libcuda.so.1").cuGraphDebugDotPrint(C.c_void_p(graph.raw_cuda_graph()), str(path).encode(), 1) == 0
    found = re.findall(r"\{ID \| (\d+) \(topoId: \d+\) \| (\w+)", path.read_text())
    return [name for _, name in sorted(found, key=lambda f: int(f[0]))]
