"""Which kernels a call launches, for tests that are about one of several: the call is
captured into a graph, whose nodes name their kernels and grids."""

import re
import warnings

NODE = re.compile(r"topoId: (\d+)\) \| (\w+)\\<\\<\\<(?:\\\{)?([\d,]+)(?:\\\})?,(\d+),")


def launched(call, tmp_path):
    """[(mangled name, grid, threads)] of the kernels of call(), in their order."""
    import torch

    call()  # whatever a first call sets up
    torch.cuda.synchronize()
    graph, path = torch.cuda.CUDAGraph(keep_graph=True), tmp_path / "graph.dot"
    graph.enable_debug_mode()
    with torch.cuda.graph(graph):
        call()
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")  # the dump announces itself
        graph.debug_dump(str(path))
    nodes = sorted(NODE.findall(path.read_text()), key=lambda n: -int(n[0]))
    assert nodes, "no kernel in the graph"
    return [(name, tuple(int(x) for x in grid.split(",")), int(threads)) for _, name, grid, threads in nodes]
