"""Which of the library's kernels a call launches: the call is captured into a graph and the graph's kernel nodes are named.
Tests of a kernel's special cases assert with it that the sizes they use still reach that kernel."""
import torch


def _ok(r):
    assert int(r[0]) == 0, r[0]
    return r[1:] if len(r) > 2 else r[1]


def launched(call):
    """mangled names of the kernels of `call` (which has run once before, so that nothing is set up during the capture)"""
    from cuda.bindings import driver

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    _, n = _ok(driver.cuGraphGetNodes(raw, 0))
    names = []
    for node in _ok(driver.cuGraphGetNodes(raw, n))[0]:
        if _ok(driver.cuGraphNodeGetType(node)) != driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        p = _ok(driver.cuGraphKernelNodeGetParams(node))
        name = _ok(driver.cuFuncGetName(p.func)) if int(p.func) else _ok(driver.cuKernelGetName(p.kern))
        names.append(name.decode())
    return names


def assert_launches(call, *kernels):
    """every one of `kernels` (parts of mangled names) is among what `call` launches"""
    names = launched(call)
    for k in kernels:
        assert any(k in n for n in names), f"{k} not among {names}"
