"""Which kernels a call launches, from the nodes of a graph that it was captured into."""


def kernel_names(call):
    """Names (mangled) of the kernels that `call` launches, in no particular order; the call runs once before the capture."""
    import torch
    from cuda.bindings import driver

    def done(answer):
        assert int(answer[0]) == 0, answer[0]
        return answer[1:]
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        keep = call()
    handle = driver.CUgraph(graph.raw_cuda_graph())
    count = done(driver.cuGraphGetNodes(handle, 0))[-1]
    names = []
    for node in done(driver.cuGraphGetNodes(handle, count))[0]:
        if done(driver.cuGraphNodeGetType(node))[0] != driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        params = done(driver.cuGraphKernelNodeGetParams(node))[0]
        name = done(driver.cuFuncGetName(params.func))[0] if int(params.func) else done(driver.cuKernelGetName(params.kern))[0]
        names.append(name.decode())
    del keep
    return names
