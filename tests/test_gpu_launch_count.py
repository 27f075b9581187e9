"""The launch count of the decoder's operators against the kernel nodes of a captured call."""
import pytest
import torch

from sparsesam_b200 import _lib, ops

cudart = pytest.importorskip("cuda.bindings.runtime")
pytestmark = pytest.mark.gpu


def captured(f, device):
    """(kernels in the graph of f, launches counted while it was captured)"""
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        f()
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        n0 = _lib.launch_count
        with torch.cuda.graph(graph, stream=side):
            f()
        counted = _lib.launch_count - n0
    err, _, n = cudart.cudaGraphGetNodes(graph.raw_cuda_graph())
    assert not int(err)
    err, nodes, n = cudart.cudaGraphGetNodes(graph.raw_cuda_graph(), n)
    kinds = [cudart.cudaGraphNodeGetType(x)[1] for x in nodes[:n]]
    return sum(k == cudart.cudaGraphNodeType.cudaGraphNodeTypeKernel for k in kinds), counted


def training(f, *shapes, dtype, device):
    g = torch.Generator().manual_seed(0)
    leaves = [torch.randn(s, generator=g).to(device, dtype).requires_grad_(True) for s in shapes]
    dout = torch.randn(shapes[0], generator=g).to(device, dtype)
    return lambda: torch.autograd.grad(f(*leaves), leaves, dout)


@pytest.mark.parametrize("name", ["layernorm", "groupnorm_resident", "groupnorm_streamed", "groupnorm_batches", "few_keys",
                                  "few_rows", "long", "fp32"])
def test_count_is_the_kernels(cuda_device, name):
    half, dev = torch.bfloat16, cuda_device
    gn = lambda x, w, b: ops.groupnorm_act(x, 8, w, b, 1e-5, "gelu")  # noqa: E731
    q = lambda n: (2, n, 4, 32)  # noqa: E731
    f = {"layernorm": lambda: training(lambda x, w, b: ops.layernorm_gelu_half(x, w, b, 1e-6, True), (500, 64), (64,), (64,),
                                       dtype=half, device=dev),
         "groupnorm_resident": lambda: training(gn, (2, 100, 64), (64,), (64,), dtype=half, device=dev),
         "groupnorm_streamed": lambda: training(gn, (2, 200 * 200, 64), (64,), (64,), dtype=half, device=dev),
         "groupnorm_batches": lambda: training(gn, (5, 132 * 136, 512), (512,), (512,), dtype=half, device=dev),
         "few_keys": lambda: training(ops.cross_attn, q(300), q(9), q(9), dtype=half, device=dev),
         "few_rows": lambda: training(ops.cross_attn, q(9), q(300), q(300), dtype=half, device=dev),
         "long": lambda: training(ops.cross_attn, q(200), q(300), q(300), dtype=half, device=dev),
         "fp32": lambda: training(ops.cross_attn, q(20), q(30), q(30), dtype=torch.float32, device=dev)}[name]()
    nodes, counted = captured(f, dev)
    assert nodes == counted > 1


def test_calls_that_launch_nothing_count_nothing(cuda_device):
    x = torch.zeros(0, 4, 2, 16, dtype=torch.float16, device=cuda_device)
    n0 = _lib.launch_count
    ops.cross_attn(x, x, x)
    ops.layernorm_gelu_half(torch.zeros(0, 32, dtype=torch.float16, device=cuda_device), *[torch.ones(
        32, dtype=torch.float16, device=cuda_device)] * 2, 1e-6, True)
    assert _lib.launch_count == n0
