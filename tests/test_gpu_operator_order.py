"""The decoder's operators in an order that streams, events and captured branches set: their kernels are set up under the
end of the kernel before them (programmatic launch), and wait for everything that the stream waits for."""
import pytest
import torch

from sparsesam_b200 import ops

pytestmark = pytest.mark.gpu


def inputs(dev):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(dev, torch.bfloat16)  # noqa: E731
    return {"image": r(8, 4096, 8, 16), "tokens": r(8, 9, 8, 16), "maps": r(8, 96 * 96, 64), "w": r(64), "b": r(64)}


def work(t, other, sync):
    """A chain on two streams with a dependence at every step: `other` runs its function on the second stream, between
    two events; sync is called after every step."""
    t = dict(t)
    out = []
    for _ in range(4):
        x = ops.cross_attn(t["tokens"], t["image"], t["image"])
        sync()
        y = other(lambda x=x: ops.cross_attn(t["image"], x, x))
        sync()
        m = other(lambda: ops.groupnorm_act(t["maps"], 8, t["w"], t["b"], 1e-5, "gelu"))
        sync()
        z = ops.cross_attn(x, y, y)
        sync()
        buf = torch.empty_like(m)
        buf.copy_(m)                          # a copy between two kernels
        n = ops.layernorm_gelu_half(buf, t["w"], t["b"], 1e-6, True)
        sync()
        big = torch.zeros_like(y)             # a fill before one
        y = ops.cross_attn(big, z, z)
        sync()
        t["tokens"], t["image"], t["maps"] = z, y, n
        out += [x, y, z, n]
    return out


@pytest.mark.parametrize("captured", [False, True])
def test_two_streams_that_wait_for_one_another(cuda_device, captured):
    t = inputs(cuda_device)
    expect = [x.clone() for x in work(t, lambda f: f(), torch.cuda.synchronize)]
    torch.cuda.synchronize()
    main, side = torch.cuda.Stream(cuda_device), torch.cuda.Stream(cuda_device)
    held = []

    def other(f):
        side.wait_stream(main)
        with torch.cuda.stream(side):
            y = f()
        main.wait_stream(side)
        held.append(y)                        # its memory belongs to the other stream
        return y

    main.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(main):
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=main):
                got = work(t, other, lambda: None)
            for _ in range(3):
                graph.replay()
        else:
            for _ in range(3):
                got = work(t, other, lambda: None)
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(zip(expect, got)):
        assert torch.equal(x, y), i
