"""ops.groupnorm_act and the gradients of ops.layernorm_gelu_half against their definitions in 64 bits.

Tolerances. Every kernel computes in fp32 and rounds once: half a step (u = eps / 2 of the type) of
the value, plus fp32 noise. The normalised value t = (x - mu) rstd carries a handful of roundings of
t and the errors of mu (2^-24 of its size, a few pairwise merges) and of rstd; z = t w + b one more;
the activations' slopes are below 1.13. 32 * 2^-24 of (|t w| + |b| + |mu| rstd |w|) covers them; the
LayerNorm's GELU adds its formula's 1.5e-7 |x|. Gradients: each group mean is a sum over n values of
random sign, whose rounding stays below 2^-24 * 64 of the mean magnitude (partial sums of at most a
few hundred terms per thread, then pairwise), likewise dw and db relative to the sum of magnitudes.
"""
import math

import pytest
import torch

from sparsesam_b200 import hq, ops

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS24 = 2.0 ** -24


def act_and_slope(z, act):
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "gelu":
        phi = torch.special.ndtr(z)
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    return z, torch.ones_like(z)


def reference(x, groups, w, b, eps, act, dout):
    """[(value, what its fp32 roundings scale with)] of out, dx, dw, db for x (N, ..., C), in 64 bits."""
    shape = x.shape
    N, C = shape[0], shape[-1]
    cg = C // groups
    x4 = x.double().reshape(N, -1, groups, cg)
    wd, bd = w.double().view(groups, cg), b.double().view(groups, cg)
    mean = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    mu = mean(x4)
    rstd = 1 / torch.sqrt(mean((x4 - mu) ** 2) + eps)
    t = (x4 - mu) * rstd
    z = t * wd + bd
    y, slope = act_and_slope(z, act)
    zsize = (t * wd).abs() + bd.abs() + (mu.abs() * rstd * wd.abs()) + y.abs()
    d = dout.double().reshape(x4.shape)
    g = d * slope
    # the slope's own error: it changes by at most 1.13 (GELU's second derivative) per unit of z
    gsize = d.abs() * (slope.abs() + (zsize if act in ("gelu", "silu") else 0.0))
    tsize = t.abs() + mu.abs() * rstd
    h = g * wd
    dx = rstd * (h - mean(h) - t * mean(h * t))
    hs = gsize * wd.abs()
    dxs = rstd * (hs + mean(hs) + tsize * mean(hs * tsize) * 2)
    return [(y.reshape(shape), zsize.reshape(shape)), (dx.reshape(shape), dxs.reshape(shape)),
            ((g * t).sum((0, 1)).reshape(C), (gsize * tsize).sum((0, 1)).reshape(C)),
            (g.sum((0, 1)).reshape(C), gsize.sum((0, 1)).reshape(C))]


def check(got, ref, dtype, extra=0.0, skip=None):
    u = torch.finfo(DTYPES[dtype]).eps / 2
    tiny = torch.finfo(DTYPES[dtype]).tiny * u * 8
    for i, (name, y, (r, size)) in enumerate(zip(("out", "dx", "dw", "db"), got, ref)):
        assert y.dtype == DTYPES[dtype] and y.shape == r.shape, name
        allow = u * r.abs() + ((32 if i == 0 else 96) * EPS24 + extra) * size + tiny
        over = (y.double() - r).abs() - allow
        if skip is not None and i < 2:
            over = over[~skip]
        assert over.max().item() <= 0, f"{name}: {over.max().item():.3e} past its bound"


def make(dev, shape, dtype, seed=0, shift=0.5, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    dt, C = DTYPES[dtype], shape[-1]
    x = (torch.randn(*shape, generator=g) * scale + shift).to(dt).to(dev)
    w = (torch.randn(C, generator=g) * 0.3 + 1).to(dt).to(dev)
    b = (torch.randn(C, generator=g) * 0.3).to(dt).to(dev)
    return x, w, b, torch.randn(*shape, generator=g).to(dt).to(dev)


def run(fn, x, w, b, dout):
    x, w, b = (t.detach().requires_grad_(True) for t in (x, w, b))
    out = fn(x, w, b)
    return [out.detach(), *torch.autograd.grad(out, (x, w, b), dout)]


def off_border(x, groups, w, b, eps):
    """Where ReLU's input is so near zero that its sign is the rounding's."""
    (z, size), *_ = reference(x, groups, w, b, eps, "none", torch.zeros_like(x))
    return z.abs() <= 32 * EPS24 * size


GN = [((1, 64, 64, 256), 8), ((2, 7, 9, 32), 32), ((3, 67, 45, 96), 4), ((1, 1, 1, 8), 1), ((5, 1, 3, 16), 4),
      ((2, 200, 200, 64), 8), ((1, 16, 2000, 24), 3), ((33, 5, 40), 5), ((2, 300, 512), 1), ((1, 50, 1024), 16),
      ((40, 9, 72), 12)]


@pytest.mark.parametrize("act", list(ops.ACTIVATIONS))
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape,groups", GN, ids=lambda s: str(s).replace(" ", ""))
def test_groupnorm(cuda_device, shape, groups, dtype, act):
    x, w, b, do = make(cuda_device, shape, dtype)
    got = run(lambda x, w, b: ops.groupnorm_act(x, groups, w, b, 1e-5, act), x, w, b, do)
    skip = off_border(x, groups, w, b, 1e-5) if act == "relu" else None
    ref = reference(x, groups, w, b, 1e-5, act, do)
    if skip is not None and skip.any():      # those elements' share of the sums is the rounding's too
        ref[2] = (ref[2][0], ref[2][1] * 2.0 ** 20)
        ref[3] = (ref[3][0], ref[3][1] * 2.0 ** 20)
    check(got, ref, dtype, skip=skip)
    assert torch.equal(ops.groupnorm_act(x, groups, w, b, 1e-5, act), got[0])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_groupnorm_far_mean_and_outlier(cuda_device, dtype):
    """A mean hundreds of deviations from zero, and a first pixel thousands of deviations out."""
    x, w, b, do = make(cuda_device, (2, 128, 128, 32), dtype, shift=300.0, scale=1.0)
    check(run(lambda x, w, b: ops.groupnorm_act(x, 4, w, b, 1e-5, "none"), x, w, b, do),
          reference(x, 4, w, b, 1e-5, "none", do), dtype)
    x, w, b, do = make(cuda_device, (2, 128, 128, 32), dtype)
    x[:, 0, 0] = 5000.0
    check(run(lambda x, w, b: ops.groupnorm_act(x, 4, w, b, 1e-5, "silu"), x, w, b, do),
          reference(x, 4, w, b, 1e-5, "silu", do), dtype)


def test_groupnorm_special_values(cuda_device):
    """A constant map gives act(b); a NaN stays inside its sample and group."""
    for act in ops.ACTIVATIONS:
        x, w, b, _ = make(cuda_device, (2, 5, 6, 16), "fp32")
        y = ops.groupnorm_act(torch.full_like(x, 7.0), 4, w, b, 1e-5, act)
        want = act_and_slope(b.double(), act)[0].expand_as(y)
        assert (y.double() - want).abs().max() < 1e-6
        x[1, 2, 3, 5] = math.nan
        y = ops.groupnorm_act(x, 4, w, b, 1e-5, act)
        bad = torch.zeros_like(x, dtype=torch.bool)
        bad[1, ..., 4:8] = True
        assert torch.equal(torch.isnan(y), bad)


def test_groupnorm_equal_bits_and_graph(cuda_device):
    x, w, b, do = make(cuda_device, (3, 40, 50, 64), "bf16")
    f = lambda x, w, b: ops.groupnorm_act(x, 8, w, b, 1e-5, "gelu")  # noqa: E731
    want = run(f, x, w, b, do)
    assert all(torch.equal(p, q) for p, q in zip(want, run(f, x, w, b, do)))
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        f(*leaves)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = f(*leaves)
            grads = torch.autograd.grad(y, leaves, do)
            y = y.detach()
    torch.cuda.current_stream().wait_stream(side)
    x2 = make(cuda_device, (3, 40, 50, 64), "bf16", seed=8)[0]
    with torch.no_grad():
        leaves[0].copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip([y, *grads], run(f, x2, w, b, do)))


def test_groupnorm_gradient_layouts(cuda_device):
    """A gradient that arrives in another memory order, or one scalar spread over all."""
    x, w, b, do = make(cuda_device, (2, 9, 10, 32), "fp16")
    f = lambda x, w, b: ops.groupnorm_act(x, 4, w, b, 1e-5, "relu")  # noqa: E731
    want = run(f, x, w, b, do)
    turned = do.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    assert all(torch.equal(p, q) for p, q in zip(want, run(f, x, w, b, turned)))
    one = torch.ones((), dtype=torch.float16, device=cuda_device).expand(x.shape)
    assert all(torch.equal(p, q) for p, q in zip(run(f, x, w, b, torch.ones_like(x)), run(f, x, w, b, one)))


def test_groupnorm_empty(cuda_device):
    x, w, b, do = make(cuda_device, (0, 5, 16), "fp32")
    got = run(lambda x, w, b: ops.groupnorm_act(x, 2, w, b), x, w, b, do)
    assert got[0].shape == (0, 5, 16) and not got[2].any() and not got[3].any()


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,C", [(1, 32), (4096, 256), (777, 64), (100003, 128), (5, 256), (33000, 32)])
def test_layernorm_gradients(cuda_device, rows, C, dtype, gelu):
    x, w, b, do = make(cuda_device, (rows, C), dtype)
    got = run(lambda x, w, b: ops.layernorm_gelu_half(x, w, b, 1e-6, gelu), x, w, b, do)
    ref = reference(x.view(rows, 1, C), 1, w, b, 1e-6, "gelu" if gelu else "none", do.view(rows, 1, C))
    ref[:2] = [(r.view(rows, C), s.view(rows, C)) for r, s in ref[:2]]
    check(got, ref, dtype, extra=2e-7)       # the forward's GELU formula, see the module text
    with torch.no_grad():                    # the forward is the same kernel with and without gradients
        assert torch.equal(got[0], ops.layernorm_gelu_half(x, w, b, 1e-6, gelu))
    again = run(lambda x, w, b: ops.layernorm_gelu_half(x, w, b, 1e-6, gelu), x, w, b, do)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


def test_layernorm_gradient_reaches_the_decoder_norms(cuda_device):
    """hq.LayerNorm2d and hq.RowLayerNorm in half precision pass their gradients on."""
    for mod, shape in ((hq.LayerNorm2d(64, gelu=True), (2, 64, 8, 8)), (hq.RowLayerNorm(64), (2, 30, 64))):
        mod = mod.to(cuda_device, torch.bfloat16)
        x = torch.randn(*shape, device=cuda_device, dtype=torch.bfloat16)
        if x.dim() == 4:
            x = x.to(memory_format=torch.channels_last)
        x.requires_grad_(True)
        mod(x).float().square().sum().backward()
        for t in (x, mod.weight, mod.bias):
            assert t.grad is not None and t.grad.abs().sum() > 0


def test_layernorm_without_channels(cuda_device):
    x = torch.zeros(3, 0, dtype=torch.float16, device=cuda_device, requires_grad=True)
    w = torch.zeros(0, dtype=torch.float16, device=cuda_device)
    out = ops.layernorm_gelu_half(x, w, w, 1e-6, False)
    assert out.shape == (3, 0)
    out.sum().backward()
    assert x.grad.shape == (3, 0)
