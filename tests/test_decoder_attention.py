"""hq.DecoderAttention where torch computes its attention (the host, dtypes and heads that the kernel does not take)."""
import copy
import math

import pytest
import torch

from sparsesam_b200 import _lib, hq

gpu = pytest.mark.gpu
LENS = torch.tensor([25, 0, 7], dtype=torch.int32)


def attention(device="cpu", dtype=torch.float32, dim=64, heads=4):
    torch.manual_seed(0)
    mod = hq.DecoderAttention(dim, heads, 2).to(device, dtype)
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(device, dtype)  # noqa: E731
    return mod, r(3, 9, dim), r(3, 25, dim), r(3, 25, dim)


def near(x, y, dtype=torch.float32):
    """Two ways of computing some five rounded layers of unit size."""
    eps = torch.finfo(dtype).eps
    assert x.shape == y.shape and (x.double() - y.double()).abs().max() <= 16 * eps * max(1.0, y.abs().max().item())


def test_masked_places_hold_anything_on_torchs_path():
    """What the kernel promises holds elsewhere too: absent keys and queries without keys may be NaN or infinite."""
    mod, q, k, v = attention()
    gone = torch.arange(25)[None] >= LENS[:, None]
    want = mod(q, torch.where(gone[..., None], 0.0, k), torch.where(gone[..., None], 0.0, v), key_lens=LENS)
    k, v, q = k.clone(), v.clone(), q.clone()
    k[gone], v[gone], q[1] = math.nan, math.inf, math.nan
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = mod(*leaves, key_lens=LENS)
    near(out, want)
    near(out[1], mod.out_proj.bias.expand(9, -1))
    for t, there in zip(torch.autograd.grad(out.square().sum(), leaves), (torch.tensor([True, False, True]), ~gone, ~gone)):
        assert torch.isfinite(t[there]).all() and not t[~there].any()


@gpu
def test_masked_places_hold_anything_where_torch_computes(cuda_device):
    """Heads of 12 channels, which the kernel does not take."""
    mod, q, k, v = attention(cuda_device, dim=96, heads=4)
    lens = LENS.to(cuda_device)
    gone = torch.arange(25, device=cuda_device)[None] >= lens[:, None]
    want = copy.deepcopy(mod).cpu()(q.cpu(), k.cpu(), v.cpu(), key_lens=LENS)
    k[gone], v[gone], q[1] = math.nan, math.inf, math.nan
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = mod(*leaves, key_lens=lens)
    near(out.cpu(), want)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(out.square().sum(), leaves))


def test_one_query_set_for_a_batch():
    mod, q, k, v = attention()
    near(mod(q[:1], k, v), mod(q[:1].expand(3, -1, -1), k, v))


@gpu
def test_one_query_set_for_a_batch_on_the_gpu(cuda_device):
    mod, q, k, v = attention(cuda_device)
    near(mod(q[:1], k, v), mod(q[:1].expand(3, -1, -1), k, v))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tq,tk,dim,kernel", [(8, 4096, 128, True), (4096, 8, 128, True), (64, 64, 256, False), (9, 9, 256, True),
                                              (1000, 1000, 512, False)])
def test_sizes_go_where_they_are_faster(cuda_device, tq, tk, dim, kernel, dtype):
    """Sizes that torch's attention took less time for before the kernels came still go there, unless there is a mask."""
    torch.manual_seed(4)
    mod = hq.DecoderAttention(dim, 8).to(cuda_device, dtype)
    q, k = torch.randn(16, tq, dim, device=cuda_device, dtype=dtype), torch.randn(16, tk, dim, device=cuda_device, dtype=dtype)
    lens = torch.full((16,), tk, dtype=torch.int32, device=cuda_device)
    with torch.no_grad():
        n0 = _lib.launch_count
        plain = mod(q, k, k)
        assert (_lib.launch_count > n0) == kernel
        n0 = _lib.launch_count
        near(mod(q, k, k, key_lens=lens), plain, dtype)
        assert _lib.launch_count > n0


@gpu
@pytest.mark.parametrize("kind", ["plain", "lens", "mask"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_more_prompts_than_one_call_takes(cuda_device, dtype, kind):
    """65,537 prompts, which torch's attention refuses in half precision: the rows and gradients of two calls."""
    torch.manual_seed(5)
    mod = hq.DecoderAttention(16, 2).to(cuda_device, dtype)
    n, most = 65537, 40000
    x, y = torch.randn(n, 2, 16, device=cuda_device).to(dtype), torch.randn(n, 5, 16, device=cuda_device).to(dtype)
    kw = {}
    if kind == "lens":
        kw["key_lens"] = torch.randint(0, 6, (n,), device=cuda_device, dtype=torch.int32)
    if kind == "mask":
        kw["key_mask"] = torch.rand(n, 5, device=cuda_device) < 0.5

    def run(at):
        a, b = x[at].clone().requires_grad_(True), y[at].clone().requires_grad_(True)
        out = mod(a, b, b, **{k: t[at] for k, t in kw.items()})
        return [out.detach(), *torch.autograd.grad(out.float().square().sum(), (a, b))]

    whole = run(slice(0, n))
    parts = [torch.cat(t) for t in zip(run(slice(0, most)), run(slice(most, n)))]
    # the attention's rows are the same; the projections' matrix products may be cut differently
    for w, p in zip(whole, parts):
        assert (w.double() - p.double()).abs().max() <= 8 * torch.finfo(dtype).eps * p.abs().max()
