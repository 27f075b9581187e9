"""ops.cross_attn against its definition in 64 bits: lengths, heads, masks, strides, gradients.

Tolerances. A half result is the fp32 result rounded once (half a step, u = eps / 2 of the
type) plus what the kernel's own arithmetic adds: products of half inputs are exact in fp32,
probabilities and their gradients enter the second product as two half terms (2 u^2 of their
value), so an element is off by at most u |o| + 4 u^2 sum_j p_j |v_j| + fp32 noise. fp32
kernels: logits carry D roundings, exp2 an absolute logit error of (|s| + D) 2^-24 in the
exponent (|s| < 30 for these inputs, D <= 128), and each sum over n terms at most
log2-many-to-n roundings of random sign: 2^-24 (30 + 2 sqrt(D) + 2 sqrt(n)) < 2^-24 * 256
for n <= 4096 of the sum of the terms' magnitudes.
"""
import math

import pytest
import torch

from sparsesam_b200 import _lib, ops

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
NOISE = 256 * 2.0 ** -24


def make(dev, B, Tq, Tk, H, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    r = lambda *s: torch.randn(*s, generator=g).to(dt).to(dev)  # noqa: E731
    return r(B, Tq, H, D), r(B, Tk, Hk, D), r(B, Tk, Hk, D), r(B, Tq, H, D)


def there(B, Tk, lens, mask, dev):
    ok = torch.ones(B, Tk, dtype=torch.bool, device=dev)
    if lens is not None:
        ok &= torch.arange(Tk, device=dev)[None] < lens[:, None]
    if mask is not None:
        ok &= mask
    return ok


def reference(q, k, v, dout=None, scale=None, lens=None, mask=None):
    """[(value, sum of the last product's magnitudes)] of out (, dq, dk, dv) in 64 bits."""
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    G = H // Hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    ok = there(B, Tk, lens, mask, q.device)
    clean = lambda t: torch.where(ok[:, :, None, None], t.double(), 0.0)  # noqa: E731
    spread = lambda t: t.repeat_interleave(G, dim=2)  # noqa: E731
    qd, kd, vd = q.double(), spread(clean(k)), spread(clean(v))
    s = torch.einsum("bqhd,bkhd->bhqk", qd, kd) * scale
    s = s.masked_fill(~ok[:, None, None, :], -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    res = [(torch.einsum("bhqk,bkhd->bqhd", p, vd), torch.einsum("bhqk,bkhd->bqhd", p, vd.abs()))]
    if dout is None:
        return res
    do = dout.double()
    dp = torch.einsum("bqhd,bkhd->bhqk", do, vd)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    # dS itself is a difference of magnitude p (sum |do v| + its mean): what its roundings scale with
    dpa = torch.einsum("bqhd,bkhd->bhqk", do.abs(), vd.abs())
    dsa = p * (dpa + (p * dpa).sum(-1, keepdim=True)) * scale
    fold = lambda t: t.unflatten(2, (Hk, G)).sum(3)  # noqa: E731
    res.append((torch.einsum("bhqk,bkhd->bqhd", ds, kd), torch.einsum("bhqk,bkhd->bqhd", dsa, kd.abs())))
    res.append((fold(torch.einsum("bhqk,bqhd->bkhd", ds, qd)), fold(torch.einsum("bhqk,bqhd->bkhd", dsa, qd.abs()))))
    res.append((fold(torch.einsum("bhqk,bqhd->bkhd", p, do)), fold(torch.einsum("bhqk,bqhd->bkhd", p, do.abs()))))
    return res


def check(got, ref, dtype):
    u = torch.finfo(DTYPES[dtype]).eps / 2
    tiny = torch.finfo(DTYPES[dtype]).tiny * u * 2       # half a step of the subnormals, and a margin of four
    for name, y, (r, size) in zip(("out", "dq", "dk", "dv"), got, ref):
        assert y.dtype == DTYPES[dtype] and y.shape == r.shape
        allow = u * r.abs() + (NOISE + (4 * u * u if dtype != "fp32" else 0.0)) * size + 4 * tiny
        over = ((y.double() - r).abs() - allow).max().item()
        assert over <= 0, f"{name}: {over:.3e} past its bound, worst error {(y.double() - r).abs().max().item():.3e}"


def run(q, k, v, dout=None, **kw):
    if dout is None:
        return [ops.cross_attn(q, k, v, **kw)]
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = ops.cross_attn(q, k, v, **kw)
    return [out.detach(), *torch.autograd.grad(out, (q, k, v), dout)]


SHAPES = [  # B, Tq, Tk, H, Hk, D
    (1, 1, 1, 1, 1, 16), (2, 1, 7, 2, 2, 16), (1, 8, 4096, 8, 8, 16), (3, 5, 65, 4, 2, 32), (2, 17, 1, 2, 2, 32),
    (2, 129, 9, 8, 8, 16), (1, 300, 64, 2, 1, 64), (2, 65, 130, 6, 2, 64), (1, 33, 257, 2, 2, 128),
    (2, 16, 16, 1, 1, 8), (1, 40, 100, 3, 1, 24), (1, 7, 515, 2, 2, 40), (2, 70, 31, 2, 2, 80), (1, 1, 3000, 4, 1, 32),
    (2, 1000, 3, 2, 2, 16), (1, 50, 70, 2, 2, 112), (2, 150, 200, 2, 2, 40), (1, 300, 260, 4, 2, 64), (1, 129, 1030, 1, 1, 56),
    (8, 128, 128, 8, 8, 64), (1, 1000, 65, 2, 1, 64),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients(cuda_device, shape, dtype):
    q, k, v, do = make(cuda_device, *shape, dtype)
    check(run(q, k, v, do), reference(q, k, v, do), dtype)
    check(run(q, k, v), reference(q, k, v), dtype)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(4, 9, 70, 2, 2, 16), (4, 100, 20, 4, 2, 32), (4, 3, 700, 2, 1, 64), (4, 70, 90, 2, 2, 16),
                                   (4, 130, 300, 2, 1, 64)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["lens", "mask", "both"])
def test_masks(cuda_device, shape, dtype, kind):
    """Lengths (past the end, zero and negative ones too) and masks; what is masked holds NaN and infinities."""
    B, Tk = shape[0], shape[2]
    q, k, v, do = make(cuda_device, *shape, dtype, seed=1)
    lens = mask = None
    if kind != "mask":
        lens = torch.tensor([Tk // 2, 0, Tk + 5, 1] if kind == "lens" else [Tk // 2, -3, Tk, 17], dtype=torch.int32,
                            device=cuda_device)
    if kind != "lens":
        mask = torch.rand(B, Tk, generator=torch.Generator().manual_seed(2)).lt(0.6).to(cuda_device)
        mask[2] = False
        mask[3] = False
        mask[3, 13] = True
    gone = ~there(B, Tk, lens, mask, cuda_device)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device=cuda_device).to(q.dtype)
    k[gone] = bad[torch.arange(int(gone.sum()), device=cuda_device) % 3][:, None, None]
    v[gone] = bad[torch.arange(int(gone.sum()), device=cuda_device) % 3][:, None, None]
    got = run(q, k, v, do, key_lens=lens, key_mask=mask)
    check(got, reference(q, k, v, do, lens=lens, mask=mask), dtype)
    empty = ~there(B, Tk, lens, mask, cuda_device).any(1)
    assert empty.any()
    assert torch.all(got[0][empty] == 0) and torch.all(got[1][empty] == 0)
    assert torch.all(got[2][gone] == 0) and torch.all(got[3][gone] == 0)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_single_key_has_no_query_gradient(cuda_device, dtype):
    """With one key the softmax is constant: out = v, and dq, dk are exactly zero."""
    q, k, v, do = make(cuda_device, 2, 37, 1, 2, 2, 16, dtype)
    out, dq, dk, _ = run(q, k, v, do)
    assert torch.equal(out, v.expand_as(out)) and not dq.any() and not dk.any()


def test_large_logits_and_scale(cuda_device):
    """Logits of some hundreds (a peaked softmax) and an explicit scale."""
    for dtype in DTYPES:
        q, k, v, do = make(cuda_device, 2, 20, 100, 2, 2, 32, dtype, seed=3)
        # exactly representable scaling, so that the logits' own error stays 2^-24 of their size
        q = q * 8
        u = torch.finfo(DTYPES[dtype]).eps / 2
        ref = reference(q, k, v, scale=1.0)
        size = (8 * 32) * 2.0 ** -24 * 8        # |s| up to 8 * 32, a few roundings of that size in the exponent
        (y,) = run(q, k, v, scale=1.0)
        allow = u * ref[0][0].abs() + (size + 4 * u * u + NOISE) * ref[0][1] + 1e-7
        assert torch.all((y.double() - ref[0][0]).abs() <= allow)


def test_strides_and_broadcast(cuda_device):
    """Head-major views, rows inside a wider buffer, one image's keys shared by all prompts (batch
    stride 0), and gradients that arrive transposed; dk, dv of the shared keys are the sum."""
    g = torch.Generator().manual_seed(4)
    dev = cuda_device
    qkv = torch.randn(3, 50, 3, 4, 32, generator=g).to(torch.bfloat16).to(dev)
    q = qkv[:, :20, 0]
    k = qkv[:1, :, 1].expand(3, -1, -1, -1)
    v = torch.randn(3, 4, 50, 32, generator=g).to(torch.bfloat16).to(dev).transpose(1, 2)
    do = torch.randn(3, 4, 20, 32, generator=g).to(torch.bfloat16).to(dev).transpose(1, 2)
    check(run(q, k, v, do), reference(q, k, v, do), "bf16")
    leaf = qkv[:1, :, 1].clone().requires_grad_(True)
    out = ops.cross_attn(q, leaf.expand(3, -1, -1, -1), v)
    (gk,) = torch.autograd.grad(out, leaf, do)
    ref = reference(q, k, v, do)[2][0].sum(0, keepdim=True)
    assert (gk.double() - ref).abs().max() <= 2.0 ** -7 * ref.abs().max()
    odd = do.new_zeros(3, 20, 4, 33)[..., 1:].copy_(do)          # rows that start off a 16-byte boundary
    qq = q.detach().clone().requires_grad_(True)
    (gq,) = torch.autograd.grad(ops.cross_attn(qq, k, v), qq, odd)
    (gq2,) = torch.autograd.grad(ops.cross_attn(qq, k, v), qq, do)
    assert torch.equal(gq, gq2)


def test_partial_gradients(cuda_device):
    q, k, v, do = make(cuda_device, 2, 9, 70, 2, 2, 16, "bf16")
    full = run(q, k, v, do)
    for i in range(3):
        ins = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        (g,) = torch.autograd.grad(ops.cross_attn(*ins), ins[i], do)
        assert torch.equal(g, full[i + 1])


def test_status_becomes_the_library_error(cuda_device):
    """A refusal of the C entry that the wrapper does not foresee (a 65536th batch entry)."""
    q = torch.zeros(65536, 1, 1, 8, dtype=torch.float16, device=cuda_device)
    with pytest.raises(_lib.SparseSAMError) as e:
        ops.cross_attn(q, q, q)
    assert e.value.status == _lib.SSAM_ERR_UNSUPPORTED and e.value.fn == "ssam_cross_attn_fwd"


def test_gradients_are_not_differentiated_again(cuda_device):
    """Asking for a graph of the backward pass is fine; differentiating it is an error, not a silent zero."""
    q, k, v, do = make(cuda_device, 1, 4, 9, 1, 1, 16, "fp32")
    q.requires_grad_(True)
    (g,) = torch.autograd.grad(ops.cross_attn(q, k, v), q, do, create_graph=True)
    assert torch.equal(g.detach(), run(q.detach(), k, v, do)[1])
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()
    assert q.grad is None


def test_empty_sets(cuda_device):
    q, k, v, do = make(cuda_device, 2, 5, 6, 2, 2, 16, "fp32")
    out, dq, dk, dv = run(q, k[:, :0], v[:, :0], do)
    assert out.shape == q.shape and not out.any() and not dq.any() and dk.shape == (2, 0, 2, 16)
    out, dq, dk, dv = run(q[:, :0], k, v, do[:, :0])
    assert out.shape == (2, 0, 2, 16) and not dk.any() and not dv.any()
    assert run(q[:0], k[:0], v[:0])[0].shape == (0, 5, 2, 16)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(1, 8, 4096, 8, 8, 16), (2, 2000, 11, 4, 4, 16), (1, 200, 1000, 2, 1, 64)],
                         ids=lambda s: "x".join(map(str, s)))
def test_equal_calls_give_equal_bits(cuda_device, shape, dtype):
    q, k, v, do = make(cuda_device, *shape, dtype)
    a = run(q, k, v, do)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(a, run(q, k, v, do)))


def test_gradient_matches_differences(cuda_device):
    """Directional derivative of sum(out * do) in fp32 against central differences of the definition in 64 bits."""
    q, k, v, do = make(cuda_device, 1, 6, 40, 2, 1, 16, "fp32", seed=5)
    _, dq, dk, dv = run(q, k, v, do)
    g = torch.Generator().manual_seed(6)
    dirs = [torch.randn(t.shape, generator=g).to(cuda_device).double() for t in (q, k, v)]

    def f(e):
        a, b, c = (t.double() + e * d for t, d in zip((q, k, v), dirs))
        s = torch.einsum("bqhd,bkhd->bhqk", a, b.repeat_interleave(2, 2)) / 4.0
        return (torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), c.repeat_interleave(2, 2)) * do.double()).sum()

    num = ((f(1e-5) - f(-1e-5)) / 2e-5).item()
    ana = sum((x.double() * d).sum().item() for x, d in zip((dq, dk, dv), dirs))
    size = sum((x.double() * d).abs().sum().item() for x, d in zip((dq, dk, dv), dirs))
    assert abs(num - ana) <= 1e-5 * size      # differences: e^2 terms and 64-bit cancellation stay under 1e-7


def test_graph_replay_and_side_stream(cuda_device):
    """Captured forward and backward replay on new inputs; a call on a side stream."""
    q, k, v, do = make(cuda_device, 2, 8, 300, 4, 4, 16, "bf16")
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b, c = (t.clone().requires_grad_(True) for t in (q, k, v))
        first = [ops.cross_attn(a, b, c).detach()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = ops.cross_attn(a, b, c)
            grads = torch.autograd.grad(out, (a, b, c), do)
            out = out.detach()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], run(q, k, v)[0])
    q2, k2, v2, do2 = make(cuda_device, 2, 8, 300, 4, 4, 16, "bf16", seed=9)
    with torch.no_grad():
        a.copy_(q2), b.copy_(k2), c.copy_(v2)
    do.copy_(do2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip([out, *grads], run(q2, k2, v2, do2)))


def test_offsets_past_32_bits(cuda_device):
    """Keys of a long cache whose byte offsets pass 2^32 (a strided view: rows far apart)."""
    step = 1 << 26                                          # 2^26 elements between tokens
    buf = torch.empty(step * 40 + 64, dtype=torch.float16, device=cuda_device)
    q, k, v, _ = make(cuda_device, 1, 3, 40, 1, 1, 16, "fp16")
    far = buf.as_strided((1, 40, 1, 16), (step, step, 16, 1), 16)
    far.copy_(k)
    vfar = buf.as_strided((1, 40, 1, 16), (step, step, 16, 1), 32)
    vfar.copy_(v)
    check(run(q, far, vfar), reference(q, k, v), "fp16")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", [(2, 150, 200, 2, 1, 128), (1, 130, 70, 6, 2, 96), (3, 50, 90, 6, 2, 72), (2, 1, 300, 140, 1, 64),
                                   (2, 257, 1030, 2, 2, 128), (1, 400, 37, 3, 3, 16), (1, 20, 260, 2, 2, 128),
                                   (1, 3, 700, 90, 3, 32)],
                         ids=lambda s: "x".join(map(str, s)))
def test_long_sides(cuda_device, shape, dtype):
    """Tiles of 128 query rows that cross from one head of a group to the next, two panels of channels."""
    q, k, v, do = make(cuda_device, *shape, dtype, seed=7)
    B, Tk = shape[0], shape[2]
    check(run(q, k, v, do), reference(q, k, v, do), dtype)
    mask = torch.rand(B, Tk, generator=torch.Generator().manual_seed(8)).lt(0.7).to(cuda_device)
    mask[0, : Tk // 2] = False
    lens = torch.full((B,), Tk - 3, dtype=torch.int32, device=cuda_device)
    gone = ~there(B, Tk, lens, mask, cuda_device)
    k[gone] = math.nan
    v[gone] = math.inf
    got = run(q, k, v, do, key_lens=lens, key_mask=mask)
    check(got, reference(q, k, v, do, lens=lens, mask=mask), dtype)
    assert not got[2][gone].any() and not got[3][gone].any()


@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("low", [-20, -6])
def test_half_gradients_of_any_size(cuda_device, D, low):
    """fp16: values and incoming gradients that grow by 2^10 each along the walk, so that the power of two that
    dS enters its products with has to follow; small ones (from 2^-26) and large ones (to 2^12)."""
    q, k, v, do = make(cuda_device, 2, 300, 400, 2, 2, D, "fp16", seed=9)
    rise = lambda n: torch.exp2(torch.arange(n, device=cuda_device) * 10 // n).half()  # noqa: E731
    v = v * rise(400)[None, :, None, None] * 2.0 ** -6
    do = do * rise(300)[None, :, None, None] * 2.0 ** low
    check(run(q, k, v, do), reference(q, k, v, do), "fp16")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("Tq,Tk,D", [(90, 100, 64), (90, 100, 128), (100, 9, 16), (9, 100, 16), (200, 9, 32)])
def test_far_rows_of_every_kernel(cuda_device, dtype, Tq, Tk, D):
    """All three inputs and the incoming gradient strided so that their offsets pass 2^31 elements."""
    step = (1 << 31) // 80
    step -= step % 8
    buf = torch.empty(step * 200 + 4 * D, dtype=DTYPES[dtype], device=cuda_device)
    q, k, v, do = make(cuda_device, 1, Tq, Tk, 1, 1, D, dtype, seed=12)
    expect = run(q, k, v, do)
    far = []
    for i, t in enumerate((q, k, v, do)):
        f = buf.as_strided(t.shape, (step, step, D, 1), i * D)
        far.append(f.copy_(t))
    got = run(*far)
    assert all(torch.equal(x, y) for x, y in zip(got, expect))


@pytest.mark.parametrize("Tq,Tk", [(3, 400), (400, 5), (100, 100)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_far_negative_logits(cuda_device, dtype, Tq, Tk):
    """Logits of -7e36, all alike: still a softmax, of equal weights; not a row without keys."""
    q, k, v, _ = make(cuda_device, 1, Tq, Tk, 2, 2, 16, dtype, seed=13)
    q, k = torch.full_like(q, -(2.0 ** 60)), torch.full_like(k, 2.0 ** 60)
    (out,) = run(q, k, v)
    mean = v.double().mean(1, keepdim=True).expand(-1, Tq, -1, -1)
    u = torch.finfo(DTYPES[dtype]).eps / 2
    size = v.double().abs().mean(1, keepdim=True)
    assert torch.all((out.double() - mean).abs() <= u * mean.abs() + (4 * u * u + NOISE) * size)
