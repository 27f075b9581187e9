"""Calls of the decoder's operators that random inputs do not make: weights far below the largest one, values that are
not finite beside ones that are, logits at the end of fp32. Bounds as derived in test_gpu_cross_attention.py and
test_gpu_norms.py; where something else is allowed, the test says why."""
import ctypes
import math

import pytest
import torch
from test_gpu_cross_attention import DTYPES, NOISE, check, make, reference, run, there

from sparsesam_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def ids(s):
    return "x".join(map(str, s))


# B, Tq, Tk, H, Hk, D of every forward kernel of the half types: few rows (one head and two per fragment, three and four
# tiles of rows, two per row of a group), few keys (the same), tcgen05 (one and two panels of channels; split and whole)
FORWARD = [(1, 3, 4096, 2, 2, 16), (40, 8, 600, 8, 8, 16), (40, 12, 300, 8, 8, 16), (1, 20, 700, 2, 2, 64), (2, 3, 900, 4, 2, 32),
           (1, 5, 300, 1, 1, 128), (2, 70, 64, 1, 1, 16), (3, 50, 8, 2, 2, 16), (3, 50, 15, 2, 2, 16), (1, 40, 30, 2, 1, 64),
           (1, 200, 1000, 2, 1, 64), (1, 130, 900, 2, 2, 128), (8, 128, 128, 8, 8, 64), (1, 70, 100, 1, 1, 24)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("far", [17.0, 19.5, 21.75])
@pytest.mark.parametrize("shape", FORWARD, ids=ids)
def test_weights_far_below_the_largest(cuda_device, shape, far, dtype):
    """One key has nearly all the weight and a value of zero: the result is what the others' weights of e^-far (2^-24 to
    2^-31) carry, and has the digits of its own type."""
    B, Tq, Tk, H, Hk, D = shape
    q, k, v, _ = make(cuda_device, *shape, dtype, seed=21)
    q[..., 0], k[..., 0] = 1.0, 0.0
    q[..., 1:], k[..., 1:] = q[..., 1:] / 16, k[..., 1:] / 16     # the other logits differ a little
    sink = Tk // 2
    k[:, sink] = 0.0
    k[:, sink, :, 0] = far
    v = v.abs() * 512 + 512
    v[:, sink] = 0.0
    got = run(q, k, v, scale=1.0)
    check(got, reference(q, k, v, scale=1.0), dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("far", [19.5, 23.0])
@pytest.mark.parametrize("shape", FORWARD, ids=ids)
def test_gradients_of_weights_far_below_the_largest(cuda_device, shape, far, dtype):
    """Keys of small weight (2^-28, 2^-33) below a large incoming gradient, and channels that only they reach: dq of those
    channels, dk and dv of those keys keep the digits of the type."""
    B, Tq, Tk, H, Hk, D = shape
    q, k, v, do = make(cuda_device, *shape, dtype, seed=22)
    q[..., 0], k[..., 0] = 1.0, 0.0
    q[..., 1:], k[..., 1:] = q[..., 1:] / 16, k[..., 1:] / 16
    near = min(3, Tk // 2)
    k[:, :near] = 0.0
    k[:, :near, :, 0] = far                                        # the near keys share the weight
    v = v / 16                                                     # keeps dk below fp16's 65504
    do = do.abs() * 256 + 256
    got = run(q, k, v, do, scale=1.0)
    check(got, reference(q, k, v, do, scale=1.0), dtype)


def close(y, ref, dtype, where=...):
    """y against (value, size of the terms), as check(), at `where`."""
    u = torch.finfo(DTYPES[dtype]).eps / 2
    r, size = ref
    allow = u * r.abs() + (NOISE + (4 * u * u if dtype != "fp32" else 0.0)) * size + 8 * torch.finfo(DTYPES[dtype]).tiny * u
    err = (y.double() - r).abs()[where]
    assert torch.all(err <= allow[where]), (err - allow[where]).max().item()


BAD = [math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", ["lens", "mask"])
@pytest.mark.parametrize("shape", FORWARD, ids=ids)
def test_queries_without_keys(cuda_device, shape, kind, dtype):
    """Two padded entries of a batch have no keys, and queries and incoming gradients that are whatever their memory
    held: zero rows and zero gradients there, and the other entries' as ever."""
    shape = (4, *shape[1:])
    q, k, v, do = make(cuda_device, *shape, dtype, seed=23)
    lens = mask = None
    if kind == "lens":
        lens = torch.tensor([shape[2], 0, (shape[2] + 1) // 2, 0], dtype=torch.int32, device=cuda_device)
    else:
        mask = torch.rand(4, shape[2], generator=torch.Generator().manual_seed(24)).lt(0.7).to(cuda_device)
        mask[::2, 0] = True
        mask[1::2] = False
    clean = q.clone(), do.clone()
    for t in (q, do):
        n = t[1::2].numel()
        t[1::2] = torch.tensor(BAD, device=cuda_device).to(t.dtype)[torch.arange(n, device=cuda_device) % 3].view(2, *t.shape[1:])
    out, dq = run(q, k, v, do, key_lens=lens, key_mask=mask)[:2]
    ref = reference(clean[0], k, v, clean[1], lens=lens, mask=mask)
    assert not out[1::2].any() and not dq[1::2].any()
    check([out, dq], ref, dtype)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", ["lens", "mask"])
@pytest.mark.parametrize("which", ["q", "dout"])
@pytest.mark.parametrize("shape", FORWARD, ids=ids)
def test_absent_keys_have_no_gradient(cuda_device, shape, which, kind, dtype):
    """A query, or its incoming gradient, that is not finite: keys that are not there keep zero gradients, and the other
    queries' rows are theirs."""
    shape = (4, *shape[1:])
    q, k, v, do = make(cuda_device, *shape, dtype, seed=25)
    Tq, Tk = shape[1:3]
    lens = mask = None
    if kind == "lens":
        lens = torch.tensor([Tk, Tk // 2, 1, 0], dtype=torch.int32, device=cuda_device)
    else:
        mask = torch.rand(4, Tk, generator=torch.Generator().manual_seed(26)).lt(0.6).to(cuda_device)
        mask[:3, 1] = True
        mask[3] = False
    ref = reference(q, k, v, do, lens=lens, mask=mask)
    bad = torch.zeros(q.shape[:3], dtype=torch.bool, device=cuda_device)
    for i in range(4):
        bad[i, (7 * i + 1) % Tq] = True
        (q if which == "q" else do)[i, (7 * i + 1) % Tq] = BAD[i % 3]
    out, dq, dk, dv = run(q, k, v, do, key_lens=lens, key_mask=mask)
    gone = ~there(4, Tk, lens, mask, cuda_device)
    assert not dk[gone].any() and not dv[gone].any()
    close(out, ref[0], dtype, ~bad if which == "q" else ...)
    close(dq, ref[1], dtype, ~bad)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("which", ["q", "k", "v"])
@pytest.mark.parametrize("shape", FORWARD, ids=ids)
def test_heads_do_not_meet(cuda_device, shape, which, dtype):
    """Values that are not finite in one key head, or in its queries: the other heads are theirs."""
    B, Tq, Tk, H, Hk, D = shape
    H, Hk = max(H, 4), max(H, 4) * Hk // H
    q, k, v, do = make(cuda_device, B, Tq, Tk, H, Hk, D, dtype, seed=27)
    G = H // Hk
    ref = reference(q, k, v, do)
    for i, value in enumerate(BAD):
        a, b, c = q.clone(), k.clone(), v.clone()
        h = i % Hk
        {"q": a[:, :, h * G : (h + 1) * G], "k": b[:, :, h : h + 1], "v": c[:, :, h : h + 1]}[which][:, 0, :, i] = value
        got = run(a, b, c, do)
        for n, (y, r) in enumerate(zip(got, ref)):
            others = torch.arange(y.shape[2], device=cuda_device) // (G if n < 2 else 1) != h
            close(y, r, dtype, (slice(None), slice(None), others))
        if which == "q":                                           # and the other queries of the head itself
            close(got[0], ref[0], dtype, (slice(None), slice(1, None)))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", FORWARD, ids=ids)
def test_logits_at_the_end_of_fp32(cuda_device, shape, dtype):
    """Every logit -3.2e38 (in base 2): equal weights, not a row without keys; the base-2 logit is finite down to -3.4e38."""
    q, k, v, _ = make(cuda_device, *shape, dtype, seed=28)
    q.zero_(), k.zero_()
    q[..., 0], k[..., 0] = -(2.0 ** 64), 2.0 ** 63 * 1.3125         # <q, k> = -2.23e38, log2(e) times that -3.22e38
    (out,) = run(q, k, v, scale=1.0)
    mean = v.double().mean(1, keepdim=True).repeat_interleave(shape[3] // shape[4], 2).expand(out.shape)
    size = v.double().abs().mean(1, keepdim=True).repeat_interleave(shape[3] // shape[4], 2).expand(out.shape)
    close(out, (mean, size), dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", FORWARD, ids=ids)
def test_results_before_they_are_rounded(cuda_device, shape, dtype):
    """out_f32 and lse of the C entry: what the terms of P and V leave out shows here, without the result's rounding. One
    key has a weight just above a half and a value just above one, of which a bf16 term leaves most, the others are 0."""
    B, Tq, Tk, H, Hk, D = shape
    q, k, v, _ = make(cuda_device, *shape, dtype, seed=29)
    g = torch.Generator().manual_seed(30)
    q.zero_(), k.zero_()
    q[..., 0] = (torch.rand(B, Tq, H, generator=g) / 32 + math.log(Tk - 1)).to(q)
    k[:, Tk // 3, :, 0] = 1.0
    v.zero_()
    v[:, Tk // 3] = (1 + torch.rand(B, Hk, D, generator=g) / 128).to(v)
    out, out32 = torch.empty_like(q), torch.empty(B, Tq, H, D, device=cuda_device)
    lse = torch.empty(B, H, Tq, device=cuda_device)
    strides = (ctypes.c_int64 * 12)(*(x for t in (q, k, v, out) for x in t.stride()[:3]))
    _lib.call("ssam_cross_attn_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, B, Tq, Tk, H, Hk, D,
              {"fp16": 0, "bf16": 1}[dtype], 1.0, None, None, out.data_ptr(), out32.data_ptr(), lse.data_ptr(),
              torch.cuda.current_stream().cuda_stream)
    u = torch.finfo(q.dtype).eps / 2
    r, size = reference(q, k, v, scale=1.0)[0]
    assert torch.all((out32.double() - r).abs() <= (NOISE + 4 * u * u) * size)
    assert torch.equal(out, out32.to(out.dtype))
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double().repeat_interleave(H // Hk, 2))
    want = torch.logsumexp(s, -1) / math.log(2.0)
    assert torch.all((lse.double() - want).abs() <= NOISE + 2.0 ** -22 * want.abs())
