"""The operators together, as the decoder uses them: attention layers, a segmentation head of convolution, GroupNorm
and activation, and the whole mask decoder, forward and backward.

Tolerances. fp32 on the GPU against the same modules in 64 bits on the CPU: a value is a chain of some 40 layers of
sums over at most 2304 terms; each adds roundings of random sign, 2^-24 sqrt(2304) of its magnitude, together below
40 * 48 * 2^-24 = 1.2e-4 of a tensor's 2-norm. Half precision against fp32: each of the 40 layers rounds its value
once, u = eps / 2 of random sign and independent, 6.4 u of the norm, with a factor of 4 for the norm layers and the
softmax, which divide by a spread smaller than the values: 26 u (fp16 0.0127, bf16 0.10). To that come the signs that
ReLU reads: an input with an error of rms e = 6.4 u of its spread has the other sign with probability phi(0) E|error| =
0.4 * 0.8 e, and then a whole component of the gradient (one of the half that pass) is there or not: sqrt(0.32 e / 0.5) =
0.8 sqrt(e) of the norm (fp16 0.045, bf16 0.13). In fp32 that term is 0.8 sqrt(6.4 * 2^-24) = 5e-4."""
import copy

import pytest
import torch

from sparsesam_b200 import _lib, hq, ops

pytestmark = pytest.mark.gpu


def half_bound(dt):
    u = torch.finfo(dt).eps / 2
    return 26 * u + 0.8 * (6.4 * u) ** 0.5


def off(x, ref):
    return ((x.detach().double().cpu() - ref.double().cpu()).norm() / ref.double().norm().cpu()).item()


@pytest.fixture(autouse=True)
def exact_fp32():
    old = torch.backends.cuda.matmul.allow_tf32, torch.backends.cudnn.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = torch.backends.cudnn.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32, torch.backends.cudnn.allow_tf32 = old


class Head(torch.nn.Module):
    """Image tokens read padded prompts, then convolution -> GroupNorm -> ReLU twice on their map."""

    def __init__(self, c=64):
        super().__init__()
        self.attn = hq.DecoderAttention(c, 4)
        self.norm = hq.RowLayerNorm(c)
        self.c1, self.n1 = torch.nn.Conv2d(c, c, 3, padding=1), hq.GroupNormAct2d(8, c, act="relu")
        self.c2, self.n2 = torch.nn.Conv2d(c, c, 3, padding=1), hq.GroupNormAct2d(8, c, act="gelu")

    def forward(self, tokens, prompts, lens, side):
        t = self.norm(tokens + self.attn(tokens, prompts, prompts, key_lens=lens))
        m = t.view(t.shape[0], side, side, -1).permute(0, 3, 1, 2)
        m = self.n1(self.c1(m).contiguous(memory_format=torch.channels_last))
        return self.n2(self.c2(m).contiguous(memory_format=torch.channels_last))


def step(mod, ins, fixed, dout):
    ins = [t.detach().requires_grad_(True) for t in ins]
    mod.zero_grad(set_to_none=True)
    out = mod(*ins, *fixed)
    outs = out if isinstance(out, tuple) else (out,)
    torch.autograd.backward(outs, [d.to(o) for d, o in zip(dout, outs)])
    return [o.detach() for o in outs] + [t.grad for t in ins] + [p.grad for p in mod.parameters() if p.grad is not None]


def test_segmentation_head_trains(cuda_device):
    g = torch.Generator().manual_seed(0)
    torch.manual_seed(0)
    mod, side, B = Head().double(), 12, 3
    ins = [torch.randn(B, side * side, 64, generator=g).double(), torch.randn(B, 9, 64, generator=g).double()]
    lens = torch.tensor([9, 4, 0], dtype=torch.int32)
    dout = [torch.randn(B, 64, side, side, generator=g).double()]
    ref = step(mod, ins, (lens, side), dout)
    for dt, bound in ((torch.float32, 6.2e-4), (torch.float16, half_bound(torch.float16)),
                      (torch.bfloat16, half_bound(torch.bfloat16))):
        m = copy.deepcopy(mod).to(cuda_device, dt)
        n0 = _lib.launch_count
        got = step(m, [t.to(cuda_device, dt) for t in ins], (lens.to(cuda_device), side), dout)
        assert _lib.launch_count > n0
        assert len(got) == len(ref)
        for x, r in zip(got, ref):
            if r.norm() > 1e-6 * r.numel() ** 0.5:        # the key bias has no gradient: softmax does not see it
                assert off(x, r) <= bound


class Decode(torch.nn.Module):
    def __init__(self, dec):
        super().__init__()
        self.dec = dec

    def forward(self, image, sparse, interm, pe, dense):
        return self.dec(image, pe, sparse, dense, False, True, [interm])


def test_mask_decoder_trains(cuda_device):
    """Masks, IoU and every parameter's gradient of MaskDecoderHQ, two images with one box prompt each."""
    g = torch.Generator().manual_seed(1)
    torch.manual_seed(1)
    dec = hq.MaskDecoderHQ(transformer_dim=64, transformer=hq.TwoWayTransformer(2, 64, 4, 128), vit_dim=96,
                           iou_head_hidden_dim=64)
    hq.init_prompt_decoder_weights(dec, 3)
    mod = Decode(dec).double()
    ins = [torch.randn(2, 64, 16, 16, generator=g).double(), torch.randn(2, 2, 64, generator=g).double(),
           torch.randn(2, 16, 16, 96, generator=g).double()]
    pe = torch.randn(1, 64, 16, 16, generator=g).double()
    dense = torch.randn(2, 64, 16, 16, generator=g).double() * 0.1
    dout = [torch.randn(2, 1, 64, 64, generator=g).double(), torch.randn(2, 1, generator=g).double()]
    ref = step(mod, ins, (pe, dense), dout)
    for dt, bound in ((torch.float32, 6.2e-4), (torch.float16, half_bound(torch.float16))):
        m = copy.deepcopy(mod).to(cuda_device, dt)
        got = step(m, [t.to(cuda_device, dt) for t in ins], (pe.to(cuda_device, dt), dense.to(cuda_device, dt)), dout)
        assert len(got) == len(ref)
        biggest = max(r.norm() / r.numel() ** 0.5 for r in ref)
        for x, r in zip(got, ref):
            # the relative error of a tensor that is small beside its neighbours is theirs
            size = max(r.norm().item(), (1e-2 * biggest * r.numel() ** 0.5).item())
            assert (x.double().cpu() - r).norm().item() <= bound * size, (tuple(r.shape), dt)


def test_decoder_attention_matches_its_torch_form(cuda_device):
    """hq.DecoderAttention on the GPU against the same module on the CPU, with padded keys."""
    torch.manual_seed(2)
    for dim, heads, rate in ((256, 8, 2), (256, 8, 1), (48, 2, 1)):
        mod = hq.DecoderAttention(dim, heads, rate)
        q, k = torch.randn(3, 40, dim), torch.randn(3, 25, dim)
        lens = torch.tensor([25, 0, 7], dtype=torch.int32)
        mask = torch.rand(3, 25) < 0.7
        for kw in ({}, {"key_lens": lens}, {"key_mask": mask}, {"key_lens": lens, "key_mask": mask}):
            want = mod(q, k, k, **kw).detach()
            got = copy.deepcopy(mod).to(cuda_device)(q.to(cuda_device), k.to(cuda_device), k.to(cuda_device),
                                                     **{n: t.to(cuda_device) for n, t in kw.items()})
            assert off(got, want) <= 1e-5


def test_group_norm_module(cuda_device):
    """hq.GroupNormAct2d: channels-last maps through the kernel, other layouts and dtypes through torch, one result."""
    x = torch.randn(2, 32, 7, 9)
    for act in ops.ACTIVATIONS:
        mod = hq.GroupNormAct2d(4, 32, act=act)
        torch.nn.init.normal_(mod.weight)
        torch.nn.init.normal_(mod.bias)
        want = mod.double()(x.double()).detach()
        mod = mod.to(cuda_device).float()
        n0 = _lib.launch_count
        a = mod(x.to(cuda_device).contiguous(memory_format=torch.channels_last))
        assert _lib.launch_count > n0 and a.is_contiguous(memory_format=torch.channels_last)
        n0 = _lib.launch_count
        b = mod(x.to(cuda_device))
        assert _lib.launch_count == n0
        assert off(a, want) <= 1e-6 and off(b, want) <= 1e-6
    with pytest.raises(ValueError):
        hq.GroupNormAct2d(4, 32, act="tanh")


def test_attention_of_many_shapes_side_by_side(cuda_device):
    """Calls on two streams at once: results as one after the other."""
    g = torch.Generator().manual_seed(3)
    cases = []
    for Tq, Tk in ((8, 4096), (4096, 8), (300, 200), (1, 5000)):
        q = torch.randn(2, Tq, 4, 32, generator=g).to(cuda_device, torch.bfloat16)
        k = torch.randn(2, Tk, 4, 32, generator=g).to(cuda_device, torch.bfloat16)
        cases.append((q, k, ops.cross_attn(q, k, k)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    outs = []
    for i, (q, k, _) in enumerate(cases * 4):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.cross_attn(q, k, k))
    torch.cuda.synchronize()
    assert all(torch.equal(o, c[2]) for o, c in zip(outs, cases * 4))


def test_attention_of_many_prompts(cuda_device):
    """More prompts than one launch takes: the same rows as in two calls."""
    torch.manual_seed(0)
    attn = hq.DecoderAttention(16, 2).to(cuda_device)
    x = torch.randn(65537, 2, 16, device=cuda_device)
    with torch.no_grad():
        whole = attn(x, x, x)
        parts = torch.cat([attn(t, t, t) for t in x.split(40000)])
    # fp32 of two orders of summation: unit-size logits and values, 4 eps of them
    assert (whole - parts).abs().max() <= 4 * torch.finfo(torch.float32).eps * parts.abs().max() * 2


@pytest.mark.parametrize("captured", [False, True])
def test_calls_behind_one_another(cuda_device, captured):
    """Each call reads what the one before has written, in memory that earlier calls have just given back: the same
    bits as with a synchronisation after each. Short and long sides, resident and streamed maps, gradients."""
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(cuda_device)  # noqa: E731
    tokens, image, rows = r(8, 9, 8, 16), r(8, 4096, 8, 16), r(2, 200, 2, 64)
    maps, w, b = r(16, 128 * 128, 64), r(64), r(64)

    def chain(wait):
        t, i, y, m = tokens, image, rows, maps
        out = []
        for _ in range(3):
            t = wait(ops.cross_attn(t, i, i))
            i = wait(ops.cross_attn(i, t, t))
            y = wait(ops.cross_attn(y, y, y))
            m = wait(ops.groupnorm_act(m, 8, w, b, 1e-5, "gelu"))
            y = wait(ops.groupnorm_act(y.reshape(2, 400, 64), 4, w, b, 1e-5, "silu")).view(2, 200, 2, 64)
            y = wait(ops.layernorm_gelu_half(y.contiguous(), w, b, 1e-6, True))
        leaves = [x.detach().requires_grad_(True) for x in (t, i, y, m, w, b)]
        o = wait(ops.cross_attn(leaves[0], leaves[1], leaves[1]))
        p = wait(ops.cross_attn(leaves[2], leaves[2], leaves[2]))
        n = wait(ops.groupnorm_act(leaves[3], 8, leaves[4], leaves[5], 1e-5, "gelu"))
        q = wait(ops.layernorm_gelu_half(p, leaves[4], leaves[5], 1e-6, True))
        grads = torch.autograd.grad([o, q, n], leaves, [tokens, rows, maps])
        return [*(x.detach() for x in (t, i, y, m, o, p, n, q)), *grads]

    def settle(x):
        torch.cuda.synchronize()
        return x

    expect = [x.clone() for x in chain(settle)]
    torch.cuda.synchronize()
    if captured:
        side = torch.cuda.Stream(cuda_device)
        side.wait_stream(torch.cuda.current_stream(cuda_device))
        with torch.cuda.stream(side):
            chain(lambda x: x)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                got = chain(lambda x: x)
        for _ in range(3):
            graph.replay()
    else:
        for _ in range(3):
            got = chain(lambda x: x)
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(zip(expect, got)):
        assert torch.isfinite(x.float()).all() and torch.equal(x, y), i
