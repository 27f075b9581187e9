"""The decoder's modules where torch follows the program through its operators: scripts, traces, compilers, vmap and
other transforms, forward-mode differentiation, dispatch modes. They see torch's attention and norms; the operators
themselves are errors there and never leave a hole in a trace or drop a tangent."""
import copy

import pytest
import torch
import torch.autograd.forward_ad as fwd
from test_decoder_attention import LENS, attention, near
from torch.utils.flop_counter import FlopCounterMode

from sparsesam_b200 import hq, ops

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------
# On the host
# ---------------------------------------------------------------------------
def test_script():
    mod, q, k, v = attention()
    script = torch.jit.script(mod)
    near(script(q, k, v), mod(q, k, v))
    mask = torch.rand(3, 25, generator=torch.Generator().manual_seed(2)) < 0.6
    near(script(q, k, v, LENS, mask), mod(q, k, v, LENS, mask))


def plain_calls(device="cpu"):
    x = torch.randn(2, 6, 2, 16).to(device, torch.float16)
    w = torch.ones(32).to(device, torch.float16)
    y = torch.randn(2, 6, 32).to(device, torch.float16)
    return {"cross_attn": (lambda x: ops.cross_attn(x, x, x), x),
            "groupnorm_act": (lambda y: ops.groupnorm_act(y, 4, w, w), y),
            "layernorm_gelu_half": (lambda y: ops.layernorm_gelu_half(y, w, w, 1e-6, True), y)}


@pytest.mark.parametrize("name", ["cross_attn", "groupnorm_act", "layernorm_gelu_half"])
def test_operators_refuse_what_would_not_see_them(name):
    """Before anything else, so also for tensors without a GPU."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x = plain_calls()[name]
    with pytest.raises(RuntimeError, match="plain tensors"):
        torch.jit.trace(f, x)
    with pytest.raises(RuntimeError, match="plain tensors"):
        torch.vmap(f)(x[None])
    with pytest.raises(RuntimeError, match="plain tensors"):
        torch.func.grad(lambda t: f(t).sum())(x)
    with pytest.raises(RuntimeError, match="plain tensors"):
        make_fx(f)(x)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="plain tensors"):
            f(fwd.make_dual(x, torch.ones_like(x)))
    with pytest.raises(ValueError, match="CUDA"):
        f(x)


# ---------------------------------------------------------------------------
# On the GPU
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attention_is_traced_and_scripted(cuda_device, dtype):
    mod, q, k, v = attention(cuda_device, dtype)
    want = mod(q, k, v)
    traced = torch.jit.trace(mod, (q, k, v), check_trace=False)   # its check would compare it with the kernel
    near(traced(q, k, v), want, dtype)
    near(traced(q + 1, k - 1, v), mod(q + 1, k - 1, v), dtype)
    near(torch.jit.script(mod)(q, k, v), want, dtype)


@gpu
def test_attention_is_compiled_whole(cuda_device):
    mod, q, k, v = attention(cuda_device)
    near(torch.compile(mod, backend="eager", fullgraph=True)(q, k, v), mod(q, k, v))
    near(torch.export.export(mod, (q, k, v)).module()(q, k, v), mod(q, k, v))


@gpu
def test_attention_under_transforms(cuda_device):
    mod, q, k, v = attention(cuda_device)
    qs = torch.stack([q, q + 1])
    near(torch.vmap(lambda t: mod(t, k, v))(qs), torch.stack([mod(t, k, v) for t in qs]))
    leaf = q.clone().requires_grad_(True)
    near(torch.func.grad(lambda t: mod(t, k, v).square().sum())(q), torch.autograd.grad(mod(leaf, k, v).square().sum(), leaf)[0])


@gpu
def test_attention_carries_tangents(cuda_device):
    """Forward mode through torch's decomposed attention; its fused forms raise, which is an answer too."""
    from torch.nn.attention import SDPBackend, sdpa_kernel
    mod, q, k, v = attention(cuda_device)
    t = torch.randn_like(q)
    host = copy.deepcopy(mod).cpu()
    with torch.no_grad(), sdpa_kernel(SDPBackend.MATH), fwd.dual_level():
        got = fwd.unpack_dual(mod(fwd.make_dual(q, t), k, v)).tangent
        want = fwd.unpack_dual(host(fwd.make_dual(q.cpu(), t.cpu()), k.cpu(), v.cpu())).tangent
    assert got is not None
    near(got.cpu(), want)


@gpu
def test_attention_is_counted(cuda_device):
    mod, q, k, v = attention(cuda_device, torch.float16)
    with FlopCounterMode(display=False) as c:
        mod(q, k, v)
    linear = 2 * 3 * 64 * 32 * (9 + 25 + 25 + 9)
    assert c.get_total_flops() >= linear + 4 * 3 * 4 * 9 * 25 * 8


@gpu
@pytest.mark.parametrize("name", ["norm2d", "rows", "group"])
def test_half_norms_are_traced_and_mapped(cuda_device, name):
    torch.manual_seed(0)
    mod, x = {"norm2d": (hq.LayerNorm2d(64, gelu=True), torch.randn(2, 64, 5, 6)),
              "rows": (hq.RowLayerNorm(64), torch.randn(2, 9, 64)),
              "group": (hq.GroupNormAct2d(8, 64, act="silu"), torch.randn(2, 64, 5, 6))}[name]
    mod, x = mod.to(cuda_device, torch.float16), x.to(cuda_device, torch.float16)
    if x.dim() == 4:
        x = x.contiguous(memory_format=torch.channels_last)
    want = mod(x)
    traced = torch.jit.trace(mod, x, check_trace=False)
    near(traced(x), want, torch.float16)
    near(traced(x * 2 - 1), mod(x * 2 - 1), torch.float16)
    near(torch.vmap(mod)(torch.stack([x, x + 1]))[0], want, torch.float16)


@gpu
@pytest.mark.parametrize("name", ["norm2d", "rows", "group"])
def test_half_norms_run_under_a_compiler(cuda_device, name):
    """Not as one graph: the operators are called between two."""
    torch.manual_seed(0)
    mod, x = {"norm2d": (hq.LayerNorm2d(64, gelu=True), torch.randn(2, 64, 5, 6)),
              "rows": (hq.RowLayerNorm(64), torch.randn(2, 9, 64)),
              "group": (hq.GroupNormAct2d(8, 64, act="silu"), torch.randn(2, 64, 5, 6))}[name]
    mod, x = mod.to(cuda_device, torch.float16), x.to(cuda_device, torch.float16)
    if x.dim() == 4:
        x = x.contiguous(memory_format=torch.channels_last)
    near(torch.compile(mod, backend="eager")(x) + 1, mod(x) + 1, torch.float16)
