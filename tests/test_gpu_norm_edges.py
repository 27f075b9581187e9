"""Calls of ops.groupnorm_act and of the half LayerNorm's gradient that random inputs do not make: values that are not
finite beside ones that are, samples cut into several launches, ReLU's parameter gradients without its border. Bounds as
derived in test_gpu_norms.py."""
import math

import pytest
import torch
from test_gpu_norms import DTYPES, EPS24, check, make, off_border, reference, run

from sparsesam_b200 import _lib, hq, ops

pytestmark = pytest.mark.gpu


def within(got, ref, dtype, where, extra=0.0):
    """check() of the elements at `where` (one index per result). Against the definition rather than bit for bit: two
    channels share a reciprocal, so that the last digit of fp32 is the pair's."""
    u = torch.finfo(DTYPES[dtype]).eps / 2
    for i, (y, (r, size), at) in enumerate(zip(got, ref, where)):
        allow = u * r.abs() + ((32 if i == 0 else 96) * EPS24 + extra) * size + torch.finfo(DTYPES[dtype]).tiny * u * 8
        assert torch.all(((y.double() - r).abs() <= allow)[at]), i


@pytest.mark.parametrize("act", list(ops.ACTIVATIONS))
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("shape,groups", [((2, 5, 6, 16), 16), ((2, 7, 8, 24), 8), ((3, 9, 40), 8), ((2, 300, 300, 24), 8)],
                         ids=lambda s: str(s).replace(" ", ""))
def test_what_is_not_finite_stays_in_its_group(cuda_device, shape, groups, value, dtype, act):
    """One value of sample 1, in a group of one, three or five channels: out and dx outside of that group, dw and db
    outside of its channels are as without it."""
    x, w, b, do = make(cuda_device, shape, dtype)
    if act == "relu":
        do = torch.where(off_border(x, groups, w, b, 1e-5), torch.zeros_like(do), do)
    f = lambda x, w, b: ops.groupnorm_act(x, groups, w, b, 1e-5, act)  # noqa: E731
    ref = reference(x, groups, w, b, 1e-5, act, do)
    cg = shape[-1] // groups
    for g in (0, 1, groups - 1):
        y = x.clone()
        y.view(shape[0], -1, shape[-1])[1, 3, g * cg + cg // 2] = value
        spoilt = torch.zeros_like(x, dtype=torch.bool)
        spoilt[1, ..., g * cg : (g + 1) * cg] = True
        here = spoilt.flatten(0, -2).any(0)
        got = run(f, y, w, b, do)
        within(got, ref, dtype, (~spoilt, ~spoilt, ~here, ~here))
        assert act == "relu" or not torch.isfinite(got[0][spoilt]).any()     # ReLU's value of -infinity is 0


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_parameters_that_are_not_finite_stay_in_their_channel(cuda_device, value, dtype):
    x, w, b, do = make(cuda_device, (5, 100, 64), dtype)
    for f, groups, eps in ((lambda x, w, b: ops.layernorm_gelu_half(x, w, b, 1e-6, True), 1, 1e-6),
                           (lambda x, w, b: ops.groupnorm_act(x, 8, w, b, 1e-5, "gelu"), 8, 1e-5)):
        flat = (lambda t: t.view(500, 1, 64)) if groups == 1 else (lambda t: t)
        ref = [(r.view(5, 100, 64), s.view(5, 100, 64)) if r.dim() == 3 else (r, s)
               for r, s in reference(flat(x), groups, w, b, eps, "gelu", flat(do))]
        for c in (10, 37):
            for which in (0, 1):
                p = [w.clone(), b.clone()]
                p[which][c] = value
                rest = torch.arange(64, device=cuda_device) != c
                none = torch.zeros(64, dtype=torch.bool, device=cuda_device)
                # dx of a row (of a group) goes through the sums over its channels
                other = none if groups == 1 else torch.arange(64, device=cuda_device) // 8 != c // 8
                within(run(f, x, *p, do), ref, dtype, ((..., rest), (..., other), rest, rest), extra=2e-7)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gelu_of_large_values(cuda_device, dtype):
    """GELU(z) = z and 0 far out, infinities included, next to ordinary channels."""
    x, w, b, _ = make(cuda_device, (2, 40, 16), dtype)
    big = torch.finfo(x.dtype).max
    w.zero_()
    b.copy_(torch.tensor([-1.0, big, 0.5, -big, -0.5, math.inf, 1.0, -math.inf] * 2))
    y = ops.groupnorm_act(x, 2, w, b, 1e-5, "gelu")
    want = torch.where(b.double().abs() > 100, b.double().clamp_min(0), b.double() * torch.special.ndtr(b.double()))
    u = torch.finfo(x.dtype).eps / 2
    ok = torch.isinf(want)
    assert torch.all(torch.where(ok, y.double() == want, (y.double() - want).abs() <= u * want.abs() + 2e-7))


@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("dtype,C", [("fp16", 512), ("bf16", 512), ("fp32", 256)])
def test_groupnorm_in_several_launches(cuda_device, dtype, C, act):
    """Five samples of 18 MB: two launches of up to three forward, three of up to two backward."""
    x, w, b, do = make(cuda_device, (5, 132, 136, C), dtype)
    x += torch.arange(5, device=cuda_device).view(5, 1, 1, 1) / 4           # every sample its own mean
    check(run(lambda x, w, b: ops.groupnorm_act(x, 8, w, b, 1e-5, act), x, w, b, do), reference(x, 8, w, b, 1e-5, act, do), dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape,groups", [((1, 64, 64, 256), 8), ((2, 200, 200, 64), 8), ((3, 67, 45, 96), 4)],
                         ids=lambda s: str(s).replace(" ", ""))
def test_relu_parameter_gradients(cuda_device, shape, groups, dtype):
    """No gradient comes in where ReLU's input is within rounding of zero: the sums then have their ordinary bound."""
    x, w, b, do = make(cuda_device, shape, dtype)
    do = torch.where(off_border(x, groups, w, b, 1e-5), torch.zeros_like(do), do)
    check(run(lambda x, w, b: ops.groupnorm_act(x, groups, w, b, 1e-5, "relu"), x, w, b, do),
          reference(x, groups, w, b, 1e-5, "relu", do), dtype)


def test_more_maps_than_one_launch_takes(cuda_device):
    """The operator refuses them; the module goes to torch."""
    g = torch.Generator().manual_seed(3)
    mod = hq.GroupNormAct2d(2, 8, act="silu").to(cuda_device)
    x = torch.randn(65537, 8, 2, 3, generator=g).to(cuda_device).contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        whole, parts = mod(x), torch.cat([mod(t) for t in x.split(40000)])
    # fp32 statistics of 24 values in two orders, on values of a few units
    assert (whole - parts).abs().max() <= 32 * torch.finfo(torch.float32).eps
    with pytest.raises(_lib.SparseSAMError):
        ops.groupnorm_act(x.permute(0, 2, 3, 1), 2, mod.weight, mod.bias)
