"""What the cross attention, GroupNorm and LayerNorm-gradient entry points refuse, on the host
(no kernel is launched; runs without a GPU)."""
import ctypes

import pytest
import torch

from sparsesam_b200 import _lib, ops

INV, ALIGN, UNSUP = _lib.SSAM_ERR_INVALID, _lib.SSAM_ERR_ALIGN, _lib.SSAM_ERR_UNSUPPORTED


def strides(v=64):
    return (ctypes.c_int64 * 12)(*([v] * 12))


def fwd(q=16, k=16, v=16, st=None, B=1, Tq=4, Tk=4, H=2, Hk=2, d=16, dtype=0, scale=0.25, out=16, out32=None):
    return _lib.load().ssam_cross_attn_fwd(q, k, v, strides() if st is None else st, B, Tq, Tk, H, Hk, d, dtype, scale,
                                           None, None, out, out32, None, None)


def bwd(q=16, dout=16, o32=16, lse=16, delta=16, dq=16, dk=16, dv=16, st=None, d=16, dtype=0):
    return _lib.load().ssam_cross_attn_bwd(q, 16, 16, dout, strides() if st is None else st, 1, 4, 4, 2, 2, d, dtype,
                                           0.25, None, None, o32, lse, delta, dq, dk, dv, None)


def test_cross_attention_abi():
    assert fwd(q=None) == INV and fwd(out=None) == INV
    for name in ("B", "Tq", "Tk", "H", "Hk", "d"):
        assert fwd(**{name: 0}) == INV and fwd(**{name: -1}) == INV
    assert fwd(H=3, Hk=2) == INV and fwd(dtype=3) == INV and fwd(dtype=-1) == INV
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert fwd(scale=scale) == INV
    for d in (4, 12, 136, 256):
        assert fwd(d=d) == UNSUP
    assert fwd(B=65536) == UNSUP
    assert fwd(q=8) == ALIGN and fwd(out=24) == ALIGN and fwd(out32=20) == ALIGN
    assert fwd(st=strides(12)) == ALIGN and fwd(st=strides(6), dtype=2) == ALIGN
    assert bwd(q=None) == INV and bwd(dout=None) == INV and bwd(o32=None, dtype=2) == INV and bwd(lse=None, dtype=2) == INV
    assert bwd(delta=None, dtype=2) == INV and bwd(dk=None) == INV and bwd(dv=None) == INV
    assert bwd(dout=8) == ALIGN and bwd(dq=8) == ALIGN and bwd(d=20) == UNSUP and bwd(st=strides(4)) == ALIGN
    uses = _lib.load().ssam_cross_attn_bwd_uses_stats
    assert uses(64, 16, 0) == 0 and uses(65, 16, 1) == 1 and uses(1, 16, 2) == 1 and uses(9, 72, 0) == 1 and uses(8, 128, 1) == 0
    assert bwd(dq=None, dk=None, dv=None) == 0          # nothing asked for: nothing launched


def gn(x=16, N=1, HW=4, C=16, G=2, w=16, act=0, dtype=0, out=16, mean=None, rstd=None, ws=16, n=1 << 20):
    return _lib.load().ssam_groupnorm_act_fwd(x, N, HW, C, G, w, 16, 1e-5, act, dtype, out, mean, rstd, ws, n, None)


def test_groupnorm_abi():
    lib = _lib.load()
    assert gn(x=None) == INV and gn(w=None) == INV and gn(out=None) == INV and gn(mean=16) == INV
    for name in ("N", "HW", "C", "G"):
        assert gn(**{name: 0}) == INV
    assert gn(C=16, G=3) == INV and gn(act=4) == INV and gn(dtype=3) == INV
    assert gn(C=12, G=2) == UNSUP and gn(C=2056, G=1) == UNSUP and gn(C=1028, G=1, dtype=2) == UNSUP
    assert gn(N=65536) == UNSUP
    big = dict(HW=1 << 22, C=64)                # too large for one cluster: the chunks' moments need a workspace
    need = lib.ssam_groupnorm_act_workspace_size(1, 1 << 22, 64, 2, 0, 0)
    assert need > 0 and lib.ssam_groupnorm_act_workspace_size(1, 4, 16, 2, 0, 0) == 0
    assert gn(ws=None, **big) == INV and gn(n=need - 1, **big) == INV
    assert gn(x=8) == ALIGN and gn(out=8) == ALIGN and gn(ws=8) == ALIGN
    assert lib.ssam_groupnorm_act_workspace_size(0, 4, 16, 2, 0, 0) == 0
    args = [16, 16, 1, 4, 16, 2, 16, 16, 16, 16, 0, 0, 16, 16, 16, 16, 1 << 20, None]
    for i in (0, 1, 6, 7, 8, 9, 12, 13, 14, 15):
        assert lib.ssam_groupnorm_act_bwd(*args[:i], None, *args[i + 1:]) == INV
    assert lib.ssam_groupnorm_act_bwd(*args[:12], 8, *args[13:]) == ALIGN


def test_layernorm_gradient_abi():
    lib = _lib.load()
    args = [16, 16, 4, 64, 16, 16, 1e-6, 0, 0, 16, 16, 16, 16, 1 << 20, None]
    for i in (0, 1, 4, 5, 9, 10, 11, 12):
        assert lib.ssam_layernorm_gelu_half_bwd(*args[:i], None, *args[i + 1:]) == INV
    assert lib.ssam_layernorm_gelu_half_bwd(*args[:3], 48, *args[4:]) == UNSUP
    assert lib.ssam_layernorm_gelu_half_bwd(*args[:8], 2, *args[9:]) == INV
    assert lib.ssam_layernorm_gelu_half_bwd(*args[:13], 8, None) == INV
    assert lib.ssam_layernorm_gelu_half_bwd(*args[:9], 8, *args[10:]) == ALIGN
    assert lib.ssam_layernorm_gelu_half_bwd_workspace_size(0, 64) == 0


def test_cpu_tensors_are_refused():
    t = torch.zeros(1, 4, 2, 16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.cross_attn(t, t, t)
    with pytest.raises(ValueError, match="CUDA"):
        ops.groupnorm_act(torch.zeros(1, 4, 16), 2, torch.ones(16), torch.zeros(16))
    with pytest.raises(ValueError, match="CUDA"):
        ops.layernorm_gelu_half(torch.zeros(4, 32).half(), torch.ones(32).half(), torch.zeros(32).half(), 1e-6, False)


# the device is checked last: these CPU tensors get as far as the fault that each case names
def fake(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("kwargs,error", [
    (dict(q=fake(1, 4, 32)), ValueError), (dict(k=fake(1, 5, 2, 16)), ValueError), (dict(q=fake(2, 4, 2, 16)), ValueError),
    (dict(q=fake(1, 4, 2, 32)), ValueError), (dict(q=fake(1, 4, 2, 16, dtype=torch.float32)), TypeError),
    (dict(q=fake(1, 4, 3, 16)), ValueError), (dict(q=fake(1, 16, 2, 4).transpose(1, 3)), ValueError),
    (dict(scale=0.0), ValueError), (dict(scale=float("nan")), ValueError), (dict(scale=-1.0), ValueError),
    (dict(key_lens=fake(1, dtype=torch.int64)), ValueError), (dict(key_lens=fake(2, dtype=torch.int32)), ValueError),
    (dict(key_mask=fake(1, 7, dtype=torch.bool)), ValueError), (dict(key_mask=fake(1, 6, dtype=torch.uint8)), ValueError),
])
def test_cross_attention_wrapper(kwargs, error):
    args = {"q": fake(1, 4, 2, 16), "k": fake(1, 6, 2, 16), "v": fake(1, 6, 2, 16), **kwargs}
    with pytest.raises(error) as e:
        ops.cross_attn(**args)
    assert "CUDA" not in str(e.value)


@pytest.mark.parametrize("kwargs,error", [
    (dict(groups=3), ValueError), (dict(groups=0), ValueError), (dict(act="tanh"), ValueError),
    (dict(w=fake(8)), ValueError), (dict(w=fake(16, dtype=torch.float32)), TypeError),
    (dict(x=fake(2, 16, 5).transpose(1, 2)), ValueError), (dict(x=fake(16)), ValueError),
])
def test_groupnorm_wrapper(kwargs, error):
    args = {"x": fake(2, 5, 16), "groups": 2, "w": fake(16), "b": fake(16), **kwargs}
    with pytest.raises(error) as e:
        ops.groupnorm_act(**args)
    assert "CUDA" not in str(e.value)


def test_sizes_past_32_bits():
    """More entries than the C entry points count: an error, not a size that has wrapped around."""
    q = torch.zeros(1, 1, 1, 8, dtype=torch.float16)
    for n in (2**31, 2**32 + 1):
        with pytest.raises(ValueError, match="entries"):
            ops.cross_attn(q.expand(1, n, 1, 8), q, q)
        with pytest.raises(ValueError, match="entries"):
            ops.cross_attn(q, q.expand(1, n, 1, 8), q.expand(1, n, 1, 8))
        with pytest.raises(ValueError, match="entries"):
            ops.groupnorm_act(q.expand(n, 1, 1, 8), 1, q[0, 0, 0], q[0, 0, 0])


def test_scale_whose_exponent_base_change_overflows():
    q = torch.zeros(1, 1, 1, 8, dtype=torch.float16)
    assert fwd(scale=2.5e38) == INV
    with pytest.raises(ValueError, match="scale"):
        ops.cross_attn(q, q, q, scale=2.5e38)
