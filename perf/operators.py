"""The mask decoder's operators, as cases that can be timed: cross attention between prompt
tokens and image tokens, group normalisation with an activation on channels-last maps, and the
channel LayerNorm (+ GELU) of the decoder's half-precision maps with its gradient.

`run` computes a case in plain torch operations, or, where `own` is true, by the calls of
sparsesam_b200.ops. `exact` gives the results from the definitions in 64 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
ACTS = ("none", "relu", "gelu", "silu")
MASKS = ("none", "lens", "mask")


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _attn(name, B, Tq, Tk, H, Hk, D, dtype, mask, train):
    c = {"op": "attn", "B": B, "Tq": Tq, "Tk": Tk, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "mask": mask,
         "train": train}
    return dict(c, name=name) if name else c


def _gn(name, N, H, W, C, G, dtype, act, train):
    c = {"op": "groupnorm", "N": N, "H": H, "W": W, "C": C, "G": G, "dtype": dtype, "act": act, "train": train}
    return dict(c, name=name) if name else c


def _ln(name, rows, C, dtype, gelu):
    c = {"op": "layernorm", "rows": rows, "C": C, "dtype": dtype, "gelu": gelu}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one box prompt on one 1024 x 1024 image: 6 output tokens + 2 box corners read the 64 x 64 image tokens
        # (8 heads of 16, the decoder's half-width cross attention); latency
        _attn("tokens_to_image_1", 1, 8, 4096, 8, 8, 16, "bf16", "none", False),
        # the evaluation step at batch 64: the same read for 64 images at once
        _attn("tokens_to_image_64", 64, 8, 4096, 8, 8, 16, "bf16", "none", False),
        # its counterpart at batch 64: every image token reads its image's few prompt tokens
        _attn("image_to_tokens_64", 64, 4096, 8, 8, 8, 16, "fp16", "none", False),
        # a single query (one point's token) over a 128 x 128 grid, key heads shared by pairs of query heads
        _attn("one_query_long", 1, 1, 16384, 8, 4, 32, "fp16", "none", False),
        # training the decoder in bf16: token reads with their gradients, image padding cut off by key lengths
        _attn("train_tokens_to_image", 8, 11, 4096, 8, 8, 16, "bf16", "lens", True),
        # training the decoder in fp32: image tokens read a padded, masked batch of prompt tokens
        _attn("train_image_to_tokens_fp32", 4, 4096, 13, 8, 8, 16, "fp32", "mask", True),
        # many object queries on a 64 x 64 grid at full head width, with gradients: the arithmetic-bound end
        _attn("train_queries_long", 2, 1369, 4096, 4, 4, 64, "bf16", "none", True),
        # a segmentation head's pixel map of one image: latency
        _gn("groupnorm_one_map", 1, 64, 64, 256, 8, "bf16", "relu", False),
        # upscaled maps of a training batch, with gradients
        _gn("train_groupnorm_maps", 16, 256, 256, 64, 8, "bf16", "gelu", True),
        # an odd crop in fp32, with gradients
        _gn("train_groupnorm_odd_fp32", 3, 67, 45, 96, 4, "fp32", "silu", True),
        # the image tokens' LayerNorm of one training image
        _ln("train_layernorm_tokens", 4096, 256, "bf16", False),
        # LayerNorm + GELU of the upscaled maps, batch 16 at 128 x 128
        _ln("train_layernorm_gelu_maps", 262144, 64, "fp16", True),
    ]


MOST_BYTES = 540e6
MOST_FLOPS = 30e9


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return c


def _draw(rng):
    kind = rng.choice(("tokens", "image", "single", "long", "gn", "gn", "ln"))
    dtype = rng.choice(("bf16", "fp16", "bf16", "fp16", "fp32"))
    if kind in ("tokens", "image", "single", "long"):
        B = _log_int(rng, 1, 64)
        H = rng.choice((2, 4, 8, 12))
        Hk = rng.choice((H, H, H, H // 2))
        D = rng.choice((16, 16, 32, 32, 64))
        mask = rng.choice(MASKS)
        train = rng.random() < 0.5
        if kind == "tokens":
            Tq, Tk = rng.randint(2, 40), _log_int(rng, 256, 16384)
        elif kind == "image":
            Tq, Tk = _log_int(rng, 256, 16384), rng.randint(2, 64)
        elif kind == "single":
            Tq, Tk, train = 1, _log_int(rng, 64, 65536), False
        else:
            Tq, Tk = _log_int(rng, 65, 2048), _log_int(rng, 65, 4096)
            B = rng.randint(1, 4)
        return _attn(None, B, Tq, Tk, H, Hk, D, dtype, mask, train)
    if kind == "gn":
        C = rng.choice((32, 64, 96, 128, 192, 256, 320, 512))
        G = rng.choice([g for g in (1, 4, 8, 16, 32) if C % g == 0])
        return _gn(None, _log_int(rng, 1, 32), _log_int(rng, 7, 256), _log_int(rng, 7, 256), C, G, dtype,
                   rng.choice(ACTS), rng.random() < 0.5)
    return _ln(None, _log_int(rng, 64, 300000), rng.choice((32, 64, 128, 256)), rng.choice(("bf16", "fp16")),
               rng.random() < 0.5)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale + shift).to(dt)

    s = {"case": dict(case)}
    if case["op"] == "attn":
        B, Tq, Tk, H, Hk, D = (case[n] for n in ("B", "Tq", "Tk", "H", "Hk", "D"))
        # projections of unit-variance states: (B, T, heads * D) rows, viewed as heads
        s["q"] = rand(B, Tq, H * D).view(B, Tq, H, D)
        s["k"] = rand(B, Tk, Hk * D).view(B, Tk, Hk, D)
        s["v"] = rand(B, Tk, Hk * D).view(B, Tk, Hk, D)
        s["lens"] = s["mask"] = None
        if case["mask"] == "lens":       # at least half of the keys are there; in a batch, one entry has none
            lens = torch.randint((Tk + 1) // 2, Tk + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32)
            if B > 2:
                lens[B // 2] = 0
            s["lens"] = lens
        elif case["mask"] == "mask":     # three keys of four on average
            s["mask"] = torch.rand(B, Tk, generator=g, device=DEVICE) < 0.75
        if case["train"]:
            s["dout"] = rand(B, Tq, H * D).view(B, Tq, H, D)
            s["leaves"] = [s[n].requires_grad_(True) for n in ("q", "k", "v")]
    elif case["op"] == "groupnorm":
        N, H, W, C = (case[n] for n in ("N", "H", "W", "C"))
        s["x"] = rand(N, H, W, C, scale=1.5, shift=0.5)
        s["w"], s["b"] = rand(C, scale=0.3, shift=1.0), rand(C, scale=0.3)
        if case["train"]:
            s["dout"] = rand(N, H, W, C)
            s["leaves"] = [s[n].requires_grad_(True) for n in ("x", "w", "b")]
    else:
        rows, C = case["rows"], case["C"]
        s["x"] = rand(rows, C, scale=1.5, shift=0.5)
        s["w"], s["b"] = rand(C, scale=0.3, shift=1.0), rand(C, scale=0.3)
        s["dout"] = rand(rows, C)
        s["leaves"] = [s[n].requires_grad_(True) for n in ("x", "w", "b")]
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        from sparsesam_b200 import ops
        if c["op"] == "attn":
            out = ops.cross_attn(s["q"], s["k"], s["v"], key_lens=s["lens"], key_mask=s["mask"])
        elif c["op"] == "groupnorm":
            out = ops.groupnorm_act(s["x"], c["G"], s["w"], s["b"], 1e-5, c["act"])
        else:
            out = ops.layernorm_gelu_half(s["x"], s["w"], s["b"], 1e-6, c["gelu"])
        if "dout" not in s:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, s["leaves"], s["dout"])]
    with torch.no_grad():
        if c["op"] == "attn":
            return _plain_attn(s["q"], s["k"], s["v"], s["lens"], s["mask"], s.get("dout"))
        if c["op"] == "groupnorm":
            x = s["x"]
            x4 = x.reshape(c["N"], c["H"] * c["W"], c["G"], c["C"] // c["G"])
            return _plain_norm(x, x4, (1, 3), s["w"], s["b"], 1e-5, c["act"], s.get("dout"))
        return _plain_norm(s["x"], s["x"].view(-1, 1, 1, c["C"]), (1, 3), s["w"], s["b"], 1e-6,
                           "gelu" if c["gelu"] else "none", s["dout"])


def _heads(t, group=1):
    t = t.float().transpose(1, 2)
    return t if group == 1 else t.repeat_interleave(group, dim=1)


def _plain_attn(q, k, v, lens, mask, dout):
    dt, group = q.dtype, q.shape[2] // k.shape[2]
    scale = 1.0 / math.sqrt(q.shape[3])
    qf, kf, vf = _heads(q), _heads(k, group), _heads(v, group)
    scores = torch.matmul(qf, kf.transpose(2, 3)) * scale
    if lens is not None:
        mask = torch.arange(k.shape[1], device=q.device)[None, :] < lens[:, None]
    if mask is not None:
        scores = torch.where(mask[:, None, None, :], scores, -math.inf)
    top = scores.amax(dim=3, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(dim=3, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, vf).transpose(1, 2).to(dt)
    if dout is None:
        return [out]
    do = _heads(dout)
    dv = torch.matmul(p.transpose(2, 3), do)
    dp = torch.matmul(do, vf.transpose(2, 3))
    ds = p * (dp - (p * dp).sum(dim=3, keepdim=True)) * scale
    dq = torch.matmul(ds, kf)
    dk = torch.matmul(ds.transpose(2, 3), qf)
    if group > 1:
        dk, dv = dk.unflatten(1, (-1, group)).sum(2), dv.unflatten(1, (-1, group)).sum(2)
    return [out, *(t.transpose(1, 2).to(dt) for t in (dq, dk, dv))]


def _plain_norm(x, x4, dims, w, b, eps, act, dout):
    """Normalisation of x over `dims` of its 4-D view x4 (samples, positions, groups, channels of a group)."""
    wf, bf = w.float().view(x4.shape[2:]), b.float().view(x4.shape[2:])
    xf = x4.float()
    mean = xf.mean(dim=dims, keepdim=True)
    xc = xf - mean
    rstd = torch.rsqrt((xc * xc).mean(dim=dims, keepdim=True) + eps)
    xh = xc * rstd
    z = xh * wf + bf
    if act == "relu":
        y = torch.clamp(z, min=0.0)
    elif act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        y = z * cdf
    elif act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        y = z * sig
    else:
        y = z
    out = y.to(x.dtype).view(x.shape)
    if dout is None:
        return [out]
    gz = dout.reshape(x4.shape).float()
    if act == "relu":
        gz = torch.where(z > 0, gz, 0.0)
    elif act == "gelu":
        gz = gz * (cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)))
    elif act == "silu":
        gz = gz * (sig * (1.0 + z * (1.0 - sig)))
    gx = gz * xh
    db, dw = gz.sum(dim=(0, 1)).view(-1).to(b.dtype), gx.sum(dim=(0, 1)).view(-1).to(w.dtype)
    m1 = (gz * wf).mean(dim=dims, keepdim=True)
    m2 = (gx * wf).mean(dim=dims, keepdim=True)
    dx = (rstd * (gz * wf - m1 - xh * m2)).to(x.dtype).view(x.shape)
    return [out, dx, dw, db]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = SIZES[case["dtype"]]
    if case["op"] == "attn":
        B, Tq, Tk, H, Hk, D = (case[n] for n in ("B", "Tq", "Tk", "H", "Hk", "D"))
        share = {"none": 1.0, "lens": 0.75, "mask": 0.75}[case["mask"]]
        rows, keys = B * Tq * H * D * e, B * Tk * Hk * D * e
        pairs = B * H * Tq * Tk * share
        if case["train"]:    # q, dout read, out, dq written; k, v read where they count, dk, dv written
            return {"bytes": 4 * rows + (2 * share + 2) * keys, "flops": 12.0 * D * pairs}
        return {"bytes": 2 * rows + 2 * share * keys, "flops": 4.0 * D * pairs}
    if case["op"] == "groupnorm":
        n = case["N"] * case["H"] * case["W"] * case["C"]
        train = case["train"]
    else:
        n, train = case["rows"] * case["C"], True
    return {"bytes": (4 if train else 2) * n * e + (4 if train else 2) * case["C"] * e,
            "flops": (30.0 if train else 10.0) * n}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attn":
            return _exact_attn(s)
        return _exact_norm(s)


def _exact_attn(s):
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    q = q.view(B, Tq, Hk, H // Hk, D)
    keep = torch.ones(B, Tk, dtype=torch.bool, device=q.device)
    if s["lens"] is not None:
        keep &= torch.arange(Tk, device=q.device) < s["lens"].view(B, 1)
    if s["mask"] is not None:
        keep &= s["mask"]
    a = torch.einsum("bqhgd,bkhd->bhgqk", q, k).mul_(D ** -0.5)
    a.masked_fill_(~keep.view(B, 1, 1, 1, Tk), -math.inf)
    p = torch.softmax(a, dim=-1).nan_to_num_(0.0)      # a row without keys: zeros
    del a
    out = torch.einsum("bhgqk,bkhd->bqhgd", p, v).reshape(B, Tq, H, D)
    if "dout" not in s:
        return [out]
    do = s["dout"].double().view(B, Tq, Hk, H // Hk, D)
    dv = torch.einsum("bhgqk,bqhgd->bkhd", p, do)
    dp = torch.einsum("bqhgd,bkhd->bhgqk", do, v)
    da = p * (dp - torch.einsum("bhgqk,bhgqk->bhgq", p, dp).unsqueeze(-1))
    dq = torch.einsum("bhgqk,bkhd->bqhgd", da, k).mul_(D ** -0.5).reshape(B, Tq, H, D)
    dk = torch.einsum("bhgqk,bqhgd->bkhd", da, q).mul_(D ** -0.5)
    return [out, dq, dk, dv]


def _exact_norm(s):
    c = s["case"]
    C, group = c["C"], c["C"] // c.get("G", 1)
    x = s["x"].detach().double().view(c["N"] if c["op"] == "groupnorm" else c["rows"], -1, C)
    w, b = s["w"].detach().double(), s["b"].detach().double()
    act = c["act"] if c["op"] == "groupnorm" else ("gelu" if c["gelu"] else "none")
    eps = 1e-5 if c["op"] == "groupnorm" else 1e-6
    n = x.shape[1] * group

    def per_group(t):     # sums over a sample's positions and a group's channels, spread over the channels
        return t.sum(1).view(x.shape[0], C // group, group).sum(2).repeat_interleave(group, 1).unsqueeze(1)

    d = x - per_group(x) / n
    inv = (per_group(d * d) / n + eps).pow(-0.5)
    t = d * inv
    z = t * w + b
    if act == "relu":
        y, slope = z.clamp_min(0), (z > 0).double()
    elif act == "gelu":
        phi = torch.special.ndtr(z)
        y, slope = z * phi, phi + z * torch.exp(z * z / -2) / math.sqrt(2 * math.pi)
    elif act == "silu":
        sg = torch.sigmoid(z)
        y, slope = z * sg, sg + z * sg * (1 - sg)
    else:
        y, slope = z, torch.ones_like(z)
    out = y.view(s["x"].shape)
    if "dout" not in s:
        return [out]
    g = s["dout"].double().view(x.shape) * slope
    h = g * w
    dx = (h - per_group(h) / n - t * (per_group(h * t) / n)) * inv
    return [out, dx.view(s["x"].shape), (g * t).sum((0, 1)), g.sum((0, 1))]
