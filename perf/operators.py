"""The channels-last block operators as they are measured: GroupNorm with an activation, and the matrix product with bias, activation
and residual, each forward and backward.  `run` computes a case in its plain form (elementary torch operations in 32 bits, rounded
once) or, with `own` set, by the calls a user of dig_amd makes."""
import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ACTS = ("none", "relu", "gelu", "silu")


def listed():
    gn = dict(op="gn", dtype="bf16", act="silu", ss=True, res=False, bwd=False)
    lin = dict(op="linear", dtype="bf16", act="none", bias=True, res=False, bwd=False)
    return [
        # the bottom level of a 32x32 Unet with dim 16, one image: a sampling loop with batch 1, where the launch counts
        dict(gn, name="gn fwd 1x4x4x128", B=1, P=16, C=128, G=8),
        # block1 of the bottom level (32x32, 512 channels) of the 256x256 Unet at batch 32
        dict(gn, name="gn fwd 32x32x32x512", B=32, P=1024, C=512, G=8),
        # block2 of the top level of the same Unet, with the block's residual: the largest activations there are
        dict(gn, name="gn fwd 32x256x256x64 res", B=32, P=65536, C=64, G=8, ss=False, res=True),
        # backward of block1 of the third level (64x64, 256 channels), batch 32
        dict(gn, name="gn bwd 32x64x64x256", B=32, P=4096, C=256, G=8, bwd=True),
        # backward of the LFCA's GroupNorm(1, C) + ReLU on the patch grid of 368x496 images, fp32 as that branch is trained
        dict(gn, name="gn bwd f32 8x23x31x1024", dtype="f32", act="relu", B=8, P=713, C=1024, G=1, ss=False, bwd=True),
        # the class-token MLP of the LFCA for one image of 20 classes, fp32: the smallest product
        dict(lin, name="linear fwd f32 20x384x1536", dtype="f32", act="gelu", M=20, K=384, N=1536),
        # fc1 of a ViT block, 32 images of 20 class and 196 patch tokens
        dict(lin, name="linear fwd 6912x384x1536", act="gelu", M=6912, K=384, N=1536),
        # an 81-class head on 8 images of 733 tokens: few output columns, not a multiple of any vector
        dict(lin, name="linear fwd 5864x384x81", M=5864, K=384, N=81),
        # a wide product with its residual: bound by the matrix units
        dict(lin, name="linear fwd 8192x4096x4096 res", act="silu", M=8192, K=4096, N=4096, res=True),
        # backward of fc2 of a ViT block, 32 images
        dict(lin, name="linear bwd 6912x1536x384", M=6912, K=1536, N=384, bwd=True),
        # backward of the first 1x1 convolution of the LFCA's patch MLP (1024 -> 4096, GELU), 32 images of 14x14 patches
        dict(lin, name="linear bwd 6272x1024x4096", act="gelu", M=6272, K=1024, N=4096, bwd=True),
        # backward of fc1 in fp32, 8 images of 733 tokens
        dict(lin, name="linear bwd f32 5864x384x1536", dtype="f32", act="gelu", M=5864, K=384, N=1536, bwd=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    bwd, dtype, act = rng.random() < 0.5, rng.choice(("bf16", "f32")), rng.choice(ACTS)
    if rng.random() < 0.5:
        while True:
            G = rng.choice((1, 2, 4, 8, 8, 8, 16, 32))
            C = G * _log(rng, 1, 1024 // G)
            if rng.random() < 0.6:
                C = max(8, C // 8 * 8) // G * G or G
            B, P = _log(rng, 1, 32), _log(rng, 1, 65536)
            if P * (C // G) < 8:  # the gradient of a group of so few values is a difference of equal numbers
                continue
            if B * P * C * (2 if bwd else 1) * (2 if dtype == "f32" else 1) <= 32 * 65536 * 64:
                return dict(op="gn", dtype=dtype, act=act, ss=rng.random() < 0.5, res=not bwd and rng.random() < 0.5, bwd=bwd, B=B, P=P, C=C, G=G)
    while True:
        M, K, N = _log(rng, 1, 65536), _log(rng, 4, 4096), _log(rng, 4, 4096)
        if rng.random() < 0.6:
            K, N = max(8, K // 8 * 8), max(8, N // 8 * 8)
        if M * K * N * (2 if bwd else 1) <= 8192 * 4096 * 4096:
            return dict(op="linear", dtype=dtype, act=act, bias=rng.random() < 0.8, res=not bwd and rng.random() < 0.5, bwd=bwd, M=M, K=K, N=N)


def prepare(case, seed):
    c, dt = dict(case), DTYPES[case["dtype"]]
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rnd(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        t = torch.randn(*shape, generator=g, device=DEV)
        return t.mul_(scale).add_(shift).to(dtype)

    s = {"case": c}
    if c["op"] == "gn":
        B, P, C, G = c["B"], c["P"], c["C"], c["G"]
        # activations behind a convolution: every channel has a spread and an offset of its own
        spread, offset = rnd(C, scale=0.3).exp_(), rnd(C, scale=0.5)
        s["x"] = (torch.randn(B, P, C, generator=g, device=DEV).mul_(spread).add_(offset)).to(dt)
        s["gamma"], s["beta"] = rnd(C, scale=0.3, shift=1.0), rnd(C, scale=0.3)
        s["ss"] = rnd(B, 2 * C, scale=0.3) if c["ss"] else None  # (scale | shift) of the time embedding
        s["res"] = rnd(B, P, C, dtype=dt) if c["res"] else None
        if c["bwd"]:
            s["dy"] = rnd(B, P, C, scale=0.1, dtype=dt)
            # what the forward keeps: mean and 1 / sqrt(var + eps) of each image and group
            xg = s["x"].reshape(B, P, G, C // G).float()
            mean = xg.mean((1, 3))
            var = (xg - mean[:, None, :, None]).square().mean((1, 3))
            s["mean_rstd"] = torch.stack([mean, (var + 1e-5).rsqrt()], -1)
    else:
        M, K, N = c["M"], c["K"], c["N"]
        s["x"] = rnd(M, K, dtype=dt)
        s["w"] = rnd(N, K, scale=K ** -0.5, dtype=dt)
        s["bias"] = rnd(N, scale=0.3) if c["bias"] else None
        s["res"] = rnd(M, N, dtype=dt) if c["res"] else None
        if c["bwd"]:
            s["dy"] = rnd(M, N, scale=0.1, dtype=dt)
            # what the forward keeps: the pre-activation in the storage type
            s["pre"] = None
            if c["act"] != "none":
                z = s["x"].float() @ s["w"].float().t()
                s["pre"] = (z + s["bias"] if c["bias"] else z).to(dt)
    return s


def _act(u, act):
    if act == "relu":
        return torch.where(u > 0, u, torch.zeros_like(u))
    if act == "gelu":
        return 0.5 * u * (1 + torch.erf(u * math.sqrt(0.5)))
    if act == "silu":
        return u / (1 + torch.exp(-u))
    return u


def _act_grad(u, act):
    if act == "relu":
        return (u > 0).to(u.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(u * math.sqrt(0.5))) + u * torch.exp(-0.5 * u * u) * (1 / math.sqrt(2 * math.pi))
    if act == "silu":
        sg = 1 / (1 + torch.exp(-u))
        return sg * (1 + u * (1 - sg))
    return torch.ones_like(u)


def _affine(s, C):
    """per (image, channel) factors of the normalised value: u = a * xhat + b"""
    a, b, sc = s["gamma"][None], s["beta"][None], None
    if s["ss"] is not None:
        sc, sh = 1 + s["ss"][:, :C], s["ss"][:, C:]
        a, b = a * sc, b * sc + sh
    return a[:, None], b[:, None], sc


def _plain_gn(s):
    c = s["case"]
    B, P, C, G = c["B"], c["P"], c["C"], c["G"]
    x = s["x"].float().reshape(B, P, G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    xc = x - mean
    rstd = 1 / torch.sqrt((xc * xc).mean((1, 3), keepdim=True) + 1e-5)
    a, b, _ = _affine(s, C)
    y = _act((xc * rstd).reshape(B, P, C) * a + b, c["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    return {"y": y.to(s["x"].dtype), "mean_rstd": torch.stack([mean.reshape(B, G), rstd.reshape(B, G)], -1)}


def _plain_gn_bwd(s):
    c = s["case"]
    B, P, C, G = c["B"], c["P"], c["C"], c["G"]
    mean, rstd = s["mean_rstd"][..., 0].reshape(B, 1, G, 1), s["mean_rstd"][..., 1].reshape(B, 1, G, 1)
    xh = ((s["x"].float().reshape(B, P, G, C // G) - mean) * rstd).reshape(B, P, C)
    a, b, sc = _affine(s, C)
    if c["act"] == "relu":  # a gate: the side of zero that a value lies on is decided in 64 bits
        u = ((s["x"].double().reshape(B, P, G, C // G) - mean) * rstd.double()).reshape(B, P, C)
        a64, b64, _ = _affine({k: s[k].double() if s[k] is not None else None for k in ("gamma", "beta", "ss")}, C)
        gate = (u * a64 + b64 > 0).float()
    else:
        gate = _act_grad(xh * a + b, c["act"])
    du = s["dy"].float() * gate
    s1, s2 = du.sum(1), (du * xh).sum(1)
    ga = (du * a).reshape(B, P, G, C // G)
    m1 = ga.mean((1, 3), keepdim=True)
    m2 = (ga * xh.reshape(B, P, G, C // G)).mean((1, 3), keepdim=True)
    dx = rstd * (ga - m1 - xh.reshape(B, P, G, C // G) * m2)
    out = {"dx": dx.reshape(B, P, C).to(s["x"].dtype)}
    out["dgamma"], out["dbeta"] = ((s2, s1) if sc is None else (s2 * sc, s1 * sc))
    out["dgamma"], out["dbeta"] = out["dgamma"].sum(0), out["dbeta"].sum(0)
    if sc is not None:
        out["dss"] = torch.cat([s["gamma"] * s2 + s["beta"] * s1, s1], 1)
    return out


def _plain_linear(s):
    c = s["case"]
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"]
    y = _act(z, c["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    out = {"y": y.to(s["x"].dtype)}
    if c["act"] != "none":  # kept for the backward
        out["pre"] = z.to(s["x"].dtype)
    return out


def _plain_linear_bwd(s):
    c, dt = s["case"], s["x"].dtype
    dz = s["dy"].float()
    if c["act"] != "none":
        dz = dz * _act_grad(s["pre"].float(), c["act"])
    out = {"dx": (dz @ s["w"].float()).to(dt), "dw": (dz.t() @ s["x"].float()).to(dt)}
    if s["bias"] is not None:
        out["db"] = dz.sum(0)
    return out


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "gn":
            return _plain_gn_bwd(s) if c["bwd"] else _plain_gn(s)
        return _plain_linear_bwd(s) if c["bwd"] else _plain_linear(s)
    from dig_amd import ops, train
    if c["op"] == "gn":
        if c["bwd"]:
            dx, dgamma, dbeta, dss = train.group_norm_act_bwd(s["x"], s["mean_rstd"], s["gamma"], s["beta"], s["dy"], act=c["act"], ss=s["ss"])
            out = {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
            if dss is not None:
                out["dss"] = dss
            return out
        y, mean_rstd = ops.group_norm_act(s["x"], s["gamma"], s["beta"], groups=c["G"], act=c["act"], ss=s["ss"], res=s["res"], want_stats=True)
        return {"y": y, "mean_rstd": mean_rstd}
    if c["bwd"]:
        dx, dw, db = train.linear_act_bwd(s["x"], s["w"], s["dy"], pre=s["pre"], act=c["act"], has_bias=c["bias"])
        out = {"dx": dx, "dw": dw}
        if db is not None:
            out["db"] = db
        return out
    if c["act"] == "none":
        return {"y": ops.linear_act(s["x"], s["w"], bias=s["bias"], act=c["act"], res=s["res"])}
    y, pre = ops.linear_act(s["x"], s["w"], bias=s["bias"], act=c["act"], res=s["res"], want_pre=True)
    return {"y": y, "pre": pre}


def work(case):
    c, e = case, 2 if case["dtype"] == "bf16" else 4
    if c["op"] == "gn":
        B, C, n = c["B"], c["C"], c["B"] * c["P"] * c["C"]
        small = 2 * C * 4 + B * c["G"] * 8 + (B * 2 * C * 4 if c["ss"] else 0)
        if c["bwd"]:  # x, dy -> dx and the parameters' gradients
            return {"bytes": 3 * n * e + 2 * small, "flops": 25 * n}
        return {"bytes": (2 + c["res"]) * n * e + small, "flops": 12 * n}
    M, K, N, kept = c["M"], c["K"], c["N"], c["act"] != "none"
    if c["bwd"]:  # x, w, dy (and the pre-activation) -> dx, dw, db
        return {"bytes": (2 * M * K + 2 * N * K + (1 + kept) * M * N) * e + 4 * N * c["bias"], "flops": 4 * M * N * K}
    return {"bytes": (M * K + N * K + (1 + kept + c["res"]) * M * N) * e + 4 * N * c["bias"], "flops": 2 * M * N * K}


def exact(case, seed):
    """The same values from the operators' definitions in 64 bits: the normalised tensor image by image, the gradients by the chain
    rule through the mean and the variance written out, the products by float64 matmul."""
    s, c = prepare(case, seed), case
    f64 = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and (v.numel() < 1 << 22 or c["op"] == "linear")}
    slope = {"none": lambda v: torch.ones_like(v), "relu": lambda v: v.gt(0).double(),
             "gelu": lambda v: torch.special.ndtr(v) + v * torch.exp(-v.square() / 2) / math.sqrt(2 * math.pi),
             "silu": lambda v: torch.sigmoid(v) * (1 + v * torch.sigmoid(-v))}[c["act"]]
    value = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "gelu": lambda v: v * torch.special.ndtr(v), "silu": lambda v: v * torch.sigmoid(v)}[c["act"]]
    if c["op"] == "linear":
        if c["bwd"]:
            dz = f64["dy"] * slope(f64["pre"]) if "pre" in f64 else f64["dy"]
            out = {"dx": torch.matmul(dz, f64["w"]), "dw": torch.matmul(dz.transpose(0, 1).contiguous(), f64["x"])}
            return dict(out, db=dz.sum(0)) if c["bias"] else out
        z = torch.matmul(f64["x"], f64["w"].transpose(0, 1).contiguous()) + (f64["bias"] if c["bias"] else 0)
        out = {"y": value(z) + (f64["res"] if c["res"] else 0)}
        return out if c["act"] == "none" else dict(out, pre=z)
    B, P, C, G = c["B"], c["P"], c["C"], c["G"]
    n, gamma, beta = P * (C // G), f64["gamma"], f64["beta"]
    ys, st, dg, db, dss = [], [], torch.zeros_like(gamma), torch.zeros_like(gamma), []
    for i in range(B):
        x = s["x"][i].double()
        grow, shift = (1 + f64["ss"][i, :C], f64["ss"][i, C:]) if c["ss"] else (torch.ones_like(gamma), torch.zeros_like(gamma))
        if not c["bwd"]:
            mu = x.sum(0).view(G, -1).sum(1) / n
            centred = x - mu.repeat_interleave(C // G)
            r = (centred.square().sum(0).view(G, -1).sum(1) / n + 1e-5).pow(-0.5)
            y = value((centred * r.repeat_interleave(C // G) * gamma + beta) * grow + shift)
            ys.append(y + s["res"][i].double() if c["res"] else y)
            st.append(torch.stack([mu, r], 1))
            continue
        mu, r = (f64["mean_rstd"][i, :, k].repeat_interleave(C // G) for k in (0, 1))
        hat = (x - mu) * r
        du = s["dy"][i].double() * slope((hat * gamma + beta) * grow + shift)
        p1, p2 = du.sum(0), (du * hat).sum(0)
        dg += p2 * grow
        db += p1 * grow
        dss.append(torch.cat([gamma * p2 + beta * p1, p1]))
        q1, q2 = ((gamma * grow * p).view(G, -1).sum(1).repeat_interleave(C // G) / n for p in (p1, p2))
        ys.append((du * gamma * grow - q1 - hat * q2) * r)
    if not c["bwd"]:
        return {"y": torch.stack(ys), "mean_rstd": torch.stack(st)}
    out = {"dx": torch.stack(ys), "dgamma": dg, "dbeta": db}
    return dict(out, dss=torch.stack(dss)) if c["ss"] else out
