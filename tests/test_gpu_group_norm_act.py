"""GPU tier (-m gpu): ops.group_norm_act / train.group_norm_act_bwd (csrc/gnorm.hip) against the definition in 64 bits.

Tolerances, elementwise and derived from the operations (U = 2^-24, half a step of fp32; a value stored in bf16 adds half a step of bf16,
2^-8 of it):
 * u = (x - mean) rstd a + b: mean and rstd are within a few U of their value, so u is within 8 U (|xhat a| + |b|) + 4 U |mean| rstd |a|
   (the rounding of mean is amplified by rstd a);
 * act(u): its slope is at most 1.13; exp2 / rcp / erf are good to 2 ulps, exp's argument to |u| U, which is relative in the result;
 * statistics: a thread sums at most 64 rows of one channel here, about its own first sample: (64 + 16) U of the variance, half of
   that of rstd; across threads fp64;
 * sums over pixels: at most 64 fp32 additions in a thread, then fp64: (64 + 16) U of the sum of magnitudes, plus the summands' own error."""
import math

import pytest
import torch

from dig_amd import ops, train

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield


def rnd(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(DEV)


def act64(u, act):
    return {"none": u, "relu": torch.where(u < 0, torch.zeros_like(u), u), "gelu": u * torch.special.ndtr(u), "silu": u * torch.sigmoid(u)}[act]


def slope64(u, act):
    if act == "gelu":
        return torch.special.ndtr(u) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        return torch.sigmoid(u) * (1 + u * torch.sigmoid(-u))
    return (u > 0).double() if act == "relu" else torch.ones_like(u)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(B, P, C, dtype, seed, ss=True, shift=0.5, spread=1.0):
    x = (rnd(B, P, C, seed=seed) * (spread * rnd(C, seed=seed + 1, scale=0.3).exp()) + rnd(C, seed=seed + 2, scale=shift)).to(dtype)
    gamma, beta = rnd(C, seed=seed + 3, scale=0.3, shift=1.0), rnd(C, seed=seed + 4, scale=0.3)
    return x, gamma, beta, (rnd(B, 2 * C, seed=seed + 5, scale=0.3) if ss else None)


def stats64(x, G, eps=EPS):
    B, C = x.shape[0], x.shape[-1]
    g = x.double().reshape(B, -1, G, C // G)
    mean = g.mean((1, 3))
    var = (g - mean[:, None, :, None]).square().mean((1, 3))
    return mean, (var + eps).rsqrt()


def factors(gamma, beta, ss, ss_off=0):
    a, b, C = gamma.double()[None], beta.double()[None], gamma.numel()
    sc = torch.ones_like(a)
    if ss is not None:
        sc, sh = 1 + ss[:, ss_off:ss_off + C].double(), ss[:, ss_off + C:ss_off + 2 * C].double()
        a, b = a * sc, b * sc + sh
    return a[:, None], b[:, None], sc


def check_fwd(x, gamma, beta, G, act, ss=None, res=None, ss_off=0):
    y, mr = ops.group_norm_act(x, gamma, beta, groups=G, act=act, ss=ss, ss_off=ss_off, res=res, want_stats=True)
    B, C = x.shape[0], x.shape[-1]
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous() and mr.shape == (B, G, 2) and mr.dtype == torch.float32
    mean, r = stats64(x, G)
    big = x.double().abs().amax()
    assert float(((mr[..., 0].double() - mean).abs() - 8 * U * big).max()) <= 0, "mean"
    # variance: 80 U of it, plus what the rounding of the partial means (2 U of |x|) adds to the squares
    tol_r = r * (40 * U + 4 * (U * big * r) ** 2 + 8 * U * U)
    assert float(((mr[..., 1].double() - r).abs() - tol_r).max()) <= 0, "rstd"
    rep = lambda t: t.repeat_interleave(C // G, 1)[:, None]  # noqa: E731
    x3 = x.double().reshape(B, -1, C)
    a, b, _ = factors(gamma, beta, ss, ss_off)
    xh = (x3 - rep(mean)) * rep(r)
    u = xh * a + b
    ref = act64(u, act)
    # 40 U: the tolerance of rstd itself
    tol = 1.13 * U * (50 * (xh * a).abs() + 8 * b.abs() + 12 * big * rep(r) * a.abs()) + U * (8 + 2 * u.abs()) * ref.abs()
    if res is not None:
        ref = ref + res.double().reshape(B, -1, C)
    tol = tol + U * ref.abs() + (half_step(x.dtype) * (ref.abs() + tol) if x.dtype != torch.float32 else 0)
    err = (y.double().reshape(B, -1, C) - ref).abs()
    assert float((err - tol).max()) <= 0, (float(err.max()), float((err / tol).max()))
    return y, mr


def grads64(x, mr, gamma, beta, dy, act, ss, ss_off=0):
    """(dx, dgamma, dbeta, dss) by the formulas, from the stored mean and rstd, with an elementwise tolerance of each"""
    B, C, G = x.shape[0], x.shape[-1], mr.shape[1]
    rep = lambda t: t.double().repeat_interleave(C // G, 1)[:, None]  # noqa: E731
    mean, r = rep(mr[..., 0]), rep(mr[..., 1])
    a, b, sc = factors(gamma, beta, ss, ss_off)
    d = dy.double().reshape(B, -1, C)
    xc = x.double().reshape(B, -1, C) - mean
    xh = xc * r
    u = xh * a + b
    du = d * slope64(u, act)
    # |act''| <= 0.8; the slope's own functions: 8 + 4 |u| ulps of at most 1.13
    du_tol = d.abs() * U * (0.8 * (8 * (xh * a).abs() + 8 * b.abs()) + 1.13 * (8 + 4 * u.abs())) if act in ("gelu", "silu") else d.abs() * U
    s1, s2 = du.sum(1), (du * xh).sum(1)
    t1 = (80 * U * du.abs() + du_tol).sum(1)
    t2 = ((84 * U * du.abs() + du_tol) * xh.abs()).sum(1)
    grp = lambda t: t.reshape(B, -1, G, C // G)  # noqa: E731
    n = xh.shape[1] * (C // G)
    gmean = lambda t: (t[:, None] * a).reshape(B, G, C // G).sum(-1) / n  # noqa: E731
    m1, m2 = rep(gmean(s1)), rep(gmean(s2))
    am = lambda t: rep((t[:, None] * a.abs()).reshape(B, G, C // G).sum(-1) / n)  # noqa: E731
    dx = r * (du * a - m1 - xh * m2)
    dx_tol = r * (du_tol * a.abs() + 6 * U * ((du * a).abs() + m1.abs() + 2 * (xh * m2).abs()) + am(t1) + xh.abs() * am(t2)) + 4 * U * dx.abs()
    if x.dtype != torch.float32:
        dx_tol = dx_tol + half_step(x.dtype) * (dx.abs() + dx_tol)
    out = [(dx.reshape(x.shape), dx_tol.reshape(x.shape)), ((s2 * sc).sum(0), (t2 * sc.abs() + 4 * U * (s2 * sc).abs()).sum(0)),
           ((s1 * sc).sum(0), (t1 * sc.abs() + 4 * U * (s1 * sc).abs()).sum(0))]
    if ss is not None:
        g, be = gamma.double(), beta.double()
        out.append((torch.cat([g * s2 + be * s1, s1], 1),
                    torch.cat([g.abs() * t2 + be.abs() * t1 + 4 * U * ((g * s2).abs() + (be * s1).abs()), t1 + U * s1.abs()], 1)))
    return out


def check_bwd(x, mr, gamma, beta, dy, act, ss=None, ss_off=0):
    got = train.group_norm_act_bwd(x, mr, gamma, beta, dy, act=act, ss=ss, ss_off=ss_off)
    assert got[0].dtype == x.dtype and got[0].shape == x.shape and got[0].is_contiguous() and (got[3] is None) == (ss is None)
    for name, g, (ref, tol) in zip(("dx", "dgamma", "dbeta", "dss"), got, grads64(x, mr, gamma, beta, dy, act, ss, ss_off)):
        assert g.shape == ref.shape, name
        err = (g.double() - ref).abs()
        assert float((err - tol - 1e-37).max()) <= 0, (name, float(err.max()), float((err / (tol + 1e-37)).max()))
    return got


SHAPES = [  # B, P, C, G
    (1, 1, 8, 1), (2, 1, 64, 8), (1, 16, 128, 8), (3, 37, 40, 5), (2, 100, 24, 8), (2, 49, 7, 7), (3, 65, 30, 6), (1, 300, 1, 1), (2, 33, 81, 3), (1, 2049, 64, 8),
    (4, 196, 384, 6), (2, 713, 1024, 1), (5, 64, 512, 8), (1, 9, 2056, 1), (2, 5, 4104, 9), (1, 6, 600, 600), (2, 1500, 16, 16), (1, 40, 1027, 13), (33, 4, 32, 8),
    (2, 1024, 512, 8), (1, 4096, 256, 8)]


@pytest.mark.parametrize("B,P,C,G", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_shapes(B, P, C, G, dtype):
    for i, act in enumerate(("none", "relu", "gelu", "silu")):
        x, gamma, beta, ss = make(B, P, C, dtype, seed=10 * i, ss=i % 2 == 1)
        res = rnd(B, P, C, seed=99 + i, dtype=dtype) if i >= 2 else None
        check_fwd(x, gamma, beta, G, act, ss=ss, res=res)


@pytest.mark.parametrize("B,P,C,G", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_shapes(B, P, C, G, dtype):
    for i, act in enumerate(("none", "relu", "gelu", "silu")):
        x, gamma, beta, ss = make(B, P, C, dtype, seed=10 * i + 3, ss=i % 2 == 0)
        _, mr = ops.group_norm_act(x, gamma, beta, groups=G, act=act, ss=ss, want_stats=True)
        check_bwd(x, mr, gamma, beta, rnd(B, P, C, seed=77 + i, dtype=dtype), act, ss=ss)


@pytest.mark.parametrize("B,P,C,G", [(64, 1500, 64, 8), (100, 3000, 64, 8), (200, 2100, 24, 3), (130, 700, 48, 3), (7, 700, 48, 3), (260, 40, 8, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_images(B, P, C, G, dtype):
    """batches whose backward gives a block a whole image, beside small ones of the same images"""
    x, gamma, beta, ss = make(B, P, C, dtype, seed=B + P)
    dy = rnd(B, P, C, seed=B, dtype=dtype)
    for act in ("silu", "relu"):
        _, mr = check_fwd(x, gamma, beta, G, act, ss=ss)
        check_bwd(x, mr, gamma, beta, dy, act, ss=ss)
    check_bwd(x[:3], mr[:3].contiguous(), gamma, beta, dy[:3], "gelu", ss=ss[:3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    """channel slices of a wider tensor (aligned and not), every second image, a broadcast dy, ss rows inside a wider table"""
    B, P, C, G = 3, 50, 48, 6
    wide = rnd(2 * B, P, 2 * C + 3, seed=1, dtype=dtype)
    _, gamma, beta, _ = make(1, 1, C, dtype, seed=4)
    table = rnd(B, 5 + 2 * C + 2, seed=6, scale=0.3)
    aligned = rnd(2 * B, P, 2 * C, seed=2, dtype=dtype)
    for x in (wide[::2, :, 3:3 + C], wide[::2, :, C:2 * C], aligned[::2, :, C:], aligned[1::2, :, :C], wide[::2, 7:8, :C]):
        res = aligned[::2, :x.shape[1], 8:8 + C]
        _, mr = check_fwd(x, gamma, beta, G, "silu", ss=table, ss_off=5, res=res)
        check_bwd(x, mr, gamma, beta, res, "gelu", ss=table, ss_off=5)
        check_bwd(x, mr, gamma, beta, rnd(1, 1, C, seed=8, dtype=dtype).expand(x.shape), "silu")
    x4 = rnd(2, 6, 7, 2 * C, seed=3, dtype=dtype)[..., :C]  # [B, H, W, C] with one row pitch
    _, mr = check_fwd(x4, gamma, beta, G, "relu")
    check_bwd(x4, mr, gamma, beta, rnd(2, 6, 7, C, seed=5, dtype=dtype), "relu")


def test_statistics_far_from_zero():
    """a mean 1000 spreads away from zero, and a first sample far off its group: no digits lost to the squares"""
    x, gamma, beta, _ = make(2, 777, 64, torch.float32, seed=1, ss=False, shift=0.0)
    check_fwd(x + 1000.0, gamma, beta, 8, "none")
    x[:, 0] = 300.0
    check_fwd(x, gamma, beta, 8, "silu")


def test_constant_input():
    """zero variance: rstd = eps^-1/2, y = act(beta'), and a gradient of xhat = 0"""
    x = torch.full((2, 33, 16), 3.25, device=DEV)
    gamma, beta = rnd(16, seed=1), rnd(16, seed=2)
    y, mr = check_fwd(x, gamma, beta, 4, "silu")
    assert torch.equal(mr[..., 0], torch.full((2, 4), 3.25, device=DEV))
    check_bwd(x, mr, gamma, beta, rnd(2, 33, 16, seed=3), "silu")


def test_one_value_per_group_has_no_gradient():
    x, gamma, beta, ss = make(4, 1, 24, torch.float32, seed=2)
    _, mr = ops.group_norm_act(x, gamma, beta, groups=24, act="silu", ss=ss, want_stats=True)
    dx = train.group_norm_act_bwd(x, mr, gamma, beta, rnd(4, 1, 24, seed=5), act="silu", ss=ss)[0]
    assert torch.equal(dx, torch.zeros_like(dx))


def test_relu_gate_on_the_border():
    """u within rounding distance of zero: the gate is the sign in 64 bits, in every pass"""
    B, P, C, G = 2, 400, 32, 4
    x, gamma, beta, ss = make(B, P, C, torch.float32, seed=7)
    mean, r = stats64(x, G)
    a, b, _ = factors(gamma, beta, ss)
    rep = lambda t: t.repeat_interleave(C // G, 1)[:, None]  # noqa: E731
    mr = torch.stack([mean, r], -1).float().contiguous()
    edge = (rep(mr[..., 0].double()) - b / a / rep(mr[..., 1].double())).float()  # u = 0 up to the rounding of x
    steps = torch.arange(P, device=DEV)[None, :, None] % 5 - 2
    x = edge.expand(B, P, C) * (1 + steps * 2.0 ** -23)
    check_bwd(x, mr, gamma, beta, rnd(B, P, C, seed=8), "relu", ss=ss)


def test_gradient_against_differences():
    """directional derivatives of L = sum(dy * y) of the 64-bit forward (central differences, h = 1e-5: 1e-9 of truncation, 1e-10 of
    rounding) in every input"""
    B, P, C, G = 2, 21, 24, 4
    for act in ("gelu", "silu", "none"):
        x, gamma, beta, ss = make(B, P, C, torch.float32, seed=20)
        dy = rnd(B, P, C, seed=31)
        _, mr = ops.group_norm_act(x, gamma, beta, groups=G, act=act, ss=ss, want_stats=True)
        got = train.group_norm_act_bwd(x, mr, gamma, beta, dy, act=act, ss=ss)

        def loss(xx, ga, be, s):
            mean, r = stats64(xx, G)
            a, b, _ = factors(ga, be, s)
            xh = (xx.double() - mean.repeat_interleave(C // G, 1)[:, None]) * r.repeat_interleave(C // G, 1)[:, None]
            return float((act64(xh * a + b, act) * dy.double()).sum())

        ins = [t.double() for t in (x, gamma, beta, ss)]
        for i, g in enumerate(got):
            v = rnd(*ins[i].shape, seed=40 + i).double()
            hi, lo = ([t + s * 1e-5 * v if j == i else t for j, t in enumerate(ins)] for s in (1, -1))
            diff = (loss(*hi) - loss(*lo)) / 2e-5
            scale = float((g.double().abs() * v.abs()).sum())
            assert abs(diff - float((g.double() * v).sum())) <= 400 * U * scale + 1e-6, (act, i)


def test_nan_and_inf_stay_in_their_group():
    x, gamma, beta, _ = make(2, 40, 32, torch.float32, seed=5, ss=False)
    clean, mr0 = ops.group_norm_act(x, gamma, beta, groups=4, act="silu", want_stats=True)
    for bad in (float("nan"), float("inf")):
        xb = x.clone()
        xb[1, 3, 9] = bad  # image 1, group 1
        y, mr = ops.group_norm_act(xb, gamma, beta, groups=4, act="silu", want_stats=True)
        keep = torch.ones_like(x, dtype=torch.bool)
        keep[1, :, 8:16] = False
        assert torch.equal(y[keep], clean[keep]) and not torch.isfinite(y[1, :, 8:16]).any()
        assert torch.isnan(ops.group_norm_act(xb, gamma, beta, groups=4, act="relu")[1, 3, 9])


def test_empty():
    gamma, beta, ss = rnd(16, seed=1), rnd(16, seed=2), rnd(3, 32, seed=3)
    for B, P in ((0, 5), (3, 0)):
        x = torch.empty(B, P, 16, device=DEV)
        y, mr = ops.group_norm_act(x, gamma, beta, groups=4, ss=ss[:B], want_stats=True)
        assert y.shape == x.shape and mr.shape == (B, 4, 2)
        dx, dg, db, dss = train.group_norm_act_bwd(x, mr, gamma, beta, x, ss=ss[:B])
        assert dx.shape == x.shape and not dg.any() and not db.any() and not dss.any()


def test_batch_invariant_and_reproducible():
    """an image's results are the same bits alone and inside a batch, and from call to call"""
    for B, P, C, G in ((6, 1024, 512, 8), (5, 70, 24, 3), (3, 9000, 64, 8)):
        x, gamma, beta, ss = make(B, P, C, torch.bfloat16, seed=3)
        dy = rnd(B, P, C, seed=9, dtype=torch.bfloat16)
        y, mr = ops.group_norm_act(x, gamma, beta, groups=G, ss=ss, want_stats=True)
        dx, dg, db, dss = train.group_norm_act_bwd(x, mr, gamma, beta, dy, ss=ss)
        again = train.group_norm_act_bwd(x, mr, gamma, beta, dy, ss=ss)
        assert all(torch.equal(p, q) for p, q in zip((dx, dg, db, dss), again))
        y1, mr1 = ops.group_norm_act(x[1:2], gamma, beta, groups=G, ss=ss[1:2], want_stats=True)
        d1 = train.group_norm_act_bwd(x[1:2], mr1, gamma, beta, dy[1:2], ss=ss[1:2])
        assert torch.equal(y1, y[1:2]) and torch.equal(mr1, mr[1:2]) and torch.equal(d1[0], dx[1:2]) and torch.equal(d1[3], dss[1:2])


def test_large_offsets():
    """element offsets past 2^31: the last image of a 4.3 GB tensor"""
    B, P, C, G = 33, 1 << 20, 64, 8
    x = torch.empty(B, P, C, dtype=torch.bfloat16, device=DEV).normal_()
    gamma, beta = rnd(C, seed=1), rnd(C, seed=2)
    y, mr = ops.group_norm_act(x, gamma, beta, groups=G, act="silu", want_stats=True)
    y1, mr1 = ops.group_norm_act(x[-1:].clone(), gamma, beta, groups=G, act="silu", want_stats=True)
    assert torch.equal(y[-1:], y1) and torch.equal(mr[-1:], mr1)
    del y, y1
    dx = train.group_norm_act_bwd(x, mr, gamma, beta, x, act="silu")[0]
    d1 = train.group_norm_act_bwd(x[-1:].clone(), mr1, gamma, beta, x[-1:].clone(), act="silu")[0]
    assert torch.equal(dx[-1:], d1)


def test_captured_and_replayed():
    """forward and backward in a graph, replayed on new inputs with eager work between, on a stream of its own"""
    B, P, C, G = 4, 300, 64, 8
    x, gamma, beta, ss = make(B, P, C, torch.bfloat16, seed=3)
    dy = rnd(B, P, C, seed=9, dtype=torch.bfloat16)

    def step():
        y, mr = ops.group_norm_act(x, gamma, beta, groups=G, ss=ss, want_stats=True)
        return (y, mr) + train.group_norm_act_bwd(x, mr, gamma, beta, dy, ss=ss)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for k in range(4):
        x.copy_(rnd(B, P, C, seed=50 + k, dtype=torch.bfloat16))
        dy.copy_(rnd(B, P, C, seed=60 + k, dtype=torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(p, q) for p, q in zip(outs, want)), k
