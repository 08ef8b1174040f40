"""GPU tier (-m gpu): ops.group_norm_act / train.group_norm_act_bwd where their sums and differences are at their worst, against the definition
in 64 bits.  U = 2^-24; a value stored in bf16 adds half a step of bf16, 2^-8 of it."""
import math

import pytest
import torch

from dig_amd import _lib, ops, train

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield


def rnd(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(DEV)


def act64(u, act):
    return {"none": u, "relu": torch.where(u < 0, torch.zeros_like(u), u), "gelu": u * torch.special.ndtr(u), "silu": u * torch.sigmoid(u)}[act]


def half(dtype):
    return torch.finfo(dtype).eps / 2


# one block per image and groups; split over blocks; rows that are no vectors
@pytest.mark.parametrize("P,C,G", [(33, 64, 8), (9000, 64, 8), (600, 30, 5)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_constant_groups_far_from_zero(P, C, G, dtype):
    """xhat is 0, so that y = act(beta') whatever the mean is, although rstd is eps^-1/2 = 316.  beta' = beta (1 + scale) + shift is two roundings of
    terms of |beta (1 + scale)| + |shift|; act has slope 1.13 at most and functions good to (8 + 2 |u|) U, as a fraction of the value."""
    levels = torch.tensor([300.0, -1000.0, 4000.0, 0.0, 61440.0, -2.5, 1.0, -300.0][:G], device=DEV)
    x = torch.stack([levels, levels.flip(0)]).repeat_interleave(C // G, 1)[:, None].expand(2, P, C).contiguous().to(dtype)
    gamma, beta, ss = rnd(C, seed=1, scale=0.3, shift=1.0), rnd(C, seed=2, scale=0.3), rnd(2, 2 * C, seed=3, scale=0.3)
    beta[::3] = 0.001  # near the border of ReLU's gate
    ss[:, C::3] = 0.0
    for act in ("none", "relu", "gelu", "silu"):
        y, mr = ops.group_norm_act(x, gamma, beta, groups=G, act=act, ss=ss, want_stats=True)
        assert torch.equal(mr[0, :, 0], levels) and torch.equal(mr[1, :, 0], levels.flip(0))
        scaled, shift = beta.double() * (1 + ss[:, :C].double()), ss[:, C:].double()
        u = scaled + shift
        ref = act64(u, act)
        tol = 1.13 * 4 * U * (scaled.abs() + shift.abs()) + U * (8 + 2 * u.abs()) * ref.abs()
        if dtype != torch.float32:
            tol = tol + half(dtype) * (ref.abs() + tol)
        err = (y.double() - ref[:, None]).abs()
        assert float((err - tol[:, None]).max()) <= 0, (act, float(err.max()), float((err / tol[:, None]).max()))


def stats64(x, G):
    """mean and biased variance of [B, P, C] per image and group, a part of the pixels at a time"""
    B, P, C = x.shape
    parts = [x[:, i:i + 16384].double().reshape(B, -1, G, C // G) for i in range(0, P, 16384)] if x.numel() <= 1 << 27 else None
    cut = lambda: parts if parts is not None else (x[:, i:i + 16384].double().reshape(B, -1, G, C // G) for i in range(0, P, 16384))  # noqa: E731
    n = P * (C // G)
    mean = sum(t.sum((1, 3)) for t in cut()) / n
    return mean, sum((t - mean[:, None, :, None]).square().sum((1, 3)) for t in cut()) / n


# rows that a thread adds: thousands (one row of 2048 channels at a time), hundreds, and of 30 channels that are no vectors
@pytest.mark.parametrize("P,C,G,border", [(1 << 18, 2048, 8, 128), (65536, 1024, 8, 256), (1 << 17, 2048, 1, 300), (1 << 20, 30, 5, 4000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_statistics_of_many_rows(P, C, G, border, dtype):
    """The first `border` rows, those that every thread begins with, lie 100 standard deviations off the rest.  A thread adds 32 fp32 values d = x - pivot
    and their squares.  For a run of n values the sum of d is within n U sum |d| and that of d^2 within n U S2, so that M2 = S2 - S1^2 / n is within
    n U S2 + 2 n U (sum |d|)^2 / n <= 3 n U S2.  A first run of 32 rows about the mean of its first 8 has S2 <= 5 M2: 480 U.  Those after it are about the mean of all k rows before,
    so that S2 <= M2 + (1 + 32 / k) of what the run's mean adds to the variance, together at most 2 M2 of all rows: 192 U.  That is 672 U of the variance at most, half
    of it for rstd (and 8 U for the rest: fp64 sums, their rounding, the stored value); the pivots' and the partial means' rounding (2 U of |x|) adds its square."""
    x = rnd(1, 4096, C, seed=1, dtype=dtype).repeat(1, P // 4096, 1)
    x += 100.0
    x[:, :border] = 0.0
    gamma, beta = rnd(C, seed=3, scale=0.3, shift=1.0), rnd(C, seed=4, scale=0.3)
    y, mr = ops.group_norm_act(x, gamma, beta, groups=G, act="none", want_stats=True)
    mean, var = stats64(x, G)
    r = (var + 1e-5).rsqrt()
    assert float(((mr[..., 0].double() - mean).abs() / mean.abs()).max()) <= 8 * U, "mean"
    off = ((mr[..., 1].double() - r).abs() / r).max()
    assert float(off) <= 344 * U + 4 * (100 * U * float(r.max())) ** 2, float(off) / U
    for rows in (slice(0, 70), slice(P // 2 + 1, P // 2 + 40), slice(P - 70, P)):  # and what is made of them
        rep = lambda t: t.repeat_interleave(C // G, 1)[:, None]  # noqa: E731
        xh = (x[:, rows].double() - rep(mr[..., 0].double())) * rep(mr[..., 1].double())
        ref = xh * gamma.double() + beta.double()
        tol = 8 * U * ((xh * gamma).abs() + beta.abs())
        if dtype != torch.float32:
            tol = tol + half(dtype) * (ref.abs() + tol)
        assert float(((y[:, rows].double() - ref).abs() - tol).max()) <= 0


@pytest.mark.parametrize("P,C,G", [(1 << 18, 2048, 8), (65536, 1024, 8), (1 << 20, 30, 5)])
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_sums_of_many_rows(P, C, G, act, dtype):
    """Summands of one sign, so that no error cancels: a thread adds 32 of them in fp32 at a time, the rest is fp64 but for the stored sums of a split, S1, S2 and the gradients:
    36 U of the sum of magnitudes, and 2 U more where (x - mean) rstd is a factor.  Slope of SiLU: |act''| <= 0.8, u good to 8 U of its terms, the functions
    to (8 + 4 |u|) U of at most 1.13."""
    x = rnd(1, 4096, C, seed=1, dtype=dtype).repeat(1, P // 4096, 1)
    dy = rnd(1, 4096, C, seed=2, scale=0.05, shift=1.1, dtype=dtype).repeat(1, P // 4096, 1)
    dy[:, :, ::3] = 1.1
    gamma, beta = rnd(C, seed=3, scale=0.3, shift=1.0), rnd(C, seed=4, scale=0.3)
    _, mr = ops.group_norm_act(x, gamma, beta, groups=G, act=act, want_stats=True)
    dx, dgamma, dbeta, _ = train.group_norm_act_bwd(x, mr, gamma, beta, dy, act=act)
    mean, r = (mr[0, :, k].double().repeat_interleave(C // G) for k in (0, 1))
    a, b = gamma.double(), beta.double()

    def terms(rows):
        xh, d = (x[0, rows].double() - mean) * r, dy[0, rows].double()
        if act == "none":
            return xh, d, torch.zeros_like(d)
        u = xh * a + b
        sg = torch.sigmoid(u)
        return xh, d * sg * (1 + u * (1 - sg)), d.abs() * U * (6.4 * ((xh * a).abs() + b.abs()) + 1.13 * (8 + 4 * u.abs()))

    s1, s2, t1, t2 = (torch.zeros(C, dtype=torch.float64, device=DEV) for _ in range(4))
    for xh, du, e in (terms(slice(i, i + 16384)) for i in range(0, P, 16384)):
        s1 += du.sum(0)
        s2 += (du * xh).sum(0)
        t1 += (36 * U * du.abs() + e).sum(0)
        t2 += ((38 * U * du.abs() + e) * xh.abs()).sum(0)
    for name, got, ref, tol in (("dbeta", dbeta, s1, t1), ("dgamma", dgamma, s2, t2)):
        err = (got.double() - ref).abs()
        assert float((err - tol).max()) <= 0, (name, float((err / tol).max()))
    group = lambda t: t.reshape(G, -1).sum(1).repeat_interleave(C // G) / (P * (C // G))  # noqa: E731
    m1, m2, e1, e2 = group(s1 * a), group(s2 * a), group(t1 * a.abs()), group(t2 * a.abs())
    for rows in (slice(0, 50), slice(P - 50, P)):
        xh, du, e = terms(rows)
        ref = r * (du * a - m1 - xh * m2)
        tol = r * (e * a.abs() + 6 * U * ((du * a).abs() + m1.abs() + 2 * (xh * m2).abs()) + e1 + xh.abs() * e2) + 4 * U * ref.abs()
        if dtype != torch.float32:
            tol = tol + half(dtype) * (ref.abs() + tol)
        err = (dx[0, rows].double() - ref).abs()
        assert float((err - tol).max()) <= 0, ("dx", float((err / tol).max()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_of_scale_and_shift_for_all_images(dtype):
    """an expanded row (one time step for the whole batch) gives what its copies give, in a graph too; so do rows that overlap"""
    B, P, C, G = 3, 50, 48, 6
    x, dy, res = (rnd(B, P, C, seed=i, dtype=dtype) for i in (1, 2, 3))
    gamma, beta, row = rnd(C, seed=4, shift=1.0), rnd(C, seed=5), rnd(1, 3 + 2 * C + 4, seed=6, scale=0.3)
    for ss, off in ((row[:, :2 * C].expand(B, 2 * C), 0), (row.expand(B, -1), 3), (torch.as_strided(row, (B, 2 * C), (2, 1)), 0)):
        def step(s, o):
            y, mr = ops.group_norm_act(x, gamma, beta, groups=G, ss=s, ss_off=o, res=res, want_stats=True)
            return (y, mr) + train.group_norm_act_bwd(x, mr, gamma, beta, dy, ss=s, ss_off=o)

        got, want = step(ss, off), step(ss.contiguous(), off)
        assert got[5].shape == (B, 2 * C) and all(torch.equal(p, q) for p, q in zip(got, want))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(ss, off)
    for k in range(3):
        row.copy_(rnd(*row.shape, seed=20 + k, scale=0.3))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, step(ss.contiguous(), off))), k


# 128 splits of an image, joined by the blocks that use them (8 groups) or by a launch of their own (32); vectors and single channels
@pytest.mark.parametrize("P,C,G", [(20000, 512, 8), (40001, 256, 32), (50003, 30, 5), (70001, 24, 24)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_splits(P, C, G, dtype):
    """buffers of the documented sizes and nothing behind them; the same image alone and in a batch; mean, rstd and the parameters' gradients in 64 bits (tolerances as above)"""
    B, L, dt, vec = 2, _lib.lib(), 0 if dtype == torch.bfloat16 else 1, int(C % 8 == 0)
    x, dy, gamma, beta = rnd(B, P, C, seed=1, shift=0.5, dtype=dtype), rnd(B, P, C, seed=2, dtype=dtype), rnd(C, seed=3, scale=0.3, shift=1.0), rnd(C, seed=4, scale=0.3)
    y, mr = ops.group_norm_act(x, gamma, beta, groups=G, act="silu", want_stats=True)
    grads = train.group_norm_act_bwd(x, mr, gamma, beta, dy, act="none")
    y1, mr1 = ops.group_norm_act(x[1:], gamma, beta, groups=G, act="silu", want_stats=True)
    assert torch.equal(y1, y[1:]) and torch.equal(mr1, mr[1:])
    assert torch.equal(train.group_norm_act_bwd(x[1:], mr1, gamma, beta, dy[1:], act="none")[0], grads[0][1:])
    mean, var = stats64(x, G)
    r = (var + 1e-5).rsqrt()
    assert float((mr[..., 0].double() - mean).abs().max()) <= 8 * U * float(x.double().abs().max())
    assert float(((mr[..., 1].double() - r).abs() / r).max()) <= 344 * U
    rep = lambda t: t.double().repeat_interleave(C // G, 1)[:, None]  # noqa: E731
    xh = (x.double() - rep(mr[..., 0])) * rep(mr[..., 1])
    d = dy.double()
    for got, t, n in ((grads[1], d * xh, 38), (grads[2], d, 36)):
        assert float(((got.double() - t.sum((0, 1))).abs() - n * U * t.abs().sum((0, 1))).max()) <= 0
    guard = 16384

    def buf(n, t=torch.float32):
        b = torch.full((n + guard,), 7.0, dtype=t, device=DEV)
        b[:n] = float("nan")
        return b

    at = dict(x=x, gamma=gamma, beta=beta, x_bs=P * C, x_ld=C, B=B, P=P, C=C, groups=G, dtype=dt)
    out, m2, w1, w2 = buf(B * P * C, dtype), buf(2 * B * G), buf(B * L.dig_gn_act_ws(P, C, G, 0, vec, dt)), buf(B * L.dig_gn_act_ws(P, C, G, 1, vec, dt))
    _lib.call("gn_act", out=out, mean_rstd=m2, ws=w1, act=3, eps=1e-5, **at)
    dx, dg, db = buf(B * P * C, dtype), buf(C), buf(C)
    _lib.call("gn_act_bwd", dy=dy, mean_rstd=mr, dx=dx, dgamma=dg, dbeta=db, ws=w2, dy_bs=P * C, dy_ld=C, act=0, **at)
    torch.cuda.synchronize()
    for b, want in ((out, y), (m2, mr), (dx, grads[0]), (dg, grads[1]), (db, grads[2]), (w1, None), (w2, None)):
        assert bool((b[-guard:] == 7.0).all())
        assert want is None or torch.equal(b[:-guard], want.reshape(-1))
