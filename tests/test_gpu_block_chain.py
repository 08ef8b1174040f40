"""GPU tier (-m gpu): the block operators run together as a model runs them - GroupNorm + scale/shift + SiLU, a 1x1 expansion with GELU, a
projection with the residual - forward and backward, against the definition in 64 bits; the same run captured and replayed, on streams other
than the default one, and from threads.

The tolerance is carried through the run with absolute values.  h is half a step of the storage type (2^-8 for bf16, 2^-24 for fp32), U = 2^-24.
A stage that gets its input within e gives
 * product of K terms: sum |w| e + (K + 8) U sum |x w|, and h of the stored value;
 * GELU, SiLU: slopes are at most 1.13 and change by at most 0.8 per unit of u; their functions are good to (8 + 4 |u|) U;
 * GroupNorm: a thread adds at most 32 values (x - pivot), below 8 standard deviations each, before the sums go on in fp64: the mean is off by
   32 * 8 U of a standard deviation and rstd by 64 U of itself, so xhat by at most 512 U (1 + |xhat|); the adjoint is linear in du."""
import math
import threading

import pytest
import torch

from dig_amd import _lib, ops, train

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
NORM = 512 * U
DTYPES = [torch.float32, torch.bfloat16]
NAMES = ("y", "dx", "dgamma", "dbeta", "dss", "dw1", "db1", "dw2", "db2")


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield


def rnd(*shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def inputs(B, P, C, H, dtype, seed=0):
    return dict(x=rnd(B, P, C, seed=seed, dtype=dtype), gamma=1 + rnd(C, seed=seed + 1, scale=0.1), beta=rnd(C, seed=seed + 2, scale=0.1),
                ss=rnd(B, 2 * C, seed=seed + 3, scale=0.1), w1=rnd(H, C, seed=seed + 4, scale=C ** -0.5, dtype=dtype), b1=rnd(H, seed=seed + 5, scale=0.1),
                w2=rnd(C, H, seed=seed + 6, scale=H ** -0.5, dtype=dtype), b2=rnd(C, seed=seed + 7, scale=0.1), dy=rnd(B, P, C, seed=seed + 8, dtype=dtype))


def run(t, G):
    """forward and backward of y = x + W2 gelu(W1 silu(norm(x)) + b1) + b2"""
    a, mr = ops.group_norm_act(t["x"], t["gamma"], t["beta"], groups=G, act="silu", ss=t["ss"], want_stats=True)
    h, pre = ops.linear_act(a, t["w1"], t["b1"], act="gelu", want_pre=True)
    y = ops.linear_act(h, t["w2"], t["b2"], res=t["x"])
    dh, dw2, db2 = train.linear_act_bwd(h, t["w2"], t["dy"], dw_f32=True)
    da, dw1, db1 = train.linear_act_bwd(a, t["w1"], dh, pre=pre, act="gelu", dw_f32=True)
    dx, dgamma, dbeta, dss = train.group_norm_act_bwd(t["x"], mr, t["gamma"], t["beta"], da, act="silu", ss=t["ss"])
    return y, dx, dgamma, dbeta, dss, dw1, db1, dw2, db2  # dx without the residual's part, which is dy


def exact(t, G):
    """name -> (value in 64 bits, how far off the run's may be), in the order of NAMES"""
    dt = t["x"].dtype
    hs = torch.finfo(dt).eps / 2
    hz = hs if dt == torch.bfloat16 else 0.0  # dz is rounded for the matrix units
    t = {k: v.double() for k, v in t.items()}
    x, W1, W2, dy = t["x"], t["w1"], t["w2"], t["dy"]
    B, P, C = x.shape
    H, M = W1.shape[0], B * P
    stored = lambda v, e: e + hs * (v.abs() + e)  # noqa: E731
    # norm: per (image, group), then per channel
    xg = x.reshape(B, P, G, C // G)
    mean, var = xg.mean((1, 3), keepdim=True), xg.var((1, 3), unbiased=False, keepdim=True)
    rstd = (var + 1e-5).rsqrt()
    xh = ((xg - mean) * rstd).reshape(B, P, C)
    rstd = rstd.expand(B, P, G, C // G).reshape(B, P, C)
    exh = NORM * (1 + xh.abs())
    sc, sh = 1 + t["ss"][:, None, :C], t["ss"][:, None, C:]
    gp, bp = t["gamma"] * sc, t["beta"] * sc + sh
    u = gp * xh + bp
    eu = gp.abs() * exh + 8 * U * (bp.abs() + u.abs())
    a = u * torch.sigmoid(u)
    ea = stored(a, 1.13 * eu + (8 + 4 * u.abs()) * U * a.abs())
    z = a @ W1.t() + t["b1"]
    ez = (ea + (C + 8) * U * a.abs()) @ W1.abs().t() + 2 * U * (t["b1"].abs() + z.abs())
    ep = stored(z, ez)
    h = z * torch.special.ndtr(z)
    eh = stored(h, 1.13 * ez + (8 + 4 * z.abs()) * U * h.abs())
    y = h @ W2.t() + t["b2"] + x
    ey = stored(y, (eh + (H + 8) * U * h.abs()) @ W2.abs().t() + 4 * U * (t["b2"].abs() + y.abs() + x.abs()))
    # backward
    dh = dy @ W2
    edh = stored(dh, (C + 8) * U * (dy.abs() @ W2.abs()))
    D, Hf, Eh = dy.reshape(M, C), h.reshape(M, H), eh.reshape(M, H)
    dw2, edw2 = D.t() @ Hf, D.abs().t() @ (Eh + (M + 8) * U * Hf.abs())
    db2, edb2 = D.sum(0), 265 * U * D.abs().sum(0)
    slope = torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    dz = dh * slope
    edz = 1.13 * edh + (dh.abs() + edh) * (0.8 * ep + 1.13 * (8 + 4 * (z.abs() + ep)) * U)
    edzr = edz + hz * (dz.abs() + edz)
    Z, Ez, Ezr, A, Ea = dz.reshape(M, H), edz.reshape(M, H), edzr.reshape(M, H), a.reshape(M, C), ea.reshape(M, C)
    dw1 = Z.t() @ A
    edw1 = (Ezr + (M + 8) * U * Z.abs()).t() @ (A.abs() + Ea) + Z.abs().t() @ Ea
    db1, edb1 = Z.sum(0), (Ez + 265 * U * (Z.abs() + Ez)).sum(0)
    da = dz @ W1
    eda = stored(da, (edzr + (H + 8) * U * (dz.abs() + edzr)) @ W1.abs())
    sg = torch.sigmoid(u)
    du = da * sg * (1 + u * (1 - sg))
    edu = 1.13 * eda + (da.abs() + eda) * (0.8 * eu + 1.13 * (8 + 4 * (u.abs() + eu)) * U)
    edu = edu + 265 * U * (du.abs() + edu)  # and the sums of it
    s1, es1 = du.sum(1), edu.sum(1)
    s2, es2 = (du * xh).sum(1), (edu * (xh.abs() + exh) + du.abs() * exh).sum(1)
    group = lambda v: v.reshape(B, G, C // G).sum(2, keepdim=True).expand(B, G, C // G).reshape(B, 1, C) / (P * (C // G))  # noqa: E731
    g1 = gp[:, 0]
    m1, em1 = group(g1 * s1), group(g1.abs() * es1)
    m2, em2 = group(g1 * s2), group(g1.abs() * es2)
    dx = rstd * (gp * du - m1 - xh * m2)
    terms = gp.abs() * du.abs() + m1.abs() + xh.abs() * m2.abs()
    edx = stored(dx, rstd * (gp.abs() * edu + em1 + (xh.abs() + exh) * em2 + exh * m2.abs() + NORM * terms))
    c1 = sc[:, 0]
    dgamma, edgamma = (c1 * s2).sum(0), (c1.abs() * (es2 + 4 * U * s2.abs())).sum(0)
    dbeta, edbeta = (c1 * s1).sum(0), (c1.abs() * (es1 + 4 * U * s1.abs())).sum(0)
    ga, be = t["gamma"].abs(), t["beta"].abs()
    dss = torch.cat([t["gamma"] * s2 + t["beta"] * s1, s1], 1)
    edss = torch.cat([ga * es2 + be * es1 + 4 * U * (ga * s2.abs() + be * s1.abs()), es1 + 4 * U * s1.abs()], 1)
    pairs = ((y, ey), (dx, edx), (dgamma, edgamma), (dbeta, edbeta), (dss, edss), (dw1, edw1 + U * dw1.abs()), (db1, edb1 + U * db1.abs()),
             (dw2, edw2 + U * dw2.abs()), (db2, edb2))
    return dict(zip(NAMES, pairs))


SHAPES = [  # B, P, C, H, groups
    (1, 1, 8, 8, 1), (2, 1, 64, 256, 8), (2, 196, 64, 256, 8), (3, 77, 36, 50, 6), (1, 1000, 320, 640, 32), (4, 1024, 128, 512, 32), (2, 2048, 384, 1536, 12), (5, 9, 7, 13, 7),
]


@pytest.mark.parametrize("B,P,C,H,G", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_chain(B, P, C, H, G, dtype):
    t = inputs(B, P, C, H, dtype, seed=P)
    got = run(t, G)
    for name, v, (ref, tol) in zip(NAMES, got, exact(t, G).values()):
        assert v.shape == ref.shape, name
        err = (v.double() - ref).abs()
        assert float((err - tol - 1e-30).max()) <= 0, (name, float(err.max()), float((err / (tol + 1e-30)).max()))


def same(name, got, want):
    for n, g, w in zip(NAMES, got, want):
        assert torch.equal(g, w), (name, n, float((g.double() - w.double()).abs().max()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_graphs_replayed_together(dtype):
    """two captured runs of different shapes, replayed in turn on two streams while the inputs change in place and eager runs go between"""
    shapes = [(2, 196, 64, 256, 8), (3, 300, 40, 136, 5)]
    ts = [inputs(B, P, C, H, dtype, seed=11 + i) for i, (B, P, C, H, _) in enumerate(shapes)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in shapes]
    for t, (*_, G) in zip(ts, shapes):
        run(t, G)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(t, G))
        graphs.append(g)
    for r in range(4):
        for i, t in enumerate(ts):
            fresh = inputs(*shapes[i][:4], dtype, seed=100 + 10 * r + i)
            for k in t:
                t[k].copy_(fresh[k])
        want = [run(t, s[4]) for t, s in zip(ts, shapes)]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            same(f"replay {r} of graph {i}", outs[i], want[i])


def test_streams_and_threads():
    """each thread on a stream of its own, all of them at once"""
    shapes = [(2, 196, 64, 256, 8), (3, 300, 40, 136, 5), (1, 1000, 320, 640, 32), (2, 64, 24, 48, 3)]
    ts = [inputs(B, P, C, H, torch.bfloat16 if i % 2 else torch.float32, seed=31 + i) for i, (B, P, C, H, _) in enumerate(shapes)]
    want = [run(t, s[4]) for t, s in zip(ts, shapes)]
    torch.cuda.synchronize()
    got, failed = [[] for _ in shapes], []

    def work(i):
        try:
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(6):
                    got[i].append(run(ts[i], shapes[i][4]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(shapes))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed, failed
    torch.cuda.synchronize()
    for i, runs in enumerate(got):
        assert len(runs) == 6
        for r in runs:
            same(f"thread {i}", r, want[i])


def test_images_do_not_meet():
    """garbage in one image of a batch changes nothing in the others"""
    B, P, C, H, G = 3, 100, 64, 128, 8
    t = inputs(B, P, C, H, torch.bfloat16, seed=5)
    base = run(t, G)
    bad = {k: v.clone() for k, v in t.items()}
    for k in ("x", "dy", "ss"):
        bad[k][2] = float("nan")
    got = run(bad, G)
    for n, g, w in zip(NAMES, got, base):
        if n in ("y", "dx", "dss"):
            assert torch.equal(g[:2], w[:2]), n
            assert g[2].isnan().all(), n


class Guarded:
    """buffers of exactly the documented sizes, with 64 KB behind each that nobody may write"""

    def __init__(self):
        self.all = []

    def __call__(self, name, n, dtype=torch.float32):
        if n == 0:
            return None
        t = torch.full((n + 65536 // dtype.itemsize,), 7.0, dtype=dtype, device=DEV)
        t[:n] = float("nan")
        self.all.append((name, t, n))
        return t

    def check(self, what):
        torch.cuda.synchronize()
        for name, t, n in self.all:
            assert bool((t[n:] == 7.0).all()), (what, name)

    def get(self, name):
        t, n = next((t, n) for k, t, n in self.all if k == name)
        return t[:n]


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (20, 1536, 384), (333, 81, 100), (300, 33, 1000), (16, 64, 4096), (64, 40, 8192), (700, 520, 264), (2500, 640, 72), (4200, 1000, 96), (9000, 2056, 64)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_writes_its_buffers_only(M, N, K, dtype):
    L, dt, e = _lib.lib(), 0 if dtype == torch.bfloat16 else 1, 8 if dtype == torch.bfloat16 else 4
    x, w, b, dy = rnd(M, K, seed=1, dtype=dtype), rnd(N, K, seed=2, scale=K ** -0.5, dtype=dtype), rnd(N, seed=3), rnd(M, N, seed=4, dtype=dtype)
    kp = (K + e - 1) // e * e
    G = Guarded()
    packs = dict(xpack=G("xpack", M * kp, dtype), wpack=G("wpack", N * kp, dtype))
    _lib.call("linear_act", x=x, w=w, bias=b, res=dy, out=G("out", M * N, dtype), pre=G("pre", M * N, dtype), ws=G("ws", L.dig_linear_act_ws(M, N, K, dt)), **packs,
              ldx=K, ldw=K, ldr=N, M=M, N=N, K=K, act=2, dtype=dt)
    G.check("forward")
    y, pre = ops.linear_act(x, w, b, act="gelu", res=dy, want_pre=True)
    assert torch.equal(G.get("out").view(M, N), y) and torch.equal(G.get("pre").view(M, N), pre)
    for act in (0, 2):
        for f32 in (0, 1):
            G = Guarded()
            _lib.call("linear_act_bwd", x=x, w=w, dy=dy, pre=pre, dx=G("dx", M * K, dtype), dw=G("dw", N * K, torch.float32 if f32 else dtype), db=G("db", N),
                      dz=G("dz", M * ((N + 7) // 8 * 8), dtype), ws=G("ws", L.dig_linear_act_bwd_ws(M, N, K, dt, 1)), xpack=G("xpack", M * kp, dtype),
                      wpack=G("wpack", N * kp, dtype), ldx=K, ldw=K, ldy=N, ldpre=N, M=M, N=N, K=K, act=act, dtype=dt, dw_f32=f32)
            G.check("backward")
            dx, dw, db = train.linear_act_bwd(x, w, dy, pre=pre, act="gelu" if act else "none", dw_f32=bool(f32))
            assert torch.equal(G.get("dx").view(M, K), dx) and torch.equal(G.get("dw").view(N, K), dw) and torch.equal(G.get("db"), db)


@pytest.mark.parametrize("B,P,C,G_", [(1, 1, 1, 1), (2, 16, 128, 32), (3, 37, 48, 6), (2, 300, 15, 5), (1, 5000, 24, 4), (2, 4096, 64, 32), (2, 1030, 320, 10), (1, 3, 2056, 8),
                                      (2, 20000, 64, 2), (1, 70000, 7, 7)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_writes_its_buffers_only(B, P, C, G_, dtype):
    L, dt = _lib.lib(), 0 if dtype == torch.bfloat16 else 1
    x, dy, ss = rnd(B, P, C, seed=1, dtype=dtype), rnd(B, P, C, seed=2, dtype=dtype), rnd(B, 2 * C, seed=3, scale=0.1)
    gamma, beta = 1 + rnd(C, seed=4, scale=0.1), rnd(C, seed=5, scale=0.1)
    vec = int(C % 8 == 0)
    G = Guarded()
    at = dict(x_bs=P * C, x_ld=C, B=B, P=P, C=C, groups=G_, ss_ld=2 * C, act=3, dtype=dt)
    _lib.call("gn_act", x=x, gamma=gamma, beta=beta, ss=ss, res=dy, out=G("out", B * P * C, dtype), mean_rstd=G("mr", B * G_ * 2),
              ws=G("ws", B * L.dig_gn_act_ws(P, C, G_, 0, vec, dt)), res_bs=P * C, res_ld=C, eps=1e-5, **at)
    G.check("forward")
    y, mr = ops.group_norm_act(x, gamma, beta, groups=G_, act="silu", ss=ss, res=dy, want_stats=True)
    assert torch.equal(G.get("out").view(B, P, C), y) and torch.equal(G.get("mr").view(B, G_, 2), mr)
    G = Guarded()
    _lib.call("gn_act_bwd", x=x, dy=dy, mean_rstd=mr, gamma=gamma, beta=beta, ss=ss, dx=G("dx", B * P * C, dtype), dgamma=G("dgamma", C), dbeta=G("dbeta", C),
              dss=G("dss", B * 2 * C), ws=G("ws", B * L.dig_gn_act_ws(P, C, G_, 1, vec, dt)), dy_bs=P * C, dy_ld=C, **at)
    G.check("backward")
    dx, dgamma, dbeta, dss = train.group_norm_act_bwd(x, mr, gamma, beta, dy, act="silu", ss=ss)
    assert torch.equal(G.get("dx").view(B, P, C), dx) and torch.equal(G.get("dgamma"), dgamma) and torch.equal(G.get("dbeta"), dbeta) and torch.equal(G.get("dss").view(B, -1), dss)


def test_one_row_of_scale_and_shift():
    """one image: the pitch of its only scale/shift row does not matter"""
    t = inputs(1, 50, 16, 8, torch.float32, seed=9)
    odd = torch.as_strided(t["ss"], (1, 32), (1, 1))
    a, mr = ops.group_norm_act(t["x"], t["gamma"], t["beta"], groups=4, ss=odd, want_stats=True)
    b = ops.group_norm_act(t["x"], t["gamma"], t["beta"], groups=4, ss=t["ss"])
    assert torch.equal(a, b)
    for v, w in zip(train.group_norm_act_bwd(t["x"], mr, t["gamma"], t["beta"], t["dy"], ss=odd), train.group_norm_act_bwd(t["x"], mr, t["gamma"], t["beta"], t["dy"], ss=t["ss"])):
        assert torch.equal(v, w)
