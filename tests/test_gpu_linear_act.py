"""GPU tier (-m gpu): ops.linear_act / train.linear_act_bwd (csrc/linear.hip) against the definition in 64 bits.

Tolerances, elementwise and derived from the operations (U = 2^-24; h = half a step of the storage type, 2^-8 for bf16 and U for fp32):
 * a product of K terms accumulated in fp32 in any order is within (K + 8) U sum |x w| of its value (the products of bf16 values are exact);
 * act: slope at most 1.13, exp2 / rcp / erf good to 2 ulps, exp's argument to |z| U, relative in the result;
 * dz = dy act'(z): the slope's functions 8 + 4 |z| ulps of at most 1.13, then h |dz| where it is rounded to bf16;
 * db: at most 256 fp32 additions in a thread, four threads, then fp64, of the unrounded dz.
Each stored value adds h of itself."""
import math

import pytest
import torch

from dig_amd import ops, train

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
ACTS = ("none", "relu", "gelu", "silu")


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield


def rnd(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def act64(u, act):
    return {"none": u, "relu": torch.where(u < 0, torch.zeros_like(u), u), "gelu": u * torch.special.ndtr(u), "silu": u * torch.sigmoid(u)}[act]


def slope64(u, act):
    if act == "gelu":
        return torch.special.ndtr(u) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        return torch.sigmoid(u) * (1 + u * torch.sigmoid(-u))
    return (u > 0).double() if act == "relu" else torch.ones_like(u)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def close(name, got, ref, tol):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    assert float((err - tol - 1e-37).max()) <= 0, (name, float(err.max()), float((err / (tol + 1e-37)).max()))


def check_fwd(x, w, bias, act, res, want_pre=True):
    out = ops.linear_act(x, w, bias=bias, act=act, res=res, want_pre=want_pre)
    y, pre = out if want_pre else (out, None)
    K = x.shape[-1]
    X, W = x.double().reshape(-1, K), w.double()
    z = X @ W.t()
    tz = (K + 8) * U * (X.abs() @ W.abs().t())
    if bias is not None:
        z = z + bias.double()
        tz = tz + 2 * U * (bias.double().abs() + z.abs())
    shape = (*x.shape[:-1], w.shape[0])
    assert y.shape == shape and y.dtype == x.dtype and y.is_contiguous()
    if want_pre:
        assert pre.dtype == x.dtype and pre.is_contiguous()
        close("pre", pre, z.reshape(shape), (tz + half(x.dtype) * (z.abs() + tz)).reshape(shape))
    ref = act64(z, act)
    tol = 1.13 * tz + (U * (8 + 2 * z.abs()) * ref.abs() if act in ("gelu", "silu") else 0)
    if res is not None:
        ref = ref + res.double().reshape(ref.shape)
        tol = tol + U * ref.abs()
    close("y", y, ref.reshape(shape), (tol + half(x.dtype) * (ref.abs() + tol)).reshape(shape))
    return y, pre


def check_bwd(x, w, dy, pre, act, has_bias=True, dw_f32=False, need_dx=True):
    dx, dw, db = train.linear_act_bwd(x, w, dy, pre=pre, act=act, has_bias=has_bias, dw_f32=dw_f32, need_dx=need_dx)
    N, K = w.shape
    X, W, D = x.double().reshape(-1, K), w.double(), dy.double().reshape(-1, N)
    M = X.shape[0]
    h = half(x.dtype)
    dz, tz = D, torch.zeros_like(D)
    if act != "none":
        Z = pre.double().reshape(-1, N)
        dz = D * slope64(Z, act)
        tz = D.abs() * 1.13 * U * (8 + 4 * Z.abs()) if act != "relu" else tz
    rounded = tz + (h * (dz.abs() + tz) if act in ("gelu", "silu") else 0)
    if need_dx:
        assert dx.dtype == x.dtype and dx.is_contiguous()
        ref, tol = dz @ W, (rounded + (N + 8) * U * dz.abs()) @ W.abs()
        close("dx", dx, ref.reshape(x.shape), (tol + h * (ref.abs() + tol)).reshape(x.shape))
    else:
        assert dx is None
    ho = U if dw_f32 else h
    assert dw.dtype == (torch.float32 if dw_f32 else w.dtype) and dw.is_contiguous()
    ref, tol = dz.t() @ X, (rounded + (M + 8) * U * dz.abs()).t() @ X.abs()
    close("dw", dw, ref, tol + ho * (ref.abs() + tol))
    assert (db is not None) == has_bias
    if has_bias:
        ref, tol = dz.sum(0), (tz + 264 * U * dz.abs()).sum(0)
        close("db", db, ref, tol + U * ref.abs())
    return dx, dw, db


SHAPES = [  # M, N, K
    (1, 1, 1), (1, 8, 8), (3, 5, 7), (2, 3, 64), (1, 1536, 384), (20, 1536, 384), (17, 20, 384), (128, 128, 64), (129, 136, 72), (200, 81, 96), (64, 300, 33), (257, 24, 1000),
    (1000, 16, 8), (5, 4096, 16), (300, 65, 2048), (37, 1153, 387), (2048, 8, 2048), (733, 384, 768), (1500, 12, 4), (90, 520, 260), (4100, 260, 36), (33, 40, 12), (16, 64, 4096),
    (500, 21, 515), (900, 768, 1032)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_shapes(M, N, K, dtype):
    for i, act in enumerate(ACTS):
        x, w = rnd(M, K, seed=i, dtype=dtype), rnd(N, K, seed=i + 5, scale=K ** -0.5, dtype=dtype)
        bias = rnd(N, seed=i + 9) if i != 1 else None
        res = rnd(M, N, seed=i + 11, dtype=dtype) if i >= 2 else None
        check_fwd(x, w, bias, act, res, want_pre=i != 0)


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_shapes(M, N, K, dtype):
    for i, act in enumerate(ACTS):
        x, w = rnd(M, K, seed=i, dtype=dtype), rnd(N, K, seed=i + 5, scale=K ** -0.5, dtype=dtype)
        dy, pre = rnd(M, N, seed=i + 13, dtype=dtype), rnd(M, N, seed=i + 17, dtype=dtype)
        check_bwd(x, w, dy, pre if i else None, act, has_bias=i != 1, dw_f32=i == 2, need_dx=i != 3 or M % 2 == 0)


@pytest.mark.parametrize("M,N,K", [(13302, 777, 33), (12711, 776, 72), (12800, 777, 64), (10347, 1153, 387), (9953, 1160, 1032), (10240, 1280, 384), (9409, 408, 168), (30001, 97, 45)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(M, N, K, dtype):
    """enough outputs for the largest tiles, with partial tiles on every side"""
    x, w, b = rnd(M, K, seed=M, dtype=dtype), rnd(N, K, seed=N, scale=K ** -0.5, dtype=dtype), rnd(N, seed=K)
    r = rnd(M, N, seed=M + 1, dtype=dtype)
    for act in ("none", "gelu"):
        _, pre = check_fwd(x, w, b, act, r)
    check_fwd(x, w, None, "relu", None, want_pre=False)
    check_bwd(x, w, r, pre, "gelu")
    check_bwd(x, w, r, None, "none", dw_f32=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    """channel slices of wider rows (aligned and not), a weight inside a larger one, broadcast rows"""
    M, N, K = 150, 72, 64
    xs, ws = rnd(M, 2 * K + 3, seed=1, dtype=dtype), rnd(N + 1, 3 * K + 1, seed=2, scale=0.1, dtype=dtype)
    xa, wa = rnd(3, M // 3, 2 * K, seed=3, dtype=dtype), rnd(N, 2 * K, seed=4, scale=0.1, dtype=dtype)
    rs = rnd(M, N + 5, seed=5, dtype=dtype)
    ra = rnd(M, 2 * N, seed=6, dtype=dtype)
    bias = rnd(N, seed=7)
    for x, w, r in ((xs[:, 3:3 + K], ws[1:, 1:1 + K], rs[:, 5:]), (xs[:, :K], wa[:, K:], ra[:, N:]), (xa.reshape(M, -1)[:, K:], wa[:, :K], ra[:, :N]),
                    (xa.reshape(M, -1)[:, K:], ws[:N, K:2 * K], rs[:, :N]), (rnd(1, K, seed=8, dtype=dtype).expand(M, K), wa[:, :K], ra[:, :N])):
        _, pre = check_fwd(x, w, bias, "gelu", r)
        check_bwd(x, w, r, r, "silu")
        check_bwd(x, w, r, None, "none")
        check_bwd(x, w, rnd(1, N, seed=9, dtype=dtype).expand(M, N), pre, "relu")
    check_fwd(xa[..., :K], wa[:, :K], bias, "relu", ra.reshape(3, M // 3, -1)[..., N:])
    check_fwd(xa[0, 0, :K], wa[:, :K], bias, "silu", None)  # one vector, [K] -> [N]
    check_bwd(xa[..., :K], wa[:, :K], ra.reshape(3, M // 3, -1)[..., N:], ra.reshape(3, M // 3, -1)[..., :N], "gelu")


def test_gradient_against_differences():
    """directional derivatives of L = sum(dy * y) of the 64-bit forward in x, w and bias (central differences, h = 1e-5)"""
    M, N, K = 40, 24, 32
    for act in ("none", "gelu", "silu"):
        x, w, b, dy = rnd(M, K, seed=1), rnd(N, K, seed=2, scale=0.2), rnd(N, seed=3), rnd(M, N, seed=4)
        _, pre = ops.linear_act(x, w, bias=b, act=act, want_pre=True)
        got = train.linear_act_bwd(x, w, dy, pre=pre, act=act)
        ins = [t.double() for t in (x, w, b)]
        loss = lambda X, W, B: float((act64(X @ W.t() + B, act) * dy.double()).sum())  # noqa: E731
        for i, g in enumerate(got):
            v = rnd(*ins[i].shape, seed=20 + i).double()
            hi, lo = ([t + s * 1e-5 * v if j == i else t for j, t in enumerate(ins)] for s in (1, -1))
            diff = (loss(*hi) - loss(*lo)) / 2e-5
            # the products' (max(M, N, K) + 8) U and the slope's few U, each relative to magnitudes at most 8 times the sums here
            assert abs(diff - float((g.double() * v).sum())) <= 400 * U * float((g.double().abs() * v.abs()).sum()) + 1e-5, (act, i)


def test_nan_and_inf_stay_in_their_rows():
    for dtype in (torch.float32, torch.bfloat16):
        M, N, K = 150, 136, 200
        x, w = rnd(M, K, seed=1, dtype=dtype), rnd(N, K, seed=2, scale=0.1, dtype=dtype)
        clean = ops.linear_act(x, w, act="silu")
        for bad in (float("nan"), float("inf")):
            xb = x.clone()
            xb[77, K - 1] = bad
            y = ops.linear_act(xb, w, act="silu")
            keep = torch.arange(M, device=DEV) != 77
            assert torch.equal(y[keep], clean[keep]) and not torch.equal(y[77], clean[77])
        xb = x.clone()
        xb[3] = float("nan")
        assert torch.isnan(ops.linear_act(xb, w, act="relu")[3]).all()
        xb, yb = torch.full_like(x, float("nan")), torch.full((M, N), float("nan"), dtype=dtype, device=DEV)
        check_fwd(x[:40], w, None, "none", None)  # rows behind the last one hold NaN nowhere they are read
        big = torch.cat([x, xb])
        assert torch.equal(ops.linear_act(big[:M], w, act="silu"), clean)
        dbig = torch.cat([rnd(M, N, seed=4, dtype=dtype), yb])
        assert all(torch.isfinite(t).all() for t in train.linear_act_bwd(big[:M], w, dbig[:M]))


def test_empty():
    w = rnd(16, 24, seed=1)
    x = torch.empty(0, 24, device=DEV)
    y, pre = ops.linear_act(x, w, bias=rnd(16, seed=2), act="gelu", want_pre=True)
    assert y.shape == pre.shape == (0, 16)
    dx, dw, db = train.linear_act_bwd(x, w, y, pre=pre, act="gelu")
    assert dx.shape == (0, 24) and not dw.any() and not db.any()


def test_reproducible():
    for M, N, K in ((300, 520, 260), (6912, 384, 1536), (16, 64, 4096)):
        x, w, dy = rnd(M, K, seed=1, dtype=torch.bfloat16), rnd(N, K, seed=2, scale=0.1, dtype=torch.bfloat16), rnd(M, N, seed=3, dtype=torch.bfloat16)
        y, pre = ops.linear_act(x, w, act="gelu", want_pre=True)
        a, b = (train.linear_act_bwd(x, w, dy, pre=pre, act="gelu") for _ in range(2))
        assert torch.equal(y, ops.linear_act(x, w, act="gelu")) and all(torch.equal(p, q) for p, q in zip(a, b))


def test_large_offsets():
    """element offsets past 2^31 in x and y: the last rows against the definition (another row count may take another kernel, whose sums run in
    another order: each is held to the tolerance of the definition, not to the other's bits)"""
    M, N, K = (1 << 25) + 128, 72, 72
    bf = torch.bfloat16
    x = torch.empty(M, K, dtype=bf, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(3))
    w, dy = rnd(N, K, seed=2, scale=0.1, dtype=bf), rnd(200, N, seed=4, dtype=bf)
    y = ops.linear_act(x, w, act="relu")
    X, W = x[-200:].double(), w.double()
    z = X @ W.t()
    tol = (K + 8) * U * (X.abs() @ W.abs().t())
    close("y", y[-200:], act64(z, "relu"), 1.13 * tol + half(bf) * (z.abs() + tol))
    y[-200:] = dy  # y serves as the incoming gradient
    dx, dw, db = train.linear_act_bwd(x, w, y, act="none")
    ref, tol = dy.double() @ W, (N + 8) * U * (dy.double().abs() @ W.abs())
    close("dx", dx[-200:], ref, tol + half(bf) * (ref.abs() + tol))


def test_captured_and_replayed():
    """forward and backward in a graph, replayed on new inputs with eager work between"""
    M, N, K = 300, 136, 520
    bf = torch.bfloat16
    x, w, b, dy = rnd(M, K, seed=1, dtype=bf), rnd(N, K, seed=2, scale=0.1, dtype=bf), rnd(N, seed=3), rnd(M, N, seed=4, dtype=bf)

    def step():
        y, pre = ops.linear_act(x, w, bias=b, act="gelu", want_pre=True)
        return (y, pre) + train.linear_act_bwd(x, w, dy, pre=pre, act="gelu")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for k in range(4):
        x.copy_(rnd(M, K, seed=50 + k, dtype=bf))
        dy.copy_(rnd(M, N, seed=60 + k, dtype=bf))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, step())), k
