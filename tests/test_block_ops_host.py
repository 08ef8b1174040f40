"""Refusals of the channels-last block operators, without a GPU: every one is raised before anything is allocated or launched."""
import ctypes

import pytest
import torch

from dig_amd import _lib, ops, train


class _Fake(torch.Tensor):
    """A CPU tensor that claims to live on a HIP device, so that the guards run up to (not into) an allocation."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_subclass(cls, t)

    @property
    def is_cuda(self):
        return True

    @property
    def device(self):
        return torch.device("cuda", 0)

    def get_device(self):
        return 0


LAUNCH = _lib.launch  # the tests below put a refusal in its place


def F(*shape, dtype=torch.float32):
    return _Fake(torch.zeros(*shape, dtype=dtype))


@pytest.fixture(autouse=True)
def _no_launch(monkeypatch):
    def refuse(fn, *a, **kw):
        raise AssertionError(f"dig_{fn} would have been launched")

    monkeypatch.setattr(ops, "call", refuse)
    monkeypatch.setattr(train, "call", refuse)
    monkeypatch.setattr(_lib, "launch", refuse)
    monkeypatch.setattr(train, "launch", refuse)


def test_group_norm_act_refusals():
    ok = dict(gamma=F(16), beta=F(16), groups=4)
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.group_norm_act(torch.zeros(2, 5, 16), **ok)
    with pytest.raises(RuntimeError, match="gamma lives on cpu"):
        ops.group_norm_act(F(2, 5, 16), torch.zeros(16), F(16), groups=4)
    bad = [(dict(groups=3), "do not divide"), (dict(groups=0), "do not divide"), (dict(act="tanh"), "act must be"), (dict(eps=0.0), "eps must be positive"),
           (dict(gamma=F(15)), "gamma must be"), (dict(beta=F(16, dtype=torch.bfloat16)), "beta must be"), (dict(gamma=_Fake(torch.zeros(32)[::2])), "gamma must be"),
           (dict(ss=F(2, 31)), "do not hold"), (dict(ss=F(3, 32)), "ss must be"), (dict(ss=F(2, 40), ss_off=9), "do not hold"), (dict(ss=F(2, 40), ss_off=-1), "do not hold"),
           (dict(res=F(2, 5, 8)), "res must be"), (dict(res=F(2, 5, 16, dtype=torch.bfloat16)), "res must be")]
    for kw, msg in bad:
        with pytest.raises(ValueError, match=msg):
            ops.group_norm_act(F(2, 5, 16), **dict(ok, **kw))
    with pytest.raises(ValueError, match="unsupported dtype"):
        ops.group_norm_act(F(2, 5, 16, dtype=torch.float16), **ok)
    with pytest.raises(ValueError, match="must be \\[B"):
        ops.group_norm_act(F(16), **ok)
    with pytest.raises(ValueError, match="adjacent in memory"):
        ops.group_norm_act(_Fake(torch.zeros(2, 16, 5).transpose(1, 2)), **ok)
    with pytest.raises(ValueError, match="one pitch"):
        ops.group_norm_act(_Fake(torch.zeros(2, 5, 6, 16)[:, :, :4]), **ok)


def test_group_norm_act_bwd_refusals():
    x, ga = F(2, 5, 16), F(16)
    for mr in (F(2, 4), F(2, 4, 2, dtype=torch.float64), F(3, 4, 2), _Fake(torch.zeros(2, 4, 4)[..., ::2])):
        with pytest.raises(ValueError, match="mean_rstd must be"):
            train.group_norm_act_bwd(x, mr, ga, ga, x)
    with pytest.raises(ValueError, match="do not divide"):
        train.group_norm_act_bwd(x, F(2, 3, 2), ga, ga, x)
    with pytest.raises(ValueError, match="dy must be"):
        train.group_norm_act_bwd(x, F(2, 4, 2), ga, ga, F(2, 5, 16, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="dy lives on cpu"):
        train.group_norm_act_bwd(x, F(2, 4, 2), ga, ga, torch.zeros(2, 5, 16))


def test_gn_act_c_entry_refuses():
    L = _lib.lib()
    for fn in ("gn_act", "gn_act_bwd"):
        S = _lib.STRUCTS[f"dig_{fn}_args"]
        f = getattr(L, f"dig_{fn}")
        a = S()
        assert f(ctypes.byref(a), None) == -1 and b"null pointer" in L.dig_last_error()
        for name, t in S._fields_:
            if t is ctypes.c_void_p and name not in ("ss", "res", "dss"):
                setattr(a, name, 16)
        for k, v in dict(B=2, P=5, C=16, groups=4, act=3, dtype=0).items():
            setattr(a, k, v)
        for k, v, msg in (("groups", 3, b"bad shape"), ("P", 0, b"bad shape"), ("B", -1, b"bad shape"), ("act", 4, b"act 4"), ("dtype", 2, b"dtype 2"),
                          ("B", (1 << 31) - 1, b"too many blocks")):
            old = getattr(a, k)
            setattr(a, k, v)
            assert f(ctypes.byref(a), None) == -1 and msg in L.dig_last_error(), (fn, k)
            setattr(a, k, old)
        a.ss, a.dss = 16, 16
        if fn == "gn_act":
            a.ss_ld = 31
        assert f(ctypes.byref(a), None) == -1 and b"do not hold" in L.dig_last_error()
        if fn == "gn_act":  # a shape of several launches needs a workspace
            a.ss, a.ws, a.P, a.C = None, None, 1 << 20, 64
            assert f(ctypes.byref(a), None) == -1 and b"needs a workspace" in L.dig_last_error()
    assert L.dig_gn_act_ws(0, 16, 4, 0, 1, 0) < 0 and L.dig_gn_act_ws(5, 16, 3, 0, 0, 0) < 0 and L.dig_gn_act_ws(5, 12, 3, 0, 1, 0) < 0
    assert L.dig_gn_act_ws(5, 16, 4, 0, 1, 0) == 0 and L.dig_gn_act_ws(5, 16, 4, 1, 1, 0) > 0 and L.dig_gn_act_ws(5, 16, 4, 0, 0, 0) > 0


def test_linear_act_refusals():
    x, w = F(6, 16), F(8, 16)
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.linear_act(torch.zeros(6, 16), w)
    with pytest.raises(RuntimeError, match="w lives on cpu"):
        ops.linear_act(x, torch.zeros(8, 16))
    bad = [(dict(w=F(8, 15)), "do not fit"), (dict(w=F(8, 16, 1)), "do not fit"), (dict(w=F(0, 16)), "do not fit"), (dict(w=F(8, 16, dtype=torch.bfloat16)), "x is"),
           (dict(w=_Fake(torch.zeros(16, 8).t())), "K adjacent"), (dict(bias=F(7)), "bias must be"), (dict(bias=F(8, dtype=torch.bfloat16)), "bias must be"),
           (dict(act="elu"), "act must be"), (dict(res=F(6, 7)), "res must be"), (dict(res=F(6, 8, dtype=torch.bfloat16)), "res must be"),
           (dict(res=_Fake(torch.zeros(8, 6).t())), "adjacent in memory"), (dict(x=_Fake(torch.zeros(4, 3, 2, 16)[:, :, 0][:, :2])), "one pitch")]
    for kw, msg in bad:
        with pytest.raises(ValueError, match=msg):
            ops.linear_act(**dict(dict(x=x, w=w), **kw))
    with pytest.raises(ValueError, match="unsupported dtype"):
        ops.linear_act(F(6, 16, dtype=torch.float16), F(8, 16, dtype=torch.float16))


def test_linear_act_bwd_refusals():
    x, w, dy = F(6, 16), F(8, 16), F(6, 8)
    for kw, msg in ((dict(dy=F(6, 9)), "dy must be"), (dict(act="gelu"), "needs pre"), (dict(act="gelu", pre=F(5, 8)), "pre must be"), (dict(act="x"), "act must be"),
                    (dict(dy=F(6, 8, dtype=torch.bfloat16)), "dy must be"), (dict(w=F(8, 17)), "do not fit")):
        with pytest.raises(ValueError, match=msg):
            train.linear_act_bwd(**dict(dict(x=x, w=w, dy=dy), **kw))
    with pytest.raises(RuntimeError, match="pre lives on cpu"):
        train.linear_act_bwd(x, w, dy, act="silu", pre=torch.zeros(6, 8))


def test_linear_act_c_entry_refuses():
    L = _lib.lib()
    for fn, optional in (("linear_act", ("bias", "res", "pre", "xpack", "wpack")), ("linear_act_bwd", ("pre", "dx", "db", "dz", "xpack", "wpack"))):
        S = _lib.STRUCTS[f"dig_{fn}_args"]
        f = getattr(L, f"dig_{fn}")
        a = S()
        assert f(ctypes.byref(a), None) == -1 and b"null pointer" in L.dig_last_error()
        for name, t in S._fields_:
            if t is ctypes.c_void_p and name not in optional:
                setattr(a, name, 16)
        for k, v in dict(M=6, N=8, K=16, act=0, dtype=0).items():
            setattr(a, k, v)
        for k, v, msg in (("M", 0, b"bad shape"), ("N", -1, b"bad shape"), ("K", 0, b"bad shape"), ("K", (1 << 30), b"bad shape"), ("act", 4, b"act 4"), ("act", -1, b"act -1"),
                          ("dtype", 2, b"dtype 2")):
            old = getattr(a, k)
            setattr(a, k, v)
            assert f(ctypes.byref(a), None) == -1 and msg in L.dig_last_error(), (fn, k, L.dig_last_error())
            setattr(a, k, old)
        if fn == "linear_act_bwd":
            a.act = 2
            assert f(ctypes.byref(a), None) == -1 and b"needs pre and dz" in L.dig_last_error()
        else:  # a shape whose k is split needs the workspace
            a.ws, a.M, a.N, a.K = None, 16, 64, 8192
            assert L.dig_linear_act_ws(16, 64, 8192, 0) > 0 and f(ctypes.byref(a), None) == -1 and b"needs a workspace" in L.dig_last_error()
            a.ws, a.M, a.N, a.K, a.ldx, a.ldw = 16, 4096, 512, 101, 101, 101  # rows that do not lie on 16 bytes, and no place to pack them
            assert f(ctypes.byref(a), None) == -2 and b"need xpack" in L.dig_last_error()
        if fn == "linear_act_bwd":
            a.act, a.K, a.ldx, a.ldw, a.ldy, a.N = 0, 16, 16, 16, 9, 9
            assert f(ctypes.byref(a), None) == -2 and b"need dz" in L.dig_last_error()
            a.ldx = 17
            assert f(ctypes.byref(a), None) == -2 and b"need xpack" in L.dig_last_error()
    assert L.dig_linear_act_ws(0, 8, 8, 0) < 0 and L.dig_linear_act_bwd_ws(4, 0, 8, 0, 1) < 0


def test_c_entries_refuse_pitches_and_workspaces():
    """negative pitches, workspaces off 16 bytes, and sizes whose workspace does not fit 31 bits"""
    L = _lib.lib()
    for fn, shape, pitches, ws in (("gn_act", dict(B=2, P=1 << 20, C=16, groups=4, act=3), ("x_bs", "x_ld", "res_bs", "res_ld"), b"on 16 bytes"),
                                   ("gn_act_bwd", dict(B=2, P=1 << 20, C=16, groups=4, act=3), ("x_bs", "x_ld", "dy_bs", "dy_ld"), b"on 16 bytes"),
                                   ("linear_act", dict(M=16, N=64, K=8192), ("ldx", "ldw", "ldr"), b"on 16 bytes"),
                                   ("linear_act_bwd", dict(M=16, N=64, K=64, act=1), ("ldx", "ldw", "ldy", "ldpre"), b"on 16 bytes")):
        S = _lib.STRUCTS[f"dig_{fn}_args"]
        f = getattr(L, f"dig_{fn}")
        a = S()
        for name, t in S._fields_:
            if t is ctypes.c_void_p and name not in ("ss", "dss"):
                setattr(a, name, 16)
        for k, v in shape.items():
            setattr(a, k, v)
        for k in pitches:
            setattr(a, k, -8)
            assert f(ctypes.byref(a), None) == -1 and b"negative pitch" in L.dig_last_error(), (fn, k)
            setattr(a, k, 64)
        a.ws = 24
        assert f(ctypes.byref(a), None) == -1 and ws in L.dig_last_error(), (fn, L.dig_last_error())
    for M in (1 << 30) + 1, (1 << 31) - 1:
        assert L.dig_linear_act_ws(M, 8, 8, 0) < 0 and L.dig_linear_act_bwd_ws(M, 8, 8, 0, 1) < 0
    for bwd in (0, 1):
        assert L.dig_gn_act_ws(1 << 20, 1 << 20, 1 << 20, bwd, 0, 1) < 0
    S = _lib.STRUCTS["dig_gn_act_args"]
    a = S()
    for name, t in S._fields_:
        if t is ctypes.c_void_p and name not in ("ss", "res"):
            setattr(a, name, 16)
    a.B, a.P, a.C, a.groups, a.dtype = 1, 1 << 20, 1 << 20, 1 << 20, 1
    a.x_ld = 1 + (1 << 20)  # rows off 16 bytes
    assert L.dig_gn_act(ctypes.byref(a), None) == -1 and b"too large a workspace" in L.dig_last_error()


def test_sizes_beyond_31_bits_are_refused():
    with pytest.raises(ValueError, match="larger than the kernels take"):
        LAUNCH("gn_act", 0, *([0] * 8), *([0] * 4), 1, 1 << 32, *([0] * 6), 1e-5)


def test_array_fields_do_not_run_into_the_next():
    for fn in sorted(_lib.STRUCTS):
        for name, t in _lib.STRUCTS[fn]._fields_:
            n = getattr(t, "_length_", 0)
            if n and fn.startswith("dig_") and fn.endswith("_args") and hasattr(_lib.lib(), fn[:-5]):
                with pytest.raises(IndexError, match="holds"):
                    _lib.call(fn[4:-5], **{name: [0] * (n + 1)})
                return
    pytest.skip("no argument block holds an array")
