"""Launches of 2^32 threads and more, which do not exist, are refused by the block operators' C entries before anything is launched (no GPU needed)."""
import ctypes

from dig_amd import _lib


def entry(fn, **at):
    a = _lib.STRUCTS[f"dig_{fn}_args"]()
    for name, t in a._fields_:
        if t is ctypes.c_void_p:
            setattr(a, name, 16)
    for k, v in at.items():
        setattr(a, k, v)
    rc = getattr(_lib.lib(), f"dig_{fn}")(ctypes.byref(a), None)
    return rc, _lib.lib().dig_last_error()


def test_group_norm_of_too_many_images():
    L = _lib.lib()
    for fn in ("gn_act", "gn_act_bwd"):
        pitch = dict(x_bs=16, x_ld=16, dtype=1, ss=None, act=3)
        pitch.update(dict(res=None) if fn == "gn_act" else dict(dy_bs=16, dy_ld=16))
        # one block of 512 threads an image, two of them; rows that are no vectors; a group a channel, whose partials a wave of its own joins
        for B, P, C, G in ((1 << 23, 1, 16, 1), (1 << 22, 1, 32, 2), (1 << 24, 1, 15, 1), (1 << 23, 4096, 15, 1), (1 << 21, 1, 33, 33)):
            rc, err = entry(fn, B=B, P=P, C=C, groups=G, **pitch)
            assert rc == -1 and b"too many blocks" in err, (fn, B, P, C, G, rc, err)
    assert L.dig_gn_act_ws(1, 16, 1, 0, 1, 1) == 0


def test_packing_of_too_many_rows():
    rc, err = entry("linear_act", M=1 << 26, N=8, K=511, ldx=511, ldw=511, dtype=0)
    assert rc == -1 and b"too many blocks" in err, (rc, err)
    rc, err = entry("linear_act_bwd", M=1 << 26, N=8, K=511, ldx=511, ldw=511, ldy=8, dtype=0)
    assert rc == -1 and b"too many blocks" in err, (rc, err)
