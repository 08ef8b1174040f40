"""What _lib.call and _lib.launch refuse in an argument block, without a GPU: every refusal comes before the launch."""
import pytest
import torch

from dig_amd import _lib

ROWS = dict(x=64, g=64, res=None, out=64, rows=4, C=8, dtype=1)  # of dig_rmsnorm


class _OnDevice(torch.Tensor):
    """A CPU tensor that claims to live on a HIP device."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_subclass(cls, t)

    @property
    def is_cuda(self):
        return True


@pytest.fixture(autouse=True)
def _no_launch(monkeypatch):
    e = _lib._Entry("rmsnorm")

    def refuse(*a):
        raise AssertionError("dig_rmsnorm would have been launched")

    e.func = refuse
    monkeypatch.setitem(_lib._ENTRIES, "rmsnorm", e)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 0, raising=False)


def test_a_block_that_is_in_order_reaches_the_launch():
    with pytest.raises(AssertionError, match="would have been launched"):
        _lib.call("rmsnorm", **ROWS)


@pytest.mark.parametrize("field", ["rows", "C", "dtype"])
def test_numbers_are_numbers(field):
    for v in (None, 3.0, "4", [4], torch.tensor(4), _OnDevice(torch.tensor(4))):
        with pytest.raises((TypeError, RuntimeError)) as err:
            _lib.call("rmsnorm", **dict(ROWS, **{field: v}))
        assert err.type is TypeError or "HIP-device pointers only" in str(err.value)
    with pytest.raises(TypeError, match="is a number, not None"):
        _lib.call("rmsnorm", **dict(ROWS, **{field: None}))
    with pytest.raises(TypeError, match="is a number, not a tensor"):
        _lib.call("rmsnorm", **dict(ROWS, **{field: _OnDevice(torch.tensor(4))}))


def test_float_fields():
    name, fields = next((n, f) for n, f in sorted(_lib._STRUCT_FIELDS.items()) if n == "dig_affine_act_add_args")
    at = {k: (64 if t is _lib.ctypes.c_void_p else 1) for k, t in fields}
    for v in (None, _OnDevice(torch.tensor(0.5))):
        with pytest.raises(TypeError, match="is a number"):
            _lib.call("affine_act_add", **dict(at, x_scale=v))
    with pytest.raises(TypeError, match="wrong type"):
        _lib.call("affine_act_add", **dict(at, x_scale="1"))


def test_values_past_31_bits():
    for v in (1 << 31, -(1 << 31) - 1, 1 << 70):
        with pytest.raises(ValueError, match="larger than the kernels take"):
            _lib.call("rmsnorm", **dict(ROWS, C=v))
    with pytest.raises(ValueError, match="larger than the kernels take"):
        _lib.call("rmsnorm", **dict(ROWS, rows=1 << 63))  # a 64-bit field


def test_pointers():
    for v in (2.0, "x"):
        with pytest.raises(TypeError, match="wrong type"):
            _lib.call("rmsnorm", **dict(ROWS, x=v))
    with pytest.raises(TypeError, match="has no field"):
        _lib.call("rmsnorm", **dict(ROWS, y=1))


def test_launch_tells_types_from_sizes():
    n = len(_lib._ENTRIES["rmsnorm"].blank)
    with pytest.raises(TypeError, match="wrong type"):
        _lib.launch("rmsnorm", 0, *[None] * n)
    with pytest.raises(ValueError, match="larger than the kernels take"):
        _lib.launch("rmsnorm", 0, *[1 << 70] * n)
