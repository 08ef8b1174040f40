"""GPU tier (-m gpu): ops.group_norm_act / train.group_norm_act_bwd where their sums and differences are at their worst, against the definition
in 64 bits.  U = 2^-24; a value stored in bf16 adds half a step of bf16, 2^-8 of it."""
import math

import pytest
import torch

from dig_amd import ops, train

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
