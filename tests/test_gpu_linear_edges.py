"""GPU tier (-m gpu): train.linear_act_bwd where its sums are longest, against the definition in 64 bits.  U = 2^-24."""
import pytest
import torch

from dig_amd import train

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield


def rnd(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).mul_(scale).to(dtype)


@pytest.mark.parametrize("N", [64, 256])
def test_column_sums_of_rows_off_16_bytes(N):
    """db of dy whose rows are read value by value: 256 values of a thread in fp32, up to 6 additions across the lanes and the rounding of the result; the rest is
    fp64.  The values are such that a longer sum in fp32 rounds the same way each time: 1 + 0.45 ulp(1024) is added as 1 from 1024 on."""
    M, K = 1 << 23, 8
    dy = torch.full((M, N + 1), 1.0 + 0.45 * 2.0 ** -13, device=DEV)[:, 1:]
    x, w = rnd(M, K, seed=1), rnd(N, K, seed=2)
    _, _, db = train.linear_act_bwd(x, w, dy, need_dx=False)
    ref = float(dy[0, 0].double()) * M
    assert float(((db.double() - ref).abs() / ref).max()) <= 264 * U
    pre = rnd(1, N, seed=3).expand(M, N)
    _, _, db = train.linear_act_bwd(x, w, dy, pre=pre, act="silu", need_dx=False)
    z = pre[0].double()
    sg = torch.sigmoid(z)
    ref = ref * sg * (1 + z * (1 - sg))
    tol = 264 * U * ref.abs() + float(dy[0, 0]) * M * 1.13 * U * (8 + 4 * z.abs())
    assert float(((db.double() - ref).abs() - tol).max()) <= 0


def test_every_row_counts_once():
    """dw and db over 33 million rows of small whole numbers: every partial sum is below 2^24, so that the result is exact in any order"""
    M, N, K = (1 << 25) + 128, 72, 72
    bf = torch.bfloat16
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randint(-1, 2, (M, K), generator=g, device=DEV, dtype=torch.int8).to(bf)
    wide = (torch.randint(0, 4, (M, N + 1), generator=g, device=DEV, dtype=torch.int8) == 3).to(bf)
    w = rnd(N, K, seed=6, scale=0.1, dtype=bf)
    for dy in (wide[:, :N].contiguous(), wide[:, 1:]):  # rows on 16 bytes and off them
        dx, dw, db = train.linear_act_bwd(x, w, dy, dw_f32=True)
        ref, cols = torch.zeros(N, K, dtype=torch.float64, device=DEV), torch.zeros(N, dtype=torch.float64, device=DEV)
        for i in range(0, M, 1 << 22):
            d, v = dy[i:i + (1 << 22)], x[i:i + (1 << 22)]
            ref += d.double().t().contiguous() @ v.double()
            cols += d.double().sum(0)
        assert float(cols.max()) < 2 ** 24 and float(ref.abs().max()) < 2 ** 24
        assert torch.equal(dw.double(), ref) and torch.equal(db.double(), cols)
        for rows in (slice(0, 200), slice(M - 200, M)):
            v, a = dy[rows].double() @ w.double(), dy[rows].double() @ w.double().abs()
            tol = (N + 8) * U * a
            assert float(((dx[rows].double() - v).abs() - tol - 2.0 ** -8 * (v.abs() + tol)).max()) <= 0
        del dx, dw, db
