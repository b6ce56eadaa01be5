"""Statistics of long samples whose first row is an outlier (a border, padding), against 64 bits.

D is the distance of the first row from the others.  The squares of the group are D^2 and more.  A thread takes L rows, sums about the
mean of the first U of them: L is at most 58 at these sizes, 40 where U is 4 (bfloat16 in pieces of eight) instead of 8.  With the outlier
among the first U rows the thread's squares are (1 - 1/U) D^2 and grow by (D / U)^2 a row, an addition is off by u of the sum so far:
73 u D^2 in all with U = 8, 75 u with U = 4.  From them goes ((L - U) D / U)^2 / L, whose sum is off by L u / 2 of itself: 39 u D^2 and 81 u.
The threads' means (T = 256 of them) are off by 2 u D and are joined with distances of D^2 / L in all: 4 sqrt(T) u = 64 u D^2.  That is
at most 220 u of the squares, half of it in the root; 18 u are for the roundings that come once."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-3


@pytest.mark.parametrize("level", ["constant", "random"])
@pytest.mark.parametrize("shape,groups,dtype", [
    ((1, 2_000_000, 4), 1, torch.float32), ((1, 30_000_000, 4), 2, torch.float32), ((1, 20_000_000, 8), 2, torch.bfloat16),
    ((2, 300_000, 90), 9, torch.float32), ((1, 3_000_000, 6), 3, torch.bfloat16), ((3, 1_000_001, 1), 1, torch.float32),
    ((1, 60_000, 2000), 8, torch.bfloat16), ((1, 4_000_000, 32), 4, torch.float32)])
def test_outlier_first_in_long_chunks(shape, groups, dtype, level):
    from spectrum_vae_amd import ops
    n, s, c = shape
    g = torch.Generator(device="cuda").manual_seed(c)
    x = torch.full(shape, 0.3, device="cuda")
    if level == "random":
        x += torch.randn(shape, device="cuda", generator=g)
    x[:, 0] = 1e4
    x = x.to(dtype)
    ones, zeros = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(n, groups, device="cuda"), torch.empty(n, groups, device="cuda")
    ws = torch.empty(max(ops.groupnorm_workspace(n, s, c, groups), 1), dtype=torch.uint8, device="cuda")
    ops.groupnorm_act_fwd(x, ones, zeros, y, mean, rstd, groups, EPS, None, 0.0, ws)
    d = c // groups
    for i in range(n):
        for k in range(groups):
            v = x[i, :, k * d:(k + 1) * d].double()
            var, mu = torch.var_mean(v, unbiased=False)
            want = float((var + EPS) ** -0.5)
            assert abs(float(mean[i, k]) - float(mu)) <= 8 * U * 1e4
            assert abs(float(rstd[i, k]) - want) <= 128 * U * want, abs(float(rstd[i, k]) / want - 1) / U
            z = (v[:1000] - mu) * want
            tol = 8 * U * 1e4 * want + 130 * U * z.abs() + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) * z.abs()
            assert ((y[i, :1000, k * d:(k + 1) * d].double() - z).abs() <= tol).all()
    assert np.isfinite(float(y.double().sum()))
