"""NaN behind every activation of the group norm: what is not a number in a group shows in all that comes from the group."""
import pytest
import torch

from test_gpu_groupnorm import EPS, Case

pytestmark = pytest.mark.gpu

# held with sums of whole groups, held with sums of channels, streamed
SHAPES = [((5, 8, 8, 64), 8), ((3, 20, 20, 12), 3), ((2, 96, 80, 20), 5), ((2, 200, 160, 64), 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "elu", "lrelu", "tanh", "sigmoid"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_one_nan_makes_its_group_nan_behind_any_activation(shape, groups, act, dtype):
    from spectrum_vae_amd import ops
    k = Case(shape, groups, act, dtype, seed=2)
    d = shape[-1] // groups
    n = shape[0] - 1
    hit = torch.zeros(shape, dtype=torch.bool, device="cuda")
    hit[n, :, :, d:2 * d] = True
    bad = k.xt.clone()
    bad[n, 3, 5, d + 1] = float("nan")
    clean, got = k.forward(), k.forward(bad)
    assert torch.isnan(got[0][hit]).all() and torch.equal(got[0][~hit], clean[0][~hit])
    for a, b in zip(got[1:], clean[1:]):
        assert torch.isnan(a[n, 1])
        a[n, 1] = b[n, 1]
        assert torch.equal(a, b)

    def backward(x, mean, rstd):
        dx = torch.empty_like(x)
        dg, db = (torch.empty(shape[-1], device="cuda") for _ in range(2))
        ops.groupnorm_act_bwd(x, k.dyt, k.gt, k.bt, mean, rstd, dx, dg, db, False, groups, act, 0.2, k.ws())
        return dx, dg, db

    want = backward(k.xt, *clean[1:])
    _, mean, rstd = k.forward(bad)
    dx, dg, db = backward(bad, mean, rstd)
    assert torch.isnan(dx[hit]).all() and torch.equal(dx[~hit], want[0][~hit])
    own = slice(d, 2 * d)
    assert torch.isnan(dg[own]).all()
    if act is not None:  # without an activation dbeta is the sum of dy alone
        assert torch.isnan(db[own]).all()
    for a, b in ((dg, want[1]), (db, want[2])):
        a[own] = b[own]
        assert torch.equal(a, b)


@pytest.mark.parametrize("act", ["relu", "lrelu", "elu"])
def test_zeros_of_either_sign_and_infinite_inputs_of_the_activation(act):
    """gamma 0 leaves beta alone: the activation of +-0 and of +-inf."""
    from spectrum_vae_amd import ops
    k = Case((2, 4, 4, 8), 2, act, torch.float32)
    k.gt.zero_()
    k.bt.copy_(torch.tensor([0.0, -0.0, float("inf"), -float("inf"), 1.0, -1.0, 3e38, -3e38]))
    y = torch.empty_like(k.xt)
    ops.groupnorm_act_fwd(k.xt, k.gt, k.bt, y, None, None, 2, EPS, act, 0.2, k.ws())
    low = {"relu": [0.0, 0.0, 0.0], "lrelu": [-float("inf"), -0.2, 0.2 * -3e38], "elu": [-1.0, -0.6321205588, -1.0]}[act]
    want = torch.tensor([0.0, 0.0, float("inf"), low[0], 1.0, low[1], 3e38, low[2]], device="cuda")
    assert torch.allclose(y, want.expand_as(y), rtol=1e-6, atol=0)


@pytest.mark.parametrize("which", ["gamma", "beta"])
@pytest.mark.parametrize("act", ["relu", "elu", "lrelu"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_a_parameter_that_is_nan(shape, groups, act, which):
    """Its channel is NaN forward; backward its parameters' gradients and all of its group."""
    k = Case(shape, groups, act, torch.float32, seed=3)
    d = shape[-1] // groups
    (k.gt if which == "gamma" else k.bt)[d + 1] = float("nan")
    y, mean, rstd = k.forward()
    hit = torch.zeros(shape, dtype=torch.bool, device="cuda")
    hit[..., d + 1] = True
    assert torch.isnan(y[hit]).all() and torch.isfinite(y[~hit]).all() and torch.isfinite(mean).all() and torch.isfinite(rstd).all()
    dx, dg, db = k.backward()
    hit[..., d:2 * d] = True
    assert torch.isnan(dx[hit]).all() and torch.isfinite(dx[~hit]).all()
    assert torch.isnan(dg).sum() == 1 and torch.isnan(db).sum() == 1 and torch.isnan(dg[d + 1]) and torch.isnan(db[d + 1])
