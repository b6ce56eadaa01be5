"""Gradients that share memory with each other or with what the step writes, given to ``apply_gradients``: the step is that of copies."""
import pytest
import torch

from test_gpu_adamw import _model

pytestmark = pytest.mark.gpu


def _two(bits):
    from spectrum_vae_amd.optimizers import AdamW
    out = []
    for _ in range(2):
        opt = AdamW(1e-2, state_bits=bits)
        m = _model(opt)
        m._materialize(torch.device("cuda", 0))
        out.append((opt, m, m.trainable_variables))
    out[1][1]._params.copy_(out[0][1]._params)
    return out


def _same(a, b):
    (opt, m, tv), (opt2, m2, tv2) = a, b
    assert torch.equal(m._params, m2._params)
    for v, w in zip(tv, tv2):
        assert all(torch.equal(s, t) for s, t in zip(opt.moments(v), opt2.moments(w)))


@pytest.mark.parametrize("bits", [32, 8])
def test_one_gradient_for_two_variables_and_overlapping_ones(bits):
    a, b = _two(bits)
    tv, tw = a[2], b[2]
    assert tv[1].size == tv[2].size  # gamma and beta
    flat = torch.linspace(-1, 1, 4 * tv[0].size, device="cuda")
    for step in range(2):
        g, h = flat[:tv[1].size], flat[3:3 + tv[0].size]  # they overlap, and each stands for itself
        a[0].apply_gradients([(g, tv[1]), (g, tv[2]), (h, tv[0])])
        b[0].apply_gradients([(g.clone(), tw[1]), (g.clone(), tw[2]), (h.clone(), tw[0])])
        _same(a, b)
    keep = flat.clone()
    one = torch.full((1,), 0.5, device="cuda").expand(tv[1].size)
    a[0].apply_gradients([(one, tv[1]), (one, tv[2])])
    b[0].apply_gradients([(one.clone(), tw[1]), (one.clone(), tw[2])])
    _same(a, b)
    assert torch.equal(flat, keep)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_lie_in_what_the_step_writes(bits):
    """A variable's own values as its gradient, another variable's values, and a piece of the gradient buffer."""
    a, b = _two(bits)
    tv, tw = a[2], b[2]
    a[0].apply_gradients([(tv[0].data, tv[0]), (tv[1].data, tv[2])])
    b[0].apply_gradients([(tw[0].data.clone(), tw[0]), (tw[1].data.clone(), tw[2])])
    _same(a, b)
    a[1]._grads.fill_(0.25)
    b[1]._grads.fill_(0.25)
    a[0].apply_gradients([(tv[2].grad, tv[1]), (tv[1].grad, tv[2])])
    b[0].apply_gradients([(tw[2].grad.clone(), tw[1]), (tw[1].grad.clone(), tw[2])])
    _same(a, b)
    assert (a[1]._grads == 0.25).all()


def test_the_same_calls_as_adam():
    """What Adam takes AdamW takes: without decay the two are one formula, up to the roundings of a step of 1e-2 (the root and
    the quotient of AdamW are within 1 ulp each; 2^-20 of a step covers them)."""
    from spectrum_vae_amd.optimizers import Adam, AdamW
    models = []
    for opt in (Adam(1e-2), AdamW(1e-2, weight_decay=0.0)):
        m = _model(opt)
        m._materialize(torch.device("cuda", 0))
        models.append((opt, m))
    models[1][1]._params.copy_(models[0][1]._params)
    g = torch.linspace(-1, 1, models[0][1].trainable_variables[1].size, device="cuda")
    for opt, m in models:
        tv = m.trainable_variables
        opt.apply_gradients([(g, tv[1]), (g, tv[2])])
    p, q = (m._params for _, m in models)
    assert ((p - q).abs() <= 2.0 ** -20 * 1e-2 + 2.0 ** -23 * p.abs()).all()
