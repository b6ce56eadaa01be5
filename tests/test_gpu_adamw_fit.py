"""AdamW inside the framework's training loops: batches that the forward launch gathers itself, recorded steps, a reducer between the
two halves of a step.  All of them run the same sums in the same order, so results are compared bit for bit."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(conv_layers=3, conv_layer_multiplier=2, initial_filters=8, activation="elu", kernel_size=3, conv_operations=1,
           fc_layers=0, fc_layer_size=256, dropout=0.2, latent_dimensions=0, batch_norm=False)


def _fit(bits, clip, gathers, graphs, reducer=False):
    from spectrum_vae_amd import autoencoder, losses, parallel
    from spectrum_vae_amd.optimizers import AdamW, ExponentialDecay
    model = autoencoder.CAEPadded(**CFG)
    model.build((None, 32, 32, 3))
    model._materialize(torch.device("cuda", 0))
    opt = AdamW(ExponentialDecay(5e-3, 2, 0.9, True), weight_decay=0.01, global_clipnorm=clip, state_bits=bits)
    model.compile(optimizer=opt, loss=losses.MeanSquaredError())
    model.gather_in_forward, model.use_graphs = gathers, graphs
    if reducer:
        model.distribute(parallel.GradReducer())
    X = torch.from_numpy(np.random.default_rng(3).standard_normal((130, 32, 32, 3)).astype(np.float32)).cuda()
    hist = model.fit(X, epochs=4, batch_size=48, verbose=0, seed=11)
    assert opt.iterations == 4 * 3
    mom = [t.clone() for v in model.trainable_variables for t in opt.moments(v)]
    return model._params.clone(), mom, hist.history["loss"], model


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 0.05])
def test_fit_takes_the_same_steps_in_every_form(bits, clip):
    """Three batches of 48, 48 and 34 of an epoch's 130 samples."""
    want, mom, loss, model = _fit(bits, clip, False, False)
    assert np.isfinite(loss).all() and torch.isfinite(want).all()
    for gathers, graphs, reducer in ((True, False, False), (False, True, False), (True, True, False), (False, False, True), (False, True, True)):
        got, mom2, loss2, other = _fit(bits, clip, gathers, graphs, reducer)
        assert torch.equal(want, got) and all(torch.equal(a, b) for a, b in zip(mom, mom2)), (gathers, graphs, reducer)
        assert loss == loss2, (gathers, graphs, reducer)
