"""The clip of AdamW where the squares of single gradients leave float32's range: the norm is a number, and so is the step.

Bounds as in test_gpu_adamw, u = 2^-24: the scale is the quotient of the clip and a norm formed in 64 bits, rounded once: u of itself, or
half the denormals' step, 2^-150, where it is that small.  ``slack`` is this with the roundings of the quotient in 64 bits."""
import numpy as np
import pytest
import torch

from test_gpu_adamw import F, U, Tensors

pytestmark = pytest.mark.gpu


def _clipped_step(t, clip, bits):
    from spectrum_vae_amd import ops
    norm = np.sqrt(sum(np.square(g.astype(np.float64)).sum() for g in t.grads))
    state = torch.zeros(3, dtype=torch.int64, device="cuda")
    ops.adamw_step(t.plan(), state, 1e-3, 0.9, 0.999, 1e-7, clip_norm=clip, seed=5)
    scale = clip / max(clip, norm)
    t.check(0, 1e-3, scale, seed=5, slack=1.01 * U + 2.0 ** -150 / scale)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("big", [3e19, 1e25, -3e38])
@pytest.mark.parametrize("sizes,at", [([300, 70_001, 8193], (1, 12_345)), ([300, 70_001, 8193], (1, 70_000)), ([5, 3], (0, 2))])
def test_one_gradient_far_above_the_root_of_the_largest_float(sizes, at, big, bits):
    """In an entry of 4096 elements, in a tensor's ragged end, and in a tensor of a few elements."""
    t = Tensors(sizes, bits, seed=4)
    t.grads[at[0]][at[1]] = F(big)
    t.grads_t[at[0]][at[1]] = float(F(big))
    _clipped_step(t, 1.0, bits)


def test_gradients_below_the_root_of_the_smallest_float():
    """The clip takes three quarters of gradients whose squares are all below float32's denormals."""
    t = Tensors([300, 70_001, 9], 32, seed=7)
    t.grads = [g * F(1e-24) for g in t.grads]
    for dev, g in zip(t.grads_t, t.grads):
        dev.copy_(torch.from_numpy(g))
    for x in t.m_t + t.v_t:
        x.zero_()
    t.m, t.v = [np.zeros(n, F) for n in t.sizes], [np.zeros(n, F) for n in t.sizes]
    norm = np.sqrt(sum(np.square(g.astype(np.float64)).sum() for g in t.grads))
    _clipped_step(t, 0.25 * norm, 32)
