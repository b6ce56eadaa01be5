"""AdamW on the host: gradients that share memory."""
import pytest
import torch


def _spans_meet(a, b):
    return (a.numel() > 0 and b.numel() > 0 and a.data_ptr() < b.data_ptr() + b.numel() * b.element_size()
            and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size())


def _check(grads, written):
    from spectrum_vae_amd.optimizers import _apart
    got = _apart(grads, written)
    assert len(got) == len(grads) and all(torch.equal(a, b) for a, b in zip(got, grads))
    for i, a in enumerate(got):
        assert not any(_spans_meet(a, b) for b in got[i + 1:]) and not any(_spans_meet(a, w) for w in written)
    copied = [a.data_ptr() != b.data_ptr() for a, b in zip(got, grads)]
    for i, a in enumerate(grads):  # what lies apart is not copied
        if not any(_spans_meet(a, b) for j, b in enumerate(grads) if j != i) and not any(_spans_meet(a, w) for w in written):
            assert not copied[i]
    return copied


def test_gradients_are_copied_where_they_share_memory():
    flat, params = torch.arange(64.0), torch.arange(100.0, 132.0)
    codes = torch.arange(32, dtype=torch.uint8)
    a, b = flat[:8], flat[8:16]
    assert _check([a, b], [params, codes]) == [False, False]
    assert sum(_check([a, a], [params])) == 1
    assert sum(_check([a, a, a, b], [params])) == 2
    assert sum(_check([flat[:20], flat[4:8], flat[16:24], flat[23:30], flat[40:50]], [params])) in (2, 3)
    assert _check([params[:8], a], [params]) == [True, False]
    assert _check([params[4:5], params[4:5], params], [params]) == [True, True, True]
    assert _check([flat[:0], flat[:0], a], [flat[20:]]) == [False, False, False]
    assert _check([flat[4:30], flat[2:3]], [flat[10:12], params]) == [True, False]  # begins ahead of what is written
    assert _check([flat, flat[20:21]], [flat[10:12], flat[40:41]]) == [True, True]
    assert _check([], [params]) == []


@pytest.mark.parametrize("seed", range(200))
def test_any_gradients_end_up_apart(seed):
    g = torch.Generator().manual_seed(seed)
    flat = torch.arange(60.0)

    def cut():
        i, j = sorted(torch.randint(0, 61, (2,), generator=g).tolist())
        return flat[i:j]

    n, m = (int(torch.randint(1, 6, (1,), generator=g)) for _ in range(2))
    edges = sorted(torch.randint(0, 61, (2 * m,), generator=g).tolist())
    _check([cut() for _ in range(n)], [flat[i:j] for i, j in zip(edges[::2], edges[1::2])])


class _Model:
    """What an optimizer sees of a model."""

    def __init__(self, sizes):
        self._params = torch.zeros(sum(sizes))
        self.trainable_variables = [type("V", (), {"size": n, "name": "v"})() for n in sizes]


@pytest.mark.parametrize("make", ["Adam", "AdamW", "AdamW8"])
def test_a_model_in_the_place_of_one_that_is_gone_starts_with_moments_of_its_own(make):
    """An id is given out again once its object is gone."""
    import gc

    from spectrum_vae_amd.optimizers import Adam, AdamW
    opt = Adam() if make == "Adam" else AdamW(state_bits=8 if make == "AdamW8" else 32)
    for i in range(20):
        m = _Model([300, 5 + i])
        slots = opt._slots_for(m)
        assert all(not t.any() for t in slots)
        assert slots[0].numel() == (256 * 3 if make == "AdamW8" else 305 + i)
        assert opt._slots_for(m)[0] is slots[0]
        for t in slots:
            t.fill_(1)
        del m, slots
        gc.collect()


def test_a_variable_in_the_place_of_an_excluded_one_is_decayed():
    import gc

    from spectrum_vae_amd.optimizers import AdamW
    opt = AdamW(weight_decay=0.1)

    class V:
        name = "kernel"

    kept = V()
    opt.exclude_from_weight_decay(var_list=[V(), kept])
    gc.collect()
    others = [V() for _ in range(20)]
    assert opt._decay_of(kept) == 0.0 and all(opt._decay_of(v) == 0.1 for v in others)
