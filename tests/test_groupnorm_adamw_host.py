"""Group norm and AdamW without a GPU: the 8-bit moments' rounding in the oracle, layer and optimizer construction, and every
refusal that the host makes before a launch."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import np_ops
from oracle.np_ops import Moments8


def _values(rng, n, signed):
    x = (rng.standard_normal(n) * np.exp(3 * rng.standard_normal(n))).astype(np.float32)
    x[rng.integers(0, n, n // 8)] = 0.0
    return x if signed else x * x


@pytest.mark.parametrize("width", [4, 5])
@pytest.mark.parametrize("n", [1, 255, 256, 257, 2000])
def test_moments8_round_to_a_neighbouring_code(width, n):
    rng = np.random.default_rng(n * width)
    x = _values(rng, n, width == 4)
    lo, _ = Moments8.encode(x, np.zeros(n, np.int64), width)
    hi, e = Moments8.encode(x, np.full(n, 65535), width)
    down, up = Moments8.decode(lo, e, width).astype(np.float64), Moments8.decode(hi, e, width).astype(np.float64)
    xd = x.astype(np.float64)
    # cut off towards zero (a positive second moment's smallest code excepted), or the code above: at most one step
    # of a value's own binade, 2^-3 of it, or the smallest code
    smallest = 2.0 ** (np.repeat(e.astype(np.float64), 256)[:n] - 129 - ((1 << width) - 1))
    step = np.maximum(np.abs(xd) / 8, smallest)
    if width == 4:
        assert (np.abs(down) <= np.abs(xd)).all()
    assert (np.abs(down - xd) <= step).all() and (np.abs(up - xd) <= step).all()
    assert (np.abs(up) >= np.abs(xd) * (1 - 2.0 ** -18)).all()
    if width == 5:
        assert (down[x > 0] > 0).all() and (down[x == 0] == 0).all()


def test_moments8_codes_are_fixed_points_and_rounding_is_unbiased():
    for width, codes in ((4, np.arange(256)), (5, np.arange(256))):
        exps = np.array([130], np.uint8)
        vals = Moments8.decode(codes.astype(np.uint8), exps, width)
        for r in (0, 65535):
            again, e = Moments8.encode(vals, np.full(256, r), width)
            assert e[0] == 130 and (Moments8.decode(again, e, width) == vals).all()
    x = np.zeros(256 * 400, np.float32)
    x[0::256] = 1.0
    x[1::256] = 0.3  # between codes 0.28125 and 0.3125
    m_bits, v_bits = Moments8.random_bits(len(x), 0, 7, 1833)
    for width, bits in ((4, m_bits), (5, v_bits)):
        codes, e = Moments8.encode(x, bits, width)
        got = Moments8.decode(codes, e, width)[1::256]
        assert set(np.unique(got)) <= {np.float32(0.28125), np.float32(0.3125)}
        # 400 draws of a step of 1/32 at 0.6: standard deviation of the mean 0.03125 * sqrt(0.24 / 400) = 7.7e-4
        assert abs(got.mean() - 0.3) < 5 * 7.7e-4


def test_moments8_blocks_with_nothing_finite_nothing_at_all_and_tiny_values():
    z = np.zeros(256, np.float32)
    codes, e = Moments8.encode(z, np.full(256, 65535), 4)
    assert e[0] == 0 and not Moments8.decode(codes, e, 4).any()
    for bad in (np.nan, np.inf):
        x = z.copy()
        x[5] = bad
        codes, e = Moments8.encode(x, np.zeros(256, np.int64), 5)
        assert e[0] == 255 and np.isnan(Moments8.decode(codes, e, 5)).all()
    x = z.copy()
    x[0], x[1] = 1e-40, 3e-45  # float32 denormals
    codes, e = Moments8.encode(x, np.zeros(256, np.int64), 5)
    assert e[0] == 0
    assert abs(Moments8.decode(codes, e, 5)[0] - x[0]) <= x[0] / 8 + 2e-45


def test_group_norm_oracle_against_differences():
    rng = np.random.default_rng(0)
    x, dy = rng.standard_normal((2, 3, 2, 6)), rng.standard_normal((2, 3, 2, 6))
    gamma, beta = rng.standard_normal(6), rng.standard_normal(6)
    for act in (None, "elu", "tanh", "sigmoid", "lrelu", "relu"):
        _, mean, rstd = np_ops.group_norm(x, gamma, beta, 3, 1e-3, act)
        dx, dg, db = np_ops.group_norm_bwd(x, dy, gamma, beta, mean, rstd, 3, act)
        h = 1e-6
        for i in [(0, 0, 0, 0), (1, 2, 1, 5), (0, 1, 1, 3)]:
            e = np.zeros_like(x)
            e[i] = h
            num = ((np_ops.group_norm(x + e, gamma, beta, 3, 1e-3, act)[0] - np_ops.group_norm(x - e, gamma, beta, 3, 1e-3, act)[0]) * dy).sum() / (2 * h)
            assert abs(num - dx[i]) < 1e-6 * max(1, abs(num)) + 1e-7
        for k in range(6):
            e = np.zeros(6)
            e[k] = h
            num = ((np_ops.group_norm(x, gamma + e, beta, 3, 1e-3, act)[0] - np_ops.group_norm(x, gamma - e, beta, 3, 1e-3, act)[0]) * dy).sum() / (2 * h)
            assert abs(num - dg[k]) < 1e-6 * max(1, abs(num)) + 1e-7
            num = ((np_ops.group_norm(x, gamma, beta + e, 3, 1e-3, act)[0] - np_ops.group_norm(x, gamma, beta - e, 3, 1e-3, act)[0]) * dy).sum() / (2 * h)
            assert abs(num - db[k]) < 1e-6 * max(1, abs(num)) + 1e-7


# ------------------------------------------------------------------------------------------------ construction
def test_group_normalization_layer_builds_and_folds_its_activation():
    from spectrum_vae_amd import nn, unet
    l = nn.GroupNormalization(groups=4)
    assert l.build((8, 8, 12)) == (8, 8, 12) and l.count_params() == 24
    inst = nn.GroupNormalization(groups=-1)
    inst.build((4, 4, 6))
    assert inst.groups == 6
    with pytest.raises(ValueError, match="do not split"):
        nn.GroupNormalization(groups=5).build((8, 8, 12))
    with pytest.raises(ValueError, match="normalization"):
        unet.convolution(8, (2, 2), (2, 2), normalization="layer")
    block = unet.convolution(64, (2, 2), (2, 2), normalization="group")
    block.build((8, 8, 3))
    assert isinstance(block.layers[1], nn.GroupNormalization) and block.layers[1].fused_act == ("lrelu", 0.2)
    assert block.layers[2].folded
    gen, disc = unet.Generator(normalization="group"), unet.Discriminator(normalization="group")
    gen.build_graph((1, 32, 32, 1))
    disc.build_graph((1, 32, 32, 4))
    ref = unet.Generator()
    ref.build_graph((1, 32, 32, 1))
    assert [v.shape for v in gen.trainable_variables] == [v.shape for v in ref.trainable_variables]
    assert not gen.non_trainable_variables  # no moving statistics


def test_adamw_arguments():
    from spectrum_vae_amd.optimizers import AdamW
    for bad in (dict(weight_decay=-1.0), dict(global_clipnorm=0.0), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW(**bad)
    opt = AdamW(weight_decay=0.1)

    class V:
        name = "conv2d/bias"

    v = V()
    assert opt._decay_of(v) == 0.1
    opt.exclude_from_weight_decay(var_names=["bias"])
    assert opt._decay_of(v) == 0.0
    opt.exclude_from_weight_decay(var_list=[v])
    assert opt._decay_of(v) == 0.0
    opt._plans[0] = (None, None)
    with pytest.raises(ValueError, match="before the first step"):
        opt.exclude_from_weight_decay()
    with pytest.raises(ValueError, match="slabs"):
        opt.apply_model(None, slabs=[1])


def test_epsilons_out_of_range():
    from spectrum_vae_amd import _lib
    from spectrum_vae_amd.optimizers import AdamW
    with pytest.raises(ValueError, match="epsilon"):
        AdamW(epsilon=1e-13)
    p = 4096  # never read: the calls are refused before a launch
    for eps in (0.0, 1e-13, float("nan")):
        assert _lib.lib.sv_adamw_step(p, 1, 32, p, 1e-3, 0.9, 0.999, eps, 10, 0.9, 1, 1.0, 0.0, 0, 0, p, 1 << 20, None) == -1
        assert "epsilon" in _lib.last_error()
    for eps in (-1e-3, float("nan")):
        assert _lib.lib.sv_groupnorm_act_fwd(p, p, p, p, p, p, 2, 4, 8, 2, eps, 0, 0.2, p, 1 << 20, 0, None) == -1
        assert "epsilon" in _lib.last_error()


def test_more_workgroups_than_a_launch_takes():
    from spectrum_vae_amd import _lib
    p = 4096  # never read
    for n, s, c, g in ((1 << 24, 1, 32, 4), (1 << 23, 300, 130, 2)):
        need = _lib.lib.sv_groupnorm_workspace_bytes(n, s, c, g)
        assert _lib.lib.sv_groupnorm_act_fwd(p, p, p, p, p, p, n, s, c, g, 1e-3, 0, 0.2, p, need, 0, None) == -1
        assert "too many" in _lib.last_error()
        assert _lib.lib.sv_groupnorm_act_bwd(p, p, p, p, p, p, p, p, p, 0, n, s, c, g, 0, 0.2, p, need, 0, None) == -1
        assert "too many" in _lib.last_error()


# ------------------------------------------------------------------------------------------------ refusals
def test_groupnorm_refusals():
    from spectrum_vae_amd import _lib, ops
    lib = _lib.lib
    ok = dict(n=2, s=4, c=8, g=2, act=0, dtype=0, ws=1 << 20)

    def fwd(**kw):
        a = {**ok, **kw}
        p = 4096  # never read: the call is refused before a launch
        return lib.sv_groupnorm_act_fwd(p, p, p, a.get("y", p), a.get("mean", p), a.get("rstd", p), a["n"], a["s"], a["c"], a["g"],
                                        1e-3, a["act"], 0.2, a.get("wsp", p), a["ws"], a["dtype"], None)

    def bwd(**kw):
        a = {**ok, **kw}
        p = 4096
        return lib.sv_groupnorm_act_bwd(p, a.get("dy", p), p, p, a.get("mean", p), p, p, a.get("dgamma", p), p, 0, a["n"], a["s"],
                                        a["c"], a["g"], a["act"], 0.2, a.get("wsp", p), a["ws"], a["dtype"], None)

    for call in (fwd, bwd):
        for kw in (dict(n=-1), dict(s=0), dict(c=0), dict(c=5000, g=1), dict(g=3), dict(g=0), dict(act=6), dict(act=-1),
                   dict(n=1 << 40, s=1 << 20)):
            assert call(**kw) == -1, kw
        assert call(dtype=2) == -2
        assert call(ws=8) == -4 and call(wsp=None) == -4
    assert fwd(mean=None) == -1 and fwd(y=None) == -1
    assert bwd(dy=None) == -1 and bwd(dgamma=None) == -1 and bwd(mean=None) == -1
    assert fwd(n=0, wsp=None, ws=0) == 0
    assert lib.sv_groupnorm_workspace_bytes(2, 0, 8, 2) == 0 and lib.sv_groupnorm_workspace_bytes(2, 4, 8, 3) == 0
    x = torch.zeros(2, 4, 8)
    one, st = torch.zeros(8), torch.zeros(2, 2)
    with pytest.raises(_lib.SpectrumHipError, match="no CPU fallback"):
        ops.groupnorm_act_fwd(x, one, one, x.clone(), st, st.clone(), 2, 1e-3, None, 0.0, None)
    with pytest.raises(ValueError, match="do not split"):
        ops.groupnorm_act_fwd(x, one, one, x.clone(), st, st.clone(), 3, 1e-3, None, 0.0, None)
    with pytest.raises(ValueError, match="one shape"):
        ops.groupnorm_act_fwd(x, one, one, x[:1], st, st.clone(), 2, 1e-3, None, 0.0, None)
    with pytest.raises(ValueError, match="go together"):
        ops.groupnorm_act_fwd(x, one, one, x.clone(), st, None, 2, 1e-3, None, 0.0, None)
    with pytest.raises(ValueError, match="channels"):
        ops.groupnorm_act_fwd(x, one[:4], one, x.clone(), st, st.clone(), 2, 1e-3, None, 0.0, None)
    with pytest.raises(ValueError, match=r"\[N\]\[groups\]"):
        ops.groupnorm_act_fwd(x, one, one, x.clone(), st[:1], st.clone(), 2, 1e-3, None, 0.0, None)
    with pytest.raises(ValueError, match="saved statistics"):
        ops.groupnorm_act_bwd(x, x, one, one, None, None, x.clone(), one, one, False, 2, None, 0.0, None)


def _table(*rows):
    from spectrum_vae_amd._lib import AdamWTensor
    t = (AdamWTensor * len(rows))()
    for e, r in zip(t, rows):
        base = r.get("at", 1 << 20)
        d = dict(theta=base, grad=base + (1 << 16), m=base + (2 << 16), v=base + (3 << 16), m_exp=base + (4 << 16),
                 v_exp=base + (5 << 16), theta_bf16=None, n=1000, weight_decay=0.1, reserved=0)
        d.update({k: v for k, v in r.items() if k != "at"})
        for k, v in d.items():
            setattr(e, k, v)
    return t


def _fill(table, bits=32, nbytes=None):
    from spectrum_vae_amd import _lib
    chunks = C.c_int64(0)
    need = _lib.lib.sv_adamw_plan_bytes(table, len(table), C.byref(chunks))
    image = (C.c_char * max(need, 1))()
    return _lib.lib.sv_adamw_plan_fill(table, len(table), bits, image, need if nbytes is None else nbytes), chunks.value


def test_adamw_plan_refusals():
    from spectrum_vae_amd import _lib
    two = 1 << 24
    assert _fill(_table({}, {"at": two})) == (0, 2)
    assert _fill(_table({}, {"at": two, "n": 0, "theta": None})) == (0, 1)
    assert _fill(_table({"n": 8193}))[1] == 3
    assert _fill(_table({}), bits=8)[0] == 0
    for kw, text in ((dict(theta=None), "null"), (dict(theta=(1 << 20) + 2), "aligned"), (dict(weight_decay=-1.0), "decay"),
                     (dict(weight_decay=float("nan")), "decay"), (dict(grad=1 << 20), "overlap"),
                     (dict(m=(1 << 20) + 3996), "overlap")):
        assert _fill(_table(kw))[0] == -1, kw
        assert text in _lib.last_error(), (kw, _lib.last_error())
    assert _fill(_table({}, {}))[0] == -1  # the same tensor twice
    assert "overlap" in _lib.last_error()
    assert _fill(_table({"m_exp": None}), bits=8)[0] == -1
    assert _fill(_table({}), bits=16)[0] == -1
    assert _fill(_table({}), nbytes=8)[0] == -4
    assert _lib.lib.sv_adamw_plan_bytes(_table({"n": -1}), 1, C.byref(C.c_int64(0))) == 0


def test_adamw_step_refusals():
    from spectrum_vae_amd import _lib, ops
    lib = _lib.lib

    def step(plan=4096, chunks=1, bits=32, state=4096, b1=0.9, b2=0.999, eps=1e-7, rate=0.9, clip=0.0, ws=4096,
             nbytes=1 << 20):
        return lib.sv_adamw_step(plan, chunks, bits, state, 1e-3, b1, b2, eps, 10, rate, 1, 1.0, clip, 0, 0, ws, nbytes, None)

    for kw in (dict(plan=None), dict(state=None), dict(chunks=-1), dict(bits=4), dict(b1=1.0), dict(b2=-0.1),
               dict(eps=0.0), dict(rate=0.0), dict(clip=-1.0), dict(clip=1.0, ws=None), dict(plan=4097)):
        assert step(**kw) == -1, kw
    assert step(clip=1.0, nbytes=8) == -4
    assert lib.sv_adamw_decode(None, None, None, 5, 0, None) == -1 and lib.sv_adamw_decode(None, None, None, 0, 0, None) == 0
    t = torch.zeros(10)
    with pytest.raises(_lib.SpectrumHipError, match="no CPU fallback"):
        ops.AdamWPlan([t], [t], [t], [t], 0.0)
    with pytest.raises(ValueError, match="empty"):
        ops.AdamWPlan([], [], [], [], 0.0)
    with pytest.raises(ValueError, match="sizes"):
        ops.AdamWPlan([t], [t[:5]], [t], [t], 0.0)
    with pytest.raises(ValueError, match="parameters and"):
        ops.AdamWPlan([t], [t], [t], [t], [0.0, 0.0])
    with pytest.raises(ValueError, match="one exponent"):
        e = torch.zeros(2, dtype=torch.uint8)
        ops.AdamWPlan([t], [t], [t.byte()], [t.byte()], 0.0, m_exp=[e], v_exp=[e])
    with pytest.raises(ValueError, match="go together"):
        ops.AdamWPlan([t], [t], [t], [t], 0.0, m_exp=[e])
