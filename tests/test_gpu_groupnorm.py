"""Group norm + activation on the GPU against the float64 oracle.

Bounds, u = 2^-24 (half a step of float32):
 * z: the mean is off by at most 8 u max|x| of its group (sums of parts about a value of the group, joined in 64 bits), rstd by
   32 u relative (its half of a relative error of at most 64 u in the sum of squares, 64 rows a thread); xhat, the product and
   the sum add a rounding each:  e_z = |gamma| (8 u max|x| rstd + 34 u |xhat|) + 2 u (|z| + |beta|).
 * activations: slopes at most 1, their own error below 3e-7.  bfloat16 outputs: 2^-8 relative.
 * backward, from given statistics: e_z = 4 u (|xhat gamma| + |beta|); the slope moves by at most e_z away from a corner
   (relu / lrelu inputs keep clear of it, checked) and has an error below 3e-7 of its own; sums of n terms: 128 u of the sum of
   magnitudes (chains of at most 64 in a thread, then joined).
"""
import numpy as np
import pytest
import torch

from oracle import np_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-3


def _dev(a, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)


def _host(t):
    return t.detach().double().cpu().numpy()


class Case:
    def __init__(self, shape, groups, act, dtype, seed=0, shift=1.0):
        rng = np.random.default_rng(seed + sum(shape))
        self.shape, self.groups, self.act, self.dtype = shape, groups, act, dtype
        c = shape[-1]
        x = rng.standard_normal(shape) * (0.3 + rng.random(c)) + shift * rng.standard_normal(c)
        self.xt = _dev(x, dtype)
        self.gamma, self.beta = (1 + 0.2 * rng.standard_normal(c)).astype(np.float32), (0.2 * rng.standard_normal(c)).astype(np.float32)
        self.dyt = _dev(rng.standard_normal(shape), dtype)
        self.x, self.dy = _host(self.xt), _host(self.dyt)
        self.gt, self.bt = _dev(self.gamma), _dev(self.beta)
        self.half = 0.0 if dtype == torch.float32 else 2.0 ** -8

    def per_channel(self, a):
        """[N, G] -> broadcastable over [N, ..., C]."""
        c = self.shape[-1]
        return np.repeat(a, c // self.groups, axis=1).reshape((self.shape[0],) + (1,) * (len(self.shape) - 2) + (c,))

    def ws(self):
        from spectrum_vae_amd import ops
        n, c = self.shape[0], self.shape[-1]
        nbytes = ops.groupnorm_workspace(n, int(np.prod(self.shape[1:-1])), c, self.groups)
        return torch.full((max(nbytes, 1),), 255, dtype=torch.uint8, device="cuda")  # NaN wherever it is read unwritten

    def forward(self, xt=None, y=None):
        from spectrum_vae_amd import ops
        xt = self.xt if xt is None else xt
        y = torch.empty_like(xt) if y is None else y
        mean, rstd = (torch.empty(self.shape[0], self.groups, device="cuda") for _ in range(2))
        ops.groupnorm_act_fwd(xt, self.gt, self.bt, y, mean, rstd, self.groups, EPS, self.act, 0.2, self.ws())
        return y, mean, rstd

    def check_forward(self, y, mean, rstd):
        want, mu, rs = np_ops.group_norm(self.x, self.gamma, self.beta, self.groups, EPS, self.act)
        n, c, g = self.shape[0], self.shape[-1], self.groups
        big = np.abs(self.x).reshape(n, -1, g, c // g).max(axis=(1, 3))
        assert (np.abs(_host(mean) - mu) <= 8 * U * big).all()
        assert (np.abs(_host(rstd) - rs) <= rs * (33 * U + (8 * U * big * rs) ** 2)).all()
        xhat = (self.x - self.per_channel(mu)) * self.per_channel(rs)
        z = xhat * self.gamma + self.beta
        e_z = np.abs(self.gamma) * (self.per_channel(8 * U * big * rs) + 34 * U * np.abs(xhat)) + 2 * U * (np.abs(z) + np.abs(self.beta))
        err = np.abs(_host(y) - want)
        tol = e_z + 3e-7 + self.half * np.abs(want)
        assert np.isfinite(_host(y)).all() and (err <= tol).all(), (err / tol).max()

    def backward(self, xt=None, dyt=None, dx=None, accumulate=False, dgamma=None, dbeta=None):
        from spectrum_vae_amd import ops
        xt, dyt = self.xt if xt is None else xt, self.dyt if dyt is None else dyt
        _, mu, rs = np_ops.group_norm(self.x, self.gamma, self.beta, self.groups, EPS, self.act)
        self.mean, self.rstd = _dev(mu), _dev(rs)
        dx = torch.empty_like(xt) if dx is None else dx
        c = self.shape[-1]
        dgamma = torch.full((c,), float("nan"), device="cuda") if dgamma is None else dgamma
        dbeta = torch.full((c,), float("nan"), device="cuda") if dbeta is None else dbeta
        ops.groupnorm_act_bwd(xt, dyt, self.gt, self.bt, self.mean, self.rstd, dx, dgamma, dbeta, accumulate, self.groups,
                              self.act, 0.2, self.ws())
        return dx, dgamma, dbeta

    def check_backward(self, dx, dgamma, dbeta, base=None):
        mu, rs = _host(self.mean), _host(self.rstd)
        want, dg, db = np_ops.group_norm_bwd(self.x, self.dy, self.gamma, self.beta, mu, rs, self.groups, self.act)
        n, c, g = self.shape[0], self.shape[-1], self.groups
        xhat = (self.x - self.per_channel(mu)) * self.per_channel(rs)
        z = xhat * self.gamma + self.beta
        e_z = 4 * U * (np.abs(xhat * self.gamma) + np.abs(self.beta))
        if self.act in ("relu", "lrelu"):
            assert (np.abs(z) > e_z).all(), "an input lies on the corner: this seed cannot be used"
        e_s = 0.0 if self.act in (None, "relu", "lrelu") else e_z + 3e-7
        dz = self.dy * np_ops.act_slope(z, self.act)
        e_dz = np.abs(self.dy) * e_s + 3 * U * np.abs(dz)
        axes = tuple(range(len(self.shape) - 1))
        for got, exact, weight, extra in ((dgamma, dg, np.abs(xhat), 3 * U), (dbeta, db, np.ones_like(xhat), 0.0)):
            tol = ((e_dz + (128 * U + extra) * np.abs(dz)) * weight).sum(axis=axes) + U * np.abs(exact)
            err = np.abs(_host(got) - exact - (0 if base is None else base))
            tol = tol + (0 if base is None else 2 * U * (np.abs(exact) + abs(base)))
            assert (err <= tol).all(), (err / np.maximum(tol, 1e-300)).max()
        v = lambda a: a.reshape(n, -1, g, c // g)  # noqa: E731
        gz, e_gz = dz * self.gamma, e_dz * np.abs(self.gamma) + U * np.abs(dz * self.gamma)
        c1 = v(gz).mean(axis=(1, 3))
        c2 = v(gz * xhat).mean(axis=(1, 3))
        e_c1 = v(e_gz + 128 * U * np.abs(gz)).mean(axis=(1, 3)) + U * np.abs(c1)
        e_c2 = v((e_gz + 131 * U * np.abs(gz)) * np.abs(xhat)).mean(axis=(1, 3)) + U * np.abs(c2)
        p = self.per_channel
        size = np.abs(gz) + np.abs(p(c1)) + np.abs(xhat * p(c2))
        tol = p(rs) * (e_gz + p(e_c1) + np.abs(xhat) * p(e_c2) + 6 * U * size) + self.half * np.abs(want)
        err = np.abs(_host(dx) - want)
        assert (err <= tol).all(), (err / tol).max()


SHAPES = [
    ((1, 1, 1, 8), 2), ((2, 1, 1, 6), 6), ((3, 5, 7, 12), 3), ((2, 8, 8, 64), 8), ((5, 4, 4, 90), 9), ((1, 33, 31, 10), 5),
    ((4, 16, 16, 128), 32), ((2, 3, 5, 7), 1), ((2, 2, 3, 7), 7), ((9, 6), 2), ((3, 300), 4), ((2, 9, 1000), 8),
    ((1, 64, 64, 64), 8), ((2, 160, 128, 16), 4), ((1, 2, 2, 4096), 1), ((1, 3, 2, 4095), 5), ((130, 2, 2, 32), 8),
    ((2, 40, 40, 36), 2), ((1, 257, 129, 24), 3), ((3, 96, 4), 4), ((2, 50, 50, 66), 11),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_group_norm(shape, groups, dtype):
    k = Case(shape, groups, "elu", dtype)
    k.check_forward(*k.forward())
    k.check_backward(*k.backward())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "elu", "lrelu", "tanh", "sigmoid"])
@pytest.mark.parametrize("shape,groups", [((3, 9, 5, 24), 4), ((1, 70, 70, 12), 3), ((2, 16, 16, 64), 8)])
def test_activations(shape, groups, act, dtype):
    k = Case(shape, groups, act, dtype, seed=5)
    k.check_forward(*k.forward())
    k.check_backward(*k.backward())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((2, 8, 8, 64), 8), ((1, 70, 66, 64), 8), ((3, 5, 7, 12), 3)])
def test_tensors_off_every_alignment_and_their_neighbours(shape, groups, dtype):
    """Every tensor starts one element behind an aligned address; what lies in front of and behind the outputs stays."""
    k = Case(shape, groups, "lrelu", dtype, seed=11)
    n = int(np.prod(shape))

    def off(t=None):
        whole = torch.full((n + 17,), 7.0, dtype=dtype, device="cuda")
        if t is not None:
            whole[1:n + 1] = t.reshape(-1)
        return whole, whole[1:n + 1].view(shape)

    (_, x), (yw, y), (_, dy), (dxw, dx) = off(k.xt), off(), off(k.dyt), off()
    k.check_forward(*k.forward(x, y))
    k.check_backward(*k.backward(x, dy, dx))
    for w in (yw, dxw):
        assert w[0] == 7 and (w[n + 1:] == 7).all()
    # the same values as on aligned tensors
    assert torch.allclose(y.float(), k.forward()[0].float(), rtol=2e-2 if dtype == torch.bfloat16 else 1e-5, atol=1e-5)


def test_values_far_from_zero_keep_their_variance():
    """A level 300 times the spread: the variance comes from differences to a value of the group, not from squares."""
    rng = np.random.default_rng(2)
    for shape in [(2, 16, 16, 16), (1, 96, 96, 16)]:
        k = Case(shape, 4, None, torch.float32)
        k.xt = _dev(300.0 + rng.standard_normal(shape))
        k.x = _host(k.xt)
        y, mean, rstd = k.forward()
        want, mu, rs = np_ops.group_norm(k.x, k.gamma, k.beta, 4, EPS, None)
        assert np.abs(_host(mean) - mu).max() <= 8 * U * 305
        assert (np.abs(_host(rstd) - rs) / rs).max() <= 33 * U + (8 * U * 305) ** 2
        # the mean's error, up to half a step at 300, is what y carries
        assert np.abs(_host(y) - want).max() <= 2 * (8 * U * 305) * rs.max() + 1e-5


def test_outlier_first_and_constant_groups():
    k = Case((2, 40, 40, 8), 2, None, torch.float32)
    k.xt[:, 0, 0, :] = 1e4  # the values that sums are formed about
    k.xt[1, :, :, 4:] = 3.0  # variance exactly 0
    k.x = _host(k.xt)
    y, mean, rstd = k.forward()
    _, mu, rs = np_ops.group_norm(k.x, k.gamma, k.beta, 2, EPS, None)
    # one chunk's threads sum up to 64 rows about the outlier: relative error of its part of the squares below 64^2 u
    assert (np.abs(_host(rstd) - rs) / rs).max() <= 64 ** 2 * U
    assert (np.abs(_host(mean) - mu) <= 8 * U * 1e4).all()
    assert torch.allclose(y[1, :, :, 4:], k.bt[4:].expand(40, 40, 4), atol=0, rtol=0)


def test_not_finite_values_stay_in_their_group():
    k = Case((3, 20, 20, 12), 3, "elu", torch.float32)
    clean, _, _ = k.forward()
    dclean, _, _ = k.backward()
    bad, badg = k.xt.clone(), k.dyt.clone()
    bad[1, 3, 3, 5] = float("nan")
    bad[2, 0, 0, 0] = float("inf")
    badg[0, 1, 1, 9] = float("nan")
    y, _, _ = k.forward(bad)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[1, :, :, 4:8] = True
    hit[2, :, :, 0:4] = True
    assert not torch.isfinite(y[hit]).any() and torch.equal(y[~hit], clean[~hit])
    dx, dg, db = k.backward(None, badg)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[0, :, :, 8:12] = True
    assert not torch.isfinite(dx[hit]).any() and torch.equal(dx[~hit], dclean[~hit])
    assert torch.isnan(dg[9]) and torch.isnan(db[9]) and torch.isfinite(dg[:9]).all()


@pytest.mark.parametrize("shape,groups", [((5, 8, 8, 64), 8), ((2, 80, 80, 20), 5)])
def test_accumulation_no_samples_and_no_statistics(shape, groups):
    from spectrum_vae_amd import ops
    k = Case(shape, groups, "tanh", torch.float32)
    c = shape[-1]
    dg, db = torch.full((c,), 2.5, device="cuda"), torch.full((c,), 2.5, device="cuda")
    k.check_backward(*k.backward(accumulate=True, dgamma=dg, dbeta=db), base=2.5)
    # inference: no statistics handed out
    y = torch.empty_like(k.xt)
    ops.groupnorm_act_fwd(k.xt, k.gt, k.bt, y, None, None, groups, EPS, k.act, 0.2, k.ws())
    assert torch.equal(y, k.forward()[0])
    # no samples: parameter gradients are zero, or what they were
    none, st = k.xt[:0], torch.empty(0, groups, device="cuda")
    ops.groupnorm_act_fwd(none, k.gt, k.bt, none.clone(), st, st.clone(), groups, EPS, k.act, 0.2, None)
    keep = dg.clone()
    ops.groupnorm_act_bwd(none, none, k.gt, k.bt, st, st.clone(), none.clone(), dg, db, True, groups, k.act, 0.2, None)
    assert torch.equal(dg, keep)
    ops.groupnorm_act_bwd(none, none, k.gt, k.bt, st, st.clone(), none.clone(), dg, db, False, groups, k.act, 0.2, None)
    assert not dg.any() and not db.any()


@pytest.mark.parametrize("shape,groups,dtype", [((6, 8, 8, 64), 8, torch.float32), ((2, 96, 80, 32), 4, torch.bfloat16)])
def test_repeats_other_streams_and_graph_replays_give_the_same_bits(shape, groups, dtype):
    from spectrum_vae_amd import ops
    k = Case(shape, groups, "elu", dtype)
    y, mean, rstd = k.forward()
    dx, dg, db = k.backward()
    first = [t.clone() for t in (y, mean, rstd, dx, dg, db)]
    ws = k.ws()

    def both():
        ops.groupnorm_act_fwd(k.xt, k.gt, k.bt, y, mean, rstd, groups, EPS, k.act, 0.2, ws)
        ops.groupnorm_act_bwd(k.xt, k.dyt, k.gt, k.bt, k.mean, k.rstd, dx, dg, db, False, groups, k.act, 0.2, ws)

    def same():
        return all(torch.equal(a, b) for a, b in zip(first, (y, mean, rstd, dx, dg, db)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in (y, mean, rstd, dx, dg, db):
            t.fill_(7)
        both()
    torch.cuda.current_stream().wait_stream(side)
    assert same()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for _ in range(3):
        for t in (y, mean, rstd, dx, dg, db):
            t.fill_(7)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert same()


def test_gradients_against_differences():
    """d sum(y * w) along a random direction, from the kernels' own forward pass: a step h moves the loss by h times the
    derivative; float32 outputs round it by about 1e-7 * sqrt(count) * |w| / h."""
    k = Case((2, 6, 5, 16), 4, "tanh", torch.float32, seed=3)
    y, mean, rstd = k.forward()
    dx, dg, db = k.backward()
    rng = np.random.default_rng(9)
    direction = rng.standard_normal(k.shape)
    direction /= np.linalg.norm(direction)
    h = 0.05
    up, down = (k.forward(_dev(k.x + s * h * direction))[0] for s in (1, -1))
    num = ((_host(up) - _host(down)) * k.dy).sum() / (2 * h)
    ana = (_host(dx) * direction).sum()
    # rounding: 960 outputs off by up to 3e-7 each way over 2 h; the third derivative's share: checked with the oracle
    f = lambda t: (np_ops.group_norm(k.x + t * direction, k.gamma, k.beta, 4, EPS, "tanh")[0] * k.dy).sum()  # noqa: E731
    curve = abs((f(h) - f(-h)) / (2 * h) - (f(1e-5) - f(-1e-5)) / 2e-5)
    assert abs(num - ana) <= 2 * curve + 2 * 6e-7 * np.abs(k.dy).sum() / (2 * h) / np.sqrt(960) + 1e-4


# Rows and channels that lie on both sides of every length at which the work is laid out differently: samples kept on the chip from
# 64 rows of one line to some thousands, more samples than one and more slabs than one, groups that end inside a slab, samples too
# long to keep with few and with many parts.
LAYOUTS = [
    ((33, 16, 64), 8), ((33, 64, 64), 8), ((33, 65, 64), 8), ((33, 129, 64), 8), ((33, 257, 64), 8), ((33, 1024, 64), 8),
    ((17, 1025, 64), 8), ((33, 1100, 64), 4), ((33, 2049, 32), 4), ((33, 257, 40), 8), ((70, 520, 40), 8), ((33, 1030, 40), 8),
    ((70, 2050, 20), 4), ((150, 12, 256), 16), ((151, 50, 96), 12), ((9, 100, 512), 4), ((3, 300, 1500), 12), ((2, 300, 4000), 32),
    ((2, 5000, 36), 9), ((4, 8200, 27), 3), ((20, 4100, 6), 2), ((1, 70_000, 8), 8), ((300, 1, 48), 3), ((2100, 3, 6), 3),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", LAYOUTS)
def test_every_layout(shape, groups, dtype):
    k = Case(shape, groups, "tanh", dtype, seed=17)
    k.check_forward(*k.forward())
    k.check_backward(*k.backward())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((5, 8, 8, 64), 8), ((2, 96, 80, 36), 4), ((3, 300, 1500), 12)])
def test_in_place(shape, groups, dtype):
    """y may be x, and dx may be dy or x: every element is read before it is written, by the thread that writes it."""
    k = Case(shape, groups, "elu", dtype, seed=1)
    y, mean, rstd = k.forward()
    x = k.xt.clone()
    got = k.forward(x, x)
    assert all(torch.equal(a, b) for a, b in zip(got, (y, mean, rstd)))
    want = k.backward()
    dy, x = k.dyt.clone(), k.xt.clone()
    for got in (k.backward(None, dy, dy), k.backward(x, None, x)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def _reference_pieces(x, dy, gamma, beta, mean, rstd, act_slope, act):
    """z, dz, xhat in float64 of rows [r, C] of one sample."""
    c = x.shape[-1]
    rep = lambda t: t.double().repeat_interleave(c // t.numel())  # noqa: E731
    xhat = (x.double() - rep(mean)) * rep(rstd)
    z = xhat * gamma.double() + beta.double()
    return xhat, act(z), (dy.double() * act_slope(z) if dy is not None else None)


@pytest.mark.parametrize("shape,groups", [((1, 68_000_000, 32), 4), ((600_000, 64, 64), 8)])
def test_more_than_2_to_the_31_elements(shape, groups):
    """One sample, and many, of more elements than 31 bits count.  Chains of up to L = 68e6 / 2048 / 64 = 519 rows a thread: a mean
    is off by at most L u of the mean magnitude (below 2 at unit spread), likewise the backward means and the channel sums."""
    from spectrum_vae_amd import ops
    n, s, c = shape
    L, half = 520, 2.0 ** -8
    g = torch.Generator(device="cuda").manual_seed(5)
    x, dy = (torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for t in (x, dy):
        for part in t.view(-1).split(1 << 28):
            part.normal_(0.25, 1.0, generator=g)
    gamma, beta = 1 + 0.1 * torch.randn(c, device="cuda", generator=g), 0.1 * torch.randn(c, device="cuda", generator=g)
    y, mean, rstd = torch.empty_like(x), torch.empty(n, groups, device="cuda"), torch.empty(n, groups, device="cuda")
    ws = torch.empty(ops.groupnorm_workspace(n, s, c, groups), dtype=torch.uint8, device="cuda")
    ops.groupnorm_act_fwd(x, gamma, beta, y, mean, rstd, groups, EPS, "tanh", 0.0, ws)
    slope = lambda z: 1 - torch.tanh(z) ** 2  # noqa: E731
    d = c // groups
    per = 1 << 20
    looked = [0] if n == 1 else [0, 1, n // 2, n - 1]
    sums = {}
    for i in looked:
        tot, sq = torch.zeros(groups, device="cuda", dtype=torch.float64), torch.zeros(groups, device="cuda", dtype=torch.float64)
        for a in range(0, s, per):
            q = x[i, a:a + per].double().view(-1, groups, d)
            tot += q.sum(dim=(0, 2))
            sq += (q * q).sum(dim=(0, 2))
        mu = tot / (s * d)
        rs = (sq / (s * d) - mu * mu + EPS).rsqrt()
        assert ((mean[i].double() - mu).abs() <= 2 * L * U).all()
        assert ((rstd[i].double() / rs - 1).abs() <= 2 * L * U).all()
        sums[i] = (mu, rs)
        for a in (0, s // 2, s - 7):
            _, want, _ = _reference_pieces(x[i, a:a + 7], None, gamma, beta, mu, rs, slope, torch.tanh)
            assert ((y[i, a:a + 7].double() - want).abs() <= half * want.abs() + 8 * L * U).all()
    dx, dgamma, dbeta = y, torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    ops.groupnorm_act_bwd(x, dy, gamma, beta, mean, rstd, dx, dgamma, dbeta, False, groups, "tanh", 0.0, ws)
    for i in looked:
        c1, c2 = torch.zeros(groups, device="cuda", dtype=torch.float64), torch.zeros(groups, device="cuda", dtype=torch.float64)
        for a in range(0, s, per):
            xhat, _, dz = _reference_pieces(x[i, a:a + per], dy[i, a:a + per], gamma, beta, mean[i], rstd[i], slope, torch.tanh)
            gz = (dz * gamma.double()).view(-1, groups, d)
            c1 += gz.sum(dim=(0, 2))
            c2 += (gz * xhat.view(-1, groups, d)).sum(dim=(0, 2))
        c1, c2 = (t.repeat_interleave(d) / (s * d) for t in (c1, c2))
        for a in (0, s // 2, s - 7):
            xhat, _, dz = _reference_pieces(x[i, a:a + 7], dy[i, a:a + 7], gamma, beta, mean[i], rstd[i], slope, torch.tanh)
            want = rstd[i].double().repeat_interleave(d) * (dz * gamma.double() - c1 - xhat * c2)
            assert ((dx[i, a:a + 7].double() - want).abs() <= half * want.abs() + 8 * L * U * (1 + xhat.abs() + dz.abs())).all()
    dg, db, mag = (torch.zeros(c, device="cuda", dtype=torch.float64) for _ in range(3))
    rows, step = x.view(-1, c), per // s * s if n > 1 else per
    for a in range(0, n * s, step):
        q = slice(a, a + step)
        st = (mean, rstd) if n == 1 else (mean[a // s:(a + step) // s], rstd[a // s:(a + step) // s])
        at = [t.double().repeat_interleave(d, dim=1).repeat_interleave(1 if n == 1 else s, dim=0) for t in st]
        xhat = (rows[q].double() - at[0]) * at[1]
        dz = dy.view(-1, c)[q].double() * slope(xhat * gamma.double() + beta.double())
        dg += (dz * xhat).sum(dim=0)
        db += dz.sum(dim=0)
        mag += (dz.abs() * (1 + xhat.abs())).sum(dim=0)
    # up to L terms in a chain, and 10 u of each term's own (statistics, activation, products)
    assert ((dgamma.double() - dg).abs() <= (L + 10) * U * mag).all() and ((dbeta.double() - db).abs() <= (L + 10) * U * mag).all()


def test_two_calls_at_once_and_two_graphs_with_one_workspace():
    """Calls on two streams with workspaces of their own do not disturb each other; two recorded graphs that share a workspace
    give the eager bits in any order of replays, with other work in between."""
    from spectrum_vae_amd import ops
    a, b = Case((3, 120, 100, 48), 6, "elu", torch.bfloat16), Case((4, 64, 70, 20), 4, "tanh", torch.float32)
    want = [[t.clone() for t in (*k.forward(), *k.backward())] for k in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for st, k in zip(streams, (a, b)):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append((*k.forward(), *k.backward()))
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))
    nbytes = max(ops.groupnorm_workspace(k.shape[0], k.shape[1] * k.shape[2], k.shape[3], k.groups) for k in (a, b))
    ws = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
    graphs, outs = [], []
    for k in (a, b):
        y, mean, rstd = torch.empty_like(k.xt), *(torch.empty(k.shape[0], k.groups, device="cuda") for _ in range(2))
        dx, dg, db = torch.empty_like(k.xt), *(torch.empty(k.shape[-1], device="cuda") for _ in range(2))

        def run():
            ops.groupnorm_act_fwd(k.xt, k.gt, k.bt, y, mean, rstd, k.groups, EPS, k.act, 0.2, ws)
            ops.groupnorm_act_bwd(k.xt, k.dyt, k.gt, k.bt, k.mean, k.rstd, dx, dg, db, False, k.groups, k.act, 0.2, ws)

        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append(graph)
        outs.append((y, mean, rstd, dx, dg, db))
    for order in ((0, 1), (1, 0), (0, 0), (1, 1)):
        for i in order:
            for t in outs[i]:
                t.fill_(7)
            graphs[i].replay()
            torch.zeros(1000, device="cuda").add_(1)
        torch.cuda.synchronize()
        for i in set(order):
            assert all(torch.equal(x, y) for x, y in zip(outs[i], want[i]))


def test_strided_tensors_and_other_types_are_refused():
    from spectrum_vae_amd import ops
    k = Case((2, 4, 4, 8), 2, None, torch.float32)
    y, st = torch.empty_like(k.xt), torch.empty(2, 2, device="cuda")
    call = lambda x, y, ws=None: ops.groupnorm_act_fwd(x, k.gt, k.bt, y, st, st.clone(), 2, EPS, None, 0.0, k.ws() if ws is None else ws)  # noqa: E731
    for bad in (k.xt.transpose(1, 2), k.xt.half(), k.xt.double()):
        with pytest.raises((TypeError, ValueError)):
            call(bad, y)
    with pytest.raises((TypeError, ValueError)):
        call(k.xt, y.to(torch.bfloat16))
    with pytest.raises(ValueError, match="one device"):
        ops.groupnorm_act_fwd(k.xt, k.gt.cpu(), k.bt, y, st, st.clone(), 2, EPS, None, 0.0, k.ws())
    from spectrum_vae_amd import _lib
    with pytest.raises(_lib.SpectrumHipError, match="workspace"):
        call(k.xt, y, k.ws()[:16])


def test_a_view_of_half_a_call_goes_back_as_a_call_of_its_own():
    """The generated half of a discriminator's [real; generated] call: the gradient through the view is that of a call on those
    samples alone, and inference gives what the training call gave."""
    from spectrum_vae_amd import unet
    rng = np.random.default_rng(6)
    disc = unet.Discriminator(normalization="group")
    disc.build_graph((1, 32, 32, 4))
    disc._materialize(torch.device("cuda", 0))
    both = torch.from_numpy(rng.standard_normal((6, 32, 32, 4)).astype(np.float32)).cuda()
    z = disc.forward_raw(both, True, bn_groups=2).clone()
    dz = torch.from_numpy(rng.standard_normal(tuple(z[3:].shape)).astype(np.float32)).cuda()
    view = disc._calls[0].group_view(1)
    view.param_grads = False
    disc.zero_grad_raw()
    through = disc.backward(view, dz, need_dx=True).clone()
    assert not disc._grads.any()
    alone = unet.Discriminator(normalization="group")
    alone.build_graph((1, 32, 32, 4))
    alone._materialize(torch.device("cuda", 0))
    alone._params.copy_(disc._params)
    z_alone = alone.forward_raw(both[3:].contiguous(), True).clone()
    # layers of other extents may sum in another order
    assert torch.allclose(z_alone, z[3:], rtol=1e-4, atol=1e-5)
    dx = alone.backward(alone._calls[0], dz.clone(), need_dx=True)
    assert float((dx - through).norm() / through.norm()) <= 1e-4
    one = disc.predict(both[4:5].cpu().numpy(), batch_size=1)
    assert np.allclose(one.reshape(-1), z[4].cpu().numpy().reshape(-1), rtol=1e-4, atol=1e-5)
