"""AdamW over many tensors on the GPU against the oracle.

Bounds, u = 2^-24: the moments take three roundings of their terms, m off by 4 u (|b1 m| + |(1 - b1) g|); the step
alpha m / (sqrt(v) + eps) takes 8 u of itself and what m and v (3 u) bring, theta two roundings.  8-bit codes are held to exact
equality with the oracle's encoding of the moments that the same float32 operations give (numpy rounds each as IEEE)."""
import numpy as np
import pytest
import torch

from oracle import np_ops
from oracle.np_ops import Moments8

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F = np.float32


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


class Tensors:
    """Host copies and device tensors of a list of parameters; ``off``: elements in front of each (alignment)."""

    def __init__(self, sizes, bits, seed=0, off=0, copies=True, decay=0.1):
        rng = np.random.default_rng(seed)
        self.sizes, self.bits = sizes, bits
        self.theta = [rng.standard_normal(n).astype(F) * F(0.1) for n in sizes]
        spread = [np.exp(2 * rng.standard_normal(n)).astype(F) for n in sizes]
        self.grads = [(rng.standard_normal(n).astype(F) * s * F(1e-2)) for n, s in zip(sizes, spread)]
        self.m = [(rng.standard_normal(n).astype(F) * s * F(3e-3)) for n, s in zip(sizes, spread)]
        self.v = [(np.square(rng.standard_normal(n).astype(F) * s * F(1e-2)) + F(1e-10)) for n, s in zip(sizes, spread)]
        self.decay = [decay if i % 2 == 0 else 0.0 for i in range(len(sizes))]
        if bits == 8:
            half = [np.full(n, 1 << 15) for n in sizes]
            self.m_code = [Moments8.encode(a, h, 4) for a, h in zip(self.m, half)]
            self.v_code = [Moments8.encode(a, h, 5) for a, h in zip(self.v, half)]
            self.m = [Moments8.decode(c, e, 4) for c, e in self.m_code]
            self.v = [Moments8.decode(c, e, 5) for c, e in self.v_code]

        def put(arrays, dtype=None):
            out = []
            for a in arrays:
                t = _dev(a, dtype)
                whole = torch.full((a.size + off + 9,), 77, dtype=t.dtype, device="cuda")
                whole[off:off + a.size] = t
                out.append(whole[off:off + a.size])
                self.whole.append((whole, off, a.size))
            return out

        self.whole = []
        self.theta_t, self.grads_t = put(self.theta), put(self.grads)
        self.lp_t = put(self.theta, torch.bfloat16) if copies else None
        self.me_t = self.ve_t = None
        if bits == 8:
            self.m_t, self.v_t = put([c for c, _ in self.m_code]), put([c for c, _ in self.v_code])
            self.me_t, self.ve_t = put([e for _, e in self.m_code]), put([e for _, e in self.v_code])
        else:
            self.m_t, self.v_t = put(self.m), put(self.v)

    def plan(self):
        from spectrum_vae_amd import ops
        return ops.AdamWPlan(self.theta_t, self.grads_t, self.m_t, self.v_t, self.decay, m_exp=self.me_t, v_exp=self.ve_t,
                             params_lp=self.lp_t)

    def check(self, it, lr, scale=1.0, seed=0, slack=0.0):
        """The device tensors after one step from the host copies, which are moved on; ``slack``: relative error of the
        gradients' common scale."""
        blocks = np.cumsum([0] + [-(-n // 256) for n in self.sizes])
        b1, b2 = 0.9, 0.999
        for i, n in enumerate(self.sizes):
            g64 = self.grads[i].astype(np.float64) * scale
            th, m, v = np_ops.adamw_step(self.theta[i], g64, self.m[i].astype(np.float64), self.v[i].astype(np.float64), it, lr,
                                         self.decay[i])
            e_g = np.abs(g64) * (U + slack)
            e_m = 4 * U * (np.abs(b1 * self.m[i]) + np.abs((1 - b1) * g64)) + (1 - b1) * e_g
            e_v = 5 * U * v + 2 * (1 - b2) * np.abs(g64) * e_g
            alpha = lr * np.sqrt(1 - b2 ** (it + 1)) / (1 - b1 ** (it + 1))
            step = alpha * m / (np.sqrt(v) + 1e-7)
            e_step = 8 * U * np.abs(step) + alpha * e_m / (np.sqrt(v) + 1e-7) + np.abs(step) * e_v / np.maximum(2 * v, 1e-300)
            got = self.theta_t[i].double().cpu().numpy()
            tol = e_step + 4 * U * (np.abs(self.theta[i]) + np.abs(th))
            assert (np.abs(got - th) <= tol).all(), (i, n, (np.abs(got - th) / tol).max())
            if self.lp_t is not None:
                assert torch.equal(self.lp_t[i], self.theta_t[i].to(torch.bfloat16))
            if self.bits == 32:
                for t, want, e in ((self.m_t[i], m, e_m), (self.v_t[i], v, e_v)):
                    assert (np.abs(t.double().cpu().numpy() - want) <= e + 1e-44).all()
                self.m[i], self.v[i] = self.m_t[i].cpu().numpy(), self.v_t[i].cpu().numpy()
            else:
                gs = self.grads[i] * F(scale)
                mf = F(b1) * self.m[i] + F(1 - b1) * gs
                vf = F(b2) * self.v[i] + F(1 - b2) * (gs * gs)
                r = Moments8.random_bits(n, int(blocks[i]), it, seed)
                for val, rnd, width, ct, et, name in ((mf, r[0], 4, self.m_t[i], self.me_t[i], "m"), (vf, r[1], 5, self.v_t[i], self.ve_t[i], "v")):
                    code, exp = Moments8.encode(val, rnd, width)
                    assert np.array_equal(et.cpu().numpy(), exp), (i, name)
                    if slack == 0.0:
                        assert np.array_equal(ct.cpu().numpy(), code), (i, name)
                self.m[i] = Moments8.decode(self.m_t[i].cpu().numpy(), self.me_t[i].cpu().numpy(), 4)
                self.v[i] = Moments8.decode(self.v_t[i].cpu().numpy(), self.ve_t[i].cpu().numpy(), 5)
            self.theta[i] = self.theta_t[i].cpu().numpy()
        for whole, off, n in self.whole:  # what lies around every buffer
            assert (whole[:off] == 77).all() and (whole[off + n:] == 77).all()


SIZES = [[1], [3, 1, 2], [256], [255, 257, 4096, 4097, 1], [0, 5, 0, 300], [216, 8, 1152, 16, 4608, 32, 4608, 16, 1152, 8, 216, 3],
         [70_001], [9, 40_000, 4095, 8193]]


@pytest.mark.parametrize("off", [0, 1, 4])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s))[:24])
def test_three_steps(sizes, bits, off):
    from spectrum_vae_amd import ops
    t = Tensors(sizes, bits, seed=sum(sizes), off=off, copies=off != 4)
    plan = t.plan()
    state = torch.tensor([7, 0, 0], dtype=torch.int64, device="cuda")
    for it in (7, 8, 9):
        ops.adamw_step(plan, state, 1e-3, 0.9, 0.999, 1e-7, 4, 0.9, True, 0.5, seed=99)
        t.check(it, np_ops.exponential_decay(1e-3, it, 4, 0.9, True), 0.5, seed=99)
    host = state.cpu()
    assert int(host[0]) == 10 and int(host[2]) == 0
    lr = host[1:2].view(torch.float32)
    assert abs(float(lr[1]) - np_ops.exponential_decay(1e-3, 9, 4, 0.9, True)) < 1e-9


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [1e-3, 1e9])
def test_clip_by_the_global_norm(clip, bits):
    from spectrum_vae_amd import ops
    t = Tensors([300, 70_001, 1, 8193], bits, seed=4)
    norm = 0.5 * np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in t.grads))
    state = torch.zeros(3, dtype=torch.int64, device="cuda")
    ops.adamw_step(t.plan(), state, 1e-3, 0.9, 0.999, 1e-7, grad_scale=0.5, clip_norm=clip, seed=5)
    # squares summed in chains of 16 in 32 bits, then in 64: 16 u of the norm's square, half of it in the norm
    t.check(0, 1e-3, 0.5 * clip / max(clip, norm), seed=5, slack=10 * U if clip < norm else 0.0)


def test_gradients_that_are_not_finite():
    from spectrum_vae_amd import ops
    for bits in (32, 8):
        t = Tensors([600, 300], bits, seed=1)
        before = [a.copy() for a in t.theta]
        t.grads_t[0][300] = float("nan")
        t.grads_t[1][2] = float("inf")
        state = torch.zeros(3, dtype=torch.int64, device="cuda")
        ops.adamw_step(t.plan(), state, 1e-3, 0.9, 0.999, 1e-7, seed=5)
        finite = [torch.isfinite(x).cpu().numpy() for x in t.theta_t]
        assert not finite[0][300] and finite[0].sum() == 599 and finite[1].sum() == 299 and not finite[1][2]
        if bits == 8:  # their blocks of 256, and no others
            out = torch.empty(600, device="cuda")
            ops.adamw_decode(t.m_t[0], t.me_t[0], out, False)
            assert torch.isnan(out[256:512]).all() and torch.isfinite(out[:256]).all() and torch.isfinite(out[512:]).all()
            assert t.ve_t[1].cpu().tolist()[0] == 255
        t = Tensors([600, 300], bits, seed=1)
        t.grads_t[0][300] = float("inf")
        ops.adamw_step(t.plan(), torch.zeros(3, dtype=torch.int64, device="cuda"), 1e-3, 0.9, 0.999, 1e-7, clip_norm=1.0)
        assert not torch.isfinite(t.theta_t[0]).any() and not torch.isfinite(t.theta_t[1]).any()
        assert before[0].size == 600


def test_moments_of_nothing_and_of_very_small_values():
    """All-zero gradients and moments leave all zero; magnitudes down to float32's denormals keep their blocks' scale."""
    from spectrum_vae_amd import ops
    t = Tensors([512, 256], 8, seed=2, copies=False, decay=0.0)
    for x in t.m_t + t.v_t + t.me_t + t.ve_t + t.grads_t:
        x.zero_()
    small = np.zeros(256, F)
    small[:4] = [1e-18, -3e-19, 5e-21, 1e-30]
    t.grads_t[1].copy_(_dev(small))
    t.grads = [np.zeros(512, F), small]
    t.m, t.v = [np.zeros(512, F), np.zeros(256, F)], [np.zeros(512, F), np.zeros(256, F)]
    state = torch.zeros(3, dtype=torch.int64, device="cuda")
    ops.adamw_step(t.plan(), state, 1e-3, 0.9, 0.999, 1e-7, seed=3)
    assert np.array_equal(t.theta_t[0].cpu().numpy(), t.theta[0])
    t.check(0, 1e-3, seed=3)
    assert not t.m_t[0].any() and not t.v_t[0].any() and not t.me_t[0].any()


def test_second_moments_in_8_bits_follow_the_gradients():
    """1500 steps of gradients of size 0.1 from second moments of 1: in 64 bits v goes to 0.01 + 0.99 * 0.999^1500 = 0.2308.
    Rounding to nearest would leave every v at 1.  The mean over n = 16384 elements: a code's step is at most 1/8 of v and a step
    moves v by about 0.001 v, so a rounding has variance of at most 0.001 / 8 v^2, 1500 of them (each then shrunk by its later
    decay) at most 0.19 v_0^2 in all, and the mean of the elements is off by at most 5 sqrt(0.19 / 16384) = 0.017."""
    from spectrum_vae_amd import ops
    n = 16384
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    u8 = lambda k: torch.zeros(k, dtype=torch.uint8, device="cuda")  # noqa: E731
    code, exp = Moments8.encode(np.ones(n, F), np.zeros(n, np.int64), 5)
    theta, grad, m, v, me, ve = z(n), z(n).fill_(0.1), u8(n), _dev(code), u8(n // 256), _dev(exp)
    plan = ops.AdamWPlan([theta], [grad], [m], [v], 0.0, m_exp=[me], v_exp=[ve])
    state = torch.zeros(3, dtype=torch.int64, device="cuda")
    for _ in range(1500):
        ops.adamw_step(plan, state, 1e-5, 0.9, 0.999, 1e-7, seed=11)
    out = z(n)
    ops.adamw_decode(v, ve, out, True)
    want = 0.01 + 0.99 * 0.999 ** 1500
    assert abs(float(out.double().mean()) - want) <= 0.017
    ops.adamw_decode(m, me, out, False)
    # m is at 0.1 but for its own rounding, a step of 1/8 each time, of which 0.9^k is left after k steps: sqrt(1 / (64 * 4 * 0.19))
    assert abs(float(out.double().mean()) - 0.1) <= 5 * 0.1 * 0.15 / np.sqrt(n) + 1e-6


@pytest.mark.parametrize("bits", [32, 8])
def test_repeats_clearing_streams_and_graph_replays(bits):
    from spectrum_vae_amd import ops
    sizes = [216, 8, 70_001, 1]

    def steps(run):
        t = Tensors(sizes, bits, seed=8)
        plan, state = t.plan(), torch.zeros(3, dtype=torch.int64, device="cuda")
        run(lambda **kw: ops.adamw_step(plan, state, 1e-3, 0.9, 0.999, 1e-7, 2, 0.5, False, clip_norm=0.3, seed=6, **kw), t)
        torch.cuda.synchronize()
        assert int(state[0]) == 4
        return t.theta_t + t.m_t + t.v_t + t.lp_t

    def eager(step, t):
        for _ in range(4):
            step()

    want = steps(eager)

    def clearing(step, t):
        keep = [g.clone() for g in t.grads_t]
        for _ in range(4):
            step(zero_grad=True)
            assert not any(g.any() for g in t.grads_t)
            for g, k in zip(t.grads_t, keep):
                g.copy_(k)

    def side_stream(step, t):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(4):
                step()
        torch.cuda.current_stream().wait_stream(side)

    def replayed(step, t):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            torch.zeros(1000, device="cuda").add_(1)

    for run in (eager, clearing, side_stream, replayed):
        assert all(torch.equal(a, b) for a, b in zip(want, steps(run))), run.__name__


def test_a_plan_of_many_tensors_and_refusals_on_the_device():
    from spectrum_vae_amd import _lib, ops
    t = Tensors([17] * 700 + [5000], 32, seed=3)
    state = torch.zeros(3, dtype=torch.int64, device="cuda")
    ops.adamw_step(t.plan(), state, 1e-3, 0.9, 0.999, 1e-7)
    t.check(0, 1e-3)
    a = torch.zeros(64, device="cuda")
    b = [torch.zeros(64, device="cuda") for _ in range(3)]
    with pytest.raises(_lib.SpectrumHipError, match="overlap"):
        ops.AdamWPlan([a, a], [b[0], b[0]], [b[1], b[1]], [b[2], b[2]], 0.0)
    with pytest.raises(ValueError, match="contiguous"):
        ops.AdamWPlan([a[::2]], [b[0][:32]], [b[1][:32]], [b[2][:32]], 0.0)
    with pytest.raises(TypeError):
        ops.AdamWPlan([a.double()], [b[0]], [b[1]], [b[2]], 0.0)
    with pytest.raises(ValueError, match="another device"):
        ops.AdamWPlan([a], [b[0].cpu()], [b[1]], [b[2]], 0.0)
    plan = ops.AdamWPlan([a], [b[0]], [b[1]], [b[2]], 0.0)
    with pytest.raises(ValueError, match="state"):
        ops.adamw_step(plan, state[:2], 1e-3, 0.9, 0.999, 1e-7)


@pytest.mark.parametrize("clip", [0.0, 0.5])
@pytest.mark.parametrize("bits,sizes", [(32, [2_000_001]), (8, [2_000_001]), (32, [9_000_000, 3, 700_001]), (8, [9_000_000, 3, 700_001]),
                                        (32, [20_000_003, 70]), (8, [30_000_003, 70])])
def test_large_tensors_by_samples(bits, sizes, clip):
    """More entries than workgroups, one to four workgroups an entry, and more bytes than the caches hold; blocks of 256 drawn from
    all over, the first and the last (incomplete) ones among them, against the oracle."""
    from spectrum_vae_amd import ops
    rng = np.random.default_rng(sum(sizes) + bits)
    g = torch.Generator(device="cuda").manual_seed(bits)
    randn = lambda n: torch.randn(n, device="cuda", generator=g)  # noqa: E731
    theta, grads = [0.1 * randn(n) for n in sizes], [1e-2 * randn(n) for n in sizes]
    lp = [torch.empty(n, dtype=torch.bfloat16, device="cuda") for n in sizes]
    blocks = [-(-n // 256) for n in sizes]
    if bits == 8:
        m, v = ([torch.randint(0, 256, (n,), dtype=torch.uint8, device="cuda", generator=g) for n in sizes] for _ in range(2))
        me, ve = ([torch.randint(115, 121, (b,), dtype=torch.uint8, device="cuda", generator=g) for b in blocks] for _ in range(2))
    else:
        m, v, me, ve = [1e-3 * randn(n) for n in sizes], [1e-4 * randn(n) ** 2 for n in sizes], None, None
    before = [[t.clone() for t in ts] for ts in (theta, m, v, *((me, ve) if bits == 8 else ()))]
    norm = float(torch.sqrt(sum((t.double() ** 2).sum() for t in grads)))
    scale = clip / max(clip, norm) if clip else 1.0
    state = torch.tensor([3, 0, 0], dtype=torch.int64, device="cuda")
    plan = ops.AdamWPlan(theta, grads, m, v, 0.1, m_exp=me, v_exp=ve, params_lp=lp)
    ops.adamw_step(plan, state, 1e-3, 0.9, 0.999, 1e-7, clip_norm=clip, seed=21)
    assert int(state[0]) == 4
    alpha = 1e-3 * np.sqrt(1 - 0.999 ** 4) / (1 - 0.9 ** 4)
    slack = 10 * U if clip else 0.0  # of the norm, as in the test of the clip
    first = np.cumsum([0] + blocks)
    for i, n in enumerate(sizes):
        assert torch.equal(lp[i], theta[i].to(torch.bfloat16))
        for b in sorted({0, blocks[i] - 1, *rng.integers(0, blocks[i], 60).tolist()}):
            s = slice(256 * b, min(256 * b + 256, n))
            pick = lambda t: t[s].cpu().numpy()  # noqa: E731
            if bits == 8:
                old = [Moments8.decode(pick(before[1 + j][i]), before[3 + j][i][b:b + 1].cpu().numpy(), 4 + j) for j in (0, 1)]
            else:
                old = [pick(before[1][i]), pick(before[2][i])]
            g64 = pick(grads[i]).astype(np.float64) * scale
            th, mw, vw = np_ops.adamw_step(pick(before[0][i]), g64, old[0].astype(np.float64), old[1].astype(np.float64), 3, 1e-3, 0.1)
            e_g = np.abs(g64) * (U + slack)
            e_m = 4 * U * (np.abs(0.9 * old[0]) + np.abs(0.1 * g64)) + 0.1 * e_g
            e_v = 5 * U * vw + 2e-3 * np.abs(g64) * e_g
            step = alpha * mw / (np.sqrt(vw) + 1e-7)
            e_step = 8 * U * np.abs(step) + alpha * e_m / (np.sqrt(vw) + 1e-7) + np.abs(step) * e_v / np.maximum(2 * vw, 1e-300)
            assert (np.abs(pick(theta[i]) - th) <= e_step + 4 * U * (np.abs(pick(before[0][i])) + np.abs(th))).all(), (i, b)
            if bits == 32:
                assert (np.abs(pick(m[i]) - mw) <= e_m).all() and (np.abs(pick(v[i]) - vw) <= e_v).all(), (i, b)
            elif not clip:
                gs = pick(grads[i])
                rnd = Moments8.random_bits(s.stop - s.start, int(first[i]) + b, 3, 21)
                for val, r, width, ct, et in ((F(0.9) * old[0] + F(1 - 0.9) * gs, rnd[0], 4, m[i], me[i]),
                                              (F(0.999) * old[1] + F(1 - 0.999) * (gs * gs), rnd[1], 5, v[i], ve[i])):
                    code, exp = Moments8.encode(val, r, width)
                    assert int(et[b]) == exp[0] and np.array_equal(pick(ct), code), (i, b, width)
    if bits == 8:  # decoding of the same sizes
        for i, n in enumerate(sizes):
            out = torch.empty(n, device="cuda")
            for second, ct, et in ((False, m[i], me[i]), (True, v[i], ve[i])):
                ops.adamw_decode(ct, et, out, second)
                for b in sorted({0, blocks[i] - 1, *rng.integers(0, blocks[i], 20).tolist()}):
                    s = slice(256 * b, min(256 * b + 256, n))
                    want = Moments8.decode(ct[s].cpu().numpy(), et[b:b + 1].cpu().numpy(), 5 if second else 4)
                    assert np.array_equal(out[s].cpu().numpy(), want)


def test_decoding_more_than_the_caches_hold():
    from spectrum_vae_amd import ops
    n = 70_000_003
    g = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.randint(0, 256, (n,), dtype=torch.uint8, device="cuda", generator=g)
    exps = torch.randint(0, 256, (-(-n // 256),), dtype=torch.uint8, device="cuda", generator=g)
    whole = torch.full((n + 9,), 7.0, device="cuda")
    for second in (False, True):
        for off in (0, 1):  # with and without 16-byte accesses
            out = whole[off:off + n]
            ops.adamw_decode(codes, exps, out, second)
            for b in (0, 1, 1000, 136_718, exps.numel() - 1):
                s = slice(256 * b, min(256 * b + 256, n))
                want = Moments8.decode(codes[s].cpu().numpy(), exps[b:b + 1].cpu().numpy(), 5 if second else 4)
                assert np.array_equal(out[s].cpu().numpy(), want, equal_nan=True)
            assert (whole[n + 1:] == 7).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_two_plans_at_once_and_two_recordings_of_each(bits):
    """Plans of different tensors stepped on two streams at once, eagerly and by graphs recorded twice from one plan: the bits of
    steps one after the other."""
    from spectrum_vae_amd import ops

    def make(seed):
        t = Tensors([300, 70_001, 8193, 4096 * 70], bits, seed=seed)
        return t, t.plan(), torch.zeros(3, dtype=torch.int64, device="cuda")

    def step(plan, state):
        ops.adamw_step(plan, state, 1e-3, 0.9, 0.999, 1e-7, clip_norm=0.2, seed=3)

    alone = [make(s) for s in (1, 2)]
    for _, plan, state in alone:
        for _ in range(5):
            step(plan, state)
    torch.cuda.synchronize()
    both = [make(s) for s in (1, 2)]
    graphs = []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for (_, plan, state), st in zip(both, streams):  # two eager steps, then three replays of two recordings
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step(plan, state)
            step(plan, state)
    torch.cuda.synchronize()
    for _, plan, state in both:
        pair = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                step(plan, state)
            pair.append(g)
        graphs.append(pair)
    for k in (0, 1, 0):
        for pair, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                pair[k].replay()
    torch.cuda.synchronize()
    for (a, _, sa), (b, _, sb) in zip(alone, both):
        assert int(sa[0]) == int(sb[0]) == 5
        assert all(torch.equal(x, y) for x, y in zip(a.theta_t + a.m_t + a.v_t + a.lp_t, b.theta_t + b.m_t + b.v_t + b.lp_t))


# ------------------------------------------------------------------------------------------------ in models
def _model(optimizer, dtype="float32"):
    from spectrum_vae_amd import losses, mixed_precision
    from spectrum_vae_amd.model import SequentialModel
    from spectrum_vae_amd.nn import Conv2D, Conv2DTranspose, GroupNormalization, LeakyReLU
    mixed_precision.set_global_policy(dtype)
    try:
        m = SequentialModel([Conv2D(16, (2, 2), strides=(2, 2), padding="same", use_bias=False), GroupNormalization(4), LeakyReLU(0.2),
                             Conv2DTranspose(3, (2, 2), strides=(2, 2), padding="same", activation="tanh")], name="gn_net")
    finally:
        mixed_precision.set_global_policy("float32")
    m.compile(optimizer=optimizer, loss=losses.MeanSquaredError())
    m.build((None, 8, 8, 3))
    return m


def test_group_norm_model_trained_with_adamw_matches_a_float64_restatement():
    """Five steps of fit's own path (eager, recorded, replayed) against torch in float64 on the CPU."""
    from spectrum_vae_amd.optimizers import AdamW, ExponentialDecay
    opt = AdamW(ExponentialDecay(1e-2, 2, 0.9, True), weight_decay=0.05, global_clipnorm=0.05)
    opt.exclude_from_weight_decay(var_names=["gamma", "beta", "bias"])
    model = _model(opt)
    rng = np.random.default_rng(0)
    x = rng.standard_normal((8, 8, 8, 3)).astype(F)
    model._materialize(torch.device("cuda", 0))
    p = [torch.from_numpy(v.numpy().astype(np.float64)).requires_grad_() for v in model.trainable_variables]
    names = [v.name for v in model.trainable_variables]
    mom = [(np.zeros(q.shape), np.zeros(q.shape)) for q in p]
    xt = torch.from_numpy(x.astype(np.float64))
    b = model._step_buffers(8, (8, 8, 3))
    b["x"].copy_(torch.from_numpy(x))
    losses_gpu, losses_cpu = [], []
    for it in range(5):
        model.train_on_device_batch(b, True, 8.0)
        losses_gpu.append(float(b["loss"]))
        h = torch.nn.functional.conv2d(xt.permute(0, 3, 1, 2), p[0].permute(3, 2, 0, 1), stride=2)
        h = torch.nn.functional.group_norm(h, 4, p[1], p[2], 1e-3)
        h = torch.nn.functional.leaky_relu(h, 0.2)
        h = torch.tanh(torch.nn.functional.conv_transpose2d(h, p[3].permute(3, 2, 0, 1), p[4], stride=2)).permute(0, 2, 3, 1)
        loss = ((h - xt) ** 2).mean()
        losses_cpu.append(float(loss.detach()))
        grads = torch.autograd.grad(loss, p)
        norm = float(torch.sqrt(sum((g * g).sum() for g in grads)))
        lr = np_ops.exponential_decay(1e-2, it, 2, 0.9, True)
        for i, g in enumerate(grads):
            wd = 0.0 if any(k in names[i] for k in ("gamma", "beta", "bias")) else 0.05
            th, m, v = np_ops.adamw_step(p[i].detach().numpy(), g.numpy() * 0.05 / max(norm, 0.05), *mom[i], it, lr, wd)
            mom[i] = (m, v)
            p[i] = torch.from_numpy(th).requires_grad_()
    # the first loss is a forward pass in float32; a step of lr per weight at most follows each, and Adam's m / sqrt(v) turns
    # relative gradient errors (about 1e-5) into changes of the same share of a step
    assert abs(losses_gpu[0] - losses_cpu[0]) <= 1e-5 * losses_cpu[0]
    np.testing.assert_allclose(losses_gpu, losses_cpu, rtol=1e-4)
    for v, q in zip(model.trainable_variables, p):
        assert np.abs(v.numpy() - q.detach().numpy()).max() <= 5 * 1e-2 * 2e-3, v.name


@pytest.mark.parametrize("dtype", ["float32", "mixed_bfloat16"])
def test_recorded_steps_equal_eager_ones_with_8_bit_moments(dtype):
    from spectrum_vae_amd.optimizers import AdamW
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((8, 8, 8, 3)).astype(F)).cuda()
    runs = []
    for graphs in (False, True):
        opt = AdamW(1e-2, state_bits=8)
        model = _model(opt, dtype)
        model.use_graphs = graphs
        model._materialize(torch.device("cuda", 0))
        b = model._step_buffers(8, (8, 8, 3))
        b["x"].copy_(x)
        for _ in range(5):
            model.train_on_device_batch(b, True, 8.0)
        runs.append((model._params.clone(), [t.clone() for v in model.trainable_variables for t in opt.moments(v)], model._params_lp))
        assert opt.iterations == 5
    assert torch.equal(runs[0][0], runs[1][0])
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))
    if dtype != "float32":
        assert torch.equal(runs[1][2], runs[1][0].to(torch.bfloat16))


def test_apply_gradients_for_some_variables_and_for_all():
    from spectrum_vae_amd.optimizers import AdamW
    for bits in (32, 8):
        whole, part = AdamW(1e-2, state_bits=bits), AdamW(1e-2, state_bits=bits)
        a, b = _model(whole), _model(part)
        for m in (a, b):
            m._materialize(torch.device("cuda", 0))
            m._grads.copy_(torch.linspace(-1, 1, m._grads.numel(), device="cuda"))
        whole.apply_gradients([(v.grad, v) for v in a.trainable_variables])
        part.apply_gradients([(v.grad.clone(), v) for v in b.trainable_variables])
        for v, w in zip(a.trainable_variables, b.trainable_variables):
            assert torch.equal(v.data, w.data)
            assert all(torch.equal(s, t) for s, t in zip(whole.moments(v), part.moments(w)))
        keep = [v.data.clone() for v in b.trainable_variables]
        part.apply_gradients([(v.grad * 2, v) for v in b.trainable_variables[1:3]])
        moved = [not torch.equal(k, v.data) for k, v in zip(keep, b.trainable_variables)]
        assert moved == [False, True, True, False, False]
        with pytest.raises(ValueError, match="twice"):
            part.apply_gradients([(v.grad, v) for v in [b.trainable_variables[0]] * 2])


def test_unet_gan_steps_with_group_norm_and_adamw():
    """Generator and discriminator with group norm, 8-bit AdamW: recorded steps give the bits of eager ones; every gradient of
    the group norm layers is live."""
    from spectrum_vae_amd import run_unet, unet
    from spectrum_vae_amd.optimizers import AdamW
    rng = np.random.default_rng(2)
    X, y = rng.standard_normal((4, 32, 32, 1)).astype(F), rng.standard_normal((4, 32, 32, 3)).astype(F)
    runs = []
    for graphs in (False, True):
        gen, disc = unet.Generator(normalization="group"), unet.Discriminator(normalization="group")
        gen.build_graph((1, 32, 32, 1))
        disc.build_graph((1, 32, 32, 4))
        opts = [AdamW(1e-3, beta_1=0.5, state_bits=8), AdamW(1e-3, beta_1=0.5, state_bits=8)]
        got = [[float(v) for v in run_unet.train_step(gen, disc, *opts, X, y, use_graph=graphs)] for _ in range(4)]
        assert np.isfinite(got).all()
        runs.append((got, gen._params.clone(), disc._params.clone()))
        for m, o in ((gen, opts[0]), (disc, opts[1])):
            assert o.iterations == 4
            for v in m.trainable_variables:
                assert o.moments(v)[1].abs().max() > 0, v.name
    assert runs[0][0] == runs[1][0]
    assert torch.equal(runs[0][1], runs[1][1]) and torch.equal(runs[0][2], runs[1][2])
