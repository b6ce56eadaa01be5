"""Every compiled form of the held group norm, in both directions and types, against 64 bits: pieces a thread, threads, elements of a
piece, sums of whole groups or of channels, nontemporal accesses.

Which form a call takes is a rule on sizes and alignment, so a changed threshold changes what a list of shapes runs: the first test fails
once a compiled form is left out.  The others compare with 64 bits; bounds, u = 2^-24, as in test_gpu_groupnorm: a mean is off by 8 u of the
group's largest value, rstd by 33 u, z by e_z = |gamma| (8 u max|x| rstd + 34 u |xhat|) + 2 u (|z| + |beta|), the activation by 3e-7, sums
of n terms by 128 u of the sum of magnitudes, bfloat16 results by 2^-8."""
import pytest
import torch

U = 2.0 ** -24
EPS = 1e-3
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}

# samples, rows, channels, groups, bytes that every address is a multiple of (and not of twice as much, below 256)
SHAPES = [
    (1, 1, 1, 1, 64), (1, 1, 2, 1, 256), (1, 1, 2, 2, 64), (1, 1, 4, 1, 16), (1, 1, 4, 4, 16), (1, 1, 8, 2, 256),
    (1, 1, 48, 3, 16), (1, 1, 96, 3, 16), (1, 33, 9, 1, 64), (1, 65, 9, 3, 64), (1, 33, 18, 3, 16), (1, 137, 6, 3, 16),
    (1, 65, 18, 2, 256), (1, 33, 36, 4, 256), (1, 257, 6, 3, 16), (1, 131, 12, 3, 256), (1, 67, 36, 4, 16), (1, 259, 12, 3, 16),
    (1, 74, 48, 3, 16), (1, 137, 48, 3, 16), (1, 78, 96, 3, 16), (1, 130, 96, 3, 16), (55, 130, 9, 1, 256),
    (50, 132, 18, 3, 64), (25, 149, 36, 3, 16), (25, 276, 24, 8, 16), (49, 581, 6, 3, 256), (118, 267, 9, 1, 256),
    (48, 532, 12, 3, 256), (28, 280, 48, 3, 16), (3, 260, 512, 16, 256), (119, 543, 9, 1, 16), (135, 267, 18, 2, 16),
    (127, 1031, 6, 3, 16), (118, 33, 300, 1, 16), (120, 1026, 10, 1, 256), (116, 1027, 12, 3, 256), (118, 2408, 6, 3, 16),
    (38, 66, 900, 3, 64), (14, 518, 320, 32, 16), (120, 1102, 24, 3, 256), (56, 519, 128, 2, 16), (151, 2093, 12, 3, 16),
    (28, 1053, 160, 32, 256), (61, 2062, 48, 3, 256), (129, 2090, 24, 3, 256), (1677, 1251, 16, 1, 16),
    (1289, 413, 64, 16, 256), (2883, 115, 128, 32, 256), (690, 95, 1024, 4, 256), (796, 659, 128, 1, 256),
    (1728, 152, 256, 16, 256), (276, 119, 2048, 32, 256), (1565, 21, 2048, 32, 256), (1539, 684, 64, 1, 256),
]


def _compiled():
    out = set()
    for name, size in (("float32", 4), ("bfloat16", 2)):
        for backward in (False, True):
            for piece in (1, 2, 4, 8):
                if piece * size > 16:
                    continue
                for held, threads in ((2, 256), (4, 256), (8, 256), (8, 512), (8, 1024), (16, 1024)):
                    if held * piece * size > (128 if backward else 256):  # bytes of a tensor that a thread holds
                        continue
                    for whole in (False, True):
                        if whole and piece * size < 8:
                            continue
                        if backward and size == 2 and piece == 8 and (held, threads) == (8, 1024) and not whole:
                            continue  # its registers do not suffice
                        for nontemporal in (0, 1, 2) if whole and piece * size == 16 else (0,):
                            out.add((name, backward, held, threads, piece, whole, nontemporal))
    return out


def test_the_shapes_reach_every_compiled_form():
    from spectrum_vae_amd import ops
    reached = set()
    for n, s, c, groups, alignment in SHAPES:
        for name, dtype in TYPES.items():
            for backward in (False, True):
                f = ops.groupnorm_form(n, s, c, groups, backward, dtype, alignment)
                reached.add((name, backward, f.held, f.threads, f.piece, f.whole_groups, f.nontemporal))
    assert not _compiled() - reached, sorted(_compiled() - reached)


def test_forms_of_calls_out_of_range_are_refused():
    from spectrum_vae_amd import _lib, ops
    for bad in ((0, 4, 8, 2), (2, 0, 8, 2), (2, 4, 5000, 1), (2, 4, 8, 3), (2, 4, 8, 0), (1 << 40, 1 << 20, 8, 2)):
        with pytest.raises(_lib.SpectrumHipError):
            ops.groupnorm_form(*bad, False, torch.float32)
    for alignment in (0, 3, -4):
        with pytest.raises(_lib.SpectrumHipError, match="alignment"):
            ops.groupnorm_form(2, 4, 8, 2, False, torch.float32, alignment)
    with pytest.raises(TypeError, match="float16"):
        ops.groupnorm_form(2, 4, 8, 2, False, torch.float16)
    f = ops.groupnorm_form(2, 512 * 512, 128, 32, False, torch.bfloat16)
    assert f.held == 0 and f.chunks > 1


def _at(t, alignment):
    """The values at an address that is a multiple of ``alignment`` and of no more (below 256)."""
    skip = 0 if alignment >= 256 else alignment // t.element_size()
    whole = torch.empty(t.numel() + 512, dtype=t.dtype, device=t.device)
    first = -(whole.data_ptr() // t.element_size()) % (256 // t.element_size()) + skip
    out = whole[first:first + t.numel()].view(t.shape)
    assert out.data_ptr() % alignment == 0 and (alignment >= 256 or out.data_ptr() % (2 * alignment) != 0)
    return out.copy_(t)


def _elu(z):
    return torch.where(z > 0, z, torch.expm1(z))


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("n,s,c,groups,alignment", SHAPES)
def test_form(n, s, c, groups, alignment, name):
    from spectrum_vae_amd import ops
    dtype, d = TYPES[name], c // groups
    half = 0.0 if dtype == torch.float32 else 2.0 ** -8
    g = torch.Generator(device="cuda").manual_seed(n * s + c)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    x = _at((randn(n, s, c) * (0.3 + torch.rand(c, device="cuda", generator=g)) + randn(c)).to(dtype), alignment)
    dy = _at(randn(n, s, c).to(dtype), alignment)
    gamma, beta = 1 + 0.2 * randn(c), 0.2 * randn(c)
    y, dx = _at(torch.empty_like(x), alignment), _at(torch.empty_like(x), alignment)
    mean, rstd = (torch.empty(n, groups, device="cuda") for _ in range(2))
    ws = torch.full((max(ops.groupnorm_workspace(n, s, c, groups), 1),), 255, dtype=torch.uint8, device="cuda")
    ops.groupnorm_act_fwd(x, gamma, beta, y, mean, rstd, groups, EPS, "elu", 0.0, ws)

    rep = lambda t: t.repeat_interleave(d, dim=1)[:, None, :]  # noqa: E731
    xd, ga, be = x.double(), gamma.double(), beta.double()
    v = xd.view(n, s, groups, d)
    var, mu = torch.var_mean(v, dim=(1, 3), unbiased=False)
    rs = (var + EPS) ** -0.5
    big = v.abs().amax(dim=(1, 3))
    assert ((mean.double() - mu).abs() <= 8 * U * big).all()
    assert ((rstd.double() - rs).abs() <= rs * (33 * U + (8 * U * big * rs) ** 2)).all()
    xhat = (xd - rep(mu)) * rep(rs)
    z = xhat * ga + be
    want = _elu(z)
    tol = ga.abs() * (rep(8 * U * big * rs) + 34 * U * xhat.abs()) + 2 * U * (z.abs() + be.abs()) + 3e-7 + half * want.abs()
    assert ((y.double() - want).abs() <= tol).all()
    del want, tol, z

    mean, rstd = mu.float(), rs.float()
    dg, db = (torch.full((c,), float("nan"), device="cuda") for _ in range(2))
    ws.fill_(255)
    ops.groupnorm_act_bwd(x, dy, gamma, beta, mean, rstd, dx, dg, db, False, groups, "elu", 0.0, ws)
    rs = rstd.double()
    xhat = (xd - rep(mean.double())) * rep(rs)
    z = xhat * ga + be
    e_slope = 4 * U * ((xhat * ga).abs() + be.abs()) + 3e-7
    dyd = dy.double()
    dz = dyd * torch.where(z > 0, torch.ones_like(z), torch.exp(z))
    e_dz = dyd.abs() * e_slope + 3 * U * dz.abs()
    for got, exact, weight, extra in ((dg, (dz * xhat).sum(dim=(0, 1)), xhat.abs(), 3 * U), (db, dz.sum(dim=(0, 1)), 1.0, 0.0)):
        bound = ((e_dz + (128 * U + extra) * dz.abs()) * weight).sum(dim=(0, 1)) + U * exact.abs()
        assert ((got.double() - exact).abs() <= bound).all()
    gz, e_gz = dz * ga, e_dz * ga.abs() + U * (dz * ga).abs()
    mean_of = lambda t: t.view(n, s, groups, d).mean(dim=(1, 3))  # noqa: E731
    c1, c2 = mean_of(gz), mean_of(gz * xhat)
    e_c1 = mean_of(e_gz + 128 * U * gz.abs()) + U * c1.abs()
    e_c2 = mean_of((e_gz + 131 * U * gz.abs()) * xhat.abs()) + U * c2.abs()
    want = rep(rs) * (gz - rep(c1) - xhat * rep(c2))
    size = gz.abs() + rep(c1).abs() + (xhat * rep(c2)).abs()
    tol = rep(rs) * (e_gz + rep(e_c1) + xhat.abs() * rep(e_c2) + 6 * U * size) + half * want.abs()
    assert ((dx.double() - want).abs() <= tol).all()
