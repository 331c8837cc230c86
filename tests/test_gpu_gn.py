"""Group norm + activation (csrc/gn.hip) against the definition in 64 bits.

Tolerances, per value: half a step of the output type (``eps / 2`` relative), and for the f32 arithmetic
``L * 2^-24`` of the magnitudes that enter, with L = the longest chain of f32 additions a sum goes through (a thread
adds at most 256 rows in these shapes, then 16 terms of a fold at most per level) plus 16 single operations.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def _k():
    from distributed_training_pytorch_amd.ops import kernels
    return kernels


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    return z * torch.sigmoid(z) if act == "silu" else z


def _ref_stats(x, groups, eps):
    n, c = x.shape[0], x.shape[-1]
    v = x.double().reshape(n, -1, groups, c // groups)
    mean = v.mean((1, 3))
    var = v.var((1, 3), unbiased=False)
    return mean, (var + eps).rsqrt(), v.abs().mean((1, 3)) + mean.abs()


def _ref(x, gamma, beta, groups, eps, act):
    n, c = x.shape[0], x.shape[-1]
    v = x.double().reshape(n, -1, groups, c // groups)
    mean, rstd, _ = _ref_stats(x, groups, eps)
    xh = ((v - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(x.shape)
    z = xh * gamma.double() + beta.double()
    return _act(z, act), xh, z


def _ref_bwd(x, dy, gamma, beta, groups, eps, act):
    n, c = x.shape[0], x.shape[-1]
    _, xh, z = _ref(x, gamma, beta, groups, eps, act)
    _, rstd, _ = _ref_stats(x, groups, eps)
    d = dy.double()
    if act == "relu":
        dz = d * (z > 0)
    elif act == "silu":
        s = torch.sigmoid(z)
        dz = d * (s + z * s * (1 - s))
    else:
        dz = d
    dims = tuple(range(x.dim() - 1))
    dgamma, dbeta = (dz * xh).sum(dims), dz.sum(dims)
    e, xg = (dz * gamma.double()).reshape(n, -1, groups, c // groups), xh.reshape(n, -1, groups, c // groups)
    m1, m2 = e.mean((1, 3), keepdim=True), (e * xg).mean((1, 3), keepdim=True)
    dx = ((e - m1 - xg * m2) * rstd[:, None, :, None]).reshape(x.shape)
    mag = ((e.abs() + e.abs().mean((1, 3), keepdim=True) + xg.abs() * (e * xg).abs().mean((1, 3), keepdim=True))
           * rstd[:, None, :, None]).reshape(x.shape)
    return dx, dgamma, dbeta, mag, (dz * xh).abs().sum(dims), dz.abs().sum(dims)


def _inputs(shape, dtype, seed=0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=g, device="cuda") * (0.5 + torch.rand(c, generator=g, device="cuda"))
         + 0.5 * torch.randn(c, generator=g, device="cuda") + shift).to(dtype)
    dy = torch.randn(shape, generator=g, device="cuda").to(dtype)
    gamma = 1 + 0.3 * torch.randn(c, generator=g, device="cuda")
    beta = 0.3 * torch.randn(c, generator=g, device="cuda")
    return x, dy, gamma, beta


def _check(got, ref, mag, name, chain=288):
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + chain * U * mag
    if got.dtype == F16:
        tol = tol + 2.0 ** -25          # half a step of its subnormals
    err = (got.double() - ref).abs()
    worst = (err / tol.clamp_min(1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, "%s: an element is %.2f times its tolerance off" % (name, worst)


SHAPES = [  # shape, groups
    ((1, 1, 1, 8), 8),              # one value a group: variance zero
    ((2, 1, 1, 64), 4),             # one pixel
    ((3, 64), 16),                  # no spatial axes
    ((2, 3, 5, 7), 1),              # all channels one group, odd channels
    ((4, 14, 14, 512), 32),
    ((2, 28, 28, 512), 32),
    ((2, 56, 56, 256), 32),
    ((1, 112, 112, 128), 32),
    ((2, 27, 19, 60), 12),
    ((3, 9, 33, 36), 12),           # three channels a group
    ((2, 17, 13, 96), 96),          # a group a channel
    ((1, 7, 5, 2058), 3),           # wide rows
    ((1, 2, 3, 4096), 2),
    ((300, 2, 2, 16), 4),           # many small images
    ((2, 1001, 24), 4),             # one long axis
]


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_gn_fwd(shape, groups, dtype, act):
    k = _k()
    x, _, gamma, beta = _inputs(shape, dtype)
    y, stats = k.gn_fwd(x, gamma, beta, groups, eps=1e-5, act=act)
    ref, xh, z = _ref(x, gamma, beta, groups, 1e-5, act)
    mean, rstd, mag = _ref_stats(x, groups, 1e-5)
    _check(stats[..., 0], mean, mag, "mean")
    # var is off by chain * U of E[(x - p)^2] <= 2 (var + (mean - p)^2); here |mean - p| <= 6 std: rstd by half of that
    _check(stats[..., 1], rstd, rstd * 40 * (1 + 0 * mag), "rstd")
    # |dy/dz| <= 1.1; xhat is off by the statistics' errors and its own three operations
    zmag = gamma.double().abs() * (xh.abs() * 40 + (mag * rstd).repeat_interleave(shape[-1] // groups, -1).view(
        (shape[0],) + (1,) * (len(shape) - 2) + (shape[-1],))) + beta.double().abs()
    _check(y, ref, 1.1 * zmag, "y")


def test_gn_data_beyond_the_caches():
    """272 MB (backward: 544 MB): more than the last-level cache, read past it up to the last 240 MiB.  The same bounds
    as the small shapes: a thread adds 74 rows."""
    test_gn_fwd((6, 381, 331, 180), 12, BF16, "relu")
    test_gn_bwd((6, 381, 331, 180), 12, BF16, "silu")


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_gn_bwd(shape, groups, dtype, act):
    k = _k()
    x, dy, gamma, beta = _inputs(shape, dtype, seed=1)
    mean, rstd, _ = _ref_stats(x, groups, 1e-5)
    stats = torch.stack((mean, rstd), -1).float()
    if act == "relu":                        # keep gradients away from signs that f32 cannot decide
        z = _ref(x, gamma, beta, groups, 1e-5, act)[2]
        dy = torch.where(z.abs() > 1e-4, dy, torch.zeros_like(dy))
    dg, db = torch.empty(shape[-1], device="cuda"), torch.empty(shape[-1], device="cuda")
    dx = k.gn_bwd(x, dy, gamma, beta, stats, groups, dg, db, act=act)
    rdx, rdg, rdb, mag, mg, mb = _ref_bwd(x, dy, gamma, beta, groups, 1e-5, act)
    zmag = 1 + _ref(x, gamma, beta, groups, 1e-5, act)[2].abs().amax().item()      # d(act')/dz <= 1: its slope enters
    extra = (x.double().abs().amax() + 1) * rstd.amax()                          # rounding of x - mean, per unit of xhat
    _check(dx, rdx, mag * (zmag + extra), "dx")
    _check(dg, rdg, mg * zmag + mb * extra, "dgamma")
    _check(db, rdb, mb * (zmag + extra), "dbeta")


def test_gn_mean_far_from_zero():
    """mean / std = 1000 in f32: E[x^2] - mean^2 would lose 1e6 * 2^-24 = 6 % of the variance."""
    k = _k()
    x, _, gamma, beta = _inputs((2, 31, 17, 48), F32, shift=1000.0)
    y, stats = k.gn_fwd(x, gamma, beta, 6, act="none")
    ref, xh, _ = _ref(x, gamma, beta, 6, 1e-5, "none")
    mean, rstd, _ = _ref_stats(x, 6, 1e-5)
    # rstd: relative chain * U * E[(x-p)^2] / var <= 288 * U * 40; the mean: half a step of 1000
    _check(stats[..., 1], rstd, rstd * 40, "rstd")
    assert ((stats[..., 0].double() - mean).abs() <= 1000 * 2 * U + 288 * U * 3).all()
    assert ((y.double() - ref).abs() <= 4 * 1000 * U * rstd.max() * gamma.abs().max() + 288 * U * 40 * (1 + ref.abs())).all()


def test_gn_poison_stays_in_its_group():
    k = _k()
    x, dy, gamma, beta = _inputs((3, 8, 8, 32), F32)
    clean, _ = k.gn_fwd(x, gamma, beta, 4, act="relu")
    x2 = x.clone()
    x2[1, 3, 2, 9] = float("nan")       # group 1 of image 1
    x2[2, 0, 0, 31] = float("inf")      # group 3 of image 2
    y, stats = k.gn_fwd(x2, gamma, beta, 4, act="relu")
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[1, :, :, 8:16] = True
    bad[2, :, :, 24:] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])
    dg, db = torch.empty(32, device="cuda"), torch.empty(32, device="cuda")
    dx = k.gn_bwd(x2, dy, gamma, beta, stats, 4, dg, db, act="none")
    assert torch.isfinite(dx[~bad]).all() and torch.isnan(dx[bad]).all()


@pytest.mark.parametrize("gdtype", [F32, BF16])
def test_gn_param_gradients_accumulate(gdtype):
    k = _k()
    x, dy, gamma, beta = _inputs((3, 11, 6, 40), BF16, seed=2)
    y, stats = k.gn_fwd(x, gamma, beta, 5, act="silu")
    dg0, db0 = torch.full((40,), 7.0, device="cuda", dtype=gdtype), torch.full((40,), -3.0, device="cuda", dtype=gdtype)
    dg, db = torch.empty(40, device="cuda", dtype=gdtype), torch.empty(40, device="cuda", dtype=gdtype)
    a = k.gn_bwd(x, dy, gamma, beta, stats, 5, dg, db, act="silu")
    b = k.gn_bwd(x, dy, gamma, beta, stats, 5, dg0, db0, act="silu", beta_g=1.0, beta_b=1.0)
    assert torch.equal(a, b)
    e = torch.finfo(gdtype).eps
    for once, more, was in ((dg, dg0, 7.0), (db, db0, -3.0)):
        want = once.double() + was
        assert ((more.double() - want).abs() <= e * (once.double().abs() + want.abs())).all()


def test_gn_gradient_against_differences():
    k = _k()
    x, dy, gamma, beta = _inputs((2, 4, 5, 12), F32, seed=3)
    _, stats = k.gn_fwd(x, gamma, beta, 3, act="silu")
    dg, db = torch.empty(12, device="cuda"), torch.empty(12, device="cuda")
    dx = k.gn_bwd(x, dy, gamma, beta, stats, 3, dg, db, act="silu")
    g = torch.Generator(device="cuda").manual_seed(9)

    def loss(x_, ga, be):
        return (k.gn_fwd(x_, ga, be, 3, act="silu")[0].double() * dy.double()).sum().item()

    h = 2.0 ** -6
    for t, grad, put in ((x, dx, 0), (gamma, dg, 1), (beta, db, 2)):
        v = torch.randn(t.shape, generator=g, device="cuda")
        v = v / v.norm()
        args = [x, gamma, beta]
        up, down = list(args), list(args)
        up[put], down[put] = t + h * v, t - h * v
        fd = (loss(*up) - loss(*down)) / (2 * h)
        want = (grad.double() * v.double()).sum().item()
        # third-order term h^2/6 |f'''| with |f'''| <~ 10 |dy|_1-ish directions of unit length, and rounding 2^-20 / h
        assert abs(fd - want) <= 10 * h * h + 480 * 2.0 ** -22 / h, (put, fd, want)


def test_gn_repeats_bit_for_bit_on_streams_and_in_graphs():
    k = _k()
    x, dy, gamma, beta = _inputs((5, 27, 19, 64), BF16, seed=4)

    def both(x_, dy_):
        y, st = k.gn_fwd(x_, gamma, beta, 8, act="relu")
        dg, db = torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
        return y, st, k.gn_bwd(x_, dy_, gamma, beta, st, 8, dg, db, act="relu"), dg, db

    first = both(x, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = both(x, dy)
    again = both(x, dy)                         # on the default stream, next to the other one
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    xs, graphs = [x.clone(), torch.flip(x, (0,)).contiguous()], []
    for v in xs:                                # two graphs share no scratch
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            out = both(v, dy)
        graphs.append((g, out))
    for rep in range(3):
        for v, (g, out) in zip(xs, graphs):
            v.mul_(0.5 if rep == 1 else 1.0)
            g.replay()
        for v, (g, out) in zip(xs, graphs):
            for a, b in zip(out, both(v, dy)):
                assert torch.equal(a, b)


def test_gn_empty_batch():
    k = _k()
    ga = torch.ones(16, device="cuda")
    x = torch.empty((0, 4, 4, 16), device="cuda")
    y, st = k.gn_fwd(x, ga, ga, 4)
    dg, db = torch.full((16,), 5.0, device="cuda"), torch.full((16,), 5.0, device="cuda")
    dx = k.gn_bwd(x, x, ga, ga, st, 4, dg, db, beta_b=1.0)
    assert y.shape == x.shape == dx.shape and st.shape == (0, 4, 2)
    assert (dg == 0).all() and (db == 5).all()


def test_gn_bwd_refuses_one_tensor_for_both_parameter_gradients():
    k = _k()
    x, dy, gamma, beta = _inputs((2, 3, 3, 16), BF16)
    _, stats = k.gn_fwd(x, gamma, beta, 4)
    d = torch.zeros(16, device="cuda")
    with pytest.raises(ValueError, match="share their memory"):
        k.gn_bwd(x, dy, gamma, beta, stats, 4, d, d)
    with pytest.raises(ValueError, match="share their memory"):
        k.gn_bwd(x, dy, gamma, beta, stats, 4, d, beta)


def _check_stats(stats, x, groups, name):
    """Statistics against 64 bits.  U = 2^-24.  A thread's squares: 3 U a term (difference, square), at most 16 additions in
    one launch; in two passes runs of 8 and one addition a run of at most 16 runs: 24 U in all.  A set's centre is off by
    2 U of its size, which moves the variance by 2 * 2 U of (centre - mean) * size summed over the sets: the centres
    deviate as little as the values, so 2 * 2 U times what the largest |x - mean| of a set is to the spread, <= 32 U.  rstd: half
    of the variance's error, and 2 U of its own: 30 U; twice that is allowed.  The mean: 2 U of a set's centre, 8 U of
    adding up a set."""
    mean, rstd, mag = _ref_stats(x, groups, 1e-5)
    err = ((stats[..., 1].double() - rstd).abs() / rstd).max().item()
    assert err <= 60 * U, "%s: rstd is %.3g off" % (name, err)
    err = ((stats[..., 0].double() - mean).abs() / mag).max().item()
    assert err <= 10 * U, "%s: mean is %.3g of E|x| off" % (name, err)


STAT_SHAPES = [((2, 56, 56, 64), 16, False), ((3, 14, 14, 60), 12, False), ((2, 30, 31, 8), 1, False), ((2, 5, 7, 33), 3, False),
               ((2, 128, 128, 64), 1, True), ((1, 301, 257, 24), 4, True), ((1, 200, 200, 9), 3, True),
               ((1, 48, 40, 4000), 2, True)]


@pytest.mark.parametrize("far", [30.0, 300.0, 1e4, 1e6])
@pytest.mark.parametrize("where", ["first", "last", "corner rows"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape,groups,two_passes", STAT_SHAPES)
def test_gn_statistics_beside_values_far_from_the_others(shape, groups, two_passes, dtype, where, far):
    """A group's first value, its last one, or the image's first row and column, `far` standard deviations from the rest:
    sums around such a value cancel (around the first: 7e-3 of rstd at 1000)."""
    if dtype == F16 and far > 6e4:
        far = 6e4
    k = _k()
    n, c = shape[0], shape[-1]
    hw = 1
    for d in shape[1:-1]:
        hw *= d
    dt = k.GN_DTYPES[dtype]
    slab = k._gn_workspace(n, hw, c, groups, dt, 0) == 0
    assert slab != two_passes, "the shape does not reach the path that it is here for"
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(shape, generator=g, device="cuda")
    first = torch.arange(0, c, c // groups, device="cuda")
    if where == "first":
        x[:, 0, 0, first] = far
    elif where == "last":
        x[:, -1, -1, first] = -far
    else:
        x[:, 0], x[:, :, 0] = far, far
    x = x.to(dtype)
    gamma, beta = 1 + 0.3 * torch.randn(c, generator=g, device="cuda"), 0.3 * torch.randn(c, generator=g, device="cuda")
    y, stats = k.gn_fwd(x, gamma, beta, groups, act="none")
    _check_stats(stats, x, groups, "%s %g" % (where, far))
    ref, xh, _ = _ref(x, gamma, beta, groups, 1e-5, "none")
    mean, rstd, mag = _ref_stats(x, groups, 1e-5)
    mag = (mag * rstd).repeat_interleave(c // groups, -1).view(n, 1, 1, c)
    _check(y, ref, gamma.double().abs() * (xh.abs() + mag) + beta.double().abs(), "y", chain=70)


@pytest.mark.parametrize("shape,groups,two_passes", STAT_SHAPES)
def test_gn_statistics_of_a_large_common_mean(shape, groups, two_passes):
    """mean / std = 1e4 in f32, with and without a zero corner: the centres of a thread's values are of the mean's
    size, and 2 U of that is 2e4 U of a standard deviation; what it moves the variance by is summed over at least
    500 values with signs of their own: 2 * 2e4 U / sqrt(500) of it, half of that of rstd."""
    k = _k()
    g = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(shape, generator=g, device="cuda") + 1e4
    ones = torch.ones(shape[-1], device="cuda")
    for corner in (False, True):
        if corner:
            x[:, 0, 0, ::shape[-1] // groups] = 0
        _, stats = k.gn_fwd(x, ones, ones, groups, act="none")
        mean, rstd, _ = _ref_stats(x, groups, 1e-5)
        m = x[0].numel() // groups
        err = ((stats[..., 1].double() - rstd).abs() / rstd).max().item()
        assert err <= 60 * U + 4 * 2e4 * U / m ** 0.5, "corner %s: rstd is %.3g off" % (corner, err)
        assert ((stats[..., 0].double() - mean).abs() <= 4 * U * 1e4).all()


def test_gn_bwd_refuses_parameter_gradients_inside_what_is_read():
    k = _k()
    x, dy, gamma, beta = _inputs((2, 3, 3, 16), F32)
    _, stats = k.gn_fwd(x, gamma, beta, 4)
    d, flat = torch.zeros(16, device="cuda"), torch.zeros(40, device="cuda")
    for dg, db in ((x.view(-1)[:16], d), (d, dy.view(-1)[16:32]), (stats.view(-1), d), (flat[:16], flat[12:28])):
        with pytest.raises(ValueError, match="share their memory"):
            k.gn_bwd(x, dy, gamma, beta, stats, 4, dg, db)


def test_gn_of_one_channel_and_two_thousand_million_pixels():
    """The longest image that is taken: row numbers up to 2^31 - 2^21.  (Sums of a thread: 4,100 rows.)"""
    k = _k()
    hw = 2 ** 31 - 2 ** 21 - 1
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty((1, hw, 1), device="cuda", dtype=BF16)
    part = 1 << 28
    for i in range(0, hw, part):
        v = x[0, i:i + part, 0]
        v.copy_(torch.randn(v.shape, generator=g, device="cuda") + i / hw)
    one, zero = torch.ones(1, device="cuda"), torch.zeros(1, device="cuda")
    y, stats = k.gn_fwd(x, one, zero, 1, act="none")
    pieces = [x[0, i:i + part, 0] for i in range(0, hw, part)]
    mean = sum(v.double().sum().item() for v in pieces) / hw
    var = sum((v.double() - mean).square().sum().item() for v in pieces) / hw
    rstd = (var + 1e-5) ** -0.5
    # (runs of eight in a thread: 512 additions of squares, each U of the sum)
    assert abs(stats[0, 0, 1].item() - rstd) <= 600 * U * rstd and abs(stats[0, 0, 0].item() - mean) <= 10 * U * (1 + mean)
    for lo in (0, hw // 2, hw - 100_000):
        _check(y[0, lo:lo + 100_000, 0], (x[0, lo:lo + 100_000, 0].double() - mean) * rstd, 1 + 0 * y[0, lo:lo + 100_000, 0].double(),
               "y", chain=1200)
    dg, db = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    dx = k.gn_bwd(x, y, one, zero, stats, 1, dg, db, act="none")
    # dy = xhat: dgamma = sum xhat^2, dbeta = sum xhat, dx = 0 up to the rounding of y (2^-8 of it)
    sq = sum((y[0, i:i + part, 0].double() * (x[0, i:i + part, 0].double() - mean) * rstd).sum().item() for i in range(0, hw, part))
    assert abs(dg.item() - sq) <= 4200 * U * sq
    assert dx[0, -100_000:].abs().max().item() <= 8 * 2.0 ** -8 * rstd and dx[0, :100_000].abs().max().item() <= 8 * 2.0 ** -8 * rstd


@pytest.mark.parametrize("value", [0.0, 1e4, 3.1415927, -1e-30, 3e38])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape,groups,two_passes", STAT_SHAPES)
def test_gn_of_equal_values(shape, groups, two_passes, dtype, value):
    """Variance zero: the mean is the value, y is beta, rstd eps^-1/2 (U of its own, U / 2 of eps as an f32)."""
    k = _k()
    x = torch.full(shape, value, device="cuda").to(dtype)
    gamma, beta = torch.full((shape[-1],), 2.0, device="cuda"), torch.linspace(-1, 1, shape[-1], device="cuda")
    y, stats = k.gn_fwd(x, gamma, beta, groups, act="none")
    assert (stats[..., 0] == x.view(-1)[0].float()).all()
    assert (stats[..., 1].double() - 1e-5 ** -0.5).abs().max() <= 1.5 * U * 1e-5 ** -0.5
    assert torch.equal(y, beta.to(dtype).expand_as(y))
