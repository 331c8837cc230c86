"""Newton-Schulz orthogonalisation and the Muon step (csrc/muon.hip) against the iteration in 64 bits.

Tolerance of O (relative, 2-norm).  A segment of three steps multiplies by Q with eigenvalues up to a^3 = 41; each of
the about ten products behind it rounds its operands and its result at 2^-23 of their size, so Q is off by at most
10 * 2^-22 * 41 = 1e-4 of 1, and O by as much of itself when X lies along few directions of size about 1 (its worst
case: rank one).  The segment of two adds a tenth of that.  A direction of size s < 1 is worse only by what the
iteration itself makes of it: one f32 rounding of G moves it by 2^-24 |G| / s.  NS_TOL is twice 1e-4.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
COEFFS = (3.4445, -4.7750, 2.0315)
NS_TOL = 2e-4
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _k():
    from distributed_training_pytorch_amd.ops import kernels
    return kernels


def _ns64(g, steps=5, coeffs=COEFFS, eps=1e-7):
    a, b, c = coeffs
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    x = x / (x.norm() + eps)
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if tall else x


def _matrix(rows, cols, kind, seed=0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "full":
        x = torch.randn(rows, cols, generator=g, device="cuda")
    else:
        r = 1 if kind == "rank1" else min(16, rows, cols)
        x = torch.randn(rows, r, generator=g, device="cuda") @ torch.randn(r, cols, generator=g, device="cuda")
        if kind == "noise":
            x = x + 0.05 * torch.randn(rows, cols, generator=g, device="cuda")
    return x.to(dtype)


def _rel(got, ref):
    return ((got.double() - ref).norm() / ref.norm().clamp_min(1e-300)).item()


SHAPES = [(1, 1), (1, 7), (7, 1), (3, 64), (64, 27), (64, 64), (65, 65), (64, 576), (128, 1152), (200, 100), (333, 1001),
          (1001, 333), (512, 4608), (2304, 512), (129, 127), (1024, 1024), (70, 5000), (700, 2100)]


@pytest.mark.parametrize("kind", ["full", "noise", "rank16", "rank1"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_newton_schulz(rows, cols, kind):
    k = _k()
    g = _matrix(rows, cols, kind)
    o = k.newton_schulz(g, out_dtype=F32)
    assert o.shape == g.shape and o.dtype == F32
    assert _rel(o, _ns64(g)) <= NS_TOL


@pytest.mark.parametrize("din", [F32, BF16, F16])
@pytest.mark.parametrize("dout", [F32, BF16, F16])
def test_newton_schulz_types(din, dout):
    k = _k()
    g = _matrix(96, 260, "noise", dtype=din)
    o = k.newton_schulz(g, out_dtype=dout)
    assert o.dtype == dout
    assert _rel(o, _ns64(g)) <= NS_TOL + HALF[dout]
    assert k.newton_schulz(g).dtype == din


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 7])
def test_newton_schulz_steps_and_coefficients(steps):
    k = _k()
    g = _matrix(150, 410, "noise", seed=3)
    for coeffs in (COEFFS, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5)):
        assert _rel(k.newton_schulz(g, steps=steps, coeffs=coeffs, out_dtype=F32), _ns64(g, steps, coeffs)) <= NS_TOL


def test_newton_schulz_any_magnitude():
    k = _k()
    g = _matrix(100, 300, "full")
    ref = _ns64(g)
    for s in (1e-30, 1e-18, 1e18, 1e30):                # squares leave f32's range
        assert _rel(k.newton_schulz(g * s, eps=1e-40, out_dtype=F32), ref) <= NS_TOL
    # eps is part of the formula: |g| and eps of one size halve X_0
    small = g / g.norm() * 1e-7
    assert _rel(k.newton_schulz(small, out_dtype=F32), _ns64(small)) <= NS_TOL
    assert (k.newton_schulz(torch.zeros(70, 90, device="cuda")) == 0).all()
    # entries of very different size: one large value, the rest tiny
    spread = torch.full((64, 200), 1e-6, device="cuda")
    spread[3, 5] = 1.0
    assert _rel(k.newton_schulz(spread, out_dtype=F32), _ns64(spread)) <= NS_TOL


def test_newton_schulz_nan_and_inf_are_not_hidden():
    k = _k()
    for v in (float("nan"), float("inf")):
        g = _matrix(64, 100, "full")
        g[3, 4] = v
        assert torch.isnan(k.newton_schulz(g, out_dtype=F32)).any()
    # ... and stay in their own matrix of a stack
    s = torch.stack([_matrix(70, 130, "full", seed=i) for i in range(3)])
    clean = k.newton_schulz(s)
    s[1, 0, 0] = float("nan")
    o = k.newton_schulz(s)
    assert torch.equal(o[0], clean[0]) and torch.equal(o[2], clean[2]) and torch.isnan(o[1]).any()


def test_newton_schulz_stacks_and_lists():
    k = _k()
    s = torch.stack([_matrix(33, 65, "noise", seed=i) for i in range(30)])      # more than one native call
    o = k.newton_schulz(s, out_dtype=F32)
    for i in range(30):
        assert torch.equal(o[i], k.newton_schulz(s[i].contiguous(), out_dtype=F32))
    mats = [_matrix(r, c, "noise", seed=r) for r, c in ((64, 27), (300, 70), (5, 9))]
    for m, q in zip(mats, k.newton_schulz(mats, out_dtype=F32)):
        assert q.shape == m.shape and _rel(q, _ns64(m)) <= NS_TOL
    assert k.newton_schulz([]) == []
    assert k.newton_schulz(torch.empty(0, 5, device="cuda")).shape == (0, 5)
    assert k.newton_schulz(torch.empty(2, 4, 0, device="cuda")).shape == (2, 4, 0)


def _muon_state(shapes, gdtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ps = [torch.randn(s, generator=g, device="cuda") * math.sqrt(2 / max(s)) for s in shapes]
    gs = [(1e-3 * _matrix(s[0], s[1], "noise", seed=i + 1)).to(gdtype) for i, s in enumerate(shapes)]
    ms = [1e-3 * _matrix(s[0], s[1], "noise", seed=i + 100) for i, s in enumerate(shapes)]
    return ps, gs, ms


@pytest.mark.parametrize("adjust", ["match_rms_adamw", "original"])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("gdtype", [F32, BF16])
def test_muon_step(gdtype, nesterov, adjust):
    k = _k()
    shapes = [(64, 27), (64, 576), (256, 1152), (10, 512), (300, 70)]
    ps, gs, ms = _muon_state(shapes, gdtype)
    lps = [None if i == 1 else torch.zeros_like(p, dtype=BF16) for i, p in enumerate(ps)]
    w64, m64 = [p.double() for p in ps], [m.double() for m in ms]
    lr, mu, wd, gsc = 0.02, 0.95, 0.1, 0.5
    for step in range(3):
        k.muon_step(ps, gs, ms, lps, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, adjust_lr=adjust, grad_scale=gsc)
        for i, s in enumerate(shapes):
            d = gs[i].double() * gsc
            m64[i] = mu * m64[i] + (1 - mu) * d
            u = (1 - mu) * d + mu * m64[i] if nesterov else m64[i]
            adj = 0.2 * math.sqrt(max(s)) if adjust == "match_rms_adamw" else math.sqrt(max(1, s[0] / s[1]))
            o = _ns64(u)
            w64[i] = w64[i] * (1 - lr * wd) - lr * adj * o
            # momentum: three roundings a step; weights: the update's NS_TOL and two roundings a step
            assert (ms[i].double() - m64[i]).norm() <= 4 * (step + 1) * 2.0 ** -24 * (m64[i].norm() + d.norm())
            assert (ps[i].double() - w64[i]).norm() <= (step + 1) * (lr * adj * NS_TOL * o.norm() + 4 * 2.0 ** -24 * w64[i].norm())
            if lps[i] is not None:
                assert torch.equal(lps[i], ps[i].to(BF16))


def test_muon_step_leaves_what_lies_around_it():
    k = _k()
    ps, gs, ms = _muon_state([(65, 130)], F32)
    flat = [torch.full((65 * 130 + 128,), 7.5, device="cuda", dtype=t) for t in (F32, F32, BF16)]
    view = [f[64:64 + 65 * 130].view(65, 130) for f in flat]
    view[0].copy_(ps[0])
    view[1].copy_(ms[0])
    k.muon_step([view[0]], gs, [view[1]], [view[2]], lr=0.01)
    for f in flat:
        assert (f[:64] == 7.5).all() and (f[64 + 65 * 130:] == 7.5).all()


def test_muon_repeats_bit_for_bit_on_streams_and_in_graphs():
    k = _k()
    shapes = [(64, 576), (300, 70), (128, 1152)]

    def fresh(seed=0):
        ps, gs, ms = _muon_state(shapes, BF16, seed)
        return ps, gs, ms, [p.to(BF16) for p in ps]

    a = fresh()
    k.muon_step(*a, lr=0.01)
    b, c = fresh(), fresh()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        k.muon_step(*b, lr=0.01)
    k.muon_step(*c, lr=0.01)                    # next to the other one
    torch.cuda.synchronize()
    for x, y, z in zip(a, b, c):
        for t, u, v in zip(x, y, z):
            assert torch.equal(t, u) and torch.equal(t, v)
    states = [fresh(0), fresh(5)]
    want = [fresh(0), fresh(5)]
    graphs = []
    for st in states:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            k.muon_step(*st, lr=0.01)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        for st in want:
            k.muon_step(*st, lr=0.01)
        for st, w in zip(states, want):
            for x, y in zip(st, w):
                for t, u in zip(x, y):
                    assert torch.equal(t, u)


def _tol_of_long_sums(m):
    """NS_TOL plus what sums of m products lose.  Behind three steps Q is a^3 I and a matrix of about a^3 / m: Q X adds up
    one term a^3 X and m small ones that cancel it, in m / 32 instructions, each of which rounds a partial sum (between
    a^3 X and X, squares a third of the first's on average) off by up to 2^-23 of it (3^-1/2 of that on average; the unit
    need not round to nearest).  The second segment multiplies what lies across G's directions by a^2: an error of
    a^5 2^-23 / 3 = 1.9e-5 an instruction, independent of each other, next to the 1e-4 that NS_TOL is twice of.  (At
    1980 x 2010 and rank one 2.0e-4, at 4150 x 4210 3.0e-4; a loop of f32 products 3.7e-4 and 5.2e-4, by the same sums.)"""
    return 2 * math.sqrt((NS_TOL / 2) ** 2 + m / 32 * (COEFFS[0] ** 5 * 2.0 ** -23 / 3) ** 2)


# m x n, and the tile sides of: Gram, polynomial, P A with P Q, Q X between segments, last Q X.  No side a multiple of 128
# or 192.
TILED = [(1980, 2010, (64, 64, 64, 128, 128)), (2450, 2530, (128, 128, 192, 192, 192)), (4150, 4210, (192, 192, 192, 192, 192))]


@pytest.mark.parametrize("kind", ["full", "noise", "rank1"])
@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("m,n,sides", TILED)
def test_newton_schulz_in_large_tiles(m, n, sides, tall, kind):
    """The 192- and 128-wide tiles (staged through LDS) in every product of the chain, with tiles that end inside the
    matrix."""
    from distributed_training_pytorch_amd import _lib
    rows, cols = (n, m) if tall else (m, n)
    assert tuple(_lib.hip().dtp_ns_tile(rows, cols, p) for p in range(5)) == sides
    g = _matrix(rows, cols, kind, seed=rows)
    o = _k().newton_schulz(g, out_dtype=F32)
    assert _rel(o, _ns64(g)) <= _tol_of_long_sums(m)
    if kind == "noise":                                # a wrong tile is off by its own size, roundings spread over the rows
        d = (o.double() - _ns64(g)).abs()
        rows_off = (d.norm(dim=1) / _ns64(g).norm(dim=1)).max().item()
        assert rows_off <= 10 * _tol_of_long_sums(m)
        assert torch.equal(_k().newton_schulz(g.to(BF16).float(), out_dtype=F16), _k().newton_schulz(g.to(BF16), out_dtype=F16))


def test_muon_step_of_large_matrices_beside_small_ones():
    """Matrices with a short side above 1024 are worked off alone, the others together, in any order of the list."""
    k = _k()
    shapes = [(64, 576), (2450, 2530), (30, 70), (2530, 2450), (1100, 1200), (512, 300)]
    ps, gs, ms = _muon_state(shapes, F32)
    lps = [torch.zeros_like(p, dtype=BF16) for p in ps]
    w64, m64 = [p.double() for p in ps], [m.double() for m in ms]
    lr, mu, wd = 0.02, 0.95, 0.1
    k.muon_step(ps, gs, ms, lps, lr=lr, momentum=mu, weight_decay=wd)
    for i, s in enumerate(shapes):
        d = gs[i].double()
        m64[i] = mu * m64[i] + (1 - mu) * d
        o = _ns64((1 - mu) * d + mu * m64[i])
        adj = 0.2 * math.sqrt(max(s))
        w64[i] = w64[i] * (1 - lr * wd) - lr * adj * o
        assert (ms[i].double() - m64[i]).norm() <= 4 * 2.0 ** -24 * (m64[i].norm() + d.norm())
        assert (ps[i].double() - w64[i]).norm() <= lr * adj * _tol_of_long_sums(min(s)) * o.norm() + 4 * 2.0 ** -24 * w64[i].norm(), s
        assert torch.equal(lps[i], ps[i].to(BF16))


@pytest.mark.parametrize("rows,cols", [(64, 64), (7, 50), (100, 128), (900, 40), (200, 300)])
@pytest.mark.parametrize("eps", [1e-37, 1e-40])
def test_newton_schulz_of_zero_and_next_to_it(rows, cols, eps):
    """1 / (|G| + eps) leaves f32 here; X_0 does not.  (eps is an f32 in the formula: 1e-40 is 7e-6 off as one.)"""
    k = _k()
    assert (k.newton_schulz(torch.zeros(rows, cols, device="cuda"), eps=eps, out_dtype=F32) == 0).all()
    for size in (1e-38, 1e-36):
        g = _matrix(rows, cols, "full") * size
        assert _rel(k.newton_schulz(g, eps=eps, out_dtype=F32), _ns64(g, eps=torch.tensor(eps, dtype=F32).item())) <= NS_TOL
    ps, gs, ms = [torch.randn(rows, cols, device="cuda")], [torch.zeros(rows, cols, device="cuda")], [torch.zeros(rows, cols, device="cuda")]
    was = ps[0].clone()
    k.muon_step(ps, gs, ms, [None], lr=0.5, weight_decay=0.0, eps=eps)
    assert torch.equal(ps[0], was)


@pytest.mark.parametrize("rows,cols", [(1, 2 ** 20), (2 ** 20, 3), (40, 300_001), (200_003, 130)])
def test_newton_schulz_of_very_long_matrices(rows, cols):
    """The longest sides that are taken.  The Gram matrix adds n / 32 products' sums, shared by 32 waves: off by at most
    n / 1024 of 2^-24, along G's own directions, where |dO/O| <= 4 |dA/A|."""
    k = _k()
    g = _matrix(rows, cols, "full")
    tol = NS_TOL + 4 * max(rows, cols) / 1024 * 2.0 ** -24
    assert _rel(k.newton_schulz(g, out_dtype=F32), _ns64(g)) <= tol


def test_newton_schulz_takes_twelve_steps():
    """Behind five steps singular values lie in [0.68, 1.13], where a step multiplies an error by
    |a + 3 b x^2 + 5 c x^4| <= 1.71."""
    k = _k()
    for rows, cols in ((64, 64), (300, 170)):
        g = _matrix(rows, cols, "noise", seed=8)
        assert _rel(k.newton_schulz(g, steps=12, out_dtype=F32), _ns64(g, 12)) <= 1.71 ** 7 * NS_TOL
