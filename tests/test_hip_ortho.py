"""suave_orthogonalize / suave_muon_step (suave_amd.operators) against the definition in float64.

Tolerance.  The iteration multiplies a perturbation of X_k by up to a^(steps - k) (a = 3.4445, the slope of the step's
polynomial at 0), so rounding noise cannot be bounded usefully by the worst direction.  The bound is taken from the arithmetic
itself: the same iteration is run with every stored factor rounded as documented -- binary32 for float32 matrices, one
fp16 plane (X, A and B times 2^12) for bfloat16 ones -- and exact products in between; the kernel, whose sums differ in order and whose roundings therefore fall
elsewhere, may be FOUR times as far from float64 in the 2-norm (two independent errors of that size differ by sqrt(2); the three
plane products add sqrt(3) 2^-24), plus the rounding of the result (2^-8 for bfloat16).  Single entries: 64 times that rms.

A matrix with few directions may be rounded luckily by that iteration, so what the LAST step alone may add in binary32 is allowed on
top, per singular direction sigma <= 1.2, lambda = sigma^2 <= 1.45: two roundings of each term of (a + b lambda + c lambda^2) sigma:
2 (3.44 + 6.93 + 4.28) 1.2 2^-24 = 35 2^-24.  That is sqrt(s) times as much in the 2-norm of a matrix with short side s."""

import math

import pytest

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315


def _iterate(u, steps, eps, rnd):
    import torch

    x = u.double()
    x = rnd(x / (torch.linalg.matrix_norm(x) + eps))
    tall = u.shape[0] > u.shape[1]
    for k in range(steps):
        G = rnd(x.t() @ x if tall else x @ x.t())
        P = rnd(B * G + C * (G @ G) + A * torch.eye(G.shape[0], dtype=torch.float64, device=u.device))
        x = x @ P if tall else P @ x
        if k + 1 < steps:
            x = rnd(x)
    return x


def _exact(u, steps=5, eps=1e-7):
    return _iterate(u, steps, eps, lambda t: t)


def _tolerance(u, want, steps=5, eps=1e-7):
    import torch

    if u.dtype == torch.bfloat16:
        rnd = lambda t: (t * 4096.0).half().double() / 4096.0  # noqa: E731
    else:
        rnd = lambda t: t.float().double()  # noqa: E731
    off = float(torch.linalg.matrix_norm(_iterate(u, steps, eps, rnd) - want))
    size, s, bf = float(torch.linalg.matrix_norm(want)), min(u.shape), u.dtype == torch.bfloat16
    last = 35 * 2.0 ** -24
    return 4 * off + last * math.sqrt(s) + (4 * 2.0 ** -24 + (2.0 ** -8 if bf else 2.0 ** -24)) * size


def _check(got, u, steps=5, eps=1e-7):
    import torch

    want = _exact(u, steps, eps)
    tol = _tolerance(u, want, steps, eps)
    e = got.double() - want
    assert bool(torch.isfinite(got).all())
    assert float(torch.linalg.matrix_norm(e)) <= tol, (tuple(u.shape), float(torch.linalg.matrix_norm(e)) / tol)
    assert float(e.abs().max()) <= 64 * tol / math.sqrt(u.numel()) + (2.0 ** -8 if u.dtype == torch.bfloat16 else 0.0) * float(want.abs().max())


def _random(r, c, seed, dtype, scale=1e-3):
    import torch

    g = torch.Generator(device="cuda:0").manual_seed(seed)
    t = min(r, c, 4)
    low = torch.randn((r, t), generator=g, device="cuda:0") @ torch.randn((t, c), generator=g, device="cuda:0")
    return ((torch.randn((r, c), generator=g, device="cuda:0") + 0.3 * low) * scale).to(dtype)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (8, 8), (64, 64), (65, 64), (63, 130), (130, 63), (129, 129), (300, 20), (20, 300), (257, 1000),
          (1000, 257), (513, 515)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("r,c", SHAPES)
def test_one_matrix_matches_the_definition(r, c, dtype):
    import torch
    from suave_amd import operators as ops

    u = _random(r, c, r * 1000 + c, getattr(torch, dtype))
    _check(ops.orthogonalize([u])[0], u)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_lists_of_any_shapes_and_every_tile_size(dtype):
    """More matrices than one group of launches takes; shapes large enough for the larger tiles; one call equals many."""
    import torch
    from suave_amd import operators as ops

    dt = getattr(torch, dtype)
    us = [_random(5 + 13 * i, 200 - 7 * i, i, dt) for i in range(27)]
    together = ops.orthogonalize(us)
    for u, o in zip(us, together):
        _check(o, u)
        assert torch.equal(ops.orthogonalize([u])[0], o)
    big = [_random(1100, 2200, 1, dt), _random(2050, 1030, 2, dt), _random(1500, 1500, 3, dt), _random(3000, 2900, 4, dt)]
    for u, o in zip(big, ops.orthogonalize(big)):
        _check(o, u)


def test_steps_and_eps():
    import torch
    from suave_amd import operators as ops

    for steps in (1, 2, 3, 7):
        for u in (_random(90, 150, 5, torch.float32), _random(150, 90, 6, torch.bfloat16)):
            _check(ops.orthogonalize([u], steps=steps)[0], u, steps=steps)
    u = _random(60, 100, 7, torch.float32)
    _check(ops.orthogonalize([u], eps=0.5)[0], u, eps=0.5)


def test_sizes_of_the_input():
    """Norms below eps (the iteration is then still growing X), subnormal and huge entries, zeros, non-finite entries."""
    import torch
    from suave_amd import operators as ops

    for scale in (1e-9, 1e-12, 1e-25, 1e-36, 1e20, 1e35):
        u = _random(70, 40, 8, torch.float32, scale)
        got, want = ops.orthogonalize([u])[0], _exact(u)
        if scale < 1e-30:  # binary32 of the tiny result itself is all that is asked
            assert float((got.double() - want).abs().max()) <= 2.0 ** -18 * float(want.abs().max()) + 1e-44
        else:
            assert float(torch.linalg.matrix_norm(got.double() - want)) <= _tolerance(u, want)
    z = torch.zeros(33, 50, device="cuda:0")
    n, f = _random(40, 30, 9, torch.float32), _random(40, 30, 10, torch.float32)
    n[3, 4], f[39, 29] = float("nan"), float("inf")
    good = _random(31, 45, 11, torch.float32)
    oz, on, of, og = ops.orthogonalize([z, n, f, good])
    assert bool((oz == 0).all()) and bool(torch.isnan(on).all()) and bool(torch.isnan(of).all())
    _check(og, good)


def test_strides_in_place_and_what_lies_outside():
    import torch
    from suave_amd import operators as ops

    for dt in (torch.float32, torch.bfloat16):
        us = [_random(70, 101, 1, dt), _random(101, 37, 2, dt)]
        want = ops.orthogonalize(us)
        hold = [torch.full((u.shape[0], u.shape[1] + 9), 5.0, dtype=dt, device="cuda:0") for u in us]
        views = [h[:, 3:3 + u.shape[1]] for h, u in zip(hold, us)]
        for v, u in zip(views, us):
            v.copy_(u)
        ops.orthogonalize(views, out=views)
        for h, v, w in zip(hold, views, want):
            assert torch.equal(v, w) and bool((h[:, :3] == 5).all()) and bool((h[:, 3 + w.shape[1]:] == 5).all())


@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (False, 0.1)])
def test_muon_steps_match_the_definition(nesterov, decay):
    import torch
    from suave_amd import operators as ops

    shapes = [(256, 205), (128, 256), (256, 32), (90, 7), (5, 300)]
    p = [_random(r, c, i, torch.float32, 0.05) for i, (r, c) in enumerate(shapes)]
    m = [torch.zeros_like(t) for t in p]
    lr = [0.02, 0.01, 0.05, 0.02, 0.03]
    for step in range(3):
        g = [_random(r, c, 50 + 10 * step + i, torch.float32) for i, (r, c) in enumerate(shapes)]
        p0, m0 = [t.double() for t in p], [t.double() for t in m]
        ops.muon_step(p, g, m, lr=lr, momentum=0.9, nesterov=nesterov, weight_decay=decay)
        for i in range(len(shapes)):
            m1 = 0.9 * m0[i] + g[i].double()
            assert float((m[i].double() - m1).abs().max()) <= 2.0 ** -23 * float(m1.abs().max()) * 2
            u = (g[i].double() + 0.9 * m1 if nesterov else m1).float()
            o = _exact(u)
            s = lr[i] * math.sqrt(max(1.0, shapes[i][0] / shapes[i][1]))
            want = p0[i] * (1 - lr[i] * decay) - s * o
            # the update's own tolerance, its input's rounding (u in binary32: once more that size), the result's
            tol = s * 2 * _tolerance(u, o) + 2.0 ** -23 * float(torch.linalg.matrix_norm(want))
            assert float(torch.linalg.matrix_norm(p[i].double() - want)) <= tol


def test_views_of_flat_buffers():
    """Parameters as the engine keeps them: one flat buffer, row strides rounded up to 4; pads and biases stay as they were."""
    import torch
    from suave_amd import operators as ops

    flat = torch.full((3000,), 0.5, device="cuda:0")
    grad, mom = torch.randn(3000, device="cuda:0"), torch.zeros(3000, device="cuda:0")
    def view(t): return [t[8:8 + 20 * 24].view(20, 24)[:, :21], t[1000:1000 + 40 * 12].view(40, 12)[:, :10]]
    ops.muon_step(view(flat), view(grad), view(mom), lr=0.1)
    touched = torch.zeros(3000, dtype=torch.bool, device="cuda:0")
    for v in view(touched):
        v.fill_(True)
    assert bool((flat[~touched] == 0.5).all()) and bool((mom[~touched] == 0).all()) and bool((flat[touched] != 0.5).any())
    want = 0.5 - 0.1 * 2.0 * _exact(view(grad)[1] * 1.95)  # sqrt(40 / 10) = 2
    assert float((view(flat)[1].double() - want).abs().max()) <= 1e-5


def test_empty_lists_and_refusals():
    import torch
    from suave_amd import lib as slib
    from suave_amd import operators as ops

    assert ops.orthogonalize([]) == [] and ops.muon_step([], [], [], lr=0.1) is None
    u = _random(8, 12, 1, torch.float32)
    for bad, msg in (([u, u.bfloat16()], "types"), ([u.half()], "types"), ([u.t()], "contiguous"), ([u[:0]], "at least one"), ([u[0]], "matrix"),
                     ([u, u.cpu()], "must be on")):
        with pytest.raises(ValueError, match=msg):
            ops.orthogonalize(bad)
    with pytest.raises(ValueError, match="shape"):
        ops.orthogonalize([u], out=[torch.empty(12, 8, device="cuda:0")])
    for kw in (dict(steps=0), dict(steps=17), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(slib.SuaveHipError):
            ops.orthogonalize([u], **kw)
    z = torch.zeros_like(u)
    for kw in (dict(lr=-1.0), dict(lr=float("inf")), dict(lr=0.1, momentum=1.0), dict(lr=0.1, weight_decay=-0.1)):
        with pytest.raises(slib.SuaveHipError):
            ops.muon_step([u], [u], [z], **kw)
    with pytest.raises(ValueError, match="types"):
        ops.muon_step([u.bfloat16()], [u], [z], lr=0.1)
    with pytest.raises(ValueError, match="shape"):
        ops.muon_step([u], [u[:4]], [z], lr=0.1)
    with pytest.raises(slib.SuaveHipError, match="GPU"):
        ops.orthogonalize([u.cpu()])


def test_other_stream_and_captured_graph():
    import torch
    from suave_amd import operators as ops

    us = [_random(100, 60, 1, torch.float32), _random(64, 200, 2, torch.float32)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.orthogonalize(us)
    torch.cuda.current_stream().wait_stream(side)
    b = ops.orthogonalize(us)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    p, m = [torch.randn_like(u) for u in us], [torch.zeros_like(u) for u in us]
    p2, m2 = [t.clone() for t in p], [t.clone() for t in m]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.orthogonalize(us)
        ops.muon_step(p, us, m, lr=0.05)
    for seed in (3, 4, 5):
        for i, u in enumerate(us):
            u.copy_(_random(u.shape[0], u.shape[1], seed + 10 * i, torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        ops.muon_step(p2, us, m2, lr=0.05)
        assert all(torch.equal(x, y) for x, y in zip(out, ops.orthogonalize(us)))
        assert all(torch.equal(x, y) for x, y in zip(p + m, p2 + m2))


@pytest.mark.parametrize("r,c", [(1, 5), (3, 50), (4, 400), (8, 8), (40, 500), (96, 39), (127, 300), (1000, 77)])
def test_short_sides_in_bfloat16_are_off_by_their_rounding_alone(r, c):
    """Up to 127 the bfloat16 iteration is binary32's: with d its error, the result is bf16(O + d), so it is off by at most
    |bf16(O) - O| + 3 |d| (rounding moves by at most |d| where its argument does, twice, and d itself)."""
    import torch
    from suave_amd import operators as ops

    u = _random(r, c, r + c, torch.bfloat16)
    want = _exact(u)
    got = ops.orthogonalize([u, _random(200, 300, 1, torch.bfloat16)])[0]
    norm = torch.linalg.matrix_norm
    assert float(norm(got.double() - want)) <= float(norm(want.bfloat16().double() - want)) + 3 * _tolerance(u.float(), want)
    assert torch.equal(got, ops.orthogonalize([u])[0])


@pytest.mark.parametrize("r,c", [(1, 1), (1, 39), (42, 1), (3, 392), (16, 16), (16, 2239), (16, 2240), (2240, 16), (7, 3000), (52, 4)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_short_sides_up_to_sixteen_are_rounded_once(r, c, dtype):
    """Up to 16 the whole iteration is one of small matrices in doubles: the result is off by its own rounding (half a step, 2^-24 or
    2^-8 relative), or by the general bound where the matrix is too long for that."""
    import torch
    from suave_amd import operators as ops

    dt = getattr(torch, dtype)
    u = _random(r, c, 7 * r + c, dt)
    want, (got,) = _exact(u), ops.orthogonalize([u])
    if min(r, c) * (max(r, c) | 1) <= 35840:
        half = torch.finfo(dt).eps / 2
        # the doubles' own errors, 2^-53 times 3.4445^5, are lost in it
        assert bool(((got.double() - want).abs() <= half * want.abs() * (1 + 1e-6) + 1e-11).all())
    else:
        _check(got, u)
    p, m = torch.zeros(r, c, device="cuda:0"), torch.zeros(r, c, device="cuda:0")
    ops.muon_step([p], [u.float()], [m], lr=1.0, momentum=0.5, nesterov=True)
    assert torch.equal(m, u.float())
    s = math.sqrt(max(1.0, r / c))
    tol = s * 2 * _tolerance((1.5 * u.double()).float(), want) + 2.0 ** -23 * s * float(torch.linalg.matrix_norm(want))
    assert float(torch.linalg.matrix_norm(p.double() + s * want)) <= tol


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shapes", [[(1024, 4096), (4096, 1024)], [(700, 3001), (650, 2900), (2500, 690), (1000, 2000)]])
def test_long_lists_of_large_matrices_are_each_matrix_alone(shapes, dtype):
    """More blocks than CUs: other tiles, the same sums, so the same bits; and the definition."""
    import torch
    from suave_amd import operators as ops

    us = [_random(r, c, 3 * r + c, getattr(torch, dtype)) for r, c in shapes]
    together = ops.orthogonalize(us)
    for u, got in zip(us, together):
        assert torch.equal(got, ops.orthogonalize([u])[0])
    _check(together[-1], us[-1])
