"""Calls of suave_amd.operators at the edges of their ranges: rows of subnormal numbers, lists that share a choice of tile,
tensors with one row far larger than the others, classes that no row gives a chance, and what a served model keeps."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -149  # binary32's smallest number


def _subnormal_rows(cols):
    """Rows of both signs whose largest element is m STEP: their scale, m / 127 STEP rounded, has few bits, and m / scale reaches 190."""
    rows = []
    for m in (1, 63, 64, 65, 100, 127, 128, 150, 190, 191, 300, 317, 500, 5000, 16000, 16129, 20000, 10 ** 6):
        for sign in (1, -1):
            j = np.rint(np.linspace(-m, m, cols)).astype(np.int64)
            j[cols // 2] = m
            rows.append(sign * j)
    return np.stack(rows).astype(np.float64) * STEP


def _definition(x):
    """q (-127 .. 127) and scale of float64 rows that binary32 holds."""
    s = (np.abs(x).max(axis=1).astype(np.float32) * (np.float32(1) / np.float32(127))).astype(np.float32)
    ok = s > 0
    q = np.where(ok[:, None], np.rint(x / np.where(ok, s, 1).astype(np.float64)[:, None]), 0.0)
    return np.clip(q, -127, 127), s


@pytest.mark.parametrize("cols", [8, 61, 700, 5000])
def test_subnormal_rows_saturate(cols):
    import torch
    from suave_amd import operators as ops

    x = _subnormal_rows(cols)
    wq, ws = _definition(x)
    t = torch.from_numpy(x.astype(np.float32)).cuda()
    assert np.array_equal(t.cpu().numpy().astype(np.float64), x)
    q, s = ops.quantize_rows(t)
    assert np.array_equal(s.cpu().numpy(), ws)
    assert np.array_equal(q.cpu().numpy().astype(np.float64), wq)
    # q through the product with 127 times the identity: 127 q s, rounded once (127 127 7874 STEP, of the largest row, has 27 bits)
    if cols > 700:
        return
    eye = torch.zeros((cols, (cols + 15) // 16 * 16), dtype=torch.int8, device="cuda:0")
    eye[:, :cols] = torch.eye(cols, device="cuda:0").mul(127).to(torch.int8)
    one = torch.ones(cols, device="cuda:0")
    want = (127.0 * wq * ws.astype(np.float64)[:, None]).astype(np.float32)
    n = len(x)
    for rows in ([range(i, min(i + 5, n)) for i in range(0, n, 5)] + [range(n), [i % n for i in range(100)]]):  # few rows: quantised inside the product
        rows = list(rows)
        got = ops.linear_quantized(t[rows].contiguous(), eye[:, :cols], one)
        assert np.array_equal(got.cpu().numpy(), want[rows]), len(rows)


def _random(r, c, seed, dtype):
    import torch

    g = torch.Generator(device="cuda:0").manual_seed(seed)
    return (torch.randn((r, c), generator=g, device="cuda:0") * 1e-3).to(dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shapes", [[(3000, 3000), (3000, 3000)], [(2300, 3000), (1100, 2600), (3000, 2300)], [(1500, 1500), (2900, 2100)]])
def test_a_matrix_is_the_same_in_any_list(shapes, dtype):
    """Sizes whose tile depends on how much work the list holds: every matrix has the bits that it has alone."""
    import torch
    from suave_amd import operators as ops

    us = [_random(r, c, 5 * r + c + i, getattr(torch, dtype)) for i, (r, c) in enumerate(shapes)]
    for u, got in zip(us, ops.orthogonalize(us)):
        assert torch.equal(got, ops.orthogonalize([u])[0]), tuple(u.shape)


def test_growing_sizes_of_one_block():
    """Matrices that go through one block, their LDS growing from call to call past 64 KB: what an earlier call was allowed is not enough."""
    import torch
    from suave_amd import operators as ops

    from tests.test_hip_ortho import _check

    for shapes in ([(40, 40)], [(65, 64)], [(63, 130)], [(128, 128)], [(16, 1100)], [(16, 1800)], [(16, 2239)], [(100, 90), (128, 128)]):
        us = [_random(r, c, r + c, torch.float32) for r, c in shapes]
        for u, got in zip(us, ops.orthogonalize(us)):
            _check(got, u)


def _ce_case(n, c, d, dtype, seed):
    import torch

    g = torch.Generator(device="cuda:0").manual_seed(seed)
    x = torch.randn((n, d), generator=g, device="cuda:0")
    w = torch.randn((c, d), generator=g, device="cuda:0") * (2.0 / math.sqrt(d))
    b = torch.randn(c, generator=g, device="cuda:0") * 0.3
    y = torch.randint(0, c, (n,), generator=g, device="cuda:0", dtype=torch.int32)
    return x.to(dtype), w.to(dtype), b, y, torch.rand(c, generator=g, device="cuda:0") + 0.5


def _rows_alone(x, w, b, y, cw, got, large_row):
    """Every row against float64, each by bounds of ITS OWN size.

    Logits: with X_i = |x_i| max |W_c| over the classes that count, off by LOGIT_i = 2^-20 X_i + 2^-23 max |l_i|
    (tests/test_hip_linear_ce.py); lse by twice that and 2^-23 (log C + 3 + |lse|), the loss by one more LOGIT_i.
    G = f (p - [c = y]), f the row's share of the weight: p is off by 4 LOGIT_i + 2^-21 of itself, G is held to 2^-8 (bf16), 2^-11 (one
    fp16 plane) or 2^-22, and no finer than 2^-38 of the largest f.  (Row `large_row`, if any: its logits lie so far apart that its p are 0
    and 1.)  x and W are held to 2^-23 of themselves, but in the sums over rows and classes no finer than 2^-38 of the tensor's largest
    element; sums in fp32: 2^-20 of their absolute terms; the result's own rounding."""
    import torch

    xd, wd = x.double(), w.double()
    l = xd @ wd.t() + b.double()
    lse = torch.logsumexp(l, dim=1)
    row_w = torch.ones_like(lse) if cw is None else cw.double()[y.long()]
    loss = row_w * (lse - l.gather(1, y.long()[:, None])[:, 0])
    count = torch.isfinite(b)
    size = xd.norm(dim=1) * wd.norm(dim=1)[count].max()
    logit = 2.0 ** -20 * size + 2.0 ** -23 * l[:, count].abs().amax(dim=1)

    def within(name, e, lim):
        assert bool((e <= lim).all()), (name, float((e / lim).max()))

    lim = 2 * logit + 2.0 ** -23 * (math.log(len(b)) + 3 + lse.abs())
    within("lse", (got["lse"].double() - lse).abs(), lim)
    within("row_loss", (got["row_loss"].double() - loss).abs(), row_w * (lim + logit) + 2.0 ** -23 * loss.abs())
    if "dx" not in got:
        return
    f = (row_w / row_w.sum())[:, None]
    p = torch.exp(l - lse[:, None])
    G = p.clone()
    G[torch.arange(len(y), device=y.device), y.long()] -= 1.0
    if large_row is not None:
        logit[large_row] = 0.0
    bf = x.dtype == torch.bfloat16
    half = 2.0 ** -22 if not bf else 2.0 ** -11 if cw is not None or len(y) <= 8 else 2.0 ** -8
    dG = f * ((4 * logit[:, None] + 2.0 ** -21) * p + half * G.abs()) + 2.0 ** -38 * f.max()
    G, u = G * f, torch.finfo(x.dtype).eps / 2
    dX, dW = (2.0 ** -23 * t.abs() + 2.0 ** -38 * t.abs().max() for t in (xd, wd))
    for name, want, lim, mag in (("dx", G @ wd, dG @ wd.abs() + G.abs() @ dW, G.abs() @ wd.abs()),
                                 ("dweight", G.t() @ xd, dG.t() @ xd.abs() + G.abs().t() @ dX, G.abs().t() @ xd.abs())):
        within(name, (got[name].double() - want).abs(), (lim + 2.0 ** -20 * mag) * 1.01 + u * want.abs() * 1.01 + 1e-38)


@pytest.mark.parametrize("n,c,d", [(1, 80, 9), (8, 300, 40), (12, 90, 24), (64, 1000, 32), (300, 200, 70), (90, 700, 300), (40, 257, 3), (700, 1500, 130),
                                   (2000, 1500, 40)])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_large_row_does_not_reach_the_others(n, c, d, weighted, dtype):
    """One row of x, and one class that is never predicted (bias -inf), 10^4 .. 10^9 times as large as the others: the losses of the
    other rows are as exact as without them, the gradients to 2^-38 of the largest."""
    import torch
    from suave_amd import operators as ops

    at = min(5, n - 1)
    for factor in (1e4, 1e6, 1e9):
        for which in ("row", "class", "both"):
            x, w, b, y, cw = _ce_case(n, c, d, getattr(torch, dtype), seed=n + c + d)
            cw = cw if weighted else None
            y = torch.where(y == 7, torch.full_like(y, 8), y)
            if which != "class":
                x[at] *= factor
            if which != "row":
                w[7] *= factor
                b[7] = -float("inf")
            large = None if which == "class" else at
            only = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw, grad=False)
            got = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
            _rows_alone(x, w, b, y, cw, only, large)
            _rows_alone(x, w, b, y, cw, got, large)
            assert torch.equal(only["row_loss"], got["row_loss"]) or (dtype == "bfloat16" and (weighted or n <= 8))


def test_replays_with_and_without_large_rows():
    """A captured call takes the scales from the data of each replay."""
    import torch
    from suave_amd import operators as ops

    for n, c, d in ((40, 120, 24), (300, 700, 300)):  # (maxima found inside the packing launch, or by one of their own)
        x, w, b, y, cw = _ce_case(n, c, d, torch.float32, seed=1)
        x0, w0 = x.clone(), w.clone()
        ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
        for fx, fw in ((1.0, 1.0), (1e7, 1.0), (1.0, 1e-7), (1.0, 1.0), (1e5, 1e-5)):
            x.copy_(x0)
            w.copy_(w0)
            x[3] *= fx
            w[5] *= fw
            eager = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(out[k], eager[k]) for k in eager)
            _rows_alone(x, w, b, y, cw, out, 3 if fx > 1 else None)


def test_gradient_of_a_class_without_a_chance():
    """Classes whose probability is 2^-12 .. 2^-40 in every row: their row of dweight by itself, not beside the largest.  G is held
    in two fp16 planes relative to the largest row weight: off by 2^-22 of itself (and of exp's argument, 64 here: 2^-17) or by 2^-38."""
    import torch
    from suave_amd import operators as ops

    x, w, b, y, _ = _ce_case(200, 400, 48, torch.float32, seed=3)
    low = torch.arange(20, 35, device="cuda:0")
    b[low] = -torch.arange(8.0, 38.0, 2.0, device="cuda:0")
    y = torch.where((y >= 20) & (y < 35), torch.full_like(y, 1), y)
    got = ops.linear_cross_entropy(x, w, y, bias=b)
    l = x.double() @ w.double().t() + b.double()
    G = torch.softmax(l, dim=1)
    G[torch.arange(200, device="cuda:0"), y.long()] -= 1.0
    want, size = (G.t() @ x.double()) / 200, (G.abs().t() @ x.double().abs()) / 200
    lim = 2.0 ** -17 * size[low] + 2.0 ** -38 * x.double().abs().mean(dim=0) + 1e-38
    e = (got["dweight"].double() - want).abs()[low]
    assert bool((e <= lim).all()), float((e / lim).max())


def test_calibration_is_of_the_classifier_itself(tmp_path):
    """The temperature outlives the 8-bit weights (quantize_classifier(False), save): fitted while they serve, it is the one fitted without."""
    import pandas as pd
    from suave_amd.model import SUAVE
    from suave_amd.types import Schema

    rng = np.random.default_rng(1)
    n = 300
    df = pd.DataFrame({"a": rng.normal(size=n), "c": rng.integers(0, 3, n)})
    y = (df["a"].to_numpy() > 0.2).astype(int) + df["c"].to_numpy()
    m = SUAVE(Schema({"a": {"type": "real"}, "c": {"type": "cat", "n_classes": 3}}), behaviour="supervised", latent_dim=8, n_components=2,
              hidden_dims=(32, 16), random_state=0)
    m.fit(df, y=y, warmup_epochs=1, kl_warmup_epochs=1, head_epochs=2, finetune_epochs=1, decoder_refine_epochs=1)
    m.calibrate(df, y)
    want, proba = m._temperature_scaler.state_dict(), m.predict_proba(df)
    m.quantize_classifier()
    assert not np.array_equal(m.predict_proba(df), proba)
    m._temperature_scaler = type(m._temperature_scaler)()  # (a fit starts from the temperature it finds)
    m.calibrate(df, y)
    assert m._temperature_scaler.state_dict() == want
    path = m.save(tmp_path / "m.pt") or tmp_path / "m.pt"
    assert np.array_equal(SUAVE.load(path).predict_proba(df), proba)
    m.quantize_classifier(False)
    assert np.array_equal(m.predict_proba(df), proba)
