"""Calls of suave_amd.operators at the edges of their ranges: rows of subnormal numbers, lists that share a choice of tile, and
what a served model keeps."""

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
