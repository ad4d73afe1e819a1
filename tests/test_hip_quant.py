"""suave_quantize_rows / suave_linear_quantized (suave_amd.operators) against their definition in float64.

q and scale are held to equality: the scale is a correctly rounded binary32 quotient, q the exact nearest integer (ties to
even) of x / scale.  The product's integer sums are exact; out = fma(float(sum), s_x * s_w, b) rounds three times in binary32
(the sum, the product of the scales, the result): 3 * 2^-24 of |s_x s_w sum| plus 2^-24 of the result, and a bfloat16 result
once more (2^-8)."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _quantized(x):
    """(q, scale) of the definition, int64 / float32, on the host in float64."""
    x = x.double().cpu().numpy()
    with np.errstate(all="ignore"):
        s = (np.abs(x).max(axis=1).astype(np.float32) * (np.float32(1) / np.float32(127))).astype(np.float32)
        ok = np.isfinite(s) & (s > 0)
        q = np.where(ok[:, None], np.rint(x / np.where(ok, s, 1).astype(np.float64)[:, None]), 0.0)
    return np.clip(q, -127, 127).astype(np.int64), s


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 15), (5, 16), (7, 17), (130, 100), (4, 1023), (9, 1040), (6, 2049), (3, 4111), (2, 9000)])
def test_rows_are_the_nearest_integers(n, k, dtype):
    import torch
    from suave_amd import operators as ops

    g = torch.Generator(device="cuda:0").manual_seed(n * 100 + k)
    x = torch.randn((n, k), generator=g, device="cuda:0") * torch.logspace(-6, 6, n, device="cuda:0")[:, None]
    x = x.to(getattr(torch, dtype))
    q, s = ops.quantize_rows(x)
    wq, wsc = _quantized(x)
    assert np.array_equal(s.cpu().numpy(), wsc) and np.array_equal(q.cpu().numpy().astype(np.int64), wq)
    assert q.stride(0) % 16 == 0 and bool((q.as_strided((n, q.stride(0)), (q.stride(0), 1))[:, k:] == 0).all())


def test_borders_ties_and_odd_rows():
    """Values on and next to half-integers of the scale, rows of zeros, tiny and huge rows, infinities and NaN."""
    import torch
    from suave_amd import operators as ops

    rows = []
    for amax in (127.0, 1.0, 3.0, 0.37, 1e30, 1e-30, 1e-38, 1e-42, 3e-45):
        s = np.float32(np.float32(amax) * (np.float32(1) / np.float32(127)))
        half = (np.arange(-127, 127) + 0.5) * np.float64(s)
        v = half.astype(np.float32)
        rows.append(np.concatenate([[amax], v, np.nextafter(v, np.float32(1e38)), np.nextafter(v, np.float32(-1e38))]).astype(np.float32))
    x = np.stack(rows)
    x = np.clip(x, -x[:, :1], x[:, :1])
    t = torch.from_numpy(x).cuda()
    q, s = ops.quantize_rows(t)
    wq, wsc = _quantized(t)
    assert np.array_equal(s.cpu().numpy(), wsc) and np.array_equal(q.cpu().numpy().astype(np.int64), wq)
    x = torch.ones((4, 40), device="cuda:0")
    x[0], x[1, 3], x[2, 39] = 0.0, float("inf"), float("nan")
    q, s = ops.quantize_rows(x)
    assert float(s[0]) == 0 and math.isinf(float(s[1])) and math.isnan(float(s[2])) and float(s[3]) == np.float32(1) / np.float32(127)
    assert bool((q[:3] == 0).all()) and bool((q[3] == 127).all())
    w, ws = ops.quantize_rows(torch.randn(20, 40, device="cuda:0"))
    b = torch.randn(20, device="cuda:0")
    out = ops.linear_quantized(x, w, ws, bias=b)
    assert torch.equal(out[0], b) and bool(torch.isnan(out[1:3]).all()) and bool(torch.isfinite(out[3]).all())


def _check_product(x, w, ws, b, out):
    import torch

    xq, xs = _quantized(x)
    xs = torch.from_numpy(xs.astype(np.float64)).cuda()
    sums = torch.from_numpy(xq.astype(np.float64)).cuda() @ w.double().t()
    core = sums * xs[:, None] * ws.double()[None, :]
    want = core + (0.0 if b is None else b.double())
    u = 2.0 ** -8 if x.dtype == torch.bfloat16 else 0.0
    lim = 3.01 * 2.0 ** -24 * core.abs() + (2.0 ** -24 + u) * 1.001 * want.abs() + 1e-38
    e = (out.double() - want).abs()
    assert bool((e <= lim).all()), float((e / lim).max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 1000, 256), (2, 65, 15), (15, 63, 129), (16, 200, 64), (17, 130, 100), (32, 64, 300),
                                   (33, 257, 48), (64, 500, 2049), (65, 100, 33), (128, 128, 128), (200, 333, 517), (300, 70, 1000),
                                   (4100, 4200, 130), (3, 50000, 77)])
def test_product_matches_the_definition(m, n, k, dtype):
    import torch
    from suave_amd import operators as ops

    g = torch.Generator(device="cuda:0").manual_seed(m * 31 + n * 7 + k)
    x = (torch.randn((m, k), generator=g, device="cuda:0") * 3).to(getattr(torch, dtype))
    w, ws = ops.quantize_rows(torch.randn((n, k), generator=g, device="cuda:0"))
    b = torch.randn(n, generator=g, device="cuda:0") if (m + n) % 2 else None
    out = ops.linear_quantized(x, w, ws, bias=b)
    _check_product(x, w, ws, b, out)
    assert torch.equal(ops.linear_quantized(x, w, ws, bias=b), out)


def test_longest_sums_are_exact():
    """All levels at +-127 over the longest rows: the sum is 127^2 * 131072, one short of 2^31's range."""
    import torch
    from suave_amd import operators as ops

    k = 131072
    for m in (3, 70):
        x = torch.full((m, k), 2.0, device="cuda:0")
        x[1] = -2.0
        w = torch.full((130, k), 127, dtype=torch.int8, device="cuda:0")
        w[5] = -127
        ws = torch.ones(130, device="cuda:0")
        _check_product(x, w, ws, None, ops.linear_quantized(x, w, ws))


def test_strides_and_what_lies_outside():
    import torch
    from suave_amd import operators as ops

    g = torch.Generator(device="cuda:0").manual_seed(3)
    for m in (5, 40, 100):
        for dt in (torch.float32, torch.bfloat16):
            xb = torch.full((m, 90), float("nan"), dtype=dt, device="cuda:0")
            xb[:, 3:73] = torch.randn((m, 70), generator=g, device="cuda:0").to(dt)
            wq, ws = ops.quantize_rows(torch.randn((150, 70), generator=g, device="cuda:0"))
            wb = torch.randint(-128, 128, (150, 112), generator=g, device="cuda:0").to(torch.int8)  # other bytes behind the rows
            wb[:, 16:86] = wq
            ob = torch.full((m, 161), 7.0, dtype=dt, device="cuda:0")
            out = ops.linear_quantized(xb[:, 3:73], wb[:, 16:86], ws, out=ob[:, 5:155])
            _check_product(xb[:, 3:73], wq, ws, None, out)
            assert bool((ob[:, :5] == 7).all()) and bool((ob[:, 155:] == 7).all())


def test_empty_calls_and_refusals():
    import torch
    from suave_amd import lib as slib
    from suave_amd import operators as ops

    x = torch.randn(4, 20, device="cuda:0")
    w, ws = ops.quantize_rows(torch.randn(6, 20, device="cuda:0"))
    assert ops.linear_quantized(x[:0], w, ws).shape == (0, 6)
    q, s = ops.quantize_rows(x[:0])
    assert q.shape == (0, 20) and s.shape == (0,)
    for kw, msg in ((dict(weight=w.contiguous()), "16 bytes"), (dict(weight=w.float()), "types"), (dict(x=x[:, :7]), "columns"),
                    (dict(weight_scale=ws[:3]), "vector"), (dict(bias=ws.double()), "type"), (dict(x=x.half()), "types"),
                    (dict(out=torch.empty(4, 6, device="cuda:0", dtype=torch.bfloat16)), "types"), (dict(weight=w.cpu()), "must be on"),
                    (dict(x=x.t().contiguous().t()), "contiguous")):
        a = dict(x=x, weight=w, weight_scale=ws)
        a.update(kw)
        with pytest.raises(ValueError, match=msg):
            ops.linear_quantized(a.pop("x"), a.pop("weight"), a.pop("weight_scale"), **a)
    with pytest.raises(slib.SuaveHipError, match="131072"):
        big = torch.zeros(1, 131073, device="cuda:0")
        ops.linear_quantized(big, torch.zeros((1, 131088), dtype=torch.int8, device="cuda:0")[:, :131073], ws[:1])
    with pytest.raises(slib.SuaveHipError, match="GPU"):
        ops.quantize_rows(x.cpu())


def test_other_stream_and_captured_graph():
    import torch
    from suave_amd import operators as ops

    g = torch.Generator(device="cuda:0").manual_seed(5)
    w, ws = ops.quantize_rows(torch.randn((300, 200), generator=g, device="cuda:0"))
    for m in (3, 50, 90):
        x = torch.randn((m, 200), generator=g, device="cuda:0")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = ops.linear_quantized(x, w, ws)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, ops.linear_quantized(x, w, ws))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear_quantized(x, w, ws)
        for _ in range(3):
            x.copy_(torch.randn((m, 200), generator=g, device="cuda:0"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.linear_quantized(x, w, ws))


def test_many_rows_against_torch_on_the_device():
    """Scales and integers as torch gives them on the device (amax / 127.0, the quotient decided in 64 bits), over enough rows that
    quotients fall next to half-integers."""
    import torch
    from suave_amd import operators as ops

    g = torch.Generator(device="cuda:0").manual_seed(11)
    for dt in (torch.float32, torch.bfloat16):
        x = torch.randn((3000, 1000), generator=g, device="cuda:0").to(dt)
        q, s = ops.quantize_rows(x)
        ts = x.float().abs().amax(dim=1) / 127.0
        assert torch.equal(s, ts)
        assert torch.equal(q.double(), torch.round(x.double() / ts.double()[:, None]))
    # the same rows a few at a time, where the product quantises them itself
    x = torch.randn((16, 250), generator=g, device="cuda:0")
    one = torch.eye(250, device="cuda:0").mul(127).to(torch.int8)
    w = torch.zeros((250, 256), dtype=torch.int8, device="cuda:0")
    w[:, :250] = one
    ts = x.abs().amax(dim=1) / 127.0
    got = ops.linear_quantized(x, w[:, :250], torch.ones(250, device="cuda:0"))
    assert torch.equal(got, torch.round(x.double() / ts.double()[:, None]).float() * 127 * ts[:, None])
