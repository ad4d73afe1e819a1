"""suave_linear_ce (suave_amd.operators.linear_cross_entropy) against the definition in float64.

Tolerances, in units of the type's half step u = finfo.eps / 2 (fp32 2^-24, bf16 2^-8):

* logits: fp32 operands enter as two fp16 planes, each product is off by at most 3 * 2^-24 of |x||w|, and K products are
  added in fp32: |error of l| <= (3 + K / 16) 2^-24 sum_k |x_k w_k| + 2^-24 |l| -- taken as LOGIT = 2^-20 * max_i |x_i| |W_c|
  (K <= 2048; sums of random sign stay far below).  bf16 operands multiply exactly: the same bound covers the additions.
* lse: an error of the logits moves it by at most itself.  exp of a binary32 argument a has a relative error of at most
  (|a| + 1) 2^-23 (rounding of a log2 e, hardware exp2), and the terms' errors enter the sum weighted by their share p: sum p |a| <= log C;
  two such exponentials (within a strip, between strips) and the logarithm: 2^-23 (log C + 3).  The result itself is
  rounded twice (M + log S, M): 2^-23 |lse|.  So LSE = 2 LOGIT + 2^-23 (log C + 3 + |lse|), and a row loss, the difference
  of lse and a logit, is off by at most w (LSE + LOGIT + 2^-23 |l|) + 2^-24 |row loss|.
* G: p = exp(l - lse) has a relative error of 4 LOGIT + 2^-22; bf16 rounds it once more (2^-8).
* gradients: the bound of G times sum |G| |W| (dx), sum |G| |x| (dW), sum |G| (db), plus the rounding of the result.
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _case(n, c, d, dtype, weighted, seed, drop=0.1, spread=2.0):
    import torch

    g = torch.Generator(device="cuda:0").manual_seed(seed)
    x = torch.randn((n, d), generator=g, device="cuda:0")
    w = torch.randn((c, d), generator=g, device="cuda:0") * (spread / math.sqrt(d))
    b = torch.randn(c, generator=g, device="cuda:0") * 0.3
    y = torch.randint(0, c, (n,), generator=g, device="cuda:0", dtype=torch.int32)
    if drop and n > 1:
        y = torch.where(torch.rand(n, generator=g, device="cuda:0") < drop, torch.full_like(y, -1), y)
        y[0] = c - 1
    cw = torch.rand(c, generator=g, device="cuda:0") + 0.25 if weighted else None
    return x.to(dtype), w.to(dtype), b, y, cw


def _reference(x, w, b, y, cw, weight_sum=None, scale=1.0):
    """(loss, row_loss, lse, dx, dW, db, |G|W, |G|x, |G|) in float64 on the CPU's float64 units of the device."""
    import torch

    xd, wd = x.double(), w.double()
    live = y >= 0
    xd = torch.where(live[:, None], xd, torch.zeros_like(xd))
    l = xd @ wd.t() + (0.0 if b is None else b.double())
    lse = torch.logsumexp(l, dim=1)
    yi = y.clamp_min(0).long()
    wt = (torch.ones_like(lse) if cw is None else cw.double()[yi]) * live
    per = torch.where(wt != 0, wt * (lse - l.gather(1, yi[:, None])[:, 0]), torch.zeros_like(lse))
    total = wt.sum() if weight_sum is None else weight_sum.double().reshape(())
    f = torch.zeros_like(wt) if float(total) == 0 else scale * wt / total
    p = torch.exp(l - lse[:, None])
    G = p.clone()
    G[torch.arange(len(y), device=y.device), yi] -= 1.0
    G = torch.where(f[:, None] != 0, G * f[:, None], torch.zeros_like(G))
    # what an entry of G may be off by, relative: the target's entry has the absolute error of p
    mag = torch.where(f[:, None] != 0, (G.abs() + p * f.abs()[:, None]), torch.zeros_like(G))
    loss = per.sum() / total if float(total) != 0 else torch.zeros_like(total)
    return dict(loss=loss, row_loss=per, lse=lse, dx=G @ wd, dweight=G.t() @ xd, dbias=G.sum(0),
                mdx=mag @ wd.abs(), mdw=mag.t() @ xd.abs(), mdb=mag.sum(0), l=l)


def _lse_error(logit, c, lse):
    return 2 * logit + 2.0 ** -23 * (math.log(c) + 3 + float(lse[lse.isfinite()].abs().max()))


def _check(got, ref, x, w, y, grad=True):
    import torch

    bf = x.dtype == torch.bfloat16
    live = y >= 0
    xn = x.double()[live].norm(dim=1).max() if bool(live.any()) else torch.zeros((), device=x.device, dtype=torch.float64)
    logit = 2.0 ** -20 * float(xn * w.double().norm(dim=1).max()) + 2.0 ** -23 * float(ref["l"][torch.isfinite(ref["l"])].abs().max())
    u = torch.finfo(x.dtype).eps / 2
    wmax = float((ref["row_loss"].abs() / (ref["lse"].abs() + 1)).max()) + 1.5
    err = _lse_error(logit, w.shape[0], ref["lse"])
    assert float((got["lse"].double() - ref["lse"]).abs().max()) <= err
    assert float((got["row_loss"].double() - ref["row_loss"]).abs().max()) <= 2 * err * wmax
    assert bool((got["row_loss"][~live] == 0).all())
    assert abs(float(got["loss"]) - float(ref["loss"])) <= 2 * err + 2.0 ** -23 * abs(float(ref["loss"]))
    if not grad:
        return
    eg = 4 * logit + 2.0 ** -21 + (2.0 ** -8 if bf else 0.0)
    for name, mag, round_ in (("dx", "mdx", u), ("dweight", "mdw", u), ("dbias", "mdb", 2.0 ** -24)):
        e = (got[name].double() - ref[name]).abs()
        lim = (4 * logit + 2.0 ** -21 if name == "dbias" else eg) * ref[mag] + round_ * ref[name].abs() * 1.01 + 1e-30
        # sums in fp32 and the planes' cross terms: 2^-20 of the largest magnitude
        lim = lim + 2.0 ** -20 * ref[mag].max() + (1e-38 if not bf else 1e-37)
        assert bool((e <= lim).all()), (name, float((e / lim).max()))
    assert bool((got["dx"][~live] == 0).all())


SHAPES = [(1, 1, 1), (1, 2, 3), (3, 65, 7), (16, 100, 32), (17, 129, 8), (64, 1000, 40), (65, 257, 64), (255, 100, 33), (300, 513, 130),
          (1000, 70, 500), (129, 5003, 96), (2, 20000, 17), (513, 1030, 256)]


@pytest.mark.parametrize("n,c,d", SHAPES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_loss_and_gradients_match_the_definition(n, c, d, dtype):
    import torch
    from suave_amd import operators as ops

    dt = getattr(torch, dtype)
    weighted = (n + c + d) % 2 == 0
    x, w, b, y, cw = _case(n, c, d, dt, weighted, seed=n * 7 + c * 3 + d)
    got = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw, loss_scale=0.75)
    ref = _reference(x, w, b, y, cw, scale=0.75)
    _check(got, ref, x, w, y)
    # the loss alone gives the same loss, and a second call the same bits
    only = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw, grad=False)
    assert torch.equal(only["row_loss"], got["row_loss"]) and "dx" not in only
    again = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw, loss_scale=0.75)
    assert all(torch.equal(again[k], got[k]) for k in got)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_several_pieces_of_the_classes(dtype):
    """A batch whose logit gradient does not fit one piece (n * C * bytes > 192 MiB)."""
    import torch
    from suave_amd import operators as ops

    dt = getattr(torch, dtype)
    n, c, d = (6000, 9001, 72) if dtype == "float32" else (6000, 17001, 72)
    x, w, b, y, cw = _case(n, c, d, dt, True, seed=5)
    assert n * c * (4 if dtype == "float32" else 2) > (192 << 20)
    _check(ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw), _reference(x, w, b, y, cw), x, w, y)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_operands_and_results(dtype):
    """Row strides beyond the row, addresses off 16 bytes, and nothing written outside the rows of the results."""
    import torch
    from suave_amd import operators as ops

    dt = getattr(torch, dtype)
    n, c, d = 70, 300, 48
    x, w, b, y, cw = _case(n, c, d, dt, True, seed=9)
    xs = torch.full((n, d + 13), float("nan"), dtype=dt, device="cuda:0")
    xs[:, 5:5 + d] = x
    for off, extra in ((0, 16), (1, 8), (3, 5)):
        wsb = torch.full((c, d + extra), float("nan"), dtype=dt, device="cuda:0")
        wsb[:, off:off + d] = w
        dxb = torch.full((n, d + 7), 3.0, dtype=dt, device="cuda:0")
        dwb = torch.full((c, d + 9), 3.0, dtype=dt, device="cuda:0")
        got = ops.linear_cross_entropy(xs[:, 5:5 + d], wsb[:, off:off + d], y, bias=b, class_weight=cw, dx=dxb[:, 2:2 + d],
                                       dweight=dwb[:, 4:4 + d])
        _check(got, _reference(x, w, b, y, cw), x, w, y)
        assert bool((dxb[:, :2] == 3).all()) and bool((dxb[:, 2 + d:] == 3).all())
        assert bool((dwb[:, :4] == 3).all()) and bool((dwb[:, 4 + d:] == 3).all())


def test_rows_left_out_do_not_matter_whatever_they_hold():
    import torch
    from suave_amd import operators as ops

    for dt in (torch.float32, torch.bfloat16):
        x, w, b, y, cw = _case(200, 700, 64, dt, True, seed=3)
        y[5], y[100:140] = -1, -100
        bad = x.clone()
        bad[5], bad[100:120], bad[120:140] = float("nan"), float("inf"), -float("inf")
        got, want = ops.linear_cross_entropy(bad, w, y, bias=b, class_weight=cw), ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
        for k in ("loss", "row_loss", "dx", "dweight", "dbias"):
            assert torch.equal(got[k], want[k]), k
        none = ops.linear_cross_entropy(bad, w, torch.full_like(y, -1), bias=b, class_weight=cw)
        assert float(none["loss"]) == 0 and all(bool((none[k] == 0).all()) for k in ("row_loss", "dx", "dweight", "dbias"))
        # rows whose class weighs nothing
        zero = cw.clone()
        zero[y[y >= 0].long()] = 0.0
        none = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=zero)
        assert float(none["loss"]) == 0 and all(bool((none[k] == 0).all()) for k in ("row_loss", "dx", "dweight", "dbias"))


def test_target_beyond_the_classes_is_loud():
    import torch
    from suave_amd import operators as ops

    x, w, b, y, cw = _case(40, 90, 16, torch.float32, True, seed=2)
    y[7] = 90
    got = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
    assert math.isnan(float(got["loss"])) and math.isnan(float(got["row_loss"][7])) and bool(torch.isfinite(got["row_loss"][:7]).all())
    assert bool(torch.isnan(got["dweight"]).all()) and bool(torch.isnan(got["dbias"]).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_classes_that_are_never_predicted(dtype):
    """bias = -inf, whole 64-class strips of it included; a target among them has an infinite loss, all of them NaN."""
    import torch
    from suave_amd import operators as ops

    dt = getattr(torch, dtype)
    x, w, b, y, _ = _case(50, 400, 24, dt, False, seed=4, drop=0)
    b[64:320] = -float("inf")
    y = torch.where((y >= 64) & (y < 320), torch.full_like(y, 10), y)
    got = ops.linear_cross_entropy(x, w, y, bias=b)
    keep = torch.tensor([i for i in range(400) if not 64 <= i < 320], device="cuda:0")
    small = ops.linear_cross_entropy(x, w[keep].contiguous(), torch.where(y >= 320, y - 256, y), bias=b[keep].contiguous())
    ref = _reference(x, w[keep], b[keep], torch.where(y >= 320, y - 256, y), None)
    _check(small, ref, x, w[keep], y)
    full = dict(got, dweight=got["dweight"][keep], dbias=got["dbias"][keep])
    _check(full, ref, x, w[keep], y)
    assert bool((got["dweight"][64:320] == 0).all()) and bool((got["dbias"][64:320] == 0).all())
    y[3] = 100
    hit = ops.linear_cross_entropy(x, w, y, bias=b)
    assert math.isinf(float(hit["row_loss"][3])) and float(hit["row_loss"][3]) > 0 and math.isinf(float(hit["loss"]))
    assert bool(torch.isfinite(hit["dx"]).all())
    gone = ops.linear_cross_entropy(x, w, y, bias=torch.full_like(b, -float("inf")))
    assert math.isnan(float(gone["loss"])) or math.isinf(float(gone["loss"]))


def test_large_and_small_scales():
    """fp32 operands far outside fp16's range, logits up to +-1e4 and down to 1e-8."""
    import torch
    from suave_amd import operators as ops

    for sx, sw in ((1e6, 1e-6), (1e-9, 3e8), (1e-20, 1e-20), (30.0, 100.0)):
        x, w, b, y, cw = _case(130, 200, 65, torch.float32, True, seed=6, spread=1.0)
        x, w = x * sx, w * sw
        got, ref = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw), _reference(x, w, b, y, cw)
        logit = 2.0 ** -20 * float(x.double().norm(dim=1).max() * w.double().norm(dim=1).max()) + 2.0 ** -23 * float(ref["l"].abs().max())
        assert float((got["lse"].double() - ref["lse"]).abs().max()) <= _lse_error(logit, 200, ref["lse"])
        for k in ("dx", "dweight"):
            m = ref["mdx" if k == "dx" else "mdw"].max()
            assert float((got[k].double() - ref[k]).abs().max()) <= float(m) * (4 * logit + 2.0 ** -19), k


def test_weight_sum_loss_sum_and_accumulation():
    import torch
    from suave_amd import operators as ops

    x, w, b, y, cw = _case(90, 150, 20, torch.float32, True, seed=8)
    ws = torch.tensor([321.0], device="cuda:0")
    acc = torch.full((1,), 5.0, dtype=torch.float64, device="cuda:0")
    got = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw, weight_sum=ws, loss_sum=acc, loss_rows=90.0)
    _check(got, _reference(x, w, b, y, cw, weight_sum=ws), x, w, y)
    assert abs(float(acc) - 5.0 - 90.0 * float(got["loss"])) <= 1e-5 * abs(float(acc))
    # two shards of the batch with the whole batch's weight sum add up to the whole batch
    total = cw[y.clamp_min(0).long()].where(y >= 0, torch.zeros_like(cw[:1])).sum().reshape(1)
    whole = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
    parts = [ops.linear_cross_entropy(x[a:e].contiguous(), w, y[a:e].contiguous(), bias=b, class_weight=cw, weight_sum=total) for a, e in ((0, 31), (31, 90))]
    for k in ("dweight", "dbias"):
        s = parts[0][k] + parts[1][k]
        assert float((s - whole[k]).abs().max()) <= 2.0 ** -19 * float(whole[k].abs().max())


def test_gradient_matches_differences():
    """Central differences of the float64 definition at the kernel's gradient, along random directions."""
    import torch
    from suave_amd import operators as ops

    x, w, b, y, cw = _case(40, 130, 24, torch.float32, True, seed=11)
    got = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
    g = torch.Generator(device="cuda:0").manual_seed(1)
    h = 1e-4
    for name, t in (("dx", x), ("dweight", w), ("dbias", b)):
        v = torch.randn(t.shape, generator=g, device="cuda:0").double()
        args = {"dx": x.double(), "dweight": w.double(), "dbias": b.double()}
        f = []
        for s in (h, -h):
            a = dict(args)
            a[name] = args[name] + s * v
            f.append(float(_reference(a["dx"], a["dweight"], a["dbias"], y, cw)["loss"]))
        want = (f[0] - f[1]) / (2 * h)
        have = float((got[name].double() * v).sum())
        # third derivatives of the loss along v times h^2 / 6, and the gradient's own error
        assert abs(have - want) <= 2e-6 * float(v.norm()) ** 3 * 0.02 + 1e-5 * float((got[name].double() * v).abs().sum()), name


def test_empty_batch_and_refusals():
    import torch
    from suave_amd import lib as slib
    from suave_amd import operators as ops

    x, w, b, y, _ = _case(8, 70, 12, torch.float32, False, seed=1)
    got = ops.linear_cross_entropy(x[:0], w, y[:0], bias=b)
    assert float(got["loss"]) == 0 and bool((got["dweight"] == 0).all()) and bool((got["dbias"] == 0).all()) and got["dx"].shape == (0, 12)
    for kw, msg in ((dict(targets=y.long()), "int32"), (dict(weight=w.bfloat16()), "types"), (dict(weight=w[:, :5]), "columns"),
                    (dict(x=x.t()), "columns|contiguous"), (dict(bias=b[:5]), "vector"), (dict(targets=y[:3]), "vector"),
                    (dict(x=x.half(), weight=w.half()), "types"), (dict(dx=torch.empty(8, 11, device="cuda:0")), "shape"),
                    (dict(weight=w.cpu()), "must be on")):
        a = dict(x=x, weight=w, targets=y)
        a.update(kw)
        with pytest.raises(ValueError, match=msg):
            ops.linear_cross_entropy(a.pop("x"), a.pop("weight"), a.pop("targets"), **a)
    with pytest.raises(slib.SuaveHipError, match="GPU"):
        ops.linear_cross_entropy(x.cpu(), w, y)


def test_other_stream_and_captured_graph():
    """The call runs on the current stream and replays from a captured graph: new inputs in the same buffers, eager work
    and synchronisations in between."""
    import torch
    from suave_amd import operators as ops

    x, w, b, y, cw = _case(300, 500, 40, torch.float32, True, seed=12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
    torch.cuda.current_stream().wait_stream(side)
    eager = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
    assert all(torch.equal(on_side[k], eager[k]) for k in eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
    for seed in (21, 22, 23):
        x2, w2, b2, y2, cw2 = _case(300, 500, 40, torch.float32, True, seed=seed)
        for dst, src in ((x, x2), (w, w2), (b, b2), (y, y2), (cw, cw2)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw)
        assert all(torch.equal(out[k], eager[k]) for k in eager)


# float32 from 256 columns on, and few classes: other paths through the kernels than the sizes above
@pytest.mark.parametrize("n,c,d", [(1, 300, 256), (33, 257, 300), (700, 1111, 261), (95, 5001, 512), (1100, 200, 40), (1025, 256, 256),
                                   (2049, 3, 20), (1024, 256, 8)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_wide_rows_and_few_classes(n, c, d, dtype):
    import torch
    from suave_amd import operators as ops

    dt = getattr(torch, dtype)
    x, w, b, y, cw = _case(n, c, d, dt, c % 2 == 1, seed=n + c + d)
    got = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw, loss_scale=1.5)
    _check(got, _reference(x, w, b, y, cw, scale=1.5), x, w, y)
    again = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw, loss_scale=1.5)
    assert all(torch.equal(again[k], got[k]) for k in got)
    only = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw, grad=False)
    assert torch.equal(only["row_loss"], got["row_loss"]) and torch.equal(only["loss"], got["loss"])


@pytest.mark.parametrize("c,d", [(400, 256), (250, 24), (700, 300)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_masked_classes_and_rows_on_every_path(c, d, dtype):
    """Strips of 64 classes at -inf or at the type's lowest value, a target among the former, rows left out that hold NaN."""
    import torch
    from suave_amd import operators as ops

    dt = getattr(torch, dtype)
    for low in (-float("inf"), torch.finfo(torch.float32).min):
        x, w, b, y, _ = _case(50, c, d, dt, False, seed=4, drop=0)
        b[64:192] = low
        y = torch.where((y >= 64) & (y < 192), torch.full_like(y, 10), y)
        y[7] = -1
        keep = torch.tensor([i for i in range(c) if not 64 <= i < 192], device="cuda:0")
        ref = _reference(x, w[keep], b[keep], torch.where(y >= 192, y - 128, y), None)
        bad = x.clone()
        bad[7] = float("nan")
        got = ops.linear_cross_entropy(bad, w, y, bias=b)
        full = dict(got, dweight=got["dweight"][keep], dbias=got["dbias"][keep])
        got["lse"][7] = full["lse"][7] = float(ref["lse"][7])  # not defined for a row that is left out
        _check(full, ref, x, w[keep], y)
        assert bool((got["dweight"][64:192] == 0).all()) and bool((got["dbias"][64:192] == 0).all())
    b[64:192] = -float("inf")
    y[3] = 100
    hit = ops.linear_cross_entropy(x, w, y, bias=b)
    assert math.isinf(float(hit["row_loss"][3])) and float(hit["row_loss"][3]) > 0 and math.isinf(float(hit["loss"]))
    assert bool(torch.isfinite(hit["dx"]).all()) and bool(torch.isfinite(hit["dweight"]).all())
    # the target's entry of G is -1 / rows there: seen in the bias gradient
    assert abs(float(hit["dbias"][100]) + 1.0 / 49) <= 2.0 ** -22


@pytest.mark.parametrize("n,c,d,weighted", [(1, 768, 56, False), (1, 1000, 500, False), (2, 300, 32, False), (8, 2000, 40, False),
                                            (5, 25418, 133, True), (300, 290, 48, True)])
def test_bfloat16_gradients_are_off_by_their_rounding_alone(n, c, d, weighted):
    """Where one entry of G can dominate a row of dweight (few rows, class weights) G has fp16's 2^-11 (half a step): with e the error of the
    unrounded gradient, |e| <= (2^-11 + 4 LOGIT + 2^-20) sum |G| |x|, the result is off by its own rounding + 3 |e|."""
    import torch
    from suave_amd import operators as ops

    x, w, b, y, cw = _case(n, c, d, torch.bfloat16, weighted, seed=n + 3 * c + d, drop=0.0)
    got, ref = ops.linear_cross_entropy(x, w, y, bias=b, class_weight=cw), _reference(x, w, b, y, cw)
    logit = 2.0 ** -20 * float(x.double().norm(dim=1).max() * w.double().norm(dim=1).max()) + 2.0 ** -23 * float(ref["l"].abs().max())
    norm = torch.linalg.matrix_norm
    for name, mag in (("dx", "mdx"), ("dweight", "mdw")):
        e = (2.0 ** -11 + 4 * logit + 2.0 ** -20) * float(norm(ref[mag]))
        assert float(norm(got[name].double() - ref[name])) <= float(norm(ref[name].bfloat16().double() - ref[name])) + 3 * e, name
