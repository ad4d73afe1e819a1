"""The many-class head, the orthogonalised update and the 8-bit head as the engine and the model use them, one after the
other: ``supervised.ManyClassHead`` (suave_linear_ce), ``Engine.muon_step`` (suave_muon_step beside suave_adam_step),
``supervised.QuantizedHead`` (suave_quantize_rows, suave_linear_quantized).

Tolerances: gradients of the head against autograd in float64 at 2^-18 of their largest entry (D <= 64 products of
binary32 grade, 2^-22 each, and exp of logits below 20: 2^-23 * 21 relative); the orthogonalised update's own bound
(tests/test_hip_ortho.py); 8-bit logits against the exact integers in float64: three binary32 roundings."""

import math

import numpy as np
import pytest

from tests.test_hip_head import _engine, _head
from tests.test_hip_ortho import _exact, _tolerance

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -18


def _table(cols, n, dev):
    from suave_amd.engine import PackedTable
    from tests.helpers import synth_packed

    return PackedTable(*synth_packed(cols, n, 0.1, seed=4), dev)


def _reference(clf, latent, y, keep=None, scale=1.0):
    """(loss, dweight, dbias, dlatent) by autograd in float64."""
    import torch
    from torch.nn import functional as F

    x = latent.double().requires_grad_(True)
    w, b = clf.linear.weight.detach().double().requires_grad_(True), clf.linear.bias.detach().double().requires_grad_(True)
    cw = clf.class_weight.double() if clf._use_weight else None
    loss = F.cross_entropy((x if keep is None else x * keep.double()) @ w.t() + b, y, weight=cw)
    (loss * scale).backward()
    return loss.detach(), w.grad, b.grad, x.grad


def _near(got, want, tol=TOL):
    return float((got.double() - want).abs().max()) <= tol * float(want.abs().max()) + 1e-12


@pytest.mark.parametrize("C,D,dropout,weighted,n", [(2, 5, 0.0, False, 3), (65, 32, 0.0, True, 700), (1000, 32, 0.25, True, 300),
                                                    (257, 64, 0.1, False, 1)])
def test_many_class_head_matches_autograd(C, D, dropout, weighted, n):
    import torch
    from suave_amd import supervised as sup

    clf = _head(C, D, dropout, weighted)
    before = clf.linear.weight.detach().clone()
    head = sup.ManyClassHead(clf)
    assert torch.equal(clf.linear.weight, before) and clf.linear.weight.data_ptr() == head.flat.data_ptr()
    g = torch.Generator(device="cuda:0").manual_seed(5)
    latent = torch.randn((n, D), device="cuda:0", generator=g)
    y = torch.randint(0, C, (n,), device="cuda:0", generator=g)
    rows, key = torch.arange(40, 40 + n, device="cuda:0"), 77
    keep = None
    if dropout:
        drop = sup.RowKeyedDropout(dropout)
        drop.ctx = (rows, key)
        keep = drop(torch.ones_like(latent))
    clf.eval()
    got = head.loss(latent, y, loss_scale=0.7, rows=rows, key=key)
    loss, dw, db, dx = _reference(clf, latent, y, keep, 0.7)
    assert _near(got["loss"], loss) and _near(got["dlatent"], dx)
    assert _near(head._dw, dw) and _near(head._db, db)
    assert not clf.training and (clf._final_dropout is None or (not clf._final_dropout.training and clf._final_dropout.ctx is None))
    plain = head.loss(latent, y, training=False)
    assert set(plain) == {"loss", "row_loss"} and _near(plain["loss"], _reference(clf, latent, y)[0])


def test_heads_with_hidden_layers_are_refused():
    import torch
    from suave_amd import supervised as sup

    with pytest.raises(ValueError, match="hidden"):
        sup.ManyClassHead(sup.ClassificationHead(8, 5, hidden_dims=(4,)).to("cuda:0"))
    with pytest.raises(ValueError, match="GPU"):
        sup.ManyClassHead(sup.ClassificationHead(8, 5))
    with pytest.raises(Exception, match="GPU"):
        sup.QuantizedHead(sup.ClassificationHead(8, 5))


def test_sizes_the_classes_state():
    import torch
    from suave_amd import supervised as sup

    with torch.device("meta"):
        big = sup.ClassificationHead(1 << 15, 1 << 15)
    big.linear.weight = torch.nn.Parameter(torch.empty(1, device="cuda:0").expand(1 << 15, 1 << 15), requires_grad=False)
    with pytest.raises(ValueError, match="2\\^30"):
        sup.ManyClassHead(big)
    # more rows than one call serves: the same as in two
    clf = _head(3, 4, 0.0, False)
    q = sup.QuantizedHead(clf)
    x = torch.randn((1 << 20) + 5, 4, device="cuda:0")
    a = q(x)
    assert torch.equal(a[:1 << 20], q(x[:1 << 20])) and torch.equal(a[1 << 20:], q(x[1 << 20:]))


@pytest.mark.parametrize("frozen", [(), ("decoder",), ("encoder", "decoder", "prior")])
def test_engine_muon_step(frozen):
    import torch

    cols, om, eng = _engine(D=32)
    twin = _engine(D=32)[2]
    mats = eng.hidden_matrices()
    assert sorted(mats) == [f"{s}.backbone.{i}.weight" for s in ("decoder", "encoder") for i in (0, 2)]
    lr = {k: 0.0 if k in frozen else v for k, v in (("encoder", 0.02), ("decoder", 0.01), ("prior", 0.02))}
    adam = {k: 0.0 if k in frozen else v for k, v in (("encoder", 1e-3), ("decoder", 5e-4), ("prior", 1e-3))}
    view = lambda t, m: t.as_strided((m[1], m[2]), (m[3], 1), m[0])  # noqa: E731
    inside = torch.zeros_like(eng.params, dtype=torch.bool)
    for o, r, _, ld in mats.values():
        inside[o:o + r * ld] = True
    g = torch.Generator(device="cuda:0").manual_seed(3)
    for step in range(2):
        eng.grads.copy_(torch.randn(eng.grads.shape, device="cuda:0", generator=g) * 1e-3)
        twin.grads.copy_(eng.grads)
        p0, m0 = eng.params.double(), eng.exp_avg.double()
        eng.muon_step(lr, adam_lr=adam)
        twin.adam_step(adam)
        for name in ("params", "exp_avg", "exp_avg_sq"):  # everything else is adam_step's
            a, b = getattr(eng, name), getattr(twin, name)
            assert torch.equal(a[~inside], b[~inside]), name
        assert float(eng.exp_avg_sq[inside].abs().max()) == 0.0
        for name, m in mats.items():
            group = name.split(".")[0]
            p, q = view(eng.params, m).double(), view(p0, m)
            if group in frozen:
                assert torch.equal(p, q) and float(view(eng.exp_avg, m).abs().max()) == 0.0
                continue
            gr = view(eng.grads, m).double()
            m1 = 0.95 * view(m0, m) + gr
            u = (gr + 0.95 * m1).float()
            o = _exact(u)
            s = lr[group] * math.sqrt(max(1.0, m[1] / m[2]))
            want = q - s * o
            # the update's bound, its input's rounding (once more that size), the result's
            tol = s * 2 * _tolerance(u, o) + 2.0 ** -23 * float(torch.linalg.matrix_norm(want))
            assert float(torch.linalg.matrix_norm(p - want)) <= tol
        pads = inside.clone()
        for m in mats.values():
            view(pads, m).fill_(False)
        assert torch.equal(eng.params[pads].double(), p0[pads])
    assert eng.adam_t == twin.adam_t == 2


def test_train_update_and_serve():
    """Two steps of a joint training step with 500 classes -- ELBO forward, head loss on its latent, ELBO backward with the
    head's gradient, Muon on the hidden layers, Adam on the rest -- then the 8-bit logits of what was trained."""

    import torch
    from suave_amd import supervised as sup

    C, D, N, B = 500, 32, 900, 333
    cols, om, eng = _engine(D=D)
    table = _table(cols, N, eng.device)
    clf = _head(C, D, 0.0, True)
    head = sup.ManyClassHead(clf)
    g = torch.Generator(device="cuda:0").manual_seed(9)
    y = torch.randint(0, C, (N,), device="cuda:0", generator=g)
    mats = eng.hidden_matrices()
    view = lambda t, m: t.as_strided((m[1], m[2]), (m[3], 1), m[0])  # noqa: E731
    for step in range(2):
        kw = dict(beta_scale=1.3, tau=1.0, seed=3, step=step)
        latent = eng.elbo(table, 10 * step, B, grad=False, training=True, want=("latent",), **kw)["latent"]
        t = y[10 * step:10 * step + B]
        loss, dw, db, dx = _reference(clf, latent, t)
        w0 = head.flat.clone()
        got = head.step(eng, latent, t, 1e-2)
        assert _near(got["loss"], loss) and _near(got["dlatent"], dx) and _near(head._dw, dw) and _near(head._db, db)
        # Adam's own formula in binary32 on the gradient the kernel gave
        ref = _engine(D=D)[2]
        p, m, v = (w0.clone(), torch.zeros_like(w0), torch.zeros_like(w0)) if step == 0 else (w0.clone(), keep_m, keep_v)
        ref.adam_flat(p, head.grads, m, v, step + 1, 1e-2)
        assert torch.equal(p, head.flat) and torch.equal(clf.linear.weight.reshape(-1), head.flat[:C * D])
        keep_m, keep_v = m, v
        eng.elbo(table, 10 * step, B, training=True, dlatent=got["dlatent"].contiguous(), **kw)
        p0, m0 = eng.params.double(), eng.exp_avg.double()
        eng.muon_step(0.02, adam_lr=1e-3)
        for m_ in mats.values():
            gr = view(eng.grads, m_).double()
            u = (gr + 0.95 * (0.95 * view(m0, m_) + gr)).float()
            o = _exact(u)
            s = 0.02 * math.sqrt(max(1.0, m_[1] / m_[2]))
            want = view(p0, m_) - s * o
            tol = s * 2 * _tolerance(u, o) + 2.0 ** -23 * float(torch.linalg.matrix_norm(want))
            assert float(torch.linalg.matrix_norm(view(eng.params, m_).double() - want)) <= tol
    post = eng.encode(table, 0, N)["mean"]
    served = head.quantized()
    logits = served(post)
    w, x = clf.linear.weight.detach(), post
    sw, sx = w.abs().amax(1) / 127.0, x.abs().amax(1) / 127.0
    q = lambda a, s: torch.round(a.double() / torch.where(s == 0, torch.ones_like(s), s).double()[:, None])  # noqa: E731
    want = (q(x, sx) @ q(w, sw).t()) * sx.double()[:, None] * sw.double()[None] + clf.linear.bias.detach().double()
    assert float((logits.double() - want).abs().max()) <= 3 * 2.0 ** -24 * float((want.abs() + clf.linear.bias.detach().abs().max()).max())
    # and against the head itself: half a step of either scale per product
    full = x.double() @ w.double().t() + clf.linear.bias.double()
    bound = (x.double().abs().sum(1)[:, None] * sw.double()[None] / 2 + w.double().abs().sum(1)[None] * sx.double()[:, None] / 2
             + D * sx.double()[:, None] * sw.double()[None] / 4)
    assert bool(((logits.double() - full).abs() <= bound * (1 + 1e-6) + 1e-6).all())
    snapshot = logits.clone()
    head.flat.mul_(2.0)  # the serving form is a snapshot
    assert torch.equal(served(post), snapshot)


def test_operators_in_two_graphs_share_nothing():
    """Loss, update and serving captured together, twice, replayed in turn with eager work between: every replay is the
    eager result."""

    import torch
    from suave_amd import operators as ops

    g = torch.Generator(device="cuda:0").manual_seed(1)

    def state(n, c, d, h):
        r = lambda *s: torch.randn(s, device="cuda:0", generator=g)  # noqa: E731
        return dict(x=r(n, d), w1=r(h, d) / d, m=torch.zeros(h, d, device="cuda:0"), w=r(c, h) / 8,
                    y=torch.randint(0, c, (n,), device="cuda:0", generator=g, dtype=torch.int32))

    def run(s):
        a = ops.linear_cross_entropy(s["h"], s["w"], s["y"])
        g1 = a["dweight"].t().contiguous()[:, :s["w1"].shape[1]].contiguous()  # any gradient of w1's shape
        ops.muon_step([s["w1"]], [g1], [s["m"]], lr=0.02)
        q, sc = ops.quantize_rows(s["w"])
        return a["loss"], a["dx"], s["w1"].clone(), ops.linear_quantized(s["h"], q, sc)

    states, graphs = [], []
    for n, c, d, h in ((200, 300, 40, 70), (1100, 200, 20, 33)):
        s = state(n, c, d, h)
        s["h"] = torch.relu(s["x"] @ s["w1"].t())
        start = {k: s[k].clone() for k in ("w1", "m")}
        run(s)
        torch.cuda.synchronize()
        for k, v in start.items():
            s[k].copy_(v)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(s)
        states.append((s, {k: v.clone() for k, v in s.items()}, out))
        graphs.append(graph)
    for turn in range(3):
        for (s, eager, out), graph in zip(states, graphs):
            h = torch.relu(torch.randn(s["h"].shape, device="cuda:0", generator=g))
            s["h"].copy_(h)
            eager["h"].copy_(h)
            want = run(eager)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), turn


def test_backward_in_a_graph_while_an_eager_graph_lives():
    """The operators keep no autograd graph: a captured call on leaves that an eager graph still holds is ordinary work."""

    import torch
    from suave_amd import supervised as sup

    clf = _head(300, 16, 0.0, False)
    head = sup.ManyClassHead(clf)
    latent = torch.randn(64, 16, device="cuda:0").requires_grad_(True)
    y = torch.randint(0, 300, (64,), device="cuda:0", dtype=torch.int32)
    eager = clf.loss(clf(latent), y.long())  # alive during the capture
    head.loss(latent, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = head.loss(latent, y)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        loss, dw, db, dx = _reference(clf, latent.detach(), y.long())
        assert _near(out["loss"], loss) and _near(out["dlatent"], dx) and _near(head._dw, dw)
    eager.backward()
    assert _near(latent.grad, dx, 1e-5)


def test_model_serves_quantized_logits_on_request():
    import pandas as pd
    import torch
    from suave_amd.model import SUAVE
    from suave_amd.types import Schema

    rng = np.random.default_rng(0)
    n = 400
    df = pd.DataFrame({"a": rng.normal(size=n), "b": rng.normal(size=n), "c": rng.integers(0, 3, n)})
    y = rng.integers(0, 70, n)
    schema = Schema({"a": {"type": "real"}, "b": {"type": "real"}, "c": {"type": "cat", "n_classes": 3}})
    m = SUAVE(schema, behaviour="supervised", latent_dim=8, n_components=2, hidden_dims=(32, 16), random_state=0)
    with pytest.raises(RuntimeError):
        m.quantize_classifier()
    kw = dict(warmup_epochs=1, kl_warmup_epochs=1, head_epochs=1, finetune_epochs=1, decoder_refine_epochs=1)
    m.fit(df, y=y, **kw)
    before = m._compute_logits(df)
    proba = m.predict_proba(df)
    m.quantize_classifier()
    served = m._compute_logits(df)
    clf = m._classifier
    post = m._posterior_mean(m._table(df)).double()
    w = clf.linear.weight.detach().double()
    sw, sx = w.abs().amax(1) / 127, post.abs().amax(1) / 127
    bound = post.abs().sum(1)[:, None] * sw / 2 + w.abs().sum(1) * sx[:, None] / 2 + 8 * sx[:, None] * sw / 4
    full = post @ w.t() + clf.linear.bias.detach().double()
    assert not np.array_equal(served, before)
    assert bool(((torch.from_numpy(served).to(full).double() - full).abs() <= bound * (1 + 1e-6) + 1e-5).all())
    assert m.predict_proba(df).shape == proba.shape
    m.quantize_classifier(False)
    assert np.array_equal(m._compute_logits(df), before) and np.array_equal(m.predict_proba(df), proba)
    m.quantize_classifier().fit(df, y=y, **kw)  # a new fit serves its own head, unquantised
    assert np.array_equal(m._compute_logits(df), before)
