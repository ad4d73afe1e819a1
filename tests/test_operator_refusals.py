"""What the operators' entry points refuse before they touch the GPU: the C-ABI's own checks, called without one, and the
sizes of the structures the binding mirrors."""

import ctypes as C

import pytest

from suave_amd import lib as slib
from suave_amd.plan import LinearCeT, LinearQuantizedT, MuonMatrixT, OrthoMatrixT

P = 0x100000  # a pointer no refused call follows


@pytest.fixture(scope="module")
def lib():
    return slib.load()


def _refused(lib, rc, text):
    assert rc != 0
    msg = lib.suave_last_error().decode()
    assert text in msg, msg


def test_structures_match_the_header():
    assert C.sizeof(LinearCeT) == 16 + 8 + 4 * 8 + 4 * 8 + 8 + 4 * 8 + 2 * 16 + 8 + 16
    assert C.sizeof(LinearQuantizedT) == 16 + 8 + 4 * 8 + 4 * 8 + 16
    assert C.sizeof(OrthoMatrixT) == 40 and C.sizeof(MuonMatrixT) == 64


def _ce(**kw):
    h = LinearCeT()
    base = dict(dtype=0, n_classes=100, dim=32, n_rows=7, x=P, ld_x=32, weight=2 * P, ld_weight=32, targets=3 * P, loss_scale=1.0,
                loss_rows=1.0, dx=4 * P, ld_dx=32, dweight=5 * P, ld_dweight=32, dbias=6 * P, workspace=7 * P, workspace_bytes=1 << 40)
    base.update(kw)
    for k, v in base.items():
        setattr(h, k, v)
    return h


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "dtype"), (dict(n_classes=0), "n_classes"), (dict(n_classes=(1 << 24) + 1), "n_classes"), (dict(dim=0), "dim"),
    (dict(dim=32769), "dim"), (dict(n_rows=-1), "n_rows"), (dict(n_rows=(1 << 24) + 1), "n_rows"),
    (dict(n_rows=1 << 20, n_classes=(1 << 18) + 1), "2^38"), (dict(ld_x=31), "stride"), (dict(ld_weight=31), "stride"),
    (dict(ld_x=(1 << 22) + 1), "stride"), (dict(ld_dx=31), "ld_dx"), (dict(ld_dweight=31), "ld_dweight")])
def test_linear_ce_sizes(lib, kw, text):
    n = C.c_size_t(0)
    _refused(lib, lib.suave_linear_ce_workspace_bytes(C.byref(_ce(**kw)), C.byref(n)), text)
    _refused(lib, lib.suave_linear_ce(C.byref(_ce(**kw)), None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(weight=None), "null"), (dict(targets=None), "null"), (dict(x=P + 2), "aligned"),
    (dict(dtype=1, weight=2 * P + 1), "aligned"), (dict(dx=P), "output"), (dict(dweight=2 * P), "output"), (dict(dx=5 * P), "output"),
    (dict(workspace=None), "workspace"), (dict(workspace=7 * P + 128), "workspace"), (dict(workspace_bytes=100), "too small")])
def test_linear_ce_pointers(lib, kw, text):
    _refused(lib, lib.suave_linear_ce(C.byref(_ce(**kw)), None), text)


def test_linear_ce_workspace_depends_on_what_is_asked(lib):
    def size(**kw):
        n = C.c_size_t(0)
        assert lib.suave_linear_ce_workspace_bytes(C.byref(_ce(workspace=None, workspace_bytes=0, **kw)), C.byref(n)) == 0
        return n.value

    full = size()
    assert size(dx=None, dweight=None, dbias=None) < full
    # the statistics of strips of 64 classes and one piece of the gradient, not the logits
    big = dict(n_rows=1 << 16, n_classes=1 << 17, dim=64, ld_x=64, ld_weight=64, ld_dx=64, ld_dweight=64, dtype=1)
    assert size(**big) < 0.2 * 2 * (1 << 33)
    assert size(n_rows=0) > 0
    _refused(lib, lib.suave_linear_ce_workspace_bytes(C.byref(_ce()), None), "null")
    _refused(lib, lib.suave_linear_ce_workspace_bytes(None, C.byref(C.c_size_t(0))), "null")
    _refused(lib, lib.suave_linear_ce(None, None), "null")


def test_quantize_rows(lib):
    def call(x=P, dtype=0, rows=3, cols=20, ld_x=20, q=2 * P, ld_q=32, scale=3 * P):
        return lib.suave_quantize_rows(x, dtype, rows, cols, ld_x, q, ld_q, scale, None)

    for kw, text in ((dict(dtype=7), "dtype"), (dict(rows=-1), "rows"), (dict(rows=(1 << 30) + 1), "rows"), (dict(cols=0), "cols"),
                     (dict(ld_x=19), "ld_x"), (dict(ld_q=31), "ld_q"), (dict(ld_q=16), "ld_q"), (dict(x=None), "null"),
                     (dict(scale=None), "null"), (dict(q=2 * P + 8), "aligned")):
        _refused(lib, call(**kw), text)
    assert call(rows=0, x=None, q=None, scale=None) == 0


def test_linear_quantized(lib):
    def h(**kw):
        s = LinearQuantizedT()
        base = dict(dtype=0, n_out=10, n_in=20, n_rows=3, x=P, ld_x=20, weight=2 * P, ld_weight=32, weight_scale=3 * P, out=4 * P,
                    ld_out=10, workspace=5 * P, workspace_bytes=1 << 40)
        base.update(kw)
        for k, v in base.items():
            setattr(s, k, v)
        return s

    for kw, text in ((dict(dtype=-1), "dtype"), (dict(n_rows=-1), "n_rows"), (dict(n_in=0), "n_in"), (dict(n_in=131073, ld_x=131073), "131072"),
                     (dict(n_out=0), "n_out"), (dict(ld_x=19), "stride"), (dict(ld_out=9), "stride"), (dict(ld_weight=24), "ld_weight"),
                     (dict(ld_weight=16), "ld_weight"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(weight=2 * P + 4), "aligned"),
                     (dict(workspace=5 * P + 1), "workspace"), (dict(workspace_bytes=8), "too small")):
        _refused(lib, lib.suave_linear_quantized(C.byref(h(**kw)), None), text)
    assert lib.suave_linear_quantized(C.byref(h(n_rows=0)), None) == 0
    _refused(lib, lib.suave_linear_quantized(None, None), "null")


def _ortho(*mats):
    arr = (OrthoMatrixT * max(len(mats), 1))()
    for a, kw in zip(arr, mats):
        for k, v in dict(dict(in_=P, out=2 * P, ld_in=8, ld_out=8, rows=5, cols=8), **kw).items():
            setattr(a, k, v)
    return arr


def test_orthogonalize(lib):
    def call(arr, n, dtype=0, steps=5, eps=1e-7, ws=3 * P, nbytes=1 << 40):
        return lib.suave_orthogonalize(arr, n, dtype, steps, eps, ws, nbytes, None)

    for kw, text in ((dict(rows=0), "row"), (dict(cols=0), "column"), (dict(rows=40000, cols=40000, ld_in=40000, ld_out=40000), "32768"),
                     (dict(ld_in=7), "stride"), (dict(ld_out=7), "stride"), (dict(in_=None), "null")):
        _refused(lib, call(_ortho(kw), 1), text)
    one = _ortho({})
    for kw, text in ((dict(dtype=3), "dtype"), (dict(steps=0), "steps"), (dict(steps=17), "steps"), (dict(eps=0.0), "eps"),
                     (dict(eps=float("nan")), "eps"), (dict(ws=None), "workspace"), (dict(ws=3 * P + 64), "workspace"), (dict(nbytes=0), "too small")):
        _refused(lib, call(one, 1, **kw), text)
    for second in (dict(out=2 * P, in_=5 * P), dict(in_=2 * P, out=5 * P), dict(out=P, in_=5 * P)):
        _refused(lib, call(_ortho({}, second), 2), "another matrix")
    assert call(one, 0, ws=None, nbytes=0) == 0
    _refused(lib, call(None, 1), "null")


def test_muon(lib):
    def call(*mats, momentum=0.9, decay=0.0, steps=5, ws=9 * P):
        arr = (MuonMatrixT * len(mats))()
        for a, kw in zip(arr, mats):
            for k, v in dict(dict(param=P, grad=2 * P, momentum=3 * P, ld_param=8, ld_grad=8, ld_momentum=8, rows=5, cols=8, lr=0.1), **kw).items():
                setattr(a, k, v)
        return lib.suave_muon_step(arr, len(mats), momentum, 1, decay, steps, 1e-7, ws, 1 << 40, None)

    for kw, text in ((dict(param=None), "null"), (dict(ld_momentum=7), "stride"), (dict(lr=-1.0), "lr"), (dict(lr=float("inf")), "lr"),
                     (dict(momentum=P), "three"), (dict(grad=3 * P), "three")):
        _refused(lib, call(kw), text)
    _refused(lib, call({}, dict(grad=5 * P, momentum=6 * P)), "twice")
    _refused(lib, call({}, dict(grad=5 * P, param=6 * P)), "twice")
    _refused(lib, call({}, momentum=1.0), "momentum")
    _refused(lib, call({}, decay=-0.1), "weight_decay")
    _refused(lib, call({}, steps=0), "steps")
    _refused(lib, call({}, ws=None), "workspace")


def test_python_checks_without_a_gpu():
    import torch
    from suave_amd import operators as ops

    x, w, y = torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ops.linear_cross_entropy(x, w, y), lambda: ops.orthogonalize([x]), lambda: ops.quantize_rows(x),
                 lambda: ops.muon_step([x], [x.clone()], [x.clone()], lr=0.1),
                 lambda: ops.linear_quantized(x, w.to(torch.int8), torch.zeros(5))):
        with pytest.raises(slib.SuaveHipError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="length"):
        ops.muon_step([x], [], [x], lr=0.1)
    with pytest.raises(ValueError, match="lr"):
        ops.muon_step([x], [x], [x], lr=[0.1, 0.2])
    assert ops.orthogonalize([]) == [] and ops.muon_step([], [], [], lr=0.1) is None


def test_linear_quantized_outputs_that_are_inputs(lib):
    """In place: blocks that still quantise x would read what others have written."""

    def h(**kw):
        s = LinearQuantizedT()
        base = dict(dtype=0, n_out=20, n_in=20, n_rows=3, x=P, ld_x=20, weight=2 * P, ld_weight=32, weight_scale=3 * P, bias=6 * P, out=4 * P,
                    ld_out=20, workspace=5 * P, workspace_bytes=1 << 40)
        base.update(kw)
        for k, v in base.items():
            setattr(s, k, v)
        return s

    for other in ("x", "weight", "weight_scale", "bias"):
        _refused(lib, lib.suave_linear_quantized(C.byref(h(**{other: 4 * P})), None), "output is an input")


def test_muon_gradients_that_are_written(lib):
    def call(*mats):
        arr = (MuonMatrixT * len(mats))()
        for a, kw in zip(arr, mats):
            for k, v in dict(dict(ld_param=8, ld_grad=8, ld_momentum=8, rows=5, cols=8, lr=0.1), **kw).items():
                setattr(a, k, v)
        return lib.suave_muon_step(arr, len(mats), 0.9, 1, 0.0, 5, 1e-7, 9 * P, 1 << 40, None)

    one = dict(param=P, grad=2 * P, momentum=3 * P)
    for grad in (P, 3 * P):
        other = dict(param=5 * P, grad=grad, momentum=6 * P)
        _refused(lib, call(one, other), "another matrix's")
        _refused(lib, call(other, one), "another matrix's")
