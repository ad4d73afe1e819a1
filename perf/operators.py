"""Cases of the operators around a classifier with many classes: its loss and gradients without the logits
(``suave_amd.operators.linear_cross_entropy``), the orthogonalised update of hidden weight matrices
(``orthogonalize`` / ``muon_step``) and the 8-bit integer product that serves the head (``linear_quantized``).

``run`` computes an operator in its plain form (elementary torch operations) or, where ``own`` is true, by the
framework's call.  ``exact`` states each operator's definition in float64."""

import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
NS = (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # the head phase of the 20-column demo table: batches of 256, latent 32; just past the 64 classes of the small head kernel
        {"name": "ce f32 256x100x32", "op": "ce", "n": 256, "c": 100, "d": 32, "dtype": "f32", "grad": True, "weighted": False},
        # the 1024-column table's latent of 128, batches of 4096 rows, class weights as `fit` derives them
        {"name": "ce f32 4096x1000x128", "op": "ce", "n": 4096, "c": 1000, "d": 128, "dtype": "f32", "grad": True, "weighted": True},
        # odd everything: a ragged last batch, classes and widths that are multiples of nothing
        {"name": "ce f32 1777x20011x501", "op": "ce", "n": 1777, "c": 20011, "d": 501, "dtype": "f32", "grad": True, "weighted": True},
        # a head with hidden layers over a vocabulary, bf16 training
        {"name": "ce bf16 4096x32000x1024", "op": "ce", "n": 4096, "c": 32000, "d": 1024, "dtype": "bf16", "grad": True, "weighted": False},
        # scoring a few rows against a large vocabulary: the loss alone
        {"name": "ce bf16 33x100000x2048 loss", "op": "ce", "n": 33, "c": 100000, "d": 2048, "dtype": "bf16", "grad": False, "weighted": False},
        # the hidden layers of the 64-column benchmark model (hidden 256, 128; latent 32): a whole optimiser step
        {"name": "muon f32 model", "op": "muon", "shapes": "256x205,128x256,256x32,128x256", "dtype": "f32"},
        # matrices of several odd shapes at once, tall and wide
        {"name": "orthogonalize f32 odd", "op": "ortho", "shapes": "500x333,1000x77,641x640", "dtype": "f32"},
        # large hidden layers, bf16 updates
        {"name": "orthogonalize bf16 2x1024x4096", "op": "ortho", "shapes": "1024x4096,4096x1024", "dtype": "bf16"},
        # the same arithmetic where a single square matrix has to fill the card, fp32
        {"name": "orthogonalize f32 2048x2048", "op": "ortho", "shapes": "2048x2048", "dtype": "f32"},
        # one row asked for its logits: latency
        {"name": "int8 f32 1x1000x256", "op": "int8", "m": 1, "n": 1000, "k": 256, "dtype": "f32", "bias": True},
        # a small batch of requests against a large head: the weights' bytes
        {"name": "int8 bf16 16x100000x2048", "op": "int8", "m": 16, "n": 100000, "k": 2048, "dtype": "bf16", "bias": False},
        # bulk scoring: the matrix pipe
        {"name": "int8 bf16 8192x16384x2048", "op": "int8", "m": 8192, "n": 16384, "k": 2048, "dtype": "bf16", "bias": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ce", "ce", "ortho", "muon", "int8", "int8"))
    dtype = rng.choice(("f32", "bf16"))
    if op == "ce":
        while True:
            n, c, d = _log_int(rng, 1, 8192), _log_int(rng, 65, 100000), _log_int(rng, 8, 2048)
            if rng.random() < 0.5:
                c, d = (c + 7) // 8 * 8, (d + 7) // 8 * 8
            if n * c * d <= 4096 * 32000 * 1024 // (1 if dtype == "bf16" else 4) and n * c <= 1 << 27:
                return {"op": "ce", "n": n, "c": c, "d": d, "dtype": dtype, "grad": rng.random() < 0.75, "weighted": rng.random() < 0.5}
    if op == "int8":
        while True:
            m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 65, 100000), _log_int(rng, 16, 4096)
            if m * n * k <= 8192 * 16384 * 2048 and m * n <= 1 << 27:
                return {"op": "int8", "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.5}
    shapes = []
    for _ in range(rng.randint(1, 4)):
        while True:
            r, c = _log_int(rng, 1, 2500), _log_int(rng, 1, 2500)
            if r * c * min(r, c) <= 1 << 31:
                break
        shapes.append("%dx%d" % (r, c))
    return {"op": op, "shapes": ",".join(shapes), "dtype": "f32" if op == "muon" else dtype}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _gen(seed)
    dev = "cuda"
    rand = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    dt = DT[case["dtype"]]
    if case["op"] == "ce":
        n, c, d = case["n"], case["c"], case["d"]
        s = {"x": rand(n, d).to(dt), "w": (rand(c, d) * (2.0 / math.sqrt(d))).to(dt), "b": rand(c) * 0.1}
        s["y"] = torch.randint(0, c, (n,), generator=g, device=dev, dtype=torch.int32)
        s["cw"] = None
        if case["weighted"]:  # class weights, and one row in sixteen without a label
            s["cw"] = torch.rand(c, generator=g, device=dev) + 0.5
            s["y"] = torch.where(torch.rand(n, generator=g, device=dev) < 1 / 16, torch.full_like(s["y"], -1), s["y"])
        return dict(s, op="ce", grad=case["grad"])
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        ld = (k + 15) // 16 * 16
        w = rand(n, k) / math.sqrt(k)
        scale = w.abs().amax(dim=1) / 127.0
        q = torch.zeros((n, ld), dtype=torch.int8, device=dev)
        q[:, :k] = torch.round(w / scale[:, None]).clamp(-127, 127).to(torch.int8)
        return {"op": "int8", "x": rand(m, k).to(dt), "q": q[:, :k], "scale": scale, "b": rand(n) if case["bias"] else None}
    # gradients of a few directions above noise, as a batch gives them
    grads = []
    for r, c in _shapes(case):
        t = min(8, r, c)
        grads.append((rand(r, t) @ rand(t, c) * 0.3 + rand(r, c)) * 1e-3)
    if case["op"] == "ortho":
        return {"op": "ortho", "u": [t.to(dt) for t in grads]}
    return {"op": "muon", "g": grads, "m": [rand(*t.shape) * 1e-3 for t in grads],
            "p": [rand(*t.shape) / math.sqrt(t.shape[1]) for t in grads]}


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _ce_plain(x, w, b, y, cw, grad):
    xf, wf = x.float(), w.float()
    keep = y >= 0
    yi = y.clamp_min(0).long()
    l = xf @ wf.t() + b
    mx = l.amax(dim=1, keepdim=True)
    e = torch.exp(l - mx)
    se = e.sum(dim=1, keepdim=True)
    wy = (torch.ones_like(mx[:, 0]) if cw is None else cw[yi]) * keep
    rows = wy * ((mx + torch.log(se))[:, 0] - l.gather(1, yi[:, None])[:, 0])
    total = wy.double().sum()
    total = torch.where(total > 0, total, torch.ones_like(total))  # a batch without a labelled row: loss 0, gradients 0
    loss = (rows.double().sum() / total).float()
    if not grad:
        return {"loss": loss, "row_loss": rows}
    f = (wy.double() / total).float()
    gl = e * (f[:, None] / se)
    gl.scatter_add_(1, yi[:, None], -f[:, None])
    return {"loss": loss, "row_loss": rows, "dx": (gl @ wf).to(x.dtype), "dweight": (gl.t() @ xf).to(w.dtype), "dbias": gl.sum(dim=0)}


def _ns_plain(u, steps=5, eps=1e-7):
    a, b, c = NS
    tall = u.shape[0] > u.shape[1]
    x = u.t() if tall else u
    x = x.float() / (u.double().square().sum().sqrt() + eps).float()
    for _ in range(steps):
        A = x @ x.t()
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.t() if tall else x


def _int8_plain(x, q, scale, b):
    xf = x.float()
    s = xf.abs().amax(dim=1) / 127.0
    # values next to a rounding border decide in 64 bits
    xq = torch.round(xf.double() / torch.where(s > 0, s, torch.ones_like(s)).double()[:, None]).clamp(-127, 127).float()
    out = (xq @ q.float().t()) * (s[:, None] * scale[None, :])
    return (out if b is None else out + b).to(x.dtype)


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "ce":
        return _ce_plain(s["x"], s["w"], s["b"], s["y"], s["cw"], s["grad"])
    if s["op"] == "int8":
        return {"out": _int8_plain(s["x"], s["q"], s["scale"], s["b"])}
    if s["op"] == "ortho":
        return {"o": [_ns_plain(u).to(u.dtype).contiguous() for u in s["u"]]}
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        m.mul_(0.95).add_(g)
        p.add_(_ns_plain(g + 0.95 * m), alpha=-0.02 * math.sqrt(max(1.0, p.shape[0] / p.shape[1])))
    return {"p": s["p"], "m": s["m"]}


def _run_own(s):
    from suave_amd import operators as ops

    if s["op"] == "ce":
        r = ops.linear_cross_entropy(s["x"], s["w"], s["y"], bias=s["b"], class_weight=s["cw"], grad=s["grad"])
        return {k: r[k] for k in (("loss", "row_loss", "dx", "dweight", "dbias") if s["grad"] else ("loss", "row_loss"))}
    if s["op"] == "int8":
        return {"out": ops.linear_quantized(s["x"], s["q"], s["scale"], bias=s["b"])}
    if s["op"] == "ortho":
        return {"o": ops.orthogonalize(s["u"])}
    ops.muon_step(s["p"], s["g"], s["m"], lr=0.02, momentum=0.95, nesterov=True)
    return {"p": s["p"], "m": s["m"]}


# ---- what one pass cannot do without -------------------------------------------------------------------------------
def work(case):
    b = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "ce":
        n, c, d = case["n"], case["c"], case["d"]
        read = b * (n * d + c * d) + 4 * c + 4 * n + (4 * c if case["weighted"] else 0)
        return {"bytes": read + 4 * n + ((b * (n * d + c * d) + 4 * c) if case["grad"] else 0), "flops": (6 if case["grad"] else 2) * n * c * d}
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": b * m * k + n * k + 4 * n + b * m * n + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    size = flops = 0
    for r, c in _shapes(case):
        s, l = min(r, c), max(r, c)
        size += r * c
        flops += 5 * (s * s * l + s * s * s + 2 * s * s * l)  # the two symmetric products by half
    return {"bytes": size * (b * 2 if case["op"] == "ortho" else 4 * 5), "flops": flops}


# ---- definitions in 64 bits ----------------------------------------------------------------------------------------
def _ns_exact(u, eps=1e-7):
    # each step as a product from the right with the Gram matrix of the columns or from the left with that of the rows,
    # whichever is smaller, in the order the definition is written: x (a + b G + c G G)
    a, b, c = NS
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x) + eps)
    for _ in range(5):
        if x.shape[0] >= x.shape[1]:
            G = x.t() @ x
            x = a * x + b * (x @ G) + c * ((x @ G) @ G)
        else:
            G = x @ x.t()
            x = a * x + b * (G @ x) + c * (G @ (G @ x))
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "ce":
        x, w, y = s["x"].double(), s["w"].double(), s["y"].long()
        lp = torch.log_softmax(x @ w.t() + s["b"].double(), dim=1)
        rows = torch.arange(y.numel(), device=y.device)[y >= 0]
        yk = y[y >= 0]
        wk = torch.ones_like(yk, dtype=torch.float64) if s["cw"] is None else s["cw"].double()[yk]
        per = torch.zeros(y.numel(), dtype=torch.float64, device=y.device)
        per[rows] = -wk * lp[rows, yk]
        out = {"loss": per.sum() / (wk.sum() if rows.numel() else 1.0), "row_loss": per}
        if not s["grad"]:
            return out
        share = torch.zeros_like(per)
        share[rows] = wk / wk.sum()
        gl = lp.exp_()
        gl[rows, yk] -= 1.0
        gl *= share[:, None]
        return dict(out, dx=gl @ w, dweight=gl.t() @ x, dbias=gl.sum(dim=0))
    if s["op"] == "int8":
        x = s["x"].double()
        step = (x.abs().amax(dim=1).float() / 127.0).double()  # the scale is a 32-bit number
        levels = torch.where(step[:, None] > 0, torch.round(x / step[:, None]), torch.zeros_like(x))
        out = (levels * step[:, None]) @ (s["q"].double() * s["scale"].double()[:, None]).t()
        return {"out": out if s["b"] is None else out + s["b"].double()}
    if s["op"] == "ortho":
        return {"o": [_ns_exact(u) for u in s["u"]]}
    out = {"p": [], "m": []}
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        m1 = 0.95 * m.double() + g.double()
        out["m"].append(m1)
        out["p"].append(p.double() - 0.02 * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * _ns_exact(g.double() + 0.95 * m1))
    return out
