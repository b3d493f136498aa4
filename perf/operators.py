"""The dense layer and the layer norm, forward and backward, as they are measured.

linear                y = act(x W + b) + r            act: none, relu, gelu (erf), silu; optionally also z = x W + b
linear_backward       dz = dy act'(z); dx = dz W^T, dW = x^T dz, db = column sums of dz
layer_norm            y = (x - mean) rstd g + b per row, with mean and rstd (float32) for the backward pass
layer_norm_backward   dx, dg, db of it, with the gradient that reaches x past the norm (a residual branch) added to dx

`layout` says how a weight lies in memory: "kn" rows of outputs (the layout of the framework's own weights), "nk" rows of
inputs, given to the call as the transposed view.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
_ctx = None


def listed():
    lin, bwd = {"op": "linear", "residual": False, "pre": False, "layout": "kn"}, {"op": "linear_backward", "layout": "kn"}
    return [
        # the camera heads' first layer on the views of one batch: the smallest call, latency counts
        dict(lin, name="linear_heads", type="f32", m=24, k=1024, n=512, act="relu"),
        # fc7 of one image's encoder: a single row, the weights are what is read
        dict(lin, name="linear_one_row", type="f32", m=1, k=4096, n=4096, act="relu"),
        # fold2/conv1 of the local stream, one chunk of query points, in the checkpoint's own type
        dict(lin, name="linear_points_f32", type="f32", m=100000, k=1984, n=512, act="relu"),
        # fold2/conv1 of the global stream in 16 bits
        dict(lin, name="linear_points_bf16", type="bf16", m=65536, k=1536, n=512, act="relu"),
        # the second half of a residual block of odd widths in training: row counts as they come, z kept for the backward pass
        dict(lin, name="linear_ragged_f16", type="f16", m=10007, k=1000, n=777, act="gelu", residual=True, pre=True, layout="nk"),
        # a training step of a decoder layer on a chunk of points
        dict(bwd, name="linear_backward_points", type="bf16", m=65536, k=1536, n=512, act="relu"),
        # fine-tuning a camera head on a batch of embeddings
        dict(bwd, name="linear_backward_heads", type="f32", m=32, k=1024, n=512, act="relu"),
        # a layer of odd widths, weights stored by rows of inputs
        dict(bwd, name="linear_backward_ragged", type="f32", m=4099, k=515, n=257, act="silu", layout="nk"),
        # the norm of one embedding
        dict(op="layer_norm", name="layer_norm_one_row", type="f32", rows=1, d=1024),
        # the norm of a chunk's point features
        dict(op="layer_norm", name="layer_norm_points", type="bf16", rows=262144, d=512),
        # its backward pass in a residual block
        dict(op="layer_norm_backward", name="layer_norm_backward_points", type="bf16", rows=262144, d=512, residual=True),
        # a norm over an odd number of features
        dict(op="layer_norm_backward", name="layer_norm_backward_ragged", type="f32", rows=5003, d=1537, residual=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear_backward", "layer_norm", "layer_norm_backward"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op.startswith("linear"):
        m, k, n = _log(rng, 1, 131072), _log(rng, 3, 4096), _log(rng, 1, 4096)
        if rng.random() < 0.5:  # widths of networks are more often than not multiples of 32
            k, n = -(-k // 32) * 32, -(-n // 32) * 32
        m = max(1, min(m, int((2e11 if op == "linear" else 1e11) / (2 * k * n)), int(4e8 / (k + n))))
        case = {"op": op, "type": kind, "m": m, "k": k, "n": n, "act": rng.choice(["none", "relu", "gelu", "silu"]), "layout": rng.choice(["kn", "nk"])}
        return dict(case, residual=rng.random() < 0.3, pre=rng.random() < 0.3) if op == "linear" else case
    d = _log(rng, 32, 8192)
    rows = max(1, min(_log(rng, 1, 262144), (1 << 27) // d))
    case = {"op": op, "type": kind, "rows": rows, "d": d}
    return dict(case, residual=rng.random() < 0.5) if op == "layer_norm_backward" else case


def work(case):
    s = 4 if case["type"] == "f32" else 2
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": s * (m * k + k * n + n + m * n * (1 + case["residual"] + case["pre"])), "flops": 2 * m * k * n}
    if case["op"] == "linear_backward":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": s * (2 * m * k + 2 * k * n + n + m * n * (1 + (case["act"] != "none"))), "flops": 4 * m * k * n}
    e = case["rows"] * case["d"]
    if case["op"] == "layer_norm":
        return {"bytes": s * (2 * e + 2 * case["d"]) + 8 * case["rows"], "flops": 8 * e}
    return {"bytes": s * (e * (3 + case["residual"]) + 3 * case["d"]) + 8 * case["rows"], "flops": 14 * e}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(kind)

    if case["op"].startswith("linear"):
        m, k, n = case["m"], case["k"], case["n"]
        lim = math.sqrt(6.0 / (k + n))
        w = (torch.rand(k, n, generator=g, device="cuda") * (2 * lim) - lim).to(kind)
        if case["layout"] == "nk":
            w = w.t().contiguous().t()
        x = normal(m, k)
        if case["act"] == "relu":  # behind another such layer: half of the values are zero
            x = x.clamp_min_(0)
        state = {"case": case, "x": x, "w": w}
        if case["op"] == "linear":
            return dict(state, bias=normal(n, std=0.1), residual=normal(m, n) if case["residual"] else None)
        return dict(state, dy=normal(m, n), pre=normal(m, n) if case["act"] != "none" else None)
    rows, d = case["rows"], case["d"]
    x = normal(rows, d) * (0.5 + torch.rand(rows, 1, generator=g, device="cuda")).to(kind) + normal(rows, 1)
    state = {"case": case, "x": x, "weight": normal(d, std=0.2, mean=1.0)}
    if case["op"] == "layer_norm":
        return dict(state, bias=normal(d, std=0.2))
    wide = x.double()
    mean = wide.mean(1)
    rstd = 1 / torch.sqrt(wide.var(1, unbiased=False) + EPS)
    return dict(state, dy=normal(rows, d), mean=mean.float(), rstd=rstd.float(), residual=normal(rows, d) if case["residual"] else None)


def _context():
    global _ctx
    if _ctx is None:
        from disn_amd.api import Context
        _ctx = Context(0)
    return _ctx


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _linear(s, case):
    kind = s["x"].dtype
    z = s["x"].float() @ s["w"].float() + s["bias"].float()
    y = _act(z, case["act"])
    if case["residual"]:
        y = y + s["residual"].float()
    return {"y": y.to(kind), "pre": z.to(kind)} if case["pre"] else {"y": y.to(kind)}


def _linear_backward(s, case):
    kind = s["x"].dtype
    dz = s["dy"].float()
    if case["act"] != "none":
        dz = dz * _slope(s["pre"].float(), case["act"])
    return {"dx": (dz @ s["w"].float().t()).to(kind), "dw": (s["x"].float().t() @ dz).to(kind), "db": dz.sum(0).to(kind)}


def _layer_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    y = c * rstd * s["weight"].float() + s["bias"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _layer_norm_backward(s, case):
    kind = s["x"].dtype
    rstd = s["rstd"][:, None]
    h = (s["x"].float() - s["mean"][:, None]) * rstd
    dy = s["dy"].float()
    t = dy * s["weight"].float()
    dx = rstd * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
    if case["residual"]:
        dx = dx + s["residual"].float()
    return {"dx": dx.to(kind), "dweight": (dy * h).sum(0).to(kind), "dbias": dy.sum(0).to(kind)}


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        ctx = _context()
        if op == "linear":
            got = ctx.linear(state["x"], state["w"], state["bias"], residual=state["residual"], act=case["act"], want_pre=case["pre"])
            return {"y": got[0], "pre": got[1]} if case["pre"] else {"y": got}
        if op == "linear_backward":
            dx, dw, db = ctx.linear_backward(state["dy"], state["x"], state["w"], pre=state["pre"], act=case["act"])
            return {"dx": dx, "dw": dw, "db": db}
        if op == "layer_norm":
            y, mean, rstd = ctx.layer_norm(state["x"], state["weight"], state["bias"], eps=EPS, want_stats=True)
            return {"y": y, "mean": mean, "rstd": rstd}
        dx, dweight, dbias = ctx.layer_norm_backward(state["dy"], state["x"], state["mean"], state["rstd"], state["weight"], residual=state["residual"])
        return {"dx": dx, "dweight": dweight, "dbias": dbias}
    if op == "linear":
        return _linear(state, case)
    if op == "linear_backward":
        return _linear_backward(state, case)
    if op == "layer_norm":
        return _layer_norm(state)
    return _layer_norm_backward(state, case)


def exact(case, seed):
    """The definitions in 64 bits, by torch's own functions; gradients of the norm and of the activations by differentiation."""
    f = torch.nn.functional
    acts = {"none": lambda z: z, "relu": f.relu, "gelu": f.gelu, "silu": f.silu}
    s = {key: v.double() if torch.is_tensor(v) else v for key, v in prepare(case, seed).items()}
    if case["op"] == "linear":
        z = f.linear(s["x"], s["w"].t(), s["bias"])
        y = acts[case["act"]](z)
        y = y + s["residual"] if case["residual"] else y
        return {"y": y, "pre": z} if case["pre"] else {"y": y}
    if case["op"] == "linear_backward":
        dz = s["dy"]
        if case["act"] != "none":
            z = s["pre"].requires_grad_()
            dz, = torch.autograd.grad(acts[case["act"]](z), z, s["dy"])
        return {"dx": f.linear(dz, s["w"]), "dw": torch.mm(s["x"].t(), dz), "db": torch.ones(1, dz.shape[0], dtype=dz.dtype, device=dz.device).mm(dz)[0]}
    if case["op"] == "layer_norm":
        var, mean = torch.var_mean(s["x"], 1, correction=0)
        return {"y": f.layer_norm(s["x"], (case["d"],), s["weight"], s["bias"], EPS), "mean": mean, "rstd": torch.rsqrt(var + EPS)}
    x, w = s["x"].requires_grad_(), s["weight"].requires_grad_()
    b = torch.zeros_like(w).requires_grad_()
    dx, dw, db = torch.autograd.grad(f.layer_norm(x, (case["d"],), w, b, EPS), (x, w, b), s["dy"])
    return {"dx": dx + s["residual"] if case["residual"] else dx, "dweight": dw, "dbias": db}
