"""Dense layer and layer norm, forward and backward (Context.linear, linear_backward, layer_norm, layer_norm_backward),
against plain formulas in float64.

Two kinds of checks.  Small whole numbers: every product and sum is exact in float32, so results must be the float64 ones
rounded once, bit for bit, whatever the order of the sums.  Real numbers: bounds worked out from the arithmetic.  E = 2^-24
is half a step of float32, U half a step of the tensors' type; a sum of n terms in float32 is off by at most n E times the
sum of the absolute terms per rounding, and the bounds count two (the matrix cores' own order of adding is not
specified)."""
import math
import zlib

import numpy as np
import pytest
import torch

from disn_amd import _lib, api, camera

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
E = 2.0 ** -24
KINDS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = {k: torch.finfo(t).eps / 2 for k, t in KINDS.items()}
ACTS = ("none", "relu", "gelu", "silu")

# (m, k, n): empty ones; single values; few rows times a large matrix (both sums of it); small products with long and
# short sums; tiles of 128 and 256, split and whole, with edges in every direction
SIZES = [(0, 5, 4), (5, 0, 4), (3, 5, 0), (1, 1, 1), (1, 2, 7), (7, 3, 64), (17, 129, 33), (33, 515, 257), (24, 1024, 512), (16, 127, 128),
         (1, 4096, 260), (2, 1031, 1025), (5, 2049, 515), (16, 1024, 1024), (17, 1024, 1024), (1, 70000, 16), (3, 16, 70000),
         (1000, 300, 777), (130, 1032, 1025), (4099, 515, 257), (65, 20000, 130), (33000, 65, 520), (20000, 67, 1000),
         (3, 4096, 2100), (4, 2000, 3000), (3000, 900, 1100), (9000, 1100, 2000), (66000, 700, 520)]


def ints(gen, kind, *shape, top=3):
    return torch.randint(-top, top + 1, shape, generator=gen, device=DEV).to(KINDS[kind])


def gen(*seed):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(seed).encode()))


def weight(w, layout):
    """[k, n] values lying by rows of outputs or of inputs"""
    return w if layout == "kn" else w.t().contiguous().t()


def act64(z, act):
    return {"none": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[act](z)


def slope64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def same(got, want):
    assert got.shape == want.shape
    assert torch.equal(got, want.to(got.dtype)), "%d of %d values differ" % ((got != want.to(got.dtype)).sum(), got.numel())


def within(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    worst = (off / bound.clamp_min(1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, "%.3g times the bound" % worst


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_whole_numbers(ctx, m, k, n, kind, layout):
    g = gen(m, k, n, kind, layout)
    x, w, b, r = (ints(g, kind, *s) for s in ((m, k), (k, n), (n,), (m, n)))
    z = x.double() @ w.double() + b.double()
    y, pre = ctx.linear(x, weight(w, layout), b, residual=r, act="relu", want_pre=True)
    same(pre, z)
    same(y, torch.relu(z) + r.double())
    same(ctx.linear(x, weight(w, layout)), x.double() @ w.double())


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_backward_whole_numbers(ctx, m, k, n, kind, layout):
    g = gen(m, k, n, kind, layout, 1)
    # where the sum over the rows is long, values of -1, 0 and 1 keep it below 2^24
    x, w, dy, pre = (ints(g, kind, *s, top=2) for s in ((m, k), (k, n), (m, n), (m, n)))
    for act in ("relu", "none"):
        dz = dy.double() * (pre > 0) if act == "relu" else dy.double()
        dx, dw, db = ctx.linear_backward(dy, x, weight(w, layout), pre=pre if act == "relu" else None, act=act)
        same(dx, dz @ w.double().t())
        same(dw, x.double().t() @ dz)
        same(db, dz.sum(0))
    assert (dw.stride(0) == 1) == (layout == "nk") or 1 in dw.shape or 0 in dw.shape


@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1), (0, 0, 0)])
@pytest.mark.parametrize("m,k,n", [(33, 70, 50), (2100, 260, 300), (3, 1024, 1100)])
def test_linear_backward_parts(ctx, m, k, n, want):
    g = gen(m, k, n, want)
    x, w, dy, pre = (ints(g, "bf16", *s, top=2) for s in ((m, k), (k, n), (m, n), (m, n)))
    every = ctx.linear_backward(dy, x, w, pre=pre, act="relu")
    some = ctx.linear_backward(dy, x if want[1] else None, w if want[0] or not want[1] else None, pre=pre, act="relu", want_dx=bool(want[0]),
                               want_dw=bool(want[1]), want_db=bool(want[2]))
    for v, one, both in zip(want, some, every):
        assert (one is not None) == bool(v)
        if v:
            same(one, both.double())


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", [(1, 3, 5), (24, 1024, 512), (4, 1500, 800), (700, 1100, 333), (33000, 40, 520), (3000, 900, 1100)])
def test_linear_values(ctx, m, k, n, kind, act):
    g = gen(m, k, n, kind, act)
    x, w, b, r = (torch.randn(*s, generator=g, device=DEV).to(KINDS[kind]) for s in ((m, k), (k, n), (n,), (m, n)))
    w = (w.float() * k ** -0.5).to(w.dtype)
    z = x.double() @ w.double() + b.double()
    y, pre = ctx.linear(x, w, b, residual=r, act=act, want_pre=True)
    # float32: the three-term products drop less than 3 E of each; then the sum's own roundings
    zerr = 2 * (k + 4) * E * (x.double().abs() @ w.double().abs() + b.double().abs())
    within(pre, z, zerr + U[kind] * (z.abs() + zerr) + 1e-7 * (kind == "f16"))   # a half below 2^-14 has steps of 2^-24
    # |act'| <= 1.13; exp and erf of float32 are good to a few steps of values of order max(|z|, 1)
    yerr = 1.13 * zerr + 16 * E * (1 + z.abs()) + E * (act64(z, act).abs() + r.double().abs())
    want = act64(z, act) + r.double()
    within(y, want, yerr + U[kind] * (want.abs() + yerr) + 1e-7 * (kind == "f16"))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", [(1, 3, 5), (32, 1024, 512), (900, 300, 520), (5000, 130, 260), (9, 1100, 1000), (3000, 900, 1100)])
def test_linear_backward_values(ctx, m, k, n, kind, act):
    g = gen(m, k, n, kind, act, 2)
    x, w, dy, pre = (torch.randn(*s, generator=g, device=DEV).to(KINDS[kind]) for s in ((m, k), (k, n), (m, n), (m, n)))
    dx, dw, db = ctx.linear_backward(dy, x, w, pre=None if act == "none" else pre, act=act)
    dz = dy.double() * slope64(pre.double(), act)
    # slopes to a few steps of float32; dz once more to the type's own half step where it feeds 16-bit products
    zerr = 16 * E * dy.double().abs() * (1 + pre.double().abs())
    zerr16 = zerr if act == "none" or kind == "f32" else zerr + U[kind] * (dz.abs() + zerr)
    tiny = 1e-7 * (kind == "f16")
    for got, a, b, e in ((dx, dz, w.double().t(), (zerr16 + tiny) @ w.double().abs().t()),
                         (dw, x.double().t(), dz, x.double().abs().t() @ (zerr16 + tiny))):
        want, err = a @ b, e + 2 * (a.shape[1] + 4) * E * (a.abs() @ b.abs())
        within(got, want, err + U[kind] * (want.abs() + err) + tiny)
    want, err = dz.sum(0), (zerr16 + 2 * m * E * dz.abs()).sum(0)
    within(db, want, err + U[kind] * (want.abs() + err) + tiny)


@pytest.mark.parametrize("m,k,n", [(8, 12, 9), (200, 90, 70), (600, 600, 400)])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_linear_gradient_against_differences(ctx, m, k, n, act):
    g = gen(m, k, n, act, 3)
    x, w, dy = (torch.randn(*s, generator=g, device=DEV) for s in ((m, k), (k, n), (m, n)))
    w *= k ** -0.5
    b = torch.randn(n, generator=g, device=DEV)
    _, pre = ctx.linear(x, w, b, act=act, want_pre=True)
    grads = ctx.linear_backward(dy, x, w, pre=pre, act=act)
    args = [x.double(), w.double(), b.double()]
    loss = lambda a: (act64(a[0] @ a[1] + a[2], act) * dy.double()).sum()
    h = 1e-4
    for i, grad in enumerate(grads):
        v = torch.randn(args[i].shape, generator=g, device=DEV, dtype=torch.float64)
        v /= v.norm()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * v, args[i] - h * v
        slope = ((loss(up) - loss(down)) / (2 * h)).item()
        # central differences: error h^2 / 6 of a third derivative that is of the gradient's size; gradient: float32 sums
        assert abs(slope - (grad.double() * v).sum().item()) <= 2e-5 * grad.double().norm().item() + 1e-6


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", [(5, 40, 30), (3, 1100, 1000), (300, 700, 800), (33000, 40, 520), (3, 4096, 2100), (3000, 900, 1100), (9000, 1100, 2000)])
def test_linear_rows_anywhere(ctx, m, k, n, kind):
    """slices of wider buffers at odd addresses, expanded and transposed inputs, a column range as the output"""
    g = gen(m, k, n, kind, 4)
    x, w, r = ints(g, kind, m, k + 5)[:, 3:3 + k], ints(g, kind, k, n + 3)[:, 1:1 + n], ints(g, kind, m, n + 1)[:, 1:]
    want = x.double() @ w.double()
    buf = torch.full((m + 2, n + 9), 77.0, device=DEV, dtype=KINDS[kind])
    y = ctx.linear(x, w, residual=r, out=buf[1:-1, 5:5 + n])
    assert y.data_ptr() == buf[1:-1, 5:].data_ptr()
    same(y, want + r.double())
    edge = buf.clone()
    edge[1:-1, 5:5 + n] = 77.0
    assert (edge == 77.0).all()
    wt = ints(g, kind, n, k + 3)[:, 2:2 + k].t()
    same(ctx.linear(x.t().contiguous().t(), wt), x.double() @ wt.double())
    one = ints(g, kind, 1, k).expand(m, k)
    same(ctx.linear(one, w, residual=ints(g, kind, 1, n).expand(m, n) * 0), one.double() @ w.double())
    # in place on the residual
    acc = r.clone()
    same(ctx.linear(x, w, residual=acc, out=acc), want + r.double())
    # backward on the same kind of views
    dy, pre = ints(g, kind, m, n + 4, top=1)[:, 2:2 + n], ints(g, kind, m, n + 1)[:, :n]
    dz = dy.double() * (pre > 0)
    for weights in (w, wt):
        dx, dw, db = ctx.linear_backward(dy, x, weights, pre=pre, act="relu")
        same(dx, dz @ weights.double().t())
        same(dw, x.double().t() @ dz)
        same(db, dz.sum(0))
    dy1 = dy[:1].expand(m, n)
    dx, dw, db = ctx.linear_backward(dy1, one, w)
    same(dx, dy1.double() @ w.double().t())
    same(dw, one.double().t() @ dy1.double())
    same(db, dy1.double().sum(0))


def test_linear_leading_dimensions(ctx):
    g = gen(5)
    x, w = ints(g, "f32", 2, 3, 4, 20), ints(g, "f32", 20, 6)
    same(ctx.linear(x, w), x.double() @ w.double())
    same(ctx.linear(x[0, 0, 0], w), x[0, 0, 0].double() @ w.double())
    same(ctx.linear(x.transpose(0, 2), w), x.transpose(0, 2).double() @ w.double())
    dy = ints(g, "f32", 2, 3, 4, 6)
    dx, dw, db = ctx.linear_backward(dy, x, w)
    same(dx, dy.double() @ w.double().t())
    same(dw, x.double().reshape(-1, 20).t() @ dy.double().reshape(-1, 6))
    same(db, dy.double().reshape(-1, 6).sum(0))
    assert ctx.linear(x[:, :0], w).shape == (2, 0, 4, 6)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", [(20, 40, 30), (4, 1100, 1000), (300, 700, 800), (4, 4096, 2100), (3000, 900, 1100), (9000, 1100, 2000)])
def test_linear_infinities_and_nan(ctx, m, k, n, kind):
    """they reach exactly the sums that hold them, as in a chain of multiply-adds"""
    g = gen(m, k, n, kind, 6)
    x, w = ints(g, kind, m, k), ints(g, kind, k, n)
    w[w == 0] = 1.0                                        # 0 * inf would be NaN, rightly
    x[1, 7], x[2, k - 1], x[3, 0] = float("inf"), float("nan"), float("-inf")
    x[3, 5] = float("inf")
    y = ctx.linear(x, w).double()
    want = x.double() @ w.double()
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf())
    fine = want.isfinite()
    assert torch.equal(y[~want.isnan()], want[~want.isnan()].to(KINDS[kind]).double()) and fine[4 if m > 4 else 0].all()
    x[3, 5] = 1.0
    relu = ctx.linear(x, w, act="relu").double()
    assert torch.equal(relu[2].isnan(), torch.ones_like(relu[2], dtype=torch.bool))
    assert torch.equal(relu[1].isinf(), w[7] > 0) and (relu[1][w[7] < 0] == 0).all()


@pytest.mark.parametrize("m,k,n", [(20, 40, 30), (4, 1100, 1000), (300, 700, 800), (3, 4096, 2100), (3000, 900, 1100), (9000, 1100, 2000)])
def test_linear_float32_range(ctx, m, k, n):
    """the whole range of float32: values next to the largest, sums that overflow, products that are subnormal"""
    g = gen(m, k, n, 7)
    xi, w = ints(g, "f32", m, k), ints(g, "f32", k, n)
    same(ctx.linear(xi * 2.0 ** -130, w), (xi.double() @ w.double()) * 2.0 ** -130)
    x = torch.zeros(m, k, device=DEV)
    x[:, 3] = 3.4028234e38
    w = torch.zeros(k, n, device=DEV)
    w[3] = 1.0
    same(ctx.linear(x, w), x.double() @ w.double())
    x[:, 3], w[3], w[3, 1] = 1.2345e30, 1.2345e30, -1.2345e30
    y = ctx.linear(x, w)
    assert (y[:, 0] == float("inf")).all() and (y[:, 1] == float("-inf")).all()


@pytest.mark.parametrize("kind", list(KINDS))
def test_linear_longest_rows(ctx, kind):
    """sums over the largest k, on and off 16-byte boundaries, and rows of the largest n"""
    top = 1 << 22
    g = gen(kind, 9)
    x, w = ints(g, kind, 130, top, top=1), ints(g, kind, 132, top, top=1)
    want = torch.zeros(130, 132, dtype=torch.float64, device=DEV)
    for part in range(0, top, top // 8):                   # whole numbers up to 2^22: every order of the sums is exact
        c = slice(part, part + top // 8)
        want += x[:, c].double() @ w[:, c].double().t()
    same(ctx.linear(x, w.t()), want)
    off = torch.empty(130 * top + 1, dtype=x.dtype, device=DEV)[1:].view(130, top)
    off.copy_(x)
    same(ctx.linear(off, w.t()), want)
    del off
    dx, dw, db = ctx.linear_backward(x, w[0].repeat(130, 1)[:, :3].contiguous(), w[:3])   # n = top
    same(db, x.double().sum(0))
    del db, dw
    assert dx.shape == (130, 3)
    same(dx, want[:, :3])
    v = ints(g, kind, 24, top, top=1)
    same(ctx.linear(x[:40, :24].contiguous(), v)[:, -300:], x[:40, :24].double() @ v[:, -300:].double())
    y = ctx.linear(x[:2, :24].contiguous(), v[:, 1:].contiguous())
    same(y, x[:2, :24].double() @ v[:, 1:].double())


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("xs,ws", [(-120, 100), (-132, 118), (-145, 120), (118, -132), (-119, 0), (-60, -62)])
@pytest.mark.parametrize("m,k,n", [(20, 40, 30), (4, 1100, 1000), (300, 700, 800), (2000, 512, 515), (3000, 900, 1100), (40000, 200, 260)])
def test_linear_float32_smallest_values(ctx, m, k, n, xs, ws, layout):
    """values whose last bits lie next to the smallest of float32, or below those of a narrower type"""
    g = gen(m, k, n, xs, ws)
    x = (torch.randn(m, k, generator=g, device=DEV).double() * 2.0 ** xs).float()
    w = (torch.randn(k, n, generator=g, device=DEV).double() * 2.0 ** ws).float()
    # (k + 4) roundings as everywhere, and six partial sums that may each be rounded to steps of 2^-149 a term
    bound = 2 * (k + 4) * E * (x.double().abs() @ w.double().abs()) + 6 * (k + 4) * 2.0 ** -149
    within(ctx.linear(x, weight(w, layout)), x.double() @ w.double(), bound)
    dy = x.repeat(1, n // k + 1)[:, :n].contiguous()
    dx, _, _ = ctx.linear_backward(dy, x, weight(w, layout))
    within(dx, dy.double() @ w.double().t(), 2 * (n + 4) * E * (dy.double().abs() @ w.double().abs().t()) + 6 * (n + 4) * 2.0 ** -149)


@pytest.mark.parametrize("m,k,n", [(300, 700, 800), (3000, 900, 1100), (40000, 200, 260)])
def test_linear_float32_small_among_others(ctx, m, k, n):
    """rows of small values, rows of zeros and ordinary rows in one matrix"""
    g = gen(m, k, n, 8)
    x, w = torch.randn(m, k, generator=g, device=DEV), torch.randn(k, n, generator=g, device=DEV)
    x[::3] *= 2.0 ** -122
    x[1::6] = 0.0
    x[2::3, ::5] *= 2.0 ** -125
    y = ctx.linear(x, w)
    within(y, x.double() @ w.double(), 2 * (k + 4) * E * (x.double().abs() @ w.double().abs()) + 6 * (k + 4) * 2.0 ** -149)
    assert (y[1::6] == 0).all()


# layers with few inputs, few outputs or few rows: sums of up to 8 products, results of up to 8 columns, and one beyond either
NARROW = [(40000, 3, 70), (20000, 1, 515), (20000, 515, 1), (9617, 12, 2), (30011, 130, 5), (30000, 6, 257), (70001, 2, 9), (8, 3000, 2000),
          (2, 2100, 3001), (30000, 8, 8), (30000, 9, 300), (30000, 300, 9), (70000, 4, 4), (70000, 3, 1)]


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", NARROW)
def test_narrow_layers(ctx, m, k, n, kind, layout):
    test_linear_whole_numbers(ctx, m, k, n, kind, layout)
    test_linear_backward_whole_numbers(ctx, m, k, n, kind, layout)


@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", NARROW)
def test_narrow_layers_values(ctx, m, k, n, kind, act):
    test_linear_values(ctx, m, k, n, kind, act)
    test_linear_backward_values(ctx, m, k, n, kind, act)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", [(40000, 3, 70), (20000, 515, 1), (9617, 12, 2), (30000, 6, 257), (2, 2100, 3001)])
def test_narrow_layers_rows_anywhere(ctx, m, k, n, kind):
    test_linear_rows_anywhere(ctx, m, k, n, kind)
    g = gen(m, k, n, kind, 10)
    x, w, r = (ints(g, kind, *s) for s in ((m, k), (k, n), (m, n)))
    want = x.double() @ w.double() + r.double()
    assert ctx.linear(x, w, residual=r, out=r) is r        # in place
    same(r, want)


@pytest.mark.parametrize("m,k,n", [(40000, 3, 70), (30000, 515, 2)])
def test_narrow_layers_infinities_and_nan(ctx, m, k, n):
    g = gen(m, k, n, 11)
    x, w, dy = ints(g, "f32", m, k), ints(g, "f32", k, n), ints(g, "f32", m, n)
    x[7, 1], dy[9, 0] = float("nan"), float("inf")
    y = ctx.linear(x, w)
    assert torch.equal(y.isnan().any(1).nonzero().flatten(), torch.tensor([7], device=DEV))
    dx, dw, db = ctx.linear_backward(dy, x, w)
    assert torch.equal((~dx.isfinite()).any(1).nonzero().flatten(), torch.tensor([9], device=DEV))
    assert dw[1].isnan().all() and not dw[0, 1:].isnan().any() and not dw[2:, 1:].isnan().any()
    assert db[0] == float("inf") and db[1:].isfinite().all()


def norm_inputs(rows, d, kind, seed):
    g = gen(rows, d, kind, seed)
    x = (torch.randn(rows, d, generator=g, device=DEV) * (0.2 + 3 * torch.rand(rows, 1, generator=g, device=DEV)) +
         5 * torch.randn(rows, 1, generator=g, device=DEV)).to(KINDS[kind])
    return [x] + [torch.randn(*s, generator=g, device=DEV).to(KINDS[kind]) for s in ((d,), (d,), (rows, d), (rows, d))]


NORMS = [(1, 1), (3, 2), (1, 1024), (5, 7), (300, 33), (257, 128), (65, 129), (70, 511), (33, 513), (64, 1000), (31, 1024), (9, 1025), (200, 1537),
         (20, 2049), (7, 4096), (5, 4097), (3, 8191), (2, 8192), (70000, 40), (0, 16)]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows,d", NORMS)
def test_layer_norm(ctx, rows, d, kind):
    x, w, b, _, _ = norm_inputs(rows, d, kind, 0)
    eps = 1e-5
    y, mean, rstd = ctx.layer_norm(x, w, b, eps=eps, want_stats=True)
    wide = x.double()
    mu = wide.mean(1, keepdim=True)
    c = wide - mu
    var = (c * c).mean(1, keepdim=True)
    r = (var + eps) ** -0.5
    # a thread adds at most 16 values, lanes and waves another 20: 40 roundings of sums of |x| (and of c^2)
    merr = 40 * E * wide.abs().mean(1, keepdim=True)
    cerr = merr + E * c.abs()
    verr = 2 * (cerr * c.abs()).mean(1, keepdim=True) + (cerr * cerr).mean(1, keepdim=True) + 42 * E * var + E * eps
    rerr = r * (verr / (var + eps) + 4 * E)            # twice the first-order term; verr is far below var + eps
    within(mean, mu[:, 0], merr[:, 0] + 1e-45)
    within(rstd, r[:, 0], rerr[:, 0])
    want = c * r * w.double() + b.double()
    err = w.double().abs() * (cerr * r + c.abs() * rerr + 2 * E * c.abs() * r) + E * want.abs()
    within(y, want, err + U[kind] * (want.abs() + err) + 1e-7 * (kind == "f16"))
    plain = ctx.layer_norm(x, eps=eps)
    err = cerr * r + c.abs() * rerr + 2 * E * c.abs() * r
    within(plain, c * r, err + U[kind] * ((c * r).abs() + err) + 1e-7 * (kind == "f16"))


def norm_backward64(dy, x, mean, rstd, w, res):
    r = rstd.double()[:, None]
    h = (x.double() - mean.double()[:, None]) * r
    t = dy.double() * w.double()
    a1, a2 = t.mean(1, keepdim=True), (t * h).mean(1, keepdim=True)
    dx = r * (t - a1 - h * a2) + (0 if res is None else res.double())
    # per value: t and h to 3 roundings, the two means to 46 of the absolute terms, then the expression's own four
    err = r * (4 * E * t.abs() + 50 * E * t.abs().mean(1, keepdim=True) + 54 * E * h.abs() * (t * h).abs().mean(1, keepdim=True)) + 8 * E * (
        r * (t.abs() + a1.abs() + (h * a2).abs()) + (0 if res is None else res.double().abs()))
    # columns: a workgroup's threads add at most rows / 256 + 4 rows, then 16 groups, then at most 1024 / 16 + 16 partial sums
    n = dy.shape[0] / 256 + 4 + 16 + 80 + 4
    dg, db = dy.double() * h, dy.double()
    return dx, err, dg.sum(0), n * E * dg.abs().sum(0), db.sum(0), n * E * db.abs().sum(0)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows,d", NORMS)
def test_layer_norm_backward(ctx, rows, d, kind, residual):
    x, w, b, dy, res = norm_inputs(rows, d, kind, 1)
    res = res if residual else None
    _, mean, rstd = ctx.layer_norm(x, w, b, want_stats=True)
    dx, dw, db = ctx.layer_norm_backward(dy, x, mean, rstd, w, residual=res)
    tiny = 1e-7 * (kind == "f16") + 1e-40
    for got, want, err in zip((dx, dw, db), *[iter(norm_backward64(dy, x, mean, rstd, w, res)[i::2]) for i in (0, 1)]):
        within(got, want, err + U[kind] * (want.abs() + err) + tiny)
    only = ctx.layer_norm_backward(dy, x, mean, rstd, w, residual=res, want_dweight=False, want_dbias=False)
    assert only[1] is None and only[2] is None and torch.equal(only[0], dx)
    none, dw2, db2 = ctx.layer_norm_backward(dy, x, mean, rstd, w, want_dx=False)
    assert none is None and torch.equal(dw2, dw) and torch.equal(db2, db)
    dx1, _, _ = ctx.layer_norm_backward(dy, x, mean, rstd)
    want, err = norm_backward64(dy, x, mean, rstd, torch.ones_like(w), None)[:2]
    within(dx1, want, err + U[kind] * (want.abs() + err) + tiny)


@pytest.mark.parametrize("rows,d", [(6, 20), (40, 300), (3, 3000)])
def test_layer_norm_gradient_against_differences(ctx, rows, d):
    x, w, b, dy, _ = norm_inputs(rows, d, "f32", 2)
    _, mean, rstd = ctx.layer_norm(x, w, b, want_stats=True)
    grads = ctx.layer_norm_backward(dy, x, mean, rstd, w)
    args = [x.double(), w.double(), b.double()]
    loss = lambda a: (torch.nn.functional.layer_norm(a[0], (d,), a[1], a[2], 1e-5) * dy.double()).sum()
    h = 1e-4
    g = gen(rows, d)
    for i, grad in enumerate(grads):
        v = torch.randn(args[i].shape, generator=g, device=DEV, dtype=torch.float64)
        v /= v.norm()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * v, args[i] - h * v
        slope = ((loss(up) - loss(down)) / (2 * h)).item()
        assert abs(slope - (grad.double() * v).sum().item()) <= 2e-5 * grad.double().norm().item() + 1e-6


def test_layer_norm_rows_anywhere(ctx):
    x, w, b, dy, res = norm_inputs(37, 201, "bf16", 3)
    want, mean, rstd = ctx.layer_norm(x, w, b, want_stats=True)
    wide = torch.full((39, 211), 9.0, device=DEV, dtype=torch.bfloat16)
    src = wide.clone()
    src[1:-1, 5:206] = x
    y = ctx.layer_norm(src[1:-1, 5:206], w, b, out=wide[1:-1, 3:204])
    assert torch.equal(y, want)
    wide[1:-1, 3:204] = 9.0
    assert (wide == 9.0).all()
    grads = ctx.layer_norm_backward(dy, x, mean, rstd, w, residual=res)
    for a, b_ in zip(grads, ctx.layer_norm_backward(dy.t().contiguous().t(), src[1:-1, 5:206], mean, rstd, w, residual=res)):
        assert torch.equal(a, b_)
    assert torch.equal(ctx.layer_norm(x.reshape(37, 1, 201), w, b)[:, 0], want)
    assert torch.equal(ctx.layer_norm(x[3], w, b), want[3])
    one = x[:1].expand(37, 201)
    assert torch.equal(ctx.layer_norm(one, w, b), want[:1].expand(37, 201))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 200, 1500])
def test_layer_norm_special_rows(ctx, kind, d):
    """a row with an infinity or a NaN is NaN, its neighbours in the wave are not; constant rows give the bias"""
    x, w, b, dy, _ = norm_inputs(9, d, kind, 4)
    want = ctx.layer_norm(x, w, b)
    x[2, d // 2], x[5, d - 1], x[7] = float("inf"), float("nan"), 3.0
    y = ctx.layer_norm(x, w, b)
    assert y[2].isnan().all() and y[5].isnan().all()
    assert torch.equal(y[7], b)
    rest = [0, 1, 3, 4, 6, 8]
    assert torch.equal(y[rest], want[rest])


def block64(x, p, dy):
    leaves = [t.double().requires_grad_() for t in [x] + p]
    x, g, b, w1, b1, w2, b2 = leaves
    h = torch.nn.functional.layer_norm(x, (x.shape[-1],), g, b, 1e-5)
    y = torch.nn.functional.gelu(h @ w1 + b1) @ w2 + b2 + x
    return y.detach(), torch.autograd.grad(y, leaves, dy.double())


def block(ctx, x, p, dy):
    """a residual block over point features and its gradients, on the operators"""
    g, b, w1, b1, w2, b2 = p
    h, mean, rstd = ctx.layer_norm(x, g, b, want_stats=True)
    u, z = ctx.linear(h, w1, b1, act="gelu", want_pre=True)
    y = ctx.linear(u, w2, b2, residual=x)
    du, dw2, db2 = ctx.linear_backward(dy, u, w2)
    dh, dw1, db1 = ctx.linear_backward(du, h, w1, pre=z, act="gelu")
    dx, dg, db = ctx.layer_norm_backward(dh, x, mean, rstd, g, residual=dy)
    return y, (dx, dg, db, dw1, db1, dw2, db2)


def block_inputs(points, d, wide, kind, seed):
    g = gen(points, d, wide, kind, seed)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=DEV) * std).to(KINDS[kind])
    x = rnd(points, d)
    p = [1 + rnd(d, std=0.1), rnd(d, std=0.1), rnd(d, wide, std=d ** -0.5), rnd(wide, std=0.1), rnd(wide, d, std=wide ** -0.5), rnd(d, std=0.1)]
    return x, p, rnd(points, d)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("points,d,wide", [(1, 64, 128), (777, 96, 200), (5000, 256, 512)])
def test_residual_block(ctx, points, d, wide, kind):
    x, p, dy = block_inputs(points, d, wide, kind, 0)
    y, grads = block(ctx, x, p, dy)
    want, wants = block64(x, p, dy)
    # relative to the norm: seven tensors in a row are rounded to the type (half a step each, amplified at most 2 times in
    # all by layers whose gain is about 1), float32 sums of at most 5000 terms stay below 5000 E
    tol = 7 * 2 * U[kind] + 2 * 5000 * E
    for a, b in zip((y,) + grads, (want,) + wants):
        assert (a.double() - b).norm() <= tol * b.norm()


def test_inside_an_autograd_function(ctx):
    """the two halves of a layer behind torch's own gradients; y serves as the backward pass's z"""
    class Dense(torch.autograd.Function):
        @staticmethod
        def forward(c, x, w, b):
            y = ctx.linear(x, w, b, act="relu")
            c.save_for_backward(x, w, y)
            return y

        @staticmethod
        def backward(c, dy):
            x, w, y = c.saved_tensors
            return ctx.linear_backward(dy, x, w, pre=y, act="relu")

    g = gen(12)
    x, w, b = (ints(g, "f32", *s).requires_grad_() for s in ((2, 50, 70), (70, 33), (33,)))
    Dense.apply(x, w, b).sum().backward()                  # the gradient of a sum arrives as one value, expanded
    got = [t.grad for t in (x, w, b)]
    leaves = [t.detach().double().requires_grad_() for t in (x, w, b)]
    torch.relu(leaves[0] @ leaves[1] + leaves[2]).sum().backward()
    for a, want in zip(got, leaves):
        same(a, want.grad)


def test_same_bits_every_time(ctx):
    for kind in KINDS:
        x, p, dy = block_inputs(3000, 256, 300, kind, 1)
        y, grads = block(ctx, x, p, dy)
        y2, grads2 = block(ctx, x, p, dy)
        assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_captured_and_replayed(ctx, kind):
    """two graphs of one context, replayed in turn on two streams at once with eager calls between, against eager results"""
    sets = [block_inputs(pts, 256, 320, kind, s) for pts, s in ((3000, 2), (40, 3))]
    wants = [block(ctx, *s) for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(ctx, *s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block(ctx, *s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for y, grads in outs:
            for t in (y,) + grads:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        if turn % 2:
            eager = block(ctx, *sets[0])
            assert torch.equal(eager[0], wants[0][0])
        torch.cuda.synchronize()
        for (y, grads), (wy, wgrads) in zip(outs, wants):
            assert torch.equal(y, wy) and all(torch.equal(a, b) for a, b in zip(grads, wgrads)), "replay %d" % turn


def test_calls_on_two_streams(ctx):
    sets = [block_inputs(2000, 256, 300, "bf16", s) for s in (4, 5)]
    wants = [block(ctx, *s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], {0: [], 1: []}
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(block(ctx, *sets[i]))
    torch.cuda.synchronize()
    for i, want in enumerate(wants):
        for y, grads in got[i]:
            assert torch.equal(y, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[1]))


def test_more_than_2_31_values(ctx):
    """offsets beyond 32 bits, in rows and in columns"""
    m, k, n = 2_100_100, 1024, 8
    g = gen(8)
    x = torch.zeros(m, k, device=DEV, dtype=torch.bfloat16)
    x[-300:] = ints(g, "bf16", 300, k)
    x[:300] = ints(g, "bf16", 300, k)
    w, dy = ints(g, "bf16", k, n), ints(g, "bf16", m, n, top=1)
    y = ctx.linear(x, w)
    same(y[-300:], x[-300:].double() @ w.double())
    same(y[:300], x[:300].double() @ w.double())
    assert (y[300:-300] == 0).all()
    dx, dw, db = ctx.linear_backward(dy, x, w)
    same(dx[-300:], dy[-300:].double() @ w.double().t())
    same(dw, x[:300].double().t() @ dy[:300].double() + x[-300:].double().t() @ dy[-300:].double())
    same(db, dy.double().sum(0))
    del dx
    z, mean, rstd = ctx.layer_norm(x, want_stats=True)
    want, wmean, wrstd = ctx.layer_norm(x[-300:].clone(), want_stats=True)
    assert torch.equal(z[-300:], want) and torch.equal(mean[-300:], wmean) and torch.equal(rstd[-300:], wrstd)
    del z
    dx, _, _ = ctx.layer_norm_backward(x, x, mean, rstd)
    assert torch.equal(dx[-300:], ctx.layer_norm_backward(x[-300:].clone(), x[-300:].clone(), wmean, wrstd)[0])


def test_camera_heads_on_the_dense_layer(ctx):
    w = camera.random_weights(seed=5)
    emb = torch.randn(24, 1024, generator=gen(9), device=DEV)
    got, want = camera.pred_trans_mat(emb, w, ctx=ctx), camera.pred_trans_mat(emb.double().cpu().float(), w)
    # three float32 layers of at most 1024 terms, a rotation (norm 1) and a product with intrinsics of up to 150
    assert np.allclose(got.cpu().numpy(), want.numpy(), rtol=1e-4, atol=1e-3)


# ---- refusals ---------------------------------------------------------------------------------------------------------
def test_refusals_of_tensors(ctx):
    x, w = torch.ones(4, 8, device=DEV), torch.ones(8, 6, device=DEV)
    with pytest.raises(api.DisnError, match="on cuda"):
        ctx.linear(x.cpu(), w)
    with pytest.raises(api.DisnError, match="must be a torch.float32"):
        ctx.linear(x, w.half())
    with pytest.raises(api.DisnError, match="expected \\(4, 6\\)"):
        ctx.linear(x, w, residual=torch.ones(4, 5, device=DEV))
    buf = torch.ones(4, 20, device=DEV)
    for out in (x[:, :6], buf[:, 2:8]):
        with pytest.raises(api.DisnError, match="overlaps"):
            ctx.linear(buf[:, :8] if out.data_ptr() != x.data_ptr() else x, w, out=out)
    with pytest.raises(api.DisnError, match="overlaps"):
        ctx.linear(x, w, residual=buf[:, 1:7], out=buf[:, :6])
    with pytest.raises(api.DisnError, match="rows must be contiguous"):
        ctx.linear(x, w, out=torch.ones(6, 4, device=DEV).t())
    assert ctx.linear(buf[:, :8], w, out=buf[:, 8:14]).sum() == 4 * 6 * 8     # other columns of the same rows: no overlap
    with pytest.raises(api.DisnError, match="overlaps"):
        ctx.layer_norm(x, out=x)


def test_refusals_of_sizes(ctx):
    import ctypes
    lib, h, n = _lib.load(), ctx._h, ctypes.c_size_t()
    p = torch.ones(64, device=DEV).data_ptr()
    top = 1 << 22
    for big in (dict(k=top + 1, ldx=top + 1), dict(n=top + 1, ldw=top + 1, ldy=top + 1), dict(m=(1 << 30) + 1)):
        a = _lib.DisnLinear(1, 0, 0, 0, 4, 8, 8, p, 64, p, 64, None, None, 0, p, 64, None, 0)
        b = _lib.DisnLinearGrad(1, 0, 0, 0, 4, 8, 8, p, 64, p, 64, p, 64, None, 0, None, 0, None, 0, p)
        for key, v in big.items():
            setattr(a, key, v)
            setattr(b, key.replace("ldy", "lddy"), v)
        assert lib.disn_linear_workspace(h, ctypes.byref(a), ctypes.byref(n)) == -1 and b"sizes" in lib.disn_last_error(h)
        assert lib.disn_linear(h, ctypes.byref(a), None, 0, None) == -1 and b"sizes" in lib.disn_last_error(h)
        assert lib.disn_linear_backward_workspace(h, ctypes.byref(b), ctypes.byref(n)) == -1 and b"sizes" in lib.disn_last_error(h)
        assert lib.disn_linear_backward(h, ctypes.byref(b), None, 0, None) == -1 and b"sizes" in lib.disn_last_error(h)


def test_refusals_of_the_c_abi(ctx):
    """every refusal is made on the host, before anything is launched"""
    import ctypes
    t = torch.ones(64, 64, device=DEV)
    p = t.data_ptr()
    lib, h = _lib.load(), ctx._h
    n = ctypes.c_size_t()

    def linear(ws=None, size=0, **kw):
        a = _lib.DisnLinear(0, 0, 0, 0, 4, 8, 8, p, 64, p + 4096, 64, None, None, 0, p + 8192, 64, None, 0)
        for key, v in kw.items():
            setattr(a, key, v)
        return lib.disn_linear(h, ctypes.byref(a), ws, size, None), lib.disn_linear_workspace(h, ctypes.byref(a), ctypes.byref(n))

    assert linear() == (0, 0) and n.value == 0
    for bad in (dict(type=3), dict(act=4), dict(act=-1), dict(w_nk=2), dict(reserved=1), dict(m=-1), dict(k=(1 << 30) + 1), dict(x=None),
                dict(w=None), dict(y=None), dict(x=p + 2), dict(bias=p + 1), dict(ldx=7), dict(ldx=-8), dict(ldy=0), dict(ldy=7),
                dict(ldw=(1 << 31) + 1), dict(residual=p, ldr=3), dict(pre=p, ldp=1)):
        assert linear(**bad) == (-1, -1), bad
        assert b"disn_linear" in lib.disn_last_error(h)
    assert lib.disn_linear(h, None, None, 0, None) == -1 and lib.disn_linear(None, None, None, 0, None) == -1
    for k in (2000, 20000):   # a sum long enough to be split
        big = torch.ones(300, k, device=DEV)
        a = _lib.DisnLinear(0, 0, 0, 0, 300, 300, k, big.data_ptr(), k, big.data_ptr(), 300, None, None, 0, p, 300, None, 0)
        assert lib.disn_linear_workspace(h, ctypes.byref(a), ctypes.byref(n)) == 0
    assert n.value > 0
    ws = torch.empty(n.value + 16, dtype=torch.uint8, device=DEV)
    for ptr, size in ((None, 0), (ws.data_ptr(), n.value - 1), (ws.data_ptr() + 8, n.value)):
        assert lib.disn_linear(h, ctypes.byref(a), ptr, size, None) == -1
        assert b"workspace" in lib.disn_last_error(h)

    def grad(**kw):
        a = _lib.DisnLinearGrad(0, 1, 0, 0, 4, 8, 8, p, 64, p, 64, p, 64, p, 64, None, 0, None, 0, None)
        for key, v in kw.items():
            setattr(a, key, v)
        return lib.disn_linear_backward(h, ctypes.byref(a), None, 0, None)

    for bad in (dict(type=-1), dict(act=9), dict(pre=None), dict(act=0), dict(dy=None), dict(dx=p, lddx=2), dict(dx=p, lddx=64, w=None),
                dict(dw=p, lddw=64, x=None), dict(dw=p, lddw=0), dict(db=p + 2), dict(n=-1)):
        assert grad(**bad) == -1, bad

    def norm(**kw):
        a = _lib.DisnLayerNorm(0, 0, 4, 8, p, 64, None, None, 1e-5, p + 8192, 64, None, None)
        for key, v in kw.items():
            setattr(a, key, v)
        return lib.disn_layer_norm(h, ctypes.byref(a), None)

    assert norm() == 0
    for bad in (dict(type=3), dict(d=0), dict(d=8193), dict(rows=-1), dict(eps=-1e-5), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=None),
                dict(ldx=3), dict(ldy=3), dict(y=None), dict(weight=p + 1), dict(mean=p + 2)):
        assert norm(**bad) == -1, bad

    def norm_grad(**kw):
        a = _lib.DisnLayerNormGrad(0, 0, 4, 8, p, 64, p, 64, p, p, None, None, 0, None, 0, None, None)
        for key, v in kw.items():
            setattr(a, key, v)
        return lib.disn_layer_norm_backward(h, ctypes.byref(a), None, 0, None)

    assert norm_grad() == 0
    for bad in (dict(type=3), dict(d=0), dict(mean=None), dict(rstd=None), dict(dy=None), dict(x=None), dict(residual=p, ldr=3), dict(dx=p, lddx=0)):
        assert norm_grad(**bad) == -1, bad
    torch.cuda.synchronize()
