"""Dense layer and layer norm at their edges: what lies beside an operand or in a workspace reaches no result; values next to
the smallest of float32; closed gates; rows of equal values."""
import ctypes

import pytest
import torch

from disn_amd import _lib, api
from test_gpu_dense import DEV, E, KINDS, U, gen, weight, within

pytestmark = pytest.mark.gpu
BESIDE = {"zeros": 0.0, "nan": float("nan"), "inf": float("inf"), "large": -1e4, "small": 2.0 ** -16}


def beside(t, what):
    """t as columns of a wider buffer whose other columns hold `what`"""
    c = t.shape[1]
    buf = torch.full((t.shape[0], c + 12), BESIDE[what], device=DEV, dtype=t.dtype)
    if what == "small" and t.dtype is torch.float32:
        buf.fill_(2.0 ** -140)
    buf[:, 4:4 + c] = t
    return buf[:, 4:4 + c]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("wide", [128, 129, 257, 258, 259, 385, 513])
def test_columns_beside_an_operand(ctx, wide, kind):
    """a last tile of one to three columns, sums of whole stages: the same bits whatever the neighbouring columns hold"""
    g = gen(wide, kind, "beside")
    m, k = 9008, 1024
    x, w, dy = (torch.randn(*s, generator=g, device=DEV).to(KINDS[kind]) for s in ((m, k), (k, wide), (m, wide)))
    narrow, wn, dyn = (torch.randn(*s, generator=g, device=DEV).to(KINDS[kind]) for s in ((m, wide), (wide, 520), (m, 520)))
    first = None
    for what in BESIDE:
        got = (ctx.linear(x, beside(w, what)),) + ctx.linear_backward(beside(dy, what), x, beside(w, what))
        got += ctx.linear_backward(dyn, beside(narrow, what), beside(wn, what))
        got += ctx.linear_backward(dyn, beside(narrow, what), beside(wn.t().contiguous(), what).t())
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first)), what
    y = first[0]
    bound = 2 * (k + 4) * E * (x.double().abs() @ w.double().abs())
    want = x.double() @ w.double()
    within(y, want, bound + U[kind] * (want.abs() + bound) + 1e-7 * (kind == "f16"))


WORKSPACES = {"zeros": 0, "ones": -1, "subnormal": 0x00000401, "inf": 0x7f800000, "inf16": 0x7c007f80, "large": 0x7e967699}


@pytest.mark.parametrize("w_nk", [0, 1])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", [(4096, 515, 257), (4099, 512, 258), (5008, 300, 259), (6000, 1024, 513), (600, 70, 50)])
def test_contents_of_the_workspace(ctx, m, k, n, kind, w_nk):
    """the same bits whatever the workspace holds before the call"""
    g = gen(m, k, n, kind, w_nk, "workspace")
    t = KINDS[kind]
    x, w, dy, pre = (torch.randn(*s, generator=g, device=DEV).to(t) for s in ((m, k), (n, k) if w_nk else (k, n), (m, n), (m, n)))
    lib, h, size = _lib.load(), ctx._h, ctypes.c_size_t()
    stream = torch.cuda.current_stream().cuda_stream
    first = None
    for what, bits in WORKSPACES.items():
        dx, dw, db = torch.empty(m, k, device=DEV, dtype=t), torch.empty_like(w), torch.empty(n, device=DEV, dtype=t)
        a = _lib.DisnLinearGrad(api.TYPES[t], api.ACTS["silu"], w_nk, 0, m, n, k, dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), w.shape[1],
                                pre.data_ptr(), n, dx.data_ptr(), k, dw.data_ptr(), w.shape[1], db.data_ptr())
        assert lib.disn_linear_backward_workspace(h, ctypes.byref(a), ctypes.byref(size)) == 0
        assert size.value or m == 600
        ws = torch.full((size.value // 4 + 4,), bits, device=DEV, dtype=torch.int32)
        assert lib.disn_linear_backward(h, ctypes.byref(a), ws.data_ptr(), size.value, stream) == 0
        assert (ws[-3:] == bits).all()
        first = first or (dx, dw, db)
        assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), first)), what
    assert all(v.isfinite().all() for v in first)


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("xs,ws", [(-140, 20), (-140, 30), (-138, 8), (-136, 0), (30, -141), (-149, 12), (-107, 3), (-104, 80), (-111, 60)])
@pytest.mark.parametrize("m,k,n", [(300, 700, 800), (3000, 900, 1100), (3000, 512, 1100), (40000, 200, 260)])
def test_float32_values_below_the_terms(ctx, m, k, n, xs, ws, layout):
    """values that the first or the last of three narrower terms cannot hold, with others that lift their products into the range"""
    g = gen(m, k, n, xs, ws, "terms")
    x = (torch.randn(m, k, generator=g, device=DEV).double() * 2.0 ** xs).float()
    w = (torch.randn(k, n, generator=g, device=DEV).double() * 2.0 ** ws).float()
    # (k + 4) roundings as everywhere, and six partial sums that may each be rounded to steps of 2^-149 a term
    bound = 2 * (k + 4) * E * (x.double().abs() @ w.double().abs()) + 6 * (k + 4) * 2.0 ** -149
    within(ctx.linear(x, weight(w, layout)), x.double() @ w.double(), bound)
    dy = x.repeat(1, n // k + 1)[:, :n].contiguous()
    dx, _, _ = ctx.linear_backward(dy, x, weight(w, layout))
    within(dx, dy.double() @ w.double().t(), 2 * (n + 4) * E * (dy.double().abs() @ w.double().abs().t()) + 6 * (n + 4) * 2.0 ** -149)


@pytest.mark.parametrize("m,k,n", [(300, 700, 803), (3000, 900, 1101), (40000, 200, 259)])
def test_float32_smallest_values_between_zeros(ctx, m, k, n):
    """rows and columns of nothing but zeros, next to rows that hold one value below the smallest of a narrower type"""
    g = gen(m, k, n, "one")
    x, w = torch.zeros(m, k, device=DEV), torch.randn(k, n, generator=g, device=DEV)
    at = torch.randint(0, k, (m,), generator=g, device=DEV)
    x[torch.arange(m, device=DEV), at] = 2.0 ** -140
    x[::3] = torch.randn(x[::3].shape, generator=g, device=DEV)
    x[1::6] = 0.0
    w[:, ::7] = 0.0
    w *= 2.0 ** 16
    y, want = ctx.linear(x, w), x.double() @ w.double()
    bound = 2 * (k + 4) * E * (x.double().abs() @ w.double().abs()) + 6 * (k + 4) * 2.0 ** -149
    within(y, want, bound)
    assert (y[1::6] == 0).all() and (y[:, ::7] == 0).all()
    # one product a sum: exact
    one = torch.arange(2, m, 6, device=DEV)
    assert torch.equal(y[one], want[one].float())


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("m,k,n", [(1, 5, 7), (20, 40, 30), (32, 1024, 512), (2, 2100, 3001), (3000, 900, 1100), (30000, 515, 2), (40000, 3, 70)])
def test_infinite_gradients_at_a_closed_relu(ctx, m, k, n, kind, layout):
    """what is not passed does not matter, be it an infinity or a NaN; a NaN in pre is still seen"""
    g = gen(m, k, n, kind, layout, "closed")
    x, w, dy, pre = (torch.randn(*s, generator=g, device=DEV).to(KINDS[kind]) for s in ((m, k), (k, n), (m, n), (m, n)))
    w = weight(w, layout)
    pre[0, 0], pre[m - 1, n - 1] = 0.0, -0.0
    closed = pre <= 0
    dy[closed] = 1.0
    want = ctx.linear_backward(dy, x, w, pre=pre, act="relu")
    for value in (float("inf"), float("-inf"), float("nan")):
        dy[closed] = value
        for a, b in zip(ctx.linear_backward(dy, x, w, pre=pre, act="relu"), want):
            assert torch.equal(a, b), value
        _, _, db = ctx.linear_backward(dy, None, None, pre=pre, act="relu", want_dx=False, want_dw=False)
        assert db.isfinite().all()
    dy[0, 0], pre[0, 0] = float("inf"), 1.0
    dx, dw, db = ctx.linear_backward(dy, x, w, pre=pre, act="relu")
    assert not dx[0].isfinite().any() and dx[1:].isfinite().all() and db[0] == float("inf") and db[1:].isfinite().all()
    dy[0, 0], pre[0, 0] = 1.0, float("nan")
    dx, dw, db = ctx.linear_backward(dy, x, w, pre=pre, act="relu")
    assert dx[0].isnan().all() and dx[1:].isfinite().all() and db[0].isnan() and db[1:].isfinite().all()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [3, 40, 100, 200, 500, 1000, 1024, 1500, 2048, 3001, 5000, 8192])
def test_rows_of_one_value(ctx, d, kind):
    """the mean of equal values is that value, so the row gives the bias, and without an eps 0 / 0"""
    values = torch.tensor([0.1, 0.7, -1.3, 1e-3, 12345.678, 1e30 if kind != "f16" else 3e4, 3e-39 if kind != "f16" else 3e-7, 0.0], device=DEV)
    x = values.to(KINDS[kind])[:, None].expand(-1, d).contiguous()
    g = gen(d, kind, "equal")
    w, b = (torch.randn(d, generator=g, device=DEV).to(KINDS[kind]) for _ in range(2))
    y, mean, rstd = ctx.layer_norm(x, w, b, eps=1e-5, want_stats=True)
    assert torch.equal(mean, x[:, 0].float())
    assert torch.equal(y, b.expand(len(values), d))
    assert (rstd.double() - 1e-5 ** -0.5).abs().max() <= 4 * E * 1e-5 ** -0.5
    assert ctx.layer_norm(x, w, b, eps=0.0).isnan().all()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [40, 200, 1000, 1500, 3001, 8192])
def test_rows_far_from_zero(ctx, d, kind):
    """a spread that is small beside the mean: the distances from the mean are as exact as the values allow"""
    g = gen(d, kind, "far")
    step = torch.finfo(KINDS[kind]).eps                      # of values from 1 to 2
    x = (1.5 + step * torch.randint(-9, 10, (60, d), generator=g, device=DEV)).to(KINDS[kind])
    eps = 1e-30
    y, mean, rstd = ctx.layer_norm(x, eps=eps, want_stats=True)
    mu = x.double().mean(1, keepdim=True)
    c = x.double() - mu
    r = (c * c).mean(1, keepdim=True) ** -0.5
    within(mean, mu[:, 0], 2 * E * mu[:, 0])                 # a rounded value, corrected once and rounded again
    # c is off by the mean's rounding, half a step of 2^-23 at most, in every value alike
    err = 2 * 2 * E * r * (1 + (c * r).abs()) + 60 * E * (c * r).abs()
    within(y, c * r, err + U[kind] * ((c * r).abs() + err) + 1e-7 * (kind == "f16"))


def test_gelu_of_float32(ctx):
    """gelu and its slope where most values lie, to the roundings of a few operations (one input, a weight of 1: z is x)"""
    g = gen("gelu")
    z = torch.rand(60000, 1, generator=g, device=DEV) * 2.4 - 1.2
    one = torch.ones(1, 1, device=DEV)
    wide = z.double()
    cdf, density = 0.5 * torch.special.erfc(-wide / 2 ** 0.5), torch.exp(-wide * wide / 2) / (2 * torch.pi) ** 0.5
    # cdf = 0.5 + z R(z^2): R to 2.5 roundings of its value, the sum rounded once; the product with z once more
    cdferr = E * (cdf + 2.5 * (cdf - 0.5).abs())
    within(ctx.linear(z, one, act="gelu"), wide * cdf, wide.abs() * (cdferr + E * cdf) + 1e-44)
    # z times the density: a product, the exponential's argument (two roundings of at most 1.04) and its own step: 5 in all
    want = cdf + wide * density
    dx, _, _ = ctx.linear_backward(torch.ones_like(z), z, one, pre=z, act="gelu")
    within(dx, want, cdferr + 5 * E * (wide * density).abs() + E * want.abs())


def test_silu_of_float32(ctx):
    """silu and its slope over the whole range of their exponential, to the roundings of a few operations"""
    g = gen("silu")
    z = torch.cat([torch.rand(60000, 1, generator=g, device=DEV) * 110 - 80, torch.randn(20000, 1, generator=g, device=DEV)])
    one = torch.ones(1, 1, device=DEV)
    wide = z.double()
    s = torch.sigmoid(wide)
    # the exponential and the reciprocal to a step (2 E) each, three roundings of s, one of the product
    within(ctx.linear(z, one, act="silu"), wide * s, 8 * E * (wide * s).abs() + 1e-36)
    # s (1 + z (1 - s)): s to 7 E, 1 - s to 7 E s + E, two roundings of the sum, one of the product
    want = s * (1 + wide * (1 - s))
    dx, _, _ = ctx.linear_backward(torch.ones_like(z), z, one, pre=z, act="silu")
    within(dx, want, E * (8 * want.abs() + s * (2 + wide.abs() * (7 * s + 3 * (1 - s)))) + 1e-36)
    big = torch.tensor([[-1e30], [-200.0], [-100.0], [100.0], [1e30], [float("inf")], [float("nan")]], device=DEV)
    y = ctx.linear(big, one, act="silu")[:, 0]
    assert (y[:3].abs() <= 1e-36).all() and torch.equal(y[3:6], big[3:6, 0]) and y[6].isnan()
