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
