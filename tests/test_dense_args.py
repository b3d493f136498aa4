"""Dense layer and layer norm: what the wrapper makes of tensors and what it refuses, before any call into the library
(no GPU: a context that was never opened, on the CPU)."""
import pytest
import torch

from disn_amd import api


@pytest.fixture
def ctx(monkeypatch):
    c = api.Context.__new__(api.Context)
    c.device, c._index = torch.device("cpu"), -1
    c.lib = type("NoLibrary", (), {"__getattr__": lambda self, name: name})()
    monkeypatch.setattr(api.Context, "_elsewhere", lambda self: False)
    monkeypatch.setattr(api.Context, "_run", lambda *a: pytest.fail("the call should have been refused"))
    return c


def test_rows(ctx):
    t = torch.arange(120.0).reshape(6, 20)
    size = 4
    at = t.data_ptr()
    f = torch.float32
    assert ctx._rows(t, "t", f, t.shape)[1] == (at, 6, 20, 20, size)
    assert ctx._rows(t[1:4, 3:9], "t", f, (3, 6))[1] == (at + 23 * 4, 3, 6, 20, size)
    assert ctx._rows(t[2], "t", f, (20,))[1] == (t[2].data_ptr(), 1, 20, 20, size)
    assert ctx._rows(t.reshape(2, 3, 20)[:, :, :7], "t", f, (2, 3, 7))[1] == (at, 6, 7, 20, size)
    assert ctx._rows(t[:1].expand(9, 20), "t", f, (9, 20))[1] == (at, 9, 20, 0, size)
    assert ctx._rows(t[:, :1], "t", f, (6, 1))[1] == (at, 6, 1, 20, size)
    for view in (t.t(), t[:, ::2], t.reshape(2, 3, 20).transpose(0, 1), t.reshape(-1).as_strided((5, 8), (3, 1)), t.reshape(2, 3, 20)[:, :1].expand(2, 4, 20)):
        copy, m = ctx._rows(view, "t", f, view.shape)
        assert copy.is_contiguous() and torch.equal(copy, view) and m[1:4] == (view.numel() // view.shape[-1], view.shape[-1], view.shape[-1])
        with pytest.raises(api.DisnError, match="rows must be"):
            ctx._rows(view, "t", f, view.shape, copy=False)
    with pytest.raises(api.DisnError, match="rows must be"):
        ctx._rows(t[:1].expand(9, 20), "t", f, (9, 20), copy=False)


def test_weights(ctx):
    w = torch.arange(60.0).reshape(5, 12)
    f = torch.float32
    assert ctx._weight(w, "w", f)[1:] == (5, 12, 0, w.data_ptr(), 12)
    assert ctx._weight(w[:, 2:7], "w", f)[1:] == (5, 5, 0, w.data_ptr() + 8, 12)
    assert ctx._weight(w.t(), "w", f)[1:] == (12, 5, 1, w.data_ptr(), 12)
    assert ctx._weight(w[1:3, 1:9].t(), "w", f)[1:] == (8, 2, 1, w[1:, 1:].data_ptr(), 12)
    for view in (w[:, ::2], w[:1, :1].expand(5, 12), w[:1].expand(5, 12)):
        copy, _, _, nk, at, ld = ctx._weight(view, "w", f)
        assert nk == 0 and ld == view.shape[1] and torch.equal(copy, view) and at == copy.data_ptr()


def test_meet():
    row = lambda at, rows, cols, ld: (at, rows, cols, ld, 4)
    assert api._meet(row(0, 4, 8, 8), row(64, 2, 8, 8))
    assert not api._meet(row(0, 4, 8, 8), row(128, 2, 8, 8))
    assert not api._meet(row(0, 4, 8, 20), row(32, 4, 8, 20))     # columns 0..7 and 8..15 of the same rows
    assert api._meet(row(0, 4, 8, 20), row(28, 4, 8, 20))
    assert api._meet(row(32, 4, 8, 20), row(80, 4, 16, 20))       # columns 0..15 from the next row on meet 8..15
    assert not api._meet(row(32, 4, 8, 20), row(80, 4, 8, 20))
    assert api._meet(row(0, 4, 8, 20), row(32, 4, 8, 24))         # other row distances: taken to meet
    assert not api._meet(row(0, 0, 8, 8), row(0, 4, 8, 8))


@pytest.mark.parametrize("call,match", [
    (lambda c, x, w: c.linear(x.int(), w), "float32, bfloat16 or float16"),
    (lambda c, x, w: c.linear(x, w, act="tanh"), "unknown act"),
    (lambda c, x, w: c.linear(x, w.half()), "must be a torch.float32"),
    (lambda c, x, w: c.linear(x, w[0]), r"\[k, n\]"),
    (lambda c, x, w: c.linear(x, w[:5]), "expected"),
    (lambda c, x, w: c.linear(x[0, 0], w), "one dimension"),
    (lambda c, x, w: c.linear(x, w, bias=torch.zeros(4)), "bias has shape"),
    (lambda c, x, w: c.linear(x, w, bias=torch.zeros(1, 6)), "bias has shape"),
    (lambda c, x, w: c.linear(x, w, residual=torch.zeros(6)), "residual has shape"),
    (lambda c, x, w: c.linear(x, w, out=torch.zeros(4, 5)), "out has shape"),
    (lambda c, x, w: c.linear(x, w, out=torch.zeros(6, 4).t()), "rows must be"),
    (lambda c, x, w: c.linear(x, w, out=x[:, :6]), "overlaps"),
    (lambda c, x, w: c.linear(x, w, out=w[:4]), "overlaps"),
    (lambda c, x, w: c.linear(x.to_sparse(), w), "must be a"),
    (lambda c, x, w: c.linear_backward(torch.zeros(4, 6), x, w, act="relu"), "pre belongs"),
    (lambda c, x, w: c.linear_backward(torch.zeros(4, 6), x, w, pre=torch.zeros(4, 6)), "pre belongs"),
    (lambda c, x, w: c.linear_backward(torch.zeros(4, 5), x, w), "w has shape"),
    (lambda c, x, w: c.linear_backward(torch.zeros(4, 6), x[:3], w), "x has shape"),
    (lambda c, x, w: c.linear_backward(torch.zeros(4, 6), None, w), "dw needs x"),
    (lambda c, x, w: c.linear_backward(torch.zeros(4, 6), x, None), "dx needs w"),
    (lambda c, x, w: c.layer_norm(x, weight=torch.zeros(6)), "weight has shape"),
    (lambda c, x, w: c.layer_norm(x, out=x), "overlaps"),
    (lambda c, x, w: c.layer_norm_backward(x, x, torch.zeros(3), torch.zeros(4)), "mean has shape"),
    (lambda c, x, w: c.layer_norm_backward(x, x, torch.zeros(4), torch.zeros(4).half()), "rstd must be"),
    (lambda c, x, w: c.layer_norm_backward(x, x[:3], torch.zeros(4), torch.zeros(4)), "x has shape"),
    (lambda c, x, w: c.layer_norm_backward(x, x, torch.zeros(4), torch.zeros(4), residual=x[0]), "residual has shape"),
])
def test_refusals(ctx, call, match):
    with pytest.raises(api.DisnError, match=match):
        call(ctx, torch.zeros(4, 8), torch.zeros(8, 6))
