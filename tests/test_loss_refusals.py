"""What the soft assignment and the losses over it refuse, without a GPU: the C entry points by their error codes (before any
device call), the Python ones by their exceptions."""
import importlib

import pytest
import torch

ARG, WORKSPACE = 1, 3


@pytest.fixture(scope="module")
def h():
    return importlib.import_module("gan-discovery-pso_amd._lib").lib()


@pytest.fixture()
def eng(monkeypatch):
    module = importlib.import_module("gan-discovery-pso_amd.engine")
    monkeypatch.setattr(module, "_device_guard", torch.device)  # let the argument checks see CPU tensors
    monkeypatch.setattr(module._lib, "lib", lambda: pytest.fail("reached the library"))
    return module


def test_workspaces(h):
    assert h.gdpso_balance_workspace_bytes(-1, 4) == h.gdpso_balance_workspace_bytes(4, 0) == 0
    assert h.gdpso_balance_workspace_bytes(0, 4) > 0
    assert h.gdpso_code_logits_grad_workspace_bytes(0, 4, 4) == 0
    assert h.gdpso_code_logits_grad_workspace_bytes(5, 3, 4) == 0  # one split needs none
    assert h.gdpso_code_logits_grad_workspace_bytes(5000, 3, 4) >= 2 * 4 * 4 * 4


def test_code_logits_refusals(h):
    P = 64  # a pointer that nothing may follow
    ok = dict(n=4, d=8, k=3, x=P, c=P, dt=0, t=1.0, out=P)

    def call(**kw):
        a = {**ok, **kw}
        return h.gdpso_code_logits(None, a["n"], a["d"], a["k"], a["x"], a["c"], a["dt"], a["t"], a["out"])

    for bad in (dict(n=-1), dict(d=0), dict(d=4097), dict(k=0), dict(k=2 ** 20 + 1), dict(dt=3), dict(t=0.0), dict(t=-1.0), dict(t=float("nan")),
                dict(t=float("inf")), dict(x=None), dict(c=None), dict(out=None)):
        assert call(**bad) == ARG, bad
    assert call(n=0, x=None, out=None) == 0
    ws = h.gdpso_code_logits_grad_workspace_bytes(5000, 8, 3)

    def grad(n=5000, d=8, k=3, g=P, x=P, c=P, dt=0, t=1.0, dx=P, dc=P, w=P, wb=ws):
        return h.gdpso_code_logits_grad(None, n, d, k, g, x, c, dt, t, dx, dc, w, wb)

    for bad in (dict(n=-1), dict(d=0), dict(k=0), dict(dt=-1), dict(t=0.0), dict(g=None), dict(x=None), dict(c=None), dict(w=None)):
        assert grad(**bad) == ARG, bad
    assert grad(wb=ws - 1) == WORKSPACE


def test_balance_refusals(h):
    P = 64
    ws = h.gdpso_balance_workspace_bytes(4, 8)

    def call(n=4, e=8, k=2, s=P, stride=8, dt=0, i=P, ib=8, loss=P, counts=P, totals=P, mean=P, w=P, wb=ws):
        return h.gdpso_balance(None, n, e, k, s, stride, dt, i, ib, None, 1.0, loss, counts, totals, mean, None, w, wb)

    for bad in (dict(n=-1), dict(e=0), dict(e=16385, wb=2 ** 40), dict(k=0), dict(s=None), dict(stride=-1), dict(dt=3), dict(i=None), dict(ib=2), dict(loss=None),
                dict(counts=None), dict(totals=None), dict(mean=None), dict(w=None)):
        assert call(**bad) == ARG, bad
    assert call(wb=ws - 1) == WORKSPACE
    for bad in ((-1, 8, P, 8, 0), (4, 0, P, 8, 0), (4, 8, None, 8, 0), (4, 8, P, -8, 0), (4, 8, P, 8, 7)):
        assert h.gdpso_balance_grad(None, *bad, None, P, P, P, P) == ARG, bad
    assert h.gdpso_balance_grad(None, 4, 8, P, 8, 0, None, P, P, None, P) == ARG
    assert h.gdpso_balance_grad(None, 0, 8, None, 8, 0, None, None, None, None, None) == 0


def test_distill_refusals(h):
    P = 64
    ws = h.gdpso_distill_workspace_bytes(4, 8, 2)

    def call(n=4, v=8, k=2, s=P, stride=8, dt=0, t=P, tdt=0, i=P, ib=8, temp=1.0, loss=P, row=P, stats=P, w=P, wb=ws):
        return h.gdpso_distill(None, n, v, k, s, stride, dt, t, tdt, i, ib, None, temp, 1.0, loss, row, stats, None, w, wb)

    for bad in (dict(n=-1), dict(v=0), dict(k=0), dict(k=1025), dict(s=None), dict(stride=-1), dict(dt=3), dict(tdt=3), dict(t=None), dict(i=None), dict(ib=1),
                dict(temp=0.0), dict(temp=-2.0), dict(temp=float("nan")), dict(temp=1e7), dict(loss=None), dict(row=None), dict(stats=None)):
        assert call(**bad) == ARG, bad
    assert ws == 0 or call(wb=ws - 1) == WORKSPACE
    assert h.gdpso_distill_grad(None, 4, 8, 2, P, 8, 0, P, 0, P, 8, None, 1.0, P, None, P) == ARG
    assert h.gdpso_distill_grad(None, 4, 8, 0, P, 8, 0, P, 0, P, 8, None, 1.0, P, P, P) == ARG
    assert h.gdpso_distill_grad(None, 0, 8, 2, None, 8, 0, None, 0, None, 8, None, 1.0, None, None, None) == 0


def test_python_code_logits(eng):
    x, c = torch.zeros(4, 8), torch.zeros(3, 8)
    for a, b in ((x, c[0]), (x[:, :7], c), (x, torch.zeros(0, 8)), (x.double(), c.double()), (x.half(), c), (torch.tensor(1.0), c)):
        with pytest.raises(ValueError):
            eng.code_logits(a, b)
    for g in (torch.zeros(4, 4), torch.zeros(4, 3, dtype=torch.float16), torch.zeros(12)):
        with pytest.raises(ValueError):
            eng.code_logits_grad(g, x, c)


def test_python_balance(eng):
    s, i = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    for a, b, m in ((s.double(), i, None), (s, i.float(), None), (s, i[:3], None), (s, i[:, :0], None), (s, i, torch.ones(4)), (s, i, torch.ones(3, dtype=torch.bool)),
                    (torch.zeros(4, 0), i, None), (torch.tensor(1.0), i, None)):
        with pytest.raises(ValueError):
            eng.balance(a, b, mask=m)
    up = torch.ones(())
    ok, two = torch.zeros(8, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)
    for counts, totals, u in ((ok[:7], two, up), (ok.float(), two, up), (ok, ok, up), (ok, two, up.double()), (ok, two, torch.ones(2))):
        with pytest.raises(ValueError):
            eng.balance_grad(s, counts, totals, u)


def test_python_sizes_beyond_int(eng):
    """Rows beyond 2^31 would wrap around in the C ABI's int (strides of 0: no memory behind them)."""
    n = 2 ** 31 + 3
    with pytest.raises(ValueError):
        eng.code_logits(torch.zeros(1, 1).expand(n, 1), torch.zeros(1, 1))
    with pytest.raises(ValueError):
        eng.balance(torch.zeros(1, 2).expand(n, 2), torch.zeros(1, dtype=torch.int64).expand(n))
    with pytest.raises(ValueError):
        eng.distill(torch.zeros(1, 2).expand(n, 2), torch.zeros(1, 1).expand(n, 1), torch.zeros(1, 1, dtype=torch.int64).expand(n, 1))


def test_python_distill(eng):
    s, t, i = torch.zeros(4, 8), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64)
    for a, b, c, m in ((s.double(), t, i, None), (s, t.double(), i, None), (s, t[:, :1], i, None), (s, t, i.short(), None), (s, t[:3], i[:3], None),
                       (s, t[:, :0], i[:, :0], None), (s, t, i, torch.ones(4, 1, dtype=torch.bool))):
        with pytest.raises(ValueError):
            eng.distill(a, b, c, mask=m)
    with pytest.raises(ValueError):
        eng.distill_grad(s, t, i, torch.zeros(8), torch.ones(()))
    with pytest.raises(ValueError):
        eng.distill_grad(s, t, i, torch.zeros(9), torch.ones(3))
