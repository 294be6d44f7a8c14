"""CPU tests of what autograd sees of the row tables' calls (horizongs_amd.embedding, horizongs_amd.rowcache).

The native entries are replaced by their formulas on host memory; what is tested is the Python boundary
around them."""
import pytest
import torch
from torch.autograd import forward_ad

from horizongs_amd import embedding as E
from horizongs_amd import rowcache as R
from tests import rows_on_host


@pytest.fixture(autouse=True)
def on_the_host(monkeypatch):
    rows_on_host.install(monkeypatch)


IDS = torch.tensor([2, 0, 2])


def table(V=4, D=3):
    return torch.arange(float(V * D)).reshape(V, D)


def test_forward_mode_is_refused_not_dropped():
    """A dual tensor's primal needs no gradient; its tangent must not get lost on the way."""
    w, g = table(), torch.ones(3, 3)
    with forward_ad.dual_level():
        dw, dg = forward_ad.make_dual(w, torch.ones_like(w)), forward_ad.make_dual(g, torch.ones_like(g))
        for call in (lambda: E.embedding(dw, IDS, 2.0), lambda: E.embedding_grad(dg, IDS, 4),
                     lambda: E.embedding_grad(dg, IDS, 4, out=table()), lambda: E.embedding_grad(g, IDS, 4, out=dw)):
            with pytest.raises(NotImplementedError, match="jvp|forward mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp|forward mode"):
                call()
        # a backward pass along a dual gradient
        p = table().requires_grad_(True)
        with pytest.raises(NotImplementedError, match="jvp"):
            torch.autograd.grad(E.embedding(p, IDS), p, dg)
        q = g.clone().requires_grad_(True)
        with pytest.raises(NotImplementedError, match="jvp"):
            torch.autograd.grad(E.embedding_grad(q, IDS, 4), q, dw)
        # tensors without a tangent, at the same level
        assert torch.equal(E.embedding(w, IDS, 2.0), 2 * w[IDS])
        out = E.embedding_grad(g, IDS, 4, out=table())
        assert torch.equal(E.embedding_grad(g, IDS, 4) + w, out)
    assert torch.equal(E.embedding(w, IDS, 2.0), 2 * w[IDS])


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("grad", [False, True])
def test_traces_are_refused(grad):
    """A trace would hold the new tensor and not the call that fills it."""
    w, g = table().requires_grad_(grad), torch.ones(3, 3, requires_grad=grad)
    c, t = R.rowcache_alloc(4, 3, device="cpu"), table()
    for call in (lambda w, g, i: E.embedding(w, i), lambda w, g, i: E.embedding_grad(g, i, 4),
                 lambda w, g, i: E.embedding_grad(g.detach(), i, 4, out=t), lambda w, g, i: R.rowcache_read(c, i),
                 lambda w, g, i: (R.rowcache_write(c, g, i), g)[1]):
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(call, (w, g, IDS), check_trace=False)
    assert not c.scales.any() and torch.equal(t, table())


def test_sums_added_to_a_saved_table_are_seen():
    """A backward pass that saved the table as it was refuses to go on with the changed one."""
    for view in (lambda t: t, lambda t: t[1:3]):
        base = table(6, 3)
        p = torch.ones_like(base, requires_grad=True)
        y = (p * base).sum()
        E.embedding_grad(torch.empty(0, 3), IDS[:0], view(base).shape[0], out=view(base))
        assert base._version == 0  # no rows: nothing was added
        t = view(base)
        E.embedding_grad(torch.ones(2, 3), torch.tensor([1, 1]), t.shape[0], out=t)
        assert t._version == base._version == 1
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    with torch.inference_mode():
        t = table()
        E.embedding_grad(torch.ones(3, 3), IDS, 4, out=t)
    E.embedding_grad(torch.ones(3, 3), IDS, 4, out=t)  # an inference tensor has no version
    assert float(t[2, 0]) == 6 + 4
    leaf = table().requires_grad_(True)  # the documented way to a leaf
    y = leaf.square().sum()
    with torch.no_grad():
        E.embedding_grad(torch.ones(3, 3), IDS, 4, out=leaf)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_writes_to_a_saved_cache_are_seen():
    c = R.rowcache_alloc(4, 3, device="cpu")
    p = torch.ones(4, 1, requires_grad=True)
    before = c.codes._version, c.scales._version
    R.rowcache_write(c, torch.empty(0, 3), IDS[:0])
    assert (c.codes._version, c.scales._version) == before
    for saved in (c.scales, c.codes):
        y = (p * saved).sum()
        R.rowcache_write(c, torch.ones(3, 3), IDS)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    before = c.codes._version, c.scales._version
    assert torch.equal(R.rowcache_read(c, IDS), torch.ones(3, 3))
    assert (c.codes._version, c.scales._version) == before


@pytest.mark.parametrize("shape", [(), (3,), (2, 3), (0,), (2, 0), (0, 2)])
@pytest.mark.parametrize("D", [0, 1, 3])
def test_gradients_of_every_shape(shape, D):
    """Tables without columns, no ids, ids of any number of dimensions: forward, backward, second derivative."""
    V = 4
    ids = torch.randint(0, V, shape)
    w = torch.randn(V, D, requires_grad=True)
    y = E.embedding(w, ids, 2.0)
    assert y.shape == (*shape, D)
    g = torch.randn(*shape, D)
    (dw,) = torch.autograd.grad(y, w, g)
    v = w.detach().clone().requires_grad_(True)
    (want,) = torch.autograd.grad(2.0 * v[ids], v, g)
    assert torch.allclose(dw, want) and dw.shape == (V, D)
    assert torch.equal(E.embedding_grad(g, ids, V, 2.0), dw)
    assert torch.equal(E.embedding_grad(g, ids, V, 2.0, out=torch.zeros(V, D)), dw)
    q = g.clone().requires_grad_(True)
    (dq,) = torch.autograd.grad(E.embedding_grad(q, ids, V, 2.0), q, w.detach())
    assert torch.equal(dq, y.detach())
    (x,) = torch.autograd.grad(E.embedding(w, ids).square().sum(), w, create_graph=True)
    (xx,) = torch.autograd.grad(x, w, torch.ones_like(w))
    assert torch.allclose(xx, 2.0 * torch.bincount(ids.reshape(-1), minlength=V)[:, None].expand(V, D).float())
