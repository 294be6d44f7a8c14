"""GPU checks of the row tables where their calls meet the rest: autograd's counters, streams, empty and odd arguments
of the decode."""
import pytest
import torch
from torch.autograd import forward_ad

from horizongs_amd import decode as HD
from horizongs_amd import embedding as E
from horizongs_amd import rowcache as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def test_autograd_sees_every_call():
    w, ids = torch.randn(9, 32, device=DEV), torch.tensor([[3, 8], [3, -1]], device=DEV)
    g = torch.ones(2, 2, 32, device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(w, torch.ones_like(w))
        with pytest.raises(NotImplementedError, match="jvp"):
            E.embedding(dual, ids)
        with pytest.raises(NotImplementedError, match="forward mode"):
            E.embedding_grad(g, ids, 9, out=dual)
    c = R.rowcache_alloc(9, 32, device=DEV)
    p = torch.ones(9, 1, device=DEV, requires_grad=True)
    for saved, write in ((w, lambda: E.embedding_grad(g, ids, 9, out=w)), (c.codes, lambda: R.rowcache_write(c, w)),
                         (c.scales, lambda: R.rowcache_write(c, w[:4], ids.reshape(-1)))):
        y = (p * saved).sum()
        write()
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()


def test_tables_without_columns():
    w = torch.randn(5, 0, device=DEV, requires_grad=True)
    E.embedding(w, torch.zeros(2, 3, dtype=torch.int64, device=DEV)).sum().backward()
    assert w.grad.shape == (5, 0)


F, N_OFF, K = 32, 10, 35


def model(A):
    g = gen(A)
    r = lambda *s, sd=1.0: (torch.randn(*s, generator=g) * sd).to(DEV)
    t = [r(A, 3), r(A, F), r(A, N_OFF, 3, sd=0.1), r(A, 6, sd=0.1), r(3)]
    w = {}
    for h, o in (("opacity", N_OFF), ("cov", 7 * N_OFF), ("color", 3 * N_OFF)):
        w.update({f"{h}_w1": r(F, K, sd=0.2), f"{h}_b1": r(F), f"{h}_w2": r(o, F, sd=0.2), f"{h}_b2": r(o)})
    return t, w


def test_decode_of_an_empty_model():
    (anchor, feat, offset, scaling, cam), w = model(0)
    cache = R.rowcache_alloc(0, F, device=DEV)
    for vis in (None, torch.zeros(0, dtype=torch.bool, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV)):
        a = HD.decode(anchor, feat, offset, scaling, cam, w, vis)
        b = HD.decode(anchor, cache, offset, scaling, cam, w, vis)
        assert [x.shape for x in a] == [x.shape for x in b] and a[0].shape == (0, 3)


def test_decode_of_odd_arguments():
    """Indices of every integer type into a cached model; weights that a dict holds flattened."""
    (anchor, feat, offset, scaling, cam), w = model(100)
    cache = R.rowcache_alloc(100, F, device=DEV)
    R.rowcache_write(cache, feat)
    feat = R.rowcache_read(cache)
    flat = {k: v.reshape(-1) for k, v in w.items()}
    idx = torch.tensor([0, 5, 6, 50, 99], device=DEV)
    want = HD.decode(anchor, feat, offset, scaling, cam, w, idx)
    assert want[0].shape[0] > 0
    for kind in (torch.uint8, torch.int16, torch.int32, torch.int64):
        for f, m in ((cache, w), (feat, w), (feat, flat)):
            got = HD.decode(anchor, f, offset, scaling, cam, m, idx.to(kind))
            assert all(torch.equal(x, y) for x, y in zip(want, got))


# The work below is queued on a stream of its own behind products that keep it busy; inputs get their values
# there, behind the products.  A launch on any other stream would read what they held before.


def busy(a):
    for _ in range(4):
        a = a @ a
    return a


@pytest.mark.parametrize("V,n", [(50, 600), (20, 30_000), (5000, 9000), (5000, 40_000)])
def test_lookups_and_gradients_follow_their_stream(V, n):
    D, big = 32, torch.zeros(8192, 8192, device=DEV)
    busy(big)
    new_w, new_ids = torch.randn(V, D, device=DEV), torch.randint(0, V, (n,), device=DEV)
    new_g = torch.randint(-8, 9, (n, D), device=DEV).float()
    want = E.embedding(new_w, new_ids, 2.0), E.embedding_grad(new_g, new_ids, V), 3 + E.embedding_grad(new_g, new_ids, V)
    w, ids, g = torch.zeros(V, D, device=DEV), torch.zeros_like(new_ids), torch.zeros_like(new_g)
    out, s = torch.full((V, D), 3.0, device=DEV), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        busy(big)
        w.copy_(new_w), ids.copy_(new_ids), g.copy_(new_g)
        got = E.embedding(w, ids, 2.0), E.embedding_grad(g, ids, V), E.embedding_grad(g, ids, V, out=out)
        leaf = w.detach().requires_grad_(True)
        y = E.embedding(leaf, ids, 2.0)
        g.zero_(), busy(big), g.copy_(new_g)
        (dw,) = torch.autograd.grad(y, leaf, g)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    assert torch.equal(y, want[0]) and torch.equal(dw, 2 * want[1])


@pytest.mark.parametrize("n,cap", [(1, 100), (600, 100), (5000, 3000), (5000, 30_000)])
def test_cache_writes_and_reads_follow_their_stream(n, cap):
    D, big = 32, torch.zeros(8192, 8192, device=DEV)
    busy(big)
    new_x, new_slots = torch.randn(n, D, device=DEV), torch.randint(0, cap, (n,), device=DEV)
    c, d = (R.rowcache_alloc(cap, D, device=DEV) for _ in range(2))
    R.rowcache_write(c, new_x, new_slots)
    want = R.rowcache_read(c, new_slots)
    x, slots, s = torch.zeros_like(new_x), torch.zeros_like(new_slots), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        busy(big)
        x.copy_(new_x), slots.copy_(new_slots)
        R.rowcache_write(d, x, slots)
        slots.zero_(), busy(big), slots.copy_(new_slots)
        y = R.rowcache_read(d, slots)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(c.codes, d.codes) and torch.equal(c.scales, d.scales) and torch.equal(y, want)
