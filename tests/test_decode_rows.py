"""CPU tests of what the decode hands to its kernels when features come from a row cache or the colour head takes
a learned row (horizongs_amd.decode); the row tables' entries by their formulas, the decode's own call recorded."""
from types import SimpleNamespace

import pytest
import torch

from horizongs_amd import decode as HD
from horizongs_amd import rowcache as R
from tests import rows_on_host

F, N_OFF, K = 32, 10, 35


@pytest.fixture(autouse=True)
def calls(monkeypatch):
    """The arguments of the last decode, which returns nothing but placeholders."""
    rows_on_host.install(monkeypatch)
    got = []

    def apply(*a):
        got[:] = a
        return (torch.empty(0),) * 7

    monkeypatch.setattr(HD, "_check_dev", lambda *ts: None)
    monkeypatch.setattr(HD, "_Decode", SimpleNamespace(apply=apply))
    return got


def scene(A):
    g = torch.Generator().manual_seed(A)
    r = lambda *s: torch.randn(*s, generator=g)
    t = dict(anchor=r(A, 3), feat=torch.randint(-9, 10, (A, F), generator=g).float(), offset=r(A, N_OFF, 3),
             scaling=r(A, 6), cam=r(3))
    w = {}
    for h, o in (("opacity", N_OFF), ("cov", 7 * N_OFF), ("color", 3 * N_OFF)):
        w.update({f"{h}_w1": r(F, K), f"{h}_b1": r(F), f"{h}_w2": r(o, F), f"{h}_b2": r(o)})
    cache = R.rowcache_alloc(A, F, device="cpu")
    R.rowcache_write(cache, t["feat"])
    return t, w, cache


def decode(t, feat, w, visible, **kw):
    return HD.decode(t["anchor"], feat, t["offset"], t["scaling"], t["cam"], w, visible, **kw)


def compacted(calls):
    """The arrays that the decode reads, by its index."""
    anchor, feat, offset, scaling, _, idx = calls[:6]
    return [x[idx.long()] for x in (anchor, feat, offset, scaling)]


@pytest.mark.parametrize("visible", [None, torch.zeros(0, dtype=torch.bool), torch.zeros(0, dtype=torch.int64),
                                     torch.zeros(0, dtype=torch.int32)])
def test_a_cache_of_an_empty_model(calls, visible):
    t, w, cache = scene(0)
    decode(t, cache, w, visible)
    assert [tuple(x.shape) for x in compacted(calls)] == [(0, 3), (0, F), (0, N_OFF, 3), (0, 6)]


@pytest.mark.parametrize("kind", [torch.uint8, torch.int16, torch.int32, torch.int64, torch.bool, None, "lazy"])
def test_indices_of_a_cached_decode(calls, kind):
    """Every kind of index that a decode of float32 features takes."""
    t, w, cache = scene(40)
    idx = torch.tensor([3, 4, 9, 17, 39])
    if kind == torch.bool:
        visible = torch.zeros(40, dtype=kind)
        visible[idx] = True
    elif kind == "lazy":
        buf = torch.full((40,), -7, dtype=torch.int32)
        buf[:5] = idx
        visible = HD.VisibleIndex(buf, torch.tensor([0, 5]), torch.ones(40, dtype=torch.bool))
    else:
        visible, idx = (None, torch.arange(40)) if kind is None else (idx.to(kind), idx)
    decode(t, cache, w, visible)
    got = compacted(calls)
    for x, k in zip(got, ("anchor", "feat", "offset", "scaling")):
        assert torch.equal(x, t[k][idx])
    if kind != "lazy":
        decode(t, t["feat"], w, visible)
        assert all(torch.equal(x, y) for x, y in zip(got, compacted(calls)))


def test_flattened_weights(calls):
    """A dict's weights are read by their memory, whatever their shape; with a row, too."""
    t, w, cache = scene(7)
    flat = {k: v.reshape(-1) for k, v in w.items()}
    decode(t, t["feat"], flat, None)
    assert all(x is y for x, y in zip(calls[7:], flat.values()))
    row = torch.randn(5)
    first = torch.randn(F, K + 5)
    for a, b in ((first, w), (first.reshape(-1), flat)):
        decode(t, t["feat"], dict(b, color_w1=a), None, appearance=row)
        assert torch.equal(calls[7 + 8], first[:, :K])
        assert torch.allclose(calls[7 + 9], w["color_b1"] + first[:, K:] @ row, atol=1e-5)
        with pytest.raises(ValueError, match="appearance row"):
            decode(t, t["feat"], dict(b, color_w1=a), None)
        with pytest.raises(ValueError, match="does not fit"):
            decode(t, t["feat"], dict(b, color_w1=a), None, appearance=row[:4])
