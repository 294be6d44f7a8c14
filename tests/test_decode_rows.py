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
