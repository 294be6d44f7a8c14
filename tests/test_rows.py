"""CPU tests of the row tables' boundary (horizongs_amd.embedding, horizongs_amd.rowcache): what the
calls refuse, at the Python surface and at the C entries, before any device work."""
import pytest
import torch

from horizongs_amd import embedding as E
from horizongs_amd import rowcache as R

W = torch.zeros(5, 4)
I = torch.zeros(3, dtype=torch.int64)
G = torch.zeros(3, 4)


@pytest.mark.parametrize("call,match", [
    (lambda: E.embedding(torch.zeros(5), I), "rows, columns"),
    (lambda: E.embedding(W.double(), I), "float64"),
    (lambda: E.embedding(W, I, dtype=torch.int32), "int32"),
    (lambda: E.embedding(W, I.float()), "ids are needed"),
    (lambda: E.embedding(W, I.to(torch.int16)), "ids are needed"),
    (lambda: E.embedding(torch.zeros(4, 5).t(), I), "contiguous"),
    (lambda: E.embedding_grad(G.double(), I, 5), "float64"),
    (lambda: E.embedding_grad(G, I[:2], 5), "one row per id"),
    (lambda: E.embedding_grad(G, I.bool(), 5), "ids are needed"),
    (lambda: E.embedding_grad(G, I, -1), "negative"),
    (lambda: E.embedding_grad(G, I, 5, dtype=torch.float64), "float64"),
    (lambda: E.embedding_grad(G, I, 5, out=torch.zeros(6, 4)), "out is"),
    (lambda: E.embedding_grad(G, I, 5, out=torch.zeros(5, 4), dtype=torch.bfloat16), "out is"),
    (lambda: E.embedding_grad(G, I, 5, out=torch.zeros(1, 4).expand(5, 4)), "overlap"),
    (lambda: E.embedding_grad(G, I, 5, out=torch.zeros(4, 5).t()), "contiguous"),
    (lambda: R.rowcache_alloc(4, 8, "int4", device="cpu"), "format"),
    (lambda: R.rowcache_alloc(4, 8, group=24, device="cpu"), "group"),
    (lambda: R.rowcache_alloc(4, 0, device="cpu"), "columns"),
])
def test_refused_arguments(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_sums_added_to_a_table_are_not_differentiable():
    for g, out in ((G, torch.zeros(5, 4, requires_grad=True)), (G.clone().requires_grad_(True), torch.zeros(5, 4))):
        with pytest.raises(NotImplementedError, match="not differentiable"):
            E.embedding_grad(g, I, 5, out=out)


def test_cpu_tensors_are_refused():
    c = R.rowcache_alloc(5, 4, device="cpu")
    for call in (lambda: E.embedding(W, I), lambda: E.embedding_grad(G, I, 5), lambda: R.rowcache_write(c, G, I),
                 lambda: E.embedding_grad(G, I, 5, out=torch.zeros(5, 4)), lambda: R.rowcache_read(c, I),
                 lambda: R.rowcache_read(c)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


def test_refused_caches():
    c = R.rowcache_alloc(5, 40, "e4m3", group=16, device="cpu")
    assert c.codes.dtype == torch.float8_e4m3fn and c.codes.shape == (5, 40) and c.scales.shape == (5, 3)
    rows = torch.zeros(3, 40)
    bad = [((c.codes, c.scales, 24), "group"), ((c.codes.view(torch.uint8), c.scales, 16), "codes"),
           ((c.codes, c.scales, 32), "do not fit"), ((c.codes, c.scales.double(), 16), "do not fit"),
           ((c.codes[:4], c.scales, 16), "do not fit"), ((c.codes[0], c.scales, 16), "codes"),
           ((c.codes[:1].expand(5, 40), c.scales, 16), "overlap"),
           ((c.codes, c.scales[:1].expand(5, 3), 16), "overlap"),
           ((c.codes, torch.zeros(3, 5).t(), 16), "contiguous")]
    for cache, match in bad:
        with pytest.raises(ValueError, match=match):
            R.rowcache_write(cache, rows, I)
        with pytest.raises(ValueError, match=match):
            R.rowcache_read(cache, I)
    for args, match in (((rows[:, :39], I), "rows"), ((rows, I[:2]), "slots"), ((rows.double(), I), "float64"),
                        ((rows, I.float()), "ids are needed"), ((torch.zeros(6, 40), None), "6 rows, 5 slots"),
                        ((rows, I[None]), "slots")):
        with pytest.raises(ValueError, match=match):
            R.rowcache_write(c, *args)
    with pytest.raises(ValueError, match="float64"):
        R.rowcache_read(c, I, dtype=torch.float64)


def test_c_entries_refuse_before_any_launch():
    from horizongs_amd import _native as N
    lib = N.lib()

    def refused(st, word, code=-1):
        assert st == code and word in lib.hgsr_last_error().decode(), lib.hgsr_last_error()

    f, t = 64, 128  # never read: every call below is refused on the host
    refused(lib.hgsr_embed_fwd(1 << 31, 1, 4, f, 0, 4, f, 0, 1, 1.0, t, 0, None), "rows")
    refused(lib.hgsr_embed_fwd(4, 1 << 31, 4, f, 0, 4, f, 0, 1, 1.0, t, 0, None), "ids")
    refused(lib.hgsr_embed_fwd(4, 1, 0, f, 0, 4, f, 0, 1, 1.0, t, 0, None), "row length")
    refused(lib.hgsr_embed_fwd(4, 1, (1 << 21) + 1, f, 0, 4, f, 0, 1, 1.0, t, 0, None), "row length")
    refused(lib.hgsr_embed_fwd(4, 1, 4, f, 3, 4, f, 0, 1, 1.0, t, 0, None), "type")
    refused(lib.hgsr_embed_fwd(4, 1, 4, f, 0, -4, f, 0, 1, 1.0, t, 0, None), "stride")
    refused(lib.hgsr_embed_fwd(4, 1, 4, None, 0, 4, f, 0, 1, 1.0, t, 0, None), "null")
    refused(lib.hgsr_embed_bwd(4, 1, 4, f, 0, 4, f, 0, 1, 1.0, t, 0, 3, 0, f, 1 << 20, None), "stride")
    refused(lib.hgsr_embed_bwd(4, 1, 4, f, 0, 4, f, 0, 1, 1.0, None, 0, 4, 0, f, 1 << 20, None), "null")
    refused(lib.hgsr_embed_bwd(4, 1, 4, f, 0, 4, f, 0, 1, 1.0, t, 0, 5, 0, f, 1 << 20, None), "contiguous")
    refused(lib.hgsr_embed_bwd(1 << 30, 1, 64, f, 0, 4, f, 0, 1, 1.0, t, 0, 64, 0, f, 1 << 20, None), "dense gradient")
    refused(lib.hgsr_embed_bwd(1 << 20, 1 << 30, 2048, f, 0, 0, f, 0, 1, 1.0, t, 0, 2048, 0, f, 1 << 50, None), "too many")
    for V, n in ((4, 2000), (1000, 2000), (1000, 100_000)):  # each form that keeps a workspace
        need = lib.hgsr_embed_bwd_ws_bytes(V, n, 4)
        refused(lib.hgsr_embed_bwd(V, n, 4, f, 0, 4, f, 0, 1, 1.0, t, 0, 4, 0, f, 0, None), "workspace", -3)
        refused(lib.hgsr_embed_bwd(V, n, 4, f, 0, 4, f, 0, 1, 1.0, t, 0, 4, 0, None, need, None), "workspace", -3)
        assert need > 0
    assert lib.hgsr_embed_bwd_ws_bytes(4, 0, 4) == 0
    cache = (f, 4, f, 1)
    refused(lib.hgsr_rowcache_write(4, 1, 4, 24, 0, f, 0, 4, None, 0, 1, *cache, None, 0, None), "group")
    refused(lib.hgsr_rowcache_write(4, 1, 4, 32, 2, f, 0, 4, None, 0, 1, *cache, None, 0, None), "format")
    refused(lib.hgsr_rowcache_write(4, 5, 4, 32, 0, f, 0, 4, None, 0, 1, *cache, None, 0, None), "slots")
    refused(lib.hgsr_rowcache_write(4, 5000, 4, 32, 0, f, 0, 4, f, 0, 1, *cache, None, 0, None), "workspace", -3)
    ws = lib.hgsr_rowcache_write_ws_bytes
    assert ws(9, 5000, 4, 1) >= 36 and ws(9, 5000, 4, 0) == 0 and ws(9, 2048, 4, 1) == 0 and ws(9, 2048, 1 << 20, 1) >= 36
    refused(lib.hgsr_rowcache_read(4, 1, 40, 32, 0, f, 40, f, 1, None, 0, 1, t, 0, None), "stride")
    refused(lib.hgsr_rowcache_read(4, 1, 4, 32, 0, f, 4, f, 1, None, 0, 1, None, 0, None), "null")
    # nothing to do: no launch, no error
    assert lib.hgsr_embed_fwd(4, 0, 4, None, 0, 4, None, 0, 1, 1.0, None, 0, None) == 0
    assert lib.hgsr_rowcache_read(4, 0, 4, 32, 0, None, 4, None, 1, None, 0, 1, None, 0, None) == 0


def test_gradbuf_take():
    from horizongs_amd import gradbuf
    p, d = torch.zeros(3, 2), torch.zeros(3, 2)
    gradbuf.set_dest(p, d)
    assert gradbuf.take(gradbuf.key(p), (3, 2), torch.float32) is d
    assert gradbuf.take(gradbuf.key(p), (3, 2), torch.float32) is None
    gradbuf.clear()
