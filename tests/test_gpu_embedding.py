"""GPU checks of the embedding lookup and its gradient (horizongs_amd.embedding) against their formulas
in 64 bits.

Tolerances.  u = 2^-24 is half a step of f32, h half a step of the result's type (eps / 2), both relative;
2^-25 is half the smallest f16 number (bf16's and f32's lie below what the inputs reach).
  lookup: one f32 product and one rounding                       (u + h + u h) |w s|
  gradient: k - 1 additions, one product, one rounding           ((k + 1) u + h) s sum |g|, + u for the old
  value's addition where the sums are added to a table.  Sums of small whole numbers are exact in f32 in
  any order: those are compared for equality, whatever the run's length."""
import numpy as np
import pytest
import torch

from horizongs_amd import embedding as E

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half(t):
    return 0.0 if t == F32 else torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make_ids(kind, V, n, seed, dtype=torch.int64):
    g = gen(seed)
    if kind == "uniform":
        ids = torch.randint(0, V, (n,), generator=g)
    elif kind == "one":
        ids = torch.full((n,), V // 2)
    elif kind == "sorted":
        ids = torch.randint(0, V, (n,), generator=g).sort().values
    elif kind == "reversed":
        ids = torch.arange(n).flip(0) % V
    elif kind == "padded":  # -1, V and numbers far outside among them
        ids = torch.randint(0, V, (n,), generator=g)
        far = torch.tensor([-1, V, -2 ** 31, 2 ** 31 - 1])[torch.randint(0, 4, (n,), generator=g)]
        ids = torch.where(torch.rand(n, generator=g) < 0.3, far, ids)
    elif kind == "tail":  # in order, padding behind
        ids = torch.randint(0, V, (n,), generator=g).sort().values
        ids[n - n // 3:] = -1
    elif kind == "none":
        ids = torch.full((n,), -1)
    else:  # half of the entries one row, the rest spread
        ids = torch.where(torch.rand(n, generator=g) < 0.5, 0, torch.randint(0, V, (n,), generator=g))
    return ids.to(dtype)


def want_lookup(w, ids, scale):
    V = w.shape[0]
    ok = (ids >= 0) & (ids < V)
    return torch.where(ok[..., None], w.double()[ids.long().clamp(0, max(V - 1, 0))] * float(np.float32(scale)), 0.0)


def want_grad(g, ids, V, scale):
    """(sum, sum of magnitudes, terms of the longest run), 64 bits."""
    ok = (ids >= 0) & (ids < V)
    at, g = ids[ok].long(), g.double()[ok] * float(np.float32(scale))
    s = torch.zeros(V, g.shape[1], dtype=torch.float64).index_add_(0, at, g)
    m = torch.zeros(V, g.shape[1], dtype=torch.float64).index_add_(0, at, g.abs())
    return s, m, int(torch.bincount(at, minlength=1).max()) if at.numel() else 0


def check(got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float((got - want).abs().max()), got[bad][:4], want[bad][:4])


KINDS = ["uniform", "one", "sorted", "reversed", "padded", "none", "mixed"]
SIZES = [(1, 1, 1), (16, 1, 32), (5, 3, 7), (16, 300, 32), (1000, 777, 33), (300, 70, 96), (9, 129, 130), (70, 64, 515),
         (2049, 4100, 8), (40, 90, 1024), (3, 5000, 2), (100_000, 2000, 4), (7, 20_000, 16)]


@pytest.mark.parametrize("V,n,D", SIZES)
@pytest.mark.parametrize("wt,ot", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (BF16, F32), (F16, BF16)])
def test_lookup(V, n, D, wt, ot):
    w = torch.randn(V, D, generator=gen(V + n + D)).to(wt)
    wd = w.to(DEV)
    for k, kind in enumerate(KINDS):
        ids = make_ids(kind, V, n, k, torch.int32 if k % 2 else torch.int64)
        for scale in (1.0, 5.657):
            out = E.embedding(wd, ids.to(DEV), scale, dtype=ot)
            want = want_lookup(w, ids, scale)
            assert out.dtype == ot
            check(out, want, (U + half(ot)) * (1 + U) * want.abs() + (2.0 ** -25 if ot == F16 else 0))
            if scale == 1.0 and wt == ot:
                assert torch.equal(out.cpu().double(), want)


@pytest.mark.parametrize("V,n,D", SIZES)
@pytest.mark.parametrize("gt,ot", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16)])
def test_grad(V, n, D, gt, ot):
    g = torch.randn(n, D, generator=gen(3 * V + n + D)).to(gt)
    gd = g.to(DEV)
    for k, kind in enumerate(KINDS):
        ids = make_ids(kind, V, n, k, torch.int64 if k % 2 else torch.int32)
        scale = (1.0, 0.25, 5.657)[k % 3]
        dw = E.embedding_grad(gd, ids.to(DEV), V, scale, dtype=ot)
        s, m, run = want_grad(g, ids, V, scale)
        assert dw.dtype == ot and dw.shape == (V, D)
        check(dw, s, (run + 1) * U * m + half(ot) * (s.abs() + (run + 1) * U * m) + (2.0 ** -25 if ot == F16 else 0))
        assert torch.equal(dw, E.embedding_grad(gd, ids.to(DEV), V, scale, dtype=ot))  # the same bits again
        # added to a table: its named rows take the sums, the others stay as they are
        old = torch.randn(V, D, generator=gen(k)).to(ot)
        out = old.to(DEV)
        assert E.embedding_grad(gd, ids.to(DEV), V, scale, out=out) is out
        want = s + old.double()
        tol = (run + 1) * U * m + (U + half(ot)) * (want.abs() + (run + 1) * U * m)
        check(out, want, tol + (2.0 ** -25 if ot == F16 else 0))
        named = torch.zeros(V, dtype=torch.bool)
        named[ids[(ids >= 0) & (ids < V)].long()] = True
        assert torch.equal(out.cpu()[~named], old[~named])


@pytest.mark.parametrize("V,n,D,kind", [
    (16, 500_000, 32, "uniform"), (16, 300_001, 32, "one"), (1, 70_000, 4, "one"), (1_000_003, 400_000, 8, "uniform"),
    (5_000_000, 30_000, 1, "mixed"), (65_536, 40_000, 64, "mixed"), (3, 16_384, 256, "mixed"), (3, 16_385, 256, "mixed"),
    (70_000, 4096, 40, "padded"), (70_000, 4097, 40, "padded"), (2048, 1024, 640, "mixed"), (2047, 1025, 640, "mixed"),
    (300, 256, 2048, "one"), (300, 257, 2048, "one"), (1_000_000, 250_000, 32, "sorted"), (4096, 65_536, 5, "mixed"),
    (2048, 100_000, 33, "reversed"), (70_000, 40_000, 8, "one"), (2048, 100_000, 33, "sorted"),
    (50_000, 30_000, 24, "tail"), (3000, 20_000, 8, "none"), (1_500_000, 17_000, 4, "tail"), (600, 9000, 48, "tail"),
    (600, 16_384, 8, "one"), (1 << 20, 16_000, 8, "mixed"), (200, 5000, 100, "uniform"),
    (90, 32_768, 12, "uniform"), (90, 32_769, 12, "uniform"), (1 << 20, 30_000, 8, "mixed"), (1 << 20, 60_000, 8, "mixed"), (1 << 20, 8193, 8, "one"),
    (300, 8192, 24, "mixed"), (300, 8193, 24, "mixed"), (300, 1024, 2048, "one"), (300, 1025, 2048, "one"),
    (200_000_000, 30_000, 1, "mixed"), (2047, 16_384, 20, "mixed"), (2047, 16_385, 20, "mixed"),
    (2048, 16_385, 20, "mixed"), (2048, 24_576, 20, "one"), (2048, 24_577, 20, "one"), (100_000, 24_000, 20, "mixed"),
    (1600, 1000, 2048, "mixed"), (1600, 1021, 520, "one")])
def test_grad_of_whole_numbers_is_exact(V, n, D, kind):
    ids = make_ids(kind, V, n, n).to(DEV)
    g = torch.randint(-8, 9, (n, D), generator=gen(V)).to(DEV)
    at = torch.where((ids >= 0) & (ids < V), ids, V)
    want = torch.zeros(V + 1, D, dtype=torch.int64, device=DEV).index_add_(0, at, g)[:V]
    for t in (F32, BF16):
        dw = E.embedding_grad(g.to(t), ids, V, 0.5, dtype=F32)
        assert torch.equal(dw.double() * 2, want.double())
    out = torch.ones(V, D, device=DEV)
    E.embedding_grad(g.float(), ids, V, 1.0, out=out)
    assert torch.equal(out.double(), want.double() + 1)


@pytest.mark.parametrize("D,near", [(257, 4096), (33, 32_768), (2, 65_536), (600, 64)])
@pytest.mark.parametrize("order", ["sorted", "shuffled"])
def test_runs_of_many_lengths_are_exact(D, near, order):
    """Rows that about `near` ids name (what a hundred workgroups' worth of entries comes to, and one), some
    exactly as many, with rows of one or a few ids between them."""
    g0 = gen(D + near)
    length = torch.randint(near - near // 8, near + near // 8 + 1, (9,), generator=g0).tolist()
    length = [1, near, near + 1, 3, 2 * near, *length[:5], 1, 2, near - 1, *length[5:], 3 * near]
    V = 3 * len(length) + 1
    ids = torch.repeat_interleave(3 * torch.arange(len(length)) + 1, torch.tensor(length))
    if order == "shuffled":
        ids = ids[torch.randperm(ids.numel(), generator=g0)]
    ids = ids.to(DEV)
    for t in (F32, BF16):
        g = torch.randint(-8, 9, (ids.numel(), D), generator=g0).to(DEV)
        want = torch.zeros(V, D, dtype=torch.int64, device=DEV).index_add_(0, ids, g)
        assert torch.equal(E.embedding_grad(g.to(t), ids, V, dtype=F32).double(), want.double())
        out = torch.ones(V, D + 1, device=DEV)
        E.embedding_grad(g.to(t), ids, V, out=out[:, 1:])
        assert torch.equal(out[:, 1:].double(), want.double() + 1) and out[:, 0].eq(1).all()


def test_strides_and_shapes():
    g0 = gen(1)
    wide = torch.randn(50, 45, generator=g0)
    ids = torch.randint(-1, 50, (6, 4, 3), generator=g0)
    for a, b in ((0, 40), (1, 41), (4, 36), (5, 45)):  # column ranges: every alignment
        w = wide.to(DEV)[:, a:b]
        for t in (F32, BF16):
            src = wide.to(t)[:, a:b]
            out = E.embedding(wide.to(t).to(DEV)[:, a:b], ids.to(DEV), 1.0)
            assert out.shape == (6, 4, 3, b - a) and torch.equal(out.cpu().double(), want_lookup(src, ids, 1.0))
        gw = torch.randint(-8, 9, (72, 45), generator=g0).float().to(DEV)
        store = torch.zeros(50, 47, device=DEV)
        E.embedding_grad(gw[:, a:b], ids.reshape(-1).to(DEV), 50, out=store[:, a:b])
        s, _, _ = want_grad(gw.cpu()[:, a:b], ids.reshape(-1), 50, 1.0)
        assert torch.equal(store[:, a:b].cpu().double(), s)
        store[:, a:b] = 0
        assert not store.any()  # nothing beside the range was touched
        del w
    one = torch.full((), 7, dtype=torch.int32, device=DEV).expand(9)  # one id for all rows: stride 0
    assert torch.equal(E.embedding(wide.to(DEV), one), wide.to(DEV)[7].expand(9, 45))
    g = torch.ones(1, 45, device=DEV).expand(9, 45)  # one gradient for all rows
    assert float(E.embedding_grad(g, one, 50)[7].sum()) == 9 * 45
    skip = ids.reshape(-1).to(DEV)[::3]
    assert torch.equal(E.embedding(wide.to(DEV), skip).cpu().double(), want_lookup(wide, ids.reshape(-1)[::3], 1.0))
    every = wide[:1].to(DEV).expand(20, 45)  # every row of the table the same memory
    assert torch.equal(E.embedding(every, skip.clamp(0, 19)), every[:1].expand(skip.numel(), 45))


@pytest.mark.parametrize("V,n,D", [(40, 300, 24), (3, 4000, 16), (500, 9000, 40), (4000, 40_000, 16), (900, 2000, 1032)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_bits_do_not_depend_on_where_tensors_lie(V, n, D, t):
    """The same values at every element offset and row stride: the same sums, bit for bit."""
    ids = make_ids("mixed", V, n, n).to(DEV)
    g = torch.randn(n, D, generator=gen(V)).to(t).to(DEV)
    w = torch.randn(V, D, generator=gen(n)).to(t).to(DEV)
    want, rows, base = E.embedding_grad(g, ids, V, 0.3), E.embedding(w, ids, 0.3), E.embedding_grad(g, ids, V, 0.3, out=w.clone())
    for off in (1, 2, 3, 5):
        for extra in (0, 1, 6):
            place = lambda x: torch.empty(x.shape[0] * (D + extra) + off, dtype=t, device=DEV)[off:].view(x.shape[0], -1)[:, :D]
            g1, w1, o1 = place(g).copy_(g), place(w).copy_(w), place(w).copy_(w)
            assert torch.equal(E.embedding_grad(g1, ids, V, 0.3), want)
            assert torch.equal(E.embedding(w1, ids, 0.3), rows)
            assert torch.equal(E.embedding_grad(g1, ids, V, 0.3, out=o1), base)


def test_empty():
    w = torch.zeros(4, 3, device=DEV)
    e = torch.empty(0, dtype=torch.int64, device=DEV)
    assert E.embedding(w, e).shape == (0, 3)
    assert E.embedding(w, e.reshape(2, 0)).shape == (2, 0, 3)
    assert not E.embedding_grad(torch.empty(0, 3, device=DEV), e, 4).any()
    out = torch.ones(4, 3, device=DEV)
    E.embedding_grad(torch.empty(0, 3, device=DEV), e, 4, out=out)
    assert out.eq(1).all()
    none = torch.empty(0, 3, device=DEV)  # a table without rows: every id is padding
    i = torch.tensor([0, -1, 5], device=DEV)
    assert E.embedding(none, i).eq(0).all() and E.embedding_grad(torch.ones(3, 3, device=DEV), i, 0).shape == (0, 3)
    assert E.embedding(torch.empty(4, 0, device=DEV), i).shape == (3, 0)
    p = torch.empty(4, 3, device=DEV, requires_grad=True)
    E.embedding(p, e).sum().backward()
    assert p.grad.eq(0).all()


def test_non_finite_values_stay_in_their_rows():
    w = torch.ones(5, 8)
    w[1], w[2] = float("nan"), float("inf")
    out = E.embedding(w.to(DEV), torch.tensor([0, 1, 2, -1, 4], device=DEV), 2.0).cpu()
    assert out[0].eq(2).all() and out[1].isnan().all() and out[2].eq(float("inf")).all() and out[3].eq(0).all()
    g = torch.ones(5, 8)
    g[1], g[3] = float("nan"), float("inf")  # row 3 is padding: what it holds is not read into any sum
    for n in (5, 20_000):
        ids = torch.full((n,), -1)
        ids[:5] = torch.tensor([0, 1, 2, -1, 2])
        dw = E.embedding_grad(torch.cat([g, torch.full((n - 5, 8), float("nan"))]).to(DEV), ids.to(DEV), 4).cpu()
        assert dw[0].eq(1).all() and dw[1].isnan().all() and dw[2].eq(2).all() and dw[3].eq(0).all()


@pytest.mark.parametrize("V,n,D,kind", [(40, 30, 8, "uniform"), (6, 3000, 8, "one"), (900, 3000, 8, "uniform"),
                                        (60_000, 50_000, 8, "uniform"), (60_000, 50_000, 8, "sorted")])
def test_rows_without_ids_are_zeros_for_every_scale(V, n, D, kind):
    ids = make_ids(kind, V, n, 1)
    rest = torch.ones(V, dtype=torch.bool)
    rest[ids] = False
    for scale in (-2.0, float("inf"), float("nan")):
        dw = E.embedding_grad(torch.ones(n, D, device=DEV), ids.to(DEV), V, scale).cpu()
        assert rest.any() and not dw[rest].view(torch.int32).any()
        assert torch.equal(dw[~rest].isfinite(), torch.full_like(dw[~rest], np.isfinite(scale)).bool())
        assert E.embedding(torch.ones(V, D, device=DEV), torch.tensor([-1, V], device=DEV), scale).eq(0).all()


def test_autograd_and_differences():
    V, n, D, scale = 30, 50, 12, 0.5
    w = torch.randn(V, D, generator=gen(0)).to(DEV).requires_grad_(True)
    ids = make_ids("padded", V, n, 3).reshape(5, 10).to(DEV)
    c = torch.randn(5, 10, D, generator=gen(1)).to(DEV)
    out = E.embedding(w, ids, scale)
    (out * c).sum().backward()
    s, m, run = want_grad(c.cpu().reshape(n, D), ids.cpu().reshape(-1), V, scale)
    check(w.grad, s, (run + 1) * U * m)
    # differences: the lookup is linear, so a step along any direction d changes the sum by <dw, d> exactly
    d = torch.randn(V, D, generator=gen(2)).to(DEV)
    with torch.no_grad():
        step = ((E.embedding(w + d, ids, scale).double() - E.embedding(w, ids, scale).double()) * c.double()).sum()
    assert abs(float(step - (w.grad.double() * d.double()).sum())) <= 8 * U * float(
        (E.embedding(w.detach().abs() + d.abs(), ids, scale).double() * c.double().abs()).sum())
    w.grad = None
    E.embedding(w, ids, scale).sum().backward()  # the gradient of a sum: one value for every place
    s, m, run = want_grad(torch.ones(n, D), ids.cpu().reshape(-1), V, scale)
    assert torch.equal(w.grad.cpu().double(), s)
    w.grad = None
    (E.embedding(w, ids, scale).sum() + E.embedding(w, ids[0], 1.0).sum()).backward()  # two uses of a table
    s2, _, _ = want_grad(torch.ones(10, D), ids[0].cpu(), V, 1.0)
    assert torch.equal(w.grad.cpu().double(), s + s2)
    b = w.detach().to(BF16).requires_grad_(True)  # 16-bit table, f32 rows out, 16-bit gradient
    o = E.embedding(b, ids, 1.0, dtype=F32)
    o.backward(torch.ones_like(o))
    assert o.dtype == F32 and b.grad.dtype == BF16
    # second derivatives: of sum((s W[ids])^2 c) / 2 along d, 2 s^2 sum c d[ids] back to its rows
    q = w.detach().clone().requires_grad_(True)
    (x,) = torch.autograd.grad((E.embedding(q, ids, scale).square() * c).sum(), q, create_graph=True)
    (hd,) = torch.autograd.grad(x, q, d)
    gd = (2 * c.double() * want_lookup(d.cpu(), ids.cpu(), scale).to(DEV)).cpu().reshape(n, D)
    s, m, run = want_grad(gd, ids.cpu().reshape(-1), V, scale)
    check(hd, s, (run + 4) * U * m)


def test_gradient_lands_in_a_registered_destination():
    from horizongs_amd import gradbuf
    w = torch.randn(20, 8, device=DEV, requires_grad=True)
    dest = torch.full((160,), 9.0, device=DEV)
    gradbuf.set_dest(w, dest.view(20, 8))
    E.embedding(w, torch.tensor([1, 1, 3], device=DEV)).sum().backward()
    assert w.grad.data_ptr() == dest.data_ptr() and float(dest.sum()) == 24
    gradbuf.clear()


def test_other_stream():
    w = torch.randn(1000, 64, device=DEV)
    ids = torch.randint(0, 1000, (30_000,), device=DEV)
    g = torch.randint(-8, 9, (30_000, 64), device=DEV).float()
    a, b = E.embedding(w, ids, 2.0), E.embedding_grad(g, ids, 1000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c, d = E.embedding(w, ids, 2.0), E.embedding_grad(g, ids, 1000)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, c) and torch.equal(b, d)


@pytest.mark.parametrize("n", [7, 3000, 40_000])
def test_captured_and_replayed(n):
    """Two graphs over the same static inputs, replayed in turn with other work between."""
    V, D = 500, 32
    w, g = torch.randn(V, D, device=DEV), torch.zeros(n, D, device=DEV)
    ids = torch.zeros(n, dtype=torch.int64, device=DEV)
    total = torch.zeros(V, D, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        E.embedding(w, ids), E.embedding_grad(g, ids, V)
    torch.cuda.current_stream().wait_stream(s)
    graphs, res = [], []
    for k in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res.append((E.embedding(w, ids, k + 1.0), E.embedding_grad(g, ids, V, k + 1.0),
                        E.embedding_grad(g, ids, V, 1.0, out=total)))
        graphs.append(gr)
    for rep in range(4):
        ids.copy_(make_ids("mixed" if rep % 2 else "padded", V, n, rep))
        g.copy_(torch.randint(-8, 9, (n, D), generator=gen(rep)))
        torch.cuda.synchronize()
        for k, gr in enumerate(graphs):
            before = total.clone()
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(res[k][0], E.embedding(w, ids, k + 1.0))
            assert torch.equal(res[k][1], E.embedding_grad(g, ids, V, k + 1.0))
            assert torch.equal(total, E.embedding_grad(g, ids, V, 1.0, out=before))


def test_captured_training_step():
    """Forward and backward of a table captured together, replayed against the eager step."""
    w = torch.randn(200, 16, device=DEV)
    p = w.clone().requires_grad_(True)
    ids = torch.randint(0, 200, (600,), device=DEV)
    c = torch.randint(-8, 9, (600, 16), device=DEV).float()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        (E.embedding(p, ids) * c).sum().backward()
    torch.cuda.current_stream().wait_stream(s)
    p.grad = None
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        (dw,) = torch.autograd.grad(E.embedding(p, ids), p, c)
    for rep in range(3):
        ids.copy_(torch.randint(0, 200, (600,), generator=gen(rep)))
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, E.embedding_grad(c, ids, 200))


def test_table_beyond_2_31_elements():
    V, D = 2_200_000, 1024
    w = torch.zeros(V, D, dtype=BF16, device=DEV)
    ids = torch.tensor([V - 1, 0, V - 2, 2_097_152, V - 1, V], device=DEV)  # 2_097_152 * 1024 = 2^31
    rows = torch.arange(1, 7, device=DEV, dtype=F32)[:, None].expand(6, D).to(BF16)
    E.embedding_grad(rows, ids, V, out=w)
    assert w[V - 1].eq(6).all() and w[0].eq(2).all() and w[V - 2].eq(3).all() and w[2_097_152].eq(4).all()
    out = E.embedding(w, ids)
    assert out[:, 0].tolist() == [6, 2, 3, 4, 6, 0]
    dense = E.embedding_grad(rows, ids, V)  # every other row written as zeros
    assert torch.equal(dense[ids[:5]], w[ids[:5]])
    dense[ids[:5]] = 0
    assert not dense.any()


@pytest.mark.parametrize("n", [500, 3000, 40_000])
def test_table_of_140_gib(n):
    """More zeros than the threads of one launch can store a piece each."""
    V, D = 560_000, 1 << 16
    if torch.cuda.mem_get_info()[0] < 180 << 30:
        pytest.skip("180 GiB of free memory are needed")
    ids = torch.randint(0, V, (n,), generator=gen(n)).to(DEV)
    ids[:2] = torch.tensor([0, V - 1], device=DEV)
    dw = E.embedding_grad(torch.ones(1, D, device=DEV).expand(n, D), ids, V)
    count = torch.bincount(ids, minlength=V).float()
    for r in range(0, V, 20_000):
        part = dw[r:r + 20_000]
        assert torch.equal(part.amin(1), count[r:r + 20_000]) and torch.equal(part.amax(1), count[r:r + 20_000])
    del dw, part
    torch.cuda.empty_cache()


def test_rows_beyond_2_31_elements():
    n, D = 2_100_000, 1024
    ids = torch.zeros(n, dtype=torch.int32, device=DEV)
    ids[-1] = 1
    w = torch.tensor([[1.0], [2.0]], device=DEV).expand(2, D).to(BF16).contiguous()
    out = E.embedding(w, ids)
    assert out[-1].eq(2).all() and out[n - 2].eq(1).all() and out[2_097_152].eq(1).all()
    dw = E.embedding_grad(out, ids, 2, dtype=F32)
    assert dw[0].eq(n - 1).all() and dw[1].eq(2).all()


def test_module():
    m = E.Embedding(12, 8, scale=2.0, device=DEV)
    i = torch.tensor([[3, 3], [11, 0]], device=DEV)
    out = m(i)
    assert torch.equal(out, m.embedding.weight[i] * 2) and torch.equal(m.mean(), m.embedding.weight.mean(0))
    out.sum().backward()
    assert m.embedding.weight.grad[3].eq(4).all() and m.embedding.weight.grad[1].eq(0).all()


def test_gradient_by_itself_is_differentiable():
    V, n, D = 40, 90, 12
    g = torch.randn(3, 30, D, generator=gen(0)).to(DEV).requires_grad_(True)
    ids = make_ids("padded", V, n, 3).reshape(3, 30).to(DEV)
    c = torch.randn(V, D, generator=gen(1)).to(DEV)
    dw = E.embedding_grad(g, ids, V, 0.5)
    with torch.no_grad():
        assert torch.equal(dw, E.embedding_grad(g, ids, V, 0.5))
    (dw * c).sum().backward()
    assert torch.equal(g.grad.cpu().double(), want_lookup(c.cpu(), ids.cpu(), 0.5))
