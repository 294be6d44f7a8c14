"""GPU checks of the 8-bit row cache (horizongs_amd.rowcache) against its definition.

Codes and scales are whole decisions: the 64-bit quotient of two f32 numbers is never nearer to a border
between codes than 2^-27 of it without lying on it (x / s - t is a whole number of s-steps over s), far
above 64-bit rounding, so they are compared for equality.  A read is one f32 product (2^-24) and one
rounding to its type (eps / 2)."""
import numpy as np
import pytest
import torch

from horizongs_amd import rowcache as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TOP = {"int8": 127.0, "e4m3": 448.0}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def e4m3_table():
    k = np.arange(127)
    return np.where(k < 8, k * 2.0 ** -9, (8 + k % 8) * 2.0 ** (k // 8 - 10.0))


def want_write(x, fmt, group):
    """(code values, f32 scales) of rows x [n, D] (numpy, f32 values)."""
    n, D = x.shape
    G = -(-D // group)
    wide = np.zeros((n, G * group), np.float32)
    wide[:, :D] = x
    with np.errstate(invalid="ignore", over="ignore"):
        amax = np.abs(wide).reshape(n, G, group).max(2)
        s = np.maximum(amax * (np.float32(1) / np.float32(TOP[fmt])), np.float32(2.0 ** -100)).astype(np.float32)
    fine = np.isfinite(amax)
    s = np.where(fine, s, np.float32("nan"))
    per = np.repeat(np.where(fine, s, 1.0).astype(np.float64), group, 1)[:, :D]
    q = np.where(np.repeat(fine, group, 1)[:, :D], x.astype(np.float64), 0.0) / per
    if fmt == "int8":
        return np.rint(q), s
    t = e4m3_table()
    a = np.abs(q)
    hi = np.clip(np.searchsorted(t, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    k = np.where((a - t[lo] < t[hi] - a) | ((a - t[lo] == t[hi] - a) & (lo % 2 == 0)), lo, hi)
    return np.copysign(t[k], q), s


def held(cache):
    return cache.codes.float().cpu().numpy().astype(np.float64), cache.scales.cpu().numpy()


def rows_of(n, D, t, seed):
    g = gen(seed)
    x = torch.randn(n, D, generator=g) * torch.exp(1.5 * torch.randn(D, generator=g)) * \
        torch.exp(torch.randn(n, 1, generator=g))
    return x.clamp(-3e4, 3e4).to(t)  # finite in every type


SIZES = [(1, 1), (1, 32), (3, 30), (33, 7), (50, 128), (9, 129), (200, 33), (64, 64), (5, 1000), (17, 515), (700, 16)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n,D", SIZES)
def test_write_and_read(fmt, t, n, D):
    for k, group in enumerate(R.GROUPS):
        cap = 2 * n + 3
        x = rows_of(n, D, t, n + D + k)
        slots = torch.randperm(cap, generator=gen(k))[:n].to(torch.int32 if k % 2 else torch.int64)
        c = R.rowcache_alloc(cap, D, fmt, group, DEV)
        R.rowcache_write(c, x.to(DEV), slots.to(DEV))
        q, s = want_write(x.float().numpy(), fmt, group)
        codes, scales = np.zeros((cap, D)), np.zeros((cap, s.shape[1]), np.float32)
        codes[slots.numpy()], scales[slots.numpy()] = q, s
        got_c, got_s = held(c)
        np.testing.assert_array_equal(got_s, scales)
        np.testing.assert_array_equal(got_c, codes)
        want = torch.from_numpy(codes * np.repeat(scales.astype(np.float64), group, 1)[:, :D])
        for ot in (F32, F16, BF16):
            h = 0 if ot == F32 else torch.finfo(ot).eps / 2
            tiny = 2.0 ** -25 if ot == F16 else 0
            tol = (2.0 ** -24 + h) * (1 + 2.0 ** -24) * want.abs() + tiny
            over = want.abs() > torch.finfo(ot).max  # f16: rows beyond its range read back as infinities
            for sl in (None, slots):
                y = R.rowcache_read(c, None if sl is None else sl.to(DEV), dtype=ot).cpu().double()
                w, e, o = (want, tol, over) if sl is None else (want[sl.long()], tol[sl.long()], over[sl.long()])
                assert y.shape == w.shape and (((y - w).abs() <= e) | (o & y.isinf())).all()
        # the value read back is within half a step of the one written
        y = R.rowcache_read(c, slots.to(DEV)).cpu().double()
        per = torch.from_numpy(np.repeat(s.astype(np.float64), group, 1)[:, :D])
        xd = x.double()
        bound = per * 0.5 if fmt == "int8" else torch.maximum(xd.abs() * 2.0 ** -4, per * 2.0 ** -10)
        assert ((y - xd).abs() <= bound + xd.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_borders_between_codes(fmt):
    """Values on the border of two codes, and the f32 numbers beside it, at scales that are no powers of two."""
    t = np.arange(0, 128.0) if fmt == "int8" else e4m3_table()
    mid = (t[1:] + t[:-1]) / 2
    rows = []
    for amax in (1.0, 448.0, 0.3712, 1e-20, 7.7e29, 3.1e-36):
        s = np.float32(max(np.float32(amax) * (np.float32(1) / np.float32(TOP[fmt])), np.float32(2.0 ** -100)))
        b = (np.concatenate([mid, t]) * np.float64(s)).astype(np.float32)
        for x in (b, np.nextafter(b, np.float32(0)), np.nextafter(b, np.float32(np.inf))):
            x = np.minimum(x, np.float32(amax))
            for sign in (1, -1):
                row = np.zeros((len(x), 16), np.float32)
                row[:, 3], row[:, 9] = amax, sign * x
                rows.append(row)
    x = np.concatenate(rows)
    c = R.rowcache_alloc(len(x), 16, fmt, 16, DEV)
    R.rowcache_write(c, torch.from_numpy(x).to(DEV))
    q, s = want_write(x, fmt, 16)
    got_c, got_s = held(c)
    np.testing.assert_array_equal(got_s, s)
    np.testing.assert_array_equal(got_c, q)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_extreme_rows(fmt):
    big = torch.finfo(F32).max
    x = torch.zeros(10, 64)
    x[1] = big
    x[2, 5] = big
    x[2, 6] = 1e-45
    x[3] = 1e-45          # below the smallest scale: codes 0
    x[4, 40] = float("nan")
    x[5, 3] = float("inf")
    x[6, 3], x[6, 40] = -float("inf"), 2.0
    x[7] = -0.0
    x[8] = 2.0 ** -100
    x[9] = torch.arange(64) * 1e-38
    c = R.rowcache_alloc(10, 64, fmt, 32, DEV)
    R.rowcache_write(c, x.to(DEV))
    q, s = want_write(x.numpy(), fmt, 32)
    got_c, got_s = held(c)
    np.testing.assert_array_equal(got_s, s)
    np.testing.assert_array_equal(got_c, q)
    y = R.rowcache_read(c).cpu()
    assert y[0].eq(0).all() and y[3].eq(0).all() and y[7].eq(0).all()
    assert y[4, 32:].isnan().all() and y[4, :32].eq(0).all() and y[5, :32].isnan().all() and y[5, 32:].eq(0).all()
    assert y[6, :32].isnan().all() and float(y[6, 40]) == 2.0


@pytest.mark.parametrize("n,cap", [(2, 4), (70, 23), (1000, 333), (1024, 100), (1025, 100), (1100, 4), (5000, 1666),
                                   (16_385, 16_384), (40_000, 16_385), (60_000, 20_000), (60_000, 7),
                                   (33_000, 16_384), (3000, 4_000_000)])
def test_repeated_and_outside_slots(n, cap):
    """The last row of a slot stays, rows outside the cache are left out, other slots keep what they hold."""
    D = 32
    x = torch.randn(n, D, generator=gen(n))
    slots = torch.randint(-2, cap + 2, (n,), generator=gen(n + 1))
    slots[slots == 1] = 0  # slot 1 is not named
    if n > 2:
        slots[-2:] = cap - 1
    c = R.rowcache_alloc(cap, D, "int8", 32, DEV)
    base = torch.randn(min(cap, 70_000), D, generator=gen(n + 2)).repeat(-(-cap // 70_000), 1)[:cap]
    R.rowcache_write(c, base.to(DEV))
    R.rowcache_write(c, x.to(DEV), slots.to(DEV))
    final = base.clone()
    for i, k in enumerate(slots.tolist()):
        if 0 <= k < cap:
            final[k] = x[i]
    q, s = want_write(final.numpy(), "int8", 32)
    got_c, got_s = held(c)
    np.testing.assert_array_equal(got_s, s)
    np.testing.assert_array_equal(got_c, q)
    y = R.rowcache_read(c, slots.to(DEV)).cpu()
    every = R.rowcache_read(c).cpu()
    ok = (slots >= 0) & (slots < cap)
    assert y[~ok].eq(0).all() and torch.equal(y[ok], every[slots[ok]])
    one = torch.full((n,), cap - 1, device=DEV)  # one slot for every row
    R.rowcache_write(c, x.to(DEV), one)
    assert torch.equal(c.codes[cap - 1].cpu().double(), torch.from_numpy(want_write(x[-1:].numpy(), "int8", 32)[0])[0])


@pytest.mark.parametrize("n,D,group,kind", [(2048, 40, 16, "two"), (2049, 40, 16, "two"), (2048, 2048, 128, "two"),
                                            (2048, 2064, 16, "two"), (700, 33_000, 64, "two"), (1000, 16, 16, "same place"),
                                            (2048, 20, 32, "power"), (2048, 16, 16, "padded")])
def test_last_rows_of_few(n, D, group, kind):
    """Each slot named about twice, by rows of every width; slots that one hash sends to one place."""
    cap = 1 << 22 if D < 32 else n
    if kind == "same place":  # the last place of a table of 2^11, so that the search wraps around
        v = np.arange(cap, dtype=np.uint64)
        slots = torch.from_numpy(v[((v * 0x9e3779b9) & 0xffffffff) >> 21 == 2047][:n // 2].astype(np.int64)).repeat(2)
    elif kind == "power":
        slots = torch.arange(n // 2).repeat_interleave(2) << 11
    else:
        slots = torch.randint(0, n // 2, (n,), generator=gen(n + D))
        if kind == "padded":
            slots[::3] = -1
    x = torch.randn(n, D, generator=gen(D))
    c = R.rowcache_alloc(cap, D, "int8", group, DEV)
    R.rowcache_write(c, x.to(DEV), slots.to(DEV))
    last = {k: i for i, k in enumerate(slots.tolist()) if k >= 0}
    at, rows = torch.tensor(list(last)), torch.tensor(list(last.values()))
    q, s = want_write(x[rows].numpy(), "int8", group)
    np.testing.assert_array_equal(c.codes[at.to(DEV)].cpu().numpy(), q)
    np.testing.assert_array_equal(c.scales[at.to(DEV)].cpu().numpy(), s)
    rest = torch.ones(cap, dtype=torch.bool, device=DEV)
    rest[at.to(DEV)] = False
    assert not c.scales[rest].any()  # no other slot was written


@pytest.mark.parametrize("n", [1025, 2048, 2049, 30_000])
@pytest.mark.parametrize("twice", [None, 0, 2047, -2])
def test_slots_in_order(n, twice):
    """Ascending slots, as a compacted index has them, with no slot or one slot named twice."""
    cap = n + n // 2
    slots = torch.randperm(cap, generator=gen(n))[:n].sort().values
    if twice is not None and twice + 1 < n:
        slots[twice + 1] = slots[twice]
    x = torch.randn(n, 32, generator=gen(n + 1))
    c = R.rowcache_alloc(cap, 32, "int8", 32, DEV)
    R.rowcache_write(c, x.to(DEV), slots.to(DEV))
    final = torch.zeros(cap, 32)
    final[slots] = x  # the later of two equal slots
    if twice is not None and twice + 1 < n:
        final[slots[twice]] = x[twice + 1]
    q, s = want_write(final[slots].numpy(), "int8", 32)
    np.testing.assert_array_equal(c.codes[slots.to(DEV)].cpu().numpy(), q)
    np.testing.assert_array_equal(c.scales[slots.to(DEV)].cpu().numpy(), s)


def test_every_code_reads_as_its_value():
    for fmt in ("int8", "e4m3"):
        bits = torch.arange(256, dtype=torch.uint8)
        c = R.RowCache(bits.reshape(1, 256).view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).to(DEV),
                       torch.ones(1, 16, device=DEV), 16)
        y = R.rowcache_read(c).cpu().numpy()[0].astype(np.float64)
        if fmt == "int8":
            np.testing.assert_array_equal(y, np.arange(256) - 256 * (np.arange(256) > 127))
        else:
            t = np.append(e4m3_table(), np.nan)
            np.testing.assert_array_equal(y, np.concatenate([t, -t]))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_strides(fmt):
    """A cache, rows and slots that are ranges of larger tensors; what lies beside them is left as it was."""
    x = torch.randn(20, 71, generator=gen(0))
    for a, b in ((0, 64), (1, 65), (3, 43), (4, 68)):
        D = b - a
        G = -(-D // 32)
        kind = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
        codes = torch.full((30, 80), 77, dtype=torch.uint8, device=DEV)
        scales = torch.full((30, 5), 3.0, device=DEV)
        c = R.RowCache(codes.view(kind)[2:28, a:b], scales[2:28, 1:1 + G], 32)
        slots = torch.randperm(52, generator=gen(a)).to(DEV)[::2] % 26
        slots = torch.unique(slots)[:12]
        R.rowcache_write(c, x.to(DEV)[:12, a:b], slots[:12])
        n = slots.numel()
        q, s = want_write(x[:n, a:b].numpy(), fmt, 32)
        np.testing.assert_array_equal(c.codes.view(torch.uint8)[slots].view(kind).float().cpu().numpy(), q)
        np.testing.assert_array_equal(c.scales[slots].cpu().numpy(), s)
        y = R.rowcache_read(c, slots)
        want = torch.from_numpy(q * np.repeat(s.astype(np.float64), 32, 1)[:, :D])
        assert ((y.cpu().double() - want).abs() <= 2.0 ** -24 * want.abs()).all()
        inside = torch.zeros(30, 80, dtype=torch.bool, device=DEV)
        inside[2:28, a:b] = True
        assert codes[~inside].eq(77).all()
        inside = torch.zeros(30, 5, dtype=torch.bool, device=DEV)
        inside[2:28, 1:1 + G] = True
        assert scales[~inside].eq(3.0).all()
    one = R.rowcache_alloc(4, 32, fmt, 32, DEV)
    R.rowcache_write(one, torch.ones(1, 32, device=DEV).expand(4, 32))  # one row for every slot
    assert R.rowcache_read(one, torch.full((), 2, device=DEV).expand(6)).eq(1).all()


def test_empty():
    c = R.rowcache_alloc(4, 8, device=DEV)
    e = torch.empty(0, dtype=torch.int64, device=DEV)
    R.rowcache_write(c, torch.empty(0, 8, device=DEV), e)
    assert R.rowcache_read(c, e).shape == (0, 8) and not R.rowcache_read(c).any()
    none = R.rowcache_alloc(0, 8, device=DEV)
    R.rowcache_write(none, torch.ones(2, 8, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV))
    assert R.rowcache_read(none, torch.zeros(2, dtype=torch.int32, device=DEV)).eq(0).all()
    assert R.rowcache_read(none).shape == (0, 8)


@pytest.mark.parametrize("n", [1, 50, 5000])
def test_captured_and_replayed(n):
    cap, D = 3000, 64
    x, slots = torch.zeros(n, D, device=DEV), torch.zeros(n, dtype=torch.int64, device=DEV)
    a = R.rowcache_alloc(cap, D, "e4m3", 64, DEV)
    b = R.rowcache_alloc(cap, D, "e4m3", 64, DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        R.rowcache_write(a, x, slots), R.rowcache_read(a, slots)
    torch.cuda.current_stream().wait_stream(s)
    graphs, reads = [], []
    for k in range(2):  # two graphs that write one cache, replayed one after the other
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            R.rowcache_write(a, x, slots)
            reads.append(R.rowcache_read(a, slots, dtype=BF16))
        graphs.append(gr)
    R.rowcache_write(b, x, slots)
    for rep in range(4):
        x.copy_(torch.randn(n, D, generator=gen(rep)))
        slots.copy_(torch.randint(-1, cap, (n,), generator=gen(rep + 9)))
        torch.cuda.synchronize()
        graphs[rep % 2].replay()
        torch.cuda.synchronize()
        R.rowcache_write(b, x, slots)
        assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
        assert torch.equal(reads[rep % 2], R.rowcache_read(b, slots, dtype=BF16))


def test_cache_beyond_2_31_bytes():
    cap, D = 2_200_000, 1024
    c = R.rowcache_alloc(cap, D, "int8", 128, DEV)
    slots = torch.tensor([cap - 1, 0, 2_097_152, cap], device=DEV)
    x = torch.randn(4, D, generator=gen(0))
    R.rowcache_write(c, x.to(DEV), slots)
    q, s = want_write(x.numpy(), "int8", 128)
    np.testing.assert_array_equal(c.codes[slots[:3]].cpu().numpy(), q[:3])
    y = R.rowcache_read(c, slots).cpu().double()
    want = torch.from_numpy(q * np.repeat(s.astype(np.float64), 128, 1))
    assert ((y[:3] - want[:3]).abs() <= 2.0 ** -24 * want[:3].abs()).all() and y[3].eq(0).all()
    whole = R.rowcache_read(c, dtype=BF16)  # 2.25e9 values out
    assert torch.equal(whole[cap - 1], R.rowcache_read(c, slots[:1], dtype=BF16)[0]) and not whole[5:2000].any()


def test_other_stream():
    c, d = (R.rowcache_alloc(9000, 32, device=DEV) for _ in range(2))
    x, slots = torch.randn(5000, 32, device=DEV), torch.randint(0, 9000, (5000,), device=DEV)
    R.rowcache_write(c, x, slots)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        R.rowcache_write(d, x, slots)
        y = R.rowcache_read(d, slots)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(c.codes, d.codes) and torch.equal(y, R.rowcache_read(c, slots))
