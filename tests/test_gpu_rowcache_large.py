"""GPU checks of cache writes of millions of rows: more than one turn of the launches that look for repeated slots
takes, and work that grows with the rows and not with their square."""
import numpy as np
import pytest
import torch

from horizongs_amd import rowcache as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("cap", [300, 16_384, 16_385, 3_000_000])
@pytest.mark.parametrize("n", [1_048_577, 4_194_305, 9_000_001])
def test_writes_of_millions_of_rows(n, cap):
    """More rows than one turn of the launch that finds the last row of each slot takes; rows of two values,
    the row's number in both, so that the slot shows which one it holds."""
    slots = torch.randint(-1, cap + 1, (n,), generator=gen(n + cap)).to(DEV)
    slots[n - 1] = slots[0] = 7
    x = torch.empty(n, 2, device=DEV)
    x[:, 0], x[:, 1] = torch.arange(n, device=DEV) // 4096 + 1, torch.arange(n, device=DEV) % 4096 + 1
    c = R.rowcache_alloc(cap, 2, "e4m3", 16, DEV)
    R.rowcache_write(c, x, slots)
    last = torch.full((cap + 2,), -1, device=DEV).scatter_reduce_(0, (slots + 1), torch.arange(n, device=DEV), "amax")[1:cap + 1]
    want = R.rowcache_alloc(cap, 2, "e4m3", 16, DEV)
    named = torch.nonzero(last >= 0).reshape(-1)  # no slot twice, in order
    R.rowcache_write(want, x[last[named]], named)
    assert torch.equal(c.scales, want.scales) and torch.equal(c.codes.view(torch.uint8), want.codes.view(torch.uint8))
    assert int(last[7]) == n - 1 and float(c.scales[7]) == float((x[n - 1].amax() * np.float32(1 / 448)))


def test_time_grows_with_the_rows():
    """Rows in order, a number each.  Ten times the rows take ten times as long (measured: 10.1); where every
    workgroup of a launch reads something of every other's rows they take twenty times as long."""
    ms = []
    for n in (10_000_000, 100_000_000):
        slots = torch.arange(n, device=DEV, dtype=torch.int32)
        x, c = torch.ones(n, 2, device=DEV), R.rowcache_alloc(n, 2, "int8", 16, DEV)
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            R.rowcache_write(c, x, slots)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        ms.append(min(times))
    assert ms[1] < 15 * ms[0], ms
