"""Tables of many rows: the last of several pairs with the same target counts, and finding it takes no longer than in a small table."""
import pytest
import torch

from ttt_tk_b200 import tables

pytestmark = pytest.mark.gpu


def _pairs(S, n, targets, seed=0):
    g = torch.Generator().manual_seed(seed)
    source = torch.randint(-2, S + 2, (n,), generator=g, dtype=torch.int32)
    pool = torch.randperm(S, generator=g)[:targets].to(torch.int32)
    return source, pool[torch.randint(0, targets, (n,), generator=g)]


@pytest.mark.parametrize("S,n,targets", [(8192, 4096, 4096), (8193, 4096, 4096), (20000, 4096, 3), (20000, 4095, 1), (100000, 4096, 4000), (1 << 20, 2049, 2049), (9000, 1, 1),
                                         (3, 4096, 3), (70, 2, 1)])
def test_the_last_pair_counts(S, n, targets):
    source, target = _pairs(S, n, min(targets, S))
    ts = [torch.randn(S, 5, generator=torch.Generator().manual_seed(1)), torch.arange(S, dtype=torch.int64)]
    want = [t.clone() for t in ts]
    for a, b in zip(source.tolist(), target.tolist()):
        if 0 <= a < S:
            for r, t in zip(want, ts):
                r[b] = t[a]
    dev = [t.cuda() for t in ts]
    tables.copy_rows(dev, source.cuda(), target.cuda())
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, want))


def test_targets_that_fall_together():
    """Rows at distances of powers of two and of the golden ratio's multiples, which a table of marks may put in the same place."""
    S = 1 << 22
    for step in (1 << 9, 1 << 10, 2654435769 % S, 40503):
        target = (torch.arange(4096, dtype=torch.int64) * step % S).to(torch.int32)
        t = torch.arange(S, dtype=torch.int32, device="cuda")
        source = torch.arange(4096, dtype=torch.int32) + 17
        want = torch.arange(S, dtype=torch.int32)
        for a, b in zip(source.tolist(), target.tolist()):
            want[b] = a
        tables.copy_rows(t, source.cuda(), target.cuda())
        assert torch.equal(t.cpu(), want)


def test_the_time_does_not_jump():
    """4096 pairs among 8193 rows and among 8192, microseconds: some tens; a search through all later pairs took tens of times as long."""
    took = {}
    for S in (8192, 8193):
        t = torch.randn(S, 1024, device="cuda")
        g = torch.Generator().manual_seed(2)
        source, target = (torch.randperm(S, generator=g)[:4096].to(torch.int32).cuda() for _ in range(2))
        for _ in range(3):
            tables.copy_rows(t, source, target)
        best = float("inf")
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                tables.copy_rows(t, source, target)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b) * 200)
        took[S] = best
    print(took)
    assert took[8193] < 3 * took[8192], took
