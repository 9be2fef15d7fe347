"""Rows of tables of states: copied, cleared and compacted, against the same done row by row on the CPU (bit by bit)."""
import pytest
import torch

from ttt_tk_b200 import ssm, tables

pytestmark = pytest.mark.gpu

SHAPES = [((3, 64), torch.bfloat16), ((130,), torch.float32), ((7,), torch.float16), ((5,), torch.uint8), ((), torch.float64), ((2, 3, 17), torch.float32)]


def _make(S, shapes=SHAPES, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(S, *s, generator=g) * 50).to(t).cuda() for s, t in shapes]


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _copied(ts, source, target):
    out = []
    for t in ts:
        t = t.cpu()
        r = t.clone()
        for a, b in zip(source, target):
            if 0 <= a < len(t) and 0 <= b < len(t):
                r[b] = t[a]
        out.append(r)
    return out


def _check_copy(S, source, target, shapes=SHAPES):
    ts = _make(S, shapes)
    want = _copied(ts, source, target)
    assert tables.copy_rows(ts, _i32(source), _i32(target)) is None
    for a, b in zip(ts, want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("source,target", [([0], [1]), ([2, 2, 2], [0, 1, 4]), ([0, 1, 2, 3], [1, 2, 3, 0]), ([3, 1], [1, 3]), ([], []), ([1], [1]),
                                           ([-1, 0, 5, 9, 2], [2, -1, 1, 3, 4]), ([0, 1, 2], [4, 4, 4]), ([0, 99, 2, 3], [4, 4, -7, 1]),
                                           ([2 ** 31 - 1, 0], [0, -2 ** 31])])
def test_copy(source, target):
    """Forks, rings, swaps, pairs that do nothing, and several pairs with the same target, of which the last one counts."""
    _check_copy(5, source, target)


@pytest.mark.parametrize("S,n", [(1, 1), (64, 64), (300, 299), (1000, 700), (4096, 4096), (9000, 500)])
def test_copy_at_random(S, n):
    """As many pairs as there may be; more rows than a CTA marks; targets named twice."""
    g = torch.Generator().manual_seed(S)
    source, target = torch.randint(-1, S + 1, (n,), generator=g).tolist(), torch.randint(-1, S + 1, (n,), generator=g).tolist()
    _check_copy(S, source, target, [((3, 8), torch.bfloat16), ((33,), torch.float32), ((3,), torch.uint8)])
    perm = torch.randperm(S, generator=g)[:n].tolist()
    _check_copy(S, perm, perm[1:] + perm[:1], [((40,), torch.float32), ((5,), torch.float16)])


def test_copy_of_wide_rows():
    _check_copy(12, [3, 4, 5, 0], [4, 5, 3, 11], [((100003,), torch.float32), ((12, 64, 256), torch.float32), ((50001,), torch.bfloat16)])


def test_one_table_and_views_of_one_memory():
    t = torch.arange(40, dtype=torch.float32, device="cuda").view(2, 4, 5)
    tables.copy_rows(t[1], _i32([0]), _i32([3]))
    assert torch.equal(t[1, 3], t[1, 0]) and t[0, 3, 0] == 15
    tables.copy_rows([t[0], t[1]], _i32([1]), _i32([2]))      # neighbours that do not overlap
    assert torch.equal(t[0, 2], t[0, 1])


@pytest.mark.parametrize("rows", [[], [0], [4, 0, 4], [-1, 5, 2]])
def test_clear(rows):
    ts = _make(5)
    want = [t.cpu().clone() for t in ts]
    for t in want:
        for r in rows:
            if 0 <= r < 5:
                t[r] = 0
    tables.clear_rows(ts, _i32(rows))
    for a, b in zip(ts, want):
        assert torch.equal(a.cpu(), b)


def _check_compact(used, shapes=SHAPES):
    S, n = len(used), sum(used)
    ts = _make(S, shapes)
    want = [t.cpu().clone() for t in ts]
    place = [k if u else -1 for k, u in enumerate(used)]
    for a, b in zip([k for k in range(n, S) if used[k]], [k for k in range(n) if not used[k]]):
        place[a] = b
        for t in want:
            t[b] = t[a]
    got = tables.compact_rows(ts, torch.tensor(used, dtype=torch.bool, device="cuda"))
    assert got.dtype == torch.int32 and got.tolist() == place
    for a, b in zip(ts, want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("used", [[1], [0], [0, 1], [1, 0], [0, 0, 0, 1], [1, 1, 1], [0, 0], [0, 1, 0, 1, 0, 1, 1], [1, 0] * 200, [0, 1] * 257])
def test_compact(used):
    _check_compact([bool(u) for u in used])


@pytest.mark.parametrize("S,share", [(255, 0.5), (256, 0.1), (257, 0.9), (8192, 0.5)])
def test_compact_at_random(S, share):
    used = (torch.rand(S, generator=torch.Generator().manual_seed(S)) < share).tolist()
    _check_compact(used, [((3, 8), torch.bfloat16), ((33,), torch.float32)])


def test_no_rows():
    t = torch.zeros(0, 4, device="cuda")
    tables.copy_rows(t, _i32([0]), _i32([0]))
    tables.clear_rows(t, _i32([0]))
    assert tables.compact_rows(t, torch.zeros(0, dtype=torch.bool, device="cuda")).shape == (0,)
    wide = torch.zeros(3, 0, device="cuda")
    tables.copy_rows(wide, _i32([0]), _i32([1]))
    assert tables.compact_rows(wide, torch.tensor([False, True, False], device="cuda")).tolist() == [-1, 0, -1]


def test_rows_beyond_4_gigabytes():
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB")
    t = torch.zeros(3, (1 << 30) + 8, device="cuda")
    t[2, -1], t[2, 0], t[1, -1] = 5.0, 3.0, 7.0
    tables.copy_rows(t, _i32([2, 1]), _i32([0, 2]))
    assert t[0, -1] == 5 and t[0, 0] == 3 and t[2, -1] == 7
    place = tables.compact_rows(t, torch.tensor([False, True, True], device="cuda"))
    assert place.tolist() == [-1, 1, 0] and t[0, -1] == 7


def test_a_captured_graph_and_another_stream():
    ts = _make(6)
    source, target, used = _i32([0, 1]), _i32([1, 5]), torch.tensor([1, 0, 1, 0, 0, 1], dtype=torch.bool, device="cuda")
    tables.copy_rows(ts, source, target)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tables.copy_rows(ts, source, target)
        place = tables.compact_rows(ts, used)
        tables.clear_rows(ts, target)
    for k in (1, 2):
        fresh = _make(6, seed=k)
        for a, b in zip(ts, fresh):
            a.copy_(b)
        source.copy_(_i32([k, 4]))
        used.copy_(torch.tensor([0, 1, 0, 0, k == 1, 1], dtype=torch.bool))
        g.replay()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            tables.copy_rows(fresh, source, target)
            want = tables.compact_rows(fresh, used)
            tables.clear_rows(fresh, target)
        s.synchronize()
        assert torch.equal(place, want)
        for a, b in zip(ts, fresh):
            assert torch.equal(a, b)


def test_samples_of_a_request():
    """A prompt, its states forked to three samples, a step of each, one that ends, and the rest in front: every sample goes on as if it had been alone."""
    D = 96
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    w, A = r(D, 4), -torch.rand(D, generator=g).cuda()
    q = r(1, 20, 2 * D)
    windows, states = torch.full((6, 3, D), 9.0, device="cuda"), torch.full((6, D), 9.0, device="cuda")
    both = [windows, states]
    tables.clear_rows(both, _i32([4]))
    u, win = ssm.short_conv(q[..., :D], w, state=windows[4:5], return_state=True)
    y, st = ssm.gated_scan(u, q[..., D:], A, state=states[4:5], return_state=True)
    windows[4], states[4] = win[0], st[0]
    tables.copy_rows(both, _i32([4, 4]), _i32([2, 5]))
    slots = _i32([4, 2, 5])
    tokens = r(3, 3, 2 * D)      # step, sample
    alone = []
    for k in range(3):
        seq = torch.cat([q, tokens[:, k][None]], 1)
        alone.append(ssm.gated_scan(ssm.short_conv(seq[..., :D], w), seq[..., D:], A))

    def step(t, which, slots):
        x = ssm.short_conv_step(tokens[t, which][:, :D], windows, w, slots=slots)
        return ssm.gated_scan_step(x, tokens[t, which][:, D:], states, A, slots=slots)

    for t in range(3):
        which = [0, 1, 2] if t < 2 else [0, 2]
        if t == 2:      # the second sample has ended
            used = torch.zeros(6, dtype=torch.bool, device="cuda")
            used[[4, 5]] = True
            place = tables.compact_rows(both, used)
            slots = place[slots.long()]
            assert slots.tolist() == [0, -1, 1]
            slots = slots[[0, 2]]
        y = step(t, which, slots)
        for j, k in enumerate(which):
            torch.testing.assert_close(y[j], alone[k][0, 20 + t], rtol=2e-5, atol=2e-5)
