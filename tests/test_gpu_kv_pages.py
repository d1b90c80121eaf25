"""Pages copied, shared, reserved, freed and moved together: equal to plain Python (kv8_ref)."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


def to(dev, *a):
    return [torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(dev) for x in a]


def make_caches(rng, L, NB, sizes=((np.uint8, (4, 16, 32)), (np.uint8, (4,)), (np.float16, (2, 16, 8)), (np.uint8, (3,)))):
    return [rng.integers(0, 200, (L, NB, *s)).astype(t) for t, s in sizes]


def dev_caches(caches, dev):
    return [torch.from_numpy(c.copy()).to(dev) for c in caches]


def same(dev_tensors, arrays, what=""):
    for i, (d, a) in enumerate(zip(dev_tensors, arrays)):
        assert (d.cpu().numpy() == a).all(), (what, i, np.argwhere(d.cpu().numpy() != a)[:4].tolist())


class State:
    """Rows of random lengths over pages in random order, some shared."""

    def __init__(self, rng, B, mb, NB, bs, fill=0.6, L=2):
        self.rng, self.bs = rng, bs
        self.table = np.full((B, mb), -1, np.int32)
        self.seq = np.zeros(B, np.int32)
        self.ref = np.zeros(NB, np.int32)
        free = rng.permutation(NB).tolist()
        for r in range(B):
            n = int(rng.integers(0, mb * bs + 1))
            pages = -(-n // bs)
            if pages > len(free) or len(free) < NB * (1 - fill):
                continue
            self.table[r, :pages] = [free.pop() for _ in range(pages)]
            self.ref[self.table[r, :pages]] += 1
            self.seq[r] = n
        self.caches = make_caches(rng, L, NB)

    def to(self, dev):
        return to(dev, self.table, self.seq, self.ref)

    def same(self, d, dc=None, what=""):
        same(d, (self.table, self.seq, self.ref), what)
        if dc is not None:
            same(dc, self.caches, what + " caches")


@pytest.mark.parametrize("n,NB,L", [(1, 2, 1), (5, 16, 3), (190, 1000, 2), (700, 5000, 1)])
def test_copy(mk, dev, n, NB, L):
    rng = np.random.default_rng(n)
    caches = make_caches(rng, L, NB)
    src, dst = rng.integers(0, NB, (2, n))
    src[0] = (dst[0] + 1) % NB
    d, (s, t) = dev_caches(caches, dev), to(dev, src, dst)
    status = mk.kv_copy_pages(d, s, t)
    want = R.copy_pages(caches, src, dst)
    assert status.tolist() == want
    same(d, caches)
    assert n == 1 or R.REFUSED in want


def test_copy_refuses_pairs(mk, dev):
    """Pages outside, a page copied onto twice, a page copied onto and from; onto itself is done."""
    rng = np.random.default_rng(0)
    caches = make_caches(rng, 2, 12)
    src = [0, 1, 2, 3, -1, 4, 12, 5, 6, 0]
    dst = [7, 8, 8, 4, 9, 10, 9, -3, 6, 11]
    d = dev_caches(caches, dev)
    status = mk.kv_copy_pages(d, *to(dev, src, dst))
    want = R.copy_pages(caches, src, dst)
    assert status.tolist() == want == [0, 0, 2, 2, 2, 0, 2, 2, 0, 0]
    same(d, caches)


def test_copy_of_any_tensors(mk, dev):
    """Pages of odd sizes, at odd addresses; half and float caches; none written but the listed."""
    rng = np.random.default_rng(1)
    for dtype, shape in ((np.uint8, (1,)), (np.uint8, (7, 3)), (np.float32, (5,)), (np.float16, (3,)),
                         (np.uint8, (16,)), (np.float16, (4, 16, 128))):
        base = rng.integers(0, 100, (3, 10, *shape)).astype(dtype)
        flat = torch.from_numpy(np.concatenate([np.zeros(1, dtype), base.reshape(-1)])).to(dev)
        view = flat[1:].view(3, 10, *shape)
        mk.kv_copy_pages([view], *to(dev, [3, 9], [0, 4]))
        R.copy_pages([base], [3, 9], [0, 4])
        same([view], [base], str((dtype, shape)))


@pytest.mark.parametrize("B,mb,NB,bs", [(1, 1, 1, 16), (20, 12, 150, 16), (300, 5, 900, 4), (7, 300, 2500, 1)])
def test_fork_reserve_free(mk, dev, B, mb, NB, bs):
    """A long run of calls on one state, each with rows that repeat or lie outside."""
    rng = np.random.default_rng(B)
    st = State(rng, B, mb, NB, bs)
    d, dc = st.to(dev), dev_caches(st.caches, dev)
    for step in range(6):
        n = int(rng.integers(1, B + 3))
        rows = rng.integers(-1, B + 1, n)
        mk.kv_free(*d, *to(dev, rows))
        R.free(st.table, st.seq, st.ref, rows)
        st.same(d, dc, f"free {step}")
        n = int(rng.integers(1, 2 * B + 2))
        parents, kids = rng.integers(-1, B + 1, (2, n))
        got = mk.kv_fork(*d, *to(dev, parents, kids))
        assert got.tolist() == R.fork(st.table, st.seq, st.ref, parents.tolist(), kids.tolist())
        st.same(d, dc, f"fork {step}")
        n = int(rng.integers(1, B + 3))
        rows = rng.permutation(np.concatenate([np.arange(-1, B + 1)] * 2))[:n]
        more = rng.integers(0, 2 * bs + 1, n) if step % 2 else rng.integers(0, mb * bs + 2, n)
        lens = np.where((rows >= 0) & (rows < B), st.seq[np.clip(rows, 0, B - 1)] + more, 5) if step % 2 else more
        got = mk.kv_reserve(dc, *d, *to(dev, rows, lens), bs)
        assert got.tolist() == R.reserve(st.caches, st.table, st.seq, st.ref, rows, lens, bs)
        st.same(d, dc, f"reserve {step}")
        # what the counts stand for
        held = np.bincount(st.table[st.table >= 0], minlength=NB)
        assert (held == st.ref).all()


def test_reserve_serves_in_order_until_the_pages_end(mk, dev):
    """The first row that does not fit and all behind it keep everything, one that needs nothing too.
    Of NB - 1 free pages row 0 takes a copy and two, row 3 one, row 1 a copy and three; row 2, by
    then the only holder of the shared page, and row 4 need none."""
    for NB, want in ((9, [0, 0, 0, 0, 0]), (8, [0, 0, 1, 1, 1]), (5, [0, 0, 1, 1, 1]), (4, [0, 1, 1, 1, 1]),
                     (3, [1, 1, 1, 1, 1])):
        table = np.full((6, 4), -1, np.int32)
        table[0, 0] = table[1, 0] = table[2, 0] = 2  # three rows on one page, partly full
        seq = np.array([3, 3, 3, 0, 0, 0], np.int32)
        ref = np.zeros(NB, np.int32)
        ref[2] = 3
        caches = make_caches(np.random.default_rng(NB), 1, NB)
        d, dc = to(dev, table, seq, ref), dev_caches(caches, dev)
        rows, lens = [0, 3, 1, 2, 4], [40, 1, 50, 4, 0]
        got = mk.kv_reserve(dc, *d, *to(dev, rows, lens), 16)
        assert got.tolist() == R.reserve(caches, table, seq, ref, rows, lens, 16) == want, NB
        same(d, (table, seq, ref), str(NB))
        same(dc, caches, str(NB))


def test_reserve_over_many_rows_and_pages(mk, dev):
    """1024 rows; free pages far behind the first thousands; a row that takes thousands."""
    rng = np.random.default_rng(4)
    B, mb, NB, bs = 1024, 6, 30000, 8
    ref = (rng.random(NB) < 0.97).astype(np.int32)
    table = np.full((B, mb), -1, np.int32)
    seq = np.zeros(B, np.int32)
    caches = [np.zeros((1, NB, 2), np.uint8)]
    d, dc = to(dev, table, seq, ref), dev_caches(caches, dev)
    rows, lens = rng.permutation(B), rng.integers(0, 12, B)
    got = mk.kv_reserve(dc, *d, *to(dev, rows, lens), bs)
    assert got.tolist() == R.reserve(caches, table, seq, ref, rows, lens, bs)
    assert R.FULL in got.tolist()
    same(d, (table, seq, ref))
    table, seq, ref = np.full((2, 9000), -1, np.int32), np.zeros(2, np.int32), np.zeros(20000, np.int32)
    d = to(dev, table, seq, ref)
    dc = dev_caches([np.zeros((1, 20000, 1), np.uint8)], dev)
    got = mk.kv_reserve(dc, *d, *to(dev, [1, 0], [70001, 9]), bs)
    assert got.tolist() == R.reserve([np.zeros((1, 20000, 1))], table, seq, ref, [1, 0], [70001, 9], bs) == [0, 0]
    same(d, (table, seq, ref))


@pytest.mark.parametrize("B,mb,NB", [(1, 1, 1), (6, 9, 40), (60, 40, 5000), (300, 20, 9001)])
@pytest.mark.parametrize("fill", [0.1, 0.9])
def test_compact(mk, dev, B, mb, NB, fill):
    rng = np.random.default_rng(NB)
    st = State(rng, B, mb, NB, 16, fill)
    if B > 2:
        parents, kids = [0, 0], [B - 1, B - 2]
        R.free(st.table, st.seq, st.ref, kids)
        R.fork(st.table, st.seq, st.ref, parents, kids)
        st.table[1, -1] = NB + 5  # an entry that is no page
    st.ref[rng.integers(0, NB, 3)] += 1  # pages that something else holds
    d, dc = st.to(dev), dev_caches(st.caches, dev)
    moved = mk.kv_compact(dc, d[0], d[2])
    want = R.compact(st.caches, st.table, st.ref)
    assert (moved.cpu().numpy() == want).all()
    st.same(d, dc)
    n = int((st.ref > 0).sum())
    assert (st.ref[:n] > 0).all() and (st.ref[n:] == 0).all()
    again = mk.kv_compact(dc, d[0], d[2])  # nothing left to move
    st.same(d, dc)
    assert (again.cpu().numpy() == np.where(st.ref > 0, np.arange(NB), -1)).all()


def test_compact_full_and_empty(mk, dev):
    for value in (0, 1):
        ref = np.full(5000, value, np.int32)
        table = np.full((2, 3), -1, np.int32)
        caches = make_caches(np.random.default_rng(0), 1, 5000)
        d, dc = to(dev, table, ref), dev_caches(caches, dev)
        moved = mk.kv_compact(dc, *d)
        assert (moved.cpu().numpy() == (np.arange(5000) if value else -1)).all()
        same(d, (table, ref))
        same(dc, caches)


def test_copy_past_4_gib(mk, dev):
    NB = 40
    big = torch.zeros((2, NB, (1 << 32) // 64), dtype=torch.uint8, device=dev)  # 5 GiB
    big[1, 3] = 5
    big[1, 3, -1] = 9
    mk.kv_copy_pages([big], *to(dev, [3], [NB - 1]))
    assert int(big[1, NB - 1].sum()) == 5 * (big.shape[2] - 1) + 9 and int(big[1, NB - 2].sum()) == 0
    assert int(big[0].sum()) == 0


def test_stream_and_graph(mk, dev):
    """A beam step captured: freed, forked, given room; replayed over changing states."""
    rng = np.random.default_rng(7)
    B, mb, NB, bs = 12, 8, 120, 16
    st = State(rng, B, mb, NB, bs, fill=0.4)
    d, dc = st.to(dev), dev_caches(st.caches, dev)
    kids, parents = np.arange(6, 12), np.array([0, 0, 1, 1, 2, 2])
    lens = np.full(6, 20)
    dk, dp, dl = to(dev, kids, parents, lens)
    s1, s2 = (torch.empty(6, dtype=torch.int32, device=dev) for _ in range(2))
    ws = torch.empty(mk.kv_pages_workspace_bytes(NB, 6) // 4, dtype=torch.int32, device=dev)
    moved = torch.empty(NB, dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step(stream=None):
        mk.kv_free(*d, dk, stream=stream)
        mk.kv_fork(*d, dp, dk, status=s1, stream=stream)
        mk.kv_reserve(dc, *d, dk, dl, bs, status=s2, workspace=ws, stream=stream)
        mk.kv_compact(dc, d[0], d[2], moved=moved, workspace=ws, stream=stream)

    def plain():
        R.free(st.table, st.seq, st.ref, kids)
        a = R.fork(st.table, st.seq, st.ref, parents.tolist(), kids.tolist())
        b = R.reserve(st.caches, st.table, st.seq, st.ref, kids, lens, bs)
        m = R.compact(st.caches, st.table, st.ref)
        return a, b, m

    def check(what):
        a, b, m = plain()
        assert s1.tolist() == a and s2.tolist() == b and (moved.cpu().numpy() == m).all(), what
        st.same(d, dc, what)

    step(side)
    side.synchronize()
    check("stream")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        lens = rng.integers(0, mb * bs, 6)
        dl.copy_(torch.from_numpy(lens.astype(np.int32)))
        graph.replay()
        check(f"replay {i}")


def test_binding_checks(mk, dev):
    i = torch.zeros(4, dtype=torch.int32, device=dev)
    c = torch.zeros((1, 4, 2), dtype=torch.uint8, device=dev)
    with pytest.raises(ValueError, match="as many"):
        mk.kv_copy_pages([c], i, i[:3])
    with pytest.raises(ValueError, match="num_blocks"):
        mk.kv_compact([c, c[:, :3].contiguous()], i.view(2, 2), i)
    with pytest.raises(ValueError, match="contiguous"):
        mk.kv_copy_pages([torch.zeros((2, 4, 2), device=dev).transpose(0, 1)], i, i)
    with pytest.raises(TypeError):
        mk.kv_copy_pages([c], i.long(), i)
    with pytest.raises(RuntimeError, match="-3"):
        mk.kv_copy_pages([c, c], i, i)
    with pytest.raises(ValueError):
        mk.kv_copy_pages([], i, i)
