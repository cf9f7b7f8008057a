"""Step tables built on the device against a plain computation with lists, entry by entry: every number is whole, so all must be equal."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def K():
    from geneinfer_b200.ops import kernels
    return kernels


class Plain:
    """The tables as lists; the stack's places above its top keep what was there."""

    def __init__(self, R, stride, pool, page, seed=0):
        rng = np.random.default_rng(seed)
        self.R, self.stride, self.pool, self.page = R, stride, pool, page
        self.tables = np.full((R, stride), -1, dtype=np.int32)
        self.held = np.zeros(R, dtype=np.int32)
        self.free = rng.permutation(pool).astype(np.int32)
        self.n = pool

    def settle(self, lengths, counts=None, rows=None):
        """Status, and (row_start, row_req, positions, slots) where there are counts."""
        c = np.zeros_like(lengths) if counts is None else counts
        if (lengths < 0).any() or (c < 0).any() or (self.held < 0).any() or (self.held > self.stride).any() or not 0 <= self.n <= self.pool:
            return -3, None
        total = lengths.astype(np.int64) + c
        need = -(-total // self.page)
        if (need > self.stride).any():
            return -2, None
        if counts is not None and c.astype(np.int64).sum() > rows:
            return -1, None
        back, take = int(np.maximum(self.held - need, 0).sum()), int(np.maximum(need - self.held, 0).sum())
        if self.n + back > self.pool:
            return -4, None
        if take > self.n + back:
            return take - self.n - back, None
        for r in reversed(range(self.R)):
            for j in reversed(range(need[r], self.held[r])):
                self.free[self.n] = self.tables[r, j]
                self.tables[r, j] = -1
                self.n += 1
        for r in range(self.R):
            for j in range(self.held[r], need[r]):
                self.n -= 1
                self.tables[r, j] = self.free[self.n]
        self.held[:] = need
        if counts is None:
            return 0, None
        start = np.concatenate([[0], np.cumsum(c)]).astype(np.int32)
        req, pos, slot = np.full(rows, -1, dtype=np.int32), np.zeros(rows, dtype=np.int32), np.full(rows, -1, dtype=np.int32)
        for r in range(self.R):
            at = slice(start[r], start[r + 1])
            p = np.arange(lengths[r], lengths[r] + c[r])
            req[at], pos[at], slot[at] = r, p, self.tables[r, p // self.page] * self.page + p % self.page
        return 0, (start, req, pos, slot)


class Device:
    def __init__(self, plain):
        to = lambda x: torch.from_numpy(np.array(x, dtype=np.int32)).to(DEV)      # noqa: E731
        self.tables, self.held, self.free, self.n = to(plain.tables), to(plain.held), to(plain.free), to([plain.n])
        self.status = to([77])
        self.page = plain.page

    def settle(self, lengths, counts=None, rows=None):
        to = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(DEV)      # noqa: E731
        if counts is None:
            K().trim_tables(to(lengths), self.tables, self.held, self.free, self.n, self.page, self.status)
            return int(self.status), None
        out = [torch.full((n,), 77, dtype=torch.int32, device=DEV) for n in (len(lengths) + 1, rows, rows, rows)]
        K().step_tables(to(lengths), to(counts), self.tables, self.held, self.free, self.n, self.page, *out, self.status)
        return int(self.status), [x.cpu().numpy() for x in out]


def same(device, plain, got, want):
    assert got[0] == want[0]
    for a, b in ((device.tables, plain.tables), (device.held, plain.held), (device.free, plain.free)):
        assert np.array_equal(a.cpu().numpy(), b)
    assert int(device.n) == plain.n
    if want[1] is not None:
        for a, b in zip(got[1], want[1]):
            assert np.array_equal(a, b)
    elif got[1] is not None:                        # refused: nothing but the status is written
        assert all((x == 77).all() for x in got[1])


@pytest.mark.parametrize("R,page,most,rows", [(1, 16, 1, 1), (1, 1, 9, 20), (3, 16, 40, 130), (33, 7, 5, 200), (250, 16, 6, 1600), (1023, 16, 3, 4096),
                                              (1024, 8, 5, 5200), (1025, 16, 5, 4000), (2500, 64, 3, 9001), (40, 32, 900, 40000)])
def test_rounds_of_growing_rewinding_and_ending_requests(R, page, most, rows):
    """Rounds as a server has them: tokens for every request (some none), a rewind to what was kept, requests that end and start."""
    rng = np.random.default_rng(R + page)
    stride = -(-(6 * most + 40) // page)
    plain = Plain(R, stride, R * stride, page, seed=R)
    device = Device(plain)
    lengths = rng.integers(0, 40, R)
    for step in range(5):
        counts = np.where(rng.random(R) < 0.25, 0, rng.integers(0, most + 1, R))
        while counts.sum() > rows:
            counts //= 2
        want = plain.settle(lengths, counts, rows)
        assert want[0] == 0
        same(device, plain, device.settle(lengths, counts, rows), want)
        lengths = lengths + (counts * rng.random(R)).astype(np.int64)
        lengths[rng.random(R) < 0.15] = 0
        same(device, plain, device.settle(lengths), plain.settle(lengths))
    assert sorted(plain.free[:plain.n].tolist() + plain.tables[plain.tables >= 0].tolist()) == list(range(R * stride))


def test_pages_that_come_back_serve_others_in_the_same_call():
    plain = Plain(5, 8, 20, 4)
    device = Device(plain)
    for lengths, counts in (([30, 20, 0, 0, 9], [1, 4, 0, 0, 3]), ([1, 8, 0, 20, 9], [0, 0, 0, 7, 0]), ([0, 0, 0, 0, 0], [0, 0, 30, 0, 0])):
        lengths, counts = np.array(lengths), np.array(counts)
        want = plain.settle(lengths, counts, 64)
        assert want[0] == 0
        same(device, plain, device.settle(lengths, counts, 64), want)


def test_taken_and_given_back_whole_leaves_the_stack_as_it_was():
    plain = Plain(700, 12, 9000, 16, seed=5)
    device = Device(plain)
    lengths = np.random.default_rng(1).integers(0, 150, 700)
    device.settle(lengths)
    before = device.free.clone(), int(device.n)
    device.settle(lengths, np.full(700, 40), 30000)
    device.settle(lengths)
    assert int(device.n) == before[1] and torch.equal(device.free, before[0])


def test_all_or_nothing():
    plain = Plain(4, 5, 12, 4)
    device = Device(plain)
    lengths = np.array([4, 4, 4, 4])
    same(device, plain, device.settle(lengths), plain.settle(lengths))
    for lengths, counts, rows, status in (([4, 4, 4, 4], [12, 12, 12, 4], 64, 2), ([4, 4, 4, 4], [4, 4, 4, 4], 15, -1), ([4, 4, 4, 17], [0, 0, 0, 4], 64, -2),
                                          ([4, -1, 4, 4], [1, 1, 1, 1], 64, -3), ([4, 4, 4, 4], [1, 1, -5, 1], 64, -3),
                                          ([2 ** 31 - 1, 4, 4, 4], [2 ** 31 - 1, 0, 0, 0], 64, -2)):
        lengths, counts = np.array(lengths), np.array(counts)
        want = plain.settle(lengths, counts, rows)
        assert want[0] == status
        same(device, plain, device.settle(lengths, counts, rows), want)
    device.n.fill_(12)
    plain.n = 12                                             # a stack that cannot hold what comes back
    want = plain.settle(np.zeros(4, dtype=np.int64))
    assert want[0] == -4
    same(device, plain, device.settle(np.zeros(4, dtype=np.int64)), want)
    device.n.fill_(13)
    assert device.settle(np.array([4, 4, 4, 4]))[0] == -3


def test_more_rows_than_32_bits_count_are_refused():
    plain = Plain(3, 0x7fff, 10, 1 << 16)
    device = Device(plain)
    lengths, counts = np.zeros(3, dtype=np.int64), np.full(3, 2 ** 31 - 1 - (1 << 16))
    want = plain.settle(lengths, counts, 1000)
    assert want[0] == -1
    same(device, plain, device.settle(lengths, counts, 1000), want)


def test_no_requests_and_no_rows():
    plain = Plain(0, 3, 4, 16)
    device = Device(plain)
    none = np.zeros(0, dtype=np.int64)
    for rows in (0, 10, 5000):
        same(device, plain, device.settle(none, none, rows), plain.settle(none, none, rows))
    plain = Plain(3, 3, 9, 16)
    device = Device(plain)
    lengths = np.array([5, 0, 17])
    same(device, plain, device.settle(lengths, np.zeros(3, dtype=np.int64), 0), plain.settle(lengths, np.zeros(3, dtype=np.int64), 0))


def test_the_tables_are_what_the_engines_kernels_read():
    """Pages that step_tables has dealt, written through rope_store and read back at the rows' slots."""
    plain = Plain(3, 6, 18, 4, seed=3)
    device = Device(plain)
    lengths, counts = np.array([3, 0, 7]), np.array([6, 1, 3])
    status, (start, req, pos, slot) = device.settle(lengths, counts, 12)
    assert status == 0
    T, hd = 10, 16
    to = lambda x: torch.from_numpy(x).to(DEV)      # noqa: E731
    qkv = torch.randn(T, 3 * hd, generator=torch.Generator().manual_seed(1)).to(DEV)
    k, v = torch.zeros(18, 1, 4, hd, device=DEV), torch.zeros(18, 1, 4, hd, device=DEV)
    K().rope_store(qkv, to(pos[:T]), to(req[:T]), device.tables, None, None, False, torch.empty(T, hd, device=DEV), k, v, 1, 1, hd, 4)
    assert torch.equal(k.view(-1, hd)[to(slot[:T]).long()], qkv[:, hd:2 * hd]) and torch.equal(v.view(-1, hd)[to(slot[:T]).long()], qkv[:, 2 * hd:])
    assert int((k.view(-1, hd).abs().sum(1) > 0).sum()) == T


def test_on_a_stream_of_its_own_and_recorded():
    plain = Plain(300, 4, 1200, 16)
    device = Device(plain)
    lengths, counts = np.full(300, 10), np.full(300, 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with K().record() as rec:
            got = device.settle(lengths, counts, 6000)
    same(device, plain, got, plain.settle(lengths, counts, 6000))
    assert len(rec.program) == 1 and rec.program.launches == 2


def test_step_tables_refuses_what_does_not_fit():
    def ints(*shape):
        return torch.zeros(*shape, dtype=torch.int32, device=DEV)
    good = dict(lengths=ints(3), counts=ints(3), tables=ints(3, 4), held=ints(3), free_pages=ints(9), n_free=ints(1), page_size=16, row_start=ints(4),
                row_req=ints(5), positions=ints(5), slots=ints(5), status=ints(1))
    K().step_tables(**good)
    for name, value in (("lengths", ints(2)), ("lengths", ints(3).long()), ("counts", ints(4)), ("tables", ints(2, 4)), ("tables", ints(12)),
                        ("tables", ints(3, 8)[:, ::2]), ("held", ints(1)), ("free_pages", ints(9).cpu()), ("n_free", ints(2)), ("page_size", 0),
                        ("page_size", 1 << 30), ("row_start", ints(3)), ("positions", ints(4)), ("slots", ints(6)), ("row_req", ints(5).float()), ("status", ints(0))):
        with pytest.raises(K().KernelError):
            K().step_tables(**dict(good, **{name: value}))
    trim = {k: good[k] for k in ("lengths", "tables", "held", "free_pages", "n_free", "page_size", "status")}
    K().trim_tables(**trim)
    with pytest.raises(K().KernelError):
        K().trim_tables(**dict(trim, held=ints(4)))


def test_positions_beyond_32_bits_are_refused():
    """A table with room for three pages of 2^30 positions: a request of 2^31 positions is refused, one of 2^31 - 1 is not."""
    for length, count, status in ((2 ** 31 - 1, 5, -2), (2 ** 31 - 6, 6, -2), (2 ** 31 - 6, 5, 0)):
        out = [torch.full((n,), 77, dtype=torch.int32, device=DEV) for n in (2, 8, 8, 8)]
        held, tables = torch.tensor([3], dtype=torch.int32, device=DEV), torch.tensor([[0, 0, 0, -1]], dtype=torch.int32, device=DEV)
        n, free, word = (torch.tensor([v], dtype=torch.int32, device=DEV) for v in (0, 0, 77))
        if status == 0:
            held.fill_(2)
        to = lambda v: torch.tensor([v], dtype=torch.int32, device=DEV)      # noqa: E731
        K().step_tables(to(length), to(count), tables, held, free, n, 1 << 30, *out, word)
        assert int(word) == status
        if status:
            assert all(bool((x == 77).all()) for x in out) and int(held) == 3
        else:
            last = 2 ** 31 - 2
            assert out[2].tolist() == list(range(length, last + 1)) + [0] * 3 and out[3].tolist() == [p % (1 << 30) for p in range(length, last + 1)] + [-1] * 3
