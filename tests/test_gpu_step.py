"""Page tables advanced on the device, rows rotated at positions of their own
and the ends of blocks, against numpy.

Tables are whole numbers: equal to a restatement that gives and takes one page at
a time.  Rotations are equal to the bit to the two products and the sum of
float32.  Block ends are compared in 64 bits, u = 2^-24: a sum of n squares, held
by up to 1024 threads with 4 in a step and joined over a tree and 16 waves, is
off by (n / 4096 + 40) u = D u of itself, its root and inverse by D / 2 + 4, the
normed value by three more products."""
import numpy as np
import pytest

import kvad_amd as K

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.fixture()
def dctx(ctx):
    """The context and torch on one stream, so that their work is in order."""
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        ctx.set_stream(stream.cuda_stream)
        yield ctx
        torch.cuda.synchronize()
    ctx.set_stream(None)


# ---- page tables ---------------------------------------------------------------

class Tables:
    """A PageTable and its restatement."""

    def __init__(self, ctx, n_seq, max_pages, page, n_pages):
        self.ctx, self.page, self.cap = ctx, page, max_pages * page
        i32 = lambda *shape: torch.full(shape, 77, dtype=torch.int32, device="cuda")  # noqa: E731
        self.dev = dict(len=i32(n_seq), pages=i32(n_seq, max_pages), row_start=i32(n_seq + 1), free=i32(n_pages),
                        n_free=i32(1), status=i32(4))
        self.t = K.PageTable(n_seq, max_pages, page, n_pages, *[a.data_ptr() for a in self.dev.values()])
        torch.cuda.synchronize()
        self.t.init_dev(ctx)
        self.len, self.pages = [0] * n_seq, [[-1] * max_pages for _ in range(n_seq)]
        self.free, self.n_pages = list(range(n_pages - 1, -1, -1)), n_pages
        self.start, self.status = [0] * (n_seq + 1), [0, 0]
        self.check()

    def pages_of(self, n):
        return -(-n // self.page)

    def check(self):
        got = {k: v.cpu().numpy() for k, v in self.dev.items()}
        assert got["len"].tolist() == self.len
        assert got["pages"].tolist() == self.pages
        assert got["row_start"].tolist() == self.start
        assert got["n_free"][0] == len(self.free)
        assert got["free"][:len(self.free)].tolist() == self.free
        assert got["status"].tolist() == self.status + [0, 0]

    def refused(self, why):
        self.status = [why, self.status[1] + (why != 0)]
        return why

    def step(self, rows, n_rows, position=True, slot=True):
        pos = torch.full((n_rows + 3,), 55, dtype=torch.int32, device="cuda")
        slots = torch.full((n_rows + 3,), 55, dtype=torch.int64, device="cuda")
        r = dev(np.array(rows, np.int32))
        self.t.step_dev(self.ctx, r.data_ptr(), n_rows, pos.data_ptr() if position else None, slots.data_ptr() if slot else None)
        why = self.expect(rows, n_rows)
        self.check()
        if position:
            assert pos.cpu().tolist() == self.position + [55] * 3
        if slot:
            assert slots.cpu().tolist() == self.slot + [55] * 3
        return why

    def expect(self, rows, n_rows):
        self.position, self.slot, self.start = [-1] * n_rows, [-1] * n_rows, [0] * len(self.start)
        need = sum(self.pages_of(n + r) - self.pages_of(n) for n, r in zip(self.len, rows) if r > 0)
        if any(r < 0 or r > n_rows for r in rows):
            return self.refused(K.PageTable.ROWS)
        if any(n + r > self.cap for n, r in zip(self.len, rows)):
            return self.refused(K.PageTable.TOO_LONG)
        if sum(rows) > n_rows:
            return self.refused(K.PageTable.ROWS)
        if need > len(self.free):
            return self.refused(K.PageTable.SHORT)
        at = 0
        for s, r in enumerate(rows):
            for _ in range(r):
                p = self.len[s]
                if self.pages[s][p // self.page] < 0:
                    self.pages[s][p // self.page] = self.free.pop()
                self.position[at] = p
                self.slot[at] = self.pages[s][p // self.page] * self.page + p % self.page
                self.len[s] += 1
                at += 1
            self.start[s + 1] = at
        return self.refused(0)

    def release(self, keep):
        k = dev(np.array(keep, np.int32))
        self.t.release_dev(self.ctx, k.data_ptr())
        for s in reversed(range(len(self.len))):
            if 0 <= keep[s] < self.len[s]:
                for j in reversed(range(self.pages_of(keep[s]), self.pages_of(self.len[s]))):
                    self.free.append(self.pages[s][j])
                    self.pages[s][j] = -1
                self.len[s] = keep[s]
        self.refused(0)
        self.check()


@pytest.mark.parametrize("n_seq, max_pages, page, n_pages", [
    (1, 1, 32, 1), (1, 40, 64, 33), (3, 7, 32, 20), (64, 20, 32, 700), (65, 9, 128, 300), (257, 5, 64, 900), (1000, 3, 32, 2500),
    (4096, 2, 32, 6000)])
def test_steps_and_releases_as_one_page_at_a_time(dctx, n_seq, max_pages, page, n_pages):
    rng = np.random.default_rng(n_seq)
    t = Tables(dctx, n_seq, max_pages, page, n_pages)
    for turn in range(12):
        if turn % 3 == 2:
            t.release([int(rng.integers(-2, n + 2)) if rng.random() < 0.5 else -1 for n in t.len])
        most = 2 if turn % 2 else page * max_pages // 3 + 1
        rows = [int(rng.integers(0, most + 1)) if rng.random() < 0.7 else 0 for _ in range(n_seq)]
        rows = [min(r, t.cap - n) for r, n in zip(rows, t.len)]
        t.step(rows, sum(rows) + int(rng.integers(0, 9)), position=turn != 4, slot=turn != 5)
    t.release([0] * n_seq)
    assert sorted(t.free) == list(range(n_pages))


def test_a_release_undoes_a_step(dctx):
    t = Tables(dctx, 5, 9, 32, 30)
    t.step([40, 0, 33, 1, 64], 200)
    t.release([7, -1, 33, 0, 32])
    before = (list(t.free), [list(p) for p in t.pages], list(t.len))
    t.step([100, 3, 0, 32, 1], 200)
    t.release(before[2])
    assert (t.free, t.pages, t.len) == before


def test_steps_that_cannot_be_done_change_nothing(dctx):
    t = Tables(dctx, 3, 4, 32, 6)
    assert t.step([30, 40, 1], 100) == 0
    # 1 + 2 + 1 pages are taken: 98 rows behind 30 need three more of two, 33 behind 1 one
    for rows, n_rows, why in (([1, 1, 128], 300, K.PageTable.TOO_LONG), ([98, 20, 1], 300, K.PageTable.SHORT), ([0, 10, 33], 99, 0),
                              ([1, -1, 0], 9, K.PageTable.ROWS), ([2, 2, 2], 5, K.PageTable.ROWS), ([9, 0, 0], 8, K.PageTable.ROWS),
                              ([1 << 30, 1 << 30, 1 << 30], 50, K.PageTable.ROWS),
                              ([0, 0, (1 << 31) - 1], 50, K.PageTable.ROWS), ([0, 0, 0], 0, 0), ([0, 2, 0], 7, 0)):
        assert t.step(rows, n_rows) == why, rows
    assert t.status[1] == 7


@pytest.mark.parametrize("what, value, why", [("len", -1, 4), ("len", 129, 4), ("n_free", -1, 4), ("n_free", 7, 4), ("n_free", 6, 4)])
def test_tables_that_were_written_over_are_refused(dctx, what, value, why):
    t = Tables(dctx, 3, 4, 32, 6)
    t.step([33, 5, 0], 40)
    t.dev[what][0] = value
    keep, rows = dev(np.array([0, 0, -1], np.int32)), dev(np.array([0, 1, 0], np.int32))
    before = {k: v.clone() for k, v in t.dev.items()}
    t.t.release_dev(dctx, keep.data_ptr())
    assert t.dev["status"].tolist() == [why, 1, 0, 0]
    if not (what == "n_free" and value == 6):  # a step takes that stack as it is
        t.t.step_dev(dctx, rows.data_ptr(), 4)
        assert t.dev["status"].tolist() == [why, 2, 0, 0]
    assert all(torch.equal(before[k], t.dev[k]) for k in ("len", "pages", "free", "n_free"))


def test_a_captured_step_takes_each_replays_rows(dctx):
    t = Tables(dctx, 64, 40, 32, 1500)
    rows = torch.zeros(64, dtype=torch.int32, device="cuda")
    keep = torch.full((64,), -1, dtype=torch.int32, device="cuda")
    n_rows = 4000  # several workgroups
    pos = torch.zeros(n_rows, dtype=torch.int32, device="cuda")
    slot = torch.zeros(n_rows, dtype=torch.int64, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    dctx.set_stream(stream.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        t.t.release_dev(dctx, keep.data_ptr())
        t.t.step_dev(dctx, rows.data_ptr(), n_rows, pos.data_ptr(), slot.data_ptr())
    dctx.set_stream(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    rng = np.random.default_rng(1)
    for i in range(6):
        k = [int(rng.integers(0, n + 1)) if i % 2 and rng.random() < 0.3 else -1 for n in t.len]
        r = [int(x) for x in rng.integers(0, 60, 64)] if i != 4 else [200] * 64  # the fifth is more rows than there are
        keep.copy_(torch.tensor(k))
        rows.copy_(torch.tensor(r))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for s in reversed(range(64)):
            if 0 <= k[s] < t.len[s]:
                for j in reversed(range(t.pages_of(k[s]), t.pages_of(t.len[s]))):
                    t.free.append(t.pages[s][j])
                    t.pages[s][j] = -1
                t.len[s] = k[s]
        t.expect(r, n_rows)
        t.check()
        assert pos.cpu().tolist() == t.position and slot.cpu().tolist() == t.slot


@pytest.mark.parametrize("held", [77, -1, 2 ** 31 - 1])
def test_a_status_that_was_never_cleared(dctx, held):
    # a table that the caller filled, as init does but for the status: steps and
    # releases of one workgroup and of several advance it all the same
    t = Tables(dctx, 64, 40, 32, 1500)
    rng = np.random.default_rng(2)
    for n_rows, most in ((4000, 60), (900, 13), (2500, 39), (4000, 60)):
        t.dev["status"].fill_(held)
        rows = [int(r) for r in rng.integers(0, most, 64)]
        r, pos = dev(np.array(rows, np.int32)), torch.zeros(n_rows, dtype=torch.int32, device="cuda")
        t.t.step_dev(dctx, r.data_ptr(), n_rows, pos.data_ptr())
        t.expect(rows, n_rows)
        assert t.dev["status"].tolist() == [0, held, held, held] and pos.cpu().tolist() == t.position
        t.dev["status"].zero_()
        t.check()
        t.dev["status"].fill_(held)
        keep = [n // 2 if s % 3 else -1 for s, n in enumerate(t.len)]
        k = dev(np.array(keep, np.int32))
        t.t.release_dev(dctx, k.data_ptr())
        assert t.dev["status"].tolist() == [0, held, held, held]
        t.dev["status"].zero_()
        for s in reversed(range(64)):
            if 0 <= keep[s] < t.len[s]:
                for j in reversed(range(t.pages_of(keep[s]), t.pages_of(t.len[s]))):
                    t.free.append(t.pages[s][j])
                    t.pages[s][j] = -1
                t.len[s] = keep[s]
        t.check()


def test_tables_stepped_beside_each_other():
    # two tables' captured steps of several workgroups, replayed on two streams at
    # once, and a third table's calls on another context meanwhile
    streams = [torch.cuda.Stream() for _ in range(3)]
    ctxs = [K.Context(0) for _ in range(2)]
    n_rows, keep = 6000, torch.full((64,), -1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    try:
        tables, rows, graphs = [], [], []
        for i, s in enumerate(streams):
            c = ctxs[i // 2]
            c.set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                tables.append(Tables(c, 64, 100, 32, 4000 + i))
                rows.append(torch.zeros(64, dtype=torch.int32, device="cuda"))
            torch.cuda.synchronize()
            if i < 2:  # both of one context's
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    tables[i].t.release_dev(c, keep.data_ptr())
                    tables[i].t.step_dev(c, rows[i].data_ptr(), n_rows)
                graphs.append(g)
        rng = np.random.default_rng(3)
        for _ in range(8):
            new = [[int(r) for r in rng.integers(0, 90, 64)] for _ in streams]
            for r, n in zip(rows, new):
                r.copy_(torch.tensor(n))
            torch.cuda.synchronize()
            for _ in range(3):
                for g, s in zip(graphs, streams):
                    with torch.cuda.stream(s):
                        g.replay()
                tables[2].t.release_dev(ctxs[1], keep.data_ptr())
                tables[2].t.step_dev(ctxs[1], rows[2].data_ptr(), n_rows)
            torch.cuda.synchronize()
            for t, n in zip(tables, new):
                for _ in range(3):
                    t.expect(n, n_rows)
                t.check()
        del g, graphs
    finally:
        torch.cuda.synchronize()
        for c in ctxs:
            c.set_stream(None)
            c.close()


# ---- rotation --------------------------------------------------------------------

def turned(x, c, s, interleaved):
    """x [m, n_vec, 2 half] by c, s [m, 1, half], in float32."""
    half = c.shape[-1]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    p, q = a * c - b * s, b * c + a * s
    return np.stack([p, q], -1).reshape(x.shape) if interleaved else np.concatenate([p, q], -1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("m, n_vec, half, behind, off", [
    (1, 1, 32, 0, 0), (5, 16, 32, 128, 0), (48, 3, 1, 5, 1), (7, 2, 10, 3, 3), (3, 40, 64, 1024, 1), (1000, 5, 40, 0, 2), (2, 3, 128, 1, 0),
    (9, 1, 7, 0, 0)])
def test_rows_are_rotated_at_their_positions(dctx, interleaved, m, n_vec, half, behind, off):
    rng = np.random.default_rng(m + half)
    width, max_pos = n_vec * 2 * half, 50
    angle = np.arange(max_pos)[:, None] * 1e4 ** (-np.arange(half) / half)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    # rows that start at any float, some at positions that are in no table
    x = rng.standard_normal((m, width + behind)).astype(np.float32)
    pos = rng.integers(0, max_pos, m).astype(np.int32)
    pos[0] = max_pos - 1
    if m > 4:
        pos[1], pos[2], pos[3] = -1, max_pos, -2 ** 31
    ok = (pos >= 0) & (pos < max_pos)
    at = np.where(ok, pos, 0)
    want = turned(x[:, :width].reshape(m, n_vec, -1), cos[at][:, None], sin[at][:, None], interleaved).reshape(m, width)
    store = torch.full((x.size + off,), 7.0, device="cuda")
    store[off:] = dev(x).flatten()
    dx, dp, dc, ds = store[off:].view(m, -1), dev(pos), dev(cos), dev(sin)
    out = torch.full((m * (width + 3) + 1,), 9.0, device="cuda")
    o = out[1:].view(m, width + 3)
    K.rope_rows_dev(dctx, dc.data_ptr(), ds.data_ptr(), half, max_pos, dx.data_ptr(), dp.data_ptr(), m, n_vec, o.data_ptr(),
                    interleaved, x_stride=width + behind, out_stride=width + 3)
    got = o.cpu().numpy()
    np.testing.assert_array_equal(got[ok][:, :width], want[ok])
    assert (got[~ok] == 9.0).all() and (got[:, width:] == 9.0).all()
    np.testing.assert_array_equal(dx.cpu().numpy(), x)
    # in place: what is behind the vectors stays
    K.rope_rows_dev(dctx, dc.data_ptr(), ds.data_ptr(), half, max_pos, dx.data_ptr(), dp.data_ptr(), m, n_vec, dx.data_ptr(),
                    interleaved, x_stride=width + behind, out_stride=width + behind)
    x[ok, :width] = want[ok]
    np.testing.assert_array_equal(dx.cpu().numpy(), x)


def test_rotation_is_rope_devs(dctx):
    m, n_vec, half, pos0 = 9, 4, 32, 5
    x = torch.randn(m, n_vec * 2 * half, device="cuda")
    y = torch.empty_like(x)
    c, s = torch.randn(20, half, device="cuda"), torch.randn(20, half, device="cuda")
    pos = torch.arange(pos0, pos0 + m, dtype=torch.int32, device="cuda")
    for pairs in (False, True):
        K.rope_rows_dev(dctx, c.data_ptr(), s.data_ptr(), half, 20, x.data_ptr(), pos.data_ptr(), m, n_vec, y.data_ptr(), pairs)
        z = x.clone()
        K.rope_dev(dctx, c.data_ptr(), s.data_ptr(), half, z.data_ptr(), m, n_vec, pos0, pairs)
        assert torch.equal(y, z)


# ---- block ends --------------------------------------------------------------------

def block_end(x, y, post, gate, scale, pre, eps):
    """The definition in 64 bits, and the tolerances of both results."""
    x, y = x.astype(np.float64), y.astype(np.float64)
    n = x.shape[-1]
    D = n / 4096 + 40
    inv = lambda a: 1 / np.sqrt(np.mean(a * a, -1, keepdims=True) + eps)  # noqa: E731
    t = y if post is None else y * inv(y) * post.astype(np.float64)
    t = t * float(np.float32(scale)) * (1 if gate is None else gate.astype(np.float64))
    xo = x + t
    tol = U * (np.abs(xo) + (D / 2 + 10) * np.abs(t))
    if pre is None:
        return xo, tol, None, None
    w = pre.astype(np.float64)
    out = xo * inv(xo) * w
    size = np.sqrt(np.sum(xo * xo, -1, keepdims=True))
    off = np.where(size > 0, np.sqrt(np.sum(tol * tol, -1, keepdims=True)) / np.where(size > 0, size, 1), 0)
    return xo, tol * 1.01, out, 1.01 * (np.abs(w) * inv(xo) * tol + np.abs(out) * (U * (D / 2 + 7) + off)) + 1e-44


SIZES = [1, 3, 4, 63, 64, 255, 257, 511, 896, 1023, 1025, 2047, 2049, 4096, 4099, 8191, 8192, 8193, 12345, 40000]


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("post, gate, pre", [(0, "none", 1), (1, "each", 1), (1, "all", 0), (0, "each", 0), (0, "all", 1), (1, "none", 1)])
def test_block_ends(dctx, n, post, gate, pre):
    m = 1 if n > 8192 and n % 2 else 6
    rng = np.random.default_rng(n)
    normal = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, y = normal(m, n) * 3, normal(m, n) * 0.2
    if m > 1:
        x[1], y[1] = 0, 0              # eps alone under the root
        x[2] *= np.float32(2.0 ** 40)  # a stream far larger than what is added to it
        y[3] *= np.float32(2.0 ** -60)
    p, w = normal(n) if post else None, normal(n) if pre else None
    stride = n + 5 if gate == "each" else 0
    g = {"none": None, "all": normal(1, n), "each": normal(m, n + 5)}[gate]
    want_x, tol_x, want, tol = block_end(x, y, p, None if g is None else g[:, :n], 0.3, w, 1e-6)
    # rows that start at any float
    store = torch.full((4, m * n + 8), 5.0, device="cuda")
    dx, dy, xo, o = store[0, 1:1 + m * n], store[1, 3:3 + m * n], store[2, 2:2 + m * n], store[3, 1:1 + m * n]
    dx.copy_(dev(x).flatten())
    dy.copy_(dev(y).flatten())
    keep = [None if a is None else dev(a) for a in (p, g, w)]
    ptr = [None if a is None else a.data_ptr() for a in keep]

    def call(x_out, out):
        K.norm_residual_dev(dctx, dx.data_ptr(), dy.data_ptr(), m, n, 1e-6, x_out.data_ptr(), ptr[0], ptr[1], stride, 0.3, ptr[2],
                            out.data_ptr() if pre else None)

    call(xo, o)
    got_x, got = xo.cpu().numpy().reshape(m, n).copy(), o.cpu().numpy().reshape(m, n).copy()
    assert (np.abs(got_x - want_x) <= tol_x).all(), np.max(np.abs(got_x - want_x) / tol_x)
    if pre:
        assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    assert (store[:, 0] == 5.0).all() and (store[:, 3 + m * n:] == 5.0).all()
    # in place, by the same bits: the residual over x and the normed over y
    call(dx, dy)
    np.testing.assert_array_equal(dx.cpu().numpy().reshape(m, n), got_x)
    if pre:
        np.testing.assert_array_equal(dy.cpu().numpy().reshape(m, n), got)
    # and the other way round
    dx.copy_(dev(x).flatten())
    dy.copy_(dev(y).flatten())
    call(dy, dx)
    np.testing.assert_array_equal(dy.cpu().numpy().reshape(m, n), got_x)
    if pre:
        np.testing.assert_array_equal(dx.cpu().numpy().reshape(m, n), got)


def test_block_ends_of_rows_that_are_not_finite_leave_the_others(dctx):
    n = 896
    x, y = torch.randn(7, n, device="cuda"), torch.randn(7, n, device="cuda")
    w = torch.ones(n, device="cuda")
    outs = []
    for bad in (False, True):
        if bad:
            y[2, 5], x[4, 7], y[6, 0] = float("nan"), float("inf"), float("-inf")
        xo, o = torch.empty_like(x), torch.empty_like(x)
        K.norm_residual_dev(dctx, x.data_ptr(), y.data_ptr(), 7, n, 1e-6, xo.data_ptr(), post_ptr=w.data_ptr(), pre_ptr=w.data_ptr(),
                            out_ptr=o.data_ptr())
        outs.append((xo, o))
    for a, b in zip(*outs):
        assert torch.equal(a[[0, 1, 3, 5]], b[[0, 1, 3, 5]])
    assert outs[1][0][2].isnan().all() and outs[1][1][4].isnan().any() and outs[1][0][6].isnan().any()


def test_block_ends_and_rotations_are_captured(dctx):
    m, n = 33, 1536
    x, y, w = torch.randn(m, n, device="cuda"), torch.randn(m, n, device="cuda"), torch.randn(n, device="cuda")
    c, s = torch.randn(40, 32, device="cuda"), torch.randn(40, 32, device="cuda")
    pos = torch.arange(m, dtype=torch.int32, device="cuda")
    xo, o, r = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)

    def calls():
        K.norm_residual_dev(dctx, x.data_ptr(), y.data_ptr(), m, n, 1e-6, xo.data_ptr(), scale=0.5, pre_ptr=w.data_ptr(), out_ptr=o.data_ptr())
        K.rope_rows_dev(dctx, c.data_ptr(), s.data_ptr(), 32, 40, o.data_ptr(), pos.data_ptr(), m, n // 64, r.data_ptr())

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    dctx.set_stream(stream.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        calls()
    dctx.set_stream(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        x.mul_(0.5).add_(0.1 * i)
        pos.add_(1).remainder_(40)
        torch.cuda.synchronize()
        calls()
        torch.cuda.synchronize()
        want = [t.clone() for t in (xo, o, r)]
        for t in (xo, o, r):
            t.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (xo, o, r)))
