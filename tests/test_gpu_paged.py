"""The paged KV cache on the device: rows as they are rounded, and attention
over them, against numpy in 64 bits.

Rows read back are compared to the bit with the definition's own roundings.
Attention is compared with 64-bit attention over the rows as the cache holds
them.  Its tolerance, per output element: a score's products and sum are off by
at most (hd + 8) u of the sum of their magnitudes, u = 2^-24 (q in two f16
pieces is off by 2^-22 = 4 u of itself, the power-of-two scales by nothing, the
scale and log2 e by 2 u), and by 3 u of the score where it is scaled and the
reference subtracted; a weight is then off by twice that of itself against the
sum of weights, plus 8 u (exp2, the weight in two pieces, V's scale), and a sum
of L of them by L u: all times sum w |v|.  Besides, f16's least step: a weight
times its V row's scale is held to 2^-25 where 2^8 stands for the reference,
which is at most the largest weight times the largest scale that the row sees;
the codes that it multiplies are under 127 (i8, whose largest row has
127 scales in it) or 2^15 (the largest row has 2^14 in it), so a position is off
by at most 2^-32 of the largest weight times the largest value, whatever its own
weight is: L times that."""
import numpy as np
import pytest

import kvad_amd as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32_TINY = 2.0 ** -126
PRECISIONS = {"f32": K.F32, "f16": K.F16, "i8": K.I8}


def rounded(precision, x):
    """The values a cache of the precision holds for rows x [..., dims]."""
    x = np.asarray(x, np.float32)
    if precision == "f32":
        return x
    amax = np.max(np.abs(x), -1, keepdims=True)
    finite = np.isfinite(amax)
    a = np.where(finite, amax, 0).astype(np.float32)
    y = np.where(finite, x, 0).astype(np.float32)
    if precision == "f16":
        scale = np.exp2(np.maximum(np.frexp(a)[1] - 15, -126)).astype(np.float32)
        r = (y / scale).astype(np.float16).astype(np.float32) * scale
    else:
        scale = (a / np.float32(127)).astype(np.float32)
        scale = np.where(scale < F32_TINY, np.float32(0), scale)
        with np.errstate(divide="ignore"):
            inv = np.where(scale > 0, np.float32(1) / scale, np.float32(0)).astype(np.float32)
        t = (y * inv).astype(np.float32).astype(np.float64)
        code = np.clip(np.sign(t) * np.floor(np.abs(t) + 0.5), -127, 127).astype(np.float32)
        r = code * scale
    return np.where(finite, r, np.float32(np.nan)).astype(np.float32)


def reference(q, k, v, first, scale, window=0, sinks=0):
    """64-bit attention of rows q [m, H, hd] at positions first .. over k, v
    [n, kv, hd], and the tolerance of each element."""
    m, H, hd = q.shape
    n, kv = k.shape[0], k.shape[1]
    out, tol = np.zeros((m, H, hd)), np.zeros((m, H, hd))
    t = np.arange(n)
    for i in range(m):
        p = first + i
        see = t <= p
        if window:
            see &= (t > p - window) | (t < sinks)
        if not see.any():
            continue
        for h in range(H):
            g = h * kv // H
            kk, vv, qq = k[see, g].astype(np.float64), v[see, g].astype(np.float64), q[i, h].astype(np.float64)
            s = scale * (kk @ qq)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vv
            size = scale * np.max(np.abs(kk) @ np.abs(qq))
            off = 2 * ((hd + 8) * size + 3 * np.abs(s).max()) + 8 + len(s)
            tol[i, h] = U * off * (w @ np.abs(vv)) + 2.0 ** -32 * len(s) * w.max() * np.abs(vv).max()
    return out, tol


class Pool:
    """Sequences in a PagedCache with their rows at hand: pages in no order."""

    def __init__(self, ctx, rng, precision, kv, hd, page, capacity, spare=2, n_layer=1):
        self.rng, self.precision, self.kv, self.hd, self.page = rng, precision, kv, hd, page
        self.width = [-(-c // page) for c in capacity]
        n_pages = sum(self.width) + spare
        order = rng.permutation(n_pages)
        self.pages = np.full((len(capacity), max(self.width + [1])), -1, np.int32)
        at = 0
        for s, w in enumerate(self.width):
            self.pages[s, :w] = order[at:at + w]
            at += w
        self.cache = K.PagedCache(ctx, n_layer, kv, hd, n_pages, page_size=page, precision=PRECISIONS[precision])
        self.k = [np.zeros((0, kv, hd), np.float32) for _ in capacity]
        self.v = [np.zeros((0, kv, hd), np.float32) for _ in capacity]

    def batch(self, rows=None, lens=None):
        lens = [len(k) for k in self.k] if lens is None else lens
        return K.Batch.host(lens, self.pages, rows)

    def rows(self, n, std=1.0):
        return (self.rng.standard_normal((n, self.kv, self.hd)) * std).astype(np.float32)

    def push(self, counts, k=None, v=None):
        k = self.rows(sum(counts)) if k is None else k
        v = self.rows(sum(counts)) if v is None else v
        at = 0
        for s, c in enumerate(counts):
            self.k[s] = np.concatenate([self.k[s], k[at:at + c]])
            self.v[s] = np.concatenate([self.v[s], v[at:at + c]])
            at += c
        self.cache.push(0, self.batch(counts), k, v)

    def held(self, s):
        return rounded(self.precision, self.k[s]), rounded(self.precision, self.v[s])

    def check(self, counts, n_head, window=0, sinks=0, q=None, got=None, scale=None):
        """attend()'s rows against the reference."""
        m = sum(counts)
        if q is None:
            q = (self.rng.standard_normal((m, n_head, self.hd)) * 1.5).astype(np.float32)
        if got is None:
            got = self.cache.attend(0, self.batch(counts), n_head, q, window=window, sinks=sinks, scale=scale)
        f = np.float32(self.hd ** -0.5 if scale is None else scale)
        at = 0
        for s, c in enumerate(counts):
            if c:
                k, v = self.held(s)
                want, tol = reference(q[at:at + c], k, v, len(k) - c, float(f), window, sinks)
                err = np.abs(got[at:at + c] - want)
                assert np.all(err <= tol), (s, np.unravel_index(np.argmax(err - tol), err.shape), np.max(err / tol))
            at += c
        return got


@pytest.fixture(params=["rule", "8", "16", "32", "128"])
def form(request, monkeypatch):
    """Each form of the attention kernel, by the rows a workgroup takes."""
    if request.param != "rule":
        monkeypatch.setenv("KVAD_PAGED_TILE", request.param)
    return request.param


# ---- rows ----------------------------------------------------------------------

@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("kv, hd, page", [(2, 64, 32), (8, 128, 64), (1, 256, 128), (3, 80, 32), (2, 20, 64), (1, 4, 1024), (2, 132, 32)])
def test_rows_read_back_as_the_definition_rounds_them(ctx, precision, kv, hd, page):
    p = Pool(ctx, np.random.default_rng(kv * hd), precision, kv, hd, page, [100, 1, 40, 257, 33])
    p.push([5, 1, 0, 200, 32], k=p.rows(238) * np.exp(p.rng.standard_normal((238, kv, 1)) * 8).astype(np.float32))
    for counts in ([60, 0, 0, 57, 0], [1, 0, 40, 0, 1], [0, 0, 0, 0, 0], [34, 0, 0, 0, 0]):
        p.push(counts)
    lens = [len(k) for k in p.k]
    k, v = p.cache.read(0, p.batch(lens))
    np.testing.assert_array_equal(k, np.concatenate([p.held(s)[0] for s in range(5)]))
    np.testing.assert_array_equal(v, np.concatenate([p.held(s)[1] for s in range(5)]))
    # the last rows alone
    k, v = p.cache.read(0, p.batch([3, 1, 0, 33, 1]))
    np.testing.assert_array_equal(v, np.concatenate([p.held(s)[1][lens[s] - c:] for s, c in enumerate([3, 1, 0, 33, 1])]))
    np.testing.assert_array_equal(k, np.concatenate([p.held(s)[0][lens[s] - c:] for s, c in enumerate([3, 1, 0, 33, 1])]))


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
def test_rows_at_the_ends_of_the_range(ctx, precision):
    hd = 64
    p = Pool(ctx, np.random.default_rng(5), precision, 1, hd, 32, [64])
    tiny, big = np.float32(1e-45), np.finfo(np.float32).max
    rows = np.zeros((12, 1, hd), np.float32)
    rows[1, 0, 3] = tiny
    rows[2] = np.float32(1e-39)
    rows[3, 0, ::2] = F32_TINY * 127
    rows[4, 0, :] = np.linspace(-1, 1, hd) * big
    rows[5, 0, :] = np.arange(hd) * 0.5 - 8   # halves of a code, both signs
    rows[5, 0, 0] = 127.0
    rows[6, 0, 7] = np.nan
    rows[7, 0, 7] = np.inf
    rows[8, 0, 7] = -np.inf
    rows[9, 0, :] = -big
    rows[10, 0, :] = np.float32(1 + 2.0 ** -11)  # halfway between two halves
    rows[11, 0, 0], rows[11, 0, 1] = 60000.0, 1e-7
    p.push([12], k=rows, v=rows[::-1].copy())
    k, v = p.cache.read(0, p.batch([12]))
    np.testing.assert_array_equal(k, rounded(precision, rows))
    np.testing.assert_array_equal(v, rounded(precision, rows[::-1]))


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
def test_a_push_writes_its_own_slots_alone(ctx, precision):
    p = Pool(ctx, np.random.default_rng(6), precision, 2, 64, 32, [96, 96])
    p.push([90, 90])
    before = [p.held(s) for s in range(2)]
    # rows 37 .. 41 of the first sequence again, by a shorter length
    k, v = p.rows(5), p.rows(5)
    p.cache.push(0, p.batch([5, 0], [42, 90]), k, v)
    got_k, got_v = p.cache.read(0, p.batch([90, 90]))
    for s, at in ((0, 0), (1, 90)):
        want_k, want_v = before[s][0].copy(), before[s][1].copy()
        if s == 0:
            want_k[37:42], want_v[37:42] = rounded(precision, k), rounded(precision, v)
        np.testing.assert_array_equal(got_k[at:at + 90], want_k)
        np.testing.assert_array_equal(got_v[at:at + 90], want_v)


def test_layers_are_apart(ctx):
    p = Pool(ctx, np.random.default_rng(7), "f16", 2, 64, 32, [40], n_layer=3)
    rows = [p.rows(40) for _ in range(3)]
    b = p.batch([40], [40])
    for l in (2, 0, 1):
        p.cache.push(l, b, rows[l], -rows[l])
    for l in range(3):
        k, v = p.cache.read(l, b)
        np.testing.assert_array_equal(k, rounded("f16", rows[l]))
        np.testing.assert_array_equal(v, rounded("f16", -rows[l]))


# ---- attention -------------------------------------------------------------------

GEOMETRIES = [(14, 2, 64), (32, 8, 128), (4, 4, 128), (12, 2, 128), (8, 1, 96), (6, 2, 256), (5, 5, 20), (3, 1, 200), (40, 1, 64)]


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("H, kv, hd", GEOMETRIES)
def test_single_tokens(ctx, precision, H, kv, hd):
    lens = [1, 2, 31, 32, 33, 64, 65, 700]
    p = Pool(ctx, np.random.default_rng(H * hd), precision, kv, hd, 64, lens)
    p.push([n - 1 for n in lens])
    p.push([1] * len(lens))
    p.check([1] * len(lens), H)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("H, kv, hd", [(14, 2, 64), (32, 8, 128), (6, 2, 256), (5, 5, 20)])
@pytest.mark.parametrize("held, rows", [(0, 1), (0, 45), (130, 17), (31, 2), (500, 33)])
def test_chunks(ctx, form, precision, H, kv, hd, held, rows):
    p = Pool(ctx, np.random.default_rng(held + rows), precision, kv, hd, 32, [held + rows, held + rows])
    p.push([held, held])
    p.push([rows, rows])
    p.check([rows, rows], H)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
def test_ragged_batches(ctx, form, precision):
    # more sequences than a wave has lanes, some without rows, some without
    # positions
    rng = np.random.default_rng(11)
    lens = [int(n) for n in rng.integers(0, 90, 70)]
    counts = [int(rng.integers(0, min(n, 12) + 1)) for n in lens]
    p = Pool(ctx, rng, precision, 2, 64, 32, lens)
    p.push([n - c for n, c in zip(lens, counts)])
    p.push(counts)
    p.check(counts, 6)


# long prompts, whose waves take rows of their own: one workgroup's rows end
# inside, and several sequences share the launch
@pytest.mark.parametrize("precision, H, kv, hd, counts", [
    ("f16", 32, 8, 128, [1100, 0, 900]), ("i8", 32, 8, 64, [2100]), ("f32", 16, 16, 64, [700, 333, 290]),
    ("i8", 16, 16, 128, [1000, 260]), ("f32", 32, 8, 128, [1100]), ("f16", 16, 8, 256, [1500])])
def test_long_prompts(ctx, precision, H, kv, hd, counts):
    import torch

    rng = np.random.default_rng(sum(counts))
    p = Pool(ctx, rng, precision, kv, hd, 64, [n + 50 for n in counts])
    p.push([50] * len(counts))
    p.push(counts)
    m = sum(counts)
    q = (rng.standard_normal((m, H, hd)) * 1.5).astype(np.float32)
    got = p.cache.attend(0, p.batch(counts), H, q)
    at = 0
    for s, c in enumerate(counts):
        if not c:
            continue
        k, v = (torch.from_numpy(x).cuda().double() for x in p.held(s))
        pos = torch.arange(50, 50 + c, device="cuda")[:, None]
        t = torch.arange(50 + c, device="cuda")[None]
        for h in range(H):
            g = h * kv // H
            qq = torch.from_numpy(q[at:at + c, h]).cuda().double()
            kk, vv = k[:, g].contiguous(), v[:, g].contiguous()
            f = float(np.float32(hd ** -0.5))
            sc = (f * (qq @ kk.T.contiguous())).masked_fill(t > pos, float("-inf"))
            w = torch.softmax(sc, -1)
            size = (f * (qq.abs() @ kk.abs().T.contiguous())).masked_fill(t > pos, 0).amax(-1, keepdim=True)
            top = sc.masked_fill(t > pos, 0).abs().amax(-1, keepdim=True)
            tol = U * (2 * ((hd + 8) * size + 3 * top) + 8 + 50 + c) * (w @ vv.abs())
            err = (torch.from_numpy(got[at:at + c, h]).cuda().double() - w @ vv).abs()
            assert bool((err <= tol).all()), (s, h, float((err / tol).max()))
        at += c


WINDOWS = [(1, 0), (1, 1), (7, 0), (32, 4), (33, 31), (64, 32), (100, 33), (64, 200), (300, 4), (1000, 3), (50, 64), (20, 1000)]


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("window, sinks", WINDOWS)
def test_windows(ctx, form, precision, window, sinks):
    p = Pool(ctx, np.random.default_rng(window + sinks), precision, 2, 64, 32, [420, 30, 1, 333])
    p.push([400, 0, 0, 332])
    p.push([20, 30, 1, 1])
    p.check([20, 30, 1, 1], 6, window=window, sinks=sinks)


@pytest.mark.parametrize("precision", ["f16", "i8"])
def test_long_window_prompt(ctx, precision):
    # rows of their own per wave, windows that start inside tiles
    rng = np.random.default_rng(3)
    p = Pool(ctx, rng, precision, 16, 64, 64, [800])
    p.push([800])
    p.check([800], 16, window=77, sinks=5)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("held, splits", [(2000, 0), (8001, 0), (2000, 2), (2000, 7), (2000, 63), (8001, 251), (40, 2)])
def test_long_caches_split_over_the_positions(ctx, form, monkeypatch, precision, held, splits):
    # a join of few splits by a wave, of many by four, of more than a wave has
    # lanes; splits that see nothing
    if splits:
        monkeypatch.setenv("KVAD_PAGED_SPLITS", str(splits))
    p = Pool(ctx, np.random.default_rng(held), precision, 2, 128, 128, [held + 3, 700, 40])
    p.push([held, 697, 0])
    p.push([3, 3, 40])
    b = p.batch([3, 3, 40])
    assert form == "128" or p.cache.attend_ws(b, 8) > 0
    p.check([3, 3, 40], 8)
    p.check([3, 3, 40], 8, window=1500, sinks=4)
    p.check([1, 0, 2], 8, window=33, sinks=1)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
def test_scores_that_spread(ctx, form, precision):
    # the maximum rises from tile to tile, by far more than a sum can keep;
    # and a first position that takes nearly all the weight
    rng = np.random.default_rng(13)
    p = Pool(ctx, rng, precision, 1, 64, 32, [500])
    k, v = p.rows(500), p.rows(500)
    k[:, 0, 0] = np.linspace(-60, 60, 500)
    p.push([500], k=k, v=v)
    q = np.zeros((500, 2, 64), np.float32)
    q[:, 0, 0], q[:, 1, 0] = 8.0, -8.0
    q[:, :, 1:] = rng.standard_normal((500, 2, 63)) * 0.5
    p.check([500], 2, q=q)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
def test_values_of_many_sizes(ctx, form, precision):
    # V's rows from 1e-12 to 1e12: the reference follows their scales; the
    # large ones are hidden from the early rows, which stay exact
    rng = np.random.default_rng(17)
    p = Pool(ctx, rng, precision, 1, 64, 32, [300])
    v = p.rows(300) * np.exp2(np.linspace(-40, 40, 300)).astype(np.float32)[:, None, None]
    p.push([300], v=v, k=p.rows(300) * np.exp2(rng.integers(-3, 4, (300, 1, 1))).astype(np.float32))
    p.check([300], 2)


def test_rows_of_zeros(ctx, form):
    for precision in PRECISIONS:
        p = Pool(ctx, np.random.default_rng(1), precision, 1, 64, 32, [70])
        p.push([70], k=np.zeros((70, 1, 64), np.float32), v=p.rows(70))
        p.check([9], 2)
        p.push([0], k=np.zeros((0, 1, 64)), v=np.zeros((0, 1, 64)))
        p.check([3], 2, q=np.zeros((3, 2, 64), np.float32))
        z = Pool(ctx, np.random.default_rng(2), precision, 1, 64, 32, [70])
        z.push([70], v=np.zeros((70, 1, 64), np.float32))
        assert not z.cache.attend(0, z.batch([70]), 2, z.rng.standard_normal((70, 2, 64))).any()


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, np.finfo(np.float32).min])
def test_what_is_hidden_changes_nothing(ctx, form, precision, bad):
    # the same rows over pages that hold such values behind the sequence's end,
    # ahead of a row in its own chunk, and between the sinks and the window
    rng = np.random.default_rng(19)
    held, rows = 150, 20
    k, v, q = (rng.standard_normal((held + rows, 2, 64)).astype(np.float32) for _ in range(3))
    q = rng.standard_normal((rows, 4, 64)).astype(np.float32)
    outs = []
    for dirty in (False, True):
        p = Pool(ctx, np.random.default_rng(19), precision, 2, 64, 32, [224])
        if dirty:
            full = np.full((224, 2, 64), bad, np.float32)
            p.cache.push(0, K.Batch.host([224], p.pages, [224]), full, full)
        p.push([held], k=k[:held], v=v[:held])
        p.push([rows], k=k[held:], v=v[held:])
        outs.append(p.cache.attend(0, p.batch([rows]), 4, q))
        # rows after the fifth new one are such values
        k2, v2 = k[held:].copy(), v[held:].copy()
        if dirty:
            k2[5:], v2[5:] = bad, bad
        p.cache.push(0, p.batch([rows]), k2, v2)
        outs.append(p.cache.attend(0, p.batch([rows]), 4, q)[:5])
        # the positions between the sinks and the window
        if dirty:
            mid = np.full((100, 2, 64), bad, np.float32)
            p.cache.push(0, K.Batch.host([104], p.pages, [100]), mid, mid)
        outs.append(p.cache.attend(0, p.batch([5], [held + 5]), 4, q[:5], window=40, sinks=4))
    for a, b in zip(outs[:3], outs[3:]):
        assert np.all(np.isfinite(a))
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
def test_what_is_not_finite_reaches_the_rows_that_see_it(ctx, form, precision):
    p = Pool(ctx, np.random.default_rng(23), precision, 2, 64, 32, [90])
    v = p.rows(90)
    v[60, 1, 5] = np.nan
    p.push([90], v=v)
    out = p.cache.attend(0, p.batch([90]), 4, p.rng.standard_normal((90, 4, 64)).astype(np.float32))
    assert np.all(np.isfinite(out[:, :2])) and np.all(np.isfinite(out[:60]))
    assert np.all(np.isnan(out[60:, 2:]))


# ---- device arrays -----------------------------------------------------------------

def device_batch(lens, pages, rows=None, n_rows=None, starts=None, max_len=0):
    import torch

    t = {"len": torch.tensor(lens, dtype=torch.int32).cuda(), "pages": torch.from_numpy(np.ascontiguousarray(pages, np.int32)).cuda()}
    if starts is None and rows is not None:
        starts = [0] + list(np.cumsum(rows))
    if starts is not None:
        t["start"] = torch.tensor(starts, dtype=torch.int32).cuda()
        n_rows = starts[-1] if n_rows is None else n_rows
    b = K.Batch(len(lens), int(n_rows), t["len"].data_ptr(), t["pages"].data_ptr(), t["pages"].shape[1],
                row_start=t["start"].data_ptr() if "start" in t else None, max_len=max_len)
    b.tensors = t
    return b


def test_rows_outside_the_sequences_are_left_alone(ctx, form):
    import torch

    p = Pool(ctx, np.random.default_rng(29), "f16", 2, 64, 32, [3000, 50])
    p.push([3000, 50])
    q = torch.randn(9, 4, 64, device="cuda")
    for window, max_len in ((0, 0), (16, 0), (0, 60)):
        b = device_batch([3000, 50], p.pages, starts=[2, 4, 7], n_rows=9, max_len=max_len)
        out, k = torch.full((9, 4, 64), 7.0, device="cuda"), torch.full((9, 2, 64), 7.0, device="cuda")
        v = k.clone()
        torch.cuda.synchronize()
        p.cache.attend_dev(0, b, 4, q.data_ptr(), out.data_ptr(), window=window)
        p.cache.read_dev(0, b, k.data_ptr(), v.data_ptr())
        ctx.synchronize()
        for x in (out, k, v):
            x = x.cpu().numpy()
            assert np.all(x[:2] == 7) and np.all(x[7:] == 7) and not np.any(x[2:7] == 7)
        p.check([2, 3], 4, q=q.cpu().numpy()[2:7], got=out.cpu().numpy()[2:7], window=window)


def test_lengths_and_pages_that_lead_nowhere(ctx, form):
    # values the host cannot see: hidden from every row, read as zero, not written
    import torch

    p = Pool(ctx, np.random.default_rng(31), "f16", 2, 64, 32, [96, 64])
    p.push([96, 64])
    q = torch.randn(12, 4, 64, device="cuda")
    before = p.cache.read(0, p.batch([96, 64]))
    low = np.iinfo(np.int32)
    pages = p.pages.copy()
    for wrong in (-1, p.cache.n_pages, low.max, low.min):
        pages[0, 1] = wrong
        b = device_batch([96, 64], pages, rows=[6, 6])
        out, k = torch.full((12, 4, 64), 7.0, device="cuda"), torch.full((12, 2, 64), 7.0, device="cuda")
        v = k.clone()
        torch.cuda.synchronize()
        p.cache.attend_dev(0, b, 4, q.data_ptr(), out.data_ptr())
        ctx.synchronize()
        # the first sequence without its second page: its other 64 positions,
        # in order, hold the rows' own last
        kk, vv = p.held(0)
        keep = np.r_[0:32, 64:96]
        want, tol = reference(q[:6].cpu().numpy(), kk[keep], vv[keep], 58, float(np.float32(64 ** -0.5)))
        assert np.all(np.abs(out[:6].cpu().numpy() - want) <= tol)
        p.check([0, 6], 4, q=q[6:].cpu().numpy(), got=out[6:].cpu().numpy())
        # rows in the missing page: not written, read as zero
        gone = device_batch([40, 64], pages, rows=[6, 6])
        p.cache.push_dev(0, gone, q.data_ptr(), q.data_ptr())
        p.cache.push_dev(0, device_batch([96, 64], p.pages, rows=[0, 6]), v.data_ptr(), v.data_ptr())
        p.cache.read_dev(0, gone, k.data_ptr(), v.data_ptr())
        ctx.synchronize()
        assert not k[:6].any() and not v[:6].any()
        p.cache.push(0, K.Batch.host([96, 64], p.pages, [0, 6]), p.k[1][58:], p.v[1][58:])
        for a, c in zip(before, p.cache.read(0, p.batch([96, 64]))):
            np.testing.assert_array_equal(a, c)
    # lengths below the rows, negative, and past the table
    for lens in ([3, 0], [-5, low.min], [2, 1]):
        b = device_batch(lens, p.pages, rows=[6, 6])
        out = torch.full((12, 4, 64), 7.0, device="cuda")
        k, v = torch.full((12, 2, 64), 7.0, device="cuda"), torch.full((12, 2, 64), 7.0, device="cuda")
        torch.cuda.synchronize()
        p.cache.attend_dev(0, b, 4, q.data_ptr(), out.data_ptr())
        p.cache.read_dev(0, b, k.data_ptr(), v.data_ptr())
        ctx.synchronize()
        for s in range(2):
            n = max(lens[s], 0)
            assert not out[6 * s:6 * s + 6 - n].any() and not k[6 * s:6 * s + 6 - n].any()
            if n:
                kk, vv = p.held(s)
                want, tol = reference(q[6 * s + 6 - n:6 * s + 6].cpu().numpy(), kk[:n], vv[:n], 0, float(np.float32(64 ** -0.5)))
                assert np.all(np.abs(out[6 * s + 6 - n:6 * s + 6].cpu().numpy() - want) <= tol)
                np.testing.assert_array_equal(k[6 * s + 6 - n:6 * s + 6].cpu().numpy(), kk[:n])
    b = device_batch([1000, low.max], p.pages, rows=[6, 6])
    out, k = torch.full((12, 4, 64), 7.0, device="cuda"), torch.full((12, 2, 64), 7.0, device="cuda")
    v = k.clone()
    torch.cuda.synchronize()
    p.cache.push_dev(0, b, q.data_ptr(), q.data_ptr())
    p.cache.read_dev(0, b, k.data_ptr(), v.data_ptr())
    p.cache.attend_dev(0, b, 4, q.data_ptr(), out.data_ptr())
    ctx.synchronize()
    assert not k.any() and not v.any() and bool(torch.isfinite(out).all())
    for a, c in zip(before, p.cache.read(0, p.batch([96, 64]))):
        np.testing.assert_array_equal(a, c)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("offset", [0, 1])
def test_strided_rows(ctx, form, precision, offset):
    # q, k and v as one row of a joint projection, at and off 16-byte alignment
    import torch

    H, kv, hd = 6, 2, 64
    p = Pool(ctx, np.random.default_rng(37), precision, kv, hd, 32, [80, 40])
    p.push([73, 31])
    width = (H + 2 * kv) * hd + (3 if offset else 4)
    store = torch.randn(16 * width + 8, device="cuda")
    base = store.data_ptr() + 4 * offset
    rows = store[offset:offset + 16 * width].reshape(16, width)
    b = device_batch([80, 40], p.pages, rows=[7, 9])
    out = torch.full((16 * width + 8,), 7.0, device="cuda")
    kb, vb = base + 4 * H * hd, base + 4 * (H + kv) * hd
    torch.cuda.synchronize()
    p.lens = [80, 40]
    host = rows.cpu().numpy()
    q = host[:, :H * hd].reshape(16, H, hd)
    kn, vn = host[:, H * hd:(H + kv) * hd].reshape(16, kv, hd), host[:, (H + kv) * hd:(H + 2 * kv) * hd].reshape(16, kv, hd)
    p.cache.push_dev(0, b, kb, vb, k_stride=width, v_stride=width)
    p.cache.attend_dev(0, b, H, base, out.data_ptr() + 4 * offset, q_stride=width, out_stride=width)
    ctx.synchronize()
    at = 0
    for s, c in enumerate([7, 9]):
        p.k[s] = np.concatenate([p.k[s], kn[at:at + c]])
        p.v[s] = np.concatenate([p.v[s], vn[at:at + c]])
        at += c
    got = out.cpu().numpy()[offset:offset + 16 * width].reshape(16, width)
    p.check([7, 9], H, q=q, got=got[:, :H * hd].reshape(16, H, hd))
    assert np.all(got[:, H * hd:] == 7) and np.all(out.cpu().numpy()[:offset] == 7)
    back = torch.full((16 * width + 8,), 7.0, device="cuda")
    torch.cuda.synchronize()
    at_k = back.data_ptr() + 4 * offset
    p.cache.read_dev(0, b, at_k, at_k + 4 * kv * hd, k_stride=width, v_stride=width)
    ctx.synchronize()
    got = back.cpu().numpy()[offset:offset + 16 * width].reshape(16, width)
    np.testing.assert_array_equal(got[:, :kv * hd].reshape(16, kv, hd), rounded(precision, kn))
    np.testing.assert_array_equal(got[:, kv * hd:2 * kv * hd].reshape(16, kv, hd), rounded(precision, vn))
    assert np.all(got[:, 2 * kv * hd:] == 7)


def test_a_call_gives_the_same_bits_again(ctx):
    p = Pool(ctx, np.random.default_rng(41), "i8", 2, 128, 64, [5000, 700])
    p.push([5000, 700])
    q = p.rng.standard_normal((20, 8, 128)).astype(np.float32)
    a = p.cache.attend(0, p.batch([11, 9]), 8, q)
    np.testing.assert_array_equal(a, p.cache.attend(0, p.batch([11, 9]), 8, q))


def test_workspaces_of_any_size(ctx):
    # the caller's workspace: what the call asks for gives the context's bits,
    # less gives fewer splits, and nothing past it is touched
    import torch

    p = Pool(ctx, np.random.default_rng(43), "f16", 2, 64, 64, [6000])
    p.push([6000])
    q = torch.randn(2, 4, 64, device="cuda")
    b = device_batch([6000], p.pages, rows=[2])
    need = p.cache.attend_ws(b, 4)
    assert need > 0
    base = torch.empty(2, 4, 64, device="cuda")
    torch.cuda.synchronize()
    p.cache.attend_dev(0, b, 4, q.data_ptr(), base.data_ptr())
    ctx.synchronize()
    for size in (need, need + 64, need // 2, need // 7, 1, 0):
        ws = torch.full((need // 4 + 64,), 7.0, device="cuda")
        out = torch.full_like(base, 7.0)
        torch.cuda.synchronize()
        p.cache.attend_dev(0, b, 4, q.data_ptr(), out.data_ptr(), ws_ptr=ws.data_ptr(), ws_bytes=size)
        ctx.synchronize()
        assert bool((ws[-(-size // 4):] == 7).all())
        if size >= need:
            assert torch.equal(out, base)
        p.check([2], 4, q=q.cpu().numpy(), got=out.cpu().numpy())


def test_captured_calls_take_the_lengths_of_each_replay(ctx):
    # a decode step's push and attention in a graph: lengths and pages are read
    # when it runs.  Two graphs with a workspace each, replayed in turn, with
    # eager calls that move the context's scratch between them; and one without.
    import torch

    H, kv, hd = 4, 2, 64
    p = Pool(ctx, np.random.default_rng(47), "i8", kv, hd, 32, [4000, 3000])
    p.push([3900, 2900])
    stream = torch.cuda.Stream()
    fresh = K.Context(0)
    cache = K.PagedCache(fresh, 1, kv, hd, p.cache.n_pages, page_size=32, precision=K.I8)
    cache.push(0, p.batch([3900, 2900]), np.concatenate(p.k), np.concatenate(p.v))
    p.cache = cache
    try:
        fresh.set_stream(stream.cuda_stream)
        graphs = []
        for kind in ("ws", "ws", "none"):
            b = device_batch([3901, 2901], p.pages, n_rows=2, rows=None)
            q, k, v = (torch.randn(2, n, hd, device="cuda") for n in (H, kv, kv))
            out = torch.zeros(2, H, hd, device="cuda")
            need = cache.attend_ws(b, H)
            assert need > 0
            ws = torch.zeros(need // 4, device="cuda") if kind == "ws" else None
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                cache.push_dev(0, b, k.data_ptr(), v.data_ptr())
                cache.attend_dev(0, b, H, q.data_ptr(), out.data_ptr(), ws_ptr=None if ws is None else ws.data_ptr(),
                                 ws_bytes=0 if ws is None else need)
            graphs.append((g, b, q, k, v, out, ws))
        for step in range(3):
            for g, b, q, k, v, out, _ in graphs:
                for x in (q, k, v):
                    x.normal_()
                p.k = [np.concatenate([p.k[s], k[s:s + 1].cpu().numpy()]) for s in range(2)]
                p.v = [np.concatenate([p.v[s], v[s:s + 1].cpu().numpy()]) for s in range(2)]
                b.tensors["len"].copy_(torch.tensor([len(x) for x in p.k], dtype=torch.int32))
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                p.check([1, 1], H, q=q.cpu().numpy(), got=out.cpu().numpy())
            p.check([step + 2, 1], H, window=900 * step)  # an eager call between them
            fresh.reserve((8 + 8 * step) << 20)
        del graphs
    finally:
        fresh.set_stream(None)
        fresh.close()


def test_another_stream_and_context(ctx):
    import torch

    other = K.Context(0)
    stream = torch.cuda.Stream()
    try:
        p = Pool(other, np.random.default_rng(53), "f16", 2, 64, 32, [300])
        other.set_stream(stream.cuda_stream)
        p.push([300])
        q = torch.randn(300, 4, 64, device="cuda")
        out = torch.empty_like(q)
        b = device_batch([300], p.pages, rows=[300])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            p.cache.attend_dev(0, b, 4, q.data_ptr(), out.data_ptr())
            host = out.cpu()
        p.check([300], 4, q=q.cpu().numpy(), got=host.numpy())
    finally:
        other.set_stream(None)
        other.close()


def test_a_pool_past_32_bit_offsets(ctx):
    # pages whose bytes lie past 4 GiB of the pool, beside the first ones
    kv, hd, page = 8, 128, 1024
    n_pages = 2300
    cache = K.PagedCache(ctx, 1, kv, hd, n_pages, page_size=page, precision=K.I8)
    try:
        assert cache.bytes > 4.5 * 2 ** 30
        rng = np.random.default_rng(59)
        pages = np.array([[n_pages - 1, 0], [2047, n_pages - 2]], np.int32)
        lens, rows = [1500, 1030], [1500, 1030]
        k, v = (rng.standard_normal((2530, kv, hd)).astype(np.float32) for _ in range(2))
        b = K.Batch.host(lens, pages, rows)
        cache.push(0, b, k, v)
        got = cache.read(0, b)
        np.testing.assert_array_equal(got[0], rounded("i8", k))
        np.testing.assert_array_equal(got[1], rounded("i8", v))
        q = rng.standard_normal((4, 16, hd)).astype(np.float32)
        out = cache.attend(0, K.Batch.host(lens, pages, [2, 2]), 16, q)
        f = float(np.float32(hd ** -0.5))
        for s, (a, e) in enumerate(((0, 1500), (1500, 2530))):
            want, tol = reference(q[2 * s:2 * s + 2], rounded("i8", k[a:e]), rounded("i8", v[a:e]), e - a - 2, f)
            assert np.all(np.abs(out[2 * s:2 * s + 2] - want) <= tol)
    finally:
        cache.free()


def test_page_sizes_and_lengths_hint(ctx):
    # the page size and max_len change nothing but the order of sums
    rng = np.random.default_rng(61)
    for page in (32, 64, 128, 256, 512, 1024):
        p = Pool(ctx, rng, "i8", 2, 64, page, [2100, 90])
        p.push([2100, 90])
        q = rng.standard_normal((8, 4, 64)).astype(np.float32)
        for hint in (0, 1, 100, 5000):
            b = p.batch([5, 3])
            b.max_len = hint
            p.check([5, 3], 4, q=q, got=p.cache.attend(0, b, 4, q))


def test_one_token_agrees_with_the_contiguous_cache(ctx):
    # kh_attend over the same rows; it drops weights under 1e-8, at most
    # 1e-8 L of the values
    spec = K.Spec(14, 2, 64)
    p = Pool(ctx, np.random.default_rng(67), "f32", 2, 64, 64, [900])
    p.push([900])
    flat = K.KvCache(ctx, 1, 128, 128)
    flat.push(0, p.k[0], p.v[0])
    q = p.rng.standard_normal((1, 14, 64)).astype(np.float32)
    a = p.check([1], 14, q=q)
    b = K.attend(ctx, spec, q, flat, 0, 900).reshape(1, 14, 64)
    assert np.max(np.abs(a - b)) <= 1e-4 * np.max(np.abs(b))


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
def test_a_run_of_them(ctx, precision):
    # conversations as a server has them: prompts in chunks beside decoding
    # ones, a common prefix, one that ends and gives its pages to another
    rng = np.random.default_rng(71)
    H, kv, hd, page = 8, 2, 64, 32
    cache = K.PagedCache(ctx, 1, kv, hd, 40, page_size=page, precision=PRECISIONS[precision])
    free = [int(x) for x in rng.permutation(40)]
    seqs = {}

    def step(news, window=0, sinks=0):
        names = list(news)
        for s in names:
            held = seqs.setdefault(s, {"k": np.zeros((0, kv, hd), np.float32), "v": np.zeros((0, kv, hd), np.float32), "pages": []})
            while len(held["pages"]) * page < len(held["k"]) + news[s]:
                held["pages"].append(free.pop())
            for x in "kv":
                held[x] = np.concatenate([held[x], rng.standard_normal((news[s], kv, hd)).astype(np.float32)])
        table = np.full((len(names), max(len(seqs[s]["pages"]) for s in names)), -1, np.int32)
        for i, s in enumerate(names):
            table[i, :len(seqs[s]["pages"])] = seqs[s]["pages"]
        counts = [news[s] for s in names]
        b = K.Batch.host([len(seqs[s]["k"]) for s in names], table, counts)
        new = {x: np.concatenate([seqs[s][x][len(seqs[s][x]) - news[s]:] for s in names]) for x in "kv"}
        cache.push(0, b, new["k"], new["v"])
        q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
        out = cache.attend(0, b, H, q, window=window, sinks=sinks)
        at = 0
        for s in names:
            k, v = rounded(precision, seqs[s]["k"]), rounded(precision, seqs[s]["v"])
            want, tol = reference(q[at:at + news[s]], k, v, len(k) - news[s], float(np.float32(hd ** -0.5)), window, sinks)
            assert np.all(np.abs(out[at:at + news[s]] - want) <= tol), s
            at += news[s]

    step({"a": 70})
    step({"a": 1, "b": 45})
    step({"a": 1, "b": 33, "c": 3})
    # d starts from a's first page, which neither writes again
    seqs["d"] = {x: seqs["a"][x][:page].copy() for x in "kv"} | {"pages": seqs["a"]["pages"][:1]}
    step({"a": 1, "d": 9, "c": 1})
    free.extend(seqs.pop("b")["pages"])
    step({"e": 150, "a": 1, "d": 1})
    step({"e": 1, "a": 1, "c": 1, "d": 1}, window=40, sinks=4)
    lens = [len(seqs["a"]["k"])]
    k, v = cache.read(0, K.Batch.host(lens, np.array([seqs["a"]["pages"]]), lens))
    np.testing.assert_array_equal(k, rounded(precision, seqs["a"]["k"]))
    np.testing.assert_array_equal(v, rounded(precision, seqs["a"]["v"]))


def test_refusals(ctx):
    for bad in (dict(n_layer=0), dict(n_kv_head=0), dict(head_dim=0), dict(head_dim=66), dict(head_dim=260),
                dict(page_size=16), dict(page_size=48), dict(page_size=2048), dict(n_pages=0), dict(precision=K.Q8),
                dict(precision=17)):
        args = dict(n_layer=1, n_kv_head=1, head_dim=64, n_pages=2, page_size=32, precision=K.F16) | bad
        with pytest.raises(K.KvadError, match="status -1"):
            K.PagedCache(ctx, **args)
    for n_pages in (2 ** 31 - 1,):  # more bytes than the device has, or than can be counted
        with pytest.raises(K.KvadError, match="status -3"):
            K.PagedCache(ctx, 65536, 65536, 256, n_pages, page_size=1024, precision=K.F32)
        with pytest.raises(K.KvadError, match="status -3"):
            K.PagedCache(ctx, 1, 8, 128, 2 ** 24, page_size=1024, precision=K.F32)
    p = Pool(ctx, np.random.default_rng(1), "f16", 2, 64, 32, [40])
    p.push([40])
    b, c, q = p.batch([1]), p.cache, np.zeros((1, 4, 64), np.float32)
    for call in (lambda: c.attend(1, b, 4, q), lambda: c.attend(0, b, 3, np.zeros((1, 3, 64))),
                 lambda: c.attend(0, b, 0, np.zeros((1, 0, 64))), lambda: c.attend(0, b, 4, q, scale=0.0),
                 lambda: c.attend(0, b, 4, q, scale=-1.0), lambda: c.attend(0, b, 4, q, scale=float("nan")),
                 lambda: c.attend(0, b, 4, q, scale=float("inf")), lambda: c.push(1, b, np.zeros((1, 2, 64)), np.zeros((1, 2, 64))),
                 lambda: c.read(1, b), lambda: c.attend(0, K.Batch.host([65], p.pages, [1]), 4, q),
                 lambda: c.push(0, K.Batch.host([40], np.array([[0, 99]]), [9]), np.zeros((9, 2, 64)), np.zeros((9, 2, 64))),
                 lambda: c.attend_dev(0, b, 4, 16, 16, q_stride=255), lambda: c.attend_dev(0, b, 4, 16, 16, out_stride=4),
                 lambda: c.attend_dev(0, b, 4, 16, None), lambda: c.attend_dev(0, b, 4, 18, 16),
                 lambda: c.attend_dev(0, b, 4, 16, 16, ws_ptr=8, ws_bytes=100),
                 lambda: c.push_dev(0, b, 16, 16, k_stride=127), lambda: c.push_dev(0, b, 16, 17),
                 lambda: c.read_dev(0, b, None, 16), lambda: c.read_dev(0, b, 16, 16, v_stride=1)):
        with pytest.raises(K.KvadError, match="status -1"):
            call()
    none = K.Batch.host([40], p.pages, [0])
    assert c.attend(0, none, 4, np.zeros((0, 4, 64))).shape == (0, 4, 64)
    assert c.read(0, none)[0].shape == (0, 2, 64)


def test_freed_with_its_context(ctx):
    other = K.Context(0)
    cache = K.PagedCache(other, 2, 2, 64, 4)
    other.close()
    assert cache.h is None
    cache.free()


def test_a_split_call_leaves_a_captured_graph_of_another_operator_its_scratch(ctx):
    # contiguous attention over a long cache, captured with the context's
    # scratch as its first call made it; paged attention, which needs more for
    # its splits, between the replays
    import torch

    H, kv, hd, L = 8, 2, 64, 6000
    q, k, v = torch.randn(H, hd, device="cuda"), torch.randn(L, kv, hd, device="cuda"), torch.randn(L, kv, hd, device="cuda")
    want, out = torch.empty_like(q), torch.empty_like(q)
    torch.cuda.synchronize()
    fresh, stream = K.Context(0), torch.cuda.Stream()
    try:
        fresh.set_stream(stream.cuda_stream)
        K.attend_dev(fresh, K.Spec(H, kv, hd), q.data_ptr(), k.data_ptr(), v.data_ptr(), L, want.data_ptr())
        fresh.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            K.attend_dev(fresh, K.Spec(H, kv, hd), q.data_ptr(), k.data_ptr(), v.data_ptr(), L, out.data_ptr())
        p = Pool(fresh, np.random.default_rng(71), "f32", 2, 256, 64, [9000])
        p.push([9000])
        for rows in (1, 9, 40):
            assert rows == 1 or p.cache.attend_ws(p.batch([rows]), 32) > 1 << 20
            p.check([rows], 32)
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        del g
    finally:
        fresh.set_stream(None)
        fresh.close()


def test_calls_of_several_threads(ctx):
    # one context, one cache, two threads: calls in some order, each its own
    from concurrent.futures import ThreadPoolExecutor

    p = Pool(ctx, np.random.default_rng(73), "i8", 2, 64, 32, [3000, 200])
    p.push([3000, 200])
    qs = [p.rng.standard_normal((n + 1, 4, 64)).astype(np.float32) for n in range(8)]
    batches = [p.batch([n, 1]) for n in range(8)]
    alone = [p.cache.attend(0, b, 4, q) for b, q in zip(batches, qs)]
    with ThreadPoolExecutor(2) as pool:
        both = list(pool.map(lambda i: p.cache.attend(0, batches[i], 4, qs[i]), range(8)))
    for a, b in zip(alone, both):
        np.testing.assert_array_equal(a, b)


def test_out_is_not_q(ctx):
    p = Pool(ctx, np.random.default_rng(79), "f16", 2, 64, 32, [40])
    with pytest.raises(K.KvadError, match="out is not q"):
        p.cache.attend_dev(0, p.batch([1]), 4, 64, 64)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("hd", [128, 256])
def test_wide_rows_behind_masks_and_splits(ctx, form, monkeypatch, precision, hd):
    # what test_what_is_hidden_changes_nothing does with 64 dims: stale values
    # behind the end and between sinks and window, chunks and splits of them
    rng = np.random.default_rng(83)
    held, rows = 300, 37
    k, v = (rng.standard_normal((held + rows, 2, hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((rows, 4, hd)).astype(np.float32)
    for splits in ("", "3"):
        monkeypatch.setenv("KVAD_PAGED_SPLITS", splits)
        outs = []
        for dirty in (False, True):
            p = Pool(ctx, np.random.default_rng(83), precision, 2, hd, 32, [384])
            if dirty:
                full = np.full((384, 2, hd), np.nan, np.float32)
                p.cache.push(0, K.Batch.host([384], p.pages, [384]), full, full)
            p.push([held], k=k[:held], v=v[:held])
            p.push([rows], k=k[held:], v=v[held:])
            outs.append(p.check([rows], 4, q=q))
            if dirty:
                mid = np.full((100, 2, hd), np.inf, np.float32)
                p.cache.push(0, K.Batch.host([140], p.pages, [100]), mid, mid)
            outs.append(p.cache.attend(0, p.batch([rows]), 4, q, window=70, sinks=40))
            if dirty:  # and seen, they are what the rows become
                out = p.cache.attend(0, p.batch([rows]), 4, q, window=70, sinks=41)
                assert np.all(np.isnan(out))
        for a, b in zip(outs[:2], outs[2:]):
            assert np.all(np.isfinite(a))
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("hd", [128, 256])
def test_long_chunks_of_wide_f32_rows(ctx, monkeypatch, hd):
    # waves with rows of their own, and waves that share them
    for tile in ("128", "32"):
        monkeypatch.setenv("KVAD_PAGED_TILE", tile)
        p = Pool(ctx, np.random.default_rng(89), "f32", 2, hd, 64, [700, 130])
        p.push([450, 0])
        p.push([250, 130])
        p.check([250, 130], 6)
        p.check([250, 130], 6, window=100, sinks=3)


# ---- values, scales and queries at the ends of the range ------------------------------

@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("small, large", [(None, 44), (None, 90), (-100, 30), (-60, 80), (-118, 88)])
@pytest.mark.parametrize("splits", ["", "3"])
def test_small_values_before_large_ones_keep_their_weights(ctx, form, monkeypatch, precision, small, large, splits):
    # zeros (None) or rows of 2^small, then rows of 2^large, and the other way
    # round: what the small ones give is lost beside the large, but their weights
    # are half of the sum that divides
    monkeypatch.setenv("KVAD_PAGED_SPLITS", splits)
    p = Pool(ctx, np.random.default_rng(97), precision, 2, 64, 32, [200, 200])
    size = np.full((200, 1, 1), 2.0 ** large, np.float32)
    size[:100] = 0 if small is None else 2.0 ** small
    p.push([200, 200], v=p.rows(400) * np.concatenate([size, size[::-1]]))
    p.check([7, 7], 4)
    p.check([1, 30], 4, window=150, sinks=20)


# Tolerance: reference()'s, and for what f16's least step is worth where V is
# smaller than the reference follows it (i8, 127 times 2^-121): 2^-147, a position;
# and f32's own least step.  Of the whole: a weight's exponent has V's in it, up to
# 128, which f32 rounds by 2^-18, a weight by 2^-18.5, once more where the
# reference moves: 2^-16 of the norm.
@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("size", [-80, -95, -105, -112, -120, 93])
def test_values_of_one_size(ctx, form, precision, size):
    p = Pool(ctx, np.random.default_rng(101), precision, 2, 64, 32, [150, 40])
    p.push([150, 40], v=p.rows(190) * np.float32(2.0 ** size))
    q = (p.rng.standard_normal((50, 4, 64)) * 1.5).astype(np.float32)
    got = p.cache.attend(0, p.batch([30, 20]), 4, q)
    for s, (a, e) in enumerate(((0, 30), (30, 50))):
        k, v = p.held(s)
        want, tol = reference(q[a:e], k, v, len(k) - (e - a), 0.125)
        err = np.abs(got[a:e] - want)
        assert np.all(err <= tol + len(k) * 2.0 ** -147 + 2.0 ** -149), np.max(err) / np.max(np.abs(want))
        assert np.linalg.norm(err) <= 2.0 ** -16 * np.linalg.norm(want)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("scale, size", [(0.125, 1.0), (3.0, 1.0), (1e-3, 1e3), (1e-8, 1.0), (1e-20, 1e19), (1e-38, 1.0),
                                         (1e-45, 1.0), (2.0 ** 120, 2.0 ** -120), (3e38, 2.0 ** -127)])
def test_scales(ctx, form, precision, scale, size):
    # small and large ones beside queries that are zero, and of about their inverse
    p = Pool(ctx, np.random.default_rng(103), precision, 2, 64, 32, [90, 40])
    p.push([90, 40])
    q = (p.rng.standard_normal((50, 4, 64)) * size).astype(np.float32)
    q[::3] = 0
    q[1::3, 1] = 0
    p.check([20, 30], 4, q=q, scale=scale)
    p.check([20, 30], 4, q=q, scale=scale, window=37, sinks=3)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
def test_keys_of_zeros_weigh_alike_at_any_scale(ctx, form, precision):
    p = Pool(ctx, np.random.default_rng(107), precision, 2, 64, 32, [90])
    p.push([90], k=np.zeros((90, 2, 64), np.float32))
    for scale in (1e-45, 1.0, 3e38):
        p.check([20], 4, scale=scale)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("H, kv, hd", [(12, 2, 64), (32, 8, 128), (10, 1, 256)])
def test_short_sequences_share_a_workgroups_waves_in_the_widest_form(ctx, monkeypatch, precision, H, kv, hd):
    # sequences of 9 to 32 rows (x group), each over the whole of its cache:
    # 128 rows a workgroup give them its four waves, as 32 do, to the bit
    rng = np.random.default_rng(109)
    p = Pool(ctx, rng, precision, kv, hd, 64, [400, 90, 700, 300])
    p.push([400, 90, 700, 300])
    group = H // kv
    counts = [-(-9 // group), 32 // group, 0, 32 // group - 1]
    q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
    monkeypatch.setenv("KVAD_PAGED_SPLITS", "1")
    outs = []
    for tile in ("32", "128"):
        monkeypatch.setenv("KVAD_PAGED_TILE", tile)
        outs.append(p.check(counts, H, q=q, got=p.cache.attend(0, p.batch(counts), H, q)))
    np.testing.assert_array_equal(*outs)


# The error of random rows as a whole, which the bound of an element (a worst
# case) does not hold: dropping the low piece of q, a weight or a f32 row of K or
# V is an error of 2^-12 a term, and shows.  With both, each of the three pairs of
# pieces is off by 2^-22 at most, so by 2^-23 on the average; scores (standard
# deviation 1.5) by about 1.5 x 2^-23 x log2 e and some 2^-24 of their sum; a
# weight by that, exp2's 2^-23 and its own pieces; independent from one position
# to the next, as the values are: 2^-21 of the norm, sums in 32 bits included, and
# 2^-18 is eight times that.
@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("H, kv, hd, held, rows, splits", [
    (4, 2, 128, 5000, 3, ""), (4, 2, 128, 5000, 3, "9"), (2, 1, 256, 700, 20, ""), (2, 1, 256, 2000, 2, "5"),
    (6, 2, 64, 300, 40, ""), (3, 3, 64, 3000, 1, "1")])
def test_error_of_the_whole(ctx, form, monkeypatch, precision, H, kv, hd, held, rows, splits):
    monkeypatch.setenv("KVAD_PAGED_SPLITS", splits)
    p = Pool(ctx, np.random.default_rng(113), precision, kv, hd, 64, [held + rows])
    p.push([held + rows])
    q = (p.rng.standard_normal((rows, H, hd)) * 1.5).astype(np.float32)
    got = p.cache.attend(0, p.batch([rows]), H, q)
    want, _ = reference(q, *p.held(0), held, float(np.float32(hd ** -0.5)))
    assert np.linalg.norm(got - want) <= 2.0 ** -18 * np.linalg.norm(want)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
@pytest.mark.parametrize("size", [-100, -60, 60, 93])
def test_keys_of_many_sizes(ctx, form, precision, size):
    # keys and queries of inverse sizes, beside keys of zeros: common scores
    p = Pool(ctx, np.random.default_rng(127), precision, 2, 64, 32, [90, 40])
    k = p.rows(130) * np.float32(2.0 ** size)
    k[5::7] = 0
    p.push([90, 40], k=k)
    q = (p.rng.standard_normal((50, 4, 64)) * 1.5 * 2.0 ** -size).astype(np.float32)
    p.check([20, 30], 4, q=q)


@pytest.mark.parametrize("precision", ["f32", "f16", "i8"])
def test_scores_as_large_as_their_step_allows(ctx, form, precision):
    # of up to 2^24, f32's step 1 there: one key for all is a mean to the last
    # bits still, and one position ahead of all others takes the whole weight
    rng = np.random.default_rng(131)
    p = Pool(ctx, rng, precision, 1, 64, 32, [200, 200])
    one = np.zeros((200, 1, 64), np.float32)
    one[:, 0, 0] = 2.0 ** 12
    ahead = one.copy()
    ahead[77, 0, 0] = 2.0 ** 13
    v = p.rows(400)
    p.push([200, 200], k=np.concatenate([one, ahead]), v=v)
    q = np.zeros((20, 2, 64), np.float32)
    q[:, 0, 0], q[:, 1, 0] = 2.0 ** 11, -(2.0 ** 11)
    got = p.cache.attend(0, p.batch([10, 10]), 2, q, scale=1.0)
    held = [p.held(s)[1].astype(np.float64) for s in range(2)]
    for i in range(10):
        mean = held[0][:191 + i, 0].mean(0)
        assert np.max(np.abs(got[i] - mean)) <= 2.0 ** -20
        np.testing.assert_allclose(got[10 + i, 0], held[1][77, 0], rtol=2.0 ** -20, atol=2.0 ** -30)
        others = np.delete(held[1][:191 + i, 0], 77, 0).mean(0)
        assert np.max(np.abs(got[10 + i, 1] - others)) <= 2.0 ** -20
