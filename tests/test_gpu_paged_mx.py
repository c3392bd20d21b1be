"""4-bit rows (MXFP4) of the paged KV cache: what the other precisions' tests
ask of theirs, and what is these rows' own.

The attention's tolerances are the ones derived there.  Of f16's least step: a
weight times its V row's scale is held to 2^-25 where 2^8 stands for the
reference, and multiplies codes times factors of up to 6 2^12, where the row
that sets the reference has 3.5 2^12 in it, or factors as its scale is at its
least, 2^-126, and the same of its own: 2^-33 x 6 / 3.5 < 2^-32 of the largest
weight times the largest value, as for f16 rows.  Codes times factors are exact
f16, subnormals (factors of 2^-14) among them."""
import numpy as np
import pytest

import kvad_amd as K
import test_gpu_paged as T
from test_gpu_paged import Pool, device_batch, form, reference  # noqa: F401

pytestmark = pytest.mark.gpu

MX = "mxfp4"
VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def mx(x):
    """The values a cache of 4-bit rows holds for rows x [..., dims]."""
    x = np.asarray(x, np.float32)
    hd = x.shape[-1]
    finite = np.isfinite(x).all(-1, keepdims=True)
    y = np.where(finite, x, 0).astype(np.float64)
    pad = -hd % 32
    y = np.concatenate([y, np.zeros(y.shape[:-1] + (pad,))], -1).reshape(y.shape[:-1] + ((hd + pad) // 32, 32))
    amax = np.abs(y).max(-1, keepdims=True)
    e = np.full(amax.shape, -128)
    for k in range(-128, 128):
        e = np.where(amax >= 3.5 * 2.0 ** k, k, e)
    e = np.maximum(e, np.maximum(e.max(-2, keepdims=True), -114) - 26)
    t = np.abs(y) / np.exp2(e.astype(np.float64))
    mid = (VALUES[1:] + VALUES[:-1]) / 2
    code = np.zeros(t.shape, int)
    for i, m in enumerate(mid):  # to code i + 1 from the middle on, or behind it where i is even
        code += (t > m) if i % 2 == 0 else (t >= m)
    with np.errstate(over="ignore"):
        r = (np.sign(y) * VALUES[code] * np.exp2(e.astype(np.float64))).astype(np.float32)
    r = r.reshape(r.shape[:-2] + (hd + pad,))[..., :hd]
    return np.where(finite, r, np.float32(np.nan)).astype(np.float32)


@pytest.fixture(autouse=True)
def with_mx(monkeypatch):
    """The other tests' pool and reference, with these rows among the precisions."""
    others = T.rounded
    monkeypatch.setitem(T.PRECISIONS, MX, K.MXFP4)
    monkeypatch.setattr(T, "rounded", lambda precision, x: mx(x) if precision == MX else others(precision, x))


# ---- rows ----------------------------------------------------------------------

@pytest.mark.parametrize("kv, hd, page", [(2, 64, 32), (8, 128, 64), (1, 256, 128), (3, 80, 32), (2, 20, 64), (1, 4, 1024), (2, 132, 32)])
def test_rows_read_back_as_the_definition_rounds_them(ctx, kv, hd, page):
    T.test_rows_read_back_as_the_definition_rounds_them(ctx, MX, kv, hd, page)


def test_rows_at_the_ends_of_the_range(ctx):
    T.test_rows_at_the_ends_of_the_range(ctx, MX)


def test_a_push_writes_its_own_slots_alone(ctx):
    T.test_a_push_writes_its_own_slots_alone(ctx, MX)


def test_codes_ties_and_steps(ctx):
    # every middle between two values and its neighbours, at steps of all sizes;
    # largest values on both sides of where the step doubles
    mid = (VALUES[1:] + VALUES[:-1]) / 2
    near = np.concatenate([VALUES, mid, np.nextafter(mid.astype(np.float32), 9), np.nextafter(mid.astype(np.float32), 0)]).astype(np.float32)
    near = near[near < 6.9][:29]
    tops = np.array([3.5, np.nextafter(np.float32(3.5), 9), 4, 5, np.nextafter(np.float32(5), 9), 6, 6.5,
                     np.nextafter(np.float32(7), 0)], np.float32)
    exps = [-128, -127, -126, -120, -100, -3, 0, 5, 100, 125]
    rows = np.zeros((len(tops) * len(exps), 1, 64), np.float32)
    for i, (top, e) in enumerate((t, e) for t in tops for e in exps):
        with np.errstate(over="ignore"):
            rows[i, 0, :29] = np.ldexp(np.minimum(near, top), e) * np.where(np.arange(29) % 2, -1, 1)
            rows[i, 0, 29:32] = np.ldexp(top, e)
            rows[i, 0, 32:61] = np.ldexp(np.minimum(near, top), min(e, 90) - i % 30)  # a group beside it, up to 2^29 smaller
    rows = rows[np.isfinite(rows).all((1, 2))]
    p = Pool(ctx, np.random.default_rng(3), MX, 1, 64, 32, [len(rows)])
    p.push([len(rows)], k=rows, v=rows[::-1].copy())
    k, v = p.cache.read(0, p.batch([len(rows)]))
    np.testing.assert_array_equal(k, mx(rows))
    np.testing.assert_array_equal(v, mx(rows[::-1]))
    assert (np.abs(k) == 2.0 ** -129).any()  # the least value there is; infinity is test_rows_at_the_ends_of_the_range's


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_single_positions_fill_words_of_eight(ctx, hd):
    # one position a call, some again: of a word of V's codes each leaves the rest
    p = Pool(ctx, np.random.default_rng(hd), MX, 2, hd, 32, [70, 70])
    for i in range(70):
        p.push([1, 1 if i % 3 else 0])
    for at in (5, 0, 63, 32, 6, 40):
        k, v = p.rows(1), p.rows(1)
        p.cache.push(0, p.batch([1, 0], [at + 1, 46]), k, v)
        p.k[0][at], p.v[0][at] = k[0], v[0]
    lens = [len(x) for x in p.k]
    k, v = p.cache.read(0, p.batch(lens))
    for got, x in ((k, p.k), (v, p.v)):
        np.testing.assert_array_equal(got, mx(np.concatenate(x)))


@pytest.mark.parametrize("precision", [MX, "i8"])
def test_one_page_by_several_runs_of_a_push(ctx, precision):
    # a sequence's rows given as runs that end and start within words of eight
    import torch

    p = Pool(ctx, np.random.default_rng(21), precision, 2, 128, 64, [64])
    k, v = p.rows(61), p.rows(61)
    ends = [3, 4, 5, 13, 24, 27, 40, 41, 61]
    b = device_batch(ends, np.repeat(p.pages, len(ends), 0), rows=list(np.diff([0] + ends)))
    dk, dv = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    torch.cuda.synchronize()
    p.cache.push_dev(0, b, dk.data_ptr(), dv.data_ptr())
    ctx.synchronize()
    got = p.cache.read(0, p.batch([61], [61]))
    np.testing.assert_array_equal(got[0], T.rounded(precision, k))
    np.testing.assert_array_equal(got[1], T.rounded(precision, v))


def test_bytes_of_a_cache(ctx):
    for hd, d in ((64, 64), (80, 128), (128, 128), (256, 256)):
        cache = K.PagedCache(ctx, 3, 2, hd, 5, page_size=64, precision=K.MXFP4)
        assert cache.bytes == 3 * 2 * 5 * 64 * (d + d // 16 + 8)
        cache.free()


def test_error_of_normal_rows(ctx):
    # the format's own: within half a step, and of normal rows 0.09 to 0.13 of the norm
    p = Pool(ctx, np.random.default_rng(9), MX, 4, 128, 64, [500])
    p.push([500])
    k, _ = p.cache.read(0, p.batch([500]))
    e = np.linalg.norm(k - p.k[0]) / np.linalg.norm(p.k[0])
    assert 0.09 < e < 0.13


# ---- attention -------------------------------------------------------------------

@pytest.mark.parametrize("H, kv, hd", T.GEOMETRIES)
def test_single_tokens(ctx, H, kv, hd):
    T.test_single_tokens(ctx, MX, H, kv, hd)


@pytest.mark.parametrize("H, kv, hd", [(14, 2, 64), (32, 8, 128), (6, 2, 256), (5, 5, 20), (10, 5, 80)])
@pytest.mark.parametrize("held, rows", [(0, 1), (0, 45), (130, 17), (31, 2), (500, 33)])
def test_chunks(ctx, form, H, kv, hd, held, rows):  # noqa: F811
    T.test_chunks(ctx, form, MX, H, kv, hd, held, rows)


def test_ragged_batches(ctx, form):  # noqa: F811
    T.test_ragged_batches(ctx, form, MX)


@pytest.mark.parametrize("H, kv, hd, counts", [(32, 8, 128, [1100, 0, 900]), (16, 16, 64, [700, 333, 290]), (16, 8, 256, [1500])])
def test_long_prompts(ctx, H, kv, hd, counts):
    T.test_long_prompts(ctx, MX, H, kv, hd, counts)


@pytest.mark.parametrize("window, sinks", T.WINDOWS)
def test_windows(ctx, form, window, sinks):  # noqa: F811
    T.test_windows(ctx, form, MX, window, sinks)


def test_long_window_prompt(ctx):
    T.test_long_window_prompt(ctx, MX)


@pytest.mark.parametrize("held, splits", [(2000, 0), (8001, 0), (2000, 2), (2000, 7), (2000, 63), (8001, 251), (40, 2)])
def test_long_caches_split_over_the_positions(ctx, form, monkeypatch, held, splits):  # noqa: F811
    T.test_long_caches_split_over_the_positions(ctx, form, monkeypatch, MX, held, splits)


def test_scores_that_spread(ctx, form):  # noqa: F811
    T.test_scores_that_spread(ctx, form, MX)


def test_values_of_many_sizes(ctx, form):  # noqa: F811
    T.test_values_of_many_sizes(ctx, form, MX)


def test_rows_of_zeros(ctx, form):  # noqa: F811
    T.test_rows_of_zeros(ctx, form)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, np.finfo(np.float32).min])
def test_what_is_hidden_changes_nothing(ctx, form, bad):  # noqa: F811
    T.test_what_is_hidden_changes_nothing(ctx, form, MX, bad)


def test_what_is_not_finite_reaches_the_rows_that_see_it(ctx, form):  # noqa: F811
    T.test_what_is_not_finite_reaches_the_rows_that_see_it(ctx, form, MX)


@pytest.mark.parametrize("offset", [0, 1])
def test_strided_rows(ctx, form, offset):  # noqa: F811
    T.test_strided_rows(ctx, form, MX, offset)


def test_a_run_of_them(ctx):
    T.test_a_run_of_them(ctx, MX)


@pytest.mark.parametrize("hd", [128, 256])
def test_wide_rows_behind_masks_and_splits(ctx, form, monkeypatch, hd):  # noqa: F811
    T.test_wide_rows_behind_masks_and_splits(ctx, form, monkeypatch, MX, hd)


@pytest.mark.parametrize("small, large", [(None, 44), (None, 90), (-100, 30), (-60, 80), (-118, 88)])
@pytest.mark.parametrize("splits", ["", "3"])
def test_small_values_before_large_ones_keep_their_weights(ctx, form, monkeypatch, small, large, splits):  # noqa: F811
    T.test_small_values_before_large_ones_keep_their_weights(ctx, form, monkeypatch, MX, small, large, splits)


@pytest.mark.parametrize("ahead", ["0", "1"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_one_tile_or_two_at_a_time(ctx, monkeypatch, ahead, hd):
    # both ways few rows are done, to the bit: no tile, one, two, an odd number
    # of a wave's; windows that leave tiles out; splits
    p = Pool(ctx, np.random.default_rng(hd), MX, 2, hd, 32, [700, 130, 33, 1])
    p.push([690, 127, 32, 0])
    p.push([10, 3, 1, 1])
    q = (p.rng.standard_normal((15, 4, hd)) * 1.5).astype(np.float32)
    for tile in ("8", "16"):
        for splits in ("1", "3"):
            outs = []
            for each in (ahead, "0"):
                monkeypatch.setenv("KVAD_PAGED_TILE", tile)
                monkeypatch.setenv("KVAD_PAGED_SPLITS", splits)
                monkeypatch.setenv("KVAD_PAGED_AHEAD", each)
                outs.append([p.check([10, 3, 1, 1], 4, q=q), p.check([10, 3, 1, 1], 4, q=q, window=150, sinks=3)])
            for a, b in zip(*outs):
                np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("precision", [MX, "i8", "f32"])
@pytest.mark.parametrize("n_seq, kv, ragged", [(64, 8, False), (64, 8, True), (37, 8, False), (37, 9, True), (65, 8, False), (2, 200, True)])
def test_the_longest_sequences_go_first(ctx, precision, n_seq, kv, ragged):
    # more workgroups than CUs over sequences of very different lengths, none and
    # alike ones among them: each gets its own
    rng = np.random.default_rng(n_seq + kv)
    lens = [int(n) for n in rng.integers(1, 150, n_seq)]
    lens[0], lens[-1], lens[n_seq // 2] = 149, 149, 1
    counts = [1] * n_seq
    if ragged:
        counts = [int(rng.integers(0, min(n, 3) + 1)) for n in lens]
        lens[1] = counts[1] = 0
    p = Pool(ctx, rng, precision, kv, 64, 32, lens)
    p.push([n - c for n, c in zip(lens, counts)])
    p.push(counts)
    b = K.Batch.host(lens, p.pages, counts) if ragged else K.Batch.host(lens, p.pages, None, n_rows=n_seq)
    q = (rng.standard_normal((sum(counts), kv, 64)) * 1.5).astype(np.float32)
    p.check(counts, kv, q=q, got=p.cache.attend(0, b, kv, q))
    # all of one length, longest_first's other way
    same = [min(lens[0], 100)] * n_seq
    p2 = Pool(ctx, rng, precision, kv, 64, 32, same)
    p2.push(same)
    q = (rng.standard_normal((n_seq, kv, 64)) * 1.5).astype(np.float32)
    p2.check([1] * n_seq, kv, q=q, got=p2.cache.attend(0, K.Batch.host(same, p2.pages, None, n_rows=n_seq), kv, q))


@pytest.mark.parametrize("splits", ["", "3"])
@pytest.mark.parametrize("H, kv, hd, counts, lens", [
    (8, 2, 128, [1] * 9, [1, 40, 700, 33, 64, 5, 900, 2, 31]), (8, 2, 64, [0, 4, 0, 0, 1, 0, 0, 3], [9, 70, 0, 30, 300, 32, 1, 500]),
    (40, 2, 64, [0, 0, 3, 0], [5, 3, 130, 60]), (24, 1, 256, [1, 0, 2], [90, 7, 64]), (4, 4, 128, [0] * 70 + [40, 9], [20] * 70 + [300, 9])])
def test_ragged_batches_of_few_rows(ctx, monkeypatch, H, kv, hd, counts, lens, splits):
    # no more rows than sequences, of a row each or of some with many
    monkeypatch.setenv("KVAD_PAGED_SPLITS", splits)
    p = Pool(ctx, np.random.default_rng(hd + H), MX, kv, hd, 32, lens)
    p.push([n - c for n, c in zip(lens, counts)])
    p.push(counts)
    p.check(counts, H)
    p.check(counts, H, window=50, sinks=2)


@pytest.mark.parametrize("size", [-80, -95, -105, -112, -120, 93])
def test_values_of_one_size(ctx, form, size):  # noqa: F811
    T.test_values_of_one_size(ctx, form, MX, size)


@pytest.mark.parametrize("scale, size", [(0.125, 1.0), (3.0, 1.0), (1e-3, 1e3), (1e-8, 1.0), (1e-20, 1e19), (1e-38, 1.0),
                                         (1e-45, 1.0), (2.0 ** 120, 2.0 ** -120), (3e38, 2.0 ** -127)])
def test_scales(ctx, form, scale, size):  # noqa: F811
    T.test_scales(ctx, form, MX, scale, size)


def test_keys_of_zeros_weigh_alike_at_any_scale(ctx, form):  # noqa: F811
    T.test_keys_of_zeros_weigh_alike_at_any_scale(ctx, form, MX)


@pytest.mark.parametrize("H, kv, hd", [(12, 2, 64), (32, 8, 128), (10, 1, 256)])
def test_short_sequences_share_a_workgroups_waves_in_the_widest_form(ctx, monkeypatch, H, kv, hd):
    T.test_short_sequences_share_a_workgroups_waves_in_the_widest_form(ctx, monkeypatch, MX, H, kv, hd)


@pytest.mark.parametrize("H, kv, hd, held, rows, splits", [
    (4, 2, 128, 5000, 3, ""), (4, 2, 128, 5000, 3, "9"), (2, 1, 256, 700, 20, ""), (2, 1, 256, 2000, 2, "5"),
    (6, 2, 64, 300, 40, ""), (3, 3, 64, 3000, 1, "1")])
def test_error_of_the_whole(ctx, form, monkeypatch, H, kv, hd, held, rows, splits):  # noqa: F811
    T.test_error_of_the_whole(ctx, form, monkeypatch, MX, H, kv, hd, held, rows, splits)


@pytest.mark.parametrize("size", [-100, -60, 60, 93])
def test_keys_of_many_sizes(ctx, form, size):  # noqa: F811
    T.test_keys_of_many_sizes(ctx, form, MX, size)


def test_scores_as_large_as_their_step_allows(ctx, form):  # noqa: F811
    T.test_scores_as_large_as_their_step_allows(ctx, form, MX)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_groups_of_many_sizes(ctx, form, hd):  # noqa: F811
    # the 32-dim groups of a row up to 2^26 and more apart, K's and Q's the other way round
    rng = np.random.default_rng(hd)
    p = Pool(ctx, rng, MX, 2, hd, 32, [150, 40])
    groups = hd // 32
    size = np.exp2(rng.integers(-28, 1, (190, 2, groups))).astype(np.float32).repeat(32, -1)
    p.push([150, 40], k=p.rows(190) * size, v=p.rows(190) * size[::-1])
    q = rng.standard_normal((50, 4, hd)).astype(np.float32)
    q[:, :, :32] *= 2.0 ** 6
    p.check([20, 30], 4, q=q)


def test_codes_past_32_bit_offsets(ctx):
    # pages whose bytes lie past 4 GiB of the pool, beside the first ones
    kv, hd, page, n_pages = 8, 128, 1024, 4000
    cache = K.PagedCache(ctx, 1, kv, hd, n_pages, page_size=page, precision=K.MXFP4)
    try:
        assert cache.bytes > 4.3 * 2 ** 30
        rng = np.random.default_rng(59)
        pages = np.array([[n_pages - 1, 0], [3700, n_pages - 2]], np.int32)
        lens = [1500, 1030]
        k, v = (rng.standard_normal((2530, kv, hd)).astype(np.float32) for _ in range(2))
        b = K.Batch.host(lens, pages, lens)
        cache.push(0, b, k, v)
        got = cache.read(0, b)
        np.testing.assert_array_equal(got[0], mx(k))
        np.testing.assert_array_equal(got[1], mx(v))
        q = rng.standard_normal((4, 16, hd)).astype(np.float32)
        out = cache.attend(0, K.Batch.host(lens, pages, [2, 2]), 16, q)
        for s, (a, e) in enumerate(((0, 1500), (1500, 2530))):
            want, tol = reference(q[2 * s:2 * s + 2], mx(k[a:e]), mx(v[a:e]), e - a - 2, float(np.float32(hd ** -0.5)))
            assert np.all(np.abs(out[2 * s:2 * s + 2] - want) <= tol)
    finally:
        cache.free()


def test_lengths_and_pages_that_lead_nowhere(ctx, form):  # noqa: F811
    import torch

    p = Pool(ctx, np.random.default_rng(31), MX, 2, 64, 32, [96, 64])
    p.push([96, 64])
    before = p.cache.read(0, p.batch([96, 64]))
    q = torch.randn(12, 4, 64, device="cuda")
    for pages, lens in ((np.where(p.pages == p.pages[0, 1], -1, p.pages), [40, -3]),
                        (np.where(p.pages == p.pages[0, 1], p.cache.n_pages, p.pages), [40, 0]), (p.pages, [1000, -2 ** 31])):
        b = device_batch(lens, pages, rows=[6, 6])
        out, k, v = (torch.full((12, n, 64), 7.0, device="cuda") for n in (4, 2, 2))
        torch.cuda.synchronize()
        p.cache.push_dev(0, b, q.data_ptr(), q.data_ptr())
        p.cache.read_dev(0, b, k.data_ptr(), v.data_ptr())
        p.cache.attend_dev(0, b, 4, q.data_ptr(), out.data_ptr())
        ctx.synchronize()
        assert not k.any() and not v.any() and bool(torch.isfinite(out).all()) and not out[6:].any()
        for a, c in zip(before, p.cache.read(0, p.batch([96, 64]))):
            np.testing.assert_array_equal(a, c)


@pytest.mark.parametrize("precision", [MX, "i8", "f16", "f32"])
@pytest.mark.parametrize("chunk", [1, 3, 45])
@pytest.mark.parametrize("window, sinks", [(30, 0), (40, 3), (100, 1), (10, 150), (149, 0), (1 << 30, 1)])
def test_sequences_by_what_their_rows_see(ctx, precision, chunk, window, sinks):
    # more workgroups than CUs, windows that make all sequences alike, some or none,
    # in front of them a chunk behind little, sequences without rows among them
    rng = np.random.default_rng(chunk + window % 1000)
    lens = [chunk + 4] + [int(n) for n in rng.integers(1, 150, 63)]
    counts = [chunk] + [int(n > 9) for n in lens[1:]]
    counts[5] = lens[7] = counts[7] = 0
    p = Pool(ctx, rng, precision, 8, 64, 32, lens)
    p.push([n - c for n, c in zip(lens, counts)])
    p.push(counts)
    p.check(counts, 16, window=window, sinks=sinks)
    ones = [1] * 40
    p2 = Pool(ctx, rng, precision, 8, 64, 32, [max(n, 1) for n in lens[:40]])
    p2.push([max(n, 1) for n in lens[:40]])
    q = (rng.standard_normal((40, 16, 64)) * 1.5).astype(np.float32)
    b = K.Batch.host([len(k) for k in p2.k], p2.pages, None, n_rows=40)
    p2.check(ones, 16, window=window, sinks=sinks, q=q, got=p2.cache.attend(0, b, 16, q, window=window, sinks=sinks))


@pytest.mark.parametrize("precision", [MX, "i8"])
@pytest.mark.parametrize("n_seq, kv", [(2, 160), (17, 40), (63, 8), (64, 8)])
def test_sequences_of_every_length_by_levels(ctx, form, precision, n_seq, kv):  # noqa: F811
    # lengths over three orders, several of a level and of a length, few rows and
    # many, a hint of the longest that is far too small
    rng = np.random.default_rng(n_seq)
    lens = [int(n) for n in np.exp(rng.uniform(0, np.log(600), n_seq))]
    lens[0], lens[-1] = 600, 1
    lens[n_seq // 2] = lens[n_seq // 3] = 300
    counts = [min(n, int(rng.choice([0, 1, 1, 1, 3, 40]))) for n in lens]
    counts[0], counts[-1] = 1, 1
    p = Pool(ctx, rng, precision, kv, 64, 32, lens)
    p.push([n - c for n, c in zip(lens, counts)])
    p.push(counts)
    q = (rng.standard_normal((sum(counts), kv, 64)) * 1.5).astype(np.float32)
    p.check(counts, kv, q=q)
    b = p.batch(counts)
    b.max_len = 2
    p.check(counts, kv, q=q, got=p.cache.attend(0, b, kv, q))
