"""The device's page tables, rotated rows and block ends without a device: what
their entry points refuse."""
import ctypes as C

import pytest

import kvad_amd as K

LIB = K.lib
SOME = C.create_string_buffer(4096)
AT = (C.addressof(SOME) + 15) // 16 * 16


class NoDevice:
    """A context's handle that is not null; every call below is refused before it is used."""
    h = C.c_void_p(AT + 2048)


def table(**kw):
    fields = dict(n_seq=4, max_pages=8, page_size=64, n_pages=32, len=AT, pages=AT, row_start=AT, free_pages=AT, n_free=AT,
                  status=AT)
    fields.update(kw)
    t = K.PageTable()
    for name, value in fields.items():
        setattr(t, name, value)
    return t


@pytest.mark.parametrize("kw, word", [
    ({"n_seq": 0}, "sequences"), ({"n_seq": 4097}, "sequences"), ({"page_size": 0}, "pages hold"),
    ({"page_size": 16}, "pages hold"), ({"page_size": 96}, "pages hold"), ({"page_size": 2048}, "pages hold"),
    ({"max_pages": 0}, "positions"), ({"max_pages": (1 << 24) + 1}, "positions"), ({"n_pages": 0}, "pages"),
    ({"n_pages": (1 << 30) + 1}, "pages"), ({"len": None}, "null"), ({"pages": None}, "null"), ({"row_start": None}, "null"),
    ({"free_pages": None}, "null"), ({"n_free": None}, "null"), ({"status": None}, "null"), ({"len": AT + 2}, "32-bit"),
    ({"status": AT + 1}, "32-bit")])
def test_tables_that_are_refused(kw, word):
    t = table(**kw)
    for call in (lambda: t.init_dev(NoDevice), lambda: t.step_dev(NoDevice, AT, 1), lambda: t.release_dev(NoDevice, AT)):
        with pytest.raises(K.KvadError, match=word):
            call()


def test_steps_and_releases_that_are_refused():
    t = table()
    for args, word in (((None, 1), "null"), ((AT + 2, 1), "32-bit"), ((AT, 1, AT + 2), "32-bit"),
                       ((AT, 1, None, AT + 4), "64-bit"), ((AT, 1 << 30), "2\\^30")):
        with pytest.raises(K.KvadError, match=word):
            t.step_dev(NoDevice, *args)
    for keep, word in ((None, "null"), (AT + 2, "32-bit")):
        with pytest.raises(K.KvadError, match=word):
            t.release_dev(NoDevice, keep)
    assert LIB.kh_pages_init_dev(None, C.byref(t)) == -1
    assert LIB.kh_pages_step_dev(NoDevice.h, None, AT, 1, None, None) == -1
    assert LIB.kh_pages_release_dev(NoDevice.h, None, AT) == -1


def test_a_tables_batch():
    b = table(len=AT + 4, pages=AT + 8, row_start=AT + 12).batch(7, max_len=100)
    assert (b.n_seq, b.n_rows, b.len, b.pages, b.row_start, b.max_pages, b.max_len) == (4, 7, AT + 4, AT + 8, AT + 12, 8, 100)


FAR = AT + (1 << 20)


def rope(**kw):
    a = dict(cos=2 * FAR, sin=3 * FAR, half=32, max_pos=10, x=AT, position=4 * FAR, m=2, n_vec=1, out=AT, interleaved=False,
             x_stride=0, out_stride=0)
    a.update(kw)
    K.rope_rows_dev(NoDevice, a["cos"], a["sin"], a["half"], a["max_pos"], a["x"], a["position"], a["m"], a["n_vec"], a["out"],
                    a["interleaved"], a["x_stride"], a["out_stride"])


@pytest.mark.parametrize("kw, word", [
    ({"cos": None}, "null"), ({"sin": None}, "null"), ({"x": None}, "null"), ({"position": None}, "null"), ({"out": None}, "null"),
    ({"x": AT + 2}, "32-bit"), ({"position": AT + 1}, "32-bit"), ({"out": AT + 3}, "32-bit"), ({"cos": AT + 2}, "32-bit"),
    ({"m": (1 << 30) + 1}, "2\\^30"), ({"max_pos": (1 << 30) + 1}, "2\\^30"), ({"half": 1 << 20, "n_vec": 1 << 10}, "2\\^30"),
    ({"x_stride": 63}, "less than a row"), ({"out_stride": 63}, "less than a row"), ({"x_stride": 1 << 62}, "too large"),
    ({"out": AT + 4}, "apart"), ({"out": AT + 16 * 4, "m": 2}, "apart"), ({"x_stride": 128}, "apart"),
    ({"cos": AT}, "tables"), ({"sin": AT + 508}, "tables"), ({"position": AT - 4}, "positions"),
    ({"m": 1 << 30, "n_vec": 4, "out": 1 << 60}, "too many rows")])
def test_rotations_that_are_refused(kw, word):
    with pytest.raises(K.KvadError, match=word):
        rope(**kw)


def test_empty_calls_do_nothing():
    rope(m=0)
    rope(n_vec=0)
    rope(half=0)
    norm(m=0)
    norm(n=0)
    assert LIB.kh_rope_rows_dev(None, AT, AT, 1, 1, AT, 0, AT, 0, 1, 0, AT, 0) == -1
    assert LIB.kh_norm_residual_dev(None, AT, AT, None, None, 0, 1.0, None, 0, 1, 0.0, AT, None) == -1


def norm(**kw):
    a = dict(x=AT, y=FAR, m=2, n=64, eps=1e-6, x_out=AT, post=2 * FAR, gate=3 * FAR, gate_stride=0, scale=1.0, pre=4 * FAR,
             out=5 * FAR)
    a.update(kw)
    K.norm_residual_dev(NoDevice, a["x"], a["y"], a["m"], a["n"], a["eps"], a["x_out"], a["post"], a["gate"], a["gate_stride"],
                        a["scale"], a["pre"], a["out"])


@pytest.mark.parametrize("kw, word", [
    ({"x": None}, "null"), ({"y": None}, "null"), ({"x_out": None}, "null"), ({"pre": None}, "comes with"),
    ({"out": None}, "comes with"), ({"eps": -1e-6}, "eps"), ({"eps": float("nan")}, "eps"), ({"eps": float("inf")}, "eps"),
    ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"x": AT + 2}, "32-bit"),
    ({"gate": 3 * FAR + 1}, "32-bit"), ({"m": (1 << 30) + 1}, "2\\^30"), ({"n": (1 << 30) + 1}, "2\\^30"),
    ({"gate_stride": 63}, "less than a row"), ({"gate_stride": 1 << 62}, "too large"),
    ({"x": AT + 4}, "apart"), ({"y": AT + 64 * 8 - 4}, "apart"), ({"out": AT}, "apart"), ({"out": AT + 256}, "apart"),
    ({"post": 5 * FAR}, "apart"), ({"pre": AT + 64 * 4}, "apart"), ({"gate": AT - 64 * 4, "gate_stride": 64}, "apart"),
    ({"m": 1 << 30, "n": 2000, "x_out": 1 << 59, "y": 1 << 60, "out": 1 << 61, "x": 1 << 62, "pre": 8, "gate": None,
      "post": None}, "too many rows")])
def test_block_ends_that_are_refused(kw, word):
    with pytest.raises(K.KvadError, match=word):
        norm(**kw)
