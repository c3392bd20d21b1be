"""The paged KV cache without a device: where its elements lie and which bytes
the attention's lanes load for which elements (paged_layout.hpp, walked by a
host program), and the refusals of kh_batch_check and of null handles."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

import kvad_amd as K

CSRC = Path(__file__).resolve().parent.parent / "kvad_amd" / "csrc"

WALK = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "paged_layout.hpp"
using namespace kh::paged;
#define MUST(c) do { if (!(c)) { std::printf("line %d: %s (es %d d %d page %d)\n", __LINE__, #c, es, d, page); std::exit(1); } } while (0)
int main() {
    for (int es : {4, 2, 1}) for (int d : {64, 128, 256}) for (int page : {32, 64, 128, 1024}) {
        const size_t block = block_bytes(es, d, page);
        MUST(block % 16 == 0 && block < (1u << 31));
        // every byte of a block is one element's, and all are used
        std::vector<unsigned char> used(block, 0);
        auto take = [&](int off, int n) {
            MUST(off >= 0 && (size_t)off + n <= block && off % n == 0);
            for (int i = 0; i < n; i++) { MUST(!used[off + i]); used[off + i] = 1; }
        };
        for (int p = 0; p < page; p++) {
            for (int e = 0; e < d; e++) { take(k_off(es, page, p, e), es); take(v_off(es, d, page, p, e), es); }
            take(k_scale_off(es, d, page, p), 4);
            take(v_scale_off(es, d, page, p), 4);
        }
        for (unsigned char u : used) MUST(u);
        // the attention's loads: inside the block, and the elements they stand for
        const int U = 16 / es;
        std::vector<int> seen(32, 0);
        for (int n = 0; n < 32; n++) { MUST(tile_pos(n) >= 0 && tile_pos(n) < 32); seen[tile_pos(n)]++; }
        for (int v : seen) MUST(v == 1);
        // result register i of half h is row 8 (i / 4) + 4 h + i % 4: position 16 h + i
        for (int h = 0; h < 2; h++) for (int i = 0; i < 16; i++) MUST(tile_pos(8 * (i / 4) + 4 * h + i % 4) == 16 * h + i);
        for (int in_page = 0; in_page < page; in_page += TILE) for (int lane = 0; lane < 64; lane++) {
            const int n = lane & 31, h = lane >> 5;
            for (int j = 0; j < d * es / 32; j++) {
                // as the kernel adds it up: the lane's part, and the load's
                const int off = (k_load_unit(es, 0, h) * page + tile_pos(n)) * 16 + (k_load_unit(es, j, 0) * page + in_page) * 16;
                MUST((size_t)off + 16 <= block);
                for (int e = 0; e < U; e++) {
                    // element e of load j is element (j U + e) % 8 of product (j U + e) / 8
                    const int dim = k_dim(es, (j * U + e) / 8, h, (j * U + e) % 8);
                    MUST(dim >= 0 && dim < d && off + e * es == k_off(es, page, in_page + tile_pos(n), dim));
                }
            }
            for (int dt = 0; dt < d / 32; dt++) for (int c = 0; c < es; c++) {
                const int off = page * d * es + (v_load_unit(es, 0, h) * d + n) * 16 + (c * d + dt * 32) * 16 + in_page * d * es;
                MUST((size_t)off + 16 <= block);
                for (int e = 0; e < U; e++) MUST(off + e * es == v_off(es, d, page, in_page + 16 * h + c * U + e, dt * 32 + n));
            }
            // the 16x16x32 product's: row r16 of each block, quarter z
            const int r16 = lane & 15, z = lane >> 4;
            for (int b = 0; b < 2; b++) {
                for (int i = 0; i < 4; i++) MUST(few_pos(4 * z + i, b) == 8 * z + 4 * b + i);
                for (int j = 0; j < d * es / 64; j++) {
                    const int off = (few_k_unit(es, 0, z) * page + few_pos(r16, b)) * 16 + (few_k_unit(es, j, 0) * page + in_page) * 16;
                    MUST((size_t)off + 16 <= block);
                    for (int e = 0; e < U; e++) {
                        const int dim = few_k_dim(es, (j * U + e) / 8, z, (j * U + e) % 8);
                        MUST(dim >= 0 && dim < d && off + e * es == k_off(es, page, in_page + few_pos(r16, b), dim));
                    }
                }
            }
            for (int db = 0; db < d / 16; db++) for (int c = 0; c < (es == 4 ? 2 : 1); c++) {
                const int off = page * d * es + in_page * d * es + r16 * 16 + db * 256 + few_v_off(es, d, c, z);
                const int bytes = es == 1 ? 8 : 16;
                MUST((size_t)off + bytes <= block && off % bytes == 0);
                for (int e = 0; e < bytes / es; e++) MUST(off + e * es == v_off(es, d, page, in_page + 8 * z + 4 * c + e, db * 16 + r16));
            }
            for (int i = 0; i < 2; i++) {
                const int ks = 2 * page * d * es + 32 * z + 16 * i + 4 * in_page;
                MUST(ks == k_scale_off(es, d, page, in_page + 8 * z + 4 * i) && (size_t)ks + 4 * page + 16 <= block);
            }
            for (int i = 0; i < 4; i++) {
                const int ks = 2 * page * d * es + 64 * h + 16 * i + 4 * in_page;
                MUST(ks == k_scale_off(es, d, page, in_page + 16 * h + 4 * i));
                MUST(ks + 4 * page == v_scale_off(es, d, page, in_page + 16 * h + 4 * i) && (size_t)ks + 4 * page + 16 <= block);
            }
        }
    }
    std::puts("ok");
}
"""


def test_every_element_and_every_load_of_a_block(tmp_path):
    src = tmp_path / "walk.cpp"
    src.write_text(WALK)
    exe = tmp_path / "walk"
    subprocess.run(["g++", "-O2", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def batch(lens=(40, 0, 70), rows=(1, 0, 3), pages=((0, 1, -1), (-1, -1, -1), (4, 2, 3)), **kw):
    return K.Batch.host(np.array(lens), np.array(pages), None if rows is None else list(rows), **kw)


def test_a_sound_batch_passes():
    batch().check(32, 5)
    batch().check(32, 5, writes=True)
    # a common prefix may be read by both, and written by neither
    batch(lens=(40, 70), rows=(1, 1), pages=((0, 1, -1), (0, 2, 3))).check(32, 4, writes=True)
    batch(rows=None, lens=(5, 6), pages=((0,), (1,)), n_rows=4).check(32, 2)
    K.Batch.host(np.zeros(0), np.zeros((0, 1)), None, n_rows=0).check(32, 1)


@pytest.mark.parametrize("b, n_pages, word", [
    (lambda: batch(lens=(40, 0, 97)), 5, "length"),
    (lambda: batch(lens=(40, -1, 70)), 5, "length"),
    (lambda: batch(rows=(1, 1, 3)), 5, "more rows"),
    (lambda: batch(), 4, "page out of range"),
    (lambda: batch(pages=((0, -1, -1), (-1, -1, -1), (4, 2, 3))), 5, "page out of range"),
    (lambda: batch(rows=None, n_rows=4), 5, "as many rows"),
    (lambda: batch(rows=None, n_rows=0, lens=(1, 1, 99)), 5, None),
])
def test_unsound_batches_are_refused(b, n_pages, word):
    if word is None:
        b().check(32, n_pages)  # no rows: nothing is done, nothing is looked at
        return
    with pytest.raises(K.KvadError, match=word):
        b().check(32, n_pages)


def test_pages_written_twice_are_refused():
    two = batch(lens=(40, 70), rows=(1, 7), pages=((0, 1, -1), (2, 3, 1)))
    two.check(32, 4)
    with pytest.raises(K.KvadError, match="written twice"):
        two.check(32, 4, writes=True)
    # the same page twice in one sequence's own new rows
    with pytest.raises(K.KvadError, match="written twice"):
        batch(lens=(64,), rows=(64,), pages=((1, 1),)).check(32, 4, writes=True)


def test_rows_out_of_order_are_refused():
    b = batch()
    for start in ((0, 3, 1, 4), (-1, 1, 1, 4), (0, 1, 1, 5)):
        keep = np.array(start, np.int32)
        b.row_start = keep.ctypes.data
        with pytest.raises(K.KvadError, match="rows out of order"):
            b.check(32, 5)


def test_sizes_are_refused():
    b = batch()
    for field, value, word in (("n_seq", 0, "no sequences"), ("max_pages", 0, "needs lengths"), ("len", None, "needs"),
                               ("pages", None, "needs"), ("max_pages", 1 << 27, "2\\^30"), ("n_rows", (1 << 30) + 1, "2\\^30")):
        bad = batch()
        setattr(bad, field, value)
        with pytest.raises(K.KvadError, match=word):
            bad.check(32, 5)
    with pytest.raises(K.KvadError):
        b.check(0, 5)
    assert K.lib.kh_batch_check(None, 32, 5, 0) == -1


def test_null_handles_are_refused_without_a_device():
    h = C.c_void_p(7)
    assert K.lib.kh_paged_new(None, 1, 1, 64, K.F16, 64, 1, C.byref(h)) == -1 and h.value is None
    b = batch()
    some = np.zeros(4, np.float32).ctypes.data
    lib = K.lib
    assert lib.kh_paged_push(None, 0, C.byref(b), some, some) == -1
    assert lib.kh_paged_push_dev(None, 0, C.byref(b), some, 0, some, 0) == -1
    assert lib.kh_paged_read(None, 0, C.byref(b), some, some) == -1
    assert lib.kh_paged_read_dev(None, 0, C.byref(b), some, 0, some, 0) == -1
    assert lib.kh_paged_attend(None, 0, C.byref(b), 1, some, 1.0, 0, 0, some) == -1
    assert lib.kh_paged_attend_dev(None, 0, C.byref(b), 1, some, 0, 1.0, 0, 0, some, 0, None, 0) == -1
    n = C.c_size_t(5)
    assert lib.kh_paged_attend_ws(None, C.byref(b), 1, 0, 0, C.byref(n)) == -1
    assert lib.kh_paged_info(None, None, None, None) == -1
    assert lib.kh_paged_free(None) == 0
