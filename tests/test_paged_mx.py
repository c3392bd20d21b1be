"""4-bit rows of the paged KV cache without a device: where their codes, factors
and scales lie and which of them the attention's lanes load (paged_layout.hpp,
walked by a host program)."""
import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "kvad_amd" / "csrc"

WALK = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "paged_layout.hpp"
using namespace kh::paged;
#define MUST(c) do { if (!(c)) { std::printf("line %d: %s (d %d page %d)\n", __LINE__, #c, d, page); std::exit(1); } } while (0)
int main() {
    for (int d : {64, 128, 256}) for (int page : {32, 64, 128, 256, 512, 1024}) {
        const size_t block = mx_block_bytes(d, page);
        const int kf = page * d, vf = page * d + page * d / 32, groups = d / 32;
        MUST(block % 16 == 0 && block < (1u << 31) && kf % 16 == 0 && vf % 16 == 0);
        // every half byte of a block is one code's, or its byte one factor's or scale's
        std::vector<unsigned char> used(2 * block, 0);
        auto take = [&](int off, int n) {
            MUST(off >= 0 && (size_t)off + n <= block && off % n == 0);
            for (int i = 2 * off; i < 2 * (off + n); i++) { MUST(!used[i]); used[i] = 1; }
        };
        auto half = [&](int off, int odd) { MUST(off >= 0 && (size_t)off < block && !used[2 * off + odd]); used[2 * off + odd] = 1; };
        for (int p = 0; p < page; p++) {
            for (int e = 0; e < d; e++) { half(mx_k_off(page, p, e), e & 1); half(mx_v_off(d, page, p, e), p & 1); }
            for (int g = 0; g < groups; g++) { take(mx_k_factor_off(d, page, p, g), 1); take(mx_v_factor_off(d, page, p, g), 1); }
            take(mx_k_scale_off(d, page, p), 4);
            take(mx_v_scale_off(d, page, p), 4);
        }
        for (unsigned char u : used) MUST(u);
        // code e of the word at off, and what lies there
        auto k_code = [&](int off, int e, int pos, int dim) { MUST((size_t)off + 4 <= block && dim >= 0 && dim < d && off + e / 2 == mx_k_off(page, pos, dim) && (e & 1) == (dim & 1)); };
        auto v_code = [&](int off, int e, int pos, int dim) { MUST((size_t)off + 4 <= block && dim >= 0 && dim < d && off + e / 2 == mx_v_off(d, page, pos, dim) && (e & 1) == (pos & 1)); };
        for (int in_page = 0; in_page < page; in_page += TILE) {
            // the write's words of V: word i of the tile, [dim / 64][position / 8][dim % 16][dim / 16 % 4]
            for (int j = 0; j < d / 64; j++) for (int i = 0; i < 256; i++) for (int e = 0; e < 8; e++)
                v_code(mx_v_off(d, page, in_page, 0) + 4 * (i + 256 * j), e, in_page + 8 * (i >> 6) + e, 64 * j + (i >> 2 & 15) + 16 * (i & 3));
            for (int lane = 0; lane < 64; lane++) {
                // 32x32x16, as the kernel adds the offsets up: the lane's part, and the load's
                const int n = lane & 31, h = lane >> 5;
                const int k_lane = (k_load_unit(MX, 0, h) * page + mx_tile_slot(n)) * 16, pos = in_page + tile_pos(n);
                std::vector<int> dims(d, 0);
                for (int j = 0; j < d / 64; j++) for (int w = 0; w < 4; w++) for (int e = 0; e < 8; e++) {
                    const int dim = mx_k_dim(4 * j + w, h, e);
                    k_code(k_lane + (k_load_unit(MX, j, 0) * page + in_page) * 16 + 4 * w, e, pos, dim);
                    // its factor: byte 2 j + h of the position's
                    MUST(kf + tile_pos(n) * groups + in_page * groups + 2 * j + h == mx_k_factor_off(d, page, pos, dim / 32));
                    dims[dim]++;
                }
                const int kf_off = kf + tile_pos(n) * groups + in_page * groups;
                MUST(kf_off % (groups < 4 ? 2 : 4) == 0 && (size_t)kf_off + groups <= block);
                const int vc_lane = page * d / 2 + 512 * h + 16 * (n & 15) + 8 * (n >> 4), vf_lane = vf + d / 2 * h + 8 * (n >> 4);
                for (int i = 0; i < d / 32; i++) {
                    const int code = vc_lane + 1024 * (i >> 1) + 256 * (i & 1) + in_page * (d / 2);
                    const int fac = vf_lane + 16 * (i >> 1) + d / 4 * (i & 1) + in_page * (d / 32);
                    MUST(code % 8 == 0 && fac % 8 == 0 && (size_t)code + 8 <= block && (size_t)fac + 8 <= block);
                    for (int t = 0; t < 2; t++) for (int e = 0; e < 8; e++) {
                        const int dim = mx_v_dim(2 * (i >> 1) + t, n), p = in_page + 16 * h + 8 * (i & 1) + e;
                        v_code(code + 4 * t, e, p, dim);
                        MUST(fac + e == mx_v_factor_off(d, page, p, dim / 32));
                    }
                }
                // four result rows of a dim tile, one behind the other, are four such dims
                for (int dt = 0; dt < d / 32; dt++) for (int c = 0; c < 4; c++) for (int e = 0; e < 4; e++)
                    MUST(mx_v_dim(dt, 8 * c + 4 * h + e) == mx_v_dim(dt, 8 * c + 4 * h) + e);
                // 16x16x32
                const int r16 = lane & 15, z = lane >> 4;
                for (int b = 0; b < 2; b++) for (int j = 0; j < (d + 127) / 128; j++) {
                    const int p = in_page + few_pos(r16, b);
                    const int off = mx_few_k_lane(d, page, z) + mx_few_slot(r16, 0) * 16 + 256 * b + (4 * j * page + in_page) * 16;
                    MUST(off % 8 == 0 && (size_t)off + (d == 64 ? 8 : 16) <= block);
                    for (int w = 0; w < (d == 64 ? 2 : 4); w++) for (int e = 0; e < 8; e++) {
                        const int dim = mx_few_k_dim(d, 4 * j + w, z, e);
                        k_code(off + 4 * w, e, p, dim);
                        const int byte = d == 64 ? z >> 1 : 4 * j + z;
                        MUST(kf + few_pos(r16, 0) * groups + 4 * b * groups + in_page * groups + byte == mx_k_factor_off(d, page, p, dim / 32));
                    }
                }
                for (int i = 0; i < d / 64; i++) {
                    const int code = page * d / 2 + 256 * z + 16 * r16 + 1024 * i + in_page * (d / 2);
                    const int fac = vf + d / 4 * z + 16 * i + in_page * (d / 32);
                    MUST(code % 16 == 0 && fac % 16 == 0 && (size_t)code + 16 <= block && (size_t)fac + 16 <= block);
                    for (int w = 0; w < 4; w++) for (int e = 0; e < 8; e++) {
                        const int dim = 16 * (4 * i + w) + r16, p = in_page + 8 * z + e;
                        v_code(code + 4 * w, e, p, dim);
                        MUST(fac + 8 * (w / 2) + e == mx_v_factor_off(d, page, p, dim / 32));
                    }
                }
                const int scales = page * d + page * d / 16;
                MUST(scales + 4 * (16 * h + (lane & 15)) + 4 * in_page == mx_k_scale_off(d, page, in_page + 16 * h + (lane & 15)));
                MUST(scales + 4 * (8 * z + (lane & 7)) + 4 * page + 4 * in_page == mx_v_scale_off(d, page, in_page + 8 * z + (lane & 7)));
            }
        }
        // both halves and all quarters together have every dim once
        for (int few = 0; few < 2; few++) {
            std::vector<int> dims(d, 0);
            for (int s = 0; s < d / (few ? 32 : 16); s++) for (int z = 0; z < (few ? 4 : 2); z++) for (int e = 0; e < 8; e++)
                dims[few ? mx_few_k_dim(d, s, z, e) : mx_k_dim(s, z, e)]++;
            for (int v : dims) MUST(v == 1);
        }
        std::vector<int> dims(d, 0);
        for (int dt = 0; dt < d / 32; dt++) for (int n = 0; n < 32; n++) dims[mx_v_dim(dt, n)]++;
        for (int v : dims) MUST(v == 1);
    }
    std::puts("ok");
}
"""


def test_every_code_and_every_load_of_a_block(tmp_path):
    src = tmp_path / "walk.cpp"
    src.write_text(WALK)
    exe = tmp_path / "walk"
    subprocess.run(["g++", "-O2", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
