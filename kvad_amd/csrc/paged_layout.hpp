// Where the paged KV cache keeps an element, and which bytes the attention
// kernel's lanes load for which elements.  Plain integer arithmetic, shared by
// the kernels and by a host test that walks every element and every load.
//
// A layer is an array of blocks [page][KV head].  A block holds one head's
// `page` positions: K, V, then a f32 scale per position for K and for V.
// Everything is in units of 16 bytes, U = 16 / es elements, in the order in
// which the matrix cores take it, so that the attention reads both operands
// from memory straight into registers, 512 bytes a half wave, with nothing
// transposed on the way:
//   K  [dim / U][position][U dims]        a lane's unit: U dims of a position
//   V  [position / U][dim][U positions]   a lane's unit: U positions of a dim
// es is 4 (f32), 2 (f16) or 1 (i8, biased by 128); d is head_dim rounded up
// to 64, 128 or 256, the dims past head_dim zero.
#pragma once

#include <cstddef>
#include <cstdint>

#if defined(__HIPCC__)
#define KH_HD __host__ __device__ __forceinline__
#else
#define KH_HD inline
#endif

namespace kh {
namespace paged {

constexpr int TILE = 32;  // positions the attention takes at a time; divides every page

KH_HD int stored_dims(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
// Rows in 4 bits (MXFP4, "es" 0): E2M1 codes, two a byte, 32 dims of a row
// sharing a factor, a power of two kept as the high byte of its f16, all of a
// row's times the row's f32 scale.  Of a block, K's codes and V's, then K's
// factors and V's, then the scales:
//   K        [dim / 32][position][32 dims]              a lane's unit: a factor's dims
//            positions of a tile of 32 in the order of mx_slot
//   V        [position / 32][dim / 64][position / 8 % 4][dim % 16][dim / 16 % 4][8 positions]
//   factors  K [position][dim / 32], V [position / 8][dim / 32][8 positions]
// V's unit of 16 bytes is 8 positions of the four dims 16 apart that a lane of
// the 16x16x32 product has of 64: one load, where single dims would be four.
// K's order of positions: a block of 16 of the 16x16x32 product (few_pos, below)
// lies together, whole lines a load.
constexpr int MX = 0;
KH_HD int mx_slot(int pos) { return (pos & ~31) | (pos >> 2 & 1) << 4 | (pos >> 3 & 3) << 2 | (pos & 3); }
KH_HD size_t mx_block_bytes(int d, int page) { return (size_t)page * (d + d / 16 + 8); }
// the byte of a code; an even dim's (K) or position's (V) is its low half
KH_HD int mx_k_off(int page, int pos, int dim) { return (dim / 32 * page + mx_slot(pos)) * 16 + dim % 32 / 2; }
KH_HD int mx_v_off(int d, int page, int pos, int dim) {
    return page * d / 2 + pos / 32 * 16 * d + dim / 64 * 1024 + pos / 8 % 4 * 256 + dim % 16 * 16 + dim / 16 % 4 * 4 + pos % 8 / 2;
}
KH_HD int mx_k_factor_off(int d, int page, int pos, int group) { return page * d + pos * (d / 32) + group; }
KH_HD int mx_v_factor_off(int d, int page, int pos, int group) {
    return page * d + page * d / 32 + pos / 8 * (d / 4) + group * 8 + pos % 8;
}
KH_HD int mx_k_scale_off(int d, int page, int pos) { return page * d + page * d / 16 + 4 * pos; }
KH_HD int mx_v_scale_off(int d, int page, int pos) { return page * d + page * d / 16 + 4 * page + 4 * pos; }

KH_HD size_t block_bytes(int es, int d, int page) { return (size_t)2 * page * d * es + (size_t)8 * page; }

KH_HD int k_off(int es, int page, int pos, int dim) {
    const int U = 16 / es;
    return (dim / U * page + pos) * 16 + dim % U * es;
}
KH_HD int v_off(int es, int d, int page, int pos, int dim) {
    const int U = 16 / es;
    return page * d * es + (pos / U * d + dim) * 16 + pos % U * es;
}
KH_HD int k_scale_off(int es, int d, int page, int pos) { return 2 * page * d * es + 4 * pos; }
KH_HD int v_scale_off(int es, int d, int page, int pos) { return 2 * page * d * es + 4 * page + 4 * pos; }

// ---- the attention's loads ---------------------------------------------------
// S^T = K Q^T on the 32x32x16 product: result register i of a lane in half h
// is row 8 (i / 4) + 4 h + i % 4.  Row m is given position tile_pos(m), which
// makes register i of half h position 16 h + i: then the weights of a lane are
// the positions that V's operand (below) wants from that lane.
KH_HD int tile_pos(int m) { return 16 * ((m >> 2) & 1) + 4 * (m >> 3) + (m & 3); }

// K: load j (of d * es / 32) of a lane in half h is this unit of its
// position's dims.  A product takes 16 dims, 8 a half: one load for f16, half
// a load for i8, two loads for f32.
KH_HD int k_load_unit(int es, int j, int h) { return es == 4 ? 4 * (j >> 1) + 2 * h + (j & 1) : 2 * j + h; }
// The dim of element e (of 8) of product s in half h: Q's operand has the same.
KH_HD int k_dim(int es, int s, int h, int e) {
    return es == 1 ? 32 * (s >> 1) + 16 * h + 8 * (s & 1) + e : 16 * s + 8 * h + e;
}
// V: load c (of es) of a lane in half h is this unit of the tile's positions:
// positions 16 h + U c + 0 .. U - 1 of the lane's dim.
KH_HD int v_load_unit(int es, int c, int h) { return es * h + c; }

// The same for the 16x16x32 product, which few rows take: lanes in quarters,
// result register i of a lane in quarter z is row 4 z + i, and the tile's
// positions are two blocks of 16.  Row m of block b is given position
// few_pos(m, b): registers 4 b + i of quarter z are positions 8 z + 4 b + i, and
// V's operand wants positions 8 z .. 8 z + 7 of that quarter.
KH_HD int few_pos(int m, int b) { return 8 * (m >> 2) + 4 * b + (m & 3); }
// K: load j (of d * es / 64) of a lane in quarter z; a product takes 32 dims, 8
// a quarter.
KH_HD int few_k_unit(int es, int j, int z) { return es == 4 ? 8 * (j >> 1) + 2 * z + (j & 1) : 4 * j + z; }
KH_HD int few_k_dim(int es, int s, int z, int e) {
    return es == 1 ? 64 * (s >> 1) + 16 * z + 8 * (s & 1) + e : 32 * s + 8 * z + e;
}
// V: the byte offset, from the tile's first unit of the dim, of positions
// 8 z + 4 c .. (f32, two loads), 8 z .. (f16, one; i8, one of half a unit).
KH_HD int few_v_off(int es, int d, int c, int z) {
    return es == 4 ? (2 * z + c) * d * 16 : es == 2 ? z * d * 16 : (z >> 1) * d * 16 + 8 * (z & 1);
}

// The same of 4-bit rows.  32x32x16: K's load j (of d / 64) is unit 2 j + h, four
// products of a word each; V's are words of 8 positions, quarters 2 h and 2 h + 1
// of the tile, the lane's dims of 64 being two that lie beside each other in a
// unit, for the two dim tiles t of the 64.
// The lane's place among K's positions: mx_slot of the position that row m has.
KH_HD int mx_tile_slot(int m) { return mx_slot(tile_pos(m)); }
KH_HD int mx_few_slot(int m, int b) { return 16 * b + m; }
KH_HD int mx_k_dim(int s, int h, int e) { return 64 * (s >> 2) + 32 * h + 8 * (s & 3) + e; }
KH_HD int mx_v_dim(int dt, int n) { return 64 * (dt >> 1) + (n & 15) + 32 * (n >> 4) + 16 * (dt & 1); }
// 16x16x32: K's load j (of d / 128) is unit 4 j + z, four products; of 64 dims
// half of unit z / 2, two products.  V's dim block db is word db % 4 of its unit.
KH_HD int mx_few_k_dim(int d, int s, int z, int e) {
    return d == 64 ? 16 * z + 8 * s + e : 128 * (s >> 2) + 32 * z + 8 * (s & 3) + e;
}
KH_HD int mx_few_k_lane(int d, int page, int z) { return d == 64 ? (z >> 1) * page * 16 + 8 * (z & 1) : z * page * 16; }

}  // namespace paged
}  // namespace kh
