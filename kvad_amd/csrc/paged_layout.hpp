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

}  // namespace paged
}  // namespace kh
