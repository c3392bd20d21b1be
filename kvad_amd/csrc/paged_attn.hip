// Attention over the paged KV cache: out = softmax(scale q K^T) V for ragged
// batches of new rows, causal, over a sequence's whole cache or through a
// window with sinks.  One pass over the positions, the running maximum and sum
// of each row's softmax in registers.
//
// The products run on the f16 matrix cores with 32-bit results.  A f32 operand
// is cut into two f16 pieces, hi + lo, 22 bits of significand: enough that the
// result is as near the 64-bit one as f32 arithmetic is (the operands of a row
// share a power-of-two scale, so f16's exponents are wide enough).  Cache rows
// of f16, i8 codes, and 4-bit codes times their factor, are one exact f16 each:
// two products a tile, q's or the weights' pieces against them; f32 rows are two
// pieces and three products (lo by lo is below the 22 bits).  The f32 matrix cores
// run at a sixteenth of the f16 rate.  Two 4-bit codes become f16, times a factor
// (K's: a lane's unit has one), in one instruction; V's factors, one a position,
// are a product more.  The row's scale is a score's or a weight's, as the others'.
//
// A wave takes rows of one KV head (query tokens x the head's group, flattened:
// each K and V byte is read once for the whole group) and 32 positions at a
// time: S^T = K Q^T, then O^T += V^T P^T.  In the transposed form a lane keeps
// one row's weights for the positions that V's operand wants of it, so the
// weights go from one product to the next in registers, and K and V come from
// memory in operand order (paged_layout.hpp): there is no LDS in the loop.  K of
// the next tile and V of this one are loaded while the weights are computed
// (wide f32 rows: by halves, each as soon as its registers are free).
//
// Two forms of the wave's work.  many_rows: 32 rows on 32x32x16 products, each
// piece a product of its own.  few_rows: 8 or 16 rows on 16x16x32 products; with
// 8, the pieces are the two halves of the 16 columns, so that one product does
// both, and their sums meet in the scores (by a lane move) and at the end.
//
// What bounds them.  few_rows: HBM (64 sequences of up to 4000 i8 positions, 8
// heads of 128: 70 us for 362 MB, 5.1 TB/s, a large copy's rate; in 4 bits 44 us
// for 203 MB, 4.6 TB/s: of 32 long ones, a workgroup a CU, 5.6), or for one
// short sequence the trips to memory and the joining launch.  many_rows: the
// matrix cores, 47% at work, behind 6 vector instructions a product (a wave
// issues one in 8 cycles, so two waves a SIMD, all that 256 registers allow,
// just fill it): 512 tokens behind 8000, f16, 32 heads of 128: 141 us, 490
// TFLOP/s of the scores and values or 980 of the products run for them, where a
// large bf16 product of the library reaches 1200; in 4 bits 132 to 139 us, 262
// vector instructions and 32 products a tile, 112 of them for the codes.
#include <algorithm>
#include <utility>

#include "paged.hpp"

namespace kh {
namespace paged {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any float

typedef const __attribute__((address_space(4))) int32_t const_i32;

constexpr float LOW = -3.0e38f;  // a running maximum that nothing has raised
// Weights times V's scales are kept at 2^BASE times their size over the row's
// reference, which follows their bound only when it is SLACK powers of two
// behind: under 2^15, f16's range, and the sums are rescaled for few tiles.
constexpr float BASE = 8.0f, SLACK = 6.0f;
// A weight alone is as much smaller or larger as V's scales are large or small,
// and its exponent, a float, is the less exact the further it is from 0.  So UP
// powers of two of the product are in the scale, about as many as keep the weights
// near 1 where V is, and the reference takes the scales' exponent as LEAST or more:
// f32 and f16, scales of 2^82 (|v| of 2^96) to 2^-126, weights of up to 2^120, of
// which a lane adds 16, and of 2^-94 for the largest of a row, with 32 powers of
// two below it; i8, scales of 2^89 on and codes of up to 127, 2^122 and 2^-94, and
// rows with scales under 2^-121 held to up to 5 bits less.  Sums are kept at 2^-24
// of that, for millions of tiles of the first and normal floats of the second.
constexpr float SUM_SCALE = 0x1p-24f;
template <int ES>
struct VScale {
    static constexpr int UP = ES == 1 ? 13 : 20, LEAST = ES == 1 ? -121 : -126;
    static constexpr float TIMES = ES == 1 ? 0x1p13f : 0x1p20f;
};
constexpr float out_scale(int es) { return SUM_SCALE / (es == 1 ? VScale<1>::TIMES : VScale<4>::TIMES); }  // values over sum

struct Args {
    const char *pool;
    Batch b;
    const float *q;
    size_t q_stride;
    float *out;
    size_t out_stride;
    float *part, *part_ml;  // [split][row][head]: values [D], (reference, sum)
    size_t block;
    int n_kv, group, hd, n_pages, page, page_shift;
    int tiles_per, splits, split_tiles, window, sinks;
    int longest_first;
    float scale, out_scale;
};

__device__ __forceinline__ float shfl(float v, int x) { return __shfl_xor(v, x); }
// lane I's value, in each row of 16.  Not where lanes are switched off: one that
// is gives zero.
template <int I>
__device__ __forceinline__ float of_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x150 + I, 0xf, 0xf, true));
}
// A product with another lane's value is one instruction if the two are found
// beside each other: computed here, not where it is first wanted.
__device__ __forceinline__ float here_and_now(float v) {
    asm volatile("" : "+v"(v));
    return v;
}
// the largest of each row of 16, in all of its lanes
__device__ __forceinline__ unsigned row_max(unsigned v) {
    v = max(v, (unsigned)dev::dpp<dev::DPP_XOR1>((int)v));
    v = max(v, (unsigned)dev::dpp<dev::DPP_XOR2>((int)v));
    v = max(v, (unsigned)dev::dpp<dev::DPP_HALF_MIRROR>((int)v));
    return max(v, (unsigned)dev::dpp<dev::DPP_MIRROR>((int)v));
}
// f(0), f(1), ... f(N - 1), each with its number as a constant
template <typename F, int... I>
__device__ __forceinline__ void each_(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
    each_(f, std::make_integer_sequence<int, N>{});
}
// V's scale at 2^UP.  A row of V that is not finite, by its scale, or whose scale
// is too large for that (|v| from 2^122 on): no part of any sum, and NaN as a score,
// so that only rows that see it are NaN.
template <int ES>
__device__ __forceinline__ void only_finite(float &v_scale, float &k_scale) {
    const bool finite = (__builtin_bit_cast(int, v_scale) & 0x7fffffff) < 0x7f800000 - (VScale<ES>::UP << 23);
    k_scale = finite ? k_scale : __builtin_bit_cast(float, NAN_BITS);
    v_scale = finite ? v_scale * VScale<ES>::TIMES : 0.0f;
}
// the value 8 lanes on, in each row of 16
__device__ __forceinline__ float other_half(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true));
}
// A copy made here: the register that v was loaded into takes the next load at
// once, where a copy at the loop's end would wait for that load.
__device__ __forceinline__ float copy(float v) {
    float r;
    asm volatile("v_mov_b32 %0, %1" : "=v"(r) : "v"(v));
    return r;
}
__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
// A sum of weights at a reference `by` powers of two on (negative, or zero).  A
// reference holds the exponent of V's scales, so it can move by more than a
// float's exponents: rows of zeros ahead of large ones, whose sums are large and
// count in full.  So in two steps, none of which is flushed; sums of values are
// not large where the reference was low, and take one.
__device__ __forceinline__ float moved(float sum, float by) {
    const float half = exp2_(0.5f * by);
    return sum * half * half;
}

// hi + lo of two floats.  hi is cut off, not rounded: one instruction that the
// compiler cannot split into two conversions, whose ties need not agree, one
// for the product and one for the remainder.  The remainder is under 2^-10 of
// the value and exact, lo is off by 2^-22 of the value.
__device__ __forceinline__ void split2(float a, float b, h2 &hi, h2 &lo) {
    float minus = -1.0f;
    asm("" : "+s"(minus));  // known, the product would become a conversion and a subtraction
    hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
    lo = h2{(_Float16)__builtin_fmaf((float)hi.x, minus, a), (_Float16)__builtin_fmaf((float)hi.y, minus, b)};
}
__device__ __forceinline__ void split8(const float *x, h8 &hi, h8 &lo) {
    h2 h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) split2(x[2 * i], x[2 * i + 1], h[i], l[i]);
    hi = h8{h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
    lo = h8{l[0].x, l[0].y, l[1].x, l[1].y, l[2].x, l[2].y, l[3].x, l[3].y};
}

// Eight biased codes as f16: the bits of 1024 + byte are 0x6400 | byte.
__device__ __forceinline__ h8 codes8(unsigned a, unsigned b) {
    const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const h2 r0 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) + off;
    const h2 r1 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) + off;
    const h2 r2 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + off;
    const h2 r3 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + off;
    return h8{r0.x, r0.y, r1.x, r1.y, r2.x, r2.y, r3.x, r3.y};
}

// Eight 4-bit codes times their factor, a power of two as a float.
__device__ __forceinline__ h8 mx8(unsigned w, float factor) {
    const h2 r0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, factor, 0), r1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, factor, 1);
    const h2 r2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, factor, 2), r3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, factor, 3);
    return h8{r0.x, r0.y, r1.x, r1.y, r2.x, r2.y, r3.x, r3.y};
}
// Byte `i` of w, the high one of an f16 power of two, as a float.
__device__ __forceinline__ float mx_factor(unsigned w, int i) {
    return __builtin_bit_cast(float, ((w >> (8 * i) & 0xff) << 21) + (112u << 23));
}
// Eight of them as f16.
__device__ __forceinline__ h8 mx_factors(unsigned a, unsigned b) {
    const h2 r0 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0u, a, 0x010c000cu));
    const h2 r1 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0u, a, 0x030c020cu));
    const h2 r2 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0u, b, 0x010c000cu));
    const h2 r3 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0u, b, 0x030c020cu));
    return h8{r0.x, r0.y, r1.x, r1.y, r2.x, r2.y, r3.x, r3.y};
}

__device__ __forceinline__ f16v mfma(h8 a, h8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4v mfma(h8 a, h8 b, f4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

typedef unsigned u2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u2v load8(dev::rsrc_t r, unsigned voff, unsigned soff) {
    return __builtin_bit_cast(u2v, __builtin_amdgcn_raw_buffer_load_b64(r, voff, soff, 0));
}
__device__ __forceinline__ float load4(dev::rsrc_t r, unsigned voff, unsigned soff) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, voff, soff, 0));
}
__device__ __forceinline__ int4 load16(dev::rsrc_t r, unsigned voff, unsigned soff) {
    return __builtin_bit_cast(int4, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0));
}

// Where a block's scales start, K's and then V's.
template <int ES, int D>
__device__ __forceinline__ unsigned scales_at(int page) {
    return (unsigned)(ES == MX ? page * D + page * D / 16 : 2 * page * D * ES);
}
// A position's factors of K, D / 32 bytes.
template <int D>
__device__ __forceinline__ u2v load_kf(dev::rsrc_t r, unsigned voff, unsigned soff) {
    if (D == 64) return u2v{(unsigned)__builtin_amdgcn_raw_buffer_load_b16(r, voff, soff, 0), 0u};
    if (D == 128) return u2v{(unsigned)__builtin_amdgcn_raw_buffer_load_b32(r, voff, soff, 0), 0u};
    return load8(r, voff, soff);
}

// The positions a wave's rows see, as a list of 32-position tiles: those of
// the sinks, then those from the first window's start on.
struct Range {
    int front, from, n;  // tiles of the sinks apart from the rest; first tile of the rest; tiles in all
    __device__ int start(int i) const { return (i < front ? i : i - front + from) * TILE; }
};
__device__ __forceinline__ Range range_of(int p_lo, int p_hi, int cap, int window, int sinks) {
    Range r{0, 0, 0};
    const int end = min(p_hi + 1, cap);
    if (end <= 0) return r;
    const int last = (end + TILE - 1) / TILE;
    const int front = (min(sinks, end) + TILE - 1) / TILE;
    const int from = window == INT32_MAX ? 0 : max(0, p_lo - window + 1) / TILE;
    if (front < from) {
        r.front = front;
        r.from = from;
    }
    r.n = r.front + max(last - r.from, 0);
    return r;
}

// A wave's rows: those of sequence `seq` from row0 on (rows x group), nr of them
// or more; its positions' tiles from t_at up to t_end, every WS'th.
struct Job {
    int seq, head, split, seq_row, first, row0, nr;
    int p_lo, p_hi, t_at, t_end;
    Range range;
};

__device__ __forceinline__ void find_range(const Args &a, Job &w) {
    // named scalars (the vector unit divides): so is what is made of them
    w.p_lo = __builtin_amdgcn_readfirstlane(w.first + w.row0 / a.group);
    w.p_hi = __builtin_amdgcn_readfirstlane(w.first + (w.row0 + w.nr - 1) / a.group);
    w.range = range_of(w.p_lo, w.p_hi, a.b.max_pages << a.page_shift, a.window, a.sinks);
    w.t_at = 0;
    w.t_end = w.range.n;
    if (a.splits > 1) {
        w.t_at = min(w.split * a.split_tiles, w.range.n);
        // the last takes what is left: a longer sequence than max_len said
        if (w.split < a.splits - 1) w.t_end = min(w.t_at + a.split_tiles, w.range.n);
    }
}

// A tile's block and place.
struct Where {
    dev::rsrc_t r;
    int start, in_page;
    bool there;
    // V's bytes ahead of it.  Named a scalar: where the compiler computes it with
    // the vector unit, each load would be a loop over the values it may have.
    __device__ __forceinline__ unsigned v_at(int row_bytes) const {
        return (unsigned)__builtin_amdgcn_readfirstlane(in_page * row_bytes);
    }
};
struct Table {
    const_i32 *pages;
    __device__ Table(const Args &a, int seq)
        // read through the scalar cache: no wait for it is a wait for K or V
        : pages((const_i32 *)dev::uniform_ptr(a.b.pages + (size_t)seq * a.b.max_pages)) {}
    __device__ __forceinline__ int page_of(const Args &a, const Job &w, int t) const {
        return pages[w.range.start(t) >> a.page_shift];
    }
    __device__ __forceinline__ Where find(const Args &a, const Job &w, int t, int page) const {
        Where x;
        x.start = w.range.start(t);
        x.there = page >= 0 && page < a.n_pages;
        if (!x.there) page = 0;  // read, and hidden from every row
        x.in_page = x.start & (a.page - 1);
        x.r = dev::rsrc(dev::uniform_ptr(a.pool + ((size_t)page * a.n_kv + w.head) * a.block), a.block);
        return x;
    }
};

// The row of the flattened row `rr`, and where its query and its output start.
struct Row {
    int j, g, pos;
    __device__ Row(const Args &a, const Job &w, int rr) {
        j = rr / a.group;
        g = rr - j * a.group;
        pos = w.first + j;
    }
    __device__ const float *query(const Args &a, const Job &w) const {
        return a.q + (size_t)(w.seq_row + j) * a.q_stride + (size_t)(w.head * a.group + g) * a.hd;
    }
};

// Eight of a query's dims for each of NS products, the first of product s at
// dim0(s); zeros past head_dim.  Returns the largest magnitude's bits.
template <int NS, typename F>
__device__ __forceinline__ int load_q(const float *x, int hd, F dim0, float (&v)[NS][8]) {
    int amax = 0;
    float4u f[NS][2];
#pragma unroll
    for (int i = 0; i < NS; i++)
#pragma unroll
        for (int c = 0; c < 2; c++) f[i][c] = *reinterpret_cast<const float4u *>(x + min(dim0(i) + 4 * c, hd - 4));
    __builtin_amdgcn_sched_barrier(0);  // all loads ahead of the first use
#pragma unroll
    for (int i = 0; i < NS; i++) {
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[i][4 * c + e] = dim0(i) + 4 * c < hd ? f[i][c][e] : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) amax = max(amax, __builtin_bit_cast(int, v[i][e]) & 0x7fffffff);
    }
    return amax;
}
// The power of two that brings a query under 2^15, inverted, and the score, in
// powers of two, of an accumulated product of 1: not zero, by which a hidden
// position's -infinity would be NaN (scores that small are all alike: a product is
// under 2^120), and not infinite, by which a product of zero would be.
__device__ __forceinline__ float q_scale(int amax, float scale, float &rowf) {
    const int e = min(max((amax >> 23) - 126 - 15, -126), 113);
    const float f = scale * (1.44269504088896341f * __builtin_bit_cast(float, (127 + e) << 23));
    rowf = fminf(fmaxf(f, 0x1p-149f), 3.40282347e38f);
    return __builtin_bit_cast(float, (127 - e) << 23);
}
// 1 / 2^k from 2^k
__device__ __forceinline__ float inv_pow2(float s) { return __builtin_bit_cast(float, 0x7f000000 - __builtin_bit_cast(int, s)); }

// The exponent of the largest of V's scales, from the bits of it at 2^UP.
template <int ES>
__device__ __forceinline__ float scale_exp(unsigned bits) {
    return (float)max((int)(bits >> 23) - 127 - VScale<ES>::UP, VScale<ES>::LEAST);
}
// 1 / 2^k from 2^(k + UP)
template <int ES>
__device__ __forceinline__ float inv_v(float s) {
    return __builtin_bit_cast(float, 0x7f000000u + ((unsigned)VScale<ES>::UP << 23) - __builtin_bit_cast(unsigned, s));
}

// The sums of four waves over the same rows, column `col` of `cols` a lane, at
// the largest reference: two and two and then one, through lds.  Wave 0 has them.
template <int N>
__device__ __forceinline__ void join_waves(float (&o)[N], float &ref, float &sum, int wave, int lane, int col, bool tells,
                                           float *lds) {
    constexpr int SN = N < 64 ? N : 64;  // registers a step
    float(*s_ref)[32] = reinterpret_cast<float(*)[32]>(lds), (*s_sum)[32] = s_ref + 4;
    float *s_acc = lds + 256;
    if (tells) {
        s_ref[wave][col] = ref;
        s_sum[wave][col] = sum;
    }
    __syncthreads();
    float all = s_ref[0][col];
#pragma unroll
    for (int w = 1; w < 4; w++) all = fmaxf(all, s_ref[w][col]);
    const float f = exp2_(ref - all);
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) sum = sum + moved(s_sum[w][col], s_ref[w][col] - all);
    ref = all;
#pragma unroll
    for (int k = 0; k < N; k++) o[k] = o[k] * f;
#pragma unroll
    for (int half = 2; half >= 1; half /= 2) {
#pragma unroll
        for (int k0 = 0; k0 < N; k0 += SN) {
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int k = 0; k < SN; k++) s_acc[((wave - half) * SN + k) * 64 + lane] = o[k0 + k];
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int k = 0; k < SN; k++) o[k0 + k] = o[k0 + k] + s_acc[(wave * SN + k) * 64 + lane];
            }
            __syncthreads();
        }
    }
}
// its LDS, in floats
template <int N>
constexpr int join_floats() { return 256 + 2 * (N < 64 ? N : 64) * 64; }

// A lane's part of a row's result, four dims from dim(c) on in o[4 c ..]: into
// the output, or beside the other splits'.
template <int ES, int N, typename F>
__device__ __forceinline__ void put_row(const Args &a, const Job &w, const Row &row, const float (&o)[N], float ref,
                                        float sum, bool tells, int stored, F dim) {
    const size_t r = (size_t)(w.seq_row + row.j);
    const int q_head = w.head * a.group + row.g;
    if (a.splits > 1) {
        const size_t at = ((size_t)w.split * a.b.n_rows + r) * (a.n_kv * a.group) + q_head;
        if (tells) reinterpret_cast<float2 *>(a.part_ml)[at] = make_float2(ref, sum);
        if (sum == 0.0f) return;  // nothing seen here: the merge reads no values
        float *to = a.part + at * stored;
#pragma unroll
        for (int c = 0; c < N / 4; c++)
            *reinterpret_cast<float4 *>(to + dim(c)) = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
        return;
    }
    float *to = a.out + r * a.out_stride + (size_t)q_head * a.hd;
    constexpr float down = out_scale(ES);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int c = 0; c < N / 4; c++)
        if (dim(c) < a.hd)
            *reinterpret_cast<float4u *>(to + dim(c)) =
                float4u{o[4 * c] * down * inv, o[4 * c + 1] * down * inv, o[4 * c + 2] * down * inv, o[4 * c + 3] * down * inv};
}

// Rows of K and V whose raw loads many_rows has one set of registers for: two
// sets leave 128 dims one wave a SIMD and 256 none (512 f32 tokens behind 8000,
// 32 heads on 8 of 128: 286 us against 342; 16 of 256: 329 against 638 by 16 rows).
constexpr bool shares_registers(int es, int d) { return es == 4 && d >= 128; }

// 32 rows; WS waves share them (1: each has its own).
template <int ES, int D, int WS>
__device__ __forceinline__ void many_rows(const Args &a, Job &w, int wave, float *lds) {
    constexpr int NK = ES == MX ? D / 64 : D * ES / 32;  // loads of a lane for K
    constexpr int DT = D / 32;       // dim tiles of V
    constexpr int NS = D / 16;       // products over the dims
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    find_range(a, w);
    const Row row(a, w, w.row0 + min(n, w.nr - 1));

    f16v acc[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) acc[i] = f16v{0.0f};
    float ref = LOW, sum = 0.0f;  // the row's reference and this lane's part of its sum

    const int P = a.page;
    const unsigned k_lane = (unsigned)(k_load_unit(ES, 0, h) * P + (ES == MX ? mx_tile_slot(n) : tile_pos(n))) * 16;
    const unsigned v_lane = (unsigned)(P * D * ES) + (unsigned)(v_load_unit(ES, 0, h) * D + n) * 16;
    // scales: a lane holds position 16 h + lane % 16's, and takes the others of
    // its half from the lanes beside it
    const unsigned s_lane = scales_at<ES, D>(P) + 4 * (16 * h + (lane & 15));
    const Table table(a, w.seq);
    // 4-bit rows: K's factors of the lane's position, V's codes and factors of 8
    // positions, two loads for each 64 dims
    const unsigned kf_lane = (unsigned)(P * D) + (unsigned)tile_pos(n) * (D / 32);
    const unsigned vc_lane = (unsigned)(P * D / 2) + 512 * h + 16 * (n & 15) + 8 * (n >> 4);
    const unsigned vf_lane = (unsigned)(P * D + P * D / 32) + (D / 2) * h + 8 * (n >> 4);
    u2v vc[ES == MX ? D / 32 : 1], vf[ES == MX ? D / 32 : 1];
    u2v kf = {0u, 0u};
    // Wide rows (SHARED): K and V take turns in the same registers, half of
    // the dims at a time, each half loaded as soon as the other's is used.
    constexpr bool SHARED = shares_registers(ES, D);
    int4 kraw[NK], vown[SHARED || ES == MX ? 1 : DT * ES];
    int4 *const vraw = SHARED ? kraw : vown;
    float ks, vs, k_own = 0.0f;
    auto load_s = [&](const Where &x) {
        ks = load4(x.r, s_lane, 4 * x.in_page);
        vs = load4(x.r, s_lane, 4 * P + 4 * x.in_page);
        if (ES == 4) k_own = dev::bldf(x.r, (unsigned)(2 * P * D * ES) + 4 * (x.in_page + tile_pos(n)));
    };
    auto load_k = [&](const Where &x, int from, int to) {
#pragma unroll
        for (int i = from; i < to; i++) {
            const int unit = k_load_unit(ES, i, 0);
            kraw[i] = load16(x.r, k_lane, (unsigned)(unit * P + x.in_page) * 16);
        }
        if constexpr (ES == MX) kf = load_kf<D>(x.r, kf_lane, (unsigned)x.in_page * (D / 32));
    };
    auto load_v = [&](const Where &x, int from, int to) {
        if constexpr (ES == MX) {
            const unsigned at = x.v_at(D / 2), f_at = x.v_at(D / 32);
#pragma unroll
            for (int i = 0; i < D / 32; i++) {  // quarter 2 h + i % 2 of 64 dims i / 2
                vc[i] = load8(x.r, vc_lane + 1024 * (i >> 1) + 256 * (i & 1), at);
                vf[i] = load8(x.r, vf_lane + 16 * (i >> 1) + (D / 4) * (i & 1), f_at);
            }
            return;
        }
        const unsigned at = x.v_at(D * ES);
#pragma unroll
        for (int i = from; i < to; i++) {
            constexpr int E = ES == MX ? 1 : ES;
            const int dt = i / E, c = i % E;
            vraw[i] = load16(x.r, v_lane + (c * D + dt * 32) * 16, at);
        }
    };

    const int t_at = w.t_at + (WS == 1 ? 0 : wave), t_end = w.t_end;
    Where here;  // its K ahead of the query: one trip to memory, not two
    if (t_at < t_end) {
        here = table.find(a, w, t_at, table.page_of(a, w, t_at));
        load_k(here, 0, NK);
        load_s(here);
    }

    h8 qh[NS], ql[NS];
    float rowf;
    {
        float v[NS][8];
        int amax = load_q<NS>(row.query(a, w), a.hd, [&](int i) { return ES == MX ? mx_k_dim(i, h, 0) : k_dim(ES, i, h, 0); }, v);
        amax = max(amax, __shfl_xor(amax, 32));
        const float inv = q_scale(amax, a.scale, rowf);
#pragma unroll
        for (int i = 0; i < NS; i++) {
#pragma unroll
            for (int k = 0; k < 8; k++) v[i][k] = v[i][k] * inv;
            split8(v[i], qh[i], ql[i]);
        }
    }

    for (int t = t_at; t < t_end; t += WS) {
        // the next tile (this one again behind the last: the loads in flight
        // are the same at every wait, and none waits for more than its own)
        const int next_t = min(t + WS, t_end - 1), next_page = table.page_of(a, w, next_t);
        if (!SHARED) load_v(here, 0, DT * ES);
        __builtin_amdgcn_sched_barrier(0);

        // ---- scores: register i is position start + 16 h + i ----
        f16v sc = f16v{0.0f};
        if constexpr (ES == MX) {
            const unsigned f[2] = {kf.x >> (8 * h), kf.y >> (8 * h)};
#pragma unroll
            for (int i = 0; i < NK; i++) {
                const float factor = mx_factor(f[i >> 1], 2 * (i & 1));
                const unsigned word[4] = {(unsigned)kraw[i].x, (unsigned)kraw[i].y, (unsigned)kraw[i].z, (unsigned)kraw[i].w};
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const h8 k = mx8(word[c], factor);
                    sc = mfma(k, qh[4 * i + c], sc);
                    sc = mfma(k, ql[4 * i + c], sc);
                }
            }
        } else if (ES == 1) {
#pragma unroll
            for (int i = 0; i < NK; i++) {
                const h8 k0 = codes8(kraw[i].x, kraw[i].y), k1 = codes8(kraw[i].z, kraw[i].w);
                sc = mfma(k0, qh[2 * i % NS], sc);
                sc = mfma(k0, ql[2 * i % NS], sc);
                sc = mfma(k1, qh[(2 * i + 1) % NS], sc);
                sc = mfma(k1, ql[(2 * i + 1) % NS], sc);
            }
        } else if (ES == 2) {
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const h8 k = __builtin_bit_cast(h8, kraw[i % NK]);
                sc = mfma(k, qh[i], sc);
                sc = mfma(k, ql[i], sc);
            }
        } else {
            const float inv = inv_pow2(k_own);
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const float4 x = __builtin_bit_cast(float4, kraw[(2 * i) % NK]), y = __builtin_bit_cast(float4, kraw[(2 * i + 1) % NK]);
                const float f[8] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv, y.x * inv, y.y * inv, y.z * inv, y.w * inv};
                h8 kh, kl;
                split8(f, kh, kl);
                sc = mfma(kh, qh[i], sc);
                sc = mfma(kh, ql[i], sc);
                sc = mfma(kl, qh[i], sc);
                if (SHARED && (i + 1) % (NS / 2) == 0) {
                    __builtin_amdgcn_sched_barrier(0);
                    const int half = i / (NS / 2);
                    load_v(here, half * (NK / 2), (half + 1) * (NK / 2));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        const int start = here.start;
        const bool there = here.there;
        const bool edge = !there || start + TILE - 1 > w.p_lo ||
                          (a.window != INT32_MAX && start + TILE > a.sinks && start < w.p_hi - a.window + 1);
        here = table.find(a, w, next_t, next_page);
        if (!SHARED) load_k(here, 0, NK);
        // (4-bit rows: no faster for it)
        float sk = ES == MX ? ks : copy(ks), sv = ES == MX ? vs : copy(vs);
        load_s(here);
        __builtin_amdgcn_sched_barrier(0);
        only_finite<ES>(sv, sk);
        float st[16];
        each<16>([&](auto i) { st[i] = here_and_now(sc[i.value] * of_lane<i>(sk)); });
        const float v_inv = ES == 4 ? inv_v<ES>(sv) : 0.0f;

        // ---- weights ----
        unsigned vtop;
        if (edge) {
            // positions ahead of the row, behind its window, or in no page:
            // no weight, and no say in the reference
            const int lo = a.window == INT32_MAX ? 0 : row.pos - a.window + 1;
            vtop = 0;
            each<16>([&](auto i) {
                const int at = start + 16 * h + i;
                const bool seen = there & (at <= row.pos) & ((at >= lo) | (at < a.sinks));
                const unsigned bits = __builtin_bit_cast(unsigned, of_lane<i>(sv));  // with every lane at work
                st[i] = seen ? st[i] : -__builtin_inff();
                vtop = max(vtop, seen ? bits : 0u);
            });
        } else {
            vtop = row_max(__builtin_bit_cast(unsigned, sv));
        }
        float top = st[0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, st[i]);
        // the reference bounds weight times V's scale
        const float want = __builtin_fmaf(top, rowf, scale_exp<ES>(vtop));
        if (__any(want > ref + SLACK)) {
            // each row for itself: what it gives does not hang on the rows beside it
            const float all = fmaxf(want, shfl(want, 32));
            const float next = all > ref + SLACK ? all : ref;
            const float f = exp2_(ref - next);
            sum = moved(sum, ref - next);
            ref = next;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[dt][i] = acc[dt][i] * f;
        }
        const float shift = BASE - VScale<ES>::UP - ref;
        h8 ph[2], pl[2];
        {
            float x[16], part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            each<16>([&](auto i) {
                const float p = exp2_(__builtin_fmaf(st[i], rowf, shift));
                part[i & 3] = part[i & 3] + p;
                x[i] = here_and_now(p * of_lane<i>(sv));
            });
            sum = __builtin_fmaf((part[0] + part[1]) + (part[2] + part[3]), SUM_SCALE, sum);
            split8(x, ph[0], pl[0]);
            split8(x + 8, ph[1], pl[1]);
        }

        // ---- O^T += V^T P^T ----
        each<DT * 2>([&](auto k) {
            constexpr int dt = k / 2, c = k % 2;
            if constexpr (ES == MX) {
                constexpr int at = dt / 2 * 2 + c;
                const h8 v = mx8(dt % 2 ? vc[at].y : vc[at].x, 1.0f) * mx_factors(vf[at].x, vf[at].y);
                acc[dt] = mfma(v, ph[c], acc[dt]);
                acc[dt] = mfma(v, pl[c], acc[dt]);
            } else if constexpr (ES == 1) {
                const int4 r = vraw[dt];
                const h8 v = c ? codes8(r.z, r.w) : codes8(r.x, r.y);
                acc[dt] = mfma(v, ph[c], acc[dt]);
                acc[dt] = mfma(v, pl[c], acc[dt]);
            } else if constexpr (ES == 2) {
                const h8 v = __builtin_bit_cast(h8, vraw[dt * ES + c]);
                acc[dt] = mfma(v, ph[c], acc[dt]);
                acc[dt] = mfma(v, pl[c], acc[dt]);
            } else {
                const f4v x = __builtin_bit_cast(f4v, vraw[dt * ES + 2 * c]), y = __builtin_bit_cast(f4v, vraw[dt * ES + 2 * c + 1]);
                // a row that is not finite leaves finite pieces here
                float f[8];
                each<8>([&](auto e) {
                    f[e] = __builtin_amdgcn_fmed3f((e < 4 ? x[e & 3] : y[e & 3]) * of_lane<8 * c + e>(v_inv), -65504.0f, 65504.0f);
                });
                h8 vh, vl;
                split8(f, vh, vl);
                acc[dt] = mfma(vh, ph[c], acc[dt]);
                acc[dt] = mfma(vh, pl[c], acc[dt]);
                acc[dt] = mfma(vl, ph[c], acc[dt]);
                if constexpr (SHARED && (k + 1) % DT == 0) {
                    __builtin_amdgcn_sched_barrier(0);
                    load_k(here, k / DT * (NK / 2), (k / DT + 1) * (NK / 2));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        });
    }
    sum = sum + shfl(sum, 32);
    float o[D / 2];
#pragma unroll
    for (int k = 0; k < D / 2; k++) o[k] = acc[k / 16][k % 16];
    if (WS > 1) {
        join_waves(o, ref, sum, wave, lane, n, h == 0, lds);
        if (wave > 0) return;
    }
    if (n >= w.nr) return;
    put_row<ES>(a, w, row, o, ref, sum, h == 0, D, [&](int c) {
        const int row_of = 8 * (c & 3) + 4 * h;  // of the dim tile, the first of four
        return ES == MX ? mx_v_dim(c >> 2, row_of) : 32 * (c >> 2) + row_of;
    });
}

// ROWS rows, 8 or 16, shared by the workgroup's four waves.
// AHEAD, of 4-bit rows, whose tiles are small: two sets of registers for what is
// loaded, all of the next tile on its way while this one is computed.  For calls
// that give a CU one workgroup or none: there a wave has a SIMD to itself and what
// it waits for is not hidden by another (32 sequences of 16000, 8 KV heads of 128:
// 104 us against 116, 5.6 TB/s; 64 of 4000, two workgroups a CU: 57.7 against 56.4).
template <int ES, int D, int ROWS, bool AHEAD>
__device__ __forceinline__ void few_rows(const Args &a, Job &w, int wave, float *lds) {
    constexpr bool PACKED = ROWS == 8;  // columns 0 .. 7 the high pieces, 8 .. 15 the low ones
    constexpr int NK = ES == MX ? (D + 127) / 128 : D * ES / 64;  // loads of a lane for K, a block of 16 positions
    constexpr int DB = D / 16;          // dim blocks of V
    constexpr int NS = D / 32;          // products over the dims
    constexpr int NV = ES == 4 ? 2 : 1; // loads of a lane for V, a dim block
    const int lane = threadIdx.x & 63, n = lane & 15, z = lane >> 4;
    const bool low = PACKED && n >= 8;
    find_range(a, w);
    const Row row(a, w, w.row0 + min(n & (ROWS - 1), w.nr - 1));

    f4v acc[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) acc[i] = f4v{0.0f};
    float ref = LOW, sum = 0.0f;

    const int P = a.page;
    const unsigned k_lane = ES == MX ? (unsigned)(mx_few_k_lane(D, P, z) + mx_few_slot(n, 0) * 16)
                                     : (unsigned)(few_k_unit(ES, 0, z) * P + few_pos(n, 0)) * 16;
    const unsigned v_lane = ES == MX ? (unsigned)(P * D / 2) + 256 * z + 16 * n
                                     : (unsigned)(P * D * ES) + 16 * n + few_v_off(ES, D, 0, z);
    const unsigned s_lane = scales_at<ES, D>(P) + 4 * (8 * z + (lane & 7));  // scales: position 8 z + lane % 8's
    const Table table(a, w.seq);
    // 4-bit rows: K's factors of the lane's two positions, V's of 8 positions of 64 dims
    const unsigned kf_lane = (unsigned)(P * D) + (unsigned)few_pos(n, 0) * (D / 32);
    const unsigned vf_lane = (unsigned)(P * D + P * D / 32) + (D / 4) * z;
    struct Raw {  // what is loaded of a tile
        Where x;
        int4 vf[ES == MX ? D / 64 : 1];
        u2v kf[2];
        int4 kraw[2 * NK];
        int4 vraw[ES == 1 ? 1 : ES == MX ? D / 64 : DB * NV];
        u2v vraw8[ES == 1 ? DB : 1];
        float ks, vs, k_own[2];
    };
    auto load_s = [&](Raw &raw) {
        const Where &x = raw.x;
        raw.ks = load4(x.r, s_lane, 4 * x.in_page);
        raw.vs = load4(x.r, s_lane, 4 * P + 4 * x.in_page);
    };
    auto load_k = [&](Raw &raw) {
        const Where &x = raw.x;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            if constexpr (ES == MX) {
                if (D == 64) {
                    const u2v half = load8(x.r, k_lane + 256 * b, (unsigned)x.in_page * 16);
                    raw.kraw[b] = make_int4((int)half.x, (int)half.y, 0, 0);
                } else {
#pragma unroll
                    for (int i = 0; i < NK; i++)
                        raw.kraw[b * NK + i] = load16(x.r, k_lane + 256 * b, (unsigned)(4 * i * P + x.in_page) * 16);
                }
                raw.kf[b] = load_kf<D>(x.r, kf_lane + 4 * b * (D / 32), (unsigned)x.in_page * (D / 32));
                continue;
            }
#pragma unroll
            for (int i = 0; i < NK; i++) {
                const int unit = few_k_unit(ES, i, 0);
                raw.kraw[b * NK + i] = load16(x.r, k_lane + 64 * b, (unsigned)(unit * P + x.in_page) * 16);
            }
            if (ES == 4) raw.k_own[b] = dev::bldf(x.r, (unsigned)(2 * P * D * ES) + 4 * (x.in_page + few_pos(n, b)));
        }
    };
    auto load_v = [&](Raw &raw) {
        const Where &x = raw.x;
        if constexpr (ES == MX) {
            const unsigned at = x.v_at(D / 2), f_at = x.v_at(D / 32);
#pragma unroll
            for (int i = 0; i < D / 64; i++) {
                raw.vraw[i] = load16(x.r, v_lane + 1024 * i, at);
                raw.vf[i] = load16(x.r, vf_lane + 16 * i, f_at);
            }
            return;
        }
        const unsigned at = x.v_at(D * ES);
#pragma unroll
        for (int db = 0; db < DB; db++) {
            if (ES == 1) {
                raw.vraw8[db % (ES == 1 ? DB : 1)] = load8(x.r, v_lane + 256 * db, at);
            } else {
#pragma unroll
                for (int c = 0; c < NV; c++)
                    raw.vraw[(db * NV + c) % (ES == 1 ? 1 : DB * NV)] = load16(x.r, v_lane + 256 * db + c * D * 16, at);
            }
        }
    };

    const int t_at = w.t_at + wave, t_end = w.t_end;
    Raw first, second;
    first.k_own[0] = first.k_own[1] = 0.0f;
    int ahead = 0;  // the next tile's page
    if (t_at < t_end) {
        const int page = table.page_of(a, w, t_at);
        if (AHEAD) ahead = table.page_of(a, w, min(t_at + 4, t_end - 1));
        first.x = table.find(a, w, t_at, page);
        load_k(first);
        load_s(first);
        if (AHEAD) load_v(first);
    }

    h8 qh[NS], ql[PACKED ? 1 : NS];
    float rowf;
    {
        float v[NS][8];
        int amax = load_q<NS>(row.query(a, w), a.hd, [&](int i) { return ES == MX ? mx_few_k_dim(D, i, z, 0) : few_k_dim(ES, i, z, 0); }, v);
        amax = max(amax, __shfl_xor(amax, 16));
        amax = max(amax, __shfl_xor(amax, 32));
        const float inv = q_scale(amax, a.scale, rowf);
#pragma unroll
        for (int i = 0; i < NS; i++) {
#pragma unroll
            for (int k = 0; k < 8; k++) v[i][k] = v[i][k] * inv;
            h8 hi, lo;
            split8(v[i], hi, lo);
            qh[i] = low ? lo : hi;
            if (!PACKED) ql[i % (PACKED ? 1 : NS)] = lo;
        }
    }

    // one tile, out of raw, with the next one (this again behind the last) into next
    auto step = [&](Raw &raw, Raw &next, int t) {
        const int next_t = min(t + 4, t_end - 1);
        int next_page = 0;
        if constexpr (AHEAD) {
            next.x = table.find(a, w, next_t, ahead);
            ahead = table.page_of(a, w, min(t + 8, t_end - 1));
            load_k(next);
            load_s(next);
            load_v(next);
        } else {
            next_page = table.page_of(a, w, next_t);
            load_v(raw);
        }
        __builtin_amdgcn_sched_barrier(0);

        // ---- scores: register 4 b + i is position start + 8 z + 4 b + i ----
        f4v sc[2] = {f4v{0.0f}, f4v{0.0f}};
#pragma unroll
        for (int b = 0; b < 2; b++) {
            if constexpr (ES == MX) {
                // the factor of the lane's unit, all of 32 dims
                const unsigned f[2] = {raw.kf[b].x >> (D == 64 ? 8 * (z >> 1) : 8 * z), raw.kf[b].y >> (8 * z)};
#pragma unroll
                for (int i = 0; i < NK; i++) {
                    const int4 r = raw.kraw[b * NK + i];
                    const float factor = mx_factor(f[i & 1], 0);
                    const unsigned word[4] = {(unsigned)r.x, (unsigned)r.y, (unsigned)r.z, (unsigned)r.w};
#pragma unroll
                    for (int c = 0; c < (D == 64 ? 2 : 4); c++) {
                        const h8 k = mx8(word[c], factor);
                        sc[b] = mfma(k, qh[4 * i + c], sc[b]);
                        if (!PACKED) sc[b] = mfma(k, ql[(4 * i + c) % (PACKED ? 1 : NS)], sc[b]);
                    }
                }
            } else if (ES == 1) {
#pragma unroll
                for (int i = 0; i < NK; i++) {
                    const int4 r = raw.kraw[b * NK + i];
                    const h8 k0 = codes8(r.x, r.y), k1 = codes8(r.z, r.w);
                    sc[b] = mfma(k0, qh[2 * i % NS], sc[b]);
                    if (!PACKED) sc[b] = mfma(k0, ql[2 * i % (PACKED ? 1 : NS)], sc[b]);
                    sc[b] = mfma(k1, qh[(2 * i + 1) % NS], sc[b]);
                    if (!PACKED) sc[b] = mfma(k1, ql[(2 * i + 1) % (PACKED ? 1 : NS)], sc[b]);
                }
            } else {
                const float inv = ES == 4 ? inv_pow2(raw.k_own[b]) : 0.0f;
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    h8 kh, kl;
                    if (ES == 2) {
                        kh = __builtin_bit_cast(h8, raw.kraw[(b * NK + i) % (2 * NK)]);
                    } else {
                        const float4 x = __builtin_bit_cast(float4, raw.kraw[(b * NK + 2 * i) % (2 * NK)]);
                        const float4 y = __builtin_bit_cast(float4, raw.kraw[(b * NK + 2 * i + 1) % (2 * NK)]);
                        const float f[8] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv, y.x * inv, y.y * inv, y.z * inv, y.w * inv};
                        split8(f, kh, kl);
                    }
                    sc[b] = mfma(kh, qh[i], sc[b]);
                    if (!PACKED) sc[b] = mfma(kh, ql[i % (PACKED ? 1 : NS)], sc[b]);
                    if (ES == 4) sc[b] = mfma(kl, qh[i], sc[b]);
                }
            }
        }
        const int start = raw.x.start;
        const bool there = raw.x.there;
        const bool edge = !there || start + TILE - 1 > w.p_lo ||
                          (a.window != INT32_MAX && start + TILE > a.sinks && start < w.p_hi - a.window + 1);
        float sk, sv;
        if constexpr (AHEAD) {
            sk = raw.ks;
            sv = raw.vs;
        } else {
            next.x = table.find(a, w, next_t, next_page);
            load_k(next);
            sk = copy(raw.ks);
            sv = copy(raw.vs);
            load_s(next);
        }
        __builtin_amdgcn_sched_barrier(0);
        only_finite<ES>(sv, sk);
        float st[8];
        each<8>([&](auto i) {
            float s = sc[i >> 2][i.value & 3];
            if (PACKED) s = here_and_now(s + other_half(s));
            st[i] = here_and_now(s * of_lane<i>(sk));
        });
        const float v_inv = ES == 4 ? inv_v<ES>(sv) : 0.0f;

        // ---- weights ----
        unsigned vtop;
        if (edge) {
            const int lo = a.window == INT32_MAX ? 0 : row.pos - a.window + 1;
            vtop = 0;
            each<8>([&](auto i) {
                const int at = start + 8 * z + i;
                const bool seen = there & (at <= row.pos) & ((at >= lo) | (at < a.sinks));
                const unsigned bits = __builtin_bit_cast(unsigned, of_lane<i>(sv));  // with every lane at work
                st[i] = seen ? st[i] : -__builtin_inff();
                vtop = max(vtop, seen ? bits : 0u);
            });
        } else {
            vtop = row_max(__builtin_bit_cast(unsigned, sv));
        }
        float top = st[0];
#pragma unroll
        for (int i = 1; i < 8; i++) top = fmaxf(top, st[i]);
        const float want = __builtin_fmaf(top, rowf, scale_exp<ES>(vtop));
        if (__any(want > ref + SLACK)) {
            float all = fmaxf(want, shfl(want, 16));
            all = fmaxf(all, shfl(all, 32));
            const float next = all > ref + SLACK ? all : ref;
            const float f = exp2_(ref - next);
            sum = moved(sum, ref - next);
            ref = next;
#pragma unroll
            for (int db = 0; db < DB; db++) acc[db] = acc[db] * f;
        }
        const float shift = BASE - VScale<ES>::UP - ref;
        h8 ph, pl;
        {
            float x[8], part[2] = {0.0f, 0.0f};
            each<8>([&](auto i) {
                const float p = exp2_(__builtin_fmaf(st[i], rowf, shift));
                part[i & 1] = part[i & 1] + p;
                x[i] = here_and_now(p * of_lane<i>(sv));
            });
            sum = __builtin_fmaf(part[0] + part[1], SUM_SCALE, sum);
            split8(x, ph, pl);
            if (low) ph = pl;
        }

        // ---- O^T += V^T P^T ----
#pragma unroll
        for (int db = 0; db < DB; db++) {
            h8 vh, vl;
            if constexpr (ES == MX) {
                const int4 r = raw.vraw[db / 4], f = raw.vf[db / 4];
                const unsigned word = (unsigned)(db % 4 == 0 ? r.x : db % 4 == 1 ? r.y : db % 4 == 2 ? r.z : r.w);
                vh = mx8(word, 1.0f) * (db % 4 < 2 ? mx_factors((unsigned)f.x, (unsigned)f.y) : mx_factors((unsigned)f.z, (unsigned)f.w));
            } else if (ES == 1) {
                const u2v r = raw.vraw8[db % (ES == 1 ? DB : 1)];
                vh = codes8(r.x, r.y);
            } else if (ES == 2) {
                vh = __builtin_bit_cast(h8, raw.vraw[db % (ES == 1 ? 1 : DB * NV)]);
            } else {
                const f4v x = __builtin_bit_cast(f4v, raw.vraw[(2 * db) % (ES == 1 ? 1 : DB * NV)]);
                const f4v y = __builtin_bit_cast(f4v, raw.vraw[(2 * db + 1) % (ES == 1 ? 1 : DB * NV)]);
                float f[8];
                each<8>([&](auto e) {
                    f[e] = __builtin_amdgcn_fmed3f((e < 4 ? x[e & 3] : y[e & 3]) * of_lane<e>(v_inv), -65504.0f, 65504.0f);
                });
                split8(f, vh, vl);
            }
            acc[db] = mfma(vh, ph, acc[db]);
            if (!PACKED) acc[db] = mfma(vh, pl, acc[db]);
            if (ES == 4) acc[db] = mfma(vl, ph, acc[db]);
        }
    };
    for (int t = t_at; t < t_end; t += 4) {
        step(first, AHEAD ? second : first, t);
        if constexpr (AHEAD) {
            t += 4;
            if (t >= t_end) break;
            step(second, first, t);
        }
    }
    sum = sum + shfl(sum, 16);
    sum = sum + shfl(sum, 32);
    float o[D / 4];
#pragma unroll
    for (int k = 0; k < D / 4; k++) {
        o[k] = acc[k / 4][k % 4];
        if (PACKED) o[k] = o[k] + other_half(o[k]);
    }
    join_waves(o, ref, sum, wave, lane, n, z == 0, lds);
    if (wave > 0 || n >= w.nr) return;
    put_row<ES>(a, w, row, o, ref, sum, z == 0, D, [&](int c) { return 16 * c + 4 * z; });
}

constexpr int FEW = 8;  // rows (x group) of a sequence that few_rows takes beside longer ones

// Waves a SIMD by the registers that the loop holds: many_rows' 32 columns, or
// few_rows' query, sums, K, V and the rest.
constexpr int waves_for(int es, int d, int rows, bool ahead = false) {
    if (rows > 16) return d == 256 ? 1 : 2;
    const int regs = d / 8 * (rows / 8) + d / 4 + (es != MX ? d * es / 4 : ahead ? d / 4 + 40 : d / 8) + 60;
    return regs <= 128 ? 4 : regs <= 172 ? 3 : regs <= 250 ? 2 : 1;
}

// find_seq of up to 64 sequences, those whose rows see the most positions first: where
// there are more workgroups than CUs, the last to start, or to have a CU's memory to
// themselves, are then short ones (64 sequences of 1333 to 4000, 8 KV heads of 128:
// 4-bit rows 47 us against 44, i8 72 against 67).  By levels of what a row sees, found
// bit by bit, and as they come within one: ranking all 64 takes each wave 0.5 us, as
// much as one of many_rows' turns (a prompt of 900 behind 40 sequences of 500 to 4000,
// 32 heads on 8, i8: 62 us, ranked 66.5, as they come 60.5, or 84 with the prompt in
// front).  Few rows go before many that see as much, whose workgroups are more than
// places and fill what the others leave (a prompt of 3000 beside 63 single rows behind
// 3000 to 4000, 12 heads on 2, f16: 98 us, by length 126).  Sequences that see about as
// many stay as they come, as a window makes them (3 chunks and 40 single rows, window
// 512, i8: 30.2 us, and with the single rows in front 36.4).
constexpr int LEVELS = 64;  // that find_longest_first tells apart, of the longest sequence
template <int ROWS, typename F>
__device__ __forceinline__ bool find_longest_first(const Args &a, int tile, F count, int &seq, Seq &s, int &local, int &n) {
    const int lane = threadIdx.x & 63;
    Seq mine{0, 0, 0};
    if (lane < a.b.n_seq) mine.load(a.b, lane);
    const int tiles = count(mine);
    const bool few = ROWS <= 16 || mine.n * a.group <= FEW;
    int seen = min(mine.len, a.window);
    seen += min(mine.len - seen, a.sinks);
    const unsigned long long some = __ballot(tiles > 0);
    const int seen0 = __builtin_amdgcn_readlane(seen, some ? __builtin_ctzll(some) : 0);
    // the level that the tile is in, and how many tiles those above have
    int level = 0, above = 0, mine_level = 0;
    if (__ballot(tiles > 0 && abs(seen - seen0) > seen0 / 8)) {
        mine_level = min((seen >> (a.longest_first - 1)) + (few && a.window == INT32_MAX), LEVELS - 1);
        level = LEVELS - 1;
#pragma unroll
        for (int step = LEVELS / 2; step > 0; step /= 2) {
            const bool over = mine_level > level - step;
            const int sum = a.b.row_start ? __builtin_amdgcn_readlane(dev::wave_scan(over ? tiles : 0), 63)
                                          : __builtin_popcountll(__ballot(over && tiles > 0)) * a.tiles_per;
            if (sum <= tile) {
                level -= step;
                above = sum;
            }
        }
    }
    const int there = mine_level == level ? tiles : 0;
    const int first = above + dev::wave_scan(there) - there;
    const unsigned long long here = __ballot(tile >= first && tile - first < there);
    if (!here) return false;  // past the last tile
    seq = __builtin_ctzll(here);
    n = __builtin_amdgcn_readlane(tiles, seq);
    local = tile - __builtin_amdgcn_readlane(first, seq);
    s = mine.of_lane(seq);
    return true;
}

// A workgroup takes ROWS rows: its waves share 8, 16 or 32, or take 32 of 128
// each; with 32 and 128 a sequence of FEW rows or less goes to few_rows.  Where
// 128 leave 32 or less to a workgroup, its waves share those: one wave alone would
// go over the whole of the positions (a prompt of 3000 beside 63 single tokens
// behind 3000 to 4000, 32 heads on 2 of 128: i8 282 us against 183, f32 517 against
// 390).
template <int ES, int D, int ROWS, bool AHEAD = false>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(waves_for(ES, D, ROWS, AHEAD))))
void attn_kernel(Args a) {
    constexpr int REGS = ROWS > 16 ? D / 2 : D / 4;  // of a lane, that join_waves takes
    __shared__ __attribute__((aligned(16))) float lds[join_floats<REGS>()];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Job w;
    int rest = blockIdx.x;
    w.head = rest % a.n_kv;
    rest /= a.n_kv;
    w.split = rest % a.splits;
    const int tile = rest / a.splits;
    Seq seq;
    int local, tiles;
    auto count = [&](const Seq &q) { return (q.n * a.group + ROWS - 1) / ROWS; };
    if (a.longest_first) {
        if (!find_longest_first<ROWS>(a, tile, count, w.seq, seq, local, tiles)) return;
    } else if (a.b.row_start) {
        if (!find_seq(a.b, tile, count, w.seq, seq, local, tiles)) return;
    } else {
        tiles = a.tiles_per;
        w.seq = tile / tiles;
        local = tile - w.seq * tiles;
        seq.load(a.b, w.seq);
    }
    w.seq_row = seq.row0;
    const int seq_rows = seq.n;
    w.first = seq.len - seq_rows;
    // later rows see more: they go first
    w.row0 = (tiles - 1 - local) * ROWS;
    w.nr = min(seq_rows * a.group - w.row0, ROWS);
    if constexpr (ROWS <= 16) {
        few_rows<ES, D, ROWS, AHEAD>(a, w, wave, lds);
    } else if (seq_rows * a.group <= FEW) {
        few_rows<ES, D, FEW, false>(a, w, wave, lds);
    } else if (ROWS == 32 || w.nr <= 32) {
        many_rows<ES, D, 4>(a, w, wave, lds);
    } else if constexpr (ROWS == 128) {
        w.row0 += 32 * wave;
        w.nr = min(w.nr - 32 * wave, 32);
        if (w.nr > 0) many_rows<ES, D, 1>(a, w, wave, nullptr);
    }
}

// The splits of a row and head, joined at the largest reference, by WM waves:
// one, or four that take every fourth split where there are many and the rows
// few enough for a workgroup each at once (one decoded token of 14 heads, 128
// splits: 10.4 us in all against 20.2; 20 tokens of 32 heads, 10 splits: 18.5
// against 16.9).
template <int D, int WM>
__global__ __launch_bounds__(256) void merge_kernel(Args a) {
    const int n_head = a.n_kv * a.group;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const size_t item = WM == 1 ? (size_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (item >= (size_t)a.b.n_rows * n_head) return;
    const int row = (int)(item / n_head);
    // rows that no sequence has stay as they are
    if (row < first_row(a.b, 0)) return;
    if (a.b.row_start && row >= clampi(a.b.row_start[a.b.n_seq], 0, a.b.n_rows)) return;
    const size_t step = (size_t)a.b.n_rows * n_head;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + item;
    float all = LOW;
    for (int i = lane; i < a.splits; i += 64) all = fmaxf(all, ml[i * step].x);  // of those that saw nothing LOW
    for (int o = 1; o < 64; o <<= 1) all = fmaxf(all, __shfl_xor(all, o));
    constexpr int E = D / 64, AT_ONCE = WM == 1 ? 8 : 16;  // loads in flight
    typedef float fe __attribute__((ext_vector_type(E)));
    fe acc = {};
    float sum = 0.0f;
    for (int base = 0; base < a.splits; base += 64) {
        const int n = min(a.splits - base, 64), i = base + lane;
        const float2 m = i < a.splits ? ml[i * step] : make_float2(LOW, 0.0f);
        const float *from = a.part + ((size_t)base * step + item) * D + E * lane;
        for (int k = WM == 1 ? 0 : wave; k < n; k += WM * AT_ONCE) {
            fe v[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++)
                v[u] = *reinterpret_cast<const fe *>(from + (size_t)min(k + u * WM, n - 1) * step * D);
            // a lane keeps a split's weight; a split that saw nothing has no
            // values, and what was read in their place counts for nothing
            const float f = m.y == 0.0f ? 0.0f : exp2_(m.x - all);
            const unsigned long long has = __ballot(m.y != 0.0f);
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                const int j = k + u * WM;
                if (j < n && (has >> j & 1))
                    acc = acc + v[u] * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), j));
            }
        }
        sum = sum + (m.y == 0.0f ? 0.0f : moved(m.y, m.x - all));
    }
    for (int o = 1; o < 64; o <<= 1) sum = sum + __shfl_xor(sum, o);
    if (WM > 1) {
        __shared__ float s_acc[WM][D];
        *reinterpret_cast<fe *>(&s_acc[wave][E * lane]) = acc;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 1; w < WM; w++) acc = acc + *reinterpret_cast<const fe *>(&s_acc[w][E * lane]);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    float *o = a.out + (size_t)row * a.out_stride + (item - (size_t)row * n_head) * a.hd;
#pragma unroll
    for (int e = 0; e < E; e++)
        if (E * lane + e < a.hd) o[E * lane + e] = acc[e] * a.out_scale * inv;
}

template <int ES, int D>
int launch(const Args &a, const AttnPlan &p, unsigned blocks, size_t items, hipStream_t stream) {
    if (ES == MX && p.ahead) {
        if (p.tile_rows == 8) attn_kernel<ES, D, 8, ES == MX><<<blocks, 256, 0, stream>>>(a);
        else attn_kernel<ES, D, 16, ES == MX><<<blocks, 256, 0, stream>>>(a);
    } else if (p.tile_rows == 8) attn_kernel<ES, D, 8><<<blocks, 256, 0, stream>>>(a);
    else if (p.tile_rows == 16) attn_kernel<ES, D, 16><<<blocks, 256, 0, stream>>>(a);
    else if (p.tile_rows == 32) attn_kernel<ES, D, 32><<<blocks, 256, 0, stream>>>(a);
    else attn_kernel<ES, D, 128><<<blocks, 256, 0, stream>>>(a);
    KH_HIP(hipGetLastError());
    if (p.splits > 1) {
        if (p.join_waves > 1) merge_kernel<D, 4><<<(unsigned)items, 256, 0, stream>>>(a);
        else merge_kernel<D, 1><<<(unsigned)((items + 3) / 4), 256, 0, stream>>>(a);
        KH_HIP(hipGetLastError());
    }
    return KH_OK;
}

template <int ES>
int launch_d(int d, const Args &a, const AttnPlan &p, unsigned blocks, size_t items, hipStream_t s) {
    if (d == 64) return launch<ES, 64>(a, p, blocks, items, s);
    if (d == 128) return launch<ES, 128>(a, p, blocks, items, s);
    return launch<ES, 256>(a, p, blocks, items, s);
}

size_t up_to(size_t n, size_t m) { return (n + m - 1) / m; }
// Waves that join a row's splits (merge_kernel): they take 16 each, one alone 8, a
// trip to memory.
int join_waves(size_t splits, size_t items, size_t cus) { return splits > 8 && items <= cus ? 4 : 1; }

// Splits of few_rows, bound by memory: a workgroup for each CU.  Each gets as
// many tiles as take as long as joining the splits does (a launch, 4 us): 16, or
// fewer large ones; and where all splits together save a wave less turns than
// that, there are none.
size_t few_splits(const kh_paged *kv, size_t blocks, size_t pos_tiles, size_t cus) {
    const size_t least = std::min(std::max(2048 / (kv->es * kv->d), 4), 16);
    const size_t splits = std::min(up_to(cus, blocks), up_to(pos_tiles, least));
    return up_to(pos_tiles, 4) < up_to(up_to(pos_tiles, splits), 4) + least / 4 ? 1 : splits;
}
// The same of 4-bit rows, whose tiles are so small that a CU takes more than one
// workgroup's at a time with a gain: the splits whose busiest CU ends first.  A turn
// of the four waves takes 0.85 us (128 dims), of two workgroups on a CU 1.45, of four
// 2.65; the join as many_splits counts it, and 1.2 for each trip to memory after its
// first (14 heads of 64, 32768 positions: 64 splits 10.6 us, 128 11.1).  Up to a workgroup a CU without splits:
// beyond, the CUs are filled by others' sequences.  Of 32 heads on 8 of 128, up to
// 4000 positions: 5 sequences 14.0 us against 15.7 with few_splits' rule, 12 17.0
// against 22.1, 20 22.4 against 27.5.
size_t mx_few_splits(const kh_paged *kv, size_t blocks, size_t pos_tiles, size_t cus, size_t items) {
    if (blocks > cus) return 1;
    const double dims = (kv->d + 32) / 160.0, join = 8e-6 / 2.4 * (double)items * (kv->d + 2);
    size_t splits = 1;
    double least = 0.0;
    for (size_t s = 1; s <= std::min(4 * cus / blocks, up_to(pos_tiles, 4)); s++) {
        const double each = 0.25 + 0.6 * (double)up_to(blocks * s, cus);
        const double trips = (double)up_to(s, join_waves(s, items, cus) > 1 ? 64 : 8);
        const double us = (double)up_to(up_to(pos_tiles, s), 4) * each * dims + (s > 1 ? 1.3 + 1.2 * trips + join * (double)s : 0.0);
        if (s > 1 && us >= least) continue;
        splits = s;
        least = us;
    }
    return splits;
}
// Splits of many_rows, bound by arithmetic: those whose slowest CU ends first.
// A wave's turn takes 1 us (128 dims, f16 or i8; f32 2), those of two workgroups
// on a CU together half as much again (f32, whose vector instructions are what
// counts, three quarters); a join its launch and the partials' way out and in.
// Never more workgroups than find a place at once.  5000 f16 positions, 32 heads
// on 8 of 128: 20 rows, one split 45 us, 8 or 10 of them 17, 20 of them 20; 200
// rows behind 3000, whose one split has 200 workgroups, 33 us against 37 with
// two; 512 of 14 heads of 64 behind 8000 52 us, with two 49.
size_t many_splits(const kh_paged *kv, size_t blocks, size_t pos_tiles, size_t cus, size_t resident, size_t items) {
    const double turn = (kv->d + 32) / 160.0 * (kv->es == 4 ? 2.0 : 1.0), both = kv->es == 4 ? 1.75 : 1.5;
    const double join = 8e-6 / 2.4 * (double)items * (kv->d + 2);
    size_t splits = 1;
    double least = 0.0;
    for (size_t s = 1; s <= std::min(resident / blocks, pos_tiles); s++) {
        const double us = (double)up_to(up_to(pos_tiles, s), 4) * turn * (blocks * s > cus ? both : 1.0) +
                          (s > 1 ? 2.5 + join * (double)s : 0.0);
        if (s > 1 && us >= least) continue;
        splits = s;
        least = us;
    }
    return splits;
}

}  // namespace

AttnPlan plan_attn(int cu_count, const kh_paged *kv, const Batch &b, int n_head, size_t max_len, int window, int sinks,
                   size_t ws_max) {
    AttnPlan p{};
    const size_t group = (size_t)n_head / kv->n_kv_head;
    auto tiles = [&](size_t rows) {
        return b.row_start ? (size_t)b.n_rows * group / rows + b.n_seq : b.n_seq * up_to((size_t)b.per * group, rows);
    };
    // positions a tile of rows goes over, at most, in tiles
    auto over = [&](size_t rows) {
        size_t span = max_len;
        if (window != INT32_MAX) span = std::min(span, (size_t)window + rows / group + sinks + 2 * TILE);
        return up_to(span, TILE);
    };
    // few_rows where no sequence has more rows than it takes, and for small
    // calls: up to 16 tiles a CU its way in and out is shorter (100 new tokens
    // of 32 heads of 128, f16: 5.9 us against 8.5; 300: 12.0 against 12.6; 100
    // behind 3000, i8: 30 against 26, f32: 60 against 39).  Else 128 rows a
    // workgroup, whose waves read the same K and V at about the same time, where
    // rows enough to fill as many waves as the device holds come together (a
    // 6000-token prompt, f16: 558 us against 621 with 32 and 753 with 16), 32 where
    // they do not (64 sequences of 10 to 20 new tokens, 32 heads on 8 of 128, i8: 174
    // us with 32 and 217 with 128; 300 of them, f16: 284 and 261).  Rows count, not
    // workgroups: one that a sequence's few rows leave nearly empty is no reason.
    // A ragged batch of no more rows than sequences is taken for a decoding one, of a
    // row each (4-bit rows; any batch is done right): 64 of 300 positions, 32 heads
    // on 8 of 128, 11.2 us with row_start and 12.3 as other ragged ones, 20 of 4000
    // 22.8 and 27.9.
    const bool single = b.row_start && kv->es == MX && b.n_rows <= b.n_seq;
    const size_t rows = single ? group : b.row_start ? SIZE_MAX : (size_t)b.per * group, cus = (size_t)cu_count;
    const size_t resident = cus * waves_for(kv->es, kv->d, 32);  // many_rows' workgroups
    const bool small = tiles(16) * kv->n_kv_head * over(16) <= 16 * cus;
    p.tile_rows = rows <= 8                                            ? 8
                  : rows <= 16 || small                              ? 16
                  : (size_t)b.n_rows * n_head / 128 >= resident      ? 128
                                                                     : 32;
    // for experiments, and for tests of each form: any form does any call
    const int form = env_int("KVAD_PAGED_TILE", 0);
    if (form == 8 || form == 16 || form == 32 || form == 128) p.tile_rows = form;
    p.tiles = (int)tiles(p.tile_rows);
    p.per = b.row_start ? 0 : (int)up_to((size_t)b.per * group, p.tile_rows);
    const size_t pos_tiles = over(p.tile_rows);
    const size_t blocks = (single && p.tile_rows <= 16 ? (size_t)b.n_rows * up_to(group, p.tile_rows) : (size_t)p.tiles) * kv->n_kv_head;
    p.splits = 1;
    p.split_tiles = (int)pos_tiles;
    if (p.tile_rows < 128) {
        const int forced = env_int("KVAD_PAGED_SPLITS", 0);
        size_t splits = 1;
        if (forced > 0) splits = std::min((size_t)forced, pos_tiles);
        else if (p.tile_rows <= 16 && kv->es == MX) splits = mx_few_splits(kv, blocks, pos_tiles, cus, (size_t)b.n_rows * n_head);
        else if (p.tile_rows <= 16) splits = few_splits(kv, blocks, pos_tiles, cus);
        else splits = many_splits(kv, blocks, pos_tiles, cus, resident, (size_t)b.n_rows * n_head);
        splits = std::min(splits, (size_t)1024);
        const size_t each = 4 * (size_t)b.n_rows * n_head * (kv->d + 2);
        if (ws_max / each < splits) splits = ws_max / each;
        if (splits > 1) {
            // few_rows waits for memory, and as long for one wave's tile as for
            // four: whole turns of the four waves (1500 positions, f32, 16 heads
            // of 128: 10.7 us against 12.0).  many_rows does not: the splits as
            // even as they can be (100 behind 2000, i8: 23.4 us against 24.1)
            p.split_tiles = (int)up_to(pos_tiles, splits);
            if (p.tile_rows <= 16) p.split_tiles = 4 * (int)up_to(p.split_tiles, 4);
            p.splits = (int)up_to(pos_tiles, p.split_tiles);
            p.ws_bytes = p.splits > 1 ? each * p.splits : 0;
            p.join_waves = join_waves(p.splits, (size_t)b.n_rows * n_head, cus);
        }
    }
    const size_t all = blocks * p.splits;
    p.ahead = kv->es == MX && p.tile_rows <= 16 && all <= cus;
    const int ahead = env_int("KVAD_PAGED_AHEAD", -1);  // for experiments, and for tests of both
    if (ahead >= 0) p.ahead = ahead && kv->es == MX && p.tile_rows <= 16;
    // Not through a window that is short beside the longest: it makes most sequences
    // alike, and finding that out is 0.2 to 0.6 us (64 of 3000 to 12000, 8 KV heads of
    // 128, window 256, i8: 12.0 against 11.7).
    const bool alike = window != INT32_MAX && (size_t)window < max_len / 4;
    p.longest_first = 0;
    if (p.splits == 1 && b.n_seq > 1 && b.n_seq <= 64 && all > cus && !alike) {
        p.longest_first = 1;
        while ((pos_tiles * TILE) >> (p.longest_first - 1) >= (size_t)LEVELS - 1) p.longest_first++;
    }
    return p;
}

int launch_attn(kh_ctx *ctx, const AttnCall &c, const AttnPlan &p) {
    const kh_paged *kv = c.kv;
    Args a{};
    a.pool = c.pool;
    a.b = c.b;
    a.q = c.q;
    a.q_stride = c.q_stride;
    a.out = c.out;
    a.out_stride = c.out_stride;
    const size_t items = (size_t)c.b.n_rows * c.n_head;
    a.part = static_cast<float *>(c.ws);
    a.part_ml = a.part ? a.part + (size_t)p.splits * items * kv->d : nullptr;
    a.block = kv->block;
    a.n_kv = (int)kv->n_kv_head;
    a.group = c.n_head / a.n_kv;
    a.hd = (int)kv->head_dim;
    a.n_pages = (int)kv->n_pages;
    a.page = kv->page;
    a.page_shift = kv->page_shift;
    a.tiles_per = p.per;
    a.splits = p.splits;
    a.split_tiles = p.split_tiles;
    a.longest_first = p.longest_first;  // 1 + the bits that leave LEVELS of what a row sees
    a.window = c.window;
    a.sinks = c.sinks;
    a.scale = c.scale;
    a.out_scale = out_scale(kv->es);
    const unsigned blocks = (unsigned)((size_t)p.tiles * kv->n_kv_head * p.splits);
    if (kv->es == 4) return launch_d<4>(kv->d, a, p, blocks, items, ctx->stream);
    if (kv->es == 2) return launch_d<2>(kv->d, a, p, blocks, items, ctx->stream);
    if (kv->es == 1) return launch_d<1>(kv->d, a, p, blocks, items, ctx->stream);
    return launch_d<MX>(kv->d, a, p, blocks, items, ctx->stream);
}

}  // namespace paged
}  // namespace kh
