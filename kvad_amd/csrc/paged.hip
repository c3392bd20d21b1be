// The paged KV cache: rows quantised as they are written (kh_paged_push),
// gathered and dequantised (kh_paged_read), and the C entries of both and of
// the attention over it (paged_attn.hip).
//
// Both kernels move each byte once and are bound by HBM, or by the launch for
// a few rows (20001 positions of 8 heads of 128 read from i8: 43 us for 206 MB,
// 4.8 TB/s, a large copy's rate; 4500 rows written in 13 us, 3.5 TB/s; 48 single
// rows 3.7 us).  A workgroup takes the 32 positions of one layout tile, one KV
// head, K and V: a cache unit of V runs over positions and a row over dims, so
// the tile is turned in LDS, and both sides go in whole lines: rows of
// head_dim floats, and 16-byte units 32 to 256 in a run.
#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <set>

#include "paged.hpp"

namespace kh {
namespace paged {
namespace {

struct MoveArgs {
    char *pool;
    Batch b;
    float *k, *v;              // rows in (push) or out (read)
    size_t k_stride, v_stride;
    size_t block;
    int n_kv, hd, n_pages, page, page_shift;
};

// A workgroup's tile: sequence, positions p0 .. p0 + 31 (the new rows' run
// may start or end within), row of the run's first position.
struct Tile {
    int p0, first, n, row0;
    char *block;   // null: a page out of range, or positions no table holds
};

__device__ __forceinline__ int tiles_of(int first, int n) { return n ? ((first + n - 1) >> 5) - (first >> 5) + 1 : 0; }

__device__ __forceinline__ bool find_tile(const MoveArgs &a, int tile, int head, Tile &t) {
    int seq, local, count;
    Seq s;
    auto tiles = [](const Seq &q) { return tiles_of(q.len - q.n, q.n); };
    if (!find_seq(a.b, tile, tiles, seq, s, local, count)) return false;
    t.row0 = s.row0;
    t.n = s.n;
    t.first = s.len - s.n;
    t.p0 = ((t.first >> 5) + local) * TILE;
    t.block = nullptr;
    if (t.p0 >= 0 && (t.p0 >> a.page_shift) < a.b.max_pages) {
        const int page = a.b.pages[(size_t)seq * a.b.max_pages + (t.p0 >> a.page_shift)];
        if (page >= 0 && page < a.n_pages) t.block = a.pool + ((size_t)page * a.n_kv + head) * a.block;
    }
    return true;
}

// 2^k, k in -126 .. 127
__device__ __forceinline__ float pow2(int k) { return __builtin_bit_cast(float, (k + 127) << 23); }

// The scale of a row whose largest magnitude has these bits, and its inverse.
// i8: amax / 127, and codes round half away from zero as every 8-bit quantiser
// here does.  f16 and f32: a power of two that brings the row under 2^15, so
// that f16 neither overflows nor loses small rows, and the attention can cut a
// f32 row into two f16 pieces.  A row with a NaN or an infinity: NaN.
template <int ES>
__device__ __forceinline__ float scale_of(int amax_bits, float &inv) {
    if (amax_bits >= 0x7f800000) {
        inv = 0.0f;
        return __builtin_bit_cast(float, NAN_BITS);
    }
    const float amax = __builtin_bit_cast(float, amax_bits);
    if (ES == 1) {
        const float s = amax / 127.0f;
        if (!(s >= 1.17549435e-38f)) return inv = 0.0f;
        inv = 1.0f / s;
        return s;
    }
    int e = 0;
    frexpf(amax, &e);
    const int k = max(e - 15, -126);
    inv = pow2(-k);
    return pow2(k);
}

template <int ES>
__device__ __forceinline__ unsigned code_of(float x, float inv, bool finite) {
    if (ES == 4) return __builtin_bit_cast(unsigned, x);
    const float t = finite ? x * inv : 0.0f;
    if (ES == 2) return __builtin_bit_cast(unsigned short, (_Float16)t);
    const int c = (int)fminf(fmaxf(roundf(t), -127.0f), 127.0f);
    return (unsigned)(c + 128);
}

template <int ES>
__device__ __forceinline__ float value_of(const char *p) {
    if (ES == 4) return *reinterpret_cast<const float *>(p);
    if (ES == 2) return (float)*reinterpret_cast<const _Float16 *>(p);
    return (float)((int)*reinterpret_cast<const uint8_t *>(p) - 128);
}

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any float

template <int ES>
__device__ __forceinline__ unsigned get(const char *p) {
    if (ES == 4) return *reinterpret_cast<const unsigned *>(p);
    if (ES == 2) return *reinterpret_cast<const unsigned short *>(p);
    return *reinterpret_cast<const uint8_t *>(p);
}
template <int ES>
__device__ __forceinline__ void put(char *p, unsigned code) {
    if (ES == 4) *reinterpret_cast<unsigned *>(p) = code;
    if (ES == 2) *reinterpret_cast<unsigned short *>(p) = (unsigned short)code;
    if (ES == 1) *reinterpret_cast<uint8_t *>(p) = (uint8_t)code;
}

// A tile's rows of K and V, in flight together: the way to the tile (the batch's
// arrays, then the page) is a few trips to memory, and both go it once.
template <int ES, int D>
__global__ __launch_bounds__(256) void push_kernel(MoveArgs a) {
    constexpr int U = 16 / ES, ROW = D * ES + 16;  // a row of codes in LDS, off the banks' period
    __shared__ __attribute__((aligned(16))) char s_codes[2][TILE * ROW];
    const int head = blockIdx.x % a.n_kv;
    Tile t;
    if (!find_tile(a, blockIdx.x / a.n_kv, head, t) || !t.block) return;
    const int r = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int row = t.p0 + r - t.first;  // of the sequence's new rows
    const bool mine = row >= 0 && row < t.n;
    const size_t at = (size_t)(t.row0 + (mine ? row : 0));
    const float *x[2] = {a.k + at * a.k_stride + (size_t)head * a.hd, a.v + at * a.v_stride + (size_t)head * a.hd};
    float4u f[2][D / 32];
#pragma unroll
    for (int what = 0; what < 2; what++)
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            const int d = 4 * c + 32 * j;
            f[what][j] = float4u{0.0f, 0.0f, 0.0f, 0.0f};
            if (mine && d < a.hd) f[what][j] = *reinterpret_cast<const float4u *>(x[what] + d);
        }
    const int in_page = t.p0 & (a.page - 1);
#pragma unroll
    for (int what = 0; what < 2; what++) {
        int amax = 0;
#pragma unroll
        for (int j = 0; j < D / 32; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)  // magnitudes compare as their bits do, NaN above infinity
                amax = max(amax, __builtin_bit_cast(int, (float)f[what][j][e]) & 0x7fffffff);
        for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor(amax, o));
        float inv;
        const float scale = scale_of<ES>(amax, inv);
        const bool finite = amax < 0x7f800000;
        if (mine && c == 0) {
            const int off = what ? v_scale_off(ES, D, a.page, in_page + r) : k_scale_off(ES, D, a.page, in_page + r);
            *reinterpret_cast<float *>(t.block + off) = scale;
        }
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            char *p = s_codes[what] + r * ROW + (4 * c + 32 * j) * ES;
            unsigned w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = code_of<ES>(f[what][j][e], inv, finite);
            if (ES == 4) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
            if (ES == 2) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
            if (ES == 1) *reinterpret_cast<unsigned *>(p) = w[0] | w[1] << 8 | w[2] << 16 | w[3] << 24;
        }
    }
    __syncthreads();
    const int lo = max(t.first - t.p0, 0), hi = min(t.first + t.n - t.p0, TILE);  // the tile's new positions
    for (int i = threadIdx.x; i < TILE * D / U; i += 256) {
        const int pos = i & 31, unit = i >> 5;
        if (pos >= lo && pos < hi)
            *reinterpret_cast<int4 *>(t.block + k_off(ES, a.page, in_page + pos, unit * U)) =
                *reinterpret_cast<const int4 *>(s_codes[0] + pos * ROW + unit * 16);
    }
    for (int i = threadIdx.x; i < TILE / U * D; i += 256) {
        const int dim = i % D, p = i / D * U;  // the unit's first position
        char *dst = t.block + v_off(ES, D, a.page, in_page + p, dim);
        const char *from = s_codes[1] + p * ROW + dim * ES;
        if (p >= lo && p + U <= hi) {
            unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < U; e++) w[e * ES / 4] |= get<ES>(from + e * ROW) << (e * ES % 4 * 8);
            *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            // a run that starts or ends within the unit: its own elements
            // alone, the others may be another call's
            for (int e = max(lo - p, 0); e < min(hi - p, U); e++) put<ES>(dst + e * ES, get<ES>(from + e * ROW));
        }
    }
}

template <int ES, int D>
__global__ __launch_bounds__(256) void read_kernel(MoveArgs a) {
    constexpr int U = 16 / ES, ROW = D * ES + 16, N = TILE * D / U / 256 ? TILE * D / U / 256 : 1;
    __shared__ __attribute__((aligned(16))) char s_codes[2][TILE * ROW];
    __shared__ float s_scale[2][TILE];
    const int head = blockIdx.x % a.n_kv;
    Tile t;
    if (!find_tile(a, blockIdx.x / a.n_kv, head, t)) return;
    const int in_page = t.p0 & (a.page - 1);
    if (t.block) {
        int4 u[2][N];
        const bool some = TILE * D / U >= 256 || threadIdx.x < TILE * D / U;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = threadIdx.x + 256 * j, pos = i & 31, unit = i >> 5, dim = i % D, p = i / D * U;
            if (!some) break;
            u[0][j] = *reinterpret_cast<const int4 *>(t.block + k_off(ES, a.page, in_page + pos, unit * U));
            u[1][j] = *reinterpret_cast<const int4 *>(t.block + v_off(ES, D, a.page, in_page + p, dim));
        }
        if (threadIdx.x < 2 * TILE) {
            const int what = threadIdx.x >> 5, pos = threadIdx.x & 31;
            const int off = what ? v_scale_off(ES, D, a.page, in_page + pos) : k_scale_off(ES, D, a.page, in_page + pos);
            s_scale[what][pos] = *reinterpret_cast<const float *>(t.block + off);
        }
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = threadIdx.x + 256 * j, pos = i & 31, unit = i >> 5, dim = i % D, p = i / D * U;
            if (!some) break;
            *reinterpret_cast<int4 *>(s_codes[0] + pos * ROW + unit * 16) = u[0][j];
            const unsigned w[4] = {(unsigned)u[1][j].x, (unsigned)u[1][j].y, (unsigned)u[1][j].z, (unsigned)u[1][j].w};
#pragma unroll
            for (int e = 0; e < U; e++) put<ES>(s_codes[1] + (p + e) * ROW + dim * ES, w[e * ES / 4] >> (e * ES % 4 * 8));
        }
    }
    __syncthreads();
    // a run of 8 lanes takes a row, 32 dims a step
    const int r = threadIdx.x >> 3, c = threadIdx.x & 7, row = t.p0 + r - t.first;
    if (row < 0 || row >= t.n) return;
#pragma unroll
    for (int what = 0; what < 2; what++) {
        float *y = (what ? a.v + (size_t)(t.row0 + row) * a.v_stride : a.k + (size_t)(t.row0 + row) * a.k_stride) +
                   (size_t)head * a.hd;
        const float s = t.block ? s_scale[what][r] : 0.0f;
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            const int d = 4 * c + 32 * j;
            if (d >= a.hd) break;
            float4u f = {0.0f, 0.0f, 0.0f, 0.0f};
            if (t.block) {
                const char *p = s_codes[what] + r * ROW + d * ES;
#pragma unroll
                for (int e = 0; e < 4; e++) f[e] = ES == 4 ? value_of<ES>(p + e * ES) : value_of<ES>(p + e * ES) * s;
            }
            *reinterpret_cast<float4u *>(y + d) = f;
        }
    }
}

template <int ES, int D>
void launch_move(bool push, const MoveArgs &a, unsigned blocks, hipStream_t stream) {
    if (push) push_kernel<ES, D><<<blocks, 256, 0, stream>>>(a);
    else read_kernel<ES, D><<<blocks, 256, 0, stream>>>(a);
}

template <int ES>
void launch_move_d(bool push, int d, const MoveArgs &a, unsigned blocks, hipStream_t stream) {
    if (d == 64) launch_move<ES, 64>(push, a, blocks, stream);
    else if (d == 128) launch_move<ES, 128>(push, a, blocks, stream);
    else launch_move<ES, 256>(push, a, blocks, stream);
}

bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Grid dimensions are counted in threads, in 32 bits.
constexpr size_t MAX_BLOCKS = ((size_t)1 << 32) / 256 - 1;
constexpr size_t MAX_POSITIONS = (size_t)1 << 30;

int refuse(const char *what, const char *why) { return fail(KH_EINVAL, std::string(what) + ": " + why); }

// What can be checked of a batch without reading its arrays.
int check_batch(const kh_paged *kv, size_t layer, const kh_batch *b, const char *what) {
    if (!kv || !b) return refuse(what, "null argument");
    if (layer >= kv->n_layer) return refuse(what, "no such layer");
    if (b->n_rows == 0) return KH_OK;
    if (b->n_seq == 0) return refuse(what, "rows, but no sequences");
    if (!b->len || !b->pages || b->max_pages == 0) return refuse(what, "a batch needs lengths and pages");
    if (!aligned4(b->len) || !aligned4(b->pages) || !aligned4(b->row_start))
        return refuse(what, "the batch's arrays are of 32-bit integers");
    if (!b->row_start && b->n_rows % b->n_seq)
        return refuse(what, "without row_start every sequence has as many rows");
    if (b->n_rows > MAX_POSITIONS || b->n_seq > MAX_POSITIONS || b->max_pages > MAX_POSITIONS / kv->page)
        return refuse(what, "more than 2^30 rows, sequences or positions of a sequence");
    return KH_OK;
}

Batch device_batch(const kh_batch *b) {
    return Batch{b->row_start, b->len, b->pages, (int)b->n_seq, (int)b->n_rows,
                 b->row_start ? 0 : (int)(b->n_rows / b->n_seq), (int)b->max_pages};
}

int move(const kh_paged *kv, size_t layer, const kh_batch *b, float *k, size_t k_stride, float *v, size_t v_stride,
         bool push) {
    const size_t width = kv->n_kv_head * kv->head_dim;
    MoveArgs a;
    a.pool = kv->layers[layer];
    a.b = device_batch(b);
    a.k = k;
    a.v = v;
    a.k_stride = k_stride ? k_stride : width;
    a.v_stride = v_stride ? v_stride : width;
    a.block = kv->block;
    a.n_kv = (int)kv->n_kv_head;
    a.hd = (int)kv->head_dim;
    a.n_pages = (int)kv->n_pages;
    a.page = kv->page;
    a.page_shift = kv->page_shift;
    // n rows lie in at most n / 32 + 2 tiles, and in at most n
    const size_t bound = b->n_rows / TILE + 2 * b->n_seq;
    const size_t tiles = bound < b->n_rows ? bound : b->n_rows;
    const size_t blocks = tiles * kv->n_kv_head;
    if (blocks > MAX_BLOCKS) return fail(KH_EINVAL, "kh_paged: too many rows for one launch");
    hipStream_t s = kv->ctx->stream;
    if (kv->es == 4) launch_move_d<4>(push, kv->d, a, (unsigned)blocks, s);
    else if (kv->es == 2) launch_move_d<2>(push, kv->d, a, (unsigned)blocks, s);
    else launch_move_d<1>(push, kv->d, a, (unsigned)blocks, s);
    KH_HIP(hipGetLastError());
    return KH_OK;
}

int check_move(const kh_paged *kv, size_t layer, const kh_batch *b, const float *k, size_t k_stride, const float *v,
               size_t v_stride, const char *what) {
    if (int rc = check_batch(kv, layer, b, what)) return rc;
    if (b->n_rows && (!k || !v)) return refuse(what, "null argument");
    if (!aligned4(k) || !aligned4(v)) return refuse(what, "rows are of 32-bit floats");
    const size_t width = kv->n_kv_head * kv->head_dim;
    if ((k_stride && k_stride < width) || (v_stride && v_stride < width))
        return refuse(what, "a stride is less than a row");
    return KH_OK;
}

struct Guard {
    std::lock_guard<std::recursive_mutex> lock;
    explicit Guard(kh_ctx *c) : lock(c->mu) { (void)hipSetDevice(c->device); }
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// The arrays of a host batch in the context's staging buffer, from `p` on;
// `dev` is the batch over them.
size_t batch_bytes(const kh_batch *b) {
    return up256(4 * (b->n_seq + 1)) + up256(4 * b->n_seq) + up256(4 * b->n_seq * b->max_pages);
}
int stage_batch(kh_ctx *ctx, const kh_batch *b, char *p, kh_batch *dev) {
    *dev = *b;
    if (b->row_start) {
        KH_HIP(hipMemcpyAsync(p, b->row_start, 4 * (b->n_seq + 1), hipMemcpyHostToDevice, ctx->stream));
        dev->row_start = reinterpret_cast<const int32_t *>(p);
    }
    p += up256(4 * (b->n_seq + 1));
    KH_HIP(hipMemcpyAsync(p, b->len, 4 * b->n_seq, hipMemcpyHostToDevice, ctx->stream));
    dev->len = reinterpret_cast<const int32_t *>(p);
    p += up256(4 * b->n_seq);
    KH_HIP(hipMemcpyAsync(p, b->pages, 4 * b->n_seq * b->max_pages, hipMemcpyHostToDevice, ctx->stream));
    dev->pages = reinterpret_cast<const int32_t *>(p);
    return KH_OK;
}

// What kh_batch_check and the host calls check of a batch's arrays; with `writes`
// the pages that hold new rows are collected, and one that comes twice refused.
int check_tables(const kh_batch *b, size_t page_size, size_t n_pages, bool writes) {
    const size_t cap = b->max_pages * page_size;
    const size_t per = b->row_start ? 0 : b->n_rows / b->n_seq;
    std::set<int32_t> written;
    for (size_t s = 0; s < b->n_seq; s++) {
        const std::string who = "kh_batch_check: sequence " + std::to_string(s);
        size_t rows = per;
        if (b->row_start) {
            const int32_t r0 = b->row_start[s], r1 = b->row_start[s + 1];
            if (r0 < 0 || r1 < r0 || (size_t)r1 > b->n_rows) return fail(KH_EINVAL, who + ": rows out of order");
            rows = (size_t)(r1 - r0);
        }
        if (b->len[s] < 0 || (size_t)b->len[s] > cap)
            return fail(KH_EINVAL, who + ": a length that its pages do not hold");
        const size_t len = (size_t)b->len[s];
        if (rows > len) return fail(KH_EINVAL, who + ": more rows than positions");
        for (size_t i = 0; i * page_size < len; i++) {
            const int32_t p = b->pages[s * b->max_pages + i];
            if (p < 0 || (size_t)p >= n_pages) return fail(KH_EINVAL, who + ": a page out of range");
            if (writes && rows && (i + 1) * page_size > len - rows && !written.insert(p).second)
                return fail(KH_EINVAL, who + ": a page that is written twice");
        }
    }
    return KH_OK;
}

// No exception leaves a C entry.
template <typename F>
int guarded(F f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return KH_ENOMEM;
    } catch (...) {
        return KH_EHIP;
    }
}

}  // namespace
}  // namespace paged
}  // namespace kh

using namespace kh;
using namespace kh::paged;

extern "C" {

int kh_paged_new(kh_ctx *ctx, size_t n_layer, size_t n_kv_head, size_t head_dim, int precision, size_t page_size,
                 size_t n_pages, kh_paged **out) {
    return guarded([&]() -> int {
        if (out) *out = nullptr;
        if (!ctx || !out) return fail(KH_EINVAL, "kh_paged_new: null argument");
        if (precision != KH_F32 && precision != KH_F16 && precision != KH_I8)
            return fail(KH_EINVAL, "kh_paged_new: rows are kept as KH_F32, KH_F16 or KH_I8");
        if (n_layer == 0 || n_layer > 65536 || n_kv_head == 0 || n_kv_head > 65536)
            return fail(KH_EINVAL, "kh_paged_new: needs 1 to 65536 layers and KV heads");
        if (head_dim == 0 || head_dim % 4 || head_dim > 256)
            return fail(KH_EINVAL, "kh_paged_new: head_dim is a multiple of 4 up to 256");
        if (page_size < 32 || page_size > 1024 || (page_size & (page_size - 1)))
            return fail(KH_EINVAL, "kh_paged_new: pages hold 32, 64, ... or 1024 positions");
        if (n_pages == 0 || n_pages > (size_t)INT32_MAX) return fail(KH_EINVAL, "kh_paged_new: needs 1 to 2^31 - 1 pages");
        std::unique_ptr<kh_paged> kv(new kh_paged());
        kv->ctx = ctx;
        kv->n_layer = n_layer;
        kv->n_kv_head = n_kv_head;
        kv->head_dim = head_dim;
        kv->es = precision == KH_F32 ? 4 : precision == KH_F16 ? 2 : 1;
        kv->d = stored_dims((int)head_dim);
        kv->page = (int)page_size;
        while ((1 << kv->page_shift) < kv->page) kv->page_shift++;
        kv->n_pages = n_pages;
        kv->block = block_bytes(kv->es, kv->d, kv->page);
        size_t layer_bytes;
        if (__builtin_mul_overflow(kv->block * n_kv_head, n_pages, &layer_bytes) ||
            __builtin_mul_overflow(layer_bytes, n_layer, &kv->bytes))
            return fail(KH_ENOMEM, "kh_paged_new: more bytes than can be counted");
        Guard g(ctx);
        auto give_back = [&] {
            for (char *p : kv->layers) (void)hipFree(p);
        };
        kv->layers.reserve(n_layer);
        for (size_t l = 0; l < n_layer; l++) {
            void *p = nullptr;
            hipError_t e = hipMalloc(&p, layer_bytes);
            if (e == hipSuccess) {
                kv->layers.push_back(static_cast<char *>(p));
                // slots no row was written to hold zeros, not what was there
                e = hipMemsetAsync(p, 0, layer_bytes, ctx->stream);
            }
            if (e != hipSuccess) {
                (void)hipGetLastError();
                (void)hipStreamSynchronize(ctx->stream);
                give_back();
                return hip_fail(e, "kh_paged_new");
            }
        }
        const hipError_t e = hipStreamSynchronize(ctx->stream);
        if (e != hipSuccess) {
            give_back();
            return hip_fail(e, "kh_paged_new");
        }
        *out = kv.release();
        return KH_OK;
    });
}

int kh_paged_free(kh_paged *kv) {
    if (!kv) return KH_OK;
    {
        Guard g(kv->ctx);
        (void)hipStreamSynchronize(kv->ctx->stream);
        for (char *p : kv->layers) (void)hipFree(p);
        if (kv->scratch.ptr) (void)hipFree(kv->scratch.ptr);
    }
    delete kv;
    return KH_OK;
}

int kh_paged_info(const kh_paged *kv, size_t *page_size, size_t *n_pages, size_t *bytes) {
    if (!kv) return fail(KH_EINVAL, "kh_paged_info: null argument");
    if (page_size) *page_size = (size_t)kv->page;
    if (n_pages) *n_pages = kv->n_pages;
    if (bytes) *bytes = kv->bytes;
    return KH_OK;
}

int kh_batch_check(const kh_batch *b, size_t page_size, size_t n_pages, int writes) {
    return guarded([&]() -> int {
        if (!b) return fail(KH_EINVAL, "kh_batch_check: null argument");
        kh_paged shape;  // check_batch reads the sizes alone
        shape.n_layer = 1;
        if (page_size == 0 || page_size > MAX_POSITIONS) return fail(KH_EINVAL, "kh_batch_check: bad page size");
        shape.page = (int)page_size;
        if (int rc = check_batch(&shape, 0, b, "kh_batch_check")) return rc;
        return b->n_rows ? check_tables(b, page_size, n_pages, writes != 0) : KH_OK;
    });
}

int kh_paged_push_dev(kh_paged *kv, size_t layer, const kh_batch *b, const float *k, size_t k_stride, const float *v,
                      size_t v_stride) {
    return guarded([&]() -> int {
        if (int rc = check_move(kv, layer, b, k, k_stride, v, v_stride, "kh_paged_push_dev")) return rc;
        if (b->n_rows == 0) return KH_OK;
        Guard g(kv->ctx);
        return move(kv, layer, b, const_cast<float *>(k), k_stride, const_cast<float *>(v), v_stride, true);
    });
}

int kh_paged_read_dev(const kh_paged *kv, size_t layer, const kh_batch *b, float *k, size_t k_stride, float *v,
                      size_t v_stride) {
    return guarded([&]() -> int {
        if (int rc = check_move(kv, layer, b, k, k_stride, v, v_stride, "kh_paged_read_dev")) return rc;
        if (b->n_rows == 0) return KH_OK;
        Guard g(kv->ctx);
        return move(kv, layer, b, k, k_stride, v, v_stride, false);
    });
}

int kh_paged_push(kh_paged *kv, size_t layer, const kh_batch *b, const float *k, const float *v) {
    return guarded([&]() -> int {
        if (int rc = check_move(kv, layer, b, k, 0, v, 0, "kh_paged_push")) return rc;
        if (b->n_rows == 0) return KH_OK;
        if (int rc = check_tables(b, (size_t)kv->page, kv->n_pages, true)) return rc;
        Guard g(kv->ctx);
        kh_ctx *ctx = kv->ctx;
        const size_t n = 4 * b->n_rows * kv->n_kv_head * kv->head_dim;
        int rc = ensure(ctx, ctx->io, batch_bytes(b) + 2 * up256(n));
        if (rc) return rc;
        char *p = static_cast<char *>(ctx->io.ptr);
        kh_batch dev;
        if ((rc = stage_batch(ctx, b, p, &dev))) return rc;
        p += batch_bytes(b);
        KH_HIP(hipMemcpyAsync(p, k, n, hipMemcpyHostToDevice, ctx->stream));
        KH_HIP(hipMemcpyAsync(p + up256(n), v, n, hipMemcpyHostToDevice, ctx->stream));
        if ((rc = move(kv, layer, &dev, reinterpret_cast<float *>(p), 0, reinterpret_cast<float *>(p + up256(n)), 0, true)))
            return rc;
        KH_HIP(hipStreamSynchronize(ctx->stream));
        return KH_OK;
    });
}

int kh_paged_read(const kh_paged *kv, size_t layer, const kh_batch *b, float *k, float *v) {
    return guarded([&]() -> int {
        if (int rc = check_move(kv, layer, b, k, 0, v, 0, "kh_paged_read")) return rc;
        if (b->n_rows == 0) return KH_OK;
        if (int rc = check_tables(b, (size_t)kv->page, kv->n_pages, false)) return rc;
        Guard g(kv->ctx);
        kh_ctx *ctx = kv->ctx;
        const size_t n = 4 * b->n_rows * kv->n_kv_head * kv->head_dim;
        int rc = ensure(ctx, ctx->io, batch_bytes(b) + 2 * up256(n));
        if (rc) return rc;
        char *p = static_cast<char *>(ctx->io.ptr);
        kh_batch dev;
        if ((rc = stage_batch(ctx, b, p, &dev))) return rc;
        p += batch_bytes(b);
        // rows behind the last sequence stay as they were
        KH_HIP(hipMemcpyAsync(p, k, n, hipMemcpyHostToDevice, ctx->stream));
        KH_HIP(hipMemcpyAsync(p + up256(n), v, n, hipMemcpyHostToDevice, ctx->stream));
        if ((rc = move(kv, layer, &dev, reinterpret_cast<float *>(p), 0, reinterpret_cast<float *>(p + up256(n)), 0, false)))
            return rc;
        KH_HIP(hipMemcpyAsync(k, p, n, hipMemcpyDeviceToHost, ctx->stream));
        KH_HIP(hipMemcpyAsync(v, p + up256(n), n, hipMemcpyDeviceToHost, ctx->stream));
        KH_HIP(hipStreamSynchronize(ctx->stream));
        return KH_OK;
    });
}

}  // extern "C"

namespace kh {
namespace paged {
namespace {

int check_attend(const kh_paged *kv, size_t layer, const kh_batch *b, size_t n_head, const float *q, size_t q_stride,
                 float scale, const float *out, size_t out_stride, const char *what) {
    if (int rc = check_batch(kv, layer, b, what)) return rc;
    if (n_head == 0 || n_head > 65536 || n_head % kv->n_kv_head)
        return refuse(what, "n_head is a multiple of the cache's KV heads, at most 65536");
    if (!(scale > 0.0f) || !std::isfinite(scale)) return refuse(what, "scale is positive and finite");
    if (b->n_rows == 0) return KH_OK;
    if (!q || !out) return refuse(what, "null argument");
    if (q == out) return refuse(what, "out is not q");
    if (!aligned4(q) || !aligned4(out)) return refuse(what, "rows are of 32-bit floats");
    const size_t width = n_head * kv->head_dim;
    if ((q_stride && q_stride < width) || (out_stride && out_stride < width))
        return refuse(what, "a stride is less than a row");
    if (b->n_rows * (n_head / kv->n_kv_head) > MAX_POSITIONS)
        return refuse(what, "more than 2^30 rows of a KV head");
    return KH_OK;
}

// No position is past 2^30: a window that long hides nothing.
int span(size_t n) { return n >= MAX_POSITIONS ? INT32_MAX : (int)n; }

AttnCall call_of(const kh_paged *kv, size_t layer, const kh_batch *b, size_t n_head, const float *q, size_t q_stride,
                 float scale, size_t window, size_t sinks, float *out, size_t out_stride) {
    AttnCall c{};
    c.kv = kv;
    c.pool = kv->layers[layer];
    c.b = device_batch(b);
    c.n_head = (int)n_head;
    c.q = q;
    c.q_stride = q_stride ? q_stride : n_head * kv->head_dim;
    c.out = out;
    c.out_stride = out_stride ? out_stride : n_head * kv->head_dim;
    c.scale = scale;
    c.window = window ? span(window) : INT32_MAX;
    c.sinks = window ? span(sinks) : 0;
    const size_t held = b->max_pages * (size_t)kv->page;
    c.max_len = b->max_len && b->max_len < held ? b->max_len : held;
    return c;
}

// The plan, its partials in the caller's workspace or the cache's scratch.
int attend(kh_paged *kv, AttnCall &c, void *ws, size_t ws_bytes) {
    kh_ctx *ctx = kv->ctx;
    if (ws && (reinterpret_cast<uintptr_t>(ws) & 15)) return fail(KH_EINVAL, "kh_paged_attend: ws is not 16-byte aligned");
    // the scratch may move before a captured graph runs: there the
    // call takes none and its positions are not split
    const size_t most = ws ? ws_bytes : capturing(ctx->stream) ? 0 : SIZE_MAX;
    AttnPlan p = plan_attn(ctx->cu_count, c.kv, c.b, c.n_head, c.max_len, c.window, c.sinks, most);
    c.ws = ws;
    if (!ws && p.ws_bytes) {
        if (ensure(ctx, kv->scratch, p.ws_bytes) == KH_OK) {
            c.ws = kv->scratch.ptr;
        } else {  // no room: unsplit
            (void)hipGetLastError();
            p = plan_attn(ctx->cu_count, c.kv, c.b, c.n_head, c.max_len, c.window, c.sinks, 0);
        }
    }
    const size_t blocks = (size_t)p.tiles * c.kv->n_kv_head * p.splits;
    if (blocks > MAX_BLOCKS || (p.splits > 1 && (size_t)c.b.n_rows * c.n_head > MAX_BLOCKS))
        return fail(KH_EINVAL, "kh_paged_attend: too many rows for one launch");
    return launch_attn(ctx, c, p);
}

}  // namespace
}  // namespace paged
}  // namespace kh

extern "C" {

int kh_paged_attend_ws(const kh_paged *kv, const kh_batch *b, size_t n_head, size_t window, size_t sinks,
                       size_t *bytes) {
    return guarded([&]() -> int {
        if (!bytes) return fail(KH_EINVAL, "kh_paged_attend_ws: null argument");
        *bytes = 0;
        const float some[2] = {};
        if (int rc = check_attend(kv, 0, b, n_head, some, 0, 1.0f, some + 1, 0, "kh_paged_attend_ws")) return rc;
        if (b->n_rows == 0) return KH_OK;
        const AttnCall c = call_of(kv, 0, b, n_head, nullptr, 0, 1.0f, window, sinks, nullptr, 0);
        *bytes = plan_attn(kv->ctx->cu_count, kv, c.b, c.n_head, c.max_len, c.window, c.sinks, SIZE_MAX).ws_bytes;
        return KH_OK;
    });
}

int kh_paged_attend_dev(kh_paged *kv, size_t layer, const kh_batch *b, size_t n_head, const float *q, size_t q_stride,
                        float scale, size_t window, size_t sinks, float *out, size_t out_stride, void *ws,
                        size_t ws_bytes) {
    return guarded([&]() -> int {
        if (int rc = check_attend(kv, layer, b, n_head, q, q_stride, scale, out, out_stride, "kh_paged_attend_dev"))
            return rc;
        if (b->n_rows == 0) return KH_OK;
        Guard g(kv->ctx);
        AttnCall c = call_of(kv, layer, b, n_head, q, q_stride, scale, window, sinks, out, out_stride);
        return attend(kv, c, ws, ws_bytes);
    });
}

int kh_paged_attend(kh_paged *kv, size_t layer, const kh_batch *b, size_t n_head, const float *q, float scale,
                    size_t window, size_t sinks, float *out) {
    return guarded([&]() -> int {
        if (int rc = check_attend(kv, layer, b, n_head, q, 0, scale, out, 0, "kh_paged_attend")) return rc;
        if (b->n_rows == 0) return KH_OK;
        if (int rc = check_tables(b, (size_t)kv->page, kv->n_pages, false)) return rc;
        Guard g(kv->ctx);
        kh_ctx *ctx = kv->ctx;
        const size_t n = 4 * b->n_rows * n_head * kv->head_dim;
        int rc = ensure(ctx, ctx->io, batch_bytes(b) + 2 * up256(n));
        if (rc) return rc;
        char *p = static_cast<char *>(ctx->io.ptr);
        kh_batch dev;
        if ((rc = stage_batch(ctx, b, p, &dev))) return rc;
        p += batch_bytes(b);
        KH_HIP(hipMemcpyAsync(p, q, n, hipMemcpyHostToDevice, ctx->stream));
        KH_HIP(hipMemcpyAsync(p + up256(n), out, n, hipMemcpyHostToDevice, ctx->stream));
        AttnCall c = call_of(kv, layer, &dev, n_head, reinterpret_cast<float *>(p), 0, scale, window, sinks,
                             reinterpret_cast<float *>(p + up256(n)), 0);
        if ((rc = attend(kv, c, nullptr, 0))) return rc;
        KH_HIP(hipMemcpyAsync(out, p + up256(n), n, hipMemcpyDeviceToHost, ctx->stream));
        KH_HIP(hipStreamSynchronize(ctx->stream));
        return KH_OK;
    });
}

}  // extern "C"
