// The decode step's glue between the matmuls and the attention:
// tensor::rms_norm (crates/llm/src/tensor.rs:329-333), Rope::apply and
// apply_interleaved (tensor.rs:437-472), swiglu_inplace (tensor.rs:344-350)
// and softmax_inplace (tensor.rs:297-308), on device arrays.
//
// RoPE is bit-exact: it multiplies by the caller's own cos/sin tables (the
// reference hands them out for exactly this, Rope::tables, tensor.rs:377-387)
// with the reference's two products and one sum.  RMSNorm and softmax reduce
// with a fixed tree rather than the reference's serial sum, and SwiGLU and
// softmax use the device's exp, so those agree to rounding.
//
// Beside them, with no counterpart in the reference: rows rotated at positions
// that the device holds (kh_rope_rows_dev, the same products and sums), and the
// end of a block fused with the norms around it (kh_norm_residual_dev).
#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "device.hpp"

namespace kh {
namespace {

// Fixed-order sum over a 256-thread block; every thread gets the total.
__device__ float block_sum(float v, float *s_red) {
    const int tid = threadIdx.x;
    s_red[tid] = v;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if (tid < w) s_red[tid] = s_red[tid] + s_red[tid + w];
        __syncthreads();
    }
    const float r = s_red[0];
    __syncthreads();
    return r;
}

__device__ float block_max(float v, float *s_red) {
    const int tid = threadIdx.x;
    s_red[tid] = v;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if (tid < w) s_red[tid] = fmaxf(s_red[tid], s_red[tid + w]);
        __syncthreads();
    }
    const float r = s_red[0];
    __syncthreads();
    return r;
}

// One row per workgroup: mean of squares, inv = 1 / sqrt(ms + eps),
// out = (x * inv) * w.
__global__ __launch_bounds__(256) void rms_norm_kernel(const float *x, const float *w, int n, float eps, float *out) {
    __shared__ float s_red[256];
    const float *xr = x + (size_t)blockIdx.x * n;
    float *o = out + (size_t)blockIdx.x * n;
    float s = 0.0f;
    for (int i = threadIdx.x; i < n; i += 256) {
        const float v = xr[i];
        const float sq = v * v;
        s = s + sq;
    }
    const float ms = block_sum(s, s_red) / (float)n;
    const float inv = 1.0f / sqrtf(ms + eps);
    for (int i = threadIdx.x; i < n; i += 256) {
        const float t = xr[i] * inv;
        o[i] = t * w[i];
    }
}

// Row r of x holds n_vec vectors of 2 * half at position pos0 + r.
__global__ __launch_bounds__(256) void rope_kernel(const float *cos_t, const float *sin_t, int half, float *x,
                                                  int n_vec, int pos0, int interleaved) {
    const int r = blockIdx.y;
    const size_t base = (size_t)(pos0 + r) * half;
    float *row = x + (size_t)r * n_vec * 2 * half;
    for (int j = blockIdx.x * 256 + threadIdx.x; j < n_vec * half; j += gridDim.x * 256) {
        const int v = j / half, i = j % half;
        float *xv = row + (size_t)v * 2 * half;
        const float c = cos_t[base + i], s = sin_t[base + i];
        const int ia = interleaved ? 2 * i : i, ib = interleaved ? 2 * i + 1 : i + half;
        const float a = xv[ia], b = xv[ib];
        const float ac = a * c, bs = b * s, bc = b * c, as = a * s;
        xv[ia] = ac - bs;
        xv[ib] = bc + as;
    }
}

__global__ __launch_bounds__(256) void swiglu_kernel(float *gate, const float *up, size_t n) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const float g = gate[i];
    const float silu = g / (1.0f + expf(-g));
    gate[i] = silu * up[i];
}

// One row per workgroup: max, exp(x - max), sum, times 1/sum.
__global__ __launch_bounds__(256) void softmax_kernel(float *x, int n) {
    __shared__ float s_red[256];
    float *xr = x + (size_t)blockIdx.x * n;
    float mx = -INFINITY;
    for (int i = threadIdx.x; i < n; i += 256) mx = fmaxf(mx, xr[i]);
    mx = block_max(mx, s_red);
    float s = 0.0f;
    for (int i = threadIdx.x; i < n; i += 256) {
        const float e = expf(xr[i] - mx);
        xr[i] = e;
        s = s + e;
    }
    const float inv = 1.0f / block_sum(s, s_red);
    for (int i = threadIdx.x; i < n; i += 256) xr[i] = xr[i] * inv;
}

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any float

// Rows at positions of their own: row r of x holds n_vec vectors of 2 * half
// first, at position[r]; a row whose position is outside of the tables is left
// alone.  VEC pairs a thread, one trip to memory for the position and one for
// the rest; bound by HBM (5300 rows of 40 heads of 128: 42.6 us for 219 MB, 5.1
// TB/s), or by the launch for a few rows (48 of 16 heads of 64: 2.5 us).
struct RopeRows {
    const float *cos_t, *sin_t, *x;
    const int32_t *position;
    float *out;
    size_t x_stride, out_stride;
    unsigned items;
    int half, max_pos, n_vec;
};
template <int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_rows_kernel(RopeRows a) {
    const unsigned item = blockIdx.x * 256 + threadIdx.x;
    if (item >= a.items) return;
    const unsigned chunks = (unsigned)a.half / VEC, per_row = a.n_vec * chunks, row = item / per_row;
    const unsigned in_row = item - row * per_row, v = in_row / chunks, i = (in_row - v * chunks) * VEC;
    const size_t r = row;
    const int pos = a.position[r];
    if (pos < 0 || pos >= a.max_pos) return;
    const float *x = a.x + r * a.x_stride + (size_t)v * 2 * a.half;
    float *y = a.out + r * a.out_stride + (size_t)v * 2 * a.half;
    const float *ct = a.cos_t + (size_t)pos * a.half + i, *st = a.sin_t + (size_t)pos * a.half + i;
    auto turn = [](float p, float q, float c, float s, float &yp, float &yq) {
        const float pc = p * c, qs = q * s, qc = q * c, ps = p * s;
        yp = pc - qs;
        yq = qc + ps;
    };
    if constexpr (VEC == 4) {
        const float4u c = *reinterpret_cast<const float4u *>(ct), s = *reinterpret_cast<const float4u *>(st);
        const int ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? 2 * i + 4 : i + a.half;
        const float4u p = *reinterpret_cast<const float4u *>(x + ia), q = *reinterpret_cast<const float4u *>(x + ib);
        float f[8], o[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f[e] = p[e];
            f[4 + e] = q[e];
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int ea = INTERLEAVED ? 2 * e : e, eb = INTERLEAVED ? 2 * e + 1 : e + 4;
            turn(f[ea], f[eb], c[e], s[e], o[ea], o[eb]);
        }
        *reinterpret_cast<float4u *>(y + ia) = float4u{o[0], o[1], o[2], o[3]};
        *reinterpret_cast<float4u *>(y + ib) = float4u{o[4], o[5], o[6], o[7]};
    } else {
        const int ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? 2 * i + 1 : i + a.half;
        float p, q;
        turn(x[ia], x[ib], *ct, *st, p, q);
        y[ia] = p;
        y[ib] = q;
    }
}

// The end of a block: t = post ? y / rms(y) * post : y, x' = x + scale * gate * t,
// out = x' / rms(x') * pre.
struct NormResidual {
    const float *x, *y, *post, *gate, *pre;
    float *x_out, *out;
    size_t gate_stride, m;
    float scale, eps;
    int n;
};

// Four floats from i on of a row of n; what is past its end is zero.  FOURS: n is a
// multiple of four, and a load is one instruction that nothing waits for.
template <bool FOURS>
__device__ __forceinline__ float4u load4(const float *p, int i, int n) {
    float4u v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i + 4 <= n) v = *reinterpret_cast<const float4u *>(p + i);
    if (FOURS || i + 4 <= n) return v;
#pragma unroll
    for (int e = 0; e < 3; e++)
        if (i + e < n) v[e] = p[i + e];
    return v;
}
template <bool FOURS>
__device__ __forceinline__ void store4(float *p, int i, int n, float4u v) {
    if (i + 4 <= n) *reinterpret_cast<float4u *>(p + i) = v;
    if (FOURS || i + 4 <= n) return;
#pragma unroll
    for (int e = 0; e < 3; e++)
        if (i + e < n) p[i + e] = v[e];
}
__device__ __forceinline__ float squares(float4u v) {
    const float a = v[0] * v[0], b = v[1] * v[1], c = v[2] * v[2], d = v[3] * v[3];
    return (a + b) + (c + d);
}
// The sum over the W waves of a row, in a fixed order; every lane gets it.
template <int W>
__device__ __forceinline__ float row_sum(float v, float *s_red) {
    v = dev::wave_sum(v);
    if (W == 1) return v;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) s_red[wave] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) s = s + s_red[w];
    return s;
}

// W waves hold a row, V times four floats a lane: everything is read once and
// all loads are in flight together.  With one wave a row a workgroup takes four
// rows and nothing waits at a barrier.  Bound by HBM (2050 rows of 4096, norms on
// both sides and a gate a row: 33.6 us for 168 MB, 5.0 TB/s), or by two sums one
// behind the other (48 rows of 896, one norm: 3.2 us).
template <int W, int V, bool FOURS>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void norm_residual_kernel(NormResidual a) {
    __shared__ float s_red[2][W];
    const size_t r = W == 1 ? (size_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (r >= a.m) return;  // W = 1 alone, by whole waves
    const int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x, n = a.n;
    float4u x[V], y[V], g[V], post[V], pre[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int i = 4 * (lane + 64 * W * j);
        y[j] = load4<FOURS>(a.y + r * n, i, n);
        x[j] = load4<FOURS>(a.x + r * n, i, n);
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int i = 4 * (lane + 64 * W * j);
        if (a.post) post[j] = load4<FOURS>(a.post, i, n);
        if (a.gate) g[j] = load4<FOURS>(a.gate + r * a.gate_stride, i, n);
        if (a.pre) pre[j] = load4<FOURS>(a.pre, i, n);
    }
    float sum = 0.0f;
    if (a.post) {
#pragma unroll
        for (int j = 0; j < V; j++) sum = sum + squares(y[j]);
        const float inv = 1.0f / sqrtf(row_sum<W>(sum, s_red[0]) / (float)n + a.eps);
#pragma unroll
        for (int j = 0; j < V; j++) y[j] = y[j] * inv * post[j];
    }
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j++) {
        const float4u t = a.gate ? y[j] * g[j] : y[j];
        x[j] = x[j] + t * a.scale;
        sum = sum + squares(x[j]);
        store4<FOURS>(a.x_out + r * n, 4 * (lane + 64 * W * j), n, x[j]);
    }
    if (!a.pre) return;
    const float inv = 1.0f / sqrtf(row_sum<W>(sum, s_red[1]) / (float)n + a.eps);
#pragma unroll
    for (int j = 0; j < V; j++) store4<FOURS>(a.out + r * n, 4 * (lane + 64 * W * j), n, x[j] * inv * pre[j]);
}

// Rows that registers do not hold: y is read twice, and x' again where it was
// written, each element by the thread that wrote it.  Bound by memory and by the loops'
// loads, of which a thread has few in flight (512 rows of 16384, norms on both sides and
// a gate a row: 39.2 us for the 168 MB that have to move, 4.3 TB/s; 1025 of 8193, three
// steps of which the last is nearly empty, 45 us, where 8192 are held and take 37; 32 of
// 16384 8.2 us).
__global__ __launch_bounds__(1024) void norm_residual_long_kernel(NormResidual a) {
    __shared__ float s_red[2][16];
    const size_t r = blockIdx.x;
    const int n = a.n;
    const float *x = a.x + r * n, *y = a.y + r * n, *g = a.gate ? a.gate + r * a.gate_stride : nullptr;
    float *xo = a.x_out + r * n;
    float inv = 1.0f, sum = 0.0f;
    if (a.post) {
        for (int i = 4 * threadIdx.x; i < n; i += 4096) sum = sum + squares(load4<false>(y, i, n));
        inv = 1.0f / sqrtf(row_sum<16>(sum, s_red[0]) / (float)n + a.eps);
    }
    sum = 0.0f;
    for (int i = 4 * threadIdx.x; i < n; i += 4096) {
        float4u t = load4<false>(y, i, n);
        if (a.post) t = t * inv * load4<false>(a.post, i, n);
        if (g) t = t * load4<false>(g, i, n);
        t = load4<false>(x, i, n) + t * a.scale;
        sum = sum + squares(t);
        store4<false>(xo, i, n, t);
    }
    if (!a.pre) return;
    inv = 1.0f / sqrtf(row_sum<16>(sum, s_red[1]) / (float)n + a.eps);
    for (int i = 4 * threadIdx.x; i < n; i += 4096) store4<false>(a.out + r * n, i, n, load4<false>(xo, i, n) * inv * load4<false>(a.pre, i, n));
}

// Whether two runs of floats share one; a null one shares none.
bool overlap(const float *a, size_t na, const float *b, size_t nb) {
    if (!a || !b || !na || !nb) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + 4 * nb && y < x + 4 * na;
}
bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Grid dimensions are counted in threads, in 32 bits.
constexpr size_t MAX_THREADS = ((size_t)1 << 32) - 1;

}  // namespace

int launch_swiglu(kh_ctx *ctx, float *gate, const float *up, size_t n) {
    if (n == 0) return KH_OK;
    hipLaunchKernelGGL(swiglu_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, ctx->stream, gate, up, n);
    KH_HIP(hipGetLastError());
    return KH_OK;
}

int launch_rms_norm(kh_ctx *ctx, const float *x, const float *w, size_t m, size_t n, float eps, float *out) {
    if (m == 0 || n == 0) return KH_OK;
    hipLaunchKernelGGL(rms_norm_kernel, dim3((unsigned)m), dim3(256), 0, ctx->stream, x, w, (int)n, eps, out);
    KH_HIP(hipGetLastError());
    return KH_OK;
}

}  // namespace kh

using namespace kh;

extern "C" {

int kh_rms_norm_dev(kh_ctx *ctx, const float *x, const float *w, size_t m, size_t n, float eps, float *out) {
    if (!ctx || !x || !w || !out) return fail(KH_EINVAL, "kh_rms_norm_dev: null argument");
    if (m == 0 || n == 0) return KH_OK;
    if (m > 0x7fffffff || n > 0x7fffffff) return fail(KH_EINVAL, "kh_rms_norm_dev: too large");
    std::lock_guard<std::recursive_mutex> lock(ctx->mu);
    (void)hipSetDevice(ctx->device);
    hipLaunchKernelGGL(rms_norm_kernel, dim3((unsigned)m), dim3(256), 0, ctx->stream, x, w, (int)n, eps, out);
    KH_HIP(hipGetLastError());
    return KH_OK;
}

int kh_rope_dev(kh_ctx *ctx, const float *cos_t, const float *sin_t, size_t half, float *x, size_t m,
                size_t n_vec, size_t pos0, int interleaved) {
    if (!ctx || !cos_t || !sin_t || !x) return fail(KH_EINVAL, "kh_rope_dev: null argument");
    if (m == 0 || n_vec == 0 || half == 0) return KH_OK;
    if (m > 65535 || n_vec * half > 0x7fffffff || pos0 + m > 0x7fffffff)
        return fail(KH_EINVAL, "kh_rope_dev: too large");
    std::lock_guard<std::recursive_mutex> lock(ctx->mu);
    (void)hipSetDevice(ctx->device);
    const size_t work = n_vec * half;
    const unsigned gx = (unsigned)((work + 255) / 256 < 64 ? (work + 255) / 256 : 64);
    hipLaunchKernelGGL(rope_kernel, dim3(gx, (unsigned)m), dim3(256), 0, ctx->stream, cos_t, sin_t, (int)half, x,
                       (int)n_vec, (int)pos0, interleaved);
    KH_HIP(hipGetLastError());
    return KH_OK;
}

int kh_rope_rows_dev(kh_ctx *ctx, const float *cos_t, const float *sin_t, size_t half, size_t max_pos, const float *x,
                     size_t x_stride, const int32_t *position, size_t m, size_t n_vec, int interleaved, float *out,
                     size_t out_stride) {
    return guarded([&]() -> int {
        if (!ctx) return fail(KH_EINVAL, "kh_rope_rows_dev: null argument");
        if (m == 0 || n_vec == 0 || half == 0) return KH_OK;
        if (!cos_t || !sin_t || !x || !position || !out) return fail(KH_EINVAL, "kh_rope_rows_dev: null argument");
        if (!aligned4(cos_t) || !aligned4(sin_t) || !aligned4(x) || !aligned4(position) || !aligned4(out))
            return fail(KH_EINVAL, "kh_rope_rows_dev: arrays are of 32-bit numbers");
        constexpr size_t MOST = (size_t)1 << 30;
        if (m > MOST || n_vec > MOST || half > MOST || 2 * n_vec * half > MOST || max_pos > MOST)
            return fail(KH_EINVAL, "kh_rope_rows_dev: more than 2^30 rows, positions or floats of a row");
        const size_t width = 2 * n_vec * half;
        if ((x_stride && x_stride < width) || (out_stride && out_stride < width))
            return fail(KH_EINVAL, "kh_rope_rows_dev: a stride is less than a row");
        if (x_stride > SIZE_MAX / 8 / m || out_stride > SIZE_MAX / 8 / m)
            return fail(KH_EINVAL, "kh_rope_rows_dev: a stride too large");
        RopeRows a{cos_t, sin_t, x, position, out, x_stride ? x_stride : width, out_stride ? out_stride : width, 0u, (int)half,
                   (int)max_pos, (int)n_vec};
        const bool in_place = x == out && a.x_stride == a.out_stride;
        if (!in_place && overlap(x, (m - 1) * a.x_stride + width, out, (m - 1) * a.out_stride + width))
            return fail(KH_EINVAL, "kh_rope_rows_dev: out is x, or apart from it");
        const size_t rows_out = (m - 1) * a.out_stride + width;
        if (overlap(cos_t, max_pos * half, out, rows_out) || overlap(sin_t, max_pos * half, out, rows_out) ||
            overlap(reinterpret_cast<const float *>(position), m, out, rows_out))
            return fail(KH_EINVAL, "kh_rope_rows_dev: out is apart from the tables and positions");
        const int vec = half % 4 ? 1 : 4;
        const size_t items = m * n_vec * (half / vec);
        a.items = (unsigned)items;
        if (items > MAX_THREADS - 255) return fail(KH_EINVAL, "kh_rope_rows_dev: too many rows for one launch");
        std::lock_guard<std::recursive_mutex> lock(ctx->mu);
        (void)hipSetDevice(ctx->device);
        const unsigned blocks = (unsigned)((items + 255) / 256);
        if (vec == 4) {
            if (interleaved) rope_rows_kernel<4, true><<<blocks, 256, 0, ctx->stream>>>(a);
            else rope_rows_kernel<4, false><<<blocks, 256, 0, ctx->stream>>>(a);
        } else {
            if (interleaved) rope_rows_kernel<1, true><<<blocks, 256, 0, ctx->stream>>>(a);
            else rope_rows_kernel<1, false><<<blocks, 256, 0, ctx->stream>>>(a);
        }
        KH_HIP(hipGetLastError());
        return KH_OK;
    });
}

int kh_norm_residual_dev(kh_ctx *ctx, const float *x, const float *y, const float *post_w, const float *gate,
                         size_t gate_stride, float scale, const float *pre_w, size_t m, size_t n, float eps,
                         float *x_out, float *out) {
    return guarded([&]() -> int {
        if (!ctx) return fail(KH_EINVAL, "kh_norm_residual_dev: null argument");
        if (!(eps >= 0.0f) || !std::isfinite(eps) || !std::isfinite(scale))
            return fail(KH_EINVAL, "kh_norm_residual_dev: eps and scale are finite, eps not negative");
        if (!pre_w != !out) return fail(KH_EINVAL, "kh_norm_residual_dev: out comes with pre_w");
        if (m == 0 || n == 0) return KH_OK;
        if (!x || !y || !x_out) return fail(KH_EINVAL, "kh_norm_residual_dev: null argument");
        for (const void *p : {(const void *)x, (const void *)y, (const void *)post_w, (const void *)gate, (const void *)pre_w,
                              (const void *)x_out, (const void *)out})
            if (!aligned4(p)) return fail(KH_EINVAL, "kh_norm_residual_dev: rows are of 32-bit floats");
        if (m > ((size_t)1 << 30) || n > ((size_t)1 << 30))
            return fail(KH_EINVAL, "kh_norm_residual_dev: more than 2^30 rows or floats of a row");
        if (gate_stride && gate_stride < n) return fail(KH_EINVAL, "kh_norm_residual_dev: a stride is less than a row");
        if (gate_stride > SIZE_MAX / 8 / m) return fail(KH_EINVAL, "kh_norm_residual_dev: a stride too large");
        const size_t all = m * n, gates = (m - 1) * gate_stride + n;
        bool apart = !overlap(x_out, all, out, all);
        for (const float *to : {(const float *)x_out, (const float *)out})
            apart = apart && !overlap(post_w, n, to, all) && !overlap(pre_w, n, to, all) && !overlap(gate, gates, to, all) &&
                    (x == to || !overlap(x, all, to, all)) && (y == to || !overlap(y, all, to, all));
        if (!apart) return fail(KH_EINVAL, "kh_norm_residual_dev: what is written is x or y, or apart from what is read");
        const NormResidual a{x, y, post_w, gate, pre_w, x_out, out, gate_stride, m, scale, eps, (int)n};
        const size_t waves = n <= 1024 ? 1 : n <= 4096 ? 4 : 16, groups = waves == 1 ? (m + 3) / 4 : m;
        if (groups * (waves == 1 ? 256 : 64 * waves) > MAX_THREADS)
            return fail(KH_EINVAL, "kh_norm_residual_dev: too many rows for one launch");
        std::lock_guard<std::recursive_mutex> lock(ctx->mu);
        (void)hipSetDevice(ctx->device);
        const unsigned g = (unsigned)groups;
        hipStream_t s = ctx->stream;
        auto run = [&](auto fours) {
            constexpr bool F = decltype(fours)::value;
            if (n <= 256) norm_residual_kernel<1, 1, F><<<g, 256, 0, s>>>(a);
            else if (n <= 512) norm_residual_kernel<1, 2, F><<<g, 256, 0, s>>>(a);
            else if (n <= 1024) norm_residual_kernel<1, 4, F><<<g, 256, 0, s>>>(a);
            else if (n <= 2048) norm_residual_kernel<4, 2, F><<<g, 256, 0, s>>>(a);
            else if (n <= 4096) norm_residual_kernel<4, 4, F><<<g, 256, 0, s>>>(a);
            else norm_residual_kernel<16, 2, F><<<g, 1024, 0, s>>>(a);
        };
        if (n > 8192) norm_residual_long_kernel<<<g, 1024, 0, s>>>(a);
        else if (n % 4) run(std::false_type{});
        else run(std::true_type{});
        KH_HIP(hipGetLastError());
        return KH_OK;
    });
}

int kh_swiglu_dev(kh_ctx *ctx, float *gate, const float *up, size_t n) {
    if (!ctx || !gate || !up) return fail(KH_EINVAL, "kh_swiglu_dev: null argument");
    if (n == 0) return KH_OK;
    std::lock_guard<std::recursive_mutex> lock(ctx->mu);
    (void)hipSetDevice(ctx->device);
    return launch_swiglu(ctx, gate, up, n);
}

int kh_softmax_dev(kh_ctx *ctx, float *x, size_t m, size_t n) {
    if (!ctx || !x) return fail(KH_EINVAL, "kh_softmax_dev: null argument");
    if (m == 0 || n == 0) return KH_OK;
    if (m > 0x7fffffff || n > 0x7fffffff) return fail(KH_EINVAL, "kh_softmax_dev: too large");
    std::lock_guard<std::recursive_mutex> lock(ctx->mu);
    (void)hipSetDevice(ctx->device);
    hipLaunchKernelGGL(softmax_kernel, dim3((unsigned)m), dim3(256), 0, ctx->stream, x, (int)n);
    KH_HIP(hipGetLastError());
    return KH_OK;
}

}  // extern "C"
