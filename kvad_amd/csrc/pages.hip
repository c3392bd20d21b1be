// Page tables advanced on the device (kh_pages_*): which sequence's rows come
// where, the pages they need from a stack of free ones, each row's position and
// slot, and pages given back.  No counterpart in the reference, whose caches are
// one array a conversation.
//
// Each call is one launch.  Every workgroup takes the sums over the sequences
// for itself (two numbers each, in LDS: reading them again costs less than a
// second launch), then its share of the rows and pages, each found by bisection.
// The arrays that all of them read, the lengths and the stack's height, are
// written by the last to have read them.  Whether the call can be done is known from
// the sums: all workgroups find the same, and either all do it or none.
//
// What bounds it: trips to memory one behind the other (lengths; a step's row counts,
// which the compiler loads behind the check of the length; of several workgroups the
// count of those that have read, which the first wave of each waits for; pages; what
// is written), and the launch.  Alone on an idle device, mean and least of a trace: 64
// sequences of a decode step 4.5 and 4.2 us, their release 3.6 and 3.3; 137000 new rows
// of 33 sequences, 4300 pages, 6.9 and 5.8, their release 4.7 and 4.4.  The bytes alone
// would take 0.3.
#include <algorithm>

#include "common.hpp"

namespace kh {
namespace pages {
namespace {

constexpr int THREADS = 256, MAX_SEQ = 4096, ROWS = 4;  // rows a thread takes at a time
typedef int i4 __attribute__((ext_vector_type(4), aligned(4)));
typedef long l2 __attribute__((ext_vector_type(2), aligned(8)));
constexpr int LIMIT = 1 << 30;                          // positions and rows are below it

// kh_page_table's status
enum { REASON, REFUSED };
enum { DONE, SHORT, TOO_LONG, BAD_ROWS, BAD_TABLE };

struct Args {
    int32_t *len, *pages, *row_start, *free_pages, *n_free, *status;
    const int32_t *rows;  // of a step; a release's positions to keep
    int32_t *position;
    int64_t *slot;
    int n_seq, max_pages, page_shift, n_pages, n_rows;
    int counter;  // of arrived, where there are several workgroups
};

// Workgroups of a launch that have read what its last one writes: a counter for each
// launch that may run beside others, zero between them.  The library's own, zero from
// the start whatever the caller's arrays hold, and never freed: a captured graph may
// outlive its context.
constexpr int COUNTERS = 1 << 14;
__device__ int arrived[COUNTERS];

__device__ __forceinline__ int pages_for(int positions, int shift) { return (int)(((unsigned)positions + (1u << shift) - 1) >> shift); }
// a sum that stops at LIMIT: of operands up to LIMIT, whatever their order
__device__ __forceinline__ int add(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)LIMIT); }

// What a call makes of a sequence: rows (none for a release) and pages given or
// taken back, from column `first` of its table on.
struct Change {
    int rows, pages, first, bad;
};
template <bool STEP>
__device__ __forceinline__ Change change_of(const Args &a, int len, int arg) {
    const int cap = a.max_pages << a.page_shift;
    Change c{0, 0, 0, DONE};
    if (len < 0 || len > cap) {
        c.bad = BAD_TABLE;
    } else if (STEP) {
        if (arg < 0 || arg > a.n_rows) {
            c.bad = BAD_ROWS;
        } else if (arg > cap - len) {
            c.bad = TOO_LONG;
        } else {
            c.rows = arg;
            c.first = pages_for(len, a.page_shift);
            c.pages = pages_for(len + arg, a.page_shift) - c.first;
        }
    } else if (arg >= 0 && arg < len) {
        c.first = pages_for(arg, a.page_shift);
        c.pages = pages_for(len, a.page_shift) - c.first;
    }
    return c;
}

// Of each sequence the sums before it and its length (of a release: the positions it
// keeps), in LDS; and what all workgroups find alike.
struct Sums {
    int rows[MAX_SEQ], pages[MAX_SEQ], len[MAX_SEQ];
    int wave_rows[THREADS / 64], wave_pages[THREADS / 64], wave_bad[THREADS / 64];
};
struct Totals {
    int rows, pages, bad, n_free;
};
// The sums up to and with each lane's.
template <int CTRL, int ROWS_TO>
__device__ __forceinline__ int below(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS_TO, 0xf, false);
}
__device__ __forceinline__ int scan(int v) {
    v = add(v, below<0x111, 0xf>(v));  // within rows of 16: the lane 1, 2, 4, 8 below
    v = add(v, below<0x112, 0xf>(v));
    v = add(v, below<0x114, 0xf>(v));
    v = add(v, below<0x118, 0xf>(v));
    v = add(v, below<0x142, 0xa>(v));  // the last of a row to the next one, then of two rows
    return add(v, below<0x143, 0xc>(v));
}
// With n_seq <= THREADS a thread has one sequence, and nothing is read twice.
template <bool STEP>
__device__ __forceinline__ Totals sum_up(const Args &a, Sums &s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int each = (a.n_seq + THREADS - 1) / THREADS, from = min((int)threadIdx.x * each, a.n_seq), to = min(from + each, a.n_seq);
    Totals t{0, 0, DONE, *a.n_free};
    int r = 0, p = 0, bad = DONE;
    for (int i = from; i < to; i++) {
        const int len = a.len[i], arg = a.rows[i];
        const Change c = change_of<STEP>(a, len, arg);
        s.rows[i] = r;
        s.pages[i] = p;
        s.len[i] = STEP ? len : arg;
        r = add(r, c.rows);
        p = add(p, c.pages);
        bad = max(bad, c.bad);
    }
    const int r_to = scan(r), p_to = scan(p);
    for (int why = BAD_TABLE; why > DONE; why--)
        if (__ballot(bad == why)) {
            t.bad = why;
            break;
        }
    if (lane == 63) {
        s.wave_rows[wave] = r_to;
        s.wave_pages[wave] = p_to;
        s.wave_bad[wave] = t.bad;
    }
    __syncthreads();
    int r0 = r_to - r, p0 = p_to - p;  // of the wave's lanes before this one, unless a sum has stopped: then nothing is done
    for (int w = 0; w < THREADS / 64; w++) {
        if (w < wave) {
            r0 = add(r0, s.wave_rows[w]);
            p0 = add(p0, s.wave_pages[w]);
        }
        t.rows = add(t.rows, s.wave_rows[w]);
        t.pages = add(t.pages, s.wave_pages[w]);
        t.bad = max(t.bad, s.wave_bad[w]);
    }
    for (int i = from; i < to; i++) {
        s.rows[i] = add(s.rows[i], r0);
        s.pages[i] = add(s.pages[i], p0);
    }
    __syncthreads();
    return t;
}
// The last sequence that starts at i or before it: the one that has item i.
__device__ __forceinline__ int find(const int *starts, int n, int i) {
    int lo = 0, hi = n;  // starts[lo] <= i < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Whether this workgroup is the last of the launch to have read the arrays that are
// then written; asked as soon as it has.  The first wave waits for the answer, whose it
// is (the others get false, and go on to their rows and pages).
__device__ __forceinline__ bool last_one(const Args &a) {
    if (threadIdx.x >= 64) return false;
    if (gridDim.x == 1) return true;
    int last = 0;
    if (threadIdx.x == 0) {
        last = __hip_atomic_fetch_add(&arrived[a.counter], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
        if (last) arrived[a.counter] = 0;
    }
    return __builtin_amdgcn_readfirstlane(last) != 0;
}
__device__ __forceinline__ void report(const Args &a, int reason) {
    a.status[REASON] = reason;
    if (reason != DONE) a.status[REFUSED] = a.status[REFUSED] + 1;
}

__global__ __launch_bounds__(THREADS) void step_kernel(Args a) {
    __shared__ Sums s;
    const Totals t = sum_up<true>(a, s);
    const bool last = last_one(a);
    int reason = t.bad;
    if (t.n_free < 0 || t.n_free > a.n_pages) reason = BAD_TABLE;
    else if (reason == DONE && t.rows > a.n_rows) reason = BAD_ROWS;
    else if (reason == DONE && t.pages > t.n_free) reason = SHORT;
    const int rows = reason == DONE ? t.rows : 0, need = reason == DONE ? t.pages : 0;
    const int at = blockIdx.x * THREADS + threadIdx.x, step = gridDim.x * THREADS;
    const int32_t *top = a.free_pages + t.n_free - 1;
    // pages into the tables, from the stack's top
    for (int i = at; i < need; i += step) {
        const int q = find(s.pages, a.n_seq, i);
        a.pages[(size_t)q * a.max_pages + pages_for(s.len[q], a.page_shift) + (i - s.pages[q])] = top[-i];
    }
    // positions and slots, ROWS rows a thread: of one sequence and one page, or each found by itself
    const int mask = (1 << a.page_shift) - 1;
    auto page_of = [&](int q, int position) {
        const int column = position >> a.page_shift, fresh = column - pages_for(s.len[q], a.page_shift);
        const int page = fresh < 0 ? a.pages[(size_t)q * a.max_pages + column] : top[-s.pages[q] - fresh];
        return page >= 0 && page < a.n_pages ? (int64_t)page << a.page_shift : (int64_t)-1;
    };
    auto end_of = [&](int q) { return q + 1 < a.n_seq ? s.rows[q + 1] : rows; };
    for (int i = at * ROWS; i < a.n_rows; i += step * ROWS) {
        int position[ROWS];
        int64_t slot[ROWS];
        int q = find(s.rows, a.n_seq, min(i, max(rows - 1, 0)));
        const int p0 = s.len[q] + (i - s.rows[q]);
        if (i + ROWS <= end_of(q) && i < rows && (p0 & mask) + ROWS <= mask + 1) {
            const int64_t page = page_of(q, p0);
#pragma unroll
            for (int e = 0; e < ROWS; e++) {
                position[e] = p0 + e;
                slot[e] = page < 0 ? page : page + ((p0 + e) & mask);
            }
        } else {
#pragma unroll
            for (int e = 0; e < ROWS; e++) {
                position[e] = -1;
                slot[e] = -1;
                if (i + e < rows) {
                    while (i + e >= end_of(q)) q++;
                    position[e] = s.len[q] + (i + e - s.rows[q]);
                    slot[e] = page_of(q, position[e]);
                    if (slot[e] >= 0) slot[e] += position[e] & mask;
                }
            }
        }
        if (i + ROWS <= a.n_rows) {
            if (a.position) *reinterpret_cast<i4 *>(a.position + i) = i4{position[0], position[1], position[2], position[3]};
            if (a.slot) {
                reinterpret_cast<l2 *>(a.slot + i)[0] = l2{slot[0], slot[1]};
                reinterpret_cast<l2 *>(a.slot + i)[1] = l2{slot[2], slot[3]};
            }
        } else {
#pragma unroll
            for (int e = 0; e < ROWS; e++) {
                if (a.position && i + e < a.n_rows) a.position[i + e] = position[e];
                if (a.slot && i + e < a.n_rows) a.slot[i + e] = slot[e];
            }
        }
    }
    if (blockIdx.x == 0) {
        for (int q = threadIdx.x; q < a.n_seq; q += THREADS) a.row_start[q] = reason == DONE ? s.rows[q] : 0;
        if (threadIdx.x == 0) a.row_start[a.n_seq] = rows;
    }
    if (!last) return;
    if (reason == DONE)
        for (int q = threadIdx.x; q < a.n_seq; q += 64) a.len[q] = s.len[q] + (end_of(q) - s.rows[q]);
    if (threadIdx.x == 0) {
        if (reason == DONE) *a.n_free = t.n_free - need;
        report(a, reason);
    }
}

__global__ __launch_bounds__(THREADS) void release_kernel(Args a) {
    __shared__ Sums s;
    const Totals t = sum_up<false>(a, s);
    const bool last = last_one(a);
    int reason = t.bad;
    if (t.n_free < 0 || t.n_free > a.n_pages || t.pages > a.n_pages - t.n_free || t.pages >= LIMIT) reason = BAD_TABLE;
    const int back = reason == DONE ? t.pages : 0;
    // the reverse of the order in which a step gives pages
    int32_t *top = a.free_pages + t.n_free + back - 1;
    for (int i = blockIdx.x * THREADS + threadIdx.x; i < back; i += gridDim.x * THREADS) {
        const int q = find(s.pages, a.n_seq, i);
        int32_t *entry = &a.pages[(size_t)q * a.max_pages + pages_for(s.len[q], a.page_shift) + (i - s.pages[q])];
        top[-i] = *entry;
        *entry = -1;
    }
    if (!last) return;
    if (reason == DONE)
        for (int q = threadIdx.x; q < a.n_seq; q += 64)
            if (s.len[q] >= 0) a.len[q] = min(s.len[q], a.len[q]);
    if (threadIdx.x == 0) {
        if (reason == DONE) *a.n_free = t.n_free + back;
        report(a, reason);
    }
}

__global__ __launch_bounds__(THREADS) void init_kernel(Args a) {
    const size_t at = (size_t)blockIdx.x * THREADS + threadIdx.x, step = (size_t)gridDim.x * THREADS;
    for (size_t i = at; i < (size_t)a.n_pages; i += step) a.free_pages[i] = a.n_pages - 1 - (int)i;
    for (size_t i = at; i < (size_t)a.n_seq * a.max_pages; i += step) a.pages[i] = -1;
    for (size_t i = at; i <= (size_t)a.n_seq; i += step) {
        a.row_start[i] = 0;
        if (i < (size_t)a.n_seq) a.len[i] = 0;
    }
    if (at < 4) a.status[at] = 0;
    if (at == 0) *a.n_free = a.n_pages;
}

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int refuse(const char *what, const char *why) { return fail(KH_EINVAL, std::string(what) + ": " + why); }

int check(kh_ctx *ctx, const kh_page_table *t, Args &a, const char *what) {
    if (!ctx || !t) return refuse(what, "null argument");
    if (t->n_seq == 0 || t->n_seq > MAX_SEQ) return refuse(what, "needs 1 to 4096 sequences");
    if (t->page_size < 32 || t->page_size > 1024 || (t->page_size & (t->page_size - 1)))
        return refuse(what, "pages hold 32, 64, ... or 1024 positions");
    if (t->max_pages == 0 || t->max_pages > (size_t)LIMIT / t->page_size)
        return refuse(what, "a sequence holds 1 to 2^30 positions");
    if (t->n_pages == 0 || t->n_pages > (size_t)LIMIT) return refuse(what, "needs 1 to 2^30 pages");
    if (!t->len || !t->pages || !t->row_start || !t->free_pages || !t->n_free || !t->status)
        return refuse(what, "null argument");
    for (const void *p : {t->len, t->pages, t->row_start, t->free_pages, t->n_free, t->status})
        if (!aligned(p, 4)) return refuse(what, "the table's arrays are of 32-bit integers");
    int shift = 0;
    while (((size_t)1 << shift) < t->page_size) shift++;
    a = Args{t->len, t->pages, t->row_start, t->free_pages, t->n_free, t->status, nullptr, nullptr, nullptr,
             (int)t->n_seq, (int)t->max_pages, shift, (int)t->n_pages, 0, 0};
    return KH_OK;
}
unsigned blocks_for(size_t items, unsigned most) {
    return (unsigned)std::min<size_t>(std::max<size_t>((items + THREADS - 1) / THREADS, 1), most);
}

// Which of the counters are taken: up to `used`, but for those given back.
std::mutex counters_mu;
int counters_used = 0, counters_back[COUNTERS], n_back = 0;
int take_counter() {
    std::lock_guard<std::mutex> lock(counters_mu);
    if (n_back) return counters_back[--n_back];
    return counters_used < COUNTERS ? counters_used++ : -1;
}
// The launch's counter, if it needs one: the context's, whose work is on one stream, or
// of a captured call, which may be replayed on any, its own for good.  With none left
// one workgroup does it all.
unsigned count_with(kh_ctx *ctx, unsigned blocks, Args &a) {
    if (blocks == 1) return 1;
    if (capturing(ctx->stream)) {
        a.counter = take_counter();
    } else {
        if (ctx->pages_counter < 0) ctx->pages_counter = take_counter();
        a.counter = ctx->pages_counter;
    }
    return a.counter < 0 ? 1 : blocks;
}

}  // namespace
}  // namespace pages

void free_counter(kh_ctx *ctx) {
    if (ctx->pages_counter < 0) return;
    std::lock_guard<std::mutex> lock(pages::counters_mu);
    pages::counters_back[pages::n_back++] = ctx->pages_counter;
    ctx->pages_counter = -1;
}

}  // namespace kh

using namespace kh;
using namespace kh::pages;

extern "C" {

int kh_pages_init_dev(kh_ctx *ctx, const kh_page_table *t) {
    return guarded([&]() -> int {
        Args a;
        if (int rc = check(ctx, t, a, "kh_pages_init_dev")) return rc;
        std::lock_guard<std::recursive_mutex> lock(ctx->mu);
        (void)hipSetDevice(ctx->device);
        init_kernel<<<blocks_for(std::max(t->n_pages, t->n_seq * t->max_pages), 1024), THREADS, 0, ctx->stream>>>(a);
        KH_HIP(hipGetLastError());
        return KH_OK;
    });
}

int kh_pages_step_dev(kh_ctx *ctx, const kh_page_table *t, const int32_t *rows, size_t n_rows, int32_t *position,
                      int64_t *slot) {
    return guarded([&]() -> int {
        Args a;
        if (int rc = check(ctx, t, a, "kh_pages_step_dev")) return rc;
        if (!rows) return refuse("kh_pages_step_dev", "null argument");
        if (!aligned(rows, 4) || !aligned(position, 4) || !aligned(slot, 8))
            return refuse("kh_pages_step_dev", "rows and positions are 32-bit integers, slots 64-bit ones");
        if (n_rows >= (size_t)LIMIT) return refuse("kh_pages_step_dev", "2^30 rows or more");
        a.rows = rows;
        a.n_rows = (int)n_rows;
        a.position = position;
        a.slot = slot;
        std::lock_guard<std::recursive_mutex> lock(ctx->mu);
        (void)hipSetDevice(ctx->device);
        const unsigned blocks = count_with(ctx, blocks_for(n_rows / ROWS, 2 * (unsigned)ctx->cu_count), a);
        step_kernel<<<blocks, THREADS, 0, ctx->stream>>>(a);
        KH_HIP(hipGetLastError());
        return KH_OK;
    });
}

int kh_pages_release_dev(kh_ctx *ctx, const kh_page_table *t, const int32_t *keep) {
    return guarded([&]() -> int {
        Args a;
        if (int rc = check(ctx, t, a, "kh_pages_release_dev")) return rc;
        if (!keep) return refuse("kh_pages_release_dev", "null argument");
        if (!aligned(keep, 4)) return refuse("kh_pages_release_dev", "positions to keep are 32-bit integers");
        a.rows = keep;
        std::lock_guard<std::recursive_mutex> lock(ctx->mu);
        (void)hipSetDevice(ctx->device);
        const size_t most = std::min(t->n_pages, t->n_seq * t->max_pages);
        const unsigned blocks = count_with(ctx, blocks_for(most / 2, (unsigned)ctx->cu_count), a);
        release_kernel<<<blocks, THREADS, 0, ctx->stream>>>(a);
        KH_HIP(hipGetLastError());
        return KH_OK;
    });
}

}  // extern "C"
