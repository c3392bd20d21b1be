// Internal declarations of the paged KV cache (paged.hip, paged_attn.hip).
#pragma once

#include "common.hpp"
#include "device.hpp"
#include "paged_layout.hpp"

// A pool of pages per layer (kvad_hip.h); the pages' owners are the caller's tables.
struct kh_paged {
    kh_ctx *ctx = nullptr;
    size_t n_layer = 0, n_kv_head = 0, head_dim = 0;
    int es = 0, d = 0;              // bytes an element (MX: half a byte), dims a row as it is kept
    int page = 0, page_shift = 0;
    size_t n_pages = 0;
    size_t block = 0;               // bytes of one page of one head
    size_t bytes = 0;               // of all layers
    std::vector<char *> layers;
    // Partials of split attention calls.  Its own, not the context's: no captured
    // graph names it, so it may grow whatever was captured.
    kh::Workspace scratch;
};

namespace kh {
namespace paged {

// A batch as the kernels take it: device arrays, sizes checked by the host.
struct Batch {
    const int32_t *row_start;  // or null: `per` rows each
    const int32_t *len;
    const int32_t *pages;
    int n_seq, n_rows, per, max_pages;
};

constexpr int NAN_BITS = 0x7fc00000;

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// First row of sequence i, and of the one behind it; within the rows whatever
// the table says.
__device__ __forceinline__ int first_row(const Batch &b, int i) {
    return b.row_start ? clampi(b.row_start[i], 0, b.n_rows) : i * b.per;
}
__device__ __forceinline__ int rows_of(const Batch &b, int i, int first) {
    return b.row_start ? clampi(b.row_start[i + 1], first, b.n_rows) - first : b.per;
}

// A sequence's rows and length, as a lane of find_seq holds them.
struct Seq {
    int row0, n, len;
    __device__ __forceinline__ void load(const Batch &b, int i) {
        row0 = first_row(b, i);
        n = rows_of(b, i, row0);
        len = max(b.len[i], 0);
    }
    __device__ __forceinline__ Seq of_lane(int l) const {
        return Seq{__builtin_amdgcn_readlane(row0, l), __builtin_amdgcn_readlane(n, l), __builtin_amdgcn_readlane(len, l)};
    }
};

// Which sequence the tile'th tile of the batch belongs to, a sequence s having
// count(s) of them: a wave takes the running sum of 64 counts at a time.  False
// past the last tile.  `tile` is the same in every lane; so are the results:
// the sequence's number, the tile's among its own, how many those are.
template <typename F>
__device__ __forceinline__ bool find_seq(const Batch &b, int tile, F count, int &seq, Seq &s, int &local, int &n) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < b.n_seq; base += 64) {
        Seq mine{0, 0, 0};
        if (base + lane < b.n_seq) mine.load(b, base + lane);
        const int c = count(mine);
        const int sum = dev::wave_scan(c);
        const int all = __builtin_amdgcn_readlane(sum, 63);
        if (tile < all) {
            const int l = __builtin_ctzll(__ballot(sum > tile));
            n = __builtin_amdgcn_readlane(c, l);
            local = tile - (__builtin_amdgcn_readlane(sum, l) - n);
            seq = base + l;
            s = mine.of_lane(l);
            return true;
        }
        tile -= all;
    }
    return false;
}

// An attention call over a layer (paged_attn.hip).
struct AttnCall {
    const kh_paged *kv;
    const char *pool;
    Batch b;
    int n_head;
    const float *q;
    size_t q_stride;
    float *out;
    size_t out_stride;
    float scale;
    int window, sinks;   // window INT32_MAX: none
    size_t max_len;      // positions of the longest sequence, for the split alone
    void *ws;            // partials
};
// How a call is cut up, from its sizes alone.
struct AttnPlan {
    int tile_rows;     // rows x group of a workgroup: 8, 16, 32 or 128
    int tiles;         // row tiles, or a bound on them where rows are ragged
    int per;           // tiles of each sequence where rows are not
    int splits;        // of the positions, over workgroups
    int split_tiles;   // 32-position tiles a split
    int join_waves;    // that join a row's splits
    bool ahead;        // of 4-bit rows: few_rows with two tiles' registers
    int longest_first;   // workgroups go to the sequences by what their rows see (0: as they come)
    size_t ws_bytes;   // of partials
};
AttnPlan plan_attn(int cu_count, const kh_paged *kv, const Batch &b, int n_head, size_t max_len, int window, int sinks,
                   size_t ws_max);
int launch_attn(kh_ctx *ctx, const AttnCall &c, const AttnPlan &p);

}  // namespace paged
}  // namespace kh
