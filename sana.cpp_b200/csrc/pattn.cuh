// What the paged-attention kernels share: the packing of rows, the key range of a row tile, the
// checks of device data, and the plan of a launch.
//
// Rows. The new tokens of a sequence and the query heads that read one cache head are packed into
// the rows of one tile, row = token * G + head: a cached key is then read once for the whole
// group, and a single token fills G rows.
//
// Keys. A row at position p sees j <= p and, with a window W, of those j > p - W or j < sinks. A
// tile of rows therefore walks the sinks' keys (if the window has moved past them) and then the
// keys from the first row's window to the last row's position, BN at a time; only tiles that some
// row sees in part are masked element by element.
//
// Splits. The key tiles of a row tile are shared out over blocks, `split_tiles` each; what a block
// of several finds is left in the workspace as (sum p v, max, sum p) and joined by
// paged_combine_kernel in a fixed order.
#pragma once

#include <cuda.h>

#include "encoder.h"

namespace sana {
namespace pattn {

struct Args {
    PagedAttention p;
    int G;            // query heads per cache head
    PageDivisor g_div;  // division by it
    int row_tiles;    // of BM packed rows, per sequence
    int BM, BN;
    int splits, split_tiles;
    int align;        // the keys of a window start at a multiple of it (a power of two)
    float* part;      // [splits][rows][q_heads][D]
    float2* ml;       // [splits][rows][q_heads]: (max, sum)
};

__device__ __forceinline__ Sequence sequence(const PagedAttention& p, int s, bool report) {
    return batch_sequence(p.batch, s, report, p.bad);
}

// The key tiles of packed rows [rr0, rr1) of a sequence.
struct KeyTiles {
    int pmin, pmax;   // positions of the first and last row
    int sink_end;     // keys [0, sink_end) apart from the rest (0: none)
    int lo, hi;       // keys [lo, hi)
    int n_sink, n;    // tiles of the sinks, of both
};
__host__ __device__ __forceinline__ KeyTiles key_tiles(int past, int n_new, int G, int rr0, int rr1, int window, int sinks,
                                                       int BN, int align) {
    KeyTiles k;
    const int last = n_new * G < rr1 ? n_new * G : rr1;
    k.pmin = past + rr0 / G;
    k.pmax = past + (last - 1) / G;
    k.hi = k.pmax + 1;
    k.lo = 0;
    k.sink_end = 0;
    if (window > 0) {
        const int lo = (k.pmin - window + 1) & -align;
        const int s = sinks < k.hi ? sinks : k.hi;
        if (lo > s) {
            k.lo = lo;
            k.sink_end = s;
        }
    }
    k.n_sink = (k.sink_end + BN - 1) / BN;
    k.n = k.n_sink + (k.hi - k.lo + BN - 1) / BN;
    return k;
}
__device__ __forceinline__ void key_range(const KeyTiles& k, int i, int BN, int& start, int& end) {
    if (i < k.n_sink) {
        start = i * BN;
        end = min(k.sink_end, start + BN);
    } else {
        start = k.lo + (i - k.n_sink) * BN;
        end = min(k.hi, start + BN);
    }
}
// Whether every row of the tile sees every key of [start, end).
__device__ __forceinline__ bool all_seen(const KeyTiles& k, int start, int end, int window, int sinks) {
    return end - 1 <= k.pmin && (window <= 0 || end <= sinks || start > k.pmax - window);
}
__device__ __forceinline__ bool seen(int j, int pos, int window, int sinks) {
    return j <= pos && (window <= 0 || j > pos - window || j < sinks);
}

// The soft cap of the tensor-core kernels, cap tanh(x / cap) log2(e) of a product x, in = 2 scale log2(e) / cap: by tanh z =
// 1 - 2 / (1 + e^2z) from the hardware exponential and reciprocal. Its error, whatever the score, moves a probability by at
// most cap 2^-21 of itself: up to kCheapCap 2^-11, an eighth of the rounding to bf16. Larger caps take another form.
constexpr float kCheapCap = 1024.f;
__device__ __forceinline__ float soft_cap_log2(float x, float in, float cap_log2) {
    return fmaf(-2.f * cap_log2, rcp_approx(1.f + ex2_approx(x * in)), cap_log2);
}

PageDivisor page_divisor(int d);
__device__ __forceinline__ int head_group(const Args& a, int rr) {  // the token of packed row rr: rr / G
    return static_cast<int>((__umulhi(static_cast<uint32_t>(rr), a.g_div.magic) + static_cast<uint32_t>(rr)) >> a.g_div.shift);
}
__device__ __forceinline__ int page_slot(const PagedAttention& p, int j) {  // j / page_size, 0 <= j < 2^30
    return static_cast<int>((__umulhi(static_cast<uint32_t>(j), p.page_div.magic) + static_cast<uint32_t>(j)) >> p.page_div.shift);
}

// Element offset of key j of sequence s in the cache (head 0), -1 if its page is not in the pool.
__device__ __forceinline__ long long key_offset(const PagedAttention& p, int s, int j) {
    const int slot = page_slot(p, j);
    const int page = slot < p.batch.table_width ? p.batch.table[s * p.batch.table_stride + slot] : -1;
    if (page < 0 || page >= p.cache.pages) {
        record_bad(p.bad, kBadPage);
        return -1;
    }
    return page * p.cache.page_stride + static_cast<long long>(j - slot * p.cache.page_size) * p.cache.token_stride;
}

// Whether the page of any of the keys [lo, hi) is not in the pool; the block's threads share out the pages.
__device__ __forceinline__ bool any_bad_page(const PagedAttention& p, int s, int lo, int hi) {
    bool bad = false;
    for (int j = page_slot(p, lo) + static_cast<int>(threadIdx.x), last = page_slot(p, hi - 1); j <= last;
         j += static_cast<int>(blockDim.x))
        bad = key_offset(p, s, min(max(j * p.cache.page_size, lo), hi - 1)) < 0 || bad;
    return bad;
}
// The same for the key tiles [t0, t0 + n) of a row tile.
__device__ __forceinline__ bool any_bad_page(const PagedAttention& p, int s, const KeyTiles& kt, int t0, int n, int BN) {
    bool bad = false;
    int lo, hi, unused;
    if (t0 < kt.n_sink) {
        key_range(kt, t0, BN, lo, unused);
        key_range(kt, min(kt.n_sink, t0 + n) - 1, BN, unused, hi);
        bad = any_bad_page(p, s, lo, hi);
    }
    if (t0 + n > kt.n_sink) {
        key_range(kt, max(t0, kt.n_sink), BN, lo, unused);
        key_range(kt, t0 + n - 1, BN, unused, hi);
        bad = any_bad_page(p, s, lo, hi) || bad;
    }
    return bad;
}

// Keys that one tensor copy (TMA) brings of tiles of `keys` keys: a page, or a key tile where pages are multiples of
// tiles; 0 where a page ends inside a tile or the pool's strides do not fit a tensor map.
int copy_box(const PagedCache& c, int keys);
// The pool's k or v as a tensor [pages][kv_heads][page_size][D] of boxes of `box` tokens of one head x 64 channels, in
// the 128-byte swizzle.
CUtensorMap pool_map(const PagedCache& c, const void* base, int box);

// The same of all channels at once, [pages][kv_heads][slabs][page_size][64] (head sizes that are multiples
// of 64).
CUtensorMap pool_map_slabs(const PagedCache& c, const void* base, int box);

// pattn_tc.cu: packed rows and keys of a block's tile, and the launch.
int tc_rows(int D);
int tc_keys();
void launch_tc(const Args& a, dim3 grid, cudaStream_t st);

}  // namespace pattn
}  // namespace sana
