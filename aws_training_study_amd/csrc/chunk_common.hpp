// Chunks of new tokens over the striped paged caches of several sequences:
// which sequence and position a row has, and where a position's page is.
#pragma once

#include "cache_kernels.hpp"
#include "common.hpp"
#include "paging_kernels.hpp"

namespace pcpa {
namespace chunk {

// floor(n / d) for 0 <= n < 2^31 in three instructions: m = floor(2^(31 + l) / d)
// + 1 with 2^l >= d fits 32 bits and is off from 2^(31 + l) / d by at most one,
// which n < 2^31 does not carry over a whole number.
struct Div {
    uint32_t m;
    uint32_t shift;
};
inline Div make_div(uint32_t d) {
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    return Div{(uint32_t)((1ull << (31 + l)) / d + 1), 31 + l};
}
__device__ __forceinline__ uint32_t div(uint32_t n, const Div& d) { return (uint32_t)(((uint64_t)n * d.m) >> d.shift); }

struct Desc {
    const int32_t* lengths;  // [batch]
    const int32_t* starts;   // [batch + 1], or null: `each` rows per sequence
    int32_t batch;
    int32_t num_tokens;
    int32_t each;
    Div div_each;
};

// The rows [first, first + count) of sequence b, within [0, num_tokens)
// whatever `starts` holds.
struct Span {
    int32_t first;
    int32_t count;
};
__device__ __forceinline__ Span span_of(const Desc& c, int b) {
    if (!c.starts) return Span{b * c.each, c.each};
    const int lo = min(max(c.starts[b], 0), c.num_tokens), hi = min(max(c.starts[b + 1], 0), c.num_tokens);
    return Span{lo, max(hi - lo, 0)};
}

// The sequence of row `token` (wave-uniform), or -1 for a row of none; every
// lane of the wave must be active.  The lanes count the sequences that end
// before the row, 64 at a time: a binary search is six dependent loads for 64
// sequences, this is one.
__device__ __forceinline__ int sequence_of(const Desc& c, int token) {
    if (!c.starts) return (int)div((uint32_t)token, c.div_each);
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int base = 0; base < c.batch; base += 64) {
        const bool ended = base + lane < c.batch && c.starts[base + lane + 1] <= token;
        b += __builtin_popcountll(__builtin_amdgcn_ballot_w64(ended));
    }
    if (b >= c.batch) return -1;
    const Span s = span_of(c, b);
    return token >= s.first && token < s.first + s.count ? b : -1;
}

// Over the 64 lanes, by DPP within 16 lanes and by row and half swaps beyond
// (the shuffles go through LDS, ten times the wait).  f has to be commutative;
// every lane gets the result, formed in the same order in every wave.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, true);
}
// ... over LANES (8, 16, 32 or 64) neighbouring lanes.
template <int LANES, class F>
__device__ __forceinline__ uint32_t over_lanes(uint32_t x, F f) {
    x = f(x, dpp<0xB1>(x));   // lane ^ 1
    x = f(x, dpp<0x4E>(x));   // lane ^ 2
    x = f(x, dpp<0x141>(x));  // half rows mirrored: lane 7 - i of 8
    if constexpr (LANES >= 16) x = f(x, dpp<0x140>(x));  // rows mirrored: lane 15 - i of 16
    if constexpr (LANES >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = f(r[0], r[1]);
    }
    if constexpr (LANES >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        x = f(r[0], r[1]);
    }
    return x;
}
template <int LANES>
__device__ __forceinline__ float sum_over_lanes(float x) {
    return __uint_as_float(over_lanes<LANES>(__float_as_uint(x), [](uint32_t u, uint32_t v) {
        return __float_as_uint(__uint_as_float(u) + __uint_as_float(v));
    }));
}
// Inclusive sums over the lanes before and at each lane.
__device__ __forceinline__ int inclusive_sum(int x) {
    const int lane = threadIdx.x & 63;
    // row_shr:1, 2, 4, 8 (lanes without a source add 0)
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    const int r0 = __builtin_amdgcn_readlane(x, 15), r1 = __builtin_amdgcn_readlane(x, 31);
    const int r2 = __builtin_amdgcn_readlane(x, 47);
    return x + (lane >= 48 ? r0 + r1 + r2 : lane >= 32 ? r0 + r1 : lane >= 16 ? r0 : 0);
}

struct Pages {
    const int32_t* table;  // [batch, pcp, max_local_blocks], int32 or int64 as dword pairs
    int32_t table_shift;
    int32_t num_pages;
    int32_t max_local_blocks;
    int32_t block_size;
    int32_t pcp;
    int32_t interleave;
    int32_t num_kv_heads;
    Div div_interleave, div_pcp, div_block, div_stride;  // (stride: pcp * interleave)
    int32_t capacity;      // positions of a sequence's cache: pcp * max_local_blocks * block_size
    int64_t page_stride;   // bytes of a page
    int64_t head_stride;   // bytes of one head's K (or V) of a page
};

// Entry `e` of a table whose first entry is `first` (64-bit: a batch of tables
// may pass 2^31 entries), or -1 where it names no page.
__device__ __forceinline__ int page_at(const Pages& p, int64_t first, int e) {
    const int64_t i = (first + e) << p.table_shift;
    const int page = p.table[i];
    const bool good = (unsigned)page < (unsigned)p.num_pages && !(p.table_shift && p.table[i + 1] != 0);
    return good ? page : -1;
}
__device__ __forceinline__ int64_t table_of(const Pages& p, int b) { return (int64_t)b * p.pcp * p.max_local_blocks; }

// Positions [0, keys) that rank `rank` holds: paging::owned_below for 0 <= keys < 2^31.
__device__ __forceinline__ int owned_of(const Pages& p, int keys, int rank) {
    const int round = (int)div((uint32_t)keys, p.div_stride);
    const int rest = keys - round * (p.pcp * p.interleave);
    return round * p.interleave + min(max(rest - rank * p.interleave, 0), p.interleave);
}

// Page and slot of position `pos` (page -1: none) in the table at `first`.
struct Place {
    int page;
    int slot;
};
__device__ __forceinline__ Place place_of(const Pages& p, int64_t first, int64_t pos) {
    if (pos < 0 || pos >= p.capacity) return Place{-1, 0};
    const uint32_t at = (uint32_t)pos;
    const uint32_t c = div(at, p.div_interleave), round = div(c, p.div_pcp), rank = c - round * p.pcp;
    const uint32_t local = round * p.interleave + (at - c * p.interleave);
    const uint32_t blk = div(local, p.div_block);
    // (the last round of a bucket that is no whole number of rounds)
    if (blk >= (uint32_t)p.max_local_blocks) return Place{-1, 0};
    return Place{page_at(p, first, (int)(rank * p.max_local_blocks + blk)), (int)(local - blk * p.block_size)};
}

// The smallest scale of a row: quotients by it are exact to the rounding of
// cache::div_rn, and a row of zeros needs no case of its own.
constexpr float kScaleFloor = 0x1p-80f;

}  // namespace chunk
}  // namespace pcpa
