// Causal attention of new tokens over the paged caches of their sequences.
#pragma once

#include "cache_kernels.hpp"
#include "chunk_common.hpp"
#include "tile_kernel.hpp"

namespace pcpa {
namespace chunk {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

constexpr int kTileKeys = 64;  // keys of a walk's tile: a whole number of them to a page

// The maximum before any score: finite, as keys may be hidden from a row before
// any that is not (2^(-inf - kNoScore) is 0), and no more than any finite score.
constexpr float kNoScore = -0x1.fffffep127f;

// What the merge needs to find a sequence's partial results: written by the
// sequence's first workgroup.
struct SequencePlan {
    int32_t first_item;  // of all its (range, row tile from the last on, KV head) items, KV head fastest
    int32_t ranges;      // its walk is cut into; 1: results are final
    int32_t tiles;       // row tiles
};

struct AttendArgs {
    Desc chunk;
    Pages pages;
    const uint8_t* q;
    const uint8_t* pool;
    const float* token_scales;
    uint8_t* out;
    float* lse;
    int32_t num_q_heads;
    int32_t group;
    int32_t rows_log2;     // of a workgroup's row tile
    Div div_group, div_heads;
    int32_t max_items;     // the launch's workgroups
    int32_t slots;         // workgroups that the GPU holds at once
    int32_t min_range;     // tiles a range has at least
    int32_t whole;         // tiles of a walk that is not cut
    float score_scale;     // softmax_scale * k_scale * log2(e)
    float v_scale;
    float* part_o;         // [max_items, rows, D] fp32 normalised outputs of ranges
    v2f* part_ml;          // [max_items, rows] their maxima and sums (one log of both would round
                           // the sum away where scores are large)
    SequencePlan* plans;   // [batch]
};

// One workgroup's share: row tile `tile` of sequence b and KV head `head`, the
// walk's tiles [begin, end).
struct Item {
    int b, head, tile, range;
    int begin, end;
    SequencePlan plan;
    Span span;
    int length;  // of the cache, as given
};

// Tiles of the walk over positions [0, keys): rank by rank within each 64 local
// positions, so that with chunks of 64 they follow the positions.  Tile i is
// local positions 64 (i / pcp) .. of rank i % pcp; a few may be empty.
__device__ __forceinline__ int walk_tiles(const Pages& p, int keys) {
    return p.pcp * ((owned_of(p, keys, 0) + kTileKeys - 1) / kTileKeys);
}

// The row of q and out that row `r` of the item's sequence and KV head is.
__device__ __forceinline__ int64_t row_index(const AttendArgs& a, const Item& it, int r) {
    const int token = (int)div((uint32_t)r, a.div_group);
    return (int64_t)(it.span.first + token) * a.num_q_heads + it.head * a.group + (r - token * a.group);
}

// The place of item `at` among the items of its sequence; false for none.
__device__ __forceinline__ bool place_item(const AttendArgs& a, int at, int walk, Item& it) {
    const int heads = a.pages.num_kv_heads;
    if (at < 0) return false;
    const int rest = (int)div((uint32_t)at, a.div_heads);
    it.head = at - rest * heads;
    it.range = it.plan.tiles == 1 ? rest : rest / it.plan.tiles;
    // the last rows, which see the most, first
    it.tile = it.plan.tiles - 1 - (rest - it.range * it.plan.tiles);
    // (starts that decrease may overflow the sums: no such item)
    if (it.range >= it.plan.ranges) return false;
    // (the first ranges a tile longer than the rest, if they are not equal)
    it.begin = 0;
    it.end = walk;
    if (it.plan.ranges > 1) {
        const int whole = walk / it.plan.ranges, more = walk - whole * it.plan.ranges;
        it.begin = it.range * whole + min(it.range, more);
        it.end = it.begin + whole + (it.range < more);
    }
    return true;
}

// The item of workgroup `index`; false when there is none.  Every wave of the
// workgroup finds it by itself (a launch of its own for this took longer), a
// sequence to a lane: first the work of the whole chunk, which gives the tiles a
// range should have so that all ranges fill the GPU once, then the sequence that
// the index falls into.  The first 64 KEPT sequences stay in registers, their
// loads in flight together: 256 where there are few rows and more sequences than
// 64 (200 sequences of up to 256 tokens: 17.2 -> 14.4 us; 64 of them 7.9 -> 9.2),
// else 64 (with many rows the registers have other uses: seven prompts, D 256,
// e4m3: 672 -> 702 us with 256).  Sequences of as many rows each whose walks are not cut need no
// sums (4096 workgroups of one tile each: 300 -> 268 us).
template <int KEPT>
__device__ __forceinline__ bool find_item(const AttendArgs& a, int index, int rows_per_tile, Item& it) {
    const int lane = threadIdx.x & 63, heads = a.pages.num_kv_heads, batch = a.chunk.batch;
    const bool cut = a.part_o != nullptr;
    auto tiles_of = [&](int count) { return (int)(((uint32_t)(count * a.group) + rows_per_tile - 1) / rows_per_tile); };
    // (a sequence whose rows see nothing still has an item, for their zeros)
    auto walk_of = [&](int length) { return max(walk_tiles(a.pages, min(max(length, 0), a.pages.capacity)), 1); };
    if (!cut && !a.chunk.starts) {
        const int tiles = tiles_of(a.chunk.each), per = tiles * heads;
        it.b = index / per;
        if (it.b >= batch) return false;
        it.span = span_of(a.chunk, it.b);
        it.length = a.chunk.lengths[it.b];
        it.plan = SequencePlan{it.b * per, 1, tiles};
        return place_item(a, index - it.b * per, walk_of(it.length), it);
    }
    struct Lane {
        Span span;
        int length;
    };
    auto load = [&](int base) {
        Lane x{{0, 0}, 0};
        if (base + lane < batch) x = Lane{span_of(a.chunk, base + lane), a.chunk.lengths[base + lane]};
        return x;
    };
    Lane kept[KEPT];
    int tiles[KEPT], walk[KEPT];
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
        kept[k] = Lane{{0, 0}, 0};
        if (64 * k < batch) kept[k] = load(64 * k);
    }
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
        tiles[k] = tiles_of(kept[k].span.count);
        walk[k] = walk_of(kept[k].length);
    }
    int range = 1 << 30;  // (beyond any walk)
    if (cut) {
        // f(tiles, walk) of every sequence
        auto over_all = [&](auto f) {
#pragma unroll
            for (int k = 0; k < KEPT; ++k)
                if (64 * k < batch) f(tiles[k], walk[k]);
            for (int base = 64 * KEPT; base < batch; base += 64) {
                const Lane x = load(base);
                f(tiles_of(x.span.count), walk_of(x.length));
            }
        };
        // (sums in 32-bit floats: only the range's length comes of them)
        const float slots = (float)a.slots;
        float work = 0.f, least = 0.f;
        over_all([&](int t, int w) {
            work += (float)t * (float)w;
            least += (float)t;
        });
        const float share = ceilf(sum_over_lanes<64>(work) * heads / slots);
        float length_of = fmaxf(fminf(share, 0x1p30f), (float)a.min_range);
        // Each sequence's last range is a shorter one, so that ranges of the fair
        // share are more than the GPU holds at once, and the few left over would run
        // after all others: longer ranges, until all run together.  (64 sequences
        // of 512 to 8192 tokens, 2 heads at D 256, e4m3: 83.2 -> 74.6 us.)
        if (sum_over_lanes<64>(least) * heads < slots)
            for (int tries = 0; tries < 6; ++tries) {
                // (2^-10: no more than w / length_of where that is a whole number)
                const float inv = 1.f / length_of;
                float count = 0.f;
                over_all([&](int t, int w) {
                    count += (float)t * (w <= a.whole ? 1.f : ceilf(fmaf((float)w, inv, -0x1p-10f)));
                });
                count = sum_over_lanes<64>(count) * heads;
                if (count <= slots) break;
                length_of = fminf(ceilf(fmaxf(length_of + 1.f, length_of * (count / slots))), 0x1p30f);
            }
        range = __builtin_amdgcn_readfirstlane((int)length_of);
    }
    int before = 0;
    bool found = false;
    auto look = [&](int base, const Lane& x, int t, int w) {
        const int ranges = w <= a.whole ? 1 : (w + range - 1) / range, items = t * heads * ranges, incl = inclusive_sum(items);
        const uint64_t past = __builtin_amdgcn_ballot_w64(before + incl > index);
        if (past) {
            const int src = __builtin_ctzll(past);
            auto of = [&](int y) { return __builtin_amdgcn_readlane(y, src); };
            it.b = base + src;
            it.span = Span{of(x.span.first), of(x.span.count)};
            it.length = of(x.length);
            it.plan = SequencePlan{before + of(incl) - of(items), of(ranges), of(t)};
            found = place_item(a, index - it.plan.first_item, of(w), it);
            return true;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
        return false;
    };
#pragma unroll
    for (int k = 0; k < KEPT; ++k)
        if (64 * k < batch && look(64 * k, kept[k], tiles[k], walk[k])) return found;
    for (int base = 64 * KEPT; base < batch; base += 64) {
        const Lane x = load(base);
        if (look(base, x, tiles_of(x.span.count), walk_of(x.length))) return found;
    }
    return false;
}

__device__ __forceinline__ float quarters_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarters_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// A table entry as it is read ahead (the two dwords of an int64 one; entry 0 in
// the place of none), and its page, or -1.
typedef const __attribute__((address_space(4))) int32_t* const_i32_ptr;
struct TableEntry {
    int lo, hi;
};
__device__ __forceinline__ TableEntry entry_of(const_i32_ptr table, const Pages& p, int entry) {
    const int64_t i = (int64_t)max(entry, 0) << p.table_shift;
    return TableEntry{table[i], table[i + p.table_shift]};
}
__device__ __forceinline__ int page_of(const Pages& p, const TableEntry& e) {
    const bool good = (unsigned)e.lo < (unsigned)p.num_pages && !(p.table_shift && e.hi != 0);
    return good ? e.lo : -1;
}

// ---- few rows ------------------------------------------------------------------
//
// For up to 32 rows per (sequence, KV head) - one token of a GQA group, or a few
// - or few in all, the work is reading the cache once: every wave streams its own keys, no wave
// waits for another.  A step of a wave is KEYS keys:
//   * S^T = K Q^T by 16x16x32 MFMAs.  K goes from the pages straight into the A
//     operand's registers: lane 16 g + r holds 16 bytes of the key in row r, four
//     lanes 64 bytes in a row, and Q's registers hold the same values of d in the
//     same order (the order of a sum of products is free).  Row r of tile t is key
//     8 (r / 4) + 4 t + r % 4 of 32, so that the scores of lane group g, (t, i),
//     are keys 8 g + 4 t + i: the B operand of the next product as they stand.
//   * the running maximum m, sum l and O^T of each row stay in registers; m is
//     raised only when a step exceeds it by 2^8 (as in the tile kernel).
//   * O^T += V^T P^T, P as two bf16 values, the upper half of its bits and the rest
//     (2^-16 off): rounded to one, it was as far off as the rounding of the result
//     (0.0024 of it instead of 0.0017), and these MFMAs are not what bounds.  V goes into the wave's own LDS by DMA, 16-byte chunks
//     swizzled by key so that the transposing reads find every bank once.
// The next step's K (registers) and V (LDS) load while this one is computed: 16
// KB (e4m3) or 32 KB (bf16) in flight per wave, 128 KB per CU.  The waves' results
// meet in LDS at the end.
// HBM bound once walks are long: 64 sequences of 4544 tokens, 2 heads at D 256,
// e4m3 with token scales, 57 us with the merge, 5.2 TB/s (5.5 without scales); of
// 512 to 8192 tokens 67 us, as the longest range is 21 tiles where 18 would be
// equal shares, and a tile of a range is half a step of its four waves.
template <int D, bool FP8, int RT>
struct FewShape {
    static constexpr int ROW = D * (FP8 ? 1 : 2);    // bytes of a key's row
    static constexpr int KG = D == 256 ? 1 : 2;      // 32-key groups of a step
    static constexpr int KEYS = 32 * KG;
    static constexpr int SUB = kTileKeys / KEYS;     // steps of a tile
    static constexpr int KC = ROW / 64;              // 16-byte loads of a K row per lane
    static constexpr int QK = D / 32;                // k-steps of the score MFMA
    static constexpr int DT = D / 16;
    static constexpr int V_BYTES = KEYS * ROW;
    static constexpr int V_BLOCKS = V_BYTES / 1024;  // DMA instructions of a step
    static constexpr int CH = ROW / 16;              // 16-byte chunks of a row
    // eight waves where their registers (256 each) and LDS hold it
    static constexpr int WAVES = D == 64 && !FP8 ? 8 : 4;
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int O_ROW = D + 4;              // floats: 16 rows then start in all banks
    static constexpr int V_LDS = WAVES * 2 * V_BYTES;
    static constexpr int O_LDS = WAVES * 16 * O_ROW * 4;
    static constexpr int LDS = V_LDS > O_LDS ? V_LDS : O_LDS;
    static constexpr int PER_CU = FP8 && !(D == 256 && RT == 2) ? 2 : 1;  // workgroups that fit
    static constexpr int ROWS = 16 * RT;
    static constexpr int WHOLE = ROW > 256 ? 4 : 8;  // tiles of a walk that is not cut
};

// Chunk swizzle of V's rows in LDS.  A transposing read of 8-bit values takes
// 16 keys x 16 bytes at once, one of 16-bit values 8 keys (0-3 and 8-11, or 4
// more) x 32 bytes: the keys of either then lie in different 16-byte (32-byte)
// parts of the 256 bytes that the banks span.
template <int ROW, bool FP8>
__device__ __forceinline__ constexpr int few_swizzle(int key) {
    constexpr int CH = ROW / 16;
    if constexpr (FP8) return (key / (256 / ROW)) & (CH < 16 ? CH - 1 : 15);
    if constexpr (CH == 8) return 2 * (((key >> 1) & 1) | ((key >> 2) & 2));
    return 2 * ((key & 3) | ((key >> 1) & 4));
}

template <class S>
struct FewStep {
    int n;        // keys of it that some row may see
    int rank;
    int local;    // the rank's local position of its first key
    int page;     // -1: no step
    int slot;
    int u;
    int entry;    // of the table
};

template <class S>
struct FewLoads {
    v4i k[2 * S::KG * S::KC];             // free once the scores are there
    v4f ks[2 * S::KG], vs[2 * S::KG];     // the keys' scales
};

template <int D, bool FP8, bool SCALED, int RT>
__global__ void __launch_bounds__((FewShape<D, FP8, RT>::THREADS),
                                  (FewShape<D, FP8, RT>::PER_CU * FewShape<D, FP8, RT>::WAVES / 4))
    attend_few_kernel(AttendArgs a) {
    using S = FewShape<D, FP8, RT>;
    constexpr int ROW = S::ROW, KG = S::KG, KC = S::KC, DT = S::DT, QK = S::QK;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::LDS];
    __shared__ float wave_ml[S::WAVES][16][2];

    Item it;
    if (!(a.chunk.batch <= 64 ? find_item<1>(a, blockIdx.x, S::ROWS, it) : find_item<4>(a, blockIdx.x, S::ROWS, it)))
        return;
    if (it.head == 0 && it.tile == 0 && it.range == 0 && threadIdx.x == 0 && a.plans) a.plans[it.b] = it.plan;

    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rows = it.span.count * a.group;

    // ---- this lane's rows: Q operand and the positions they see ---------------
    v8bf qop[RT][QK];
    int seen[RT];  // positions [0, seen) of the sequence
    const int row0 = it.tile * S::ROWS;
    // the tile's last row sees the most
    const int last = min(row0 + S::ROWS, rows) - 1;
    auto sees = [&](int row) {
        const int64_t np = (int64_t)it.length - it.span.count + (int)div((uint32_t)row, a.div_group) + 1;
        return (int)min(max(np, (int64_t)0), (int64_t)a.pages.capacity);
    };
    auto index_of = [&](int row) { return row_index(a, it, row); };
    const int most = __builtin_amdgcn_readfirstlane(sees(last)), least = __builtin_amdgcn_readfirstlane(sees(row0));
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = row0 + 16 * rt + r16;
        const bool ok = row < rows;
        seen[rt] = ok ? sees(row) : most;  // rows past the last mask nothing
        const uint8_t* const qrow = a.q + index_of(row) * D * 2;
#pragma unroll
        for (int c = 0; c < QK; ++c) {
            const int d = FP8 ? 64 * (c >> 1) + 16 * g + 8 * (c & 1) : 32 * c + 8 * g;
            v4i x{0, 0, 0, 0};
            if (ok) x = *(const v4i*)(qrow + d * 2);
            qop[rt][c] = __builtin_bit_cast(v8bf, x);
        }
    }
    // striping: whole rounds and the rest of what each row sees
    const int stride = a.pages.pcp * a.pages.interleave;
    auto striped = [&](int keys, int& whole, int& tail) {
        const int round = (int)div((uint32_t)keys, a.pages.div_stride);
        whole = round * a.pages.interleave;
        tail = keys - round * stride;
    };
    int rounds[RT], rest[RT], most_rounds, most_rest, least_rounds, least_rest;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) striped(seen[rt], rounds[rt], rest[rt]);
    striped(most, most_rounds, most_rest);
    striped(least, least_rounds, least_rest);
    auto owned = [&](int whole, int tail, int rank) {
        return whole + min(max(tail - rank * a.pages.interleave, 0), a.pages.interleave);
    };

    // ---- the wave's steps ----------------------------------------------------------
    const const_i32_ptr table = (const_i32_ptr)(a.pages.table + (table_of(a.pages, it.b) << a.pages.table_shift));
    const int steps = (it.end - it.begin) * S::SUB;
    // The wave's first step from step u on that has keys, its page still a table
    // entry to be read (entry -1: past the last).  Steps without keys are passed
    // over here, in scalar code: a loop body that may be skipped had two copies
    // of O^T and K in registers.
    auto step_from = [&](int u) {
        FewStep<S> s{0, 0, 0, -1, 0, u, -1};
        for (; s.u < steps; s.u += S::WAVES) {
            const uint32_t tile = it.begin + s.u / S::SUB;
            const uint32_t lt = div(tile, a.pages.div_pcp);
            const int rank = tile - lt * a.pages.pcp;
            const int local = lt * kTileKeys + (s.u % S::SUB) * S::KEYS;
            const int n = min(owned(most_rounds, most_rest, rank) - local, S::KEYS);
            const uint32_t blk = div(local, a.pages.div_block);
            if (n <= 0 || (int)blk >= a.pages.max_local_blocks) continue;
            s.n = __builtin_amdgcn_readfirstlane(n);
            s.rank = __builtin_amdgcn_readfirstlane(rank);
            s.local = __builtin_amdgcn_readfirstlane(local);
            s.entry = __builtin_amdgcn_readfirstlane(rank * a.pages.max_local_blocks + (int)blk);
            s.slot = __builtin_amdgcn_readfirstlane(local - (int)blk * a.pages.block_size);
            break;
        }
        return s;
    };
    auto read_entry = [&](const FewStep<S>& s) { return entry_of(table, a.pages, s.entry); };
    // The step with its page, from what was read ahead; steps without a page are
    // passed over.
    auto with_page = [&](FewStep<S> s, TableEntry e) {
        while (s.entry >= 0) {
            s.page = page_of(a.pages, e);
            if (s.page >= 0) break;
            s = step_from(s.u + S::WAVES);
            e = read_entry(s);
        }
        return s;
    };

    uint8_t* const my_lds = lds + wave * 2 * S::V_BYTES;
    const uint32_t my_addr = lds_address(my_lds);
    const uint32_t k_lane = (8 * (r16 >> 2) + (r16 & 3)) * ROW + 16 * g;
    // lane's chunk of DMA block 0: LDS chunk `lane` holds the swizzled one.  Block
    // i's keys differ in bits that the lane does not set: their part of the
    // swizzle is a constant.
    uint32_t v_lane;
    {
        const int key = lane / S::CH, c = lane % S::CH;
        v_lane = key * ROW + ((c ^ few_swizzle<ROW, FP8>(key)) << 4);
    }
    // transposing reads: this lane's address of d tile 0, 32-key group 0
    uint32_t v_read[FP8 ? 1 : 2];
    if constexpr (FP8) {
        const int key = 8 * g + (r16 >> 1);
        v_read[0] = my_addr + key * ROW + (few_swizzle<ROW, FP8>(key) << 4) + 8 * (r16 & 1);
    } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int key = 8 * g + 4 * s + (r16 >> 2), byte = 8 * (r16 & 3);
            v_read[s] = my_addr + key * ROW + (((byte >> 4) ^ few_swizzle<ROW, FP8>(key)) << 4) + (byte & 15);
        }
    }
    const uint8_t* const k_pool = a.pool + it.head * a.pages.head_stride;
    const int64_t v_offset = a.pages.num_kv_heads * a.pages.head_stride;
    const float* const k_scales = a.token_scales + (int64_t)it.head * a.pages.block_size;
    const int64_t vs_offset = (int64_t)a.pages.num_kv_heads * a.pages.block_size;
    FewLoads<S> L;
    auto issue_v = [&](const FewStep<S>& s, uint32_t dst) {
        if (s.page < 0) return;
        const uint8_t* const vb = k_pool + s.page * a.pages.page_stride + s.slot * ROW + v_offset;
        // (opaque, here and below: addresses that differ by a constant are formed
        // when they are used, not kept in registers for the whole walk)
        uint32_t off = v_lane;
        asm volatile("" : "+v"(off));
        static_for<0, S::V_BLOCKS>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            dma_sbase<0>(vb + 1024 * i, off ^ (few_swizzle<ROW, FP8>(64 * i / S::CH) << 4), dst + 1024 * i);
        });
    };
    auto issue_k = [&](const FewStep<S>& s) {
        if (s.page < 0) return;
        const uint8_t* const kb = k_pool + s.page * a.pages.page_stride + s.slot * ROW + k_lane;
#pragma unroll
        for (int t = 0; t < 2 * KG; ++t)
#pragma unroll
            for (int c = 0; c < KC; ++c)
                L.k[t * KC + c] = *(const v4i*)(kb + ((t >> 1) * 32 + (t & 1) * 4) * ROW + c * 64);
    };
    auto issue_scales = [&](const FewStep<S>& s) {
        if (!SCALED || s.page < 0) return;
        const float* const sc = k_scales + (int64_t)s.page * 2 * vs_offset + s.slot + 8 * g;
#pragma unroll
        for (int t = 0; t < 2 * KG; ++t) {
            L.ks[t] = *(const v4f*)(sc + (t >> 1) * 32 + (t & 1) * 4);
            L.vs[t] = *(const v4f*)(sc + vs_offset + (t >> 1) * 32 + (t & 1) * 4);
        }
    };

    float m[RT], l[RT];
    v4f o[RT][DT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = kNoScore;
        l[rt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    // ---- the walk: two steps on a table entry is read, the next step's keys load, this one
    // runs ----
    FewStep<S> ahead = step_from(wave);
    FewStep<S> st = with_page(ahead, read_entry(ahead));
    ahead = step_from(st.u + S::WAVES);
    FewStep<S> nxt = with_page(ahead, read_entry(ahead));
    ahead = step_from(nxt.u + S::WAVES);
    TableEntry entry = read_entry(ahead);
    issue_v(st, my_addr);
    issue_k(st);
    issue_scales(st);
    uint32_t buf = 0;
    while (st.page >= 0) {
        wait_vmem();
        __builtin_amdgcn_sched_barrier(0);
        issue_v(nxt, my_addr + (buf ^ S::V_BYTES));
        const FewStep<S> after = with_page(ahead, entry);
        ahead = step_from(after.u + S::WAVES);
        entry = read_entry(ahead);
        // ---- scores -----------------------------------------------------------
        v4f s[RT][2 * KG];
#pragma unroll
        for (int t = 0; t < 2 * KG; ++t) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < QK; ++c) {
                v8bf kop;
                if constexpr (FP8) {
                    const v4i x = L.k[t * KC + (c >> 1)];
                    kop = __builtin_bit_cast(v8bf, e4m3x8_to_bf16x8(x[2 * (c & 1)], x[2 * (c & 1) + 1]));
                } else {
                    kop = __builtin_bit_cast(v8bf, L.k[t * KC + c]);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    s[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop, qop[rt][c], s[rt][t], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        issue_k(nxt);
        __builtin_amdgcn_sched_barrier(0);
        // ---- V's rows that not every row sees, or none -----------------------------
        const int all = owned(least_rounds, least_rest, st.rank) - st.local;  // keys that every row sees
        if (all < S::KEYS) {
            uint8_t* const vt = my_lds + buf;
            // A value that is not finite would reach rows that do not see its key,
            // as 0 times it: such values are added to the rows that do, and
            // cleared before the product.
            for (int key = max(all, 0); key < st.n; ++key) {
                static_for<0, DT>([&](auto dc) {
                    constexpr int dt = decltype(dc)::value;
                    const int byte = (16 * dt + 4 * g) * (FP8 ? 1 : 2);
                    uint8_t* const at = vt + key * ROW + (((byte >> 4) ^ few_swizzle<ROW, FP8>(key)) << 4) + (byte & 15);
                    float v[4];
                    if constexpr (FP8) {
                        const int w = *(const int*)at;
                        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
                        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
                        v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
                    } else {
                        const v2i w = *(const v2i*)at;
                        v[0] = bf16_bits_to_f32((uint32_t)w[0] & 0xffffu), v[1] = bf16_bits_to_f32((uint32_t)w[0] >> 16);
                        v[2] = bf16_bits_to_f32((uint32_t)w[1] & 0xffffu), v[3] = bf16_bits_to_f32((uint32_t)w[1] >> 16);
                    }
                    bool bad = false;
#pragma unroll
                    for (int i = 0; i < 4; ++i) bad |= !(fabsf(v[i]) < INFINITY);
                    if (__builtin_amdgcn_ballot_w64(bad)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool hit = !(fabsf(v[i]) < INFINITY);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt)
                                if (hit && key < owned(rounds[rt], rest[rt], st.rank) - st.local) o[rt][dt][i] += v[i];
                            if (hit && r16 == 0) {
                                if constexpr (FP8)
                                    at[i] = 0;
                                else
                                    ((uint16_t*)at)[i] = 0;
                            }
                        }
                    }
                });
            }
            for (int i = st.n * S::CH + lane; i < S::KEYS * S::CH; i += 64) *(v4i*)(vt + i * 16) = v4i{0, 0, 0, 0};
            asm volatile("" ::: "memory");
            if constexpr (SCALED) {  // (nor do the scales of slots without a token mean anything)
#pragma unroll
                for (int t = 0; t < 2 * KG; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        L.vs[t][i] = 32 * (t >> 1) + 4 * (t & 1) + i < st.n - 8 * g ? L.vs[t][i] : 0.f;
            }
        }
        // ---- softmax ---------------------------------------------------------------
        v8bf pop[RT][KG], low[RT][KG];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int vis = owned(rounds[rt], rest[rt], st.rank) - st.local;
#pragma unroll
            for (int t = 0; t < 2 * KG; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[rt][t][i] *= SCALED ? L.ks[t][i] * a.score_scale : a.score_scale;
            if (all < S::KEYS) {
#pragma unroll
                for (int t = 0; t < 2 * KG; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[rt][t][i] = 32 * (t >> 1) + 4 * (t & 1) + i < vis - 8 * g ? s[rt][t][i] : -INFINITY;
            }
            float mx = s[rt][0][0];
#pragma unroll
            for (int t = 0; t < 2 * KG; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rt][t][i]);
            mx = quarters_max(mx);
            const bool raise = mx > m[rt] + 8.f;
            if (__builtin_amdgcn_ballot_w64(raise)) {
                const float next = raise ? mx : m[rt];
                const float keep = raise ? __builtin_amdgcn_exp2f(m[rt] - next) : 1.f;
                l[rt] *= keep;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= keep;
                m[rt] = next;
            }
#pragma unroll
            for (int t = 0; t < 2 * KG; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(s[rt][t][i] - m[rt]);
                    l[rt] += p;
                    const float x = SCALED ? p * L.vs[t][i] : p;
                    const float high = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
                    pop[rt][t >> 1][4 * (t & 1) + i] = (__bf16)high;
                    // (the 2^-30: where x is its own upper half, the lower is not a 0
                    // that made infinite values NaN)
                    low[rt][t >> 1][4 * (t & 1) + i] = (__bf16)fmaf(x, 0x1p-30f, x - high);
                }
        }
        issue_scales(nxt);
        // ---- O^T += V^T P^T -----------------------------------------------------------
        constexpr int READS = DT * KG;  // operands: d tile dt of 32-key group kg
        uint32_t va[FP8 ? 1 : 2];
#pragma unroll
        for (int i = 0; i < (FP8 ? 1 : 2); ++i) {
            va[i] = v_read[i] + buf;
            asm volatile("" : "+v"(va[i]));
        }
        if constexpr (FP8) {
            v2i x[2][4];
            auto read4 = [&](auto nc) {
                constexpr int n = decltype(nc)::value;
                static_for<0, 4>([&](auto ec) {
                    constexpr int op = 4 * n + decltype(ec)::value, dt = op / KG, kg = op % KG;
                    x[n & 1][decltype(ec)::value] =
                        ds_read_tr8_b64<kg * 32 * ROW>(va[0] ^ (dt << 4));
                });
            };
            read4(std::integral_constant<int, 0>{});
            static_for<0, READS / 4>([&](auto nc) {
                constexpr int n = decltype(nc)::value;
                lds_results_ready(x[n & 1]);
                if constexpr (n + 1 < READS / 4) read4(std::integral_constant<int, n + 1>{});
                static_for<0, 4>([&](auto ec) {
                    constexpr int e = decltype(ec)::value, op = 4 * n + e, dt = op / KG, kg = op % KG;
                    const v8bf vop = __builtin_bit_cast(v8bf, e4m3x8_to_bf16x8(x[n & 1][e][0], x[n & 1][e][1]));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, low[rt][kg], o[rt][dt], 0, 0, 0);
                        o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, pop[rt][kg], o[rt][dt], 0, 0, 0);
                    }
                });
            });
        } else {
            v2i x[2][4];  // two operands of two reads
            auto read2 = [&](auto nc) {
                constexpr int n = decltype(nc)::value;
                static_for<0, 2>([&](auto ec) {
                    constexpr int e = decltype(ec)::value, op = 2 * n + e, dt = op / KG, kg = op % KG;
                    constexpr int off = kg * 32 * ROW;
                    x[n & 1][2 * e] = ds_read_tr16_b64<off>(va[0] ^ (dt << 5));
                    x[n & 1][2 * e + 1] = ds_read_tr16_b64<off>(va[1] ^ (dt << 5));
                });
            };
            read2(std::integral_constant<int, 0>{});
            static_for<0, READS / 2>([&](auto nc) {
                constexpr int n = decltype(nc)::value;
                lds_results_ready(x[n & 1]);
                if constexpr (n + 1 < READS / 2) read2(std::integral_constant<int, n + 1>{});
                static_for<0, 2>([&](auto ec) {
                    constexpr int e = decltype(ec)::value, op = 2 * n + e, dt = op / KG, kg = op % KG;
                    const v4i w{x[n & 1][2 * e][0], x[n & 1][2 * e][1], x[n & 1][2 * e + 1][0], x[n & 1][2 * e + 1][1]};
                    const v8bf vop = __builtin_bit_cast(v8bf, w);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, low[rt][kg], o[rt][dt], 0, 0, 0);
                        o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vop, pop[rt][kg], o[rt][dt], 0, 0, 0);
                    }
                });
            });
        }
        st = nxt;
        nxt = after;
        buf ^= S::V_BYTES;
    }

    // ---- the waves' results meet: 16 rows at a time ---------------------------------
    float* const ol = (float*)lds;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = quarters_sum(l[rt]);
        __syncthreads();  // every wave is done with its part of the LDS
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            *(v4f*)(ol + (wave * 16 + r16) * S::O_ROW + 16 * dt + 4 * g) = o[rt][dt];
        if (g == 0) {
            wave_ml[wave][r16][0] = m[rt];
            wave_ml[wave][r16][1] = sum;
        }
        __syncthreads();
        for (int i = tid; i < 16 * (D / 4); i += S::THREADS) {
            const int j = i / (D / 4), c = i % (D / 4), row = row0 + 16 * rt + j;
            if (row >= rows) continue;
            float top = wave_ml[0][j][0];
#pragma unroll
            for (int w = 1; w < S::WAVES; ++w) top = fmaxf(top, wave_ml[w][j][0]);
            float total = 0.f;
            v4f acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < S::WAVES; ++w) {
                const float weight = __builtin_amdgcn_exp2f(wave_ml[w][j][0] - top);
                total = fmaf(weight, wave_ml[w][j][1], total);
                const v4f x = *(const v4f*)(ol + (w * 16 + j) * S::O_ROW + 4 * c);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = fmaf(weight, x[k], acc[k]);
            }
            // (a row that sees nothing: zeros.  NaN sums divide to NaN)
            const bool empty = total == 0.f;
            const float inv = empty ? 0.f : a.v_scale / total;
            const float log2sum = empty ? -INFINITY : top + __builtin_amdgcn_logf(total);
            if (it.plan.ranges > 1) {
                const int64_t prow = (int64_t)blockIdx.x * S::ROWS + 16 * rt + j;
                *(v4f*)(a.part_o + prow * D + 4 * c) = empty ? v4f{0.f, 0.f, 0.f, 0.f} : acc * inv;
                if (c == 0) a.part_ml[prow] = v2f{top, total};
            } else {
                const int64_t at = index_of(row);
                uint32_t w[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const __bf16 lo = (__bf16)(empty ? 0.f : acc[2 * k] * inv), hi = (__bf16)(empty ? 0.f : acc[2 * k + 1] * inv);
                    w[k] = (uint32_t)__builtin_bit_cast(uint16_t, lo) | ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
                }
                *(v2i*)(a.out + (at * D + 4 * c) * 2) = v2i{(int)w[0], (int)w[1]};
                if (a.lse && c == 0) a.lse[at] = log2sum * kLn2;
            }
        }
    }
}

// ---- many rows -------------------------------------------------------------------
//
// For more rows per (sequence, KV head) the products bound: the tile kernel's
// workgroups of 128 rows (tile_kernel.hpp: K and V tiles shared through LDS, both
// products on 32x32 MFMAs, bf16 operands), over the walk of this sequence's table
// and with every row's own last key.  MFMA bound, with the softmax and (e4m3) the
// widening of K and V beside it: 512 new tokens of 32768, 64 over 8 heads at D 128,
// bf16, 540 us (1.0 PFLOP/s, where a bf16 matrix product of the library reaches
// 1.3); seven prompts of up to 4096 tokens, 32 over 2 heads at D 256, e4m3 with
// token scales, 665 us (0.80).  P is rounded once to bf16: as two values, as for few
// rows, the two took 754 and 914 us.

// The sequence's walk for one workgroup: tile i of [begin, end) as find_item
// counts them.
struct ManyTile {
    int i;
    int page;   // -1: past the last
    int slot;
    int n;      // keys that some row may see
    int rank;
    int local;
    int entry;  // of the table
};

template <int D, bool FP8, bool SCALED>
__global__ void __launch_bounds__((TileShape<D, FP8, false>::THREADS), (TileShape<D, FP8, false>::PAIR ? 1 : 2))
    attend_many_kernel(AttendArgs a) {
    static_assert(!SCALED || FP8, "token scales go with e4m3 caches");
    using S = TileShape<D, FP8, false>;
    constexpr int ROW = S::ROW, CHUNKS = S::CHUNKS, QK = S::QK, DT = S::DT;
    constexpr bool F8 = S::F8, TWO = S::TILES == 2;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::LDS_BYTES];
    __shared__ __attribute__((aligned(16))) float scales[SCALED ? 2 * S::TILES * 2 * kKeyTile : 4];
    __shared__ float pair_ml[S::PAIR ? kWaves * 64 * 2 : 1];
    __shared__ int spoiled;  // a value that is not finite was taken out of some tile's V

    Item it;
    if (!find_item<1>(a, blockIdx.x, kRowsPerGroup, it)) return;
    if (threadIdx.x == 0) spoiled = 0;  // (the first tile's barrier comes before any settle_v)
    if (it.head == 0 && it.tile == 0 && it.range == 0 && threadIdx.x == 0 && a.plans) a.plans[it.b] = it.plan;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pw = S::PAIR ? wave & (kWaves - 1) : wave;  // the wave's 32-row slot
    const int kh = S::PAIR ? wave / kWaves : 0;           // PAIR: its keys (half a tile, or every second tile)
    const int j = lane & 31, h = lane >> 5, grp = lane >> 4, gl = lane & 15;

    // ---- this lane's row and what it sees ------------------------------------------
    const int rows = it.span.count * a.group, row0 = it.tile * kRowsPerGroup;
    // (rows past the last do as the last, unseen)
    const int row_c = min(row0 + pw * kRowsPerWave + j, rows - 1);
    auto sees = [&](int r) {
        const int64_t np = (int64_t)it.length - it.span.count + (int)div((uint32_t)r, a.div_group) + 1;
        return (int)min(max(np, (int64_t)0), (int64_t)a.pages.capacity);
    };
    auto index_of = [&](int r) { return row_index(a, it, r); };
    const int seen = sees(row_c);
    const int most = __builtin_amdgcn_readfirstlane(sees(min(row0 + kRowsPerGroup, rows) - 1));
    const int least = __builtin_amdgcn_readfirstlane(sees(row0));
    v8bf qop[QK];
    {
        const uint8_t* const qrow = a.q + index_of(row_c) * D * 2;
#pragma unroll
        for (int c = 0; c < QK; ++c) {
            const int d = S::WIDE ? 32 * (c >> 1) + 16 * h + 8 * (c & 1) : 16 * c + 8 * h;
            qop[c] = __builtin_bit_cast(v8bf, *(const v4i*)(qrow + d * 2));
        }
    }

    // ---- per-lane LDS and DMA offsets (the tile kernel's maps) ------------------------
    LaneMap<S> L;
    {
        const int r = lds_row<F8>(key_of_row<F8>(0, j));
        L.k_addr = r * ROW + ((h ^ chunk_swizzle<F8, CHUNKS>(r)) << 4) + (S::PAIR_HALVES ? kh * S::K_T1_ROWS * ROW : 0);
    }
    if constexpr (F8) {
        const int r = lds_row<F8>(32 * (grp >> 1) + (gl >> 1));
        L.v_addr[0] = lds_address(lds) + r * ROW + (((grp & 1) ^ chunk_swizzle_v<F8, CHUNKS>(r)) << 4) + 8 * (gl & 1);
    } else {
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            const int vkey = 8 * (grp >> 1) + 4 * s2 + (gl >> 2);
            const int dbyte = 2 * (16 * (grp & 1) + 4 * (gl & 3));
            L.v_addr[s2] = lds_address(lds) + vkey * ROW + (((dbyte >> 4) ^ chunk_swizzle_v<F8, CHUNKS>(vkey)) << 4) +
                           (dbyte & 15) + kh * 32 * ROW;
        }
    }

    // ---- the walk ------------------------------------------------------------------------
    const const_i32_ptr table = (const_i32_ptr)(a.pages.table + (table_of(a.pages, it.b) << a.pages.table_shift));
    const int end = min(it.end, walk_tiles(a.pages, most));
    // the first tile from i on with keys, its page still a table entry to be read
    // (entry -1: past the last)
    auto tile_from = [&](int i) {
        ManyTile t{i, -1, 0, 0, 0, 0, -1};
        for (; t.i < end; ++t.i) {
            const uint32_t lt = div((uint32_t)t.i, a.pages.div_pcp);
            const int rank = t.i - lt * a.pages.pcp, local = lt * kTileKeys;
            const int n = min(owned_of(a.pages, most, rank) - local, kKeyTile);
            const uint32_t blk = div((uint32_t)local, a.pages.div_block);
            if (n <= 0 || (int)blk >= a.pages.max_local_blocks) continue;
            t.n = __builtin_amdgcn_readfirstlane(n);
            t.rank = __builtin_amdgcn_readfirstlane(rank);
            t.local = __builtin_amdgcn_readfirstlane(local);
            t.entry = __builtin_amdgcn_readfirstlane(rank * a.pages.max_local_blocks + (int)blk);
            t.slot = __builtin_amdgcn_readfirstlane(local - (int)blk * a.pages.block_size);
            break;
        }
        return t;
    };
    auto read_entry = [&](const ManyTile& t) { return entry_of(table, a.pages, t.entry); };
    // the tile with its page, from the entry read ahead; tiles without a page are passed over
    auto with_page = [&](ManyTile t, TableEntry e) {
        while (t.entry >= 0) {
            t.page = page_of(a.pages, e);
            if (t.page >= 0) break;
            t = tile_from(t.i + 1);
            e = read_entry(t);
        }
        return t;
    };
    auto next_tile = [&](int i) {
        const ManyTile t = tile_from(i);
        return with_page(t, read_entry(t));
    };
    FwdArgs f{};
    f.kv = a.pool + it.head * a.pages.head_stride;
    f.head_stride = a.pages.head_stride;
    f.num_kv_heads = a.pages.num_kv_heads;
    // (opaque here and below: what a thread's index or its row gives is formed where
    // it is used; kept over the walk it cost Q's registers, parts of which were then
    // read back from memory for every tile)
    auto opaque = [](int x) {
        asm volatile("" : "+v"(x));
        return x;
    };
    auto thread = [&]() { return opaque(tid); };
    auto visible = [&](const ManyTile& t) { return owned_of(a.pages, opaque(seen), t.rank) - t.local; };
    // the thread's scale of tile t: wave 0 K's, wave 1 V's (TWO: the next two the
    // second tile's); slots without a token have none
    auto load_scale = [&](const ManyTile& t, const ManyTile& t2) {
        const bool other = TWO && (wave & 2);
        const int page = other ? t2.page : t.page, slot = other ? t2.slot : t.slot, n = other ? t2.n : t.n;
        if (page < 0 || wave >= 2 * S::TILES) return 0.f;
        const float* const of = a.token_scales +
            (((int64_t)page * 2 + (wave & 1)) * a.pages.num_kv_heads + it.head) * a.pages.block_size + slot;
        const uint32_t key = thread() & 63;
        return (int)key < n ? of[key] : 0.f;
    };

    SoftmaxState<S> st;
    st.m = kNoScore;
    st.l = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) st.o[dt] = v16f{};

    // V rows of a staged tile that not every row sees: no value there may reach
    // a row that does not, as 0 times it, unless it is finite.  Rows past the n
    // keys are cleared, and values that are not finite: those join the rows that
    // see their keys after the walk.  Called by the whole workgroup.
    auto settle_v = [&](uint8_t* v, const ManyTile& t) {
        const int tid = thread();
        const int from = max(owned_of(a.pages, least, t.rank) - t.local, 0);
        bool bad = false;
        for (int i = from * CHUNKS + tid; i < kKeyTile * CHUNKS; i += S::THREADS) {
            v4i* const at = (v4i*)(v + lds_row<F8>(i / CHUNKS) * ROW + (i % CHUNKS) * 16);
            const v4i x = *at;
            const uint32_t keep = i < t.n * CHUNKS ? ~0u : 0u;
            v4i y;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                // the values whose exponent (code) is all ones: a carry into their sign bit
                const uint32_t u = (uint32_t)x[w];
                const uint32_t ones = F8 ? (((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7
                                         : (((u & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15;
                y[w] = (int)(u & ~(ones * (F8 ? 0xffu : 0xffffu)) & keep);
                bad |= ones != 0 && keep != 0;
            }
            *at = y;
        }
        if (bad) spoiled = 1;
        __syncthreads();
    };
    auto settled = [&](const ManyTile& t) { return owned_of(a.pages, least, t.rank) - t.local >= kKeyTile; };

    ManyTile cur = next_tile(it.begin), cur2{}, ahead, ahead2{};
    TableEntry entry, entry2{};
    float scale = 0.f;
    auto stage = [&](const ManyTile& t, const ManyTile& t2, uint8_t* buf) {
        {
            const int byte = wave * 1024 + (thread() & 63) * 16, r = byte / ROW, pos = (byte % ROW) / 16;
            L.dma_off = lds_row<F8>(r) * ROW + (pos ^ chunk_swizzle<F8, CHUNKS>(r)) * 16;
            L.dma_off_v = lds_row<F8>(r) * ROW + (pos ^ chunk_swizzle_v<F8, CHUNKS>(r)) * 16;
        }
        if (t.page >= 0) stage_tile_async<S>(f, TileCursor{0, t.slot, 0, t.page * a.pages.page_stride}, buf, wave, L);
        if (TWO && t2.page >= 0)
            stage_tile_async<S>(f, TileCursor{0, t2.slot, 0, t2.page * a.pages.page_stride}, buf + 2 * S::TILE, wave, L);
        if constexpr (SCALED) scale = load_scale(t, t2);
    };
    if constexpr (TWO) cur2 = next_tile(cur.i + 1);
    stage(cur, cur2, lds);
    auto look_ahead = [&](int i) {  // (a step ahead of their use: no wait for the table's memory)
        ahead = tile_from(i);
        entry = read_entry(ahead);
        if constexpr (TWO) {
            ahead2 = tile_from(ahead.i + 1);
            entry2 = read_entry(ahead2);
        }
    };
    look_ahead((TWO ? cur2.i : cur.i) + 1);
    for (int rbuf = 0; cur.page >= 0; rbuf ^= 1) {
        const ManyTile nxt = with_page(ahead, entry);
        // (a tile without a page was passed over: the second follows anew)
        const ManyTile nxt2 = !TWO ? ManyTile{} : nxt.i < ahead2.i ? with_page(ahead2, entry2) : next_tile(nxt.i + 1);
        look_ahead((TWO ? nxt2.i : nxt.i) + 1);
        const uint32_t rt_off = rbuf * S::BUFFER;
        wait_vmem();  // this wave's loads of the current tiles have landed
        float* const sc = scales + rbuf * S::TILES * 2 * kKeyTile;
        if (const int t = thread(); SCALED && t < 128 * S::TILES) sc[t] = scale;
        __syncthreads();  // ... and every wave's; the other buffer is free
        stage(nxt, nxt2, lds + (rt_off ^ S::BUFFER));
        if (!settled(cur)) settle_v(lds + rt_off + S::TILE, cur);
        if (TWO && cur2.page >= 0 && !settled(cur2)) settle_v(lds + rt_off + 3 * S::TILE, cur2);
        const int hl = (thread() >> 5) & 1;
        if constexpr (TWO) {
            const ManyTile& t = kh ? cur2 : cur;
            if (t.page >= 0)
                compute_tile<S, 0, true, SCALED>(lds, rt_off + kh * 2 * S::TILE, visible(t),
                                                 qop, a.score_scale, L, hl, st, sc + kh * 2 * kKeyTile);
        } else {
            const int first_key = S::PAIR ? 32 * kh : 0;
            compute_tile<S, 0, true, SCALED>(lds, rt_off, visible(cur) - first_key, qop,
                                             a.score_scale, L, hl, st, sc);
        }
        cur = nxt;
        cur2 = nxt2;
    }

    // (the arguments are read anew: kept over the walk they cost it scalar
    // registers; seven prompts, D 256, e4m3: 696 -> 682 us)
    auto* args = (const __attribute__((address_space(4))) uint8_t*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    const AttendArgs& z = *(const AttendArgs*)args;
    const int lane2 = thread() & 63, h2 = lane2 >> 5;
    const int row = row0 + pw * kRowsPerWave + (lane2 & 31);

    // ---- PAIR: the two waves' results meet in the first wave of the pair ----------------
    if constexpr (S::PAIR) {
        float* const xo = (float*)lds + pw * (DT * 16 * 64);
        __syncthreads();
        if (kh == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4)
                    *(v4f*)(xo + ((4 * dt + r4) * 64 + lane2) * 4) =
                        v4f{st.o[dt][4 * r4], st.o[dt][4 * r4 + 1], st.o[dt][4 * r4 + 2], st.o[dt][4 * r4 + 3]};
            pair_ml[(pw * 64 + lane2) * 2] = st.m;
            pair_ml[(pw * 64 + lane2) * 2 + 1] = st.l;
        }
        __syncthreads();
        if (kh == 1) return;
        const float m1 = pair_ml[(pw * 64 + lane2) * 2], l1 = pair_ml[(pw * 64 + lane2) * 2 + 1];
        const float m = fmaxf(st.m, m1);
        const float w0 = __builtin_amdgcn_exp2f(st.m - m), w1 = __builtin_amdgcn_exp2f(m1 - m);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const v4f x = *(const v4f*)(xo + ((4 * dt + r4) * 64 + lane2) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) st.o[dt][4 * r4 + i] = fmaf(w1, x[i], w0 * st.o[dt][4 * r4 + i]);
            }
        st.l = fmaf(w1, l1, w0 * st.l);
        st.m = m;
    }

    if constexpr (!S::PAIR) __syncthreads();  // (spoiled is whole: PAIR has passed two barriers)
    // ---- values that are not finite, for the rows that see them (from the pages) -----------
    if (spoiled) {
        for (ManyTile t = next_tile(it.begin); t.page >= 0; t = next_tile(t.i + 1)) {
            const int vis = min(owned_of(a.pages, sees(min(row, rows - 1)), t.rank) - t.local, t.n);
            for (int key = max(owned_of(a.pages, least, t.rank) - t.local, 0); key < t.n; ++key) {
                const uint8_t* const v = f.kv + t.page * a.pages.page_stride + a.pages.num_kv_heads * a.pages.head_stride +
                                         (int64_t)(t.slot + key) * ROW + 4 * h2 * S::ES;
                if (key >= vis) continue;
                static_for<0, 4 * DT>([&](auto c) {
                    constexpr int dt = decltype(c)::value >> 2, r4 = decltype(c)::value & 3;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int d = 32 * dt + 8 * r4 + i;
                        float x;
                        if constexpr (F8)
                            x = (v[d] & 0x7f) == 0x7f ? NAN : 0.f;
                        else
                            x = bf16_bits_to_f32(((const uint16_t*)v)[d]);
                        if (!(fabsf(x) < INFINITY)) st.o[dt][4 * r4 + i] += x;
                    }
                    __builtin_amdgcn_sched_barrier(0);  // (few registers for this rare path)
                });
            }
        }
    }

    // ---- O = O^T / l, or the range's partial result ---------------------------------------
    const float total = halves_sum(st.l);
    const bool empty = total == 0.f;
    const float inv = empty ? 0.f : z.v_scale / total;
    const float log2sum = empty ? -INFINITY : st.m + __builtin_amdgcn_logf(total);
    if (row >= rows) return;
    const int64_t out_row = row_index(z, it, row);
    const bool part = it.plan.ranges > 1;
    const int64_t prow = (int64_t)blockIdx.x * kRowsPerGroup + pw * kRowsPerWave + (lane2 & 31);
    float* const po = z.part_o + prow * D;
    uint8_t* const orow = z.out + out_row * D * 2;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = 32 * dt + 8 * r4 + 4 * h2;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = empty ? 0.f : st.o[dt][4 * r4 + i] * inv;
            if (part) {
                *(v4f*)(po + d) = v4f{x[0], x[1], x[2], x[3]};
            } else {
                uint32_t w[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const __bf16 lo = (__bf16)x[2 * k], hi = (__bf16)x[2 * k + 1];
                    w[k] = (uint32_t)__builtin_bit_cast(uint16_t, lo) |
                           ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
                }
                *(v2i*)(orow + 2 * d) = v2i{(int)w[0], (int)w[1]};
            }
        }
    if (h2 == 0) {
        if (part)
            z.part_ml[prow] = v2f{st.m, total};
        else if (z.lse)
            z.lse[out_row] = log2sum * kLn2;
    }
}

// ---- ranges of one walk ----------------------------------------------------------

// A row's partial results: where they are, for the row of `token` and Q head
// `head`; false if its result is final or there is no such row.
struct Partials {
    int64_t first;  // row of the first range's partial result
    int64_t step;   // rows from one range's to the next
    int ranges;
};
__device__ __forceinline__ bool partials_of(const AttendArgs& a, int b, int token, int head, Partials& p) {
    if (b < 0) return false;
    const SequencePlan plan = a.plans[b];
    if (plan.ranges <= 1) return false;
    const Span span = span_of(a.chunk, b);
    const int kv = (int)div((uint32_t)head, a.div_group);
    const int row = (token - span.first) * a.group + (head - kv * a.group);
    const int tile = row >> a.rows_log2;
    const int64_t heads = a.pages.num_kv_heads, item = plan.first_item + ((int64_t)plan.tiles - 1 - tile) * heads + kv;
    const int64_t step = plan.tiles * heads;
    // (only with starts that decrease is there a plan that no workgroup wrote:
    // whatever it holds, nothing past the launch's items is read)
    if (plan.first_item < 0 || tile >= plan.tiles || step > a.max_items || plan.ranges > a.max_items ||
        item + (plan.ranges - 1) * step >= a.max_items)
        return false;
    p = Partials{(item << a.rows_log2) + row - (tile << a.rows_log2), step << a.rows_log2, plan.ranges};
    return true;
}

// The running merge of partial results: weights sum 2^(max - top).
struct Merged {
    float top, total;
    v4f acc;
    __device__ __forceinline__ void add(const v2f& ml, const v4f& x) {
        const float next = fmaxf(top, ml[0]);
        const float keep = __builtin_amdgcn_exp2f(top - next);
        const float weight = ml[1] * __builtin_amdgcn_exp2f(ml[0] - next);
        total = fmaf(total, keep, weight);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = fmaf(acc[k], keep, weight * x[k]);
        top = next;
    }
};

// Four values of a merged row to the output, and (first lane) its log-sum-exp.
template <int D>
__device__ __forceinline__ void store_merged(const AttendArgs& a, int64_t row, int c, float top, float total, const v4f& acc) {
    const bool empty = total == 0.f;
    const float inv = empty ? 0.f : 1.f / total;
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const __bf16 lo = (__bf16)(empty ? 0.f : acc[2 * k] * inv), hi = (__bf16)(empty ? 0.f : acc[2 * k + 1] * inv);
        w[k] = (uint32_t)__builtin_bit_cast(uint16_t, lo) | ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
    }
    *(v2i*)(a.out + (row * D + 4 * c) * 2) = v2i{(int)w[0], (int)w[1]};
    if (a.lse && c == 0) a.lse[row] = empty ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

// Rows with few ranges each: D / 4 threads go through a row's partials in turn.
// A token's Q heads are a workgroup's rows, THREADS / (D / 4) at a time.
template <int D>
__global__ void __launch_bounds__(256) merge_few_ranges_kernel(AttendArgs a) {
    constexpr int LANES = D / 4, AT_ONCE = 256 / LANES, UNROLL = 4;
    const int token = blockIdx.x, b = sequence_of(a.chunk, token);
    const int c = threadIdx.x % LANES;
    for (int head = blockIdx.y * AT_ONCE + threadIdx.x / LANES; head < a.num_q_heads; head += gridDim.y * AT_ONCE) {
        Partials p;
        if (!partials_of(a, b, token, head, p)) continue;
        Merged r{kNoScore, 0.f, v4f{0.f, 0.f, 0.f, 0.f}};
        for (int s0 = 0; s0 < p.ranges; s0 += UNROLL) {
            v2f ml[UNROLL];
            v4f x[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int64_t row = p.first + min(s0 + u, p.ranges - 1) * p.step;
                ml[u] = a.part_ml[row];
                x[u] = *(const v4f*)(a.part_o + row * D + 4 * c);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) r.add(s0 + u < p.ranges ? ml[u] : v2f{kNoScore, 0.f}, x[u]);
        }
        store_merged<D>(a, (int64_t)token * a.num_q_heads + head, c, r.top, r.total, r.acc);
    }
}

// Rows with many ranges: a workgroup of 16 waves per 64 values of a (row, Q
// head), 64 partials at a time, 16 lanes to each; the four of a wave meet in
// registers, the waves in LDS.  (32 rows of 256 ranges at D 256:
// 5.1 us; 9.0 with one wave for a row.)
constexpr int kMergeParts = 64;  // values of a workgroup
template <int D>
__global__ void __launch_bounds__(1024) merge_many_ranges_kernel(AttendArgs a) {
    constexpr int LANES = kMergeParts / 4, AT_ONCE = 1024 / LANES, UNROLL = 4, WAVES = 16;
    __shared__ v4f part[WAVES][LANES];
    __shared__ float part_ml[WAVES][2];
    const int token = blockIdx.x, head = blockIdx.y;
    const int b = sequence_of(a.chunk, token);
    Partials p;
    if (!partials_of(a, b, token, head, p)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = threadIdx.x / LANES, c = threadIdx.x % LANES;
    const int value = blockIdx.z * kMergeParts + 4 * c;
    Merged r{kNoScore, 0.f, v4f{0.f, 0.f, 0.f, 0.f}};
    for (int s0 = at; s0 < p.ranges; s0 += AT_ONCE * UNROLL) {
        v2f ml[UNROLL];
        v4f x[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int64_t row = p.first + min(s0 + u * AT_ONCE, p.ranges - 1) * p.step;
            ml[u] = a.part_ml[row];
            x[u] = *(const v4f*)(a.part_o + row * D + value);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) r.add(s0 + u * AT_ONCE < p.ranges ? ml[u] : v2f{kNoScore, 0.f}, x[u]);
    }
    // (a partial that saw nothing has the sum 0; one that is NaN has a NaN sum)
    float top = quarters_max(r.top);
    float weight = __builtin_amdgcn_exp2f(r.top - top);
    float total = quarters_sum(weight * r.total);
    v4f acc;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = quarters_sum(weight * r.acc[k]);
    if (lane < LANES) part[wave][c] = acc;
    if (lane == 0) {
        part_ml[wave][0] = top;
        part_ml[wave][1] = total;
    }
    __syncthreads();
    if (threadIdx.x >= LANES) return;
    top = part_ml[0][0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) top = fmaxf(top, part_ml[i][0]);
    total = 0.f;
    acc = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        weight = __builtin_amdgcn_exp2f(part_ml[i][0] - top);
        total = fmaf(weight, part_ml[i][1], total);
        const v4f x = part[i][c];
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = fmaf(weight, x[k], acc[k]);
    }
    store_merged<D>(a, (int64_t)token * a.num_q_heads + head, value / 4, top, total, acc);
}

}  // namespace chunk
}  // namespace pcpa
