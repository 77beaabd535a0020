// Rows of new tokens: norms and rotation of Q and K, K and V into the pages of
// their sequences, and a cache read back.
#pragma once

#include "cache_kernels.hpp"
#include "chunk_common.hpp"

namespace pcpa {
namespace chunk {

constexpr int kTokenThreads = 256;

struct RowsIn {
    const uint8_t* data;   // null: none
    int64_t token_stride;  // bytes
    int64_t head_stride;
};
struct RowsOut {
    uint8_t* data;
    int64_t token_stride;
    int64_t head_stride;
};

enum Positions : int32_t { kOfChunk = 0, kFromFirst = -1, kInt32 = 32, kInt64 = 64 };

struct TokenArgs {
    Desc chunk;
    Pages pages;          // PAGES kernels
    RowsIn q, k, v;
    RowsOut q_out, k_out, v_out;
    int32_t num_q_heads, num_kv_heads;
    // waves: q_waves of Q (q_parts a token, NG groups each), then kv_waves of K and
    // as many of V (each group of heads over token_blocks runs of NG tokens)
    int32_t q_waves, q_parts, kv_waves, token_blocks;
    int32_t waves;        // all of them: a workgroup's last may be of none
    Div div_q_parts, div_token_blocks;
    int32_t striped;      // q_out is [pcp, Hq, local_q, D]
    int32_t local_q;
    int32_t position_kind;
    const void* positions;
    int64_t first_pos;
    // rotation
    int32_t rotary_dim, interleaved;
    float amplitude, norm_eps;
    const double* turns;
    const uint8_t* q_weight;
    const uint8_t* k_weight;
    int32_t weight_f32;
    // pages
    uint8_t* pool;
    float* token_scales;  // [num_pages, 2, Hkv, block_size] or null
    float k_scale, v_scale;
};

__device__ __forceinline__ v4i to_bf16x8(const float (&x)[8]) {
    v4i r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __bf16 lo = (__bf16)x[2 * i], hi = (__bf16)x[2 * i + 1];
        r[i] = (int)((uint32_t)__builtin_bit_cast(uint16_t, lo) | ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16));
    }
    return r;
}
__host__ __device__ constexpr int token_rows(int d) { return 64 / (d / 8); }  // rows of a group

// A group is 64 / (D / 8) heads of one token's Q, K or V, a row's D values 8 to
// a lane in D / 8 neighbouring lanes.  A wave takes NG groups of one kind: of Q,
// neighbouring heads of one token; of K or V, one group of heads of neighbouring
// tokens.  Of the rotated values in the half layout a lane takes four and their
// four partners, else eight in a row: both values of a pair are in one lane.
//   ROTATE  norms and rotation of the q and k rows
//   PAGES   k and v rows go into the pages (FP8: e4m3 ones), else to k_out and
//           v_out
// HBM bound by its bytes (2 read and 1 or 2 written per value) only as long as a
// group costs less than about 180 vector and, as the four SIMDs share one scalar
// unit, 45 scalar instructions, and waits are few.  So: the groups of a wave are
// a stride apart; the rows are loaded before the tokens' places are known, which
// take two dependent loads; sums, maxima and quotients run side by side (no
// branch until the stores); sine and cosine are the hardware's (2^-23 off at most
// over 2^22 even steps of a turn).  NG is 4 where that still leaves the GPU full
// of waves, else 1: the wait is shorter (4096
// tokens of 32 + 2 + 2 heads at D 256, normed, a quarter rotated, laid out for a
// prefill: 31.7 us, 4.8 TB/s, where a 256 MiB copy reaches 5.5; 53.9 us when the
// groups took 709 vector and 782 scalar instructions instead of 509 and 265).
template <int D, bool ROTATE, bool PAGES, bool FP8, int NG>
__global__ void __launch_bounds__(kTokenThreads) token_kernel(TokenArgs a) {
    constexpr int LANES = D / 8, ROWS = token_rows(D);  // lanes of a row, rows of a group
    const int lane = threadIdx.x & 63, c = lane % LANES, r = lane / LANES;
    const int wid = __builtin_amdgcn_readfirstlane((blockIdx.x * kTokenThreads + threadIdx.x) >> 6);

    if (wid >= a.waves) return;

    // ---- the wave's groups: group i is token0 + i * dt, heads head0 + i * dh + [0, ROWS) ----
    const bool is_q = wid < a.q_waves, is_v = !is_q && wid >= a.q_waves + a.kv_waves;
    int token0, head0, dt;
    if (is_q) {
        token0 = (int)div((uint32_t)wid, a.div_q_parts);
        head0 = (wid - token0 * a.q_parts) * (NG * ROWS);
        dt = 0;
    } else {
        const int w = wid - a.q_waves - (is_v ? a.kv_waves : 0);
        const int hg = (int)div((uint32_t)w, a.div_token_blocks);
        token0 = (w - hg * a.token_blocks) * NG;
        head0 = hg * ROWS;
        dt = 1;
    }
    const int dh = (1 - dt) * ROWS, heads = is_q ? a.num_q_heads : a.num_kv_heads;
    const int tokens = dt ? min(NG, a.chunk.num_tokens - token0) : 1;
    auto there = [&](int i) { return (dt == 0 || i < tokens) && head0 + i * dh + r < heads; };

    // this lane's values of a row: [d0, d0 + 4) and [d1, d1 + 4)
    const bool turning = ROTATE && !is_v && 8 * c < a.rotary_dim;
    const bool apart = turning && !a.interleaved;
    const int d0 = apart ? 4 * c : 8 * c, d1 = apart ? 4 * c + a.rotary_dim / 2 : 8 * c + 4;

    // ---- the rows and the weights -----------------------------------------------------------
    v2i raw[NG][2];
    {
        const RowsIn in = is_q ? a.q : is_v ? a.v : a.k;
        const uint8_t* src = in.data + token0 * in.token_stride + head0 * in.head_stride;
        const int64_t step = dt ? in.token_stride : dh * in.head_stride, mine = r * in.head_stride + 2 * d0;
#pragma unroll
        for (int i = 0; i < NG; ++i, src += step) {
            raw[i][0] = raw[i][1] = v2i{0, 0};
            if (!there(i)) continue;
            raw[i][0] = *(const v2i*)(src + mine);
            raw[i][1] = *(const v2i*)(src + mine + 2 * (d1 - d0));
        }
    }
    auto unpack = [](const v2i (&x)[2], float (&y)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t w = (uint32_t)x[e >> 2][(e >> 1) & 1];
            y[e] = (e & 1) ? __uint_as_float(w & 0xffff0000u) : __uint_as_float(w << 16);
        }
    };
    const uint8_t* const weight = !ROTATE || is_v ? nullptr : is_q ? a.q_weight : a.k_weight;
    float w8[8];
    if constexpr (ROTATE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w8[e] = 1.f;
        if (weight && a.weight_f32) {
            const v4f lo = *(const v4f*)(weight + 4 * d0), hi = *(const v4f*)(weight + 4 * d1);
#pragma unroll
            for (int e = 0; e < 8; ++e) w8[e] = e < 4 ? lo[e] : hi[e - 4];
        } else if (weight) {
            const v2i x[2] = {*(const v2i*)(weight + 2 * d0), *(const v2i*)(weight + 2 * d1)};
            unpack(x, w8);
        }
    }

    // ---- the tokens' positions and places, token i in lane i --------------------------------
    int64_t pos = 0;
    Place at{-1, 0};
    bool live = lane < tokens;
    {
        const int token = token0 + min(lane, tokens - 1);
        int b = 0;
        if (a.position_kind == kOfChunk) {
            Span s{0, 0};
            int64_t length = 0;
            if (!a.chunk.starts) {
                b = (int)div((uint32_t)token, a.chunk.div_each);
                s = span_of(a.chunk, b);
                length = a.chunk.lengths[b];
            } else if (a.chunk.batch <= 64) {
                // the sequences' starts and lengths, one to a lane, in one wait
                const bool has = lane < a.chunk.batch;
                const Span mine = has ? span_of(a.chunk, lane) : Span{0, 0};
                const int len = has ? a.chunk.lengths[lane] : 0;
                const int end = has ? mine.first + mine.count : INT32_MAX;
                b = -1;
                for (int i = 0; i < tokens; ++i) {
                    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= token0 + i));
                    if (n >= a.chunk.batch) continue;
                    const Span of{__builtin_amdgcn_readlane(mine.first, n), __builtin_amdgcn_readlane(mine.count, n)};
                    const int of_length = __builtin_amdgcn_readlane(len, n);
                    if (lane == i && token0 + i >= of.first && token0 + i < of.first + of.count) {
                        b = n;
                        s = of;
                        length = of_length;
                    }
                }
            } else {
                b = -1;
                for (int i = 0; i < tokens; ++i) {
                    const int found = sequence_of(a.chunk, token0 + i);
                    b = lane == i ? found : b;
                }
                if (live && b >= 0) {
                    s = span_of(a.chunk, b);
                    length = a.chunk.lengths[b];
                }
            }
            live = live && b >= 0;
            pos = length - s.count + (token - s.first);
        } else if (a.position_kind == kFromFirst) {
            pos = a.first_pos + token;
        } else {
            pos = a.position_kind == kInt64 ? ((const int64_t*)a.positions)[token] : ((const int32_t*)a.positions)[token];
        }
        if (PAGES && !is_q && live) at = place_of(a.pages, table_of(a.pages, b), pos);
    }
    const uint64_t live_mask = __builtin_amdgcn_ballot_w64(live);
    if (!live_mask) return;

    // ---- norms and rotation ---------------------------------------------------------------------
    if (ROTATE && !is_v) {
        float cosv[4] = {1.f, 1.f, 1.f, 1.f}, sinv[4] = {};
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            if (a.rotary_dim > 0 && (i == 0 || dt)) {
                const int64_t p = ((int64_t)__builtin_amdgcn_readlane((int)(pos >> 32), i) << 32) |
                                  (uint32_t)__builtin_amdgcn_readlane((int)pos, i);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double t = (double)p * a.turns[turning ? 4 * c + e : 0];
                    const float x = (float)(t - rint(t));  // revolutions in [-1/2, 1/2]
                    sinv[e] = __builtin_amdgcn_sinf(x) * a.amplitude;
                    cosv[e] = __builtin_amdgcn_cosf(x) * a.amplitude;
                }
            }
            float x[8];
            unpack(raw[i], x);
            if (weight) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
                sum = sum_over_lanes<LANES>(sum);
                const float inv = __builtin_amdgcn_rsqf(sum * (1.f / D) + a.norm_eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= inv * w8[e];
            }
            if (turning) {
                // half layout: pairs (e, e + 4); interleaved: (2 e, 2 e + 1)
                if (a.interleaved) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float u = x[2 * e], v = x[2 * e + 1];
                        x[2 * e] = fmaf(u, cosv[e], -v * sinv[e]);
                        x[2 * e + 1] = fmaf(v, cosv[e], u * sinv[e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float u = x[e], v = x[e + 4];
                        x[e] = fmaf(u, cosv[e], -v * sinv[e]);
                        x[e + 4] = fmaf(v, cosv[e], u * sinv[e]);
                    }
                }
            }
            const v4i z = to_bf16x8(x);
            raw[i][0] = v2i{z[0], z[1]};
            raw[i][1] = v2i{z[2], z[3]};
        }
    }

    // ---- rows of q, and of k and v without pages ---------------------------------------------------
    if (is_q || !PAGES) {
        const RowsOut out = is_q ? a.q_out : is_v ? a.v_out : a.k_out;
        uint8_t* dst = out.data;
        int64_t head_stride = out.head_stride;
        if (is_q && a.striped) {
            const uint32_t ch = div((uint32_t)token0, a.pages.div_interleave), round = div(ch, a.pages.div_pcp);
            const int64_t rank = ch - round * a.pages.pcp;
            const int64_t local = (int64_t)round * a.pages.interleave + (token0 - (int64_t)ch * a.pages.interleave);
            head_stride = (int64_t)a.local_q * D * 2;
            dst += (rank * a.num_q_heads * a.local_q + local) * D * 2;
        } else {
            dst += token0 * out.token_stride;
        }
        dst += head0 * head_stride;
        const int64_t step = dt ? out.token_stride : dh * head_stride, mine = r * head_stride + 2 * d0;
#pragma unroll
        for (int i = 0; i < NG; ++i, dst += step) {
            if (!there(i) || !((live_mask >> (dt ? i : 0)) & 1)) continue;
            *(v2i*)(dst + mine) = raw[i][0];
            *(v2i*)(dst + mine + 2 * (d1 - d0)) = raw[i][1];
        }
        return;
    }
    if constexpr (PAGES) {
        // ---- e4m3 codes of the k and v rows (of their bf16 values, rotated or not) -------------
        float scale[NG];
        uint32_t code[NG][2];
        if constexpr (FP8) {
            if (a.token_scales) {
                // a row's largest finite magnitude, as a bf16 pattern (ordered as the
                // integers are)
                uint32_t m[NG], any = 0;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    m[i] = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t u = (uint32_t)raw[i][e >> 1][e & 1] & 0x7fff7fffu;
                        m[i] = max(m[i], max(u >> 16, u & 0xffffu));
                    }
                    any = max(any, m[i]);
                }
                if (__builtin_amdgcn_ballot_w64(any >= 0x7f80u)) {
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        m[i] = 0;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t u = ((uint32_t)raw[i][e >> 2][(e >> 1) & 1] >> (16 * (e & 1))) & 0x7fffu;
                            m[i] = u < 0x7f80u ? max(m[i], u) : m[i];
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    m[i] = over_lanes<LANES>(m[i], [](uint32_t u, uint32_t v) { return max(u, v); });
                    scale[i] = fmaxf(__uint_as_float(m[i] << 16) / kFp8Max, kScaleFloor);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NG; ++i) scale[i] = is_v ? a.v_scale : a.k_scale;
            }
            // as torch rounds x / scale (cache::div_rn: the same quotient in fewer
            // instructions, where its range covers the scale)
            const bool covered = a.token_scales || cache::div_rn_covers(is_v ? a.v_scale : a.k_scale);
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                float x[8];
                unpack(raw[i], x);
                if (covered) {
                    const float rcp = 1.f / scale[i];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = cache::div_rn(x[e], scale[i], rcp);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = x[e] / scale[i];
                }
                code[i][0] = cache::e4m3_codes4(x[0], x[1], x[2], x[3]);
                code[i][1] = cache::e4m3_codes4(x[4], x[5], x[6], x[7]);
            }
        }
        const int row0 = (is_v ? a.num_kv_heads : 0) + head0;  // of the page's K and V blocks
        uint8_t* const heads_at = a.pool + row0 * a.pages.head_stride;
        const int64_t mine = r * a.pages.head_stride + d0 * (FP8 ? 1 : 2);
        float* const scales_at = a.token_scales + (int64_t)(row0 + r) * a.pages.block_size;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int page = __builtin_amdgcn_readlane(at.page, i), slot = __builtin_amdgcn_readlane(at.slot, i);
            if (page < 0 || !there(i)) continue;
            uint8_t* const dst = heads_at + page * a.pages.page_stride + (int64_t)slot * D * (FP8 ? 1 : 2) + mine;
            if constexpr (FP8) {
                *(uint32_t*)dst = code[i][0];
                *(uint32_t*)(dst + (d1 - d0)) = code[i][1];
                if (a.token_scales && c == 0)
                    scales_at[(int64_t)page * 2 * a.num_kv_heads * a.pages.block_size + slot] = scale[i];
            } else {
                *(v2i*)dst = raw[i][0];
                *(v2i*)(dst + 2 * (d1 - d0)) = raw[i][1];
            }
        }
    }
}

struct ReadArgs {
    Pages pages;
    const uint8_t* pool;
    const float* token_scales;
    uint8_t* k;  // [Hkv, num_tokens, D] bf16
    uint8_t* v;
    int64_t first_pos;
    int32_t num_tokens;
    float k_scale, v_scale;
};

// A thread takes 8 values of kReads tokens' rows of one head of K (grid z 0) or V
// (z 1): the table entries, then the rows and scales of all of them in flight.
// The stores are whole lines and bypass the caches: what is read back is more
// than they hold.  (131072 tokens, 2 heads at D 256 from e4m3 with token scales:
// 76 us, 5.3 TB/s; with two stores of half lines each 129 us.)
constexpr int kReads = 4;
template <int D>
constexpr int read_tokens() {  // tokens of a workgroup
    return kTokenThreads / (D / 8) * kReads;
}
template <int D, bool FP8>
__global__ void __launch_bounds__(kTokenThreads) cache_read_kernel(ReadArgs a) {
    constexpr int ROW = D * (FP8 ? 1 : 2), LANES = D / 8, AT_ONCE = kTokenThreads / LANES;
    const int c = threadIdx.x % LANES;
    const int64_t token0 = (int64_t)blockIdx.x * (AT_ONCE * kReads) + threadIdx.x / LANES;
    const int head = blockIdx.y, which = blockIdx.z, hr = which * a.pages.num_kv_heads + head;
    Place at[kReads];
#pragma unroll
    for (int u = 0; u < kReads; ++u) {
        const int64_t token = token0 + u * AT_ONCE;
        at[u] = token < a.num_tokens
                    ? place_of(a.pages, 0, a.first_pos + token)
                    : Place{-1, 0};
    }
    v4i raw[kReads];
    float scale[kReads];
#pragma unroll
    for (int u = 0; u < kReads; ++u) {
        raw[u] = v4i{0, 0, 0, 0};
        scale[u] = which ? a.v_scale : a.k_scale;
        if (at[u].page < 0) continue;
        const uint8_t* const src = a.pool + at[u].page * a.pages.page_stride + (int64_t)hr * a.pages.head_stride +
                                   (int64_t)at[u].slot * ROW + c * (ROW / LANES);
        if constexpr (FP8) {
            const v2i x = *(const v2i*)src;
            raw[u][0] = x[0];
            raw[u][1] = x[1];
            if (a.token_scales)
                scale[u] = a.token_scales[((int64_t)at[u].page * 2 * a.pages.num_kv_heads + hr) * a.pages.block_size +
                                          at[u].slot];
        } else {
            raw[u] = *(const v4i*)src;
        }
    }
    uint8_t* const out = which ? a.v : a.k;
#pragma unroll
    for (int u = 0; u < kReads; ++u) {
        const int64_t token = token0 + u * AT_ONCE;
        if (token >= a.num_tokens) continue;
        v4i x = raw[u];
        if constexpr (FP8) {
            float y[8];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(raw[u][w], false);
                const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(raw[u][w], true);
                y[4 * w] = lo[0] * scale[u];
                y[4 * w + 1] = lo[1] * scale[u];
                y[4 * w + 2] = hi[0] * scale[u];
                y[4 * w + 3] = hi[1] * scale[u];
            }
            x = to_bf16x8(y);
        }
        __builtin_nontemporal_store(x, (v4i*)(out + (((int64_t)head * a.num_tokens + token) * D + c * 8) * 2));
    }
}

}  // namespace chunk
}  // namespace pcpa
