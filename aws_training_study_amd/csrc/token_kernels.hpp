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
    int32_t rows_per_token;  // heads of q, k and v that are there
    int32_t waves_per_token, groups_per_wave;
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

__device__ __forceinline__ float weight_at(const uint8_t* w, int d, int f32) {
    return f32 ? ((const float*)w)[d] : bf16_bits_to_f32(((const uint16_t*)w)[d]);
}

__device__ __forceinline__ v4i to_bf16x8(const float (&x)[8]) {
    v4i r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __bf16 lo = (__bf16)x[2 * i], hi = (__bf16)x[2 * i + 1];
        r[i] = (int)((uint32_t)__builtin_bit_cast(uint16_t, lo) | ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16));
    }
    return r;
}
__device__ __forceinline__ void from_bf16x8(const v4i& r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = bf16_bits_to_f32((uint32_t)r[i] & 0xffffu);
        x[2 * i + 1] = bf16_bits_to_f32((uint32_t)r[i] >> 16);
    }
}

// A wave takes one token and `groups_per_wave` groups of its rows (heads of Q,
// then K, then V): a row's D values lie 8 to a lane in D / 8 neighbouring
// lanes, 64 / (D / 8) rows at a time.  The angles of a lane's pairs depend on
// the token and the lane alone, so they are formed once for all its rows.
//   ROTATE  norms and rotation of the q and k rows
//   PAGES   k and v rows go into the pages (FP8: e4m3 ones), else to k_out and
//           v_out
// Everything is HBM bound: 2 bytes read and 1 or 2 written per value.
template <int D, bool ROTATE, bool PAGES, bool FP8>
__global__ void __launch_bounds__(kTokenThreads) token_kernel(TokenArgs a) {
    constexpr int LANES = D / 8, ROWS = 64 / LANES;  // lanes of a row, rows at a time
    const int lane = threadIdx.x & 63, c = lane % LANES;
    const int wid = __builtin_amdgcn_readfirstlane((blockIdx.x * kTokenThreads + threadIdx.x) >> 6);
    const int token = wid / a.waves_per_token, part = wid - token * a.waves_per_token;
    if (token >= a.chunk.num_tokens) return;

    // ---- the token's position and place --------------------------------------
    int64_t pos = 0;
    int b = 0;
    if (a.position_kind == kOfChunk) {
        b = sequence_of(a.chunk, token);
        if (b < 0) return;
        const Span s = span_of(a.chunk, b);
        pos = (int64_t)a.chunk.lengths[b] - s.count + (token - s.first);
    } else if (a.position_kind == kFromFirst) {
        pos = a.first_pos + token;
    } else {
        pos = a.position_kind == kInt64 ? ((const int64_t*)a.positions)[token] : ((const int32_t*)a.positions)[token];
    }
    Place at{-1, 0};
    if constexpr (PAGES) at = place_of(a.pages, table_of(a.pages, b), pos);

    // ---- cosines and sines of this lane's pairs ---------------------------------
    // half layout: lane c holds values 8c .. 8c + 7, pairs i = those modulo R / 2;
    // interleaved: pairs 4c .. 4c + 3
    const int chunks = ROTATE ? a.rotary_dim / 8 : 0;  // lanes of a row that rotate
    const bool turning = ROTATE && c < chunks;
    const bool second = turning && !a.interleaved && c >= chunks / 2;
    const int partner = lane + (second ? -chunks / 2 : chunks / 2);
    float cosv[8], sinv[8];
    if constexpr (ROTATE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = a.interleaved ? 4 * c + e / 2 : 8 * (second ? c - chunks / 2 : c) + e;
            float x = 0.f, y = 0.f;
            if (turning) {
                const double t = (double)pos * a.turns[i];
                const float r = (float)(t - rint(t));  // revolutions in [-1/2, 1/2]
                sincospif(2.f * r, &y, &x);
                x *= a.amplitude;
                y *= a.amplitude;
            }
            cosv[e] = x;
            // (a, b) -> (a cos - b sin, b cos + a sin): the sign of the partner's part
            sinv[e] = a.interleaved ? ((e & 1) ? y : -y) : (second ? y : -y);
        }
    }

    for (int g = 0; g < a.groups_per_wave; ++g) {
        const int row = (part * a.groups_per_wave + g) * ROWS + lane / LANES;
        if ((part * a.groups_per_wave + g) * ROWS >= a.rows_per_token) break;  // wave-uniform
        // which head of q, k or v
        const int nq = a.q.data ? a.num_q_heads : 0, nk = a.k.data ? a.num_kv_heads : 0;
        const bool there = row < a.rows_per_token;
        const bool is_q = there && row < nq, is_k = there && !is_q && row < nq + nk, is_v = there && !is_q && !is_k;
        const int head = is_q ? row : is_k ? row - nq : row - nq - nk;
        const RowsIn in = is_q ? a.q : is_k ? a.k : a.v;
        v4i raw{0, 0, 0, 0};
        if (there) raw = *(const v4i*)(in.data + token * in.token_stride + head * in.head_stride + c * 16);
        float x[8];
        from_bf16x8(raw, x);
        if constexpr (ROTATE) {
            const uint8_t* const w = is_q ? a.q_weight : is_k ? a.k_weight : nullptr;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
            for (int off = 1; off < LANES; off <<= 1) sum += __shfl_xor(sum, off);
            if (w) {
                const float inv = 1.f / sqrtf(sum * (1.f / D) + a.norm_eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * weight_at(w, 8 * c + e, a.weight_f32);
            }
            float y[8];  // the other value of each pair
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = __shfl(x[e], partner);
            }
            if (turning && (is_q || is_k)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = fmaf(x[e], cosv[e], y[e] * sinv[e]);
            }
            // v's rows and those without norm and rotation keep their bits
            if (is_q || is_k) raw = to_bf16x8(x);
        }
        if (is_q || (!PAGES && there)) {
            uint8_t* dst;
            if (is_q && a.striped) {
                const int il = a.pages.interleave, pcp = a.pages.pcp;
                const int ch = token / il, round = ch / pcp, rank = ch - round * pcp;
                const int local = round * il + (token - ch * il);
                dst = a.q_out.data + (((int64_t)rank * a.num_q_heads + head) * a.local_q + local) * D * 2;
            } else {
                const RowsOut out = is_q ? a.q_out : is_k ? a.k_out : a.v_out;
                dst = out.data + token * out.token_stride + head * out.head_stride;
            }
            *(v4i*)(dst + c * 16) = raw;
        }
        if constexpr (PAGES) {
            // (the row's bf16 values are what is quantised, rotated or not)
            const bool stored = (is_k || is_v) && at.page >= 0;
            const int64_t offset = at.page * a.pages.page_stride +
                                   (int64_t)(is_v ? a.num_kv_heads + head : head) * a.pages.head_stride +
                                   (int64_t)at.slot * D * (FP8 ? 1 : 2) + c * (FP8 ? 8 : 16);
            if constexpr (FP8) {
                from_bf16x8(raw, x);
                float scale = is_v ? a.v_scale : a.k_scale;
                if (a.token_scales) {
                    uint32_t m = 0;  // the largest finite magnitude's bits
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t u = __float_as_uint(x[e]) & 0x7fffffffu;
                        m = u < 0x7f800000u ? max(m, u) : m;
                    }
#pragma unroll
                    for (int off = 1; off < LANES; off <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off));
                    scale = fmaxf(__uint_as_float(m) / kFp8Max, kScaleFloor);
                    if (stored && c == 0)
                        a.token_scales[((int64_t)at.page * 2 * a.num_kv_heads + (is_v ? a.num_kv_heads : 0) + head) *
                                           a.pages.block_size + at.slot] = scale;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = x[e] / scale;
                if (stored)
                    *(v2i*)(a.pool + offset) = v2i{(int)cache::e4m3_codes4(x[0], x[1], x[2], x[3]),
                                                   (int)cache::e4m3_codes4(x[4], x[5], x[6], x[7])};
            } else if (stored) {
                *(v4i*)(a.pool + offset) = raw;
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

// Thread: 8 values of one (token, head) row of K (grid z 0) or V (z 1).
template <int D, bool FP8>
__global__ void __launch_bounds__(kTokenThreads) cache_read_kernel(ReadArgs a) {
    constexpr int LANES = D / 8;
    const int64_t id = (int64_t)blockIdx.x * kTokenThreads + threadIdx.x;
    const int token = (int)(id / LANES), c = (int)(id % LANES);
    if (token >= a.num_tokens) return;
    const int head = blockIdx.y, which = blockIdx.z;
    const Place at = place_of(a.pages, 0, a.first_pos + token);
    v4i out{0, 0, 0, 0};
    if (at.page >= 0) {
        const int hr = which * a.pages.num_kv_heads + head;
        const uint8_t* const src = a.pool + at.page * a.pages.page_stride + (int64_t)hr * a.pages.head_stride;
        if constexpr (FP8) {
            const v2i raw = *(const v2i*)(src + (int64_t)at.slot * D + c * 8);
            const float scale =
                a.token_scales ? a.token_scales[((int64_t)at.page * 2 * a.pages.num_kv_heads + hr) *
                                                    a.pages.block_size + at.slot]
                               : which ? a.v_scale : a.k_scale;
            float x[8];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(raw[w], false);
                const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(raw[w], true);
                x[4 * w] = lo[0] * scale;
                x[4 * w + 1] = lo[1] * scale;
                x[4 * w + 2] = hi[0] * scale;
                x[4 * w + 3] = hi[1] * scale;
            }
            out = to_bf16x8(x);
        } else {
            out = *(const v4i*)(src + ((int64_t)at.slot * D + c * 8) * 2);
        }
    }
    *(v4i*)((which ? a.v : a.k) + (((int64_t)head * a.num_tokens + token) * D + c * 8) * 2) = out;
}

}  // namespace chunk
}  // namespace pcpa
