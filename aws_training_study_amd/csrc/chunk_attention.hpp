// Causal attention of new tokens over the paged caches of their sequences.
#pragma once

#include "chunk_common.hpp"

namespace pcpa {
namespace chunk {

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
    float score_scale;  // softmax_scale * k_scale * log2(e)
    float v_scale;
};

template <bool FP8>
__device__ __forceinline__ float cached(const uint8_t* row, int d) {
    if constexpr (FP8) return __builtin_amdgcn_cvt_f32_fp8(row[d], 0);
    return bf16_bits_to_f32(((const uint16_t*)row)[d]);
}

// One wave per (row, Q head): scores of 64 keys at a time, a key to a lane, with
// a running maximum m and sum l (s in log2 units, p = 2^(s - m)); then the lanes
// take D / 64 values of the output each and go through the 64 probabilities.
template <int D, bool FP8>
__global__ void __launch_bounds__(64) attend_rows_kernel(AttendArgs a) {
    constexpr int PER = D / 64, ES = FP8 ? 1 : 2;
    const int lane = threadIdx.x;
    const int token = blockIdx.x, head = blockIdx.y, kv = head / a.group;
    const int b = sequence_of(a.chunk, token);
    if (b < 0) return;
    const Span span = span_of(a.chunk, b);
    const int64_t pos = (int64_t)a.chunk.lengths[b] - span.count + (token - span.first);
    const int64_t table = table_of(a.pages, b);
    const int64_t at = (int64_t)token * a.num_q_heads + head;
    const uint16_t* const q = (const uint16_t*)(a.q + at * D * 2);
    const int64_t k_off = kv * a.pages.head_stride, v_off = (a.pages.num_kv_heads + kv) * a.pages.head_stride;
    const int64_t keys = pos + 1 < a.pages.capacity ? pos + 1 : a.pages.capacity;
    float m = -INFINITY, l = 0.f, o[PER] = {};
    for (int64_t base = 0; base < keys; base += 64) {
        const Place p = base + lane < keys ? place_of(a.pages, table, base + lane) : Place{-1, 0};
        float s = -INFINITY, vs = a.v_scale;
        if (p.page >= 0) {
            const uint8_t* const row = a.pool + p.page * a.pages.page_stride + k_off + (int64_t)p.slot * D * ES;
            float dot = 0.f;
            for (int d = 0; d < D; ++d) dot = fmaf(bf16_bits_to_f32(q[d]), cached<FP8>(row, d), dot);
            if (a.token_scales) {
                const float* const sc = a.token_scales + ((int64_t)p.page * 2 * a.pages.num_kv_heads + kv) *
                                                             a.pages.block_size + p.slot;
                dot *= sc[0];
                vs *= sc[(int64_t)a.pages.num_kv_heads * a.pages.block_size];
            }
            s = dot * a.score_scale;
        }
        float top = s;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
        const float next = fmaxf(m, top);
        const float weight = p.page >= 0 ? exp2f(s - next) : 0.f;
        float sum = weight;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off);
        const float keep = m == -INFINITY ? 0.f : exp2f(m - next);
        l = l * keep + sum;
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] *= keep;
        m = next;
        for (int k = 0; k < 64; ++k) {
            const int page = __shfl(p.page, k), slot = __shfl(p.slot, k);
            const float w = __shfl(weight * vs, k);
            if (page < 0) continue;
            const uint8_t* const row = a.pool + page * a.pages.page_stride + v_off + (int64_t)slot * D * ES;
#pragma unroll
            for (int i = 0; i < PER; ++i) o[i] = fmaf(w, cached<FP8>(row, lane * PER + i), o[i]);
        }
    }
    const bool seen = m != -INFINITY;
    __bf16* const out = (__bf16*)(a.out + at * D * 2);
#pragma unroll
    for (int i = 0; i < PER; ++i) out[lane * PER + i] = (__bf16)(seen ? o[i] / l : 0.f);
    if (a.lse && lane == 0) a.lse[at] = seen ? m * kLn2 + logf(l) : -INFINITY;
}

}  // namespace chunk
}  // namespace pcpa
