// C ABI of the serving operators (include/pcp_attention_hip.h): rows of new
// tokens normed, rotated and written to the pages of their sequences
// (token_kernels.hpp), a cache read back, and the causal attention of a chunk
// over its sequences' caches (chunk_attention.hpp).
#include "chunk_attention.hpp"
#include "token_kernels.hpp"

namespace pcpa {
namespace chunk {
namespace {

constexpr int kCUs = 256;  // MI355X

// The parameters and the chunk, without the pointers that the kernels read.
int32_t check_chunk(const pcpa_params* p, const pcpa_chunk* c) {
    const int32_t st = pcpa_check_params(p);
    if (st != PCPA_OK) return st;
    if (!c) return PCPA_ERR_NULL_POINTER;
    if (c->interleave <= 0 || c->batch <= 0 || c->num_tokens < 0 || c->reserved != 0) return PCPA_ERR_BAD_SHAPE;
    if (!c->starts && c->num_tokens % c->batch) return PCPA_ERR_BAD_SHAPE;
    if (((uintptr_t)c->lengths | (uintptr_t)c->starts) & 3u) return PCPA_ERR_MISALIGNED;
    const int64_t capacity = (int64_t)p->pcp_size * p->max_local_blocks * p->block_size;
    // (256: room for the walk's rounding up)
    if (capacity > INT32_MAX - 256ll * p->pcp_size || (int64_t)p->pcp_size * c->interleave > INT32_MAX ||
        (int64_t)c->num_tokens * p->num_q_heads > INT32_MAX - 256)  // (256: a last row tile's)
        return PCPA_ERR_TOO_LARGE;
    return PCPA_OK;
}

// A launch has fewer than 2^32 threads.
bool too_many(int64_t blocks, int threads) { return blocks > (int64_t)(UINT32_MAX / threads); }

// The pages of a launch; the table holds `batch` sequences.
int32_t check_pages(const pcpa_params* p, const void* block_table, const void* kv_pages, const float* token_scales) {
    if (!block_table || !kv_pages) return PCPA_ERR_NULL_POINTER;
    if ((uintptr_t)kv_pages & 15u) return PCPA_ERR_MISALIGNED;
    if ((uintptr_t)block_table & ((p->flags & PCPA_FLAG_TABLE_INT64) ? 7u : 3u)) return PCPA_ERR_MISALIGNED;
    if ((uintptr_t)token_scales & 15u) return PCPA_ERR_MISALIGNED;
    if (token_scales && p->kv_dtype != PCPA_DTYPE_FP8_E4M3FN) return PCPA_ERR_BAD_DTYPE;
    if (token_scales && (p->k_scale != 1.f || p->v_scale != 1.f)) return PCPA_ERR_BAD_SCALE;
    return PCPA_OK;
}

Desc desc_of(const pcpa_chunk* c) {
    const int32_t each = c->starts ? 0 : c->num_tokens / c->batch;
    return Desc{c->lengths, c->starts, c->batch, c->num_tokens, each, make_div(each > 0 ? (uint32_t)each : 1u)};
}

Pages pages_of(const pcpa_params* p, int32_t interleave, const void* block_table) {
    const int64_t es = p->kv_dtype == PCPA_DTYPE_FP8_E4M3FN ? 1 : 2;
    Pages g{};
    g.table = (const int32_t*)block_table;
    g.table_shift = (p->flags & PCPA_FLAG_TABLE_INT64) ? 1 : 0;
    g.num_pages = p->num_pages;
    g.max_local_blocks = p->max_local_blocks;
    g.block_size = p->block_size;
    g.pcp = p->pcp_size;
    g.interleave = interleave;
    g.num_kv_heads = p->num_kv_heads;
    g.div_interleave = make_div((uint32_t)interleave);
    g.div_pcp = make_div((uint32_t)p->pcp_size);
    g.div_block = make_div((uint32_t)p->block_size);
    g.div_stride = make_div((uint32_t)p->pcp_size * (uint32_t)interleave);
    g.capacity = (int32_t)((int64_t)p->pcp_size * p->max_local_blocks * p->block_size);
    g.head_stride = (int64_t)p->block_size * p->head_dim * es;
    g.page_stride = 2 * (int64_t)p->num_kv_heads * g.head_stride;
    return g;
}

bool misaligned(const pcpa_rows* r) {
    return ((uintptr_t)r->data & 15u) || (r->token_stride & 7) || (r->head_stride & 7);
}
RowsIn rows_in(const pcpa_rows* r) { return RowsIn{(const uint8_t*)r->data, r->token_stride * 2, r->head_stride * 2}; }
RowsOut rows_out(const pcpa_rows* r) { return RowsOut{(uint8_t*)r->data, r->token_stride * 2, r->head_stride * 2}; }

// The square root's reciprocal takes no smaller numbers.
constexpr float kLeastEps = 0x1p-126f;

int32_t check_rotary(const pcpa_params* p, const pcpa_rotary* r) {
    if (!r) return PCPA_ERR_NULL_POINTER;
    if (r->rotary_dim < 0 || r->rotary_dim > p->head_dim || r->rotary_dim % 16) return PCPA_ERR_BAD_SHAPE;
    if (r->rotary_dim > 0 && !r->turns) return PCPA_ERR_NULL_POINTER;
    if (!isfinite(r->amplitude) || !isfinite(r->norm_eps) || !(r->norm_eps >= kLeastEps)) return PCPA_ERR_BAD_SCALE;
    const bool f32 = r->weight_dtype == PCPA_DTYPE_FP32;
    if (!f32 && r->weight_dtype != PCPA_DTYPE_BF16) return PCPA_ERR_BAD_DTYPE;
    if (((uintptr_t)r->q_weight | (uintptr_t)r->k_weight) & (f32 ? 15u : 7u)) return PCPA_ERR_MISALIGNED;
    if ((uintptr_t)r->turns & 7u) return PCPA_ERR_MISALIGNED;
    return PCPA_OK;
}

void set_rotary(TokenArgs& a, const pcpa_rotary* r) {
    a.rotary_dim = r->rotary_dim;
    a.interleaved = r->interleaved ? 1 : 0;
    a.amplitude = r->amplitude;
    a.norm_eps = r->norm_eps;
    a.turns = r->turns;
    a.q_weight = (const uint8_t*)r->q_weight;
    a.k_weight = (const uint8_t*)r->k_weight;
    a.weight_f32 = r->weight_dtype == PCPA_DTYPE_FP32;
}

template <bool ROTATE, bool PAGES, bool FP8, int NG>
const void* token_kernel_for(int head_dim) {
    return head_dim == 64    ? (const void*)token_kernel<64, ROTATE, PAGES, FP8, NG>
           : head_dim == 128 ? (const void*)token_kernel<128, ROTATE, PAGES, FP8, NG>
                             : (const void*)token_kernel<256, ROTATE, PAGES, FP8, NG>;
}

struct ReadKernel {
    const void* fn;
    int tokens;
};
template <bool FP8>
ReadKernel read_kernel_for(int d) {
    return d == 64    ? ReadKernel{(const void*)cache_read_kernel<64, FP8>, read_tokens<64>()}
           : d == 128 ? ReadKernel{(const void*)cache_read_kernel<128, FP8>, read_tokens<128>()}
                      : ReadKernel{(const void*)cache_read_kernel<256, FP8>, read_tokens<256>()};
}

template <bool ROTATE, bool PAGES, bool FP8>
int32_t launch_tokens(TokenArgs& a, const pcpa_params* p, hipStream_t stream) {
    a.num_q_heads = p->num_q_heads;
    a.num_kv_heads = p->num_kv_heads;
    const int rows = token_rows(p->head_dim), kv_groups = (p->num_kv_heads + rows - 1) / rows;
    const int q_groups = a.q.data ? (p->num_q_heads + rows - 1) / rows : 0, kinds = (a.k.data ? 1 : 0) + (a.v.data ? 1 : 0);
    const int64_t n = a.chunk.num_tokens;
    // four groups a wave once that fills half the GPU's 32 waves a CU
    const int ng = n * (q_groups + kinds * kv_groups) >= 4ll * 16 * kCUs ? 4 : 1;
    const int64_t q_parts = (q_groups + ng - 1) / ng, blocks_of_tokens = (n + ng - 1) / ng;
    const int64_t q_waves = n * q_parts, kv_waves = blocks_of_tokens * kv_groups;
    const int64_t waves = q_waves + kinds * kv_waves, per = kTokenThreads / 64, blocks = (waves + per - 1) / per;
    if (waves > INT32_MAX - per || too_many(blocks, kTokenThreads)) return PCPA_ERR_TOO_LARGE;
    a.waves = (int32_t)waves;
    a.q_waves = (int32_t)q_waves;
    a.q_parts = (int32_t)q_parts;
    a.kv_waves = (int32_t)kv_waves;
    a.token_blocks = (int32_t)blocks_of_tokens;
    a.div_q_parts = make_div((uint32_t)(q_parts > 0 ? q_parts : 1));
    a.div_token_blocks = make_div((uint32_t)blocks_of_tokens);
    void* args[] = {&a};
    const void* const fn = ng == 4 ? token_kernel_for<ROTATE, PAGES, FP8, 4>(p->head_dim)
                                   : token_kernel_for<ROTATE, PAGES, FP8, 1>(p->head_dim);
    return hipLaunchKernel(fn, dim3((unsigned)blocks), dim3(kTokenThreads), args, 0, stream) == hipSuccess
               ? PCPA_OK
               : PCPA_ERR_LAUNCH;
}

// pcpa_chunk_write, or with a rotation pcpa_chunk_prepare.
int32_t write_chunk(const pcpa_params* p, const pcpa_chunk* c, const pcpa_rotary* r, const pcpa_rows* q,
                    const pcpa_rows* k, const pcpa_rows* v, const pcpa_rows* q_out, const void* block_table,
                    void* kv_pages, float* token_scales, hipStream_t stream) {
    int32_t st = check_chunk(p, c);
    if (st != PCPA_OK) return st;
    if (r && (st = check_rotary(p, r)) != PCPA_OK) return st;
    if (!c->lengths || !k || !v || !k->data || !v->data) return PCPA_ERR_NULL_POINTER;
    if (r && (!q || !q_out || !q->data || !q_out->data)) return PCPA_ERR_NULL_POINTER;
    if ((st = check_pages(p, block_table, kv_pages, token_scales)) != PCPA_OK) return st;
    if (misaligned(k) || misaligned(v) || (r && (misaligned(q) || misaligned(q_out)))) return PCPA_ERR_MISALIGNED;
    if (c->num_tokens == 0) return PCPA_OK;
    TokenArgs a{};
    a.chunk = desc_of(c);
    a.pages = pages_of(p, c->interleave, block_table);
    a.k = rows_in(k);
    a.v = rows_in(v);
    if (r) {
        a.q = rows_in(q);
        a.q_out = rows_out(q_out);
        set_rotary(a, r);
    }
    a.position_kind = kOfChunk;
    a.pool = (uint8_t*)kv_pages;
    a.token_scales = token_scales;
    a.k_scale = p->k_scale;
    a.v_scale = p->v_scale;
    const bool fp8 = p->kv_dtype == PCPA_DTYPE_FP8_E4M3FN;
    return r ? (fp8 ? launch_tokens<true, true, true>(a, p, stream) : launch_tokens<true, true, false>(a, p, stream))
             : (fp8 ? launch_tokens<false, true, true>(a, p, stream) : launch_tokens<false, true, false>(a, p, stream));
}

// ---- attention ---------------------------------------------------------------

// A range of a walk has at least this many tiles (64 keys each).  Few rows: one
// token over 1024 to 8192 keys at D 256 took 16.4 us a call with 8, 14.5 with 4,
// 12.6 to 13.9 with 2; many: a range's start costs several tiles' time.  Short
// walks of few rows stay whole: 32 sequences of 512 tokens, 16 over 2 heads, took
// 8.6 us where ranges of two tiles took 10.9 (bf16 at D 64), 9.5 and 12.3 (e4m3 at
// D 128), 13.1 and 17.5 (e4m3 at D 256); one such sequence alone 8.2 and 9.1, 8.5
// and 9.1, 11.2 and 10.1, and at D 256 bf16 15.6 and 11.3, where 4 tiles are the
// most.
constexpr int kMinRangeFew = 2, kMinRangeMany = 8;

struct AttendKernel {
    const void* fn;
    int threads, rows, per_cu, min_range, whole;
};
// (a kernel with and without token scales has the same shape)
template <int D, bool FP8, int RT>
AttendKernel few_kernel(bool scaled) {
    using S = FewShape<D, FP8, RT>;
    return AttendKernel{scaled ? (const void*)attend_few_kernel<D, FP8, FP8, RT>
                               : (const void*)attend_few_kernel<D, FP8, false, RT>,
                        S::THREADS, S::ROWS, S::PER_CU, kMinRangeFew, S::WHOLE};
}
template <bool FP8, int RT>
AttendKernel few_kernel_for(int d, bool scaled) {
    return d == 64    ? few_kernel<64, FP8, RT>(scaled)
           : d == 128 ? few_kernel<128, FP8, RT>(scaled)
                      : few_kernel<256, FP8, RT>(scaled);
}

template <int D, bool FP8>
AttendKernel many_kernel(bool scaled) {
    using S = TileShape<D, FP8, false>;
    return AttendKernel{scaled ? (const void*)attend_many_kernel<D, FP8, FP8>
                               : (const void*)attend_many_kernel<D, FP8, false>,
                        S::THREADS, kRowsPerGroup, S::PAIR ? 1 : 2, kMinRangeMany, kMinRangeMany};
}
template <bool FP8>
AttendKernel many_kernel_for(int d, bool scaled) {
    return d == 64 ? many_kernel<64, FP8>(scaled) : d == 128 ? many_kernel<128, FP8>(scaled) : many_kernel<256, FP8>(scaled);
}

struct AttendPlan {
    AttendKernel kernel;
    int64_t items;        // workgroups of the launch
    bool ranges;          // walks may be cut into ranges
    int64_t part_ml, plans, bytes;
};

AttendPlan attend_plan(const pcpa_params* p, const pcpa_chunk* c, bool scaled = false) {
    AttendPlan w{};
    const int64_t group = p->num_q_heads / p->num_kv_heads;
    const int64_t sequences = c->num_tokens < c->batch ? c->num_tokens : c->batch;
    const bool narrow = sequences > 0 && c->num_tokens * group <= 16 * sequences;
    const bool fp8 = p->kv_dtype == PCPA_DTYPE_FP8_E4M3FN;
    const int d = p->head_dim;
    // Few rows: 32 a sequence and KV head on average, or so few in all that the
    // kernel for them runs on half of the CUs at most (8 new tokens of each of 8
    // sequences of 512, 32 over 2 heads at D 256, e4m3: 19.2 us, with the other 26.7;
    // on all of them, 128 of 128 tokens, 64 over 8 at D 128, bf16: 11.2 and 9.0)
    const int64_t few_tiles = c->num_tokens * group / 32 + sequences;
    const bool many = c->num_tokens * group > 32 * sequences && few_tiles * p->num_kv_heads > kCUs / 2;
    w.kernel = many  ? (fp8 ? many_kernel_for<true>(d, scaled) : many_kernel_for<false>(d, false))
               : fp8 ? (narrow ? few_kernel_for<true, 1>(d, scaled) : few_kernel_for<true, 2>(d, scaled))
                     : (narrow ? few_kernel_for<false, 1>(d, false) : few_kernel_for<false, 2>(d, false));
    // row tiles of one KV head: at most one that is not full per sequence
    const int64_t tiles = c->num_tokens * group / w.kernel.rows + sequences;
    const int64_t slots = (int64_t)kCUs * w.kernel.per_cu;
    const int64_t longest = (int64_t)p->pcp_size * p->max_local_blocks * p->block_size / kTileKeys;
    w.ranges = c->num_tokens > 0 && tiles * p->num_kv_heads < 4 * slots && longest > w.kernel.whole;
    // (the device sums the work in 32-bit floats, which may be less by 2^-24 for each
    // of a lane's sequences)
    w.items = tiles * p->num_kv_heads + (w.ranges ? slots + slots / 64 : 0);
    if (w.ranges) {
        const int64_t rows = w.items * w.kernel.rows;
        w.part_ml = rows * d * 4;
        w.plans = w.part_ml + rows * 8;
        w.bytes = w.plans + (int64_t)c->batch * sizeof(SequencePlan);
    }
    return w;
}

template <int D>
const void* merge_kernel_for(bool many) {
    return many ? (const void*)merge_many_ranges_kernel<D> : (const void*)merge_few_ranges_kernel<D>;
}

int32_t attend(const pcpa_params* p, const pcpa_chunk* c, const void* q, const void* kv_pages,
               const float* token_scales, const void* block_table, void* out, float* lse, void* workspace,
               int64_t workspace_bytes, hipStream_t stream) {
    int32_t st = check_chunk(p, c);
    if (st != PCPA_OK) return st;
    if (!c->lengths || !q || !out) return PCPA_ERR_NULL_POINTER;
    if ((st = check_pages(p, block_table, kv_pages, token_scales)) != PCPA_OK) return st;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15u) return PCPA_ERR_MISALIGNED;
    if ((uintptr_t)lse & 3u) return PCPA_ERR_MISALIGNED;
    const AttendPlan w = attend_plan(p, c, token_scales != nullptr);
    if (workspace_bytes < 0 || (w.bytes > 0 && (!workspace || workspace_bytes < w.bytes))) return PCPA_ERR_WORKSPACE;
    if (p->num_q_heads > 65535 || too_many(w.items, w.kernel.threads)) return PCPA_ERR_TOO_LARGE;
    if (c->num_tokens == 0) return PCPA_OK;
    AttendArgs a{};
    a.chunk = desc_of(c);
    a.pages = pages_of(p, c->interleave, block_table);
    a.q = (const uint8_t*)q;
    a.pool = (const uint8_t*)kv_pages;
    a.token_scales = token_scales;
    a.out = (uint8_t*)out;
    a.lse = lse;
    a.num_q_heads = p->num_q_heads;
    a.group = p->num_q_heads / p->num_kv_heads;
    a.rows_log2 = __builtin_ctz(w.kernel.rows);
    a.div_group = make_div((uint32_t)a.group);
    a.div_heads = make_div((uint32_t)p->num_kv_heads);
    a.max_items = (int32_t)w.items;
    a.slots = kCUs * w.kernel.per_cu;
    a.min_range = w.kernel.min_range;
    a.whole = w.kernel.whole;
    a.score_scale = p->softmax_scale * p->k_scale * kLog2e;
    a.v_scale = p->v_scale;
    if (w.ranges) {
        a.part_o = (float*)workspace;
        a.part_ml = (v2f*)((uint8_t*)workspace + w.part_ml);
        a.plans = (SequencePlan*)((uint8_t*)workspace + w.plans);
    }
    void* args[] = {&a};
    if (hipLaunchKernel(w.kernel.fn, dim3((unsigned)w.items), dim3(w.kernel.threads), args, 0, stream) != hipSuccess)
        return PCPA_ERR_LAUNCH;
    if (!w.ranges) return PCPA_OK;
    // Few rows have many ranges each: 16 waves to a row, as long as the GPU has
    // room for all rows at once
    const bool many = (int64_t)c->num_tokens * p->num_q_heads <= 2 * kCUs;
    const void* const merge = p->head_dim == 64    ? merge_kernel_for<64>(many)
                              : p->head_dim == 128 ? merge_kernel_for<128>(many)
                                                   : merge_kernel_for<256>(many);
    const int at_once = 256 / (p->head_dim / 4);
    const dim3 grid(c->num_tokens, many ? p->num_q_heads : (p->num_q_heads + at_once - 1) / at_once,
                    many ? p->head_dim / kMergeParts : 1);
    return hipLaunchKernel(merge, grid, dim3(many ? 1024 : 256), args, 0, stream) == hipSuccess ? PCPA_OK
                                                                                               : PCPA_ERR_LAUNCH;
}

}  // namespace
}  // namespace chunk
}  // namespace pcpa

extern "C" {

int32_t pcpa_rotate(const pcpa_params* p, const pcpa_chunk* c, const pcpa_rotary* r, const void* positions,
                    int32_t position_bits, int64_t first_pos, const pcpa_rows* q, const pcpa_rows* k,
                    const pcpa_rows* v, const pcpa_rows* q_out, const pcpa_rows* k_out, const pcpa_rows* v_out,
                    int32_t striped, void* stream) {
    using namespace pcpa::chunk;
    int32_t st = check_chunk(p, c);
    if (st != PCPA_OK) return st;
    if ((st = check_rotary(p, r)) != PCPA_OK) return st;
    if (!q || !k || !q_out || !k_out || !q->data || !k->data || !q_out->data || !k_out->data)
        return PCPA_ERR_NULL_POINTER;
    if ((v == nullptr) != (v_out == nullptr) || (v && (!v->data || !v_out->data))) return PCPA_ERR_NULL_POINTER;
    if (position_bits != kOfChunk && position_bits != kFromFirst && position_bits != kInt32 && position_bits != kInt64)
        return PCPA_ERR_BAD_SHAPE;
    const bool given = position_bits > 0;
    if (given != (positions != nullptr) || (position_bits == kOfChunk && !c->lengths)) return PCPA_ERR_NULL_POINTER;
    if (position_bits == kFromFirst && (c->batch != 1 || first_pos < 0 || first_pos > INT64_MAX - c->num_tokens))
        return PCPA_ERR_BAD_SHAPE;
    if (striped && (position_bits == kOfChunk || c->num_tokens % (p->pcp_size * c->interleave)))
        return PCPA_ERR_BAD_SHAPE;
    if (misaligned(q) || misaligned(k) || misaligned(k_out) || ((uintptr_t)q_out->data & 15u) ||
        (!striped && misaligned(q_out)) || (v && (misaligned(v) || misaligned(v_out))))
        return PCPA_ERR_MISALIGNED;
    if ((uintptr_t)positions & (position_bits == kInt64 ? 7u : 3u)) return PCPA_ERR_MISALIGNED;
    if (c->num_tokens == 0) return PCPA_OK;
    TokenArgs a{};
    a.chunk = desc_of(c);
    a.pages = pages_of(p, c->interleave, nullptr);
    a.q = rows_in(q);
    a.k = rows_in(k);
    a.q_out = rows_out(q_out);
    a.k_out = rows_out(k_out);
    if (v) {
        a.v = rows_in(v);
        a.v_out = rows_out(v_out);
    }
    a.striped = striped ? 1 : 0;
    a.local_q = c->num_tokens / p->pcp_size;
    a.position_kind = position_bits;
    a.positions = positions;
    a.first_pos = first_pos;
    set_rotary(a, r);
    return launch_tokens<true, false, false>(a, p, (hipStream_t)stream);
}

int32_t pcpa_chunk_write(const pcpa_params* p, const pcpa_chunk* c, const pcpa_rows* k, const pcpa_rows* v,
                         const void* block_table, void* kv_pages, float* token_scales, void* stream) {
    return pcpa::chunk::write_chunk(p, c, nullptr, nullptr, k, v, nullptr, block_table, kv_pages, token_scales,
                                    (hipStream_t)stream);
}

int32_t pcpa_chunk_prepare(const pcpa_params* p, const pcpa_chunk* c, const pcpa_rotary* r, const pcpa_rows* q,
                           const pcpa_rows* k, const pcpa_rows* v, const pcpa_rows* q_out, const void* block_table,
                           void* kv_pages, float* token_scales, void* stream) {
    if (!r) return PCPA_ERR_NULL_POINTER;
    return pcpa::chunk::write_chunk(p, c, r, q, k, v, q_out, block_table, kv_pages, token_scales,
                                    (hipStream_t)stream);
}

int32_t pcpa_cache_read(const pcpa_params* p, int32_t interleave, int64_t first_pos, int32_t num_tokens,
                        const void* block_table, const void* kv_pages, const float* token_scales, void* k, void* v,
                        void* stream) {
    using namespace pcpa::chunk;
    const pcpa_chunk c{interleave, 1, num_tokens, 0, nullptr, nullptr};
    int32_t st = check_chunk(p, &c);
    if (st != PCPA_OK) return st;
    if (first_pos < 0 || first_pos > INT64_MAX - num_tokens) return PCPA_ERR_BAD_SHAPE;
    if (!k || !v) return PCPA_ERR_NULL_POINTER;
    if ((st = check_pages(p, block_table, kv_pages, token_scales)) != PCPA_OK) return st;
    if (((uintptr_t)k | (uintptr_t)v) & 15u) return PCPA_ERR_MISALIGNED;
    if (num_tokens == 0) return PCPA_OK;
    ReadArgs a{};
    a.pages = pages_of(p, interleave, block_table);
    a.pool = (const uint8_t*)kv_pages;
    a.token_scales = token_scales;
    a.k = (uint8_t*)k;
    a.v = (uint8_t*)v;
    a.first_pos = first_pos;
    a.num_tokens = num_tokens;
    a.k_scale = p->k_scale;
    a.v_scale = p->v_scale;
    const bool fp8 = p->kv_dtype == PCPA_DTYPE_FP8_E4M3FN;
    const ReadKernel kernel = fp8 ? read_kernel_for<true>(p->head_dim) : read_kernel_for<false>(p->head_dim);
    const int64_t blocks = ((int64_t)num_tokens + kernel.tokens - 1) / kernel.tokens;
    if (p->num_kv_heads > 65535 || too_many(blocks, kTokenThreads)) return PCPA_ERR_TOO_LARGE;
    void* args[] = {&a};
    return hipLaunchKernel(kernel.fn, dim3((unsigned)blocks, p->num_kv_heads, 2), dim3(kTokenThreads), args, 0,
                           (hipStream_t)stream) == hipSuccess
               ? PCPA_OK
               : PCPA_ERR_LAUNCH;
}

int64_t pcpa_chunk_workspace_bytes(const pcpa_params* p, const pcpa_chunk* c) {
    const int32_t st = pcpa::chunk::check_chunk(p, c);
    return st == PCPA_OK ? pcpa::chunk::attend_plan(p, c).bytes : st;
}

int32_t pcpa_chunk_attention(const pcpa_params* p, const pcpa_chunk* c, const void* q, const void* kv_pages,
                             const float* token_scales, const void* block_table, void* out, float* lse,
                             void* workspace, int64_t workspace_bytes, void* stream) {
    return pcpa::chunk::attend(p, c, q, kv_pages, token_scales, block_table, out, lse, workspace, workspace_bytes,
                               (hipStream_t)stream);
}

}  // extern "C"
