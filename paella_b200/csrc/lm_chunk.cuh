// Attention of chunks of new tokens over a paged cache (pb_chunk_attn): part of lm_attn.cu, whose exponentials and products it uses.
//
//   out[r][h] = sum_j softmax_j(scale * q[r][h] . k_j) v_j   over the tokens that row r sees: up to its own position, with a window the last of them
#pragma once

namespace pb {
namespace {

struct ChunkArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t *block_table, *starts, *lens;
    int64_t q_stride, q_head, out_stride, out_head, page_stride, token_stride, head_stride, table_stride;
    int batch, tokens, q_heads, kv_heads, group, D, page, n_pages, max_new, max_len, window;
    float scale;
};

// A sequence's rows and length, as they count.
struct ChunkSeq {
    int start, rows, first, len;       // its first row, its rows, the first one's position, its tokens in the cache
};
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkArgs& a, int b, bool tell) {
    const int s0 = a.starts[b], s1 = a.starts[b + 1], l = a.lens[b];
    const int start = min(max(s0, 0), a.tokens), end = min(max(s1, start), a.tokens), len = min(max(l, 0), a.max_len);
    const int n = end - start;
    if (tell && (start != s0 || end != s1 || len != l || n > a.max_new)) atomicExch(&g_attn_flag, kFlagLmLength);
    return {start, min(n, a.max_new), len - n, len};
}

// A warp a row and head.
template <typename T>
__global__ void __launch_bounds__(128) chunk_simple_kernel(const __grid_constant__ ChunkArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (item < (int64_t)a.batch * a.max_new * a.q_heads) {          // (none of 0: no quotient by it either)
        const int b = (int)(item / ((int64_t)a.max_new * a.q_heads));
        const int i = (int)(item / a.q_heads % a.max_new), h = (int)(item % a.q_heads);
        const ChunkSeq s = chunk_seq(a, b, lane == 0 && i == 0 && h == 0);
        if (i < s.rows) {
            const T* q = static_cast<const T*>(a.q) + (s.start + i) * a.q_stride + h * a.q_head;
            float x[4], o[4] = {}, m = -INFINITY, l = 0.f;
            for (int e = 0; e < 4; ++e) x[e] = lane + 32 * e < a.D ? lm_to_f<T>(q[lane + 32 * e]) * a.scale * kLog2e : 0.f;
            const int p = s.first + i;
            for (int j = a.window ? max(0, p - a.window + 1) : 0; j <= p; ++j) {
                const int page = a.block_table[b * a.table_stride + j / a.page];
                const bool there = page >= 0 && page < a.n_pages;
                if (!there && lane == 0) atomicExch(&g_attn_flag, kFlagLmPage);
                const int64_t at = page * a.page_stride + (j % a.page) * a.token_stride + h / a.group * a.head_stride;
                float z = 0.f, v[4] = {};
                for (int e = 0; e < 4; ++e)
                    if (there && lane + 32 * e < a.D) {
                        z = fmaf(x[e], lm_to_f<T>(static_cast<const T*>(a.k)[at + lane + 32 * e]), z);
                        v[e] = lm_to_f<T>(static_cast<const T*>(a.v)[at + lane + 32 * e]);
                    }
                for (int d = 16; d > 0; d >>= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
                if (z > m) {
                    const float keep = ex2(m - z);
                    l *= keep;
                    for (int e = 0; e < 4; ++e) o[e] *= keep;
                    m = z;
                }
                const float w = ex2(z - m);
                l += w;
                for (int e = 0; e < 4; ++e) o[e] = fmaf(lm_to_f<T>(lm_from_f<T>(w)), v[e], o[e]);
            }
            T* out = static_cast<T*>(a.out) + (s.start + i) * a.out_stride + h * a.out_head;
            for (int e = 0; e < 4; ++e)
                if (lane + 32 * e < a.D) out[lane + 32 * e] = lm_from_f<T>(p < 0 ? 0.f : o[e] / l);
        }
    }
    if (nf) nf->end(job_id);
}

int check_chunk(const pb_chunk_attn_params* p, ChunkArgs& a) {
    const char* who = "pb_chunk_attn";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(p->dtype == PB_BF16 || p->dtype == PB_F16, "%s: dtype %d (PB_BF16 or PB_F16)", who, p->dtype);
    PB_REQUIRE(p->batch >= 0 && p->batch <= 1 << 24 && p->tokens >= 0 && p->q_heads >= 1 && p->kv_heads >= 1 && p->q_heads % p->kv_heads == 0 && p->q_heads <= 65536, "%s: batch %d, %d tokens, %d query heads, %d key heads", who,
               p->batch, p->tokens, p->q_heads, p->kv_heads);
    PB_REQUIRE(p->head_dim >= 8 && p->head_dim <= 128 && p->head_dim % 8 == 0, "%s: head_dim %d (a multiple of 8, 8 to 128)", who, p->head_dim);
    PB_REQUIRE(p->page_size >= 8 && p->page_size % 8 == 0 && p->page_size <= 1 << 24, "%s: page_size %d (a multiple of 8, at most 2^24)", who, p->page_size);
    PB_REQUIRE(p->n_pages >= 0 && p->n_pages <= 0x7fffffff, "%s: %lld pages", who, (long long)p->n_pages);
    PB_REQUIRE(p->max_new >= 0 && p->max_len >= 0 && p->max_len <= 1 << 30 && p->window >= 0, "%s: at most %d new tokens of %d, window %d", who, p->max_new, p->max_len, p->window);
    PB_REQUIRE(p->max_blocks >= 0 && p->max_len <= (int64_t)p->max_blocks * p->page_size, "%s: %d tokens do not fit %d pages of %d", who, p->max_len, p->max_blocks, p->page_size);
    PB_REQUIRE(fabsf(p->scale) <= 2e38f, "%s: scale is not finite, or above 2e38", who);        // (which in powers of two is finite, too)
    PB_REQUIRE(p->page_stride % 8 == 0 && p->token_stride % 8 == 0 && p->head_stride % 8 == 0 && p->page_stride > 0 && p->token_stride > 0 && p->head_stride > 0, "%s: strides of the cache are positive multiples of 8", who);
    PB_REQUIRE(p->q_stride % 8 == 0 && p->q_head_stride % 8 == 0, "%s: rows of q start on 16 bytes", who);
    PB_REQUIRE(rows_apart(p->tokens, p->out_stride, p->head_dim) && rows_apart(p->q_heads, p->out_head_stride, p->head_dim), "%s: rows of out overlap (strides %lld, %lld)", who, (long long)p->out_stride, (long long)p->out_head_stride);
    if (p->batch > 0 && p->tokens > 0 && p->max_new > 0) {
        PB_REQUIRE(p->q && p->out && p->starts && p->lens, "%s: NULL buffer", who);
        PB_REQUIRE(p->max_len == 0 || (p->k_cache && p->v_cache && p->block_table && p->n_pages > 0), "%s: a NULL cache or block_table, or a cache without pages", who);
        PB_REQUIRE(aligned(p->q, 16) && aligned(p->k_cache, 16) && aligned(p->v_cache, 16) && aligned(p->out, 2), "%s: q and the cache must be 16-byte aligned", who);
        PB_REQUIRE(aligned(p->block_table, 4) && aligned(p->starts, 4) && aligned(p->lens, 4), "%s: a table is not aligned to its elements", who);
    }
    memset(&a, 0, sizeof(a));
    a.q = p->q; a.k = p->k_cache; a.v = p->v_cache; a.out = p->out; a.block_table = p->block_table; a.starts = p->starts; a.lens = p->lens;
    a.q_stride = p->q_stride; a.q_head = p->q_head_stride; a.out_stride = p->out_stride; a.out_head = p->out_head_stride;
    a.page_stride = p->page_stride; a.token_stride = p->token_stride; a.head_stride = p->head_stride; a.table_stride = p->table_stride;
    a.batch = p->tokens > 0 && p->max_new > 0 ? p->batch : 0; a.tokens = p->tokens; a.q_heads = p->q_heads; a.kv_heads = p->kv_heads; a.group = p->q_heads / p->kv_heads; a.D = p->head_dim;
    a.page = p->page_size; a.n_pages = (int)p->n_pages; a.max_new = p->max_new < p->tokens ? p->max_new : p->tokens; a.max_len = p->max_len; a.window = p->window; a.scale = p->scale;
    return PB_OK;
}

}  // namespace
}  // namespace pb
