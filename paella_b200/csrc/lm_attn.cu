// Attention of one new token for every sequence of a batch that shares a prefix, over a paged cache.
//
//   out[b][h] = sum_j softmax_j(scale * q[b][h] . k_j) v_j   over the prefix's tokens and the sequence's own
#include <cuda.h>

#include <cmath>

#include "lm.cuh"

namespace pb {
namespace {

__device__ uint32_t g_attn_flag;

struct AttnArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t *prefix_pages, *block_table, *own_lens;
    int64_t q_stride, q_head, out_stride, out_head, page_stride, token_stride, head_stride, table_stride, n_pages;
    int batch, q_heads, group, D, page, prefix_len, max_own;
    float scale;
};

// A warp takes a query head of a sequence: lane l holds values 4 l to 4 l + 3 of the head, every key's product is a sum over the
// lanes, and the softmax's maximum and sum run along.
template <typename T>
__global__ void __launch_bounds__(128) attn_kernel(AttnArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row < (int64_t)a.batch * a.q_heads) {
        const int b = (int)(row / a.q_heads), h = (int)(row % a.q_heads), d = 4 * lane;
        const bool mine = d < a.D;
        const float to_log2 = a.scale * 1.4426950408889634f;
        float q[4] = {}, acc[4] = {}, top = -INFINITY, sum = 0.f;
        if (mine)
            for (int j = 0; j < 4; ++j) q[j] = lm_to_f<T>(static_cast<const T*>(a.q)[b * a.q_stride + h * a.q_head + d + j]);
        int own = a.max_own > 0 ? a.own_lens[b] : 0;
        if (own < 0 || own > a.max_own) {
            if (lane == 0) atomicExch(&g_attn_flag, kFlagLmLength);
            own = own < 0 ? 0 : a.max_own;
        }
        for (int i = 0; i < a.prefix_len + own; ++i) {
            const bool ahead = i < a.prefix_len;
            const int j = ahead ? i : i - a.prefix_len;
            const int page = ahead ? a.prefix_pages[j / a.page] : a.block_table[b * a.table_stride + j / a.page];
            const bool real = page >= 0 && page < a.n_pages;
            if (!real && lane == 0) atomicExch(&g_attn_flag, kFlagLmPage);
            const int64_t at = page * a.page_stride + (j % a.page) * a.token_stride + (h / a.group) * a.head_stride + d;
            float s = 0.f;
            if (real && mine)
                for (int e = 0; e < 4; ++e) s = fmaf(q[e], lm_to_f<T>(static_cast<const T*>(a.k)[at + e]), s);
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            s *= to_log2;
            const float next = fmaxf(top, s);
            const float keep = top == -INFINITY ? 0.f : exp2f(top - next), p = s == -INFINITY ? 0.f : exp2f(s - next);
            sum = sum * keep + p;
            for (int e = 0; e < 4; ++e) acc[e] = acc[e] * keep + (real && mine ? p * lm_to_f<T>(static_cast<const T*>(a.v)[at + e]) : 0.f);
            top = next;
        }
        if (mine)
            for (int e = 0; e < 4; ++e)
                static_cast<T*>(a.out)[b * a.out_stride + h * a.out_head + d + e] = lm_from_f<T>(a.prefix_len + own == 0 ? 0.f : acc[e] / sum);
    }
    if (nf) nf->end(job_id);
}

int check_attn(const pb_prefix_attn_params* p) {
    const char* who = "pb_prefix_attn";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(p->dtype == PB_BF16 || p->dtype == PB_F16, "%s: dtype %d (PB_BF16 or PB_F16)", who, p->dtype);
    PB_REQUIRE(p->batch >= 0 && p->q_heads >= 1 && p->kv_heads >= 1 && p->q_heads % p->kv_heads == 0 && p->q_heads <= 65536, "%s: batch %d, %d query heads, %d key heads", who, p->batch, p->q_heads, p->kv_heads);
    PB_REQUIRE(p->head_dim >= 8 && p->head_dim <= 128 && p->head_dim % 8 == 0, "%s: head_dim %d (a multiple of 8, 8 to 128)", who, p->head_dim);
    PB_REQUIRE(p->page_size >= 8 && p->page_size % 8 == 0, "%s: page_size %d (a multiple of 8)", who, p->page_size);
    PB_REQUIRE(p->n_pages >= 0 && p->n_pages <= 0x7fffffff, "%s: %lld pages", who, (long long)p->n_pages);
    PB_REQUIRE(p->prefix_len >= 0 && p->prefix_len <= (1 << 30) && p->max_own_len >= 0 && p->max_own_len <= (1 << 30), "%s: prefix of %d tokens, at most %d own", who, p->prefix_len, p->max_own_len);
    PB_REQUIRE(p->max_blocks >= 0 && p->max_own_len <= (int64_t)p->max_blocks * p->page_size, "%s: %d own tokens do not fit %d pages of %d", who, p->max_own_len, p->max_blocks, p->page_size);
    PB_REQUIRE(p->scale == p->scale && fabsf(p->scale) <= 3.402823466e38f, "%s: scale is not finite", who);
    PB_REQUIRE(p->page_stride % 8 == 0 && p->token_stride % 8 == 0 && p->head_stride % 8 == 0, "%s: strides of the cache are multiples of 8", who);
    PB_REQUIRE(p->q_stride % 8 == 0 && p->q_head_stride % 8 == 0, "%s: rows of q start on 16 bytes", who);
    if (p->batch > 0) {
        PB_REQUIRE(p->q && p->out && p->k_cache && p->v_cache, "%s: NULL buffer", who);
        PB_REQUIRE(aligned(p->q, 16) && aligned(p->k_cache, 16) && aligned(p->v_cache, 16) && aligned(p->out, 2), "%s: q and the cache must be 16-byte aligned", who);
        PB_REQUIRE(p->prefix_len == 0 || (p->prefix_pages && aligned(p->prefix_pages, 4)), "%s: a prefix needs its pages", who);
        PB_REQUIRE(p->max_own_len == 0 || (p->block_table && p->own_lens && aligned(p->block_table, 4) && aligned(p->own_lens, 4)), "%s: own tokens need block_table and own_lens", who);
    }
    return PB_OK;
}

}  // namespace

uint32_t* lm_attn_error_flag_ptr() {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_attn_flag) != cudaSuccess) { cudaGetLastError(); return nullptr; }
    return (uint32_t*)p;
}

}  // namespace pb

using namespace pb;

extern "C" {

int pb_prefix_attn_info(const pb_prefix_attn_params* p, pb_launch_info* out) {
    const int rc = check_attn(p);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_prefix_attn_info: NULL out");
    memset(out, 0, sizeof(*out));
    const int64_t blocks = ceil_div<int64_t>((int64_t)p->batch * p->q_heads, 4);
    PB_REQUIRE(blocks <= 0x7fffffff, "pb_prefix_attn: too many rows for one launch");
    out->num_blocks = blocks > 0 ? (uint32_t)blocks : 1u;
    out->threads_per_block = 128;
    out->regs_per_thread = p->dtype == PB_BF16 ? lm_regs(attn_kernel<__nv_bfloat16>) : lm_regs(attn_kernel<__half>);
    const uint64_t seen = (uint64_t)p->prefix_len + (uint64_t)p->batch * p->max_own_len;
    out->flops = 4ull * p->head_dim * p->q_heads * p->batch * ((uint64_t)p->prefix_len + p->max_own_len);
    out->bytes = p->batch ? 4ull * p->head_dim * (p->kv_heads * seen + (uint64_t)p->batch * p->q_heads) : 0;
    return PB_OK;
}

int pb_prefix_attn_launch(const pb_prefix_attn_params* p, void* stream, uint32_t job_id, void* notifier) {
    pb_launch_info li;
    const int rc = pb_prefix_attn_info(p, &li);
    if (rc != PB_OK) return rc;
    const AttnArgs a = {p->q, p->k_cache, p->v_cache, p->out, p->prefix_pages, p->block_table, p->own_lens, p->q_stride, p->q_head_stride, p->out_stride, p->out_head_stride,
                        p->page_stride, p->token_stride, p->head_stride, p->table_stride, p->n_pages, p->batch, p->q_heads, p->q_heads / p->kv_heads, p->head_dim, p->page_size,
                        p->prefix_len, p->max_own_len, p->scale};
    FinishedBlockNotifier* nf = (FinishedBlockNotifier*)notifier;
    const dim3 grid(li.num_blocks), block(128);
    if (p->dtype == PB_BF16) return lm_launch("pb_prefix_attn", attn_kernel<__nv_bfloat16>, grid, block, 0, (cudaStream_t)stream, 1, a, job_id, nf);
    return lm_launch("pb_prefix_attn", attn_kernel<__half>, grid, block, 0, (cudaStream_t)stream, 1, a, job_id, nf);
}

}  // extern "C"
