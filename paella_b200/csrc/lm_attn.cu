// Attention of one new token for every sequence of a batch that shares a prefix, over a paged cache.
//
//   out[b][h] = sum_j softmax_j(scale * q[b][h] . k_j) v_j   over the prefix's tokens and the sequence's own
//
// Two kernels.  The prefix is one matrix for the whole batch: the rows of all sequences' query heads that share a key head
// meet it in tiles of 128 rows x 128 keys on the tensor cores (prefix_kernel), and its keys and values are read once for 256
// rows.  A sequence's own tokens meet only its `group` query rows: that is bound by reading them, a block for each sequence and
// key head (own_kernel), which also joins the parts of the prefix with its own.  Softmax runs along with the sums: each part
// has its rows' maximum m, sum l and unscaled O, and parts join as sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i.
#include <cuda.h>

#include <cmath>

#include "lm.cuh"
#include "umma.cuh"

namespace pb {
namespace {

__device__ uint32_t g_attn_flag;

struct AttnArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t *prefix_pages, *block_table, *own_lens;
    int64_t q_stride, q_head, out_stride, out_head, page_stride, token_stride, head_stride, table_stride;
    int batch, group, D, page, n_pages, prefix_len, max_own;
    float scale;
    // the prefix's split
    int row_tiles, pairs, splits, key_tiles, box_rows;
    float* part_o;             // [kv_heads][pairs][splits][2][128][DP]
    float2* part_ml;           // the same without DP: (m, l)
    // own tokens
    int kv_heads, row_groups, ranks, early, out_vec;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kLog2e = 1.4426950408889634f;
// A row's maximum is followed only once it has grown by 2^8: until then the values are up to 2^8 times too large, which fp32 sums and the
// 16-bit values' exponents hold, and the accumulator need not be rescaled.
constexpr float kSlack = 8.f;
// fp16 has few exponents below 1: its values are scaled up by 2^5 (2^13 with the slack; the sums with them).
template <typename T> __device__ __forceinline__ constexpr float p_shift() { return sizeof(T) == 2 && std::is_same<T, __half>::value ? 5.f : 0.f; }

// ---- the prefix ----------------------------------------------------------------------------------------------
// A block takes a range of the prefix's keys for one key head and a pair of row tiles, or, where the last row tile is alone, that tile with its
// even and odd key tiles as a pair.  Warps 0-3 and 4-7: softmax of one of the pair each, a row a thread; warp 8 loads keys and values, warp 9 issues the
// products: S = Q K^T of the one tile runs while the other's softmax does.  S (128 columns) becomes P in place (64 columns of 16-bit pairs), the A
// operand of O += P V.  Tensor memory: S0 S1 O0 O1.
template <int DP> struct PrefixShape {
    static constexpr uint32_t tile = 128 * DP * 2;                   // bytes of 128 rows
    static constexpr int stages = DP == 128 ? 5 : 10;                // tiles of keys or values in flight
    static constexpr uint32_t smem = 1024 + (2 + stages) * tile;     // two tiles of queries in front of them
};

template <typename T, int DP>
__global__ void __launch_bounds__(320, 1) prefix_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int kBlocks = DP / 64, kStages = PrefixShape<DP>::stages;
    constexpr uint32_t kTile = PrefixShape<DP>::tile, kBlock = 128 * 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_full[kStages], s_empty[kStages], s_scores[2], s_probs[2], s_done[2], s_q;
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_abort;
    const uint32_t q_smem = (smem_u32(smem_raw) + 1023u) & ~1023u, ring = q_smem + 2 * kTile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int pair = blockIdx.x % a.pairs, split = (blockIdx.x / a.pairs) % a.splits, kvh = blockIdx.x / (a.pairs * a.splits);
    const int kt0 = (int)((int64_t)a.key_tiles * split / a.splits), n = (int)((int64_t)a.key_tiles * (split + 1) / a.splits) - kt0;
    const bool two = 2 * pair + 1 < a.row_tiles;      // two row tiles; otherwise one, its key tiles dealt to both softmax groups
    const int jobs = two ? 2 * n : n;                 // job i: softmax group i & 1, key tile i / 2 or i

    if (warp == 9) {
        tcgen05_alloc(smem_u32(&s_tmem), 512);
        tcgen05_relinquish();
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_scores[i]), 1);
            mbar_init(smem_u32(&s_probs[i]), 4);
            mbar_init(smem_u32(&s_done[i]), 1);
        }
        mbar_init(smem_u32(&s_q), 256);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = s_tmem;
    griddep_wait();
    griddep_launch();          // own_kernel, which reads nothing that precedes this launch in the stream but what has ended here

    if (warp == 8) {
        // Keys and values in the order in which the products ask for them.
        for (int pos = 0; pos < 2 * n; ++pos) {
            bool values;
            int t;
            if (two) { values = pos & 1; t = pos >> 1; }
            else if (pos == 0) { values = false; t = 0; }
            else if (pos == 2 * n - 1) { values = true; t = n - 1; }
            else if (pos & 1) { values = false; t = (pos + 1) >> 1; }
            else { values = true; t = (pos - 2) >> 1; }
            const int st = pos % kStages, use = pos / kStages;
            const int key0 = (kt0 + t) * 128, left = min(128, a.prefix_len - key0), boxes = (left + a.box_rows - 1) / a.box_rows;
            const bool mine = lane < boxes * kBlocks;
            const int box = lane / kBlocks, blk = lane % kBlocks, key = key0 + box * a.box_rows;
            int page = 0;
            if (mine) {
                page = __ldcg(a.prefix_pages + key / a.page);
                if (page < 0 || page >= a.n_pages) {
                    atomicExch(&g_attn_flag, kFlagLmPage);
                    page = a.n_pages;                 // outside of the map: zeros
                }
            }
            if (use > 0 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_empty[st]), (use - 1) & 1, &s_abort, &g_attn_flag, kFlagLmWait))) break;
            const uint32_t bar = smem_u32(&s_full[st]);
            if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(boxes * kBlocks * a.box_rows * 128));
            __syncwarp();
            if (mine) tma_load_4d(ring + st * kTile + blk * kBlock + box * a.box_rows * 128, values ? &vmap : &kmap, blk * 64, key % a.page, kvh, page, bar);
        }
    } else if (warp == 9) {
        constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t idesc_s = (1u << 4) | kType | ((128u >> 3) << 17) | ((128u >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | kType | (1u << 16) | (((uint32_t)DP >> 3) << 17) | ((128u >> 4) << 24);
        bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_q), 0, &s_abort, &g_attn_flag, kFlagLmWait));
        const auto stage_ready = [&](int pos) {
            return __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[pos % kStages]), (pos / kStages) & 1, &s_abort, &g_attn_flag, kFlagLmWait));
        };
        const auto scores = [&](int i) {
            const int g = i & 1, t = two ? i >> 1 : i, pos = two ? 2 * t : t == 0 ? 0 : 2 * t - 1;
            if (!stage_ready(pos)) return false;
            tcgen05_fence_after();
            const uint64_t dq = umma_desc_sw128(q_smem + (two ? g * kTile : 0)), dk = umma_desc_sw128(ring + (pos % kStages) * kTile);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    const uint64_t at = (uint64_t)((k >> 2) * (kBlock >> 4) + (k & 3) * 2);
                    tcgen05_mma_bf16(tmem + g * 128, dq + at, dk + at, idesc_s, k > 0);
                }
                tcgen05_commit(smem_u32(&s_scores[g]));
                if (!two || g == 1) tcgen05_commit(smem_u32(&s_empty[pos % kStages]));
            }
            __syncwarp();
            return true;
        };
        for (int i = 0; i < 2 && ok; ++i)
            if (i < jobs) ok = scores(i);
        for (int i = 0; i < jobs && ok; ++i) {
            const int g = i & 1, t = two ? i >> 1 : i, pos = two ? 2 * t + 1 : t == n - 1 ? 2 * n - 1 : 2 * t + 2;
            ok = stage_ready(pos);
            if (!ok) break;
            const uint32_t v_smem = ring + (pos % kStages) * kTile;
            const int left = a.prefix_len - (kt0 + t) * 128;
            if (left < 128 && (!two || g == 0)) {
                // Rows behind the last token: their P is zero, and so is what they hold, which nobody wrote or which may be NaNs.
                for (int c = lane; c < (128 - left) * 8 * kBlocks; c += 32) {
                    const int blk = c / ((128 - left) * 8), at = c % ((128 - left) * 8);
                    st_shared_v4(v_smem + blk * kBlock + left * 128 + at * 16, 0, 0, 0, 0);
                }
                fence_proxy_async();
                __syncwarp();
            }
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_probs[g]), (i >> 1) & 1, &s_abort, &g_attn_flag, kFlagLmWait));
            if (!ok) break;
            tcgen05_fence_after();
            const uint64_t dv = umma_desc_sw128_mn(v_smem, kBlock);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 8; ++k) tcgen05_mma_f16_ts(tmem + 256 + g * DP, tmem + g * 128 + k * 8, dv + (uint64_t)(k * (2048 >> 4)), idesc_o, i > 1 || k > 0);
                if (!two || g == 1) tcgen05_commit(smem_u32(&s_empty[pos % kStages]));
                if (i + 2 >= jobs) tcgen05_commit(smem_u32(&s_done[g]));
            }
            __syncwarp();
            if (i + 2 < jobs) ok = scores(i + 2);
        }
    } else {
        const int g = warp >> 2, in_tile = (warp & 3) * 32 + lane, rows = a.batch * a.group;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                       // this warp's lanes of tensor memory
        const int row = (2 * pair + (two ? g : 0)) * 128 + in_tile;
        const bool live_warp = row - lane < rows;
        if (two || g == 0) {
            const T* src = nullptr;
            if (row < rows) src = static_cast<const T*>(a.q) + (int64_t)(row / a.group) * a.q_stride + (int64_t)(kvh * a.group + row % a.group) * a.q_head;
            const uint32_t dst = q_smem + g * kTile + in_tile * 128, flip = a.scale < 0.f ? 0x80008000u : 0u;      // |scale| from here on
#pragma unroll
            for (int c = 0; c < DP / 8; ++c) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (row < rows && 8 * c < a.D) v = __ldcg(reinterpret_cast<const uint4*>(src + 8 * c));
                st_shared_v4(dst + (c >> 3) * kBlock + (((c & 7) ^ (in_tile & 7)) << 4), v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
            }
        }
        fence_proxy_async();
        mbar_arrive(smem_u32(&s_q));

        const float c = fmaxf(fabsf(a.scale) * kLog2e, 1e-38f);                  // (a scale of 0 must not meet the infinities of masked keys)
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        int done = 0;
        for (int i = g; i < jobs; i += 2, ++done) {
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_scores[g]), done & 1, &s_abort, &g_attn_flag, kFlagLmWait));
            if (!ok) break;
            if (live_warp) {
                tcgen05_fence_after();
                const int left = a.prefix_len - (kt0 + (two ? i >> 1 : i)) * 128;
                const uint32_t ts = tmem + lanes + g * 128;
                uint32_t s[128];
#pragma unroll
                for (int j = 0; j < 4; ++j) tcgen05_ld32(ts + 32 * j, s + 32 * j);
                tcgen05_wait_ld();
                if (left < 128) {
#pragma unroll
                    for (int j = 0; j < 128; ++j)
                        if (j >= left) s[j] = 0xff800000u;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 128; ++j) top[j & 3] = fmaxf(top[j & 3], __uint_as_float(s[j]));
                const float next = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                if (done == 0) {
                    m = next;
                } else if (__any_sync(0xffffffffu, (next - m) * c > kSlack)) {   // (a NaN difference, -inf to -inf, is no growth)
                    const float keep = next == m ? 1.f : ex2((m - next) * c);
                    const uint32_t to = tmem + lanes + 256 + g * DP;
#pragma unroll 1
                    for (int j = 0; j < DP; j += 32) {
                        uint32_t o[32];
                        tcgen05_ld32(to + j, o);
                        tcgen05_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tcgen05_st32(to + j, o);
                    }
                    l *= keep;
                    m = next;
                }
                const float base = m == -INFINITY ? 0.f : m * c - p_shift<T>();
                float sum[4] = {};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t p[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float x = ex2(fmaf(__uint_as_float(s[64 * h + 2 * j]), c, -base)), y = ex2(fmaf(__uint_as_float(s[64 * h + 2 * j + 1]), c, -base));
                        sum[j & 3] += x + y;
                        p[j] = lm_pack2<T>(x, y);
                    }
                    tcgen05_st32(ts + 32 * h, p);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tcgen05_wait_st();
                tcgen05_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_probs[g]));
        }
        // this block's part of the row
        const int64_t part = ((int64_t)((int64_t)kvh * a.pairs + pair) * a.splits + split) * 2 + g;
        if (ok && done > 0) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_done[g]), 0, &s_abort, &g_attn_flag, kFlagLmWait));
        if (ok && live_warp) {
            tcgen05_fence_after();
            if (row < rows) a.part_ml[part * 128 + in_tile] = make_float2(m == -INFINITY ? m : m * c, l);
            if (done > 0) {
                float* dst = a.part_o + (part * 128 + in_tile) * DP;
#pragma unroll 1
                for (int j = 0; j < DP; j += 32) {
                    uint32_t o[32];
                    tcgen05_ld32(tmem + lanes + 256 + g * DP + j, o);
                    tcgen05_wait_ld();
                    if (row < rows) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(dst + j + e) = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                    }
                }
            }
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (s_abort) {             // copies in flight end before their shared memory does
        const unsigned long long t0 = globaltimer_ns();
        for (int i = 0; i < 100000 && globaltimer_ns() - t0 < 50000; ++i) __nanosleep(500);
    }
    if (warp == 9) {
        tcgen05_fence_after();
        tcgen05_dealloc(tmem, 512);
    }
}

// ---- own tokens, and the parts together ------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// A block (or a cluster of `ranks` blocks, each a range of the tokens) takes 8 NT query rows of one sequence and key head.  A warp takes 16 tokens at a
// time, straight from global memory into the registers that the products read: the order of a head's values within a product's 16 is free as
// long as both operands have the same, and so is the order of O's rows, hence each lane's 16 bytes are as they lie.
//   S^T[token][row] = K Q^T:  lane (g, c) = (lane / 4, lane % 4) holds 8 values at 8 c of every 32 of tokens g and g + 8
//   O^T[value][row] = V^T P^T: 8 values at 8 g of every 64 of tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9
// P^T comes out of S^T with a transposition of 8 x 8 in the warp.
template <typename T, int DP, int NT>
__global__ void __launch_bounds__(128) own_kernel(const __grid_constant__ AttnArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    constexpr int R = 8 * NT, KB = DP / 32, VB = DP / 64;
    __shared__ __align__(16) float s_o[4][R][DP];
    __shared__ __align__(8) float2 s_ml[4][R];
    if (!a.early) griddep_wait();
    if (nf) nf->start(job_id);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int rank = blockIdx.x % a.ranks;
    int unit = blockIdx.x / a.ranks;
    const int zg = unit % a.row_groups;
    unit /= a.row_groups;
    const int kvh = unit % a.kv_heads, b = unit / a.kv_heads;
    const int row0 = zg * R, rows = b < a.batch ? min(R, a.group - row0) : 0;
    int own = 0;
    if (b < a.batch && a.max_own > 0) {
        own = __ldcg(a.own_lens + b);
        if (own < 0 || own > a.max_own) {
            if (threadIdx.x == 0) atomicExch(&g_attn_flag, kFlagLmLength);
            own = own < 0 ? 0 : a.max_own;
        }
    }
    const int chunks = (own + 15) / 16, first = (int)((int64_t)chunks * rank / a.ranks) + warp, last = (int)((int64_t)chunks * (rank + 1) / a.ranks);
    float o[VB][4][NT][4] = {};
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f;
    if (first < last) {
        uint4 q[NT][KB];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < KB; ++i) {
                q[t][i] = make_uint4(0, 0, 0, 0);
                if (t * 8 + g < rows && 32 * i + 8 * c < a.D)
                    q[t][i] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.q_stride + (int64_t)(kvh * a.group + row0 + t * 8 + g) * a.q_head + 32 * i + 8 * c));
            }
        const int32_t* table = a.block_table + b * a.table_stride;
        const int64_t head = (int64_t)kvh * a.head_stride;
        // where the 8 tokens at 16 chunk + 8 half lie (a page holds a multiple of 8), or -1: zeros
        const auto where = [&](int chunk, int half) -> int64_t {
            const int token = 16 * chunk + 8 * half;
            if (token >= own) return -1;
            const int at = token / a.page, page = __ldcg(table + at);
            if (page < 0 || page >= a.n_pages) {
                if (lane == 0) atomicExch(&g_attn_flag, kFlagLmPage);
                return -1;
            }
            return page * a.page_stride + (token - at * a.page) * a.token_stride + head;
        };
        uint4 k[KB][2], v[VB][4];
        const auto load_k = [&](int chunk, int64_t lo, int64_t hi) {
            const int token = 16 * chunk + g;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t base = h ? hi : lo;
                const bool there = base >= 0 && token + 8 * h < own;
                const T* src = static_cast<const T*>(a.k) + base + g * a.token_stride + 8 * c;
#pragma unroll
                for (int i = 0; i < KB; ++i) {
                    k[i][h] = make_uint4(0, 0, 0, 0);
                    if (there && 32 * i + 8 * c < a.D) k[i][h] = __ldcg(reinterpret_cast<const uint4*>(src + 32 * i));
                }
            }
        };
        const auto load_v = [&](int chunk, int64_t lo, int64_t hi) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int within = 2 * c + (e & 1);
                const int64_t base = e >> 1 ? hi : lo;
                const bool there = base >= 0 && 16 * chunk + 8 * (e >> 1) + within < own;
                const T* src = static_cast<const T*>(a.v) + base + within * a.token_stride + 8 * g;
#pragma unroll
                for (int i = 0; i < VB; ++i) {
                    v[i][e] = make_uint4(0, 0, 0, 0);
                    if (there && 64 * i + 8 * g < a.D) v[i][e] = __ldcg(reinterpret_cast<const uint4*>(src + 64 * i));
                }
            }
        };
        const float scale = a.scale * kLog2e;
        int64_t lo = where(first, 0), hi = where(first, 1);
        load_k(first, lo, hi);
        load_v(first, lo, hi);
        for (int chunk = first; chunk < last; chunk += 4) {
            const int next = chunk + 4;
            int64_t nlo = -1, nhi = -1;
            if (next < last) { nlo = where(next, 0); nhi = where(next, 1); }
            float s[NT][4] = {};
#pragma unroll
            for (int i = 0; i < KB; ++i) {
                const uint32_t a0[4] = {k[i][0].x, k[i][1].x, k[i][0].y, k[i][1].y}, a1[4] = {k[i][0].z, k[i][1].z, k[i][0].w, k[i][1].w};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    mma_16x8x16<T>(s[t], a0, q[t][i].x, q[t][i].y);
                    mma_16x8x16<T>(s[t], a1, q[t][i].z, q[t][i].w);
                }
            }
            if (next < last) load_k(next, nlo, nhi);
            const bool in0 = 16 * chunk + g < own, in1 = 16 * chunk + g + 8 < own;
            float up[NT][2];
            bool grown = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    s[t][j] = in0 ? s[t][j] * scale : -INFINITY;
                    s[t][2 + j] = in1 ? s[t][2 + j] * scale : -INFINITY;
                    float x = fmaxf(s[t][j], s[t][2 + j]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    up[t][j] = fmaxf(m[t][j], x);
                    grown |= up[t][j] - m[t][j] > kSlack;                // (from -inf, too)
                }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float keep = up[t][j] == m[t][j] ? 1.f : ex2(m[t][j] - up[t][j]);
                        m[t][j] = up[t][j];
                        l[t][j] *= keep;
#pragma unroll
                        for (int i = 0; i < VB; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) { o[i][e][t][j] *= keep; o[i][e][t][2 + j] *= keep; }
                    }
            }
            uint32_t p0[NT], p1[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float b0 = m[t][0] == -INFINITY ? 0.f : m[t][0] - p_shift<T>(), b1 = m[t][1] == -INFINITY ? 0.f : m[t][1] - p_shift<T>();
                const float x0 = ex2(s[t][0] - b0), x1 = ex2(s[t][1] - b1), y0 = ex2(s[t][2] - b0), y1 = ex2(s[t][3] - b1);
                l[t][0] += x0 + y0;
                l[t][1] += x1 + y1;
                p0[t] = transpose_8x8(lm_pack2<T>(x0, x1));
                p1[t] = transpose_8x8(lm_pack2<T>(y0, y1));
            }
#pragma unroll
            for (int i = 0; i < VB; ++i) {
                const uint32_t* w0 = &v[i][0].x; const uint32_t* w1 = &v[i][1].x; const uint32_t* w2 = &v[i][2].x; const uint32_t* w3 = &v[i][3].x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t av[4] = {__byte_perm(w0[e], w1[e], 0x5410), __byte_perm(w0[e], w1[e], 0x7632), __byte_perm(w2[e], w3[e], 0x5410), __byte_perm(w2[e], w3[e], 0x7632)};
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma_16x8x16<T>(o[i][e][t], av, p0[t], p1[t]);
                }
            }
            if (next < last) load_v(next, nlo, nhi);
        }
    }
    // this warp's part: (m, l) and O of its rows, values 64 i + 8 g + 2 e and + 1
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float x = l[t][j];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            const int row = 8 * t + 2 * c + j;
            if (g == 0) s_ml[warp][row] = make_float2(m[t][j], x);
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(&s_o[warp][row][64 * i + 8 * g + 2 * e]) = make_float2(o[i][e][t][j], o[i][e][t][2 + j]);
        }
    if (a.early) griddep_wait();                                          // the prefix's parts
    griddep_launch();
    if (a.ranks > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();

    // The parts joined: a float4 of a row for `lanes` neighbouring threads, which deal the parts out among themselves.
    const int items = rows * (DP / 4);
    int lanes = 1;
    while (lanes < 32 && items * lanes * 2 <= 128 * a.ranks) lanes *= 2;
    const int sub = threadIdx.x & (lanes - 1);
    for (int base = 0; base < items; base += 128 * a.ranks / lanes) {
        const int item = base + (rank * 128 + threadIdx.x) / lanes;
        const bool real = item < items;
        const int row = real ? item / (DP / 4) : 0, col = real ? item % (DP / 4) * 4 : 0;
        // the prefix's parts of this row
        const int flat = b * a.group + row0 + row, tile = flat >> 7, pair = tile >> 1, in_tile = flat & 127;
        const bool two = 2 * pair + 1 < a.row_tiles;
        const int64_t part0 = ((int64_t)kvh * a.pairs + pair) * a.splits * 2 + (two ? tile & 1 : 0);
        const int step = two ? 2 : 1, ahead = a.prefix_len > 0 ? (two ? a.splits : 2 * a.splits) : 0, mine = own > 0 ? 4 * a.ranks : 0;
        float top = -INFINITY;
        for (int i = sub; real && i < ahead + mine; i += lanes) {
            const int w = i - ahead;
            const float2 ml = i < ahead ? __ldcg(a.part_ml + (part0 + (int64_t)i * step) * 128 + in_tile) : ld_cluster_f2(cluster_addr(smem_u32(&s_ml[w & 3][row]), w >> 2));
            top = fmaxf(top, ml.x);
        }
        for (int k = lanes >> 1; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll 4
        for (int i = sub; real && i < ahead + mine; i += lanes) {
            const int w = i - ahead;
            const int64_t part = (part0 + (int64_t)i * step) * 128 + in_tile;
            const float2 ml = i < ahead ? __ldcg(a.part_ml + part) : ld_cluster_f2(cluster_addr(smem_u32(&s_ml[w & 3][row]), w >> 2));
            if (ml.x == -INFINITY && ml.y == 0.f) continue;               // no token, or none with a finite score: O may not have been written
            const float4 x = i < ahead ? __ldcg(reinterpret_cast<const float4*>(a.part_o + part * DP + col)) : ld_cluster_f4(cluster_addr(smem_u32(&s_o[w & 3][row][col]), w >> 2));
            const float f = ex2(ml.x - top);
            sum = fmaf(f, ml.y, sum);
            acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y); acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w);
        }
        for (int k = lanes >> 1; k > 0; k >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, k);
            acc.x += __shfl_xor_sync(0xffffffffu, acc.x, k); acc.y += __shfl_xor_sync(0xffffffffu, acc.y, k);
            acc.z += __shfl_xor_sync(0xffffffffu, acc.z, k); acc.w += __shfl_xor_sync(0xffffffffu, acc.w, k);
        }
        if (!real || sub != 0 || col >= a.D) continue;
        if (a.prefix_len + own == 0) acc = make_float4(0.f, 0.f, 0.f, 0.f), sum = 1.f;
        T* dst = static_cast<T*>(a.out) + b * a.out_stride + (int64_t)(kvh * a.group + row0 + row) * a.out_head + col;
        const float inv = 1.f / sum;
        if (a.out_vec) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(lm_pack2<T>(acc.x * inv, acc.y * inv), lm_pack2<T>(acc.z * inv, acc.w * inv));
        } else {
            dst[0] = lm_from_f<T>(acc.x * inv); dst[1] = lm_from_f<T>(acc.y * inv); dst[2] = lm_from_f<T>(acc.z * inv); dst[3] = lm_from_f<T>(acc.w * inv);
        }
    }
    if (a.ranks > 1) { cluster_arrive_relaxed(); cluster_wait(); }        // the others have read this block's part
    if (nf) nf->end(job_id);
}

typedef void (*OwnFn)(AttnArgs, uint32_t, FinishedBlockNotifier*);

template <typename T> OwnFn own_fn(int DP, int NT) {
    if (DP == 64) return NT == 1 ? own_kernel<T, 64, 1> : own_kernel<T, 64, 2>;
    return NT == 1 ? own_kernel<T, 128, 1> : own_kernel<T, 128, 2>;
}

struct AttnPlan {
    AttnArgs a;
    int DP, NT;
    bool half;
    int64_t prefix_blocks, own_blocks;
    uint64_t scratch;
    OwnFn own;
};

int plan_attn(const pb_prefix_attn_params* p, AttnPlan& pl) {
    const char* who = "pb_prefix_attn";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(p->dtype == PB_BF16 || p->dtype == PB_F16, "%s: dtype %d (PB_BF16 or PB_F16)", who, p->dtype);
    PB_REQUIRE(p->batch >= 0 && p->q_heads >= 1 && p->kv_heads >= 1 && p->q_heads % p->kv_heads == 0 && p->q_heads <= 65536, "%s: batch %d, %d query heads, %d key heads", who, p->batch, p->q_heads, p->kv_heads);
    PB_REQUIRE(p->head_dim >= 8 && p->head_dim <= 128 && p->head_dim % 8 == 0, "%s: head_dim %d (a multiple of 8, 8 to 128)", who, p->head_dim);
    PB_REQUIRE(p->page_size >= 8 && p->page_size % 8 == 0, "%s: page_size %d (a multiple of 8)", who, p->page_size);
    PB_REQUIRE(p->n_pages >= 0 && p->n_pages <= 0x7fffffff, "%s: %lld pages", who, (long long)p->n_pages);
    PB_REQUIRE(p->prefix_len >= 0 && p->prefix_len <= (1 << 30) && p->max_own_len >= 0 && p->max_own_len <= (1 << 30), "%s: prefix of %d tokens, at most %d own", who, p->prefix_len, p->max_own_len);
    PB_REQUIRE(p->max_blocks >= 0 && p->max_own_len <= (int64_t)p->max_blocks * p->page_size, "%s: %d own tokens do not fit %d pages of %d", who, p->max_own_len, p->max_blocks, p->page_size);
    PB_REQUIRE(p->n_pages > 0 || (p->prefix_len == 0 && p->max_own_len == 0) || p->batch == 0, "%s: a cache without pages", who);
    PB_REQUIRE(p->scale == p->scale && fabsf(p->scale) <= 3.402823466e38f, "%s: scale is not finite", who);
    PB_REQUIRE(p->page_stride % 8 == 0 && p->token_stride % 8 == 0 && p->head_stride % 8 == 0 && p->page_stride > 0 && p->token_stride > 0 && p->head_stride > 0, "%s: strides of the cache are positive multiples of 8", who);
    PB_REQUIRE(p->q_stride % 8 == 0 && p->q_head_stride % 8 == 0, "%s: rows of q start on 16 bytes", who);
    if (p->batch > 0) {
        PB_REQUIRE(p->q && p->out && p->k_cache && p->v_cache, "%s: NULL buffer", who);
        PB_REQUIRE(aligned(p->q, 16) && aligned(p->k_cache, 16) && aligned(p->v_cache, 16) && aligned(p->out, 2), "%s: q and the cache must be 16-byte aligned", who);
        PB_REQUIRE(p->prefix_len == 0 || (p->prefix_pages && aligned(p->prefix_pages, 4)), "%s: a prefix needs its pages", who);
        PB_REQUIRE(p->max_own_len == 0 || (p->block_table && p->own_lens && aligned(p->block_table, 4) && aligned(p->own_lens, 4)), "%s: own tokens need block_table and own_lens", who);
    }
    AttnArgs& a = pl.a;
    memset(&a, 0, sizeof(a));
    a.q = p->q; a.k = p->k_cache; a.v = p->v_cache; a.out = p->out; a.prefix_pages = p->prefix_pages; a.block_table = p->block_table; a.own_lens = p->own_lens;
    a.q_stride = p->q_stride; a.q_head = p->q_head_stride; a.out_stride = p->out_stride; a.out_head = p->out_head_stride;
    a.page_stride = p->page_stride; a.token_stride = p->token_stride; a.head_stride = p->head_stride; a.table_stride = p->table_stride;
    a.batch = p->batch; a.group = p->q_heads / p->kv_heads; a.D = p->head_dim; a.page = p->page_size; a.n_pages = (int)p->n_pages; a.prefix_len = p->prefix_len;
    a.max_own = p->max_own_len; a.scale = p->scale; a.kv_heads = p->kv_heads;
    pl.DP = p->head_dim <= 64 ? 64 : 128;
    pl.NT = a.group <= 8 ? 1 : 2;
    pl.half = p->dtype == PB_F16;
    pl.own = pl.half ? own_fn<__half>(pl.DP, pl.NT) : own_fn<__nv_bfloat16>(pl.DP, pl.NT);
    // the prefix: as many parts as give every SM a block
    const int64_t rows = (int64_t)a.batch * a.group;
    PB_REQUIRE(rows <= (1 << 24), "%s: %lld query rows for a key head", who, (long long)rows);
    a.row_tiles = (int)ceil_div<int64_t>(rows, 128);
    a.pairs = ceil_div(a.row_tiles, 2);
    a.key_tiles = ceil_div(a.prefix_len, 128);
    a.box_rows = 8;
    while (a.box_rows < 128 && p->page_size % (2 * a.box_rows) == 0) a.box_rows *= 2;
    const int64_t units = (int64_t)a.pairs * a.kv_heads;
    a.splits = 1;
    if (units > 0 && units < 148) a.splits = (int)(148 / units);
    if (a.splits > a.key_tiles) a.splits = a.key_tiles > 0 ? a.key_tiles : 1;
    pl.prefix_blocks = a.prefix_len > 0 ? units * a.splits : 0;
    const uint64_t parts = (uint64_t)pl.prefix_blocks * 2 * 128;
    pl.scratch = parts * ((uint64_t)pl.DP * 4 + 8);
    a.part_o = (float*)p->scratch;
    a.part_ml = (float2*)((char*)p->scratch + parts * pl.DP * 4);
    // own tokens
    a.row_groups = ceil_div(a.group, 8 * pl.NT);
    const int64_t own_units = (int64_t)a.batch * a.kv_heads * a.row_groups;
    a.ranks = 1;
    while (a.ranks < 8 && own_units * a.ranks < 2 * 148 && a.max_own / (2 * a.ranks) >= 128) a.ranks *= 2;
    pl.own_blocks = own_units > 0 ? own_units * a.ranks : 1;
    PB_REQUIRE(pl.prefix_blocks <= 0x7fffffff && pl.own_blocks <= 0x7fffffff, "%s: too many blocks for one launch", who);
    a.early = pl.prefix_blocks > 0;
    a.out_vec = aligned(p->out, 8) && a.out_stride % 4 == 0 && a.out_head % 4 == 0;
    return PB_OK;
}

template <typename T, int DP>
int launch_prefix(const AttnPlan& pl, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    PB_CUDA(cudaFuncSetAttribute(prefix_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PrefixShape<DP>::smem));
    return lm_launch("pb_prefix_attn (prefix)", prefix_kernel<T, DP>, dim3((unsigned)pl.prefix_blocks), dim3(320), PrefixShape<DP>::smem, st, 1, pl.a, km, vm);
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
    AttnPlan pl;
    const int rc = plan_attn(p, pl);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_prefix_attn_info: NULL out");
    memset(out, 0, sizeof(*out));
    out->num_blocks = (uint32_t)pl.own_blocks;
    out->threads_per_block = 128;
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, pl.own) == cudaSuccess) {
        out->regs_per_thread = (uint32_t)fa.numRegs;
        out->smem_per_block = (uint32_t)fa.sharedSizeBytes;
    } else {
        cudaGetLastError();
    }
    const uint64_t seen = (uint64_t)p->prefix_len + (uint64_t)p->batch * p->max_own_len;
    out->flops = 4ull * p->head_dim * p->q_heads * p->batch * ((uint64_t)p->prefix_len + p->max_own_len);
    out->bytes = p->batch ? 4ull * p->head_dim * (p->kv_heads * seen + (uint64_t)p->batch * p->q_heads) : 0;
    out->scratch_bytes = pl.scratch;
    return PB_OK;
}

int pb_prefix_attn_launch(const pb_prefix_attn_params* p, void* stream, uint32_t job_id, void* notifier) {
    AttnPlan pl;
    const int rc = plan_attn(p, pl);
    if (rc != PB_OK) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    if (pl.prefix_blocks > 0) {
        PB_REQUIRE(p->scratch != nullptr && p->scratch_bytes >= pl.scratch && aligned(p->scratch, 16), "pb_prefix_attn: %llu bytes of scratch memory are needed, 16-byte aligned (%llu given)",
                   (unsigned long long)pl.scratch, (unsigned long long)(p->scratch ? p->scratch_bytes : 0));
        // [page][head][token][value] whatever the order in memory; a dimension of one needs no stride of its own
        const uint64_t dims[4] = {(uint64_t)p->head_dim, (uint64_t)p->page_size, (uint64_t)p->kv_heads, (uint64_t)p->n_pages};
        const uint64_t strides[3] = {(uint64_t)p->token_stride * 2, p->kv_heads > 1 ? (uint64_t)p->head_stride * 2 : 16, p->n_pages > 1 ? (uint64_t)p->page_stride * 2 : 16};
        const uint32_t box[4] = {64, (uint32_t)pl.a.box_rows, 1, 1};
        const CUtensorMapDataType type = pl.half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        CUtensorMap km, vm;
        int e = encode_tiled_sw128(type, p->k_cache, 4, dims, strides, box, &km);
        if (e == PB_OK) e = encode_tiled_sw128(type, p->v_cache, 4, dims, strides, box, &vm);
        if (e == PB_OK) {
            if (pl.half) e = pl.DP == 64 ? launch_prefix<__half, 64>(pl, km, vm, st) : launch_prefix<__half, 128>(pl, km, vm, st);
            else e = pl.DP == 64 ? launch_prefix<__nv_bfloat16, 64>(pl, km, vm, st) : launch_prefix<__nv_bfloat16, 128>(pl, km, vm, st);
        }
        if (e != PB_OK) return e;
    }
    return lm_launch("pb_prefix_attn", pl.own, dim3((unsigned)pl.own_blocks), dim3(128), 0, st, pl.a.ranks, pl.a, job_id, (FinishedBlockNotifier*)notifier);
}

}  // extern "C"
