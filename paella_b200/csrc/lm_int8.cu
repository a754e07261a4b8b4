// Dense layers in 8-bit integers: activations brought to 8 bits token by token, and their product with weights that have a scale
// for each output channel.
//
//   q[t][k] = rint(x[t][k] * (127 * (1 / max_t))), s[t] = max_t / 127;   y[t][n] = act(s[t] * ws[n] * sum_k q[t][k] w[n][k] + b[n])
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "lm.cuh"
#include "umma.cuh"

namespace pb {
namespace {

__device__ uint32_t g_int8_flag;

// ---- activations to 8 bits ---------------------------------------------------------------
// Bound by memory (8192 rows of 8192 in fp16, 201 MB: 38 us, 5.2 TB/s): a row is read once, stays in registers, and leaves as a quarter or half of its bytes.
// `ROW` threads take a row (a warp a short one, the block a long one) in vectors of 16 bytes; what does not fit the registers is read a second time, from the
// caches.
struct QuantizeArgs {
    const void* x;
    int8_t* q;
    float* scale;
    int64_t x_stride, q_stride;
    int tokens, channels;
};

// rint(v * inv) for products up to 2^22: behind 1.5 x 2^23 the sum's last bits are the whole number, halves to even as rint has them.  (Conversions on the
// special-function unit kept it busy 45 % of the time.)
__device__ __forceinline__ int8_t to_int8(float v, float inv) { return (int8_t)__float_as_int(__fadd_rn(__fmul_rn(v, inv), 12582912.f)); }

template <typename T, bool WIDE, int ROW>
__global__ void __launch_bounds__(256) int8_quantize_kernel(const __grid_constant__ QuantizeArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    constexpr int V = WIDE ? 16 / (int)sizeof(T) : 1, HELD = WIDE ? 4 : 8;
    using In = LmVec<T, V>;
    using Out = LmVec<int8_t, V>;
    __shared__ float red[8];
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int me = threadIdx.x % ROW, vectors = a.channels / V, tail = vectors * V + me;
    const int64_t t = (int64_t)blockIdx.x * (256 / ROW) + threadIdx.x / ROW;
    const bool live = t < a.tokens;
    const T* row = static_cast<const T*>(a.x) + (live ? t : 0) * a.x_stride;
    const int mine = live ? vectors : 0;
    In held[HELD];
    float most = 0.f;
    bool odd = false;                                  // a NaN or an infinity
    const auto look = [&](float v) {
        v = fabsf(v);
        odd |= !(v <= 3.402823466e38f);
        most = fmaxf(most, v);
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (me + i * ROW < mine) held[i] = *reinterpret_cast<const In*>(row + (int64_t)(me + i * ROW) * V);
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (me + i * ROW < mine) {
#pragma unroll
            for (int j = 0; j < V; ++j) look(lm_to_f<T>(held[i].v[j]));
        }
    for (int i = me + HELD * ROW; i < mine; i += ROW) {
        const In x = *reinterpret_cast<const In*>(row + (int64_t)i * V);
#pragma unroll
        for (int j = 0; j < V; ++j) look(lm_to_f<T>(x.v[j]));
    }
    const bool has_tail = live && tail < a.channels;   // (fewer than V values)
    const float last = has_tail ? lm_to_f<T>(row[tail]) : 0.f;
    look(last);
    if (odd) most = INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (ROW > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
        __syncthreads();
        most = red[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) most = fmaxf(most, red[i]);
    }
    const bool zero = !(most >= 0x1p-119f) || most == INFINITY;
    const float inv = zero ? 0.f : 127.f * __fdiv_rn(1.f, most);
    if (live && me == 0) a.scale[t] = most == INFINITY ? NAN : zero ? 0.f : __fdiv_rn(most, 127.f);
    int8_t* dst = a.q + (live ? t : 0) * a.q_stride;
    const auto put = [&](int i, const In& x) {
        Out q;
#pragma unroll
        for (int j = 0; j < V; ++j) q.v[j] = zero ? (int8_t)0 : to_int8(lm_to_f<T>(x.v[j]), inv);
        *reinterpret_cast<Out*>(dst + (int64_t)i * V) = q;
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (me + i * ROW < mine) put(me + i * ROW, held[i]);
    for (int i = me + HELD * ROW; i < mine; i += ROW) put(i, *reinterpret_cast<const In*>(row + (int64_t)i * V));
    if (has_tail) dst[tail] = zero ? (int8_t)0 : to_int8(last, inv);
    if (nf) nf->end(job_id);
}

typedef void (*QuantizeFn)(QuantizeArgs, uint32_t, FinishedBlockNotifier*);
struct QuantizePlan {
    QuantizeFn fn;
    unsigned blocks;
};
template <typename T> QuantizeFn quantize_fn(bool wide, bool warp) {
    if (wide) return warp ? int8_quantize_kernel<T, true, 32> : int8_quantize_kernel<T, true, 256>;
    return warp ? int8_quantize_kernel<T, false, 32> : int8_quantize_kernel<T, false, 256>;
}

// ---- the product ---------------------------------------------------------------------------
// Y^T = W X^T on the tensor cores: operand A is 128 output channels, operand B up to 256 tokens, both as they lie in memory (rows
// of in_channels, 128 bytes a k-block, the 128-byte swizzle), the sums 32-bit integers in tensor memory, a lane for each channel.
// So a weight row's scale and bias are a thread's own, few tokens make a narrow tile instead of an empty one, and neighbouring
// lanes hold neighbouring values of y.
//
// Few tokens are bound by reading the weights, many by the tensor cores.  int8_few_kernel: a tile of 128 channels for each block, its
// reduction shared by the blocks of a cluster where the tiles alone leave SMs idle; they send their sums to the blocks that own the tokens (whole numbers:
// their order changes nothing).  Figures here and below are of launches back to back in a graph.  24 tokens, 4096 -> 14336: 13.6 us with the quantiser, 4.4 TB/s, 67 % of the copy rate; 64 tokens, 8192 -> 28672 40 to 42 us,
// 87 to 90 %.  int8_many_kernel: a pair of SMs on a tile of 256 channels, each block with its own half of the channels and half of the tokens: 32 KB a
// k-block and SM for 512 clocks of products, which the path from the L2 cache into an SM (some 60 bytes a clock) feeds; a lone SM on 128 x 256 would need
// 48 KB.  8192 tokens, 8192 -> 8192: 337 us at full clocks, 3261 TOP/s, twice the measured bf16 rate to 1 %; 390 to 400 where power holds the clocks down.
// 777 tokens, 2000 -> 5001 in fp32: 13.8 us (16.0 with one width for all tiles, 160 of them of 128 for 74 pairs): 1 for the first operands, 6 for the products, which
// wait for the L2 cache (11 TB/s), 3 for the results of all SMs at once.
struct DenseArgs {
    const float *x_scale, *w_scale, *bias;
    void* y;
    int64_t y_stride;
    int T, K, N, act;
    int kblocks, BN, stages, splits;       // BN: tokens of a tile
    int channel_tiles, token_tiles;
    int last, extra;                       // int8_many_kernel: tokens of the last tile, a multiple of 32; narrow tiles of a pair before all pairs take some
    int y_vec;                             // rows of y take 16-byte stores
};

constexpr uint32_t kABytes = 128 * 128;
constexpr int kMaxInt8Stages = 16;
constexpr int kMaxInt8Smem = 224 * 1024;


template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// Signed 8-bit operands, both along k, 32-bit integer sums.
__device__ __forceinline__ uint32_t i8_idesc(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

__device__ __forceinline__ float int8_result(int act, int acc, float s, float b) {
    float v = fmaf((float)acc, s, b);
    // (no branches; a NaN stays one)
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(act >= 1 ? 0.f : -INFINITY));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(act == 2 ? 6.f : INFINITY));
    return v;
}

__device__ __forceinline__ void wait_for_copies() {    // an aborted block's copies end before their shared memory does
    const unsigned long long t0 = globaltimer_ns();
    for (int i = 0; i < 100000 && globaltimer_ns() - t0 < 50000; ++i) __nanosleep(500);
}

template <typename Y, int HALVES>
__global__ void __launch_bounds__(192) int8_few_kernel(const __grid_constant__ DenseArgs a, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                                                       uint32_t job_id, FinishedBlockNotifier* nf) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_full[kMaxInt8Stages], s_empty[kMaxInt8Stages], s_sums, s_parts;
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_abort;
    __shared__ float s_xs[128];
    __shared__ volatile uint32_t s_never;              // an abort flag that another wait of this block does not raise
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u, half_bytes = kABytes + (uint32_t)a.BN * 128u, stage_bytes = half_bytes * HALVES;
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int rank = blockIdx.x % a.splits, tile = blockIdx.x / a.splits;
    const int n0 = tile % a.channel_tiles * 128, t0 = tile / a.channel_tiles * a.BN;
    const int kb0 = a.kblocks * rank / a.splits, nkb = a.kblocks * (rank + 1) / a.splits - kb0;
    const int tokens = min(a.BN, a.T - t0), owned = (tokens - rank + a.splits - 1) / a.splits;      // of a split reduction: tokens rank, rank + splits ...
    const uint32_t parts = ring + a.stages * stage_bytes;                                           // [rank][owned token][channel]: what the cluster's blocks send
    uint32_t cols = 32;
    while ((int)cols < a.BN) cols *= 2;
    if (warp == 5) {
        tcgen05_alloc(smem_u32(&s_tmem), cols);
        tcgen05_relinquish();
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        s_never = 0;
        for (int i = 0; i < a.stages; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_empty[i]), 1);
        }
        mbar_init(smem_u32(&s_sums), 1);
        mbar_init(smem_u32(&s_parts), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (a.splits > 1) mbar_arrive_expect_tx(smem_u32(&s_parts), (uint32_t)(a.splits * owned) * 512u);
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    if (a.splits > 1) cluster_arrive();
    const uint32_t tmem = uniform(s_tmem);
    if (warp == 4 && elect_one()) {
        // the weights come into the L2 cache while the launch that makes the activations still runs
        for (int i = 0; i < nkb * HALVES && i < 8; ++i)
            asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(&wmap), "r"((kb0 * HALVES + i) * 128), "r"(n0) : "memory");
    }
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    bool ok = true;
    if (warp == 4) {
        if (elect_one()) {
            uint32_t st = 0, parity = 1;
            for (int i = 0, x = kb0 * HALVES * 128; i < nkb; ++i) {
                if (i >= a.stages && !mbar_wait(smem_u32(&s_empty[st]), parity, &s_abort, &g_int8_flag, kFlagLmWait)) break;
                const uint32_t bar = smem_u32(&s_full[st]), at = ring + st * stage_bytes;
                mbar_arrive_expect_tx(bar, stage_bytes);
#pragma unroll
                for (uint32_t h = 0; h < HALVES; ++h, x += 128) {
                    tma_load_2d(at + h * half_bytes, &wmap, x, n0, bar);
                    tma_load_2d(at + h * half_bytes + kABytes, &xmap, x, t0, bar);
                }
                if (++st == (uint32_t)a.stages) { st = 0; parity ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        if (elect_one()) {
            const uint32_t idesc = i8_idesc(128, a.BN), step = stage_bytes >> 4;
            const uint64_t desc = umma_desc_sw128(ring);
            const uint32_t high = (uint32_t)(desc >> 32);
            uint32_t st = 0, parity = 0, low = (uint32_t)desc;
            for (int i = 0; i < nkb; ++i) {
                ok = mbar_wait(smem_u32(&s_full[st]), parity, &s_abort, &g_int8_flag, kFlagLmWait);
                if (!ok) break;
                tcgen05_fence_after();
#pragma unroll
                for (uint32_t k = 0; k < 4 * HALVES; ++k) {
                    const uint32_t at = low + (k >> 2) * (half_bytes >> 4) + 2 * (k & 3);
                    mma_i8<false>(tmem, pack_f32x2(at, high), pack_f32x2(at + (kABytes >> 4), high), idesc, (uint32_t)(i > 0) | (uint32_t)(k > 0));
                }
                tcgen05_commit(smem_u32(&s_empty[st]));
                low += step;
                if (++st == (uint32_t)a.stages) { st = 0; parity ^= 1; low = (uint32_t)desc; }
            }
            if (ok) tcgen05_commit(smem_u32(&s_sums));
        }
        __syncwarp();
    }
    const int n = n0 + 32 * (warp & 3) + lane;
    const bool mine = warp < 4 && n < a.N;
    const float ws = mine ? __ldg(a.w_scale + n) : 0.f, bias = mine && a.bias ? __ldg(a.bias + n) : 0.f;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    if (warp < 4) {
        if ((int)threadIdx.x < tokens) s_xs[threadIdx.x] = __ldcg(a.x_scale + t0 + threadIdx.x);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_sums), 0, &s_abort, &g_int8_flag, kFlagLmWait));
        tcgen05_fence_after();
        if (ok) {
            // (short loops: code that a block runs once comes from the L2 cache, line by line)
            if (a.splits == 1) {
                Y* dst = static_cast<Y*>(a.y) + (int64_t)t0 * a.y_stride + n;
#pragma unroll 1
                for (int j0 = 0; j0 < tokens; j0 += 8) {
                    uint32_t v[8];
                    tcgen05_ld8(lanes + j0, v);
                    tcgen05_wait_ld();
                    Y r[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) r[j] = lm_from_f<Y>(int8_result(a.act, (int)v[j], s_xs[(j0 + j) & 127] * ws, bias));
#pragma unroll
                    for (int j = 0; j < 8; ++j, dst += a.y_stride)
                        if (mine && j0 + j < tokens) *dst = r[j];
                }
            } else {
                cluster_wait();                        // the others' barriers are set up
                const int shift = __ffs(a.splits) - 1; // (blocks of a cluster: a power of two)
#pragma unroll 1
                for (int j0 = 0; j0 < tokens; j0 += 8) {
                    uint32_t v[8];
                    tcgen05_ld8(lanes + j0, v);
                    tcgen05_wait_ld();
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j0 + j < tokens) {
                            const uint32_t to = (uint32_t)(j0 + j) & (a.splits - 1), at = (uint32_t)(j0 + j) >> shift, theirs = (tokens - to + a.splits - 1) >> shift;
                            asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];"
                                         ::"r"(cluster_addr(parts + ((rank * theirs + at) * 128 + 32 * warp + lane) * 4u, to)), "r"(v[j]), "r"(cluster_addr(smem_u32(&s_parts), to)) : "memory");
                        }
                }
            }
        } else if (a.splits > 1) {
            cluster_wait();
        }
        if (a.splits > 1) {
            // (also a block that has given up waits for what the others send into its memory)
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_parts), 0, &s_never, &g_int8_flag, kFlagLmWait)) && ok;
            if (ok && mine) {
                Y* dst = static_cast<Y*>(a.y) + (int64_t)(t0 + rank) * a.y_stride + n;
                uint32_t from = parts + (32 * warp + lane) * 4u;
#pragma unroll 1
                for (int i = 0; i < owned; ++i, dst += a.splits * a.y_stride, from += 512) {
                    int sum = 0;
#pragma unroll 4
                    for (int r = 0; r < a.splits; ++r) {
                        int v;
                        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(from + r * owned * 512) : "memory");
                        sum += v;
                    }
                    *dst = lm_from_f<Y>(int8_result(a.act, sum, s_xs[rank + i * a.splits] * ws, bias));
                }
            }
        }
    } else if (a.splits > 1) {
        cluster_wait();
    }
    tcgen05_fence_before();
    __syncthreads();
    if (s_abort) wait_for_copies();
    if (warp == 5) {
        tcgen05_fence_after();
        tcgen05_dealloc(tmem, cols);
    }
    if (nf) nf->end(job_id);
}

constexpr uint32_t kOutBytes = 2 * 16 * 128 * 4;       // twice 32 tokens of 128 channels in 16 bits on their way out

// A pair of blocks walks its share of the tiles.  Warps 0-3 and 4-7: results, a lane a channel, 32 tokens each in turn; warp 8: copies of this block's operands; warp
// 9 of the first block: the products of both.  Two accumulators: the results of a tile leave under the products of the next.
template <typename Y>
__global__ void __launch_bounds__(320, 1) int8_many_kernel(const __grid_constant__ DenseArgs a, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                                                           uint32_t job_id, FinishedBlockNotifier* nf) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_full[kMaxInt8Stages], s_empty[kMaxInt8Stages], s_sums[2], s_read[2];
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_abort;
    __shared__ float s_xs[256];
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u, stage_bytes = kABytes + (uint32_t)a.BN * 64u, out = ring + a.stages * stage_bytes;
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int rank = blockIdx.x & 1, pairs = gridDim.x / 2;
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int i = 0; i < a.stages; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_sums[i]), 1);
            mbar_init(smem_u32(&s_read[i]), 2);        // the results warps of both blocks
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();                                    // both blocks' barriers and tensor memory are set up
    tcgen05_fence_after();
    const uint32_t tmem = uniform(s_tmem);
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();

    // Neighbouring pairs take the tokens of the same channels, then the next channels: all of them together read few rows of both operands.  The narrower tiles of
    // the last tokens come last: `extra` for each pair that has a wide tile less than others, the rest for all.
    struct Tile { int n0, t0, width; };
    const int wide = a.last < a.BN ? a.token_tiles - 1 : a.token_tiles, all = wide * a.channel_tiles, pair = blockIdx.x >> 1, short_of = all % pairs;
    const auto tile_at = [&](int turn, Tile& tile) {
        const int i = pair + turn * pairs, k = turn - (all - pair + pairs - 1) / pairs, given = a.extra * (pairs - short_of);
        if (i < all) {
            tile = {i / wide * 256, i % wide * a.BN, a.BN};
            return true;
        }
        const int n = pair < short_of ? given + k * pairs + pair : k < a.extra ? k * (pairs - short_of) + pair - short_of : given + (k - a.extra) * pairs + pair;
        tile = {n * 256, wide * a.BN, a.last};
        return a.last < a.BN && n < a.channel_tiles;
    };
    Tile tile;
    if (warp == 8) {
        uint32_t st = 0, parity = 1;
        int filled = 0;
        bool ok = true;
        for (int turn = 0; ok && tile_at(turn, tile); ++turn) {
            const int n0 = tile.n0 + 128 * rank, t0 = tile.t0 + tile.width / 2 * rank;
            for (int i = 0; i < a.kblocks; ++i) {
                if (filled == a.stages) {
                    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_empty[st]), parity, &s_abort, &g_int8_flag, kFlagLmWait));
                    if (!ok) break;
                } else {
                    ++filled;
                }
                if (elect_one()) {
                    const uint32_t bar = smem_u32(&s_full[st]), first = cluster_addr(bar, 0u), at = ring + st * stage_bytes;
                    if (rank == 0) mbar_arrive_expect_tx(bar, 2 * stage_bytes);      // both blocks' copies
                    tma_load_2d_pair(at, &wmap, i * 128, n0, first);
                    tma_load_2d_pair(at + kABytes, &xmap, i * 128, t0, first);
                }
                __syncwarp();
                if (++st == (uint32_t)a.stages) { st = 0; parity ^= 1; }
            }
        }
    } else if (warp == 9) {
        if (rank == 0) {
            const uint32_t step = uniform(stage_bytes >> 4), stages = uniform((uint32_t)a.stages);
            const uint64_t desc = umma_desc_sw128(uniform(ring));
            const uint32_t high = (uint32_t)(desc >> 32);
            uint32_t st = 0, parity = 0, low = (uint32_t)desc;
            bool ok = true;
            for (int turn = 0; ok && tile_at(turn, tile); ++turn) {
                const uint32_t acc = turn & 1, sums = tmem + 256 * acc, idesc = uniform(i8_idesc(256, tile.width));
                if (turn >= 2) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_read[acc]), (uint32_t)(turn / 2 - 1) & 1, &s_abort, &g_int8_flag, kFlagLmWait));
                if (!ok) break;
                tcgen05_fence_after();
                for (int i = 0; i < a.kblocks; ++i) {
                    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[st]), parity, &s_abort, &g_int8_flag, kFlagLmWait));
                    if (!ok) break;
                    tcgen05_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) mma_i8<true>(sums, pack_f32x2(low + 2 * k, high), pack_f32x2(low + (kABytes >> 4) + 2 * k, high), idesc, (uint32_t)(i > 0) | (uint32_t)(k > 0));
                        tcgen05_commit_pair(smem_u32(&s_empty[st]));
                    }
                    __syncwarp();
                    low += step;
                    if (++st == stages) { st = 0; parity ^= 1; low = (uint32_t)desc; }
                }
                if (ok && elect_one()) tcgen05_commit_pair(smem_u32(&s_sums[acc]));
                __syncwarp();
            }
        }
    } else {
        const int quarter = warp & 3, group = warp >> 2;
        for (int turn = 0; tile_at(turn, tile); ++turn) {
            const int acc = turn & 1, n0 = tile.n0 + 128 * rank, t0 = tile.t0, tokens = min(tile.width, a.T - t0);
            const int n = n0 + 32 * quarter + lane;
            const float ws = n < a.N ? __ldg(a.w_scale + n) : 0.f, bias = n < a.N && a.bias ? __ldg(a.bias + n) : 0.f;
            asm volatile("bar.sync 1, 256;" ::: "memory");                         // the last tile's scales and values have been read
            if (threadIdx.x < tokens) s_xs[threadIdx.x] = __ldcg(a.x_scale + t0 + threadIdx.x);
            // (the eight warps go on together or not at all: they meet at barriers)
            if (!all_of_256(mbar_wait(smem_u32(&s_sums[acc]), (turn / 2) & 1, &s_abort, &g_int8_flag, kFlagLmWait))) break;
            tcgen05_fence_after();
            for (int j0 = 32 * group; j0 < tokens; j0 += 64) {
                uint32_t v[32];
                tcgen05_ld32(tmem + ((uint32_t)quarter << 21) + 256 * acc + j0, v);
                tcgen05_wait_ld();
                if (j0 + 64 >= tokens) tcgen05_fence_before();                      // this warp's last columns: they may be written again
                const int left = min(32, tokens - j0);
                if (sizeof(Y) == 4 || !a.y_vec || n0 + 128 > a.N) {
                    // a warp's 32 channels of a token are 128 (64) bytes of a row, wherever it starts
                    Y* dst = static_cast<Y*>(a.y) + (int64_t)(t0 + j0) * a.y_stride + n;
                    Y r[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = lm_from_f<Y>(int8_result(a.act, (int)v[j], s_xs[j0 + j] * ws, bias));
                    if (left == 32 && n < a.N) {
#pragma unroll
                        for (int j = 0; j < 32; ++j, dst += a.y_stride) *dst = r[j];
                    } else if (n < a.N) {
#pragma unroll
                        for (int j = 0; j < 32; ++j, dst += a.y_stride)
                            if (j < left) *dst = r[j];
                    }
                    continue;
                }
                if constexpr (sizeof(Y) == 2) {        // two tokens a word in shared memory, [token / 2][channel], and out 16 bytes a thread
                    const uint32_t mine = out + group * (kOutBytes / 2), me = mine + (uint32_t)(32 * quarter + lane) * 4u;
#pragma unroll
                    for (int j = 0; j < 32; j += 2)
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(me + j * 256),
                                     "r"(lm_pack2<Y>(int8_result(a.act, (int)v[j], s_xs[j0 + j] * ws, bias), int8_result(a.act, (int)v[j + 1], s_xs[j0 + j + 1] * ws, bias))) : "memory");
                    asm volatile("bar.sync %0, 128;" ::"r"(2 + group) : "memory");
                    Y* dst = static_cast<Y*>(a.y) + (int64_t)(t0 + j0) * a.y_stride + n0;
                    for (int i = threadIdx.x & 127; i < 16 * 16; i += 128) {             // tokens 2 (i / 16) and + 1, channels 8 (i % 16) and up
                        const uint4 p = ld_shared_v4(mine + (i >> 4) * 512 + (i & 15) * 32), q = ld_shared_v4(mine + (i >> 4) * 512 + (i & 15) * 32 + 16);
                        Y* at = dst + (i >> 4) * 2 * a.y_stride + (i & 15) * 8;
                        if ((i >> 4) * 2 < left)
                            *reinterpret_cast<uint4*>(at) = make_uint4(__byte_perm(p.x, p.y, 0x5410), __byte_perm(p.z, p.w, 0x5410), __byte_perm(q.x, q.y, 0x5410), __byte_perm(q.z, q.w, 0x5410));
                        if ((i >> 4) * 2 + 1 < left)
                            *reinterpret_cast<uint4*>(at + a.y_stride) = make_uint4(__byte_perm(p.x, p.y, 0x7632), __byte_perm(p.z, p.w, 0x7632), __byte_perm(q.x, q.y, 0x7632), __byte_perm(q.z, q.w, 0x7632));
                    }
                    asm volatile("bar.sync %0, 128;" ::"r"(2 + group) : "memory");
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");                         // all warps have read the accumulator
            if (threadIdx.x == 0)
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr(smem_u32(&s_read[acc]), 0u)) : "memory");
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (s_abort) wait_for_copies();
    cluster_arrive();
    cluster_wait();                                    // neither block's memory goes before both have finished
    if (warp == 9) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (nf) nf->end(job_id);
}

// No tokens: the records alone.
__global__ void int8_nothing_kernel(uint32_t job_id, FinishedBlockNotifier* nf) {
    griddep_wait();
    if (nf) nf->start(job_id);
    if (nf) nf->end(job_id);
}

typedef void (*DenseFn)(DenseArgs, CUtensorMap, CUtensorMap, uint32_t, FinishedBlockNotifier*);
template <typename Y> DenseFn few_fn(int halves) { return halves == 2 ? int8_few_kernel<Y, 2> : int8_few_kernel<Y, 1>; }
struct DensePlan {
    DenseArgs a;
    bool many;
    DenseFn fn;
    unsigned blocks;
    uint32_t smem, tmem_cols;
};

int check_quantize(const pb_int8_quantize_params* p) {
    const char* who = "pb_int8_quantize";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(is_float_dtype(p->x_dtype), "%s: x_dtype %d (PB_F32, PB_BF16 or PB_F16)", who, p->x_dtype);
    PB_REQUIRE(p->tokens >= 0 && p->tokens <= (1 << 30) && p->channels >= 1 && p->channels <= (1 << 30), "%s: %d tokens of %d channels", who, p->tokens, p->channels);
    PB_REQUIRE(p->tokens == 0 || (p->x && p->q && p->scale), "%s: NULL buffer", who);
    PB_REQUIRE(aligned(p->x, dtype_bytes(p->x_dtype)) && aligned(p->scale, 4), "%s: a buffer is not aligned to its elements", who);
    PB_REQUIRE(rows_apart(p->tokens, p->q_stride, p->channels), "%s: rows of q overlap (stride %lld)", who, (long long)p->q_stride);
    return PB_OK;
}

int check_dense(const pb_int8_dense_params* p) {
    const char* who = "pb_int8_dense";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(is_float_dtype(p->y_dtype), "%s: y_dtype %d (PB_F32, PB_BF16 or PB_F16)", who, p->y_dtype);
    PB_REQUIRE(p->tokens >= 0 && p->tokens <= (1 << 30) && p->in_channels >= 1 && p->out_channels >= 1 && p->out_channels <= (1 << 30), "%s: %d tokens, %d -> %d channels", who, p->tokens, p->in_channels, p->out_channels);
    PB_REQUIRE(p->in_channels <= 131071, "%s: %d input channels could pass 32 bits (at most 131071)", who, p->in_channels);
    PB_REQUIRE(p->act >= 0 && p->act <= 2, "%s: activation %d (0 none, 1 relu, 2 relu6)", who, p->act);
    PB_REQUIRE(p->x_stride % 16 == 0 && p->w_stride % 16 == 0, "%s: rows of x and w start on 16 bytes (strides %lld, %lld)", who, (long long)p->x_stride, (long long)p->w_stride);
    PB_REQUIRE((p->x_stride >= p->in_channels || p->tokens <= 1) && (p->w_stride >= p->in_channels || p->out_channels == 1), "%s: rows overlap (strides %lld, %lld)", who, (long long)p->x_stride, (long long)p->w_stride);
    PB_REQUIRE(rows_apart(p->tokens, p->y_stride, p->out_channels), "%s: rows of y overlap (stride %lld)", who, (long long)p->y_stride);
    if (p->tokens > 0) {
        PB_REQUIRE(p->x && p->x_scale && p->w && p->w_scale && p->y, "%s: NULL buffer", who);
        PB_REQUIRE(aligned(p->x, 16) && aligned(p->w, 16), "%s: x and w must be 16-byte aligned", who);
        PB_REQUIRE(aligned(p->x_scale, 4) && aligned(p->w_scale, 4) && aligned(p->bias, 4) && aligned(p->y, dtype_bytes(p->y_dtype)), "%s: a buffer is not aligned to its elements", who);
    }
    return PB_OK;
}

int plan_quantize(const pb_int8_quantize_params* p, QuantizePlan& pl) {
    const int rc = check_quantize(p);
    if (rc != PB_OK) return rc;
    const size_t es = dtype_bytes(p->x_dtype);
    const int V = (int)(16 / es);
    const bool wide = aligned(p->x, 16) && p->x_stride % V == 0 && aligned(p->q, V) && p->q_stride % V == 0;
    // a warp holds 128 vectors of a row; longer rows take a block
    const bool warp = p->channels <= 128 * (wide ? V : 2);
    pl.fn = p->x_dtype == PB_F32 ? quantize_fn<float>(wide, warp) : p->x_dtype == PB_BF16 ? quantize_fn<__nv_bfloat16>(wide, warp) : quantize_fn<__half>(wide, warp);
    pl.blocks = p->tokens > 0 ? (unsigned)(warp ? ceil_div(p->tokens, 8) : p->tokens) : 1u;
    return PB_OK;
}

// Clocks of a launch, from what an SM does in one: products of BN tokens with 128 channels (four instructions a k-block, BN / 2 clocks each, but no fewer
// than shared memory needs for both operands at 128 bytes a clock), copies at 60 bytes a clock.
double kblock_clocks(int BN, int b_rows) {
    const double mma = 4 * std::max(BN / 2.0, 32 + b_rows / 4.0), copy = (128 + b_rows) * 128 / 60.0;
    return std::max(mma, copy);
}

int plan_dense(const pb_int8_dense_params* p, DensePlan& pl) {
    const int rc = check_dense(p);
    if (rc != PB_OK) return rc;
    DenseArgs& a = pl.a;
    a = {p->x_scale, p->w_scale, p->bias, p->y, p->y_stride, p->tokens, p->in_channels, p->out_channels, p->act};
    a.kblocks = ceil_div(a.K, 128);
    const int T = a.T > 0 ? a.T : 1;
    double best = 1e300;
    int halves = 1;            // of 128 bytes of a row in a stage of int8_few_kernel
    // One block a tile; narrower tiles, and up to 8 blocks on a reduction, only where SMs would be idle otherwise (two blocks an SM for long reductions).
    // Beside what an SM does: the weights from memory, at 22 bytes a clock for each SM that asks for them, and for parts that meet 2600 clocks and 70 a
    // token.  (24 tokens, 4096 -> 14336: 112 blocks 13.6 us, 224 that share 17.9, 224 of twelve tokens 16.8; 16384 -> 14336: 112 blocks 52, 224
    // that share 42; 64 tokens, 1024 -> 1024: 8 blocks 4.5, 16 of half the tokens 3.6, 64 that share 5.5.)
    for (int tt = ceil_div(T, 128); tt <= ceil_div(T, 16); ++tt) {
        const int BN = round_up(ceil_div(T, tt), 16), tiles = ceil_div(T, BN), pieces = BN <= 32 ? 2 : 1, few = ceil_div(a.K, 128 * pieces);
        if (tt > ceil_div(T, 128) && (int64_t)ceil_div(a.N, 128) * tiles > 148) break;
        for (int S = 1; S <= 8 && S <= few; S *= 2) {
            const double blocks = (double)ceil_div(a.N, 128) * tiles * S;
            if (S > 1 && blocks > (a.K >= 8192 ? 296 : 148)) break;
            const double work = std::ceil(blocks / 148) * ceil_div(few, S) * pieces * kblock_clocks(BN, BN), memory = (double)a.N * a.K / (22 * std::min(blocks, 148.0));
            const double clocks = std::max(work, memory) + (S > 1 ? 2600 + 70.0 * std::min(BN, T) : 0) + 10.0 * BN;
            if (clocks < best) { best = clocks; pl.many = false; a.BN = BN; a.token_tiles = tiles; a.splits = S; halves = pieces; }
        }
    }
    // pairs of SMs on 256 channels
    if (T > 64)
        for (int wide = 64; wide <= 256; wide += 32) {
            const int tiles = ceil_div(T, wide), last = round_up(T - (tiles - 1) * wide, 32);
            const int64_t rows = ceil_div(a.N, 256), full = rows * (last < wide ? tiles - 1 : tiles), narrow = rows * tiles - full;
            // (as the kernel deals them out: the most have the first pair, and the first that has a wide tile less than others)
            const double of_wide = a.kblocks * kblock_clocks(wide, wide / 2), of_narrow = a.kblocks * kblock_clocks(last, last / 2);
            for (int extra = 0; extra <= (narrow ? 4 : 0); ++extra) {
                const int64_t rest = std::max<int64_t>(narrow - extra * (74 - full % 74), 0);
                const double first = ceil_div<int64_t>(full, 74) * of_wide + ceil_div<int64_t>(rest, 74) * of_narrow, other = full / 74 * of_wide + (std::min<int64_t>(extra, narrow) + ceil_div<int64_t>(rest, 74)) * of_narrow;
                const double clocks = std::max(first, other) + 2000 + 10.0 * wide;
                if (clocks < best) { best = clocks; pl.many = true; a.BN = wide; a.token_tiles = tiles; a.last = last; a.extra = extra; a.splits = 1; }
            }
        }
    a.channel_tiles = ceil_div(a.N, pl.many ? 256 : 128);
    // Narrow tiles take 256 bytes of a row a stage: what a stage costs beside its copies and products, 230 clocks, comes half as often.
    if (!pl.many) a.kblocks = ceil_div(a.K, 128 * halves);
    const uint32_t stage = pl.many ? kABytes + (uint32_t)a.BN * 64 : (kABytes + (uint32_t)a.BN * 128) * halves;
    if (pl.many) {
        a.stages = (int)std::min<uint32_t>(kMaxInt8Stages, (kMaxInt8Smem - 1024 - kOutBytes) / stage);
        pl.smem = 1024 + a.stages * stage + kOutBytes;
        const int64_t tiles = (int64_t)a.channel_tiles * a.token_tiles;
        PB_REQUIRE(tiles <= 0x3fffffff, "pb_int8_dense: too many results for one launch");
        pl.blocks = 2 * (unsigned)std::min<int64_t>(tiles, 74);
        pl.tmem_cols = 512;
        a.splits = 2;          // blocks of a cluster
        pl.fn = p->y_dtype == PB_F32 ? int8_many_kernel<float> : p->y_dtype == PB_BF16 ? int8_many_kernel<__nv_bfloat16> : int8_many_kernel<__half>;
    } else {
        // What an SM has in flight covers the memory's latency: up to 200 KB of one block, or 100 KB each of two.  Blocks that have an SM each also keep it to
        // themselves: two of the next launch, set up beside this one's on an idle SM, would share its path to memory while others have one block.
        const uint32_t sent = a.splits > 1 ? (uint32_t)a.splits * ceil_div(a.BN, a.splits) * 512 : 0;
        const bool lone = (int64_t)a.channel_tiles * a.token_tiles * a.splits <= 148;
        uint32_t room = (lone ? 216 * 1024 : 111 * 1024) - sent;
        if (room < 2 * stage) room = 216 * 1024 - sent;
        a.stages = (int)std::min<uint32_t>(std::min<uint32_t>(kMaxInt8Stages, ceil_div(a.kblocks, a.splits)), room / stage);
        pl.smem = 1024 + a.stages * stage + sent;
        if (lone && pl.smem < 116 * 1024) pl.smem = 116 * 1024;
        const int64_t blocks = (int64_t)a.channel_tiles * a.token_tiles * a.splits;
        PB_REQUIRE(blocks <= 0x7fffffff, "pb_int8_dense: too many results for one launch");
        pl.blocks = (unsigned)blocks;
        pl.tmem_cols = 32;
        while ((int)pl.tmem_cols < a.BN) pl.tmem_cols *= 2;
        pl.fn = p->y_dtype == PB_F32 ? few_fn<float>(halves) : p->y_dtype == PB_BF16 ? few_fn<__nv_bfloat16>(halves) : few_fn<__half>(halves);
    }
    const int V = (int)(16 / dtype_bytes(p->y_dtype));
    a.y_vec = aligned(p->y, 16) && p->y_stride % V == 0;
    return PB_OK;
}

}  // namespace

uint32_t* lm_int8_error_flag_ptr() {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_int8_flag) != cudaSuccess) { cudaGetLastError(); return nullptr; }
    return (uint32_t*)p;
}

}  // namespace pb

using namespace pb;

extern "C" {

int pb_int8_quantize_info(const pb_int8_quantize_params* p, pb_launch_info* out) {
    QuantizePlan pl;
    const int rc = plan_quantize(p, pl);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_int8_quantize_info: NULL out");
    memset(out, 0, sizeof(*out));
    out->num_blocks = pl.blocks;
    out->threads_per_block = 256;
    out->smem_per_block = 32;
    out->regs_per_thread = lm_regs(pl.fn);
    out->bytes = (uint64_t)p->tokens * ((dtype_bytes(p->x_dtype) + 1) * p->channels + 4);
    return PB_OK;
}

int pb_int8_quantize_launch(const pb_int8_quantize_params* p, void* stream, uint32_t job_id, void* notifier) {
    QuantizePlan pl;
    const int rc = plan_quantize(p, pl);
    if (rc != PB_OK) return rc;
    const QuantizeArgs a = {p->x, p->q, p->scale, p->x_stride, p->q_stride, p->tokens, p->channels};
    return lm_launch("pb_int8_quantize", pl.fn, dim3(pl.blocks), dim3(256), 0, (cudaStream_t)stream, 1, a, job_id, (FinishedBlockNotifier*)notifier);
}

int pb_int8_dense_info(const pb_int8_dense_params* p, pb_launch_info* out) {
    DensePlan pl;
    const int rc = plan_dense(p, pl);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_int8_dense_info: NULL out");
    memset(out, 0, sizeof(*out));
    const uint64_t t = (uint64_t)p->tokens, k = (uint64_t)p->in_channels, n = (uint64_t)p->out_channels;
    out->num_blocks = p->tokens > 0 ? pl.blocks : 1;
    out->threads_per_block = pl.many ? 320 : 192;
    out->smem_per_block = pl.smem;
    out->regs_per_thread = lm_regs(pl.fn);
    out->tmem_cols_per_block = pl.tmem_cols;
    out->flops = 2 * t * k * n;
    out->bytes = t * k + n * k + 4 * t + (p->bias ? 8 : 4) * n + t * n * dtype_bytes(p->y_dtype);
    return PB_OK;
}

int pb_int8_dense_launch(const pb_int8_dense_params* p, void* stream, uint32_t job_id, void* notifier) {
    DensePlan pl;
    const int rc = plan_dense(p, pl);
    if (rc != PB_OK) return rc;
    if (p->tokens == 0) return lm_launch("pb_int8_dense", int8_nothing_kernel, dim3(1), dim3(192), 0, (cudaStream_t)stream, 1, job_id, (FinishedBlockNotifier*)notifier);
    const uint64_t wdims[2] = {(uint64_t)p->in_channels, (uint64_t)p->out_channels}, xdims[2] = {(uint64_t)p->in_channels, (uint64_t)p->tokens};
    // (the stride of a lone row is never used)
    const uint64_t wstride = p->out_channels > 1 ? (uint64_t)p->w_stride : round_up<uint64_t>(p->in_channels, 16), xstride = p->tokens > 1 ? (uint64_t)p->x_stride : round_up<uint64_t>(p->in_channels, 16);
    const uint32_t wbox[2] = {128, 128}, xbox[2] = {128, (uint32_t)(pl.many ? pl.a.BN / 2 : pl.a.BN)};
    CUtensorMap wmap, xmap;
    int e = encode_tiled_sw128(CU_TENSOR_MAP_DATA_TYPE_UINT8, p->w, 2, wdims, &wstride, wbox, &wmap);
    if (e == PB_OK) e = encode_tiled_sw128(CU_TENSOR_MAP_DATA_TYPE_UINT8, p->x, 2, xdims, &xstride, xbox, &xmap);
    if (e != PB_OK) return e;
    PB_CUDA(cudaFuncSetAttribute(pl.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxInt8Smem));      // (the same for every launch: other threads' may be on their way)
    return lm_launch("pb_int8_dense", pl.fn, dim3(pl.blocks), dim3(pl.many ? 320 : 192), pl.smem, (cudaStream_t)stream, pl.a.splits, pl.a, wmap, xmap, job_id, (FinishedBlockNotifier*)notifier);
}

}  // extern "C"
