// Log probabilities of given tokens with their ranks, the entropy of each row of logits, and its likeliest tokens.
//
//   log p_t = s x_t - log sum_j exp(s x_j);   H = log S - sum_j e_j d_j / S   with d_j = s (x_j - m), e_j = exp(d_j), S = sum_j e_j
//
// Bound by memory: the logits are read once (their exponentials take three quarters of the special-function units' time at that rate in 16 bits).  Each
// thread runs along its own vectors of a row with a maximum m of its own, which it follows only once it has grown by 2^16, so that sums are
// rescaled a few times a row; all of a row's threads join at its end.
//
// The likeliest tokens come out of the same pass: a thread remembers the first of its vectors with its largest logit.  Tokens are ordered by keys of
// 64 bits, the logit's order above the index's, so that no two are equal; the k-th largest of the threads' largest keys is a bound that k tokens
// reach, and exactly k threads have any.  Only their vectors are read again (from the caches), each by a warp that keeps the 32 largest keys of what it saw in order, one a lane.
#include <cmath>

#include "lm.cuh"
#include "umma.cuh"

namespace pb {
namespace {

__device__ uint32_t g_logprobs_flag;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxTop = 32, kMaxRanks = 8;
constexpr float kLog2e = 1.4426950408889634f;

struct LogprobsArgs {
    const void* logits;
    const int32_t* targets;
    float *logprobs, *entropy, *top_logprobs;
    int32_t *ranks, *top_ids;
    int64_t stride, top_stride;
    int tokens, vocab, top, ranks_of_row;      // ranks_of_row: blocks of a cluster that share a row out
    float scale, c, slack, far;                // c: scale * log2(e); 16 and 256 in powers of two as differences of logits
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}

// The logits' order as whole numbers: 0 is none of them, NaNs are the largest, both zeros are the same.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
    return __uint_as_float(order == 0xffffffffu ? 0x7fffffffu : order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t key_of(uint32_t order, int index) { return (uint64_t)order << 32 | (0x7fffffffu - (uint32_t)index); }
__device__ __forceinline__ int index_of(uint64_t key) { return (int)(0x7fffffffu - (uint32_t)key); }

// 16 bytes of logits.
template <typename T> struct Logits {
    static constexpr int V = 16 / (int)sizeof(T);
    uint4 w;
    __device__ __forceinline__ void load(const T* p) { w = __ldcg(reinterpret_cast<const uint4*>(p)); }
    // value pairs as they are multiplied
    __device__ __forceinline__ uint64_t pair(int i) const {
        const uint32_t* q = &w.x;
        if constexpr (sizeof(T) == 4) {
            return pack_f32x2(q[2 * i], q[2 * i + 1]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(q + i));
            return pack_f32x2(__float_as_uint(f.x), __float_as_uint(f.y));
        } else {
            return pack_f32x2(q[i] << 16, q[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        float lo, hi;
        unpack_f32x2(pair(i >> 1), lo, hi);
        return i & 1 ? hi : lo;
    }
    // the largest, or NaN if there is one
    __device__ __forceinline__ float top() const {
        if constexpr (sizeof(T) == 4) {
            return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2* q = reinterpret_cast<const __half2*>(&w);
            const float2 f = __half22float2(__hmax2_nan(__hmax2_nan(q[0], q[1]), __hmax2_nan(q[2], q[3])));
            return max_nan(f.x, f.y);
        } else {
            const __nv_bfloat162* q = reinterpret_cast<const __nv_bfloat162*>(&w);
            const float2 f = __bfloat1622float2(__hmax2_nan(__hmax2_nan(q[0], q[1]), __hmax2_nan(q[2], q[3])));
            return max_nan(f.x, f.y);
        }
    }
    // none below `low` (no NaN among them)
    __device__ __forceinline__ void raise(T low) {
        if constexpr (sizeof(T) == 4) {
            w = make_uint4(__float_as_uint(fmaxf(__uint_as_float(w.x), low)), __float_as_uint(fmaxf(__uint_as_float(w.y), low)), __float_as_uint(fmaxf(__uint_as_float(w.z), low)),
                           __float_as_uint(fmaxf(__uint_as_float(w.w), low)));
        } else if constexpr (std::is_same<T, __half>::value) {
            __half2* q = reinterpret_cast<__half2*>(&w);
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = __hmax2(q[i], __half2half2(low));
        } else {
            __nv_bfloat162* q = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = __hmax2(q[i], __bfloat162bfloat162(low));
        }
    }
};

template <typename T> __device__ __forceinline__ float lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -3.402823466e38f; }
template <> __device__ __forceinline__ float lowest<__nv_bfloat16>() { return -3.389531389e38f; }
template <> __device__ __forceinline__ float lowest<__half>() { return -65504.f; }

// A thread's (or a row's) sums: S = sum e, E = sum e (x - m).  m = -inf: nothing yet.
struct Sums {
    float m, S, E;
    __device__ __forceinline__ void rescale(float to, float c) {       // m <= to
        if (m != -INFINITY) {
            const float t = m - to, f = ex2(t * c);
            E = f > 0.f ? f * fmaf(S, t, E) : 0.f;
            S *= f;
        }
        m = to;
    }
    __device__ __forceinline__ void add(const Sums& o, float c) {
        if (o.S != o.S || S != S) { S = E = __uint_as_float(0x7fffffffu); return; }
        if (o.m == -INFINITY) return;
        Sums x = o;
        if (x.m > m) rescale(x.m, c);
        else x.rescale(m, c);
        S += x.S;
        E += x.E;
    }
    __device__ __forceinline__ void add_logit(float x, float c) {      // any value
        if (!(x < INFINITY)) { S = E = __uint_as_float(0x7fffffffu); return; }
        if (x == -INFINITY) return;
        if (x > m) rescale(x, c);
        const float t = x - m, e = ex2(t * c);
        if (e > 0.f) { S += e; E = fmaf(e, t, E); }
    }
};

// 32 keys, one a lane, brought into falling order; or, of a rising-then-falling sequence, its last steps.
__device__ __forceinline__ uint64_t exchange(uint64_t k, int with, bool keep_larger) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, k, with);
    return (k > o) == keep_larger ? k : o;
}
__device__ __forceinline__ uint64_t merge_32(uint64_t k, int lane) {
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) k = exchange(k, j, (lane & j) == 0);
    return k;
}
__device__ __forceinline__ uint64_t sort_32(uint64_t k, int lane) {
#pragma unroll
    for (int n = 2; n <= 32; n *= 2)
#pragma unroll
        for (int j = n / 2; j > 0; j >>= 1) k = exchange(k, j, ((lane & j) == 0) == ((lane & n) == 0));
    return k;
}
// The 32 largest of two falling sequences.
__device__ __forceinline__ uint64_t largest_32(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
    return merge_32(a > r ? a : r, lane);
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const __grid_constant__ LogprobsArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    constexpr int V = Logits<T>::V;
    __shared__ Sums s_sums[kWarps];
    __shared__ int s_before[kWarps];
    __shared__ uint64_t s_keys[TOP ? kWarps : 1][32];
    __shared__ int s_segment[kMaxTop], s_segments;
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = threadIdx.x;
    const int rank = blockIdx.x % a.ranks_of_row, row = blockIdx.x / a.ranks_of_row;
    const bool live = row < a.tokens;
    const T* x = static_cast<const T*>(a.logits) + (live ? row : 0) * a.stride;
    // the row: up to V - 1 logits until 16 bytes are aligned, n vectors, up to V - 1 more.  This block's share of the vectors; the first block has the others, too.
    const int head = live ? min((int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T), a.vocab) : 0, n = live ? (a.vocab - head) / V : 0;
    const int first = (int)((int64_t)n * rank / a.ranks_of_row), last = (int)((int64_t)n * (rank + 1) / a.ranks_of_row);
    const int loose = live && rank == 0 ? a.vocab - n * V : 0;           // logits outside of the vectors: the first `head`, and those behind
    const auto loose_index = [&](int i) { return i < head ? i : n * V + i; };
    int target = -1;
    if (live && a.targets) target = a.targets[row];
    if (target >= a.vocab && t == 0) atomicExch(&g_logprobs_flag, kFlagLmToken);
    const bool ranked = target >= 0 && target < a.vocab;
    const float wanted = ranked ? lm_to_f<T>(x[target]) : 0.f;
    const uint64_t wanted_key = ranked ? key_of(order_of(wanted), target) : ~0ull;

    Sums sums = {-INFINITY, 0.f, 0.f};
    int before = 0, at = -1;                  // logits in front of the target; the vector of the largest one
    uint32_t best = 0;
    float best_logit = -INFINITY, limit = __uint_as_float(0x7fffffffu);     // limit: vectors whose largest logit is not above it are the common ones
    T low = lm_from_f<T>(0.f);
    uint64_t S2 = 0, E2 = 0;
    const T* body = x + head;
    const uint64_t c2 = pack_f32x2(__float_as_uint(a.c), __float_as_uint(a.c));
    uint64_t minus_m = 0;
    const int with_target = ranked && target >= head && target < head + n * V ? (target - head) / V : -1;
    // The sums of the common vectors, as pairs, into the others.
    const auto fold = [&]() {
        float lo, hi, elo, ehi;
        unpack_f32x2(S2, lo, hi);
        unpack_f32x2(E2, elo, ehi);
        sums.S += lo + hi;
        sums.E += elo + ehi;
        S2 = E2 = 0;
    };
    const auto take = [&](Logits<T> v, int i) {
        const float top = v.top();
        if (TOP && top > best_logit) { best_logit = top; best = order_of(top); at = i; }
        if (!(top <= limit)) {
            // a first vector, one that is far above what came so far, or one with a NaN or infinity
            if (TOP && (top != top || top == -INFINITY) && best < order_of(top)) { best = order_of(top); at = i; best_logit = top == top ? top : INFINITY; }
            fold();
            if (top > sums.m && top < INFINITY) sums.rescale(top, a.c);
            // Logits far below the maximum are raised to `low`, where their exponentials are zeros: masks of -infinity need no case of their own.  Not where
            // logits are so large that `low` and the maximum are too near each other in their type: those go one by one.
            low = lm_from_f<T>(fmaxf(sums.m - a.far, lowest<T>()));
            const bool common = sums.m > -INFINITY && (sums.m - lm_to_f<T>(low)) * a.c >= 200.f;
            limit = common ? sums.m + a.slack : __uint_as_float(0x7fffffffu);
            minus_m = pack_f32x2(__float_as_uint(-sums.m), __float_as_uint(-sums.m));
            if (!(top <= limit)) {
#pragma unroll 1
                for (int j = 0; j < V; ++j) {
                    const float logit = v[j];
                    sums.add_logit(logit, a.c);
                    if (ranked) before += key_of(order_of(logit), head + i * V + j) > wanted_key;
                }
                return;
            }
        }
        if (ranked && top >= wanted) {
            if (i == with_target) {
#pragma unroll
                for (int j = 0; j < V; ++j) before += key_of(order_of(v[j]), head + i * V + j) > wanted_key;
            } else if (head + i * V < target) {
#pragma unroll
                for (int j = 0; j < V; ++j) before += v[j] >= wanted;
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) before += v[j] > wanted;
            }
        }
        v.raise(low);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const uint64_t d = add_f32x2(v.pair(j), minus_m);
            float lo, hi;
            unpack_f32x2(mul_f32x2(d, c2), lo, hi);
            const uint64_t e = pack_f32x2(__float_as_uint(ex2(lo)), __float_as_uint(ex2(hi)));
            S2 = add_f32x2(S2, e);
            E2 = fma_f32x2(e, d, E2);
        }
    };
    {
        constexpr int U = 4;                                              // vectors in flight
        int i = first + t;
        for (; i + (U - 1) * kThreads < last; i += U * kThreads) {
            Logits<T> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u].load(body + (int64_t)(i + u * kThreads) * V);
#pragma unroll
            for (int u = 0; u < U; ++u) take(v[u], i + u * kThreads);
        }
        for (; i < last; i += kThreads) {
            Logits<T> v;
            v.load(body + (int64_t)i * V);
            take(v, i);
        }
        fold();
    }
    uint64_t loose_key = 0;
    if (t < loose) {
        const int index = loose_index(t);
        const float v = lm_to_f<T>(x[index]);
        sums.add_logit(v, a.c);
        loose_key = key_of(order_of(v), index);
        if (ranked) before += loose_key > wanted_key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums other;
        other.m = __shfl_xor_sync(0xffffffffu, sums.m, o);
        other.S = __shfl_xor_sync(0xffffffffu, sums.S, o);
        other.E = __shfl_xor_sync(0xffffffffu, sums.E, o);
        // the same in both lanes: the lower one's first
        Sums lower = lane & o ? other : sums;
        lower.add(lane & o ? sums : other, a.c);
        sums = lower;
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (lane == 0) { s_sums[warp] = sums; s_before[warp] = before; }
    if (threadIdx.x == 0) s_segments = 0;

    if constexpr (TOP) {
        // this thread's largest key, and the k-th largest of the block's
        uint64_t mine = 0;
        if (at >= 0) {
            Logits<T> v;
            v.load(body + (int64_t)at * V);
            int j = V - 1;
#pragma unroll
            for (int e = V - 1; e >= 0; --e) j = order_of(v[e]) == best ? e : j;
            mine = key_of(best, head + at * V + j);
        }
        const auto largest_of_block = [&](uint64_t falling) {             // of the warps' falling sequences; in warp 0
            s_keys[warp][lane] = falling;
            __syncthreads();
            for (int half = kWarps / 2; half > 0; half /= 2) {
                if (warp < half) {
                    falling = largest_32(falling, s_keys[warp + half][lane], lane);
                    s_keys[warp][lane] = falling;
                }
                __syncthreads();
            }
            return s_keys[0][lane];
        };
        largest_of_block(sort_32(mine, lane));
        const uint64_t bound = s_keys[0][a.top - 1];                      // (0 where fewer threads have vectors)
        if (mine > 0 && mine >= bound) s_segment[atomicAdd(&s_segments, 1)] = t;
        __syncthreads();
        // the loose logits are in any case looked at: warp 0's first
        uint64_t list = 0;
        if (warp == 0) list = sort_32(loose_key, lane);
        for (int s = warp; s < s_segments; s += kWarps) {
            const int from = first + s_segment[s];
            for (int base = from; base < last; base += 32 * kThreads) {
                const int i = base + lane * kThreads;
                Logits<T> v;
                if (i < last) v.load(body + (int64_t)i * V);
#pragma unroll 1
                for (int j = 0; j < V; ++j) {
                    const uint64_t key = i < last ? key_of(order_of(v[j]), head + i * V + j) : 0;
                    const uint64_t least = __shfl_sync(0xffffffffu, list, 31);
                    if (__any_sync(0xffffffffu, key >= bound && key > least)) list = largest_32(list, sort_32(key >= bound ? key : 0, lane), lane);
                }
            }
        }
        largest_of_block(list);
    } else {
        __syncthreads();
    }
    if (a.ranks_of_row > 1) { cluster_arrive(); cluster_wait(); }
    if (rank == 0 && warp == 0 && live) {
        // all warps' sums of all blocks: a warp a lane, block after block
        Sums all = {-INFINITY, 0.f, 0.f};
        int count = 0;
        uint64_t list = TOP ? s_keys[0][lane] : 0;
        for (int r = 0; r < a.ranks_of_row; ++r) {
            if (lane < kWarps) {
                Sums o;
                const uint32_t from = cluster_addr(smem_u32(&s_sums[lane]), (uint32_t)r);
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.m) : "r"(from) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.S) : "r"(from + 4) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.E) : "r"(from + 8) : "memory");
                int b;
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(b) : "r"(cluster_addr(smem_u32(&s_before[lane]), (uint32_t)r)) : "memory");
                all.add(o, a.c);
                count += b;
            }
            if (TOP && r > 0) {
                uint64_t other;
                asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(other) : "r"(cluster_addr(smem_u32(&s_keys[0][lane]), (uint32_t)r)) : "memory");
                list = largest_32(list, other, lane);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            Sums other;
            other.m = __shfl_xor_sync(0xffffffffu, all.m, o);
            other.S = __shfl_xor_sync(0xffffffffu, all.S, o);
            other.E = __shfl_xor_sync(0xffffffffu, all.E, o);
            Sums lower = lane & o ? other : all;
            lower.add(lane & o ? all : other, a.c);
            all = lower;
            count += __shfl_xor_sync(0xffffffffu, count, o);
        }
        const float logs = logf(all.S);
        const bool nothing = all.m == -INFINITY && all.S == 0.f;
        const auto logprob = [&](float v) { return nothing ? -INFINITY : fmaf(0.5f * v - 0.5f * all.m, 2.f * a.scale, -logs); };      // (halves: the difference of a type's ends is finite)
        if (lane == 0) {
            if (a.logprobs && a.targets) a.logprobs[row] = target < 0 ? 0.f : ranked ? logprob(wanted) : __uint_as_float(0x7fffffffu);
            if (a.ranks && a.targets) a.ranks[row] = ranked ? 1 + count : 0;
            if (a.entropy) a.entropy[row] = nothing ? 0.f : fmaf(-all.E / all.S, a.scale, logs);
        }
        if (TOP && lane < a.top) {
            if (a.top_ids) a.top_ids[row * a.top_stride + lane] = index_of(list);
            if (a.top_logprobs) a.top_logprobs[row * a.top_stride + lane] = logprob(logit_of((uint32_t)(list >> 32)));
        }
    }
    if (a.ranks_of_row > 1) { cluster_arrive_relaxed(); cluster_wait(); }      // the first block has read what the others hold
    if (nf) nf->end(job_id);
}

typedef void (*LogprobsFn)(LogprobsArgs, uint32_t, FinishedBlockNotifier*);

struct LogprobsPlan {
    LogprobsArgs a;
    LogprobsFn fn;
    unsigned blocks;
};

int plan_logprobs(const pb_logprobs_params* p, LogprobsPlan& pl) {
    const char* who = "pb_logprobs";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(p->tokens >= 0 && p->vocab >= 1 && p->vocab <= 1 << 30, "%s: %d tokens, a vocabulary of %d", who, p->tokens, p->vocab);
    PB_REQUIRE(is_float_dtype(p->dtype), "%s: dtype %d (PB_F32, PB_BF16 or PB_F16)", who, p->dtype);
    PB_REQUIRE(p->top >= 0 && p->top <= kMaxTop && p->top <= p->vocab, "%s: top %d (0 to %d, at most vocab)", who, p->top, kMaxTop);
    PB_REQUIRE(p->scale >= 1e-6f && p->scale <= 1e6f, "%s: scale is not between 1e-6 and 1e6", who);
    if (p->tokens > 0) {
        const size_t es = dtype_bytes(p->dtype);
        PB_REQUIRE(p->logits && aligned(p->logits, es), "%s: logits are NULL or not aligned to their elements", who);
        PB_REQUIRE(p->targets || !(p->logprobs || p->ranks), "%s: logprobs and ranks need targets", who);
        PB_REQUIRE(p->top > 0 || !(p->top_ids || p->top_logprobs), "%s: top_ids and top_logprobs need top", who);
        PB_REQUIRE(p->logprobs || p->ranks || p->entropy || p->top_ids || p->top_logprobs, "%s: no output", who);
        PB_REQUIRE(aligned(p->targets, 4) && aligned(p->logprobs, 4) && aligned(p->ranks, 4) && aligned(p->entropy, 4) && aligned(p->top_ids, 4) && aligned(p->top_logprobs, 4), "%s: a buffer is not aligned to its elements", who);
        PB_REQUIRE(!(p->top_ids || p->top_logprobs) || rows_apart(p->tokens, p->top_stride, p->top), "%s: rows of top_ids overlap (stride %lld)", who, (long long)p->top_stride);
    }
    const bool top = p->top_ids || p->top_logprobs;
    LogprobsArgs& a = pl.a;
    a = {p->logits, p->targets, p->logprobs, p->entropy, p->top_logprobs, p->ranks, p->top_ids, p->logits_stride, p->top_stride, p->tokens, p->vocab, p->top, 1, p->scale, p->scale * kLog2e, 0.f, 0.f};
    a.slack = 16.f / a.c;
    a.far = 256.f / a.c;
    // Few rows: a cluster on each, as long as that gives SMs something to do and a block some vectors for each thread.
    while (a.ranks_of_row < kMaxRanks && (int64_t)p->tokens * a.ranks_of_row < 148 && p->vocab / (2 * a.ranks_of_row) >= 4096) a.ranks_of_row *= 2;
    const int64_t blocks = (int64_t)p->tokens * a.ranks_of_row;
    pl.blocks = blocks > 0 ? (unsigned)blocks : (unsigned)a.ranks_of_row;
    if (p->dtype == PB_F32) pl.fn = top ? logprobs_kernel<float, true> : logprobs_kernel<float, false>;
    else if (p->dtype == PB_BF16) pl.fn = top ? logprobs_kernel<__nv_bfloat16, true> : logprobs_kernel<__nv_bfloat16, false>;
    else pl.fn = top ? logprobs_kernel<__half, true> : logprobs_kernel<__half, false>;
    return PB_OK;
}

}  // namespace

uint32_t* lm_logprobs_error_flag_ptr() {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_logprobs_flag) != cudaSuccess) { cudaGetLastError(); return nullptr; }
    return (uint32_t*)p;
}

}  // namespace pb

using namespace pb;

extern "C" {

int pb_logprobs_info(const pb_logprobs_params* p, pb_launch_info* out) {
    LogprobsPlan pl;
    const int rc = plan_logprobs(p, pl);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_logprobs_info: NULL out");
    memset(out, 0, sizeof(*out));
    cudaFuncAttributes fa = {};
    if (cudaFuncGetAttributes(&fa, (const void*)pl.fn) != cudaSuccess) cudaGetLastError();        // (without a GPU: what the host knows)
    const uint64_t t = (uint64_t)p->tokens;
    out->num_blocks = pl.blocks;
    out->threads_per_block = kThreads;
    out->smem_per_block = (uint32_t)fa.sharedSizeBytes;
    out->regs_per_thread = (uint32_t)fa.numRegs;
    out->flops = 6 * t * p->vocab;
    out->bytes = t * (p->vocab * dtype_bytes(p->dtype) + (p->targets ? 4 : 0) + (p->logprobs ? 4 : 0) + (p->ranks ? 4 : 0) + (p->entropy ? 4 : 0) + (p->top_ids ? 4ull * p->top : 0) +
                      (p->top_logprobs ? 4ull * p->top : 0));
    return PB_OK;
}

int pb_logprobs_launch(const pb_logprobs_params* p, void* stream, uint32_t job_id, void* notifier) {
    LogprobsPlan pl;
    const int rc = plan_logprobs(p, pl);
    if (rc != PB_OK) return rc;
    return lm_launch("pb_logprobs", pl.fn, dim3(pl.blocks), dim3(kThreads), 0, (cudaStream_t)stream, pl.a.ranks_of_row, pl.a, job_id, (FinishedBlockNotifier*)notifier);
}

}  // extern "C"
