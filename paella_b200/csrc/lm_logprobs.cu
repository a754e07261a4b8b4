// Log probabilities of given tokens with their ranks, the entropy of each row of logits, and its likeliest tokens.
//
//   log p_t = s x_t - log sum_j exp(s x_j);   H = log S - sum_j e_j d_j / S   with d_j = s (x_j - m), e_j = exp(d_j), S = sum_j e_j
//
// Bound by issue slots and the exponentials beside the reading: nine instructions a logit, one of them on the special-function units, which take 59 us for what memory delivers in 82 (2048 rows of 131072 in bf16:
// 117 us, 4.6 TB/s, and 133 with the five likeliest tokens; 4096 rows of 32000 in fp16 72 us; 4 rows of 131072 in fp32 with twenty tokens 15 us).  Each
// thread runs along its own vectors of a row with a maximum m of its own, which it follows only once it has grown by 2^16, so that sums are
// rescaled a few times a row; all of a row's threads join at its end.
//
// The likeliest tokens come out of the same pass: a thread remembers the first of its vectors with its largest logit.  Tokens are ordered by keys of
// 64 bits, the logit's order above the index's, so that no two are equal.  The k-th largest of the threads' largest logits (the largest of four threads each) is a bound that k tokens reach; the few threads
// that have any have their vectors read again, from the caches, and what reaches the bound is put in order by counting, for each, those in front of it.  Where that is more than there is room for
// (rows whose large logits lie with few threads), those that came give a higher bound.
#include <cmath>

#include "lm.cuh"
#include "umma.cuh"

namespace pb {
namespace {

__device__ uint32_t g_logprobs_flag;

constexpr int kMaxTop = 32, kMaxRanks = 8, kList = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct LogprobsArgs {
    const void* logits;
    const int32_t* targets;
    float *logprobs, *entropy, *top_logprobs;
    int32_t *ranks, *top_ids;
    int64_t stride, top_stride;
    int tokens, vocab, top, ranks_of_row;      // ranks_of_row: blocks of a cluster that share a row out
    float scale, c, inv_c, slack, far;         // c: scale * log2(e); 16 and 256 in powers of two as differences of logits
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

// 32 bytes of logits, 16-byte aligned.
template <typename T> struct Logits {
    static constexpr int V = 32 / (int)sizeof(T);
    uint4 w[2];
    __device__ __forceinline__ void load(const T* p) {
        w[0] = __ldcg(reinterpret_cast<const uint4*>(p));
        w[1] = __ldcg(reinterpret_cast<const uint4*>(p) + 1);
    }
    __device__ __forceinline__ uint32_t word(int i) const { return (&w[i >> 2].x)[i & 3]; }
    // value pairs as they are multiplied
    __device__ __forceinline__ uint64_t pair(int i) const {
        if constexpr (sizeof(T) == 4) {
            return pack_f32x2(word(2 * i), word(2 * i + 1));
        } else if constexpr (std::is_same<T, __half>::value) {
            const uint32_t q = word(i);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q));
            return pack_f32x2(__float_as_uint(f.x), __float_as_uint(f.y));
        } else {
            return pack_f32x2(word(i) << 16, word(i) & 0xffff0000u);
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
            float t[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = max_nan(__uint_as_float(word(i)), __uint_as_float(word(i + 4)));
            return max_nan(max_nan(t[0], t[1]), max_nan(t[2], t[3]));
        } else {
            Two t[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = __hmax2_nan(two(i), two(i + 4));
            const Two m = __hmax2_nan(__hmax2_nan(t[0], t[1]), __hmax2_nan(t[2], t[3]));
            return max_nan(__low2float(m), __high2float(m));
        }
    }
    // none below `low` (no NaN among them)
    __device__ __forceinline__ void raise(T low) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t& x = (&w[i >> 2].x)[i & 3];
            if constexpr (sizeof(T) == 4) {
                x = __float_as_uint(fmaxf(__uint_as_float(x), low));
            } else {
                const Two m = __hmax2(two(i), both(low));
                x = *reinterpret_cast<const uint32_t*>(&m);
            }
        }
    }
    // how many are above `x`, or not below it (no NaN among them)
    template <bool OR_SAME> __device__ __forceinline__ int above(T x) const {
        if constexpr (sizeof(T) == 4) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) n += OR_SAME ? __uint_as_float(word(i)) >= x : __uint_as_float(word(i)) > x;
            return n;
        } else {
            Two n = OR_SAME ? __hge2(two(0), both(x)) : __hgt2(two(0), both(x));      // ones: whole numbers up to 256 are exact
#pragma unroll
            for (int i = 1; i < 8; ++i) n = __hadd2(n, OR_SAME ? __hge2(two(i), both(x)) : __hgt2(two(i), both(x)));
            return (int)(__low2float(n) + __high2float(n));
        }
    }

   private:
    using Two = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    __device__ __forceinline__ Two two(int i) const {
        const uint32_t x = word(i);
        return *reinterpret_cast<const Two*>(&x);
    }
    static __device__ __forceinline__ __half2 both(__half x) { return __half2half2(x); }
    static __device__ __forceinline__ __nv_bfloat162 both(__nv_bfloat16 x) { return __bfloat162bfloat162(x); }
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

// Blocks of 128 threads, eight an SM, so that one's end lies under the others' rows; 256 for few rows.  (4096 rows of 32000 in fp16 70 / 83 us, 2048 of 131072 in bf16 131 / 135.)
template <typename T, bool TOP, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) logprobs_kernel(const __grid_constant__ LogprobsArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    constexpr int V = Logits<T>::V, kWarps = kThreads / 32;
    __shared__ Sums s_sums[kWarps];
    __shared__ int s_before[kWarps];
    __shared__ uint64_t s_quads[TOP ? kThreads / 4 : 1], s_bound, s_top[TOP ? kMaxTop : 1], s_list[TOP ? kList : 1];
    __shared__ uint16_t s_who[TOP ? kThreads : 1];
    __shared__ int s_found, s_many;
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = threadIdx.x;
    const int rank = blockIdx.x % a.ranks_of_row, row = blockIdx.x / a.ranks_of_row;
    const bool live = row < a.tokens;
    const T* x = static_cast<const T*>(a.logits) + (live ? row : 0) * a.stride;
    // the row: logits until 16 bytes are aligned, n vectors, and those that are left.  This block's share of the vectors; the first block has the others, too.
    const int head = live ? min((int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T), a.vocab) : 0, n = live ? (a.vocab - head) / V : 0;
    const int first = (int)((int64_t)n * rank / a.ranks_of_row), last = (int)((int64_t)n * (rank + 1) / a.ranks_of_row);
    const int loose = live && rank == 0 ? a.vocab - n * V : 0;           // logits outside of the vectors: the first `head`, and those behind
    const T* body = x + head;
    // two vectors come while a third is worked on, the first ones while the target is looked up
    Logits<T> v[3];
    const auto load = [&](Logits<T>& to, int i) {
        if (i < last) to.load(body + (int64_t)i * V);
    };
    load(v[0], first + t);
    load(v[1], first + t + kThreads);
    int target = -1;
    if (live && a.targets) target = a.targets[row];
    if (target >= a.vocab && t == 0) atomicExch(&g_logprobs_flag, kFlagLmToken);
    const bool ranked = target >= 0 && target < a.vocab;
    const T wanted_as = ranked ? x[target] : lm_from_f<T>(0.f);
    const float wanted = lm_to_f<T>(wanted_as);
    const uint64_t wanted_key = ranked ? key_of(order_of(wanted), target) : ~0ull;

    Sums sums = {-INFINITY, 0.f, 0.f};
    int before = 0, at = -1;                  // logits in front of the target; the vector of the largest one
    uint32_t best = 0;
    float best_logit = -INFINITY, limit = __uint_as_float(0x7fffffffu);     // limit: vectors whose largest logit is not above it are the common ones
    T low = lm_from_f<T>(0.f);
    uint64_t S2[2] = {0, 0}, E2[2] = {0, 0};
    const uint64_t c2 = pack_f32x2(__float_as_uint(a.c), __float_as_uint(a.c));
    uint64_t minus_mc = 0;
    const int with_target = ranked && target >= head && target < head + n * V ? (target - head) / V : -1;
    float mc = 0.f;                           // m c, rounded: the common vectors' exponents are x c - mc, one operation
    // The sums of the common vectors, as pairs, into the others.  Their exponents are r = mc - m c too small, which mc's rounding left.
    const auto fold = [&]() {
        float lo, hi, elo, ehi;
        unpack_f32x2(add_f32x2(S2[0], S2[1]), lo, hi);
        unpack_f32x2(add_f32x2(E2[0], E2[1]), elo, ehi);
        if (lo + hi > 0.f) {
            const float r = fmaf(-sums.m, a.c, mc), f = ex2(r);
            sums.E = fmaf(fmaf(r, lo + hi, elo + ehi) * f, a.inv_c, sums.E);
            sums.S = fmaf(lo + hi, f, sums.S);
        }
        S2[0] = S2[1] = E2[0] = E2[1] = 0;
    };
    const auto take = [&](Logits<T>& v, int i) {
        const float top = v.top();
        if (TOP && top > best_logit) { best_logit = top; at = i; }
        if (!(top <= limit)) {
            // a first vector, one that is far above what came so far, or one with a NaN or infinity
            if (TOP) {
                if (top != top && best == 0) { best = 0xffffffffu; at = i; best_logit = INFINITY; }          // the first NaN: nothing comes in front of it
                else if (at < 0) at = i;
            }
            fold();
            if (top > sums.m && top < INFINITY) sums.rescale(top, a.c);
            // Logits far below the maximum are raised to `low`, where their exponentials are zeros: masks of -infinity need no case of their own.  Not where
            // logits are so large that `low` and the maximum are too near each other in their type: those go one by one.
            low = lm_from_f<T>(fmaxf(sums.m - a.far, lowest<T>()));
            // Nor where mc's rounding is so large that the exponents x c - mc leave fp32's range before `fold` can take it back, as from some 2^31 on (up to 16, an exponential is off by 2^-20 of itself).
            mc = sums.m * a.c;
            const bool common = sums.m > -INFINITY && (sums.m - lm_to_f<T>(low)) * a.c >= 200.f && fabsf(fmaf(-sums.m, a.c, mc)) <= 16.f;
            limit = common ? sums.m + a.slack : __uint_as_float(0x7fffffffu);
            minus_mc = pack_f32x2(__float_as_uint(-mc), __float_as_uint(-mc));
            if (!(top <= limit)) {
                if (top == -INFINITY) {
                    if (ranked && wanted == -INFINITY) before += max(min(target - (head + i * V), V), 0);
                    return;
                }
#pragma unroll 1
                for (int j = 0; j < V; ++j) {
                    const float logit = lm_to_f<T>(body[(int64_t)i * V + j]);
                    sums.add_logit(logit, a.c);
                    if (ranked) before += key_of(order_of(logit), head + i * V + j) > wanted_key;
                }
                return;
            }
        }
        if (ranked && top >= wanted) {
            if (i == with_target) {
#pragma unroll
                for (int j = 0; j < V; ++j) before += v[j] > wanted || (v[j] == wanted && head + i * V + j < target);
            } else {
                before += head + i * V < target ? v.template above<true>(wanted_as) : v.template above<false>(wanted_as);
            }
        }
        v.raise(low);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const uint64_t d = fma_f32x2(v.pair(j), c2, minus_mc);
            float lo, hi;
            unpack_f32x2(d, lo, hi);
            const uint64_t e = pack_f32x2(__float_as_uint(ex2(lo)), __float_as_uint(ex2(hi)));
            S2[j & 1] = add_f32x2(S2[j & 1], e);
            E2[j & 1] = fma_f32x2(e, d, E2[j & 1]);
        }
    };
    {
        int i = first + t;
        for (; i < last; i += 3 * kThreads) {
            load(v[2], i + 2 * kThreads);
            take(v[0], i);
            load(v[0], i + 3 * kThreads);
            if (i + kThreads < last) take(v[1], i + kThreads);
            load(v[1], i + 4 * kThreads);
            if (i + 2 * kThreads < last) take(v[2], i + 2 * kThreads);
        }
        fold();
    }
    if (at >= 0 && best == 0) best = order_of(best_logit);
    uint64_t loose_key = 0;
    if (t < loose) {
        const int index = t < head ? t : n * V + t;
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

    if constexpr (TOP) {
        // A bound that `top` tokens reach: the top-th largest of the quads' largest logits, each as if it were the last of its vector.
        uint64_t quad = at >= 0 ? key_of(best, head + at * V + V - 1) : 0;
#pragma unroll
        for (int o = 1; o < 4; o *= 2) {
            const uint64_t other = __shfl_xor_sync(0xffffffffu, quad, o);
            quad = other > quad ? other : quad;
        }
        if ((lane & 3) == 0) s_quads[t >> 2] = quad;
        if (t == 0) { s_bound = 0; s_found = s_many = 0; }
        __syncthreads();
        // the number of keys in front of mine
        const auto place = [&](const uint64_t* keys, int count, uint64_t mine) {
            int in_front = 0;
#pragma unroll 8
            for (int i = 0; i < count; ++i) in_front += keys[i] > mine;
            return in_front;
        };
        if (t < kThreads / 4 && s_quads[t] > 0 && place(s_quads, kThreads / 4, s_quads[t]) == a.top - 1) s_bound = s_quads[t];
        __syncthreads();
        while (true) {
            const uint64_t bound = s_bound;
            const auto found = [&](uint64_t key) {
                if (key < bound) return;
                const int i = atomicAdd(&s_found, 1);
                if (i < kList) s_list[i] = key;
            };
            if (loose_key) found(loose_key);
            // threads with a logit that may reach the bound: the warps look through their vectors in turn
            if (at >= 0 && key_of(best, head + at * V) >= bound) s_who[atomicAdd(&s_many, 1)] = (uint16_t)t;
            __syncthreads();
            const float reach = logit_of((uint32_t)(bound >> 32));
            for (int w = warp; w < s_many; w += kWarps)
                for (int i = first + s_who[w] + lane * kThreads; i < last; i += 32 * kThreads) {
                    Logits<T> v;
                    v.load(body + (int64_t)i * V);
                    uint32_t there = 0;
#pragma unroll
                    for (int j = 0; j < V; ++j) there |= (uint32_t)!(v[j] < reach) << j;
                    while (there) {
                        const int j = __ffs(there) - 1;
                        there &= there - 1;
                        found(key_of(order_of(lm_to_f<T>(body[(int64_t)i * V + j])), head + i * V + j));
                    }
                }
            __syncthreads();
            const int count = s_found;
            if (count <= kList) break;
            // More than there is room for: those that came are a bound again, a higher one.
            uint64_t mine[kList / kThreads];
            for (int k = 0; k < kList / kThreads; ++k) mine[k] = s_list[t + k * kThreads];
            for (int k = 0; k < kList / kThreads; ++k)
                if (place(s_list, kList, mine[k]) == a.top - 1) s_bound = mine[k];
            __syncthreads();
            if (t == 0) s_found = s_many = 0;
            __syncthreads();
        }
        const int count = s_found;
        for (int i = t; i < count; i += kThreads) {
            const int p = place(s_list, count, s_list[i]);
            if (p < a.top) s_top[p] = s_list[i];
        }
        for (int i = count + t; i < a.top; i += kThreads) s_top[i] = 0;   // (a block of a cluster whose share is that small)
    }
    __syncthreads();
    if (a.ranks_of_row > 1) { cluster_arrive(); cluster_wait(); }
    if (TOP && a.ranks_of_row > 1 && rank == 0) {
        // all blocks' first tokens
        static_assert(kThreads < 256 || (kMaxRanks <= kWarps && kThreads <= kList), "a warp for each block's list");
        uint64_t mine = 0;
        if (lane < a.top && warp < a.ranks_of_row) asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(mine) : "r"(cluster_addr(smem_u32(&s_top[lane]), (uint32_t)warp)) : "memory");
        __syncthreads();
        s_list[t] = mine;
        __syncthreads();
        int p = 0;
        for (int r = 0; r < a.ranks_of_row; ++r)
            for (int i = 0; i < a.top; ++i) p += s_list[32 * r + i] > mine;
        if (mine > 0 && p < a.top) s_top[p] = mine;
        __syncthreads();
    }
    if (rank == 0 && warp == 0 && live) {
        // all warps' sums of all blocks: a warp a lane, block after block
        Sums all = {-INFINITY, 0.f, 0.f};
        int count = 0;
        Sums o[kMaxRanks];
        int b[kMaxRanks];
#pragma unroll
        for (int r = 0; r < kMaxRanks; ++r) {
            o[r] = {-INFINITY, 0.f, 0.f};
            b[r] = 0;
            if (r < a.ranks_of_row && lane < kWarps) {
                const uint32_t from = cluster_addr(smem_u32(&s_sums[lane]), (uint32_t)r);
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o[r].m) : "r"(from) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o[r].S) : "r"(from + 4) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o[r].E) : "r"(from + 8) : "memory");
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(b[r]) : "r"(cluster_addr(smem_u32(&s_before[lane]), (uint32_t)r)) : "memory");
            }
        }
#pragma unroll 1
        for (int r = 0; r < kMaxRanks; ++r) {
            if (r < a.ranks_of_row) {
                all.add(o[0], a.c);
                count += b[0];
            }
#pragma unroll
            for (int k = 0; k + 1 < kMaxRanks; ++k) { o[k] = o[k + 1]; b[k] = b[k + 1]; }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            Sums other;
            other.m = __shfl_xor_sync(0xffffffffu, all.m, d);
            other.S = __shfl_xor_sync(0xffffffffu, all.S, d);
            other.E = __shfl_xor_sync(0xffffffffu, all.E, d);
            Sums lower = lane & d ? other : all;
            lower.add(lane & d ? all : other, a.c);
            all = lower;
            count += __shfl_xor_sync(0xffffffffu, count, d);
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
            const uint64_t key = s_top[lane];
            if (a.top_ids) a.top_ids[row * a.top_stride + lane] = index_of(key);
            if (a.top_logprobs) a.top_logprobs[row * a.top_stride + lane] = logprob(logit_of((uint32_t)(key >> 32)));
        }
    }
    if (a.ranks_of_row > 1) { cluster_arrive_relaxed(); cluster_wait(); }      // the first block has read what the others hold
    if (nf) nf->end(job_id);
}

typedef void (*LogprobsFn)(LogprobsArgs, uint32_t, FinishedBlockNotifier*);

struct LogprobsPlan {
    LogprobsArgs a;
    LogprobsFn fn;
    unsigned blocks, threads;
};

template <typename T> LogprobsFn pick(bool top, unsigned threads) {
    if (threads == 128) return top ? logprobs_kernel<T, true, 128> : logprobs_kernel<T, false, 128>;
    return top ? logprobs_kernel<T, true, 256> : logprobs_kernel<T, false, 256>;
}

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
    a = {p->logits, p->targets, p->logprobs, p->entropy, p->top_logprobs, p->ranks, p->top_ids, p->logits_stride, p->top_stride, p->tokens, p->vocab, p->top, 1, p->scale, p->scale * kLog2e, 0.f, 0.f, 0.f};
    a.inv_c = 1.f / a.c;
    a.slack = 16.f / a.c;
    a.far = 256.f / a.c;
    // Few rows: a cluster on each, as long as that gives SMs something to do and a block some vectors for each thread.
    while (a.ranks_of_row < kMaxRanks && (int64_t)p->tokens * a.ranks_of_row < 148 && p->vocab / (2 * a.ranks_of_row) >= 4096) a.ranks_of_row *= 2;
    const int64_t blocks = (int64_t)p->tokens * a.ranks_of_row;
    pl.blocks = blocks > 0 ? (unsigned)blocks : (unsigned)a.ranks_of_row;
    pl.threads = blocks >= 4 * 148 ? 128 : 256;                // (clusters have fewer blocks)
    if (p->dtype == PB_F32) pl.fn = pick<float>(top, pl.threads);
    else if (p->dtype == PB_BF16) pl.fn = pick<__nv_bfloat16>(top, pl.threads);
    else pl.fn = pick<__half>(top, pl.threads);
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
    out->threads_per_block = pl.threads;
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
    return lm_launch("pb_logprobs", pl.fn, dim3(pl.blocks), dim3(pl.threads), 0, (cudaStream_t)stream, pl.a.ranks_of_row, pl.a, job_id, (FinishedBlockNotifier*)notifier);
}

}  // extern "C"
