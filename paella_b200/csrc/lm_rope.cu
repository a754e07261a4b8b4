// Norms of queries and keys for each head with the rotation by position, and the same on the way into a paged cache.
//
//   z = x * w / sqrt(mean(x^2) + eps);   (a, b) -> (a c - b s, b c + a s) for the pairs of the first rot_dim values
//
// Both are bound by memory: every head is read once and written once, 4 operations a byte.  A group of lanes takes a head, each
// lane both halves of its pairs, so that the rotation needs no exchange and only the norm's sum does (three shuffles for a head
// of 128 values in 16 bits, whose group is eight lanes).  Everything is in fp32 and rounded once.  Few tokens are a chain of latencies (one token into
// the cache: 2.5 us, 48 tokens of 40 heads 2.5 to 4; launches back to back in a graph, as all figures here); for many a group takes up to eight neighbouring heads of a token.
// The two kernels add squares and multiply norm, weight and rotation in different orders, so a token's last fp32 bit depends on which of them takes it.
#include <cuda.h>

#include "lm.cuh"
#include "umma.cuh"

namespace pb {
namespace {

__device__ uint32_t g_rope_flag;

// One class of heads: queries, keys or values.  dst is found from the slot for keys and values of an append.
struct HeadSet {
    const void* src;
    void* dst;
    const float* weight;
    int64_t src_token, src_head, dst_token, dst_head;
};

struct RopeArgs {
    HeadSet set[3];            // queries, keys, values
    int first[3];              // heads before the end of each set: queries, then keys, then values
    int tokens, head_dim, rot_dim, interleaved, max_position, lanes;   // lanes: of a group, a power of two
    int slices;                // groups that share a token's heads out
    float eps, inv_dim;
    const float* cos_sin;
    const int32_t* positions;
    // an append: keys and values go to pages
    const int64_t* slots;      // NULL otherwise
    int64_t n_slots, page_stride, row_stride;
    int page_size;
    int wide_weights;          // weights are 16-byte aligned
};

// V values are an access, a lane takes CH chunks of 2 V values, a group one head of a token: few heads, or any alignment.
template <typename T, int V, int CH>
__global__ void __launch_bounds__(256) rope_kernel(const __grid_constant__ RopeArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    using Vt = LmVec<T, V>;
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int lane = threadIdx.x & (a.lanes - 1);
    const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) / a.lanes;
    const int64_t token = group >> 32 ? group / a.slices : (uint32_t)group / (uint32_t)a.slices;    // (a 64-bit quotient takes some 70 instructions)
    const int head = (int)(group - token * a.slices);
    bool live = token < a.tokens;
    int pos = 0;
    int64_t slot = 0;
    if (live && a.rot_dim) pos = a.positions[token];
    if (live && a.slots) slot = a.slots[token];
    // where this lane's chunks lie: `lo` and `hi`, V values each
    const int half = a.rot_dim / 2, turned = half / V;
    int lo[CH], hi[CH];                                  // -1 = none
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = lane + c * a.lanes;
        if (i < turned) {
            lo[c] = a.interleaved ? 2 * V * i : V * i;
            hi[c] = a.interleaved ? lo[c] + V : lo[c] + half;
        } else {
            lo[c] = a.rot_dim + 2 * V * (i - turned);
            hi[c] = lo[c] + V;
        }
        if (lo[c] >= a.head_dim) lo[c] = -1;
        if (hi[c] >= a.head_dim) hi[c] = -1;
    }
    Vt x[CH][2];
    const int kind = head < a.first[0] ? 0 : head < a.first[1] ? 1 : 2, within = head - (kind ? a.first[kind - 1] : 0);
    const HeadSet& s = a.set[kind];
    if (live) {
        const T* src = static_cast<const T*>(s.src) + token * s.src_token + within * s.src_head;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int at = p ? hi[c] : lo[c];
                if (at >= 0) x[c][p] = *reinterpret_cast<const Vt*>(src + at);
            }
    }
    bool store = true;                                   // keys and values of this token are stored
    int64_t page = 0;
    if (live && a.slots) {
        store = slot >= 0;
        if (slot >= a.n_slots) {
            if (lane == 0) atomicExch(&g_rope_flag, kFlagLmSlot);
            live = false;
        }
        page = slot >> 32 ? slot / a.page_size : (uint32_t)slot / (uint32_t)a.page_size;
        slot -= page * a.page_size;
    }
    if (live && a.rot_dim && (pos < 0 || pos >= a.max_position)) {
        if (lane == 0 && store) atomicExch(&g_rope_flag, kFlagLmPosition);
        live = false;
    }
    float co[CH][V], si[CH][V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = lane + c * a.lanes;
        if (live && i < turned) {
            const float* row = a.cos_sin + (int64_t)pos * a.rot_dim + V * i;
            constexpr int W = V < 4 ? V : 4;
#pragma unroll
            for (int j = 0; j < V; j += W) {
                const LmVec<float, W> cv = *reinterpret_cast<const LmVec<float, W>*>(row + j);
                const LmVec<float, W> sv = *reinterpret_cast<const LmVec<float, W>*>(row + half + j);
#pragma unroll
                for (int k = 0; k < W; ++k) { co[c][j + k] = cv.v[k]; si[c][j + k] = sv.v[k]; }
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) { co[c][j] = 1.f; si[c][j] = 0.f; }
        }
    }
    const int w = live && (kind == 0 || store) ? kind : -1;
    if (!__all_sync(0xffffffffu, w < 0)) {
        const float* weight = w < 0 ? nullptr : s.weight;
        T* dst = static_cast<T*>(s.dst) + within * s.dst_head + (kind && a.slots ? page * a.page_stride + slot * a.row_stride : token * s.dst_token);
        float z[CH][2][V];
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const bool there = w >= 0 && (p ? hi[c] : lo[c]) >= 0;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    z[c][p][j] = there ? lm_to_f<T>(x[c][p].v[j]) : 0.f;
                    sum += z[c][p][j] * z[c][p][j];
                }
            }
        if (__any_sync(0xffffffffu, weight != nullptr))
            for (int o = a.lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (weight) {
            const float r = rsqrtf(sum * a.inv_dim + a.eps);
            constexpr int W = V < 4 ? V : 4;             // (weights may lie at any float: wide accesses only where they do not)
            const bool wide = V >= 4 && a.wide_weights;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int at = p ? hi[c] : lo[c];
                    if (at < 0) continue;
                    if (wide) {
#pragma unroll
                        for (int j = 0; j < V; j += W) {
                            const LmVec<float, W> wv = *reinterpret_cast<const LmVec<float, W>*>(weight + at + j);
#pragma unroll
                            for (int k = 0; k < W; ++k) z[c][p][j + k] *= r * wv.v[k];
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < V; ++j) z[c][p][j] *= r * weight[at + j];
                    }
                }
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            Vt out[2];
            const int i = lane + c * a.lanes;
            const bool turn = w < 2 && i < turned;
            if (turn && a.interleaved) {
#pragma unroll
                for (int j = 0; j < V; ++j) {            // pair j of the chunk: values 2 j and 2 j + 1
                    const float A = 2 * j < V ? z[c][0][(2 * j) % V] : z[c][1][(2 * j) % V];
                    const float B = 2 * j + 1 < V ? z[c][0][(2 * j + 1) % V] : z[c][1][(2 * j + 1) % V];
                    out[(2 * j) / V].v[(2 * j) % V] = lm_from_f<T>(A * co[c][j] - B * si[c][j]);
                    out[(2 * j + 1) / V].v[(2 * j + 1) % V] = lm_from_f<T>(B * co[c][j] + A * si[c][j]);
                }
            } else if (turn) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    out[0].v[j] = lm_from_f<T>(z[c][0][j] * co[c][j] - z[c][1][j] * si[c][j]);
                    out[1].v[j] = lm_from_f<T>(z[c][1][j] * co[c][j] + z[c][0][j] * si[c][j]);
                }
            } else if (weight) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    out[0].v[j] = lm_from_f<T>(z[c][0][j]);
                    out[1].v[j] = lm_from_f<T>(z[c][1][j]);
                }
            } else {                                     // as it was, a NaN's bits too
                out[0] = x[c][0];
                out[1] = x[c][1];
            }
            if (w >= 0 && lo[c] >= 0) *reinterpret_cast<Vt*>(dst + lo[c]) = out[0];
            if (w >= 0 && hi[c] >= 0) *reinterpret_cast<Vt*>(dst + hi[c]) = out[1];
        }
    }
    if (nf) nf->end(job_id);
}

__device__ __forceinline__ uint64_t two(float x, float y) { return pack_f32x2(__float_as_uint(x), __float_as_uint(y)); }
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// 16 bytes of each half of a lane's chunk to pairs of floats, A and B of the pairs (j, j + 1), and back
template <typename T, bool interleaved>
__device__ __forceinline__ void spread(uint4 lo, uint4 hi, uint64_t (&A)[8 / sizeof(T)], uint64_t (&B)[8 / sizeof(T)]) {
    const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
    if constexpr (sizeof(T) == 4) {
        if (interleaved) {
            A[0] = pack_f32x2(l[0], l[2]); B[0] = pack_f32x2(l[1], l[3]); A[1] = pack_f32x2(h[0], h[2]); B[1] = pack_f32x2(h[1], h[3]);
        } else {
            A[0] = pack_f32x2(l[0], l[1]); A[1] = pack_f32x2(l[2], l[3]); B[0] = pack_f32x2(h[0], h[1]); B[1] = pack_f32x2(h[2], h[3]);
        }
    } else {
        if (interleaved) {
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                const float2 x = unpack2<T>(l[k]), y = unpack2<T>(l[k + 1]), u = unpack2<T>(h[k]), v = unpack2<T>(h[k + 1]);
                A[k / 2] = two(x.x, y.x); B[k / 2] = two(x.y, y.y);
                A[2 + k / 2] = two(u.x, v.x); B[2 + k / 2] = two(u.y, v.y);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 x = unpack2<T>(l[k]), u = unpack2<T>(h[k]);
                A[k] = two(x.x, x.y);
                B[k] = two(u.x, u.y);
            }
        }
    }
}
template <typename T, bool interleaved>
__device__ __forceinline__ void gather(const uint64_t (&A)[8 / sizeof(T)], const uint64_t (&B)[8 / sizeof(T)], uint4& lo, uint4& hi) {
    uint32_t l[4], h[4];
    constexpr int N = 8 / sizeof(T);
    float a[2 * N], b[2 * N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        unpack_f32x2(A[j], a[2 * j], a[2 * j + 1]);
        unpack_f32x2(B[j], b[2 * j], b[2 * j + 1]);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            l[k] = __float_as_uint(interleaved ? (k & 1 ? b[k / 2] : a[k / 2]) : a[k]);
            h[k] = __float_as_uint(interleaved ? (k & 1 ? b[2 + k / 2] : a[2 + k / 2]) : b[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            l[k] = interleaved ? lm_pack2<T>(a[k], b[k]) : lm_pack2<T>(a[2 * k], a[2 * k + 1]);
            h[k] = interleaved ? lm_pack2<T>(a[4 + k], b[4 + k]) : lm_pack2<T>(b[2 * k], b[2 * k + 1]);
        }
    }
    lo = make_uint4(l[0], l[1], l[2], l[3]);
    hi = make_uint4(h[0], h[1], h[2], h[3]);
}

// The same for many heads, in accesses of 16 bytes: a lane's values wait in shared memory, in slots of its own, so that a thread has 128 or 256 bytes on the way
// and an SM 96 or 192 KB, which cover the latency of x and, behind the position, of the rotation's row.  What the general kernel spends most on beside the
// transfers, weights and rotation for each head, is found once here: products of weight and cosine or sine of a lane's pairs, again only where
// queries end and keys begin.  16384 tokens of 40 heads of 128 in bf16, 344 MB: 72 us, 4.8 TB/s, 74 % of the copy rate (118 by the general kernel);
// what is left is a block's chain of copies, norms and heads one after the other.  Three blocks an SM leave a thread 80 registers, of which 16-bit types need 18 or 19 more and fp32
// in halves 3: those are kept in local memory.
template <typename T, int HEADS, bool interleaved>
__global__ void __launch_bounds__(256, 3) rope_many_kernel(const __grid_constant__ RopeArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    constexpr int V = 16 / (int)sizeof(T), N = V / 2;
    extern __shared__ __align__(16) uint4 s_values[];    // [2 HEADS][256]
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int lane = threadIdx.x & (a.lanes - 1);
    const uint32_t mates = (a.lanes == 32 ? 0xffffffffu : (1u << a.lanes) - 1u) << (threadIdx.x & 31 & ~(a.lanes - 1));     // the group's lanes
    const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) / a.lanes;
    const int64_t token = group >> 32 ? group / a.slices : (uint32_t)group / (uint32_t)a.slices;
    const int head0 = (int)(group - token * a.slices) * HEADS;
    bool live = token < a.tokens;
    const int count = live ? min(HEADS, a.first[2] - head0) : 0;
    int pos = 0;
    int64_t slot = 0;
    if (live && a.rot_dim) pos = a.positions[token];
    if (live && a.slots) slot = a.slots[token];
    // This lane's two vectors of V values.  In halves: V values of the first half and their partners.  Pairs side by side: vectors `lane` and `lane` + half
    // their number, so that neighbouring lanes have neighbouring bytes; what is not rotated in the same way.
    const int half = a.rot_dim / 2, turned = half / V, rest = interleaved ? a.head_dim / V : (a.head_dim - a.rot_dim) / V, first = interleaved ? lane : lane - turned;
    const int from = interleaved ? 0 : a.rot_dim, second = first + (rest + 1) / 2;
    const bool in_halves = !interleaved && lane < turned;
    const int lo = in_halves ? V * lane : first < (rest + 1) / 2 ? from + V * first : a.head_dim, hi = in_halves ? V * lane + half : second < rest ? from + V * second : a.head_dim;
    const bool turn_lo = lo < a.rot_dim, turn_hi = hi < a.rot_dim;
    const bool has_lo = lo < a.head_dim, has_hi = hi < a.head_dim;
    const auto set_of = [&](int head) { return head < a.first[0] ? 0 : head < a.first[1] ? 1 : 2; };
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&s_values[threadIdx.x]);
    for (int h = 0; h < count;) {
        const int w = set_of(head0 + h), end = min(count, a.first[w] - head0);
        const T* src = static_cast<const T*>(a.set[w].src) + token * a.set[w].src_token + (head0 + h - (w ? a.first[w - 1] : 0)) * a.set[w].src_head;
        for (; h < end; ++h, src += a.set[w].src_head) {
            if (has_lo) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + h * 8192), "l"(src + lo) : "memory");
            if (has_hi) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + h * 8192 + 4096), "l"(src + hi) : "memory");
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    bool store = true;                                   // keys and values of this token are stored
    int64_t page = 0;
    if (live && a.slots) {
        store = slot >= 0;
        if (slot >= a.n_slots) {
            if (lane == 0) atomicExch(&g_rope_flag, kFlagLmSlot);
            live = false;
        }
        page = slot >> 32 ? slot / a.page_size : (uint32_t)slot / (uint32_t)a.page_size;
        slot -= page * a.page_size;
    }
    if (live && a.rot_dim && (pos < 0 || pos >= a.max_position)) {
        if (lane == 0 && store) atomicExch(&g_rope_flag, kFlagLmPosition);
        live = false;
    }
    float cosines[V], sines[V];                          // of pairs j
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        constexpr int W = V / 2;
        const int pair = interleaved ? (p ? hi : lo) / 2 : lo + p * W;
        LmVec<float, W> c, n;
#pragma unroll
        for (int k = 0; k < W; ++k) c.v[k] = 1.f, n.v[k] = 0.f;
        if (live && (interleaved && p ? turn_hi : turn_lo)) {
            const float* row = a.cos_sin + (int64_t)pos * a.rot_dim + pair;
            c = *reinterpret_cast<const LmVec<float, W>*>(row);
            n = *reinterpret_cast<const LmVec<float, W>*>(row + half);
        }
#pragma unroll
        for (int k = 0; k < W; ++k) cosines[p * W + k] = c.v[k], sines[p * W + k] = n.v[k];
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // The norms of all heads first: eight sums over the lanes side by side, where one after the other each head would wait for three shuffles and a root.
    float* const norms = reinterpret_cast<float*>(s_values + 2 * HEADS * 256) + threadIdx.x;     // [HEADS][256]
    if (live && (a.set[0].weight || a.set[1].weight)) {
        float sum[HEADS];
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            uint64_t sum2 = 0;
            if (head0 + h < a.first[1]) {
                uint64_t A[N], B[N];
                uint4 lv = make_uint4(0, 0, 0, 0), hv = lv;
                if (has_lo) lv = s_values[2 * h * 256 + threadIdx.x];
                if (has_hi) hv = s_values[(2 * h + 1) * 256 + threadIdx.x];
                spread<T, interleaved>(lv, hv, A, B);
#pragma unroll
                for (int j = 0; j < N; ++j) sum2 = fma_f32x2(B[j], B[j], fma_f32x2(A[j], A[j], sum2));
            }
            float x, y;
            unpack_f32x2(sum2, x, y);
            sum[h] = x + y;
        }
        for (int o = a.lanes >> 1; o > 0; o >>= 1)
#pragma unroll
            for (int h = 0; h < HEADS; ++h) sum[h] += __shfl_xor_sync(mates, sum[h], o);
#pragma unroll
        for (int h = 0; h < HEADS; ++h) norms[h * 256] = rsqrtf(sum[h] * a.inv_dim + a.eps);
    }
    // Heads of one kind after another.  (The lanes of a group go through this together, the groups of a warp need not.)
    for (int h = 0; h < count && live;) {
        const int w = set_of(head0 + h), end = min(count, a.first[w] - head0);
        const HeadSet& s = a.set[w];
        if (w && !store) { h = end; continue; }
        T* dst = static_cast<T*>(s.dst) + (head0 + h - (w ? a.first[w - 1] : 0)) * s.dst_head + (w && a.slots ? page * a.page_stride + slot * a.row_stride : token * s.dst_token);
        const float* weight = s.weight;
        if (w == 2 || (!weight && !a.rot_dim)) {         // as they are, a NaN's bits too
            for (; h < end; ++h, dst += s.dst_head) {
                if (has_lo) *reinterpret_cast<uint4*>(dst + lo) = s_values[2 * h * 256 + threadIdx.x];
                if (has_hi) *reinterpret_cast<uint4*>(dst + hi) = s_values[(2 * h + 1) * 256 + threadIdx.x];
            }
            continue;
        }
        // out A = r (A ca + B nb), out B = r (B cb + A sa) with ca = wa cos, nb = -wb sin, cb = wb cos, sa = wa sin
        uint64_t ca[N], cb[N], sa[N], nb[N];
        float w_lo[V], w_hi[V];
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            float4 x = make_float4(1.f, 1.f, 1.f, 1.f), y = x;
            if (weight && has_lo) x = a.wide_weights ? *reinterpret_cast<const float4*>(weight + lo + j) : make_float4(weight[lo + j], weight[lo + j + 1], weight[lo + j + 2], weight[lo + j + 3]);
            if (weight && has_hi) y = a.wide_weights ? *reinterpret_cast<const float4*>(weight + hi + j) : make_float4(weight[hi + j], weight[hi + j + 1], weight[hi + j + 2], weight[hi + j + 3]);
            w_lo[j] = x.x; w_lo[j + 1] = x.y; w_lo[j + 2] = x.z; w_lo[j + 3] = x.w;
            w_hi[j] = y.x; w_hi[j + 1] = y.y; w_hi[j + 2] = y.z; w_hi[j + 3] = y.w;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            // (interleaved: pairs 2 j and 2 j + 1 are values 4 j to 4 j + 3 of the lane's 2 V)
            const float* w4 = 4 * j < V ? w_lo + 4 * j : w_hi + (4 * j - V);
            const uint64_t x = interleaved ? two(w4[0], w4[2]) : two(w_lo[2 * j], w_lo[2 * j + 1]), y = interleaved ? two(w4[1], w4[3]) : two(w_hi[2 * j], w_hi[2 * j + 1]);
            ca[j] = mul_f32x2(x, two(cosines[2 * j], cosines[2 * j + 1]));
            cb[j] = mul_f32x2(y, two(cosines[2 * j], cosines[2 * j + 1]));
            sa[j] = mul_f32x2(x, two(sines[2 * j], sines[2 * j + 1]));
            nb[j] = mul_f32x2(y, two(-sines[2 * j], -sines[2 * j + 1]));
        }
        for (; h < end; ++h, dst += s.dst_head) {
            uint4 lv = make_uint4(0, 0, 0, 0), hv = lv;
            if (has_lo) lv = s_values[2 * h * 256 + threadIdx.x];
            if (has_hi) hv = s_values[(2 * h + 1) * 256 + threadIdx.x];
            uint64_t A[N], B[N];
            spread<T, interleaved>(lv, hv, A, B);
            if (weight) {
                const float r = norms[h * 256];
                const uint64_t r2 = two(r, r);
#pragma unroll
                for (int j = 0; j < N; ++j) A[j] = mul_f32x2(A[j], r2), B[j] = mul_f32x2(B[j], r2);
            }
            if (weight || turn_lo) {                     // (a lane whose second vector alone turned does not exist)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const uint64_t x = A[j], y = B[j];
                    A[j] = mul_f32x2(x, ca[j]);
                    B[j] = mul_f32x2(y, cb[j]);
                    if (interleaved && 2 * j >= N ? turn_hi : turn_lo) {
                        A[j] = fma_f32x2(y, nb[j], A[j]);
                        B[j] = fma_f32x2(x, sa[j], B[j]);
                    }
                }
                gather<T, interleaved>(A, B, lv, hv);
            }
            if (has_lo) *reinterpret_cast<uint4*>(dst + lo) = lv;
            if (has_hi) *reinterpret_cast<uint4*>(dst + hi) = hv;
        }
    }
    if (nf) nf->end(job_id);
}

typedef void (*RopeFn)(RopeArgs, uint32_t, FinishedBlockNotifier*);

struct RopePlan {
    RopeArgs a;
    RopeFn fn;
    unsigned blocks;
    int smem;
};

// All accesses of V values of `es` bytes of this set are aligned to their size.
bool vectors_fit(const HeadSet& s, int heads, int V, size_t es) {
    if (!heads) return true;
    return aligned(s.src, V * es) && aligned(s.dst, V * es) && s.src_token % V == 0 && s.src_head % V == 0 && s.dst_token % V == 0 && s.dst_head % V == 0;
}

template <typename T>
RopeFn pick(bool wide, int heads, bool interleaved) {
    constexpr int VN = 16 / (int)sizeof(T);
    if (!wide) return rope_kernel<T, 1, 4>;
    if (heads == 8) return interleaved ? rope_many_kernel<T, 8, true> : rope_many_kernel<T, 8, false>;
    if (heads == 4) return interleaved ? rope_many_kernel<T, 4, true> : rope_many_kernel<T, 4, false>;
    return rope_kernel<T, VN, 1>;
}

int plan_rope(const char* who, int dtype, RopePlan& pl) {
    RopeArgs& a = pl.a;
    const size_t es = dtype_bytes(dtype);
    const int VN = (int)(16 / es);
    // 16 bytes an access where every pair's halves, every head and every row of the table allow it, single values otherwise
    bool wide = (a.rot_dim / 2) % VN == 0 && a.head_dim % VN == 0 && (a.rot_dim == 0 || aligned(a.cos_sin, 16));
    int before = 0;
    for (int i = 0; i < 3; ++i) {
        wide = wide && vectors_fit(a.set[i], a.first[i] - before, VN, es);
        before = a.first[i];
    }
    if (a.slots) wide = wide && a.page_stride % VN == 0 && a.row_stride % VN == 0;
    a.inv_dim = 1.f / (float)a.head_dim;
    a.wide_weights = aligned(a.set[0].weight, 16) && aligned(a.set[1].weight, 16);
    const int V = wide ? VN : 1;
    int chunks = a.rot_dim / 2 / V + ceil_div(a.head_dim - a.rot_dim, 2 * V);
    const int per_lane = wide ? 1 : 4;
    a.lanes = 1;
    while (a.lanes * per_lane < chunks) a.lanes *= 2;
    const int heads = a.first[2];
    // Heads of a group: eight (four of few) once that gives every SM a block and a half, one below.  (40 heads of 128 in bf16, one / four / eight: 700 tokens
    // 5.8 / 5.8 / 6.2 us, 1500 12.7 / 11.8 / 11.8, 3000 24 / 20 / 20, 16384 118 / 80 / 72.)
    int each = 1;
    if (wide && heads > 1 && (int64_t)a.tokens * ceil_div(heads, heads > 4 ? 8 : 4) * a.lanes >= 148 * 384) each = heads > 4 ? 8 : 4;
    a.slices = ceil_div(heads, each);
    const int64_t blocks = ceil_div<int64_t>((int64_t)a.tokens * a.slices * a.lanes, 256);
    PB_REQUIRE(blocks <= 0x7fffffff, "%s: %d tokens of %d heads are too many for one launch", who, a.tokens, heads);
    pl.blocks = blocks > 0 ? (unsigned)blocks : 1u;
    pl.fn = dtype == PB_F32 ? pick<float>(wide, each, a.interleaved) : dtype == PB_BF16 ? pick<__nv_bfloat16>(wide, each, a.interleaved) : pick<__half>(wide, each, a.interleaved);
    pl.smem = each >= 4 ? each * (8192 + 1024) : 0;
    return PB_OK;
}

int check_heads(const char* who, int dtype, int tokens, int q_heads, int kv_heads, int head_dim, int rot_dim, int max_position, const float* cos_sin, const int32_t* positions) {
    PB_REQUIRE(is_float_dtype(dtype), "%s: dtype %d (PB_F32, PB_BF16 or PB_F16)", who, dtype);
    PB_REQUIRE(tokens >= 0, "%s: %d tokens", who, tokens);
    PB_REQUIRE(q_heads >= 0 && kv_heads >= 0 && q_heads <= 65536 && kv_heads <= 65536, "%s: %d query heads, %d key heads", who, q_heads, kv_heads);
    PB_REQUIRE(head_dim >= 1 && head_dim <= 256, "%s: head_dim %d (1 to 256)", who, head_dim);
    PB_REQUIRE(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 2 == 0, "%s: rot_dim %d (even, 0 to head_dim %d)", who, rot_dim, head_dim);
    PB_REQUIRE(rot_dim == 0 || tokens == 0 || (max_position > 0 && cos_sin && positions && aligned(cos_sin, 4) && aligned(positions, 4)), "%s: a rotation needs cos_sin, positions and max_position", who);
    return PB_OK;
}

bool heads_apart(int64_t tokens, int heads, int head_dim, int64_t stride, int64_t head_stride) {
    return heads == 0 || (rows_apart(tokens, stride, head_dim) && rows_apart(heads, head_stride, head_dim));
}

int rope_plan(const pb_qk_rope_params* p, RopePlan& pl) {
    const char* who = "pb_qk_rope";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    const int rc = check_heads(who, p->dtype, p->tokens, p->q_heads, p->kv_heads, p->head_dim, p->rot_dim, p->max_position, p->cos_sin, p->positions);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(p->q_heads + p->kv_heads > 0, "%s: no heads", who);
    PB_REQUIRE(heads_apart(p->tokens, p->q_heads, p->head_dim, p->q_out_stride, p->q_out_head_stride) && heads_apart(p->tokens, p->kv_heads, p->head_dim, p->k_out_stride, p->k_out_head_stride),
               "%s: rows of q_out or k_out overlap", who);
    const size_t es = dtype_bytes(p->dtype);
    if (p->tokens > 0) {
        PB_REQUIRE(p->q_heads == 0 || (p->q && p->q_out), "%s: NULL q or q_out", who);
        PB_REQUIRE(p->kv_heads == 0 || (p->k && p->k_out), "%s: NULL k or k_out", who);
        PB_REQUIRE(aligned(p->q, es) && aligned(p->q_out, es) && aligned(p->k, es) && aligned(p->k_out, es) && aligned(p->q_weight, 4) && aligned(p->k_weight, 4), "%s: a buffer is not aligned to its elements", who);
    }
    RopeArgs& a = pl.a;
    memset(&a, 0, sizeof(a));
    a.set[0] = {p->q, p->q_out, p->q_weight, p->q_stride, p->q_head_stride, p->q_out_stride, p->q_out_head_stride};
    a.set[1] = {p->k, p->k_out, p->k_weight, p->k_stride, p->k_head_stride, p->k_out_stride, p->k_out_head_stride};
    a.first[0] = p->q_heads;
    a.first[1] = a.first[2] = p->q_heads + p->kv_heads;
    a.tokens = p->tokens; a.head_dim = p->head_dim; a.rot_dim = p->rot_dim; a.interleaved = p->interleaved != 0; a.max_position = p->max_position;
    a.eps = p->eps; a.cos_sin = p->cos_sin; a.positions = p->positions;
    return plan_rope(who, p->dtype, pl);
}

int append_plan(const pb_kv_append_params* p, RopePlan& pl) {
    const char* who = "pb_kv_append";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    const int rc = check_heads(who, p->dtype, p->tokens, p->q_heads, p->kv_heads, p->head_dim, p->rot_dim, p->max_position, p->cos_sin, p->positions);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(p->kv_heads > 0, "%s: no key heads", who);
    PB_REQUIRE(p->page_size >= 1 && p->n_pages >= 0 && p->n_pages <= INT64_MAX / p->page_size, "%s: %lld pages of %d rows", who, (long long)p->n_pages, p->page_size);
    PB_REQUIRE(rows_apart(p->n_pages, p->page_stride, p->head_dim) && heads_apart(p->page_size, p->kv_heads, p->head_dim, p->token_stride, p->head_stride), "%s: rows of the cache overlap", who);
    PB_REQUIRE(heads_apart(p->tokens, p->q_heads, p->head_dim, p->q_out_stride, p->q_out_head_stride), "%s: rows of q_out overlap", who);
    const size_t es = dtype_bytes(p->dtype);
    if (p->tokens > 0) {
        PB_REQUIRE(p->k && p->v && p->k_cache && p->v_cache && p->slots && aligned(p->slots, 8), "%s: NULL k, v, cache or slots", who);
        PB_REQUIRE(p->q_heads == 0 || (p->q && p->q_out), "%s: NULL q or q_out", who);
        PB_REQUIRE(aligned(p->q, es) && aligned(p->q_out, es) && aligned(p->k, es) && aligned(p->v, es) && aligned(p->k_cache, es) && aligned(p->v_cache, es) && aligned(p->q_weight, 4) && aligned(p->k_weight, 4), "%s: a buffer is not aligned to its elements", who);
    }
    RopeArgs& a = pl.a;
    memset(&a, 0, sizeof(a));
    a.set[0] = {p->q, p->q_out, p->q_weight, p->q_stride, p->q_head_stride, p->q_out_stride, p->q_out_head_stride};
    a.set[1] = {p->k, p->k_cache, p->k_weight, p->k_stride, p->k_head_stride, 0, p->head_stride};
    a.set[2] = {p->v, p->v_cache, nullptr, p->v_stride, p->v_head_stride, 0, p->head_stride};
    a.first[0] = p->q_heads;
    a.first[1] = p->q_heads + p->kv_heads;
    a.first[2] = p->q_heads + 2 * p->kv_heads;
    a.tokens = p->tokens; a.head_dim = p->head_dim; a.rot_dim = p->rot_dim; a.interleaved = p->interleaved != 0; a.max_position = p->max_position;
    a.eps = p->eps; a.cos_sin = p->cos_sin; a.positions = p->positions;
    a.slots = p->slots; a.n_slots = p->n_pages * p->page_size; a.page_size = p->page_size; a.page_stride = p->page_stride; a.row_stride = p->token_stride;
    return plan_rope(who, p->dtype, pl);
}

int rope_info(const RopePlan& pl, int dtype, pb_launch_info* out) {
    memset(out, 0, sizeof(*out));
    const RopeArgs& a = pl.a;
    const uint64_t t = (uint64_t)a.tokens, es = dtype_bytes(dtype);
    out->num_blocks = pl.blocks;
    out->threads_per_block = 256;
    out->smem_per_block = (uint32_t)pl.smem;
    out->regs_per_thread = lm_regs(pl.fn);
    out->flops = t * ((uint64_t)a.first[1] * 3 * a.rot_dim + 4ull * a.head_dim * ((a.set[0].weight ? a.first[0] : 0) + (a.set[1].weight ? a.first[1] - a.first[0] : 0)));
    out->bytes = t * (2 * es * a.head_dim * a.first[2] + (a.rot_dim ? 4ull * a.rot_dim + 4 : 0) + (a.slots ? 8 : 0));
    return PB_OK;
}

int launch_rope(const char* who, const RopePlan& pl, void* stream, uint32_t job_id, void* notifier) {
    if (pl.smem > 48 * 1024) PB_CUDA(cudaFuncSetAttribute(pl.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * (8192 + 1024)));
    return lm_launch(who, pl.fn, dim3(pl.blocks), dim3(256), (size_t)pl.smem, (cudaStream_t)stream, 1, pl.a, job_id, (FinishedBlockNotifier*)notifier);
}

}  // namespace

uint32_t* lm_rope_error_flag_ptr() {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_rope_flag) != cudaSuccess) { cudaGetLastError(); return nullptr; }
    return (uint32_t*)p;
}

}  // namespace pb

extern "C" {

int pb_qk_rope_info(const pb_qk_rope_params* p, pb_launch_info* out) {
    pb::RopePlan pl;
    const int rc = pb::rope_plan(p, pl);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_qk_rope_info: NULL out");
    return pb::rope_info(pl, p->dtype, out);
}

int pb_qk_rope_launch(const pb_qk_rope_params* p, void* stream, uint32_t job_id, void* notifier) {
    pb::RopePlan pl;
    const int rc = pb::rope_plan(p, pl);
    if (rc != PB_OK) return rc;
    return pb::launch_rope("pb_qk_rope", pl, stream, job_id, notifier);
}

int pb_kv_append_info(const pb_kv_append_params* p, pb_launch_info* out) {
    pb::RopePlan pl;
    const int rc = pb::append_plan(p, pl);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_kv_append_info: NULL out");
    return pb::rope_info(pl, p->dtype, out);
}

int pb_kv_append_launch(const pb_kv_append_params* p, void* stream, uint32_t job_id, void* notifier) {
    pb::RopePlan pl;
    const int rc = pb::append_plan(p, pl);
    if (rc != PB_OK) return rc;
    return pb::launch_rope("pb_kv_append", pl, stream, job_id, notifier);
}

}  // extern "C"
