// What stands between a block of a layer and the next one: the norm behind the block, its gate and scale, the residual, and the norm in
// front of the next block.
//
//   a = x * w' / sqrt(mean(x^2) + eps);   h = residual + scale * gate * a;   y = h * w / sqrt(mean(h^2) + eps)
//
// Bound by memory: a row is read once and written once (some 4 operations a byte), so a row stays in registers from its first load to its
// last store, in fp32.  (16384 rows of 4096: in bf16 with both norms and a gate 101 us, 5.3 TB/s; with a gate for each token and one norm 101 us, 6.6 TB/s; with residuals in fp32 125 us, 6.4 TB/s.  777 rows of 5001 in
// fp16, value by value, 25 us.  One row 2.4 us.)
#include <algorithm>
#include <cmath>

#include "lm.cuh"
#include "umma.cuh"

namespace pb {
namespace {

__device__ uint32_t g_norm_flag;

// Two rows of a block are on their way, the next one asked for when a row's results have been stored: more at a time, or sooner, come slower, where memory is what counts.  (16384 rows of 4096, all in fp32 / in
// bf16 with a gate for each token / with residuals in fp32: 171, 101, 125 us; as soon as a row has been read 162, 109, 134; six rows, as soon as that 192, 119, 125.)
constexpr int kMaxChannels = 32768, kMaxStages = 2;
constexpr uint64_t kRingBytes = 208 * 1024;      // of an SM's shared memory

struct NormArgs {
    const void *x, *gate, *residual;
    void *h, *y;
    const float *post_weight, *weight;
    int64_t x_stride, gate_stride, residual_stride, h_stride, y_stride;
    int tokens, channels, group;         // group: threads of a row, a multiple of 32
    float scale, eps, inv_channels;
    int stages;                          // of the ring
};

// 16-byte aligned bytes into shared memory, counted by a barrier.
__device__ __forceinline__ void bulk_load(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

// N values of T as they lie in memory, in accesses of up to 16 bytes, aligned to them.
template <typename T, int N>
struct Raw {
    static constexpr int A = N * sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
    LmVec<T, A> v[N / A];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < N / A; ++i) v[i] = reinterpret_cast<const LmVec<T, A>*>(p)[i];
    }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i / A].v[i % A] = lm_from_f<T>(x);
    }
    __device__ __forceinline__ float operator[](int i) const { return lm_to_f<T>(v[i / A].v[i % A]); }
};
template <typename T, int N>
__device__ __forceinline__ void store_floats(T* p, const float (&x)[N]) {
    Raw<T, N> r;
    if constexpr (sizeof(T) == 2 && N >= 2) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
        for (int i = 0; i < N; i += 2) w[i / 2] = lm_pack2<T>(x[i], x[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i / Raw<T, N>::A].v[i % Raw<T, N>::A] = lm_from_f<T>(x[i]);
    }
#pragma unroll
    for (int i = 0; i < N / Raw<T, N>::A; ++i) reinterpret_cast<LmVec<T, Raw<T, N>::A>*>(p)[i] = r.v[i];
}

// What a thread has of a row: CH pieces of V values, piece i of thread t at (i * group + t) * V.
template <typename T, typename H, int V, int CH>
struct RowPart {
    Raw<T, V> x[CH], gate[CH];
    Raw<H, V> residual[CH];
    float v[CH][V];
    // everything at once; `there`: pieces in front of the row's end
    __device__ __forceinline__ void load(const NormArgs& a, const T* px, const T* pg, const H* pr, int t, bool live) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int at = (i * a.group + t) * V;
            const bool there = live && at < a.channels;
            x[i].fill(0.f);
            gate[i].fill(1.f);
            residual[i].fill(0.f);
            if (there) x[i].load(px + at);
            if (there && pg) gate[i].load(pg + at);
            if (there && pr) residual[i].load(pr + at);
        }
    }
    __device__ __forceinline__ float squares_of_x() {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] = x[i][j];
                sum = fmaf(v[i][j], v[i][j], sum);
            }
        return sum;
    }
    // v = residual + scale * gate * (factor * post_weight) * x, stored; its squares.  `kept`: weights that the thread holds already, or NULL.
    __device__ __forceinline__ float into_residual(const NormArgs& a, float factor, int64_t row, int t, bool live, const Raw<float, V>* kept) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int at = (i * a.group + t) * V;
            const bool there = live && at < a.channels;
            if (a.post_weight && there) {
                Raw<float, V> w;
                if (kept) w = kept[i];
                else w.load(a.post_weight + at);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] *= factor * w[j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] = fmaf(a.scale, a.gate ? v[i][j] * gate[i][j] : v[i][j], residual[i][j]);
                sum = fmaf(v[i][j], v[i][j], sum);
            }
            if (a.h && there) store_floats<H, V>(static_cast<H*>(a.h) + row * a.h_stride + at, v[i]);
        }
        return sum;
    }
    __device__ __forceinline__ void normed(const NormArgs& a, float factor, int64_t row, int t, bool live, const Raw<float, V>* kept) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int at = (i * a.group + t) * V;
            if (!live || at >= a.channels) continue;
            Raw<float, V> w;
            w.fill(1.f);
            if (kept) w = kept[i];
            else if (a.weight) w.load(a.weight + at);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] *= factor * w[j];
            store_floats<T, V>(static_cast<T*>(a.y) + row * a.y_stride + at, v[i]);
        }
    }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// The sum over a group of threads (whole warps), the same in all of them.  All groups of a block come here together; calls that follow one another take turns at two arrays.
__device__ __forceinline__ float group_sum(float v, int group, float* s_part) {
    v = warp_sum(v);
    if (group == 32) return v;
    const int warps = group >> 5, first = threadIdx.x / group * warps;
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
    __syncthreads();
    float sum = 0.f;
    for (int i = 0; i < warps; ++i) sum += s_part[first + i];
    return sum;
}

// A row for `group` threads.
template <typename T, typename H, int V, int CH>
__global__ void __launch_bounds__(V > 1 && CH <= 2 ? 256 : V == 1 && CH <= 16 ? 640 : 1024, V > 1 && CH <= 2 ? 6 / CH : V == 1 && CH <= 8 ? 2 : 1) norm_kernel(const __grid_constant__ NormArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    __shared__ float s_part[2][32];
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int t = threadIdx.x % a.group;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / a.group) + threadIdx.x / a.group;
    const bool live = row < a.tokens;
    RowPart<T, H, V, CH> p;
    p.load(a, static_cast<const T*>(a.x) + row * a.x_stride, a.gate ? static_cast<const T*>(a.gate) + row * a.gate_stride : nullptr,
           a.residual ? static_cast<const H*>(a.residual) + row * a.residual_stride : nullptr, t, live);
    float sum = p.squares_of_x(), factor = 1.f;
    if (a.post_weight) factor = rsqrtf(group_sum(sum, a.group, s_part[0]) * a.inv_channels + a.eps);
    sum = p.into_residual(a, factor, row, t, live, nullptr);
    if (a.y) p.normed(a, rsqrtf(group_sum(sum, a.group, s_part[1]) * a.inv_channels + a.eps), row, t, live, nullptr);
    if (nf) nf->end(job_id);
}

// The same for many rows, which come through a ring of bulk copies in shared memory: a block takes every gridDim.x-th.  With two pieces a thread, the weights and a gate of all tokens stay in its registers,
// since the ring leaves no room for them in the first-level cache.  (16384 rows of 4096 in bf16 with both norms and such a gate: 101 us, read again for each row 133; with a piece a thread and twice the
// threads 149, with four pieces 152.)
template <typename T, typename H, int CH>
__global__ void __launch_bounds__(512, 1) norm_ring_kernel(const __grid_constant__ NormArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    constexpr bool kKeep = CH == 2;
    constexpr int V = 16 / (int)sizeof(T);
    extern __shared__ __align__(128) uint8_t s_rows[];
    __shared__ __align__(16) float s_part[2][2][16];                     // (of warps that the block does not have: zeros)
    __shared__ uint64_t s_full[kMaxStages];
    __shared__ volatile uint32_t s_abort;
    if (threadIdx.x < 64) reinterpret_cast<float*>(s_part)[threadIdx.x] = 0.f;
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int i = 0; i < a.stages; ++i) mbar_init(smem_u32(&s_full[i]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int t = threadIdx.x;
    const uint32_t x_bytes = (uint32_t)a.channels * sizeof(T), r_bytes = a.residual ? (uint32_t)a.channels * sizeof(H) : 0, g_bytes = a.gate && a.gate_stride ? x_bytes : 0, stage_bytes = x_bytes + r_bytes + g_bytes;
    const auto fetch = [&](int64_t row, int stage) {                     // one thread
        const uint32_t to = smem_u32(s_rows) + stage * stage_bytes, bar = smem_u32(&s_full[stage]);
        mbar_arrive_expect_tx(bar, stage_bytes);
        bulk_load(to, static_cast<const T*>(a.x) + row * a.x_stride, x_bytes, bar);
        if (r_bytes) bulk_load(to + x_bytes, static_cast<const H*>(a.residual) + row * a.residual_stride, r_bytes, bar);
        if (g_bytes) bulk_load(to + x_bytes + r_bytes, static_cast<const T*>(a.gate) + row * a.gate_stride, g_bytes, bar);
    };
    if (t == 0)
        for (int i = 0; i < a.stages; ++i)
            if ((int64_t)blockIdx.x + (int64_t)i * gridDim.x < a.tokens) fetch((int64_t)blockIdx.x + (int64_t)i * gridDim.x, i);
    const auto all_parts = [&](const float* part) {
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = reinterpret_cast<const float4*>(part)[i];
#pragma unroll
        for (int i = 1; i < 4; ++i) { x[0].x += x[i].x; x[0].y += x[i].y; x[0].z += x[i].z; x[0].w += x[i].w; }
        return (x[0].x + x[0].y) + (x[0].z + x[0].w);
    };
    Raw<float, V> post[CH], weight[CH];
    Raw<T, V> gate[CH];
    if (kKeep) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int at = (i * a.group + t) * V;
            post[i].fill(1.f);
            weight[i].fill(1.f);
            gate[i].fill(1.f);
            if (at < a.channels && a.post_weight) post[i].load(a.post_weight + at);
            if (at < a.channels && a.weight) weight[i].load(a.weight + at);
            if (at < a.channels && a.gate && !g_bytes) gate[i].load(static_cast<const T*>(a.gate) + at);
        }
    }
    int stage = 0, turn = 0;
    uint32_t parity = 0;
    for (int64_t row = blockIdx.x; row < a.tokens; row += gridDim.x) {
        const bool ok = mbar_wait(smem_u32(&s_full[stage]), parity, &s_abort, &g_norm_flag, kFlagLmWait);
        const T* x = reinterpret_cast<const T*>(s_rows + (size_t)stage * stage_bytes);
        RowPart<T, H, V, CH> p;
        p.load(a, x, !a.gate || (kKeep && !g_bytes) ? nullptr : g_bytes ? reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(x) + x_bytes + r_bytes) : static_cast<const T*>(a.gate),
               r_bytes ? reinterpret_cast<const H*>(reinterpret_cast<const uint8_t*>(x) + x_bytes) : nullptr, t, true);
        if (kKeep && a.gate && !g_bytes) {
#pragma unroll
            for (int i = 0; i < CH; ++i) p.gate[i] = gate[i];
        }
        float sum = warp_sum(p.squares_of_x());
        if ((t & 31) == 0) s_part[turn][0][t >> 5] = sum;
        if (!__syncthreads_and(ok)) break;                               // all have read the stage
        const float factor = a.post_weight ? rsqrtf(all_parts(s_part[turn][0]) * a.inv_channels + a.eps) : 1.f;
        sum = p.into_residual(a, factor, row, t, true, kKeep ? post : nullptr);
        if (a.y) {
            sum = warp_sum(sum);
            if ((t & 31) == 0) s_part[turn][1][t >> 5] = sum;
            __syncthreads();
            p.normed(a, rsqrtf(all_parts(s_part[turn][1]) * a.inv_channels + a.eps), row, t, true, kKeep ? weight : nullptr);
        }
        if (t == 0 && row + (int64_t)a.stages * gridDim.x < a.tokens) fetch(row + (int64_t)a.stages * gridDim.x, stage);
        turn ^= 1;
        if (++stage == a.stages) { stage = 0; parity ^= 1; }
    }
    if (s_abort) {             // copies in flight end before their shared memory does
        const unsigned long long t0 = globaltimer_ns();
        for (int i = 0; i < 100000 && globaltimer_ns() - t0 < 50000; ++i) __nanosleep(500);
    }
    if (nf) nf->end(job_id);
}

typedef void (*NormFn)(NormArgs, uint32_t, FinishedBlockNotifier*);

struct NormPlan {
    NormArgs a;
    NormFn fn;
    unsigned blocks, threads, smem;
};

// wide: 16-byte accesses of T, up to 4 pieces a thread (8 of fp32); otherwise single values, up to 32.  ring: rows through shared memory, 2 or 4 pieces.
template <typename T, typename H>
NormFn pick(bool wide, bool ring, int pieces) {
    constexpr int VN = 16 / (int)sizeof(T);
    if (ring) return pieces == 2 ? norm_ring_kernel<T, H, 2> : norm_ring_kernel<T, H, 4>;
    if constexpr (sizeof(T) == 4)
        if (wide && pieces == 8) return norm_kernel<T, H, VN, 8>;
    if (wide) return pieces == 1 ? norm_kernel<T, H, VN, 1> : pieces == 2 ? norm_kernel<T, H, VN, 2> : norm_kernel<T, H, VN, 4>;
    return pieces == 4 ? norm_kernel<T, H, 1, 4> : pieces == 8 ? norm_kernel<T, H, 1, 8> : pieces == 16 ? norm_kernel<T, H, 1, 16> : norm_kernel<T, H, 1, 32>;
}

int plan_norm(const pb_residual_norm_params* p, NormPlan& pl) {
    const char* who = "pb_residual_norm";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(p->tokens >= 0, "%s: %d tokens", who, p->tokens);
    PB_REQUIRE(p->channels >= 1 && p->channels <= kMaxChannels, "%s: %d channels (1 to %d)", who, p->channels, kMaxChannels);
    PB_REQUIRE(is_float_dtype(p->dtype) && (p->h_dtype == p->dtype || p->h_dtype == PB_F32), "%s: dtype %d, h_dtype %d (the same, or PB_F32)", who, p->dtype, p->h_dtype);
    PB_REQUIRE(std::isfinite(p->scale) && p->eps >= 0.f && std::isfinite(p->eps), "%s: scale or eps is not finite, or eps is negative", who);
    const size_t es = dtype_bytes(p->dtype), hs = dtype_bytes(p->h_dtype);
    if (p->tokens > 0) {
        PB_REQUIRE(p->x && (p->h || p->y), "%s: NULL x, or neither h nor y", who);
        PB_REQUIRE(aligned(p->x, es) && aligned(p->gate, es) && aligned(p->y, es) && aligned(p->residual, hs) && aligned(p->h, hs) && aligned(p->post_weight, 4) && aligned(p->weight, 4),
                   "%s: a buffer is not aligned to its elements", who);
        PB_REQUIRE((!p->h || rows_apart(p->tokens, p->h_stride, p->channels)) && (!p->y || rows_apart(p->tokens, p->y_stride, p->channels)), "%s: rows of h or y overlap", who);
    }
    NormArgs& a = pl.a;
    a = {p->x, p->gate, p->residual, p->h, p->y, p->post_weight, p->weight, p->x_stride, p->gate_stride, p->residual_stride, p->h_stride, p->y_stride, p->tokens, p->channels, 32, p->scale, p->eps,
         1.f / (float)p->channels, 0};
    const int VN = (int)(16 / es);
    const auto fits = [&](const void* b, int64_t stride) { return !b || (aligned(b, 16) && stride % VN == 0); };
    const bool wide = p->channels % VN == 0 && fits(p->x, p->x_stride) && fits(p->gate, p->gate_stride) && fits(p->residual, p->residual_stride) && fits(p->h, p->h_stride) && fits(p->y, p->y_stride) &&
                      aligned(p->post_weight, 16) && aligned(p->weight, 16);
    const int vectors = wide ? p->channels / VN : p->channels;
    int pieces = wide ? 1 : 4;
    while (vectors > (wide ? (pieces <= 2 ? 256 : 1024) : pieces <= 16 ? 640 : 1024) * pieces) pieces *= 2;
    a.group = round_up(ceil_div(vectors, pieces), 32);
    const int rows = a.group >= 256 ? 1 : 256 / a.group;
    pl.threads = (unsigned)(a.group * rows);
    int64_t blocks = ceil_div<int64_t>(p->tokens, rows);
    pl.smem = 0;
    // Many rows come through rings, 512 threads an SM as far as there is room for two rows of each block.  (Rows of 1024 in bf16, and from registers alone: 65536 of them 90 and 102 us, 16384 25.3 and 27.3, 8192
    // 12.7 and 13.5, 4096 7.9 and 7.5, 2400 5.3 both.  Rows of 4096: 16384 of them 92 and 124, 2048 12.5 and 12.8, 700 6.1 both.)
    bool ring = false;
    const uint64_t row_bytes = (uint64_t)p->channels * (es + (p->residual ? hs : 0) + (p->gate && p->gate_stride ? es : 0));
    if (wide && vectors >= 64 && vectors <= 2048) {
        const int each = vectors <= 1024 ? 2 : 4;
        const unsigned threads = (unsigned)round_up(ceil_div(vectors, each), 32);
        const int resident = (int)std::min<uint64_t>(std::max(1u, 512 / threads), kRingBytes / (2 * row_bytes));
        if (resident >= 1 && p->tokens >= 2 * 148 * resident) {
            ring = true;
            pieces = each;
            a.group = (int)threads;
            pl.threads = threads;
            a.stages = (int)std::min<uint64_t>(kMaxStages, kRingBytes / resident / row_bytes);
            pl.smem = (unsigned)(a.stages * row_bytes);
            blocks = 148 * resident;
        }
    }
    pl.blocks = blocks > 0 ? (unsigned)blocks : 1u;
    const bool same = p->h_dtype == p->dtype;
    if (p->dtype == PB_F32) pl.fn = pick<float, float>(wide, ring, pieces);
    else if (p->dtype == PB_BF16) pl.fn = same ? pick<__nv_bfloat16, __nv_bfloat16>(wide, ring, pieces) : pick<__nv_bfloat16, float>(wide, ring, pieces);
    else pl.fn = same ? pick<__half, __half>(wide, ring, pieces) : pick<__half, float>(wide, ring, pieces);
    return PB_OK;
}

}  // namespace

uint32_t* lm_norm_error_flag_ptr() {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_norm_flag) != cudaSuccess) { cudaGetLastError(); return nullptr; }
    return (uint32_t*)p;
}

}  // namespace pb

using namespace pb;

extern "C" {

int pb_residual_norm_info(const pb_residual_norm_params* p, pb_launch_info* out) {
    NormPlan pl;
    const int rc = plan_norm(p, pl);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_residual_norm_info: NULL out");
    memset(out, 0, sizeof(*out));
    const uint64_t t = (uint64_t)p->tokens, c = (uint64_t)p->channels, es = dtype_bytes(p->dtype), hs = dtype_bytes(p->h_dtype);
    out->num_blocks = pl.blocks;
    out->threads_per_block = pl.threads;
    cudaFuncAttributes fa = {};
    if (cudaFuncGetAttributes(&fa, (const void*)pl.fn) != cudaSuccess) cudaGetLastError();        // (without a GPU: what the host knows)
    out->smem_per_block = pl.smem + (uint32_t)fa.sharedSizeBytes;
    out->regs_per_thread = (uint32_t)fa.numRegs;
    out->flops = t * c * (2 + (p->post_weight ? 4 : 0) + (p->gate ? 1 : 0) + (p->y ? 4 : 0));
    if (t)
        out->bytes = t * c * (es * (1 + (p->y ? 1 : 0)) + hs * ((p->residual ? 1 : 0) + (p->h ? 1 : 0))) + (p->gate ? (p->gate_stride ? t : 1) * c * es : 0) +
                     4 * c * ((p->post_weight ? 1 : 0) + (p->y && p->weight ? 1 : 0));
    return PB_OK;
}

int pb_residual_norm_launch(const pb_residual_norm_params* p, void* stream, uint32_t job_id, void* notifier) {
    NormPlan pl;
    const int rc = plan_norm(p, pl);
    if (rc != PB_OK) return rc;
    if (pl.smem) PB_CUDA(cudaFuncSetAttribute(pl.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingBytes));
    return lm_launch("pb_residual_norm", pl.fn, dim3(pl.blocks), dim3(pl.threads), pl.smem, (cudaStream_t)stream, 1, pl.a, job_id, (FinishedBlockNotifier*)notifier);
}

}  // extern "C"
