// What stands between a block of a layer and the next one: the norm behind the block, its gate and scale, the residual, and the norm in
// front of the next block.
//
//   a = x * w' / sqrt(mean(x^2) + eps);   h = residual + scale * gate * a;   y = h * w / sqrt(mean(h^2) + eps)
//
// Bound by memory: a row is read once and written once (some 4 operations a byte), so a row stays in registers from its first load to its
// last store, in fp32.
#include <cmath>

#include "lm.cuh"

namespace pb {
namespace {

constexpr int kMaxChannels = 32768;

struct NormArgs {
    const void *x, *gate, *residual;
    void *h, *y;
    const float *post_weight, *weight;
    int64_t x_stride, gate_stride, residual_stride, h_stride, y_stride;
    int tokens, channels, group;         // group: threads of a row, a multiple of 32
    float scale, eps, inv_channels;
};

// N values of T at p as floats, in accesses of up to 16 bytes, aligned to them.
template <typename T, int N>
__device__ __forceinline__ void load_floats(const T* p, float (&v)[N]) {
    constexpr int A = N * sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += A) {
        const LmVec<T, A> x = *reinterpret_cast<const LmVec<T, A>*>(p + i);
#pragma unroll
        for (int j = 0; j < A; ++j) v[i + j] = lm_to_f<T>(x.v[j]);
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_floats(T* p, const float (&v)[N]) {
    constexpr int A = N * sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += A) {
        LmVec<T, A> x;
#pragma unroll
        for (int j = 0; j < A; ++j) x.v[j] = lm_from_f<T>(v[i + j]);
        *reinterpret_cast<LmVec<T, A>*>(p + i) = x;
    }
}

// The sum over a group of threads (whole warps), the same in all of them.  All groups of a block come here together.
__device__ __forceinline__ float group_sum(float v, int group, float* s_part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (group == 32) return v;
    const int warps = group >> 5, first = threadIdx.x / group * warps;
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
    __syncthreads();
    float sum = 0.f;
    for (int i = 0; i < warps; ++i) sum += s_part[first + i];
    __syncthreads();
    return sum;
}

// A row for `group` threads, each with CH pieces of V values: piece i of thread t lies at (i * group + t) * V.
template <typename T, typename H, int V, int CH>
__global__ void __launch_bounds__(1024) norm_kernel(const __grid_constant__ NormArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    __shared__ float s_part[32];
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int t = threadIdx.x % a.group;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / a.group) + threadIdx.x / a.group;
    const bool live = row < a.tokens;
    float v[CH][V];
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int at = (i * a.group + t) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = 0.f;
        if (live && at < a.channels) load_floats<T, V>(x + at, v[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) sum = fmaf(v[i][j], v[i][j], sum);
    }
    float factor = 1.f;
    if (a.post_weight) factor = rsqrtf(group_sum(sum, a.group, s_part) * a.inv_channels + a.eps);
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int at = (i * a.group + t) * V;
        if (!live || at >= a.channels) continue;
        float w[V];
        if (a.post_weight) {
            load_floats<float, V>(a.post_weight + at, w);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] *= factor * w[j];
        }
        if (a.gate) {
            load_floats<T, V>(static_cast<const T*>(a.gate) + row * a.gate_stride + at, w);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] *= w[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = 0.f;
        if (a.residual) load_floats<H, V>(static_cast<const H*>(a.residual) + row * a.residual_stride + at, w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v[i][j] = fmaf(a.scale, v[i][j], w[j]);
            sum = fmaf(v[i][j], v[i][j], sum);
        }
        if (a.h) store_floats<H, V>(static_cast<H*>(a.h) + row * a.h_stride + at, v[i]);
    }
    if (a.y) {
        factor = rsqrtf(group_sum(sum, a.group, s_part) * a.inv_channels + a.eps);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int at = (i * a.group + t) * V;
            if (!live || at >= a.channels) continue;
            float w[V];
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = 1.f;
            if (a.weight) load_floats<float, V>(a.weight + at, w);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] *= factor * w[j];
            store_floats<T, V>(static_cast<T*>(a.y) + row * a.y_stride + at, v[i]);
        }
    }
    if (nf) nf->end(job_id);
}

typedef void (*NormFn)(NormArgs, uint32_t, FinishedBlockNotifier*);

struct NormPlan {
    NormArgs a;
    NormFn fn;
    unsigned blocks, threads;
};

// wide: 16-byte accesses of T, 1 or 4 pieces a thread; otherwise single values, up to 32.
template <typename T, typename H>
NormFn pick(bool wide, int pieces) {
    constexpr int VN = 16 / (int)sizeof(T);
    if (wide) return pieces == 1 ? norm_kernel<T, H, VN, 1> : pieces == 2 ? norm_kernel<T, H, VN, 2> : pieces == 4 ? norm_kernel<T, H, VN, 4> : norm_kernel<T, H, VN, 8>;
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
         1.f / (float)p->channels};
    const int VN = (int)(16 / es);
    const auto fits = [&](const void* b, int64_t stride) { return !b || (aligned(b, 16) && stride % VN == 0); };
    const bool wide = p->channels % VN == 0 && fits(p->x, p->x_stride) && fits(p->gate, p->gate_stride) && fits(p->residual, p->residual_stride) && fits(p->h, p->h_stride) && fits(p->y, p->y_stride) &&
                      aligned(p->post_weight, 16) && aligned(p->weight, 16);
    const int vectors = wide ? p->channels / VN : p->channels;
    int pieces = wide ? 1 : 4;
    while (vectors > 1024 * pieces) pieces *= 2;
    a.group = round_up(ceil_div(vectors, pieces), 32);
    const int rows = a.group >= 256 ? 1 : 256 / a.group;
    pl.threads = (unsigned)(a.group * rows);
    const int64_t blocks = ceil_div<int64_t>(p->tokens, rows);
    pl.blocks = blocks > 0 ? (unsigned)blocks : 1u;
    const bool same = p->h_dtype == p->dtype;
    if (p->dtype == PB_F32) pl.fn = pick<float, float>(wide, pieces);
    else if (p->dtype == PB_BF16) pl.fn = same ? pick<__nv_bfloat16, __nv_bfloat16>(wide, pieces) : pick<__nv_bfloat16, float>(wide, pieces);
    else pl.fn = same ? pick<__half, __half>(wide, pieces) : pick<__half, float>(wide, pieces);
    return PB_OK;
}

}  // namespace
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
    out->regs_per_thread = lm_regs(pl.fn);
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
    return lm_launch("pb_residual_norm", pl.fn, dim3(pl.blocks), dim3(pl.threads), 0, (cudaStream_t)stream, 1, pl.a, job_id, (FinishedBlockNotifier*)notifier);
}

}  // extern "C"
