// Dense layers in 8-bit integers: activations brought to 8 bits token by token, and their product with weights that have a scale
// for each output channel.
//
//   q[t][k] = rint(x[t][k] * (127 * (1 / max_t))), s[t] = max_t / 127;   y[t][n] = act(s[t] * ws[n] * sum_k q[t][k] w[n][k] + b[n])
#include <cuda.h>

#include <cmath>

#include "lm.cuh"

namespace pb {
namespace {

// ---- activations to 8 bits ---------------------------------------------------------------
// A block takes a row: the largest magnitude first, then the row again (from the caches) for the integers.
template <typename T>
__global__ void __launch_bounds__(256) int8_quantize_kernel(const T* x, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, int tokens, int channels,
                                                            uint32_t job_id, FinishedBlockNotifier* nf) {
    __shared__ float red[8];
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int64_t t = blockIdx.x;
    if (t < tokens) {
        const T* row = x + t * x_stride;
        float most = 0.f;
        bool odd = false;                              // a NaN or an infinity
        for (int k = threadIdx.x; k < channels; k += 256) {
            const float v = fabsf(lm_to_f<T>(row[k]));
            odd |= !(v <= 3.402823466e38f);
            most = fmaxf(most, v);
        }
        if (odd) most = INFINITY;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
        __syncthreads();
        most = red[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) most = fmaxf(most, red[i]);
        const bool zero = !(most >= 0x1p-119f) || most == INFINITY;
        const float inv = zero ? 0.f : 127.f * __fdiv_rn(1.f, most);
        if (threadIdx.x == 0) scale[t] = most == INFINITY ? NAN : zero ? 0.f : __fdiv_rn(most, 127.f);
        for (int k = threadIdx.x; k < channels; k += 256) q[t * q_stride + k] = zero ? (int8_t)0 : (int8_t)__float2int_rn(lm_to_f<T>(row[k]) * inv);
    }
    if (nf) nf->end(job_id);
}

// ---- the product ---------------------------------------------------------------------------
struct DenseArgs {
    const int8_t *x, *w;
    const float *x_scale, *w_scale, *bias;
    void* y;
    int64_t x_stride, w_stride, y_stride;
    int T, K, N, act;
};

__device__ __forceinline__ float int8_result(const DenseArgs& a, int acc, float xs, float ws, float b) {
    float v = fmaf((float)acc, xs * ws, b);
    if (a.act >= 1) v = v < 0.f ? 0.f : v;             // (a NaN stays one)
    if (a.act == 2) v = v > 6.f ? 6.f : v;
    return v;
}

// 64 x 64 results of a block, four by four a thread; four products an instruction.
template <typename Y>
__global__ void __launch_bounds__(256) int8_dense_kernel(DenseArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    __shared__ int sx[16][65], sw[16][65];             // 64 bytes of each row, word by word
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, row = threadIdx.x >> 2, part = threadIdx.x & 3;
    const int tiles = (a.N + 63) / 64, t0 = (int)(blockIdx.x / tiles) * 64, n0 = (int)(blockIdx.x % tiles) * 64;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += 64) {
        const int k = k0 + 16 * part;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int r = (which ? n0 : t0) + row;
            const int8_t* src = which ? a.w + r * a.w_stride : a.x + r * a.x_stride;
            int v[4] = {0, 0, 0, 0};
            if (r < (which ? a.N : a.T) && k < a.K) {
                if (k + 16 <= a.K) {
                    *reinterpret_cast<int4*>(v) = *reinterpret_cast<const int4*>(src + k);
                } else {
                    for (int j = 0; j < a.K - k; ++j) v[j / 4] |= (int)(uint8_t)src[k + j] << (8 * (j % 4));
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) (which ? sw : sx)[4 * part + j][row] = v[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int l = 0; l < 4; ++l) acc[i][l] = __dp4a(sx[j][ty * 4 + i], sw[j][tx * 4 + l], acc[i][l]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int l = 0; l < 4; ++l) {
            const int t = t0 + ty * 4 + i, n = n0 + tx * 4 + l;
            if (t >= a.T || n >= a.N) continue;
            static_cast<Y*>(a.y)[t * a.y_stride + n] = lm_from_f<Y>(int8_result(a, acc[i][l], a.x_scale[t], a.w_scale[n], a.bias ? a.bias[n] : 0.f));
        }
    if (nf) nf->end(job_id);
}

int check_quantize(const pb_int8_quantize_params* p) {
    const char* who = "pb_int8_quantize";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(is_float_dtype(p->x_dtype), "%s: x_dtype %d (PB_F32, PB_BF16 or PB_F16)", who, p->x_dtype);
    PB_REQUIRE(p->tokens >= 0 && p->channels >= 1, "%s: %d tokens of %d channels", who, p->tokens, p->channels);
    PB_REQUIRE(p->tokens == 0 || (p->x && p->q && p->scale), "%s: NULL buffer", who);
    PB_REQUIRE(aligned(p->x, dtype_bytes(p->x_dtype)) && aligned(p->scale, 4), "%s: a buffer is not aligned to its elements", who);
    return PB_OK;
}

int check_dense(const pb_int8_dense_params* p) {
    const char* who = "pb_int8_dense";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(is_float_dtype(p->y_dtype), "%s: y_dtype %d (PB_F32, PB_BF16 or PB_F16)", who, p->y_dtype);
    PB_REQUIRE(p->tokens >= 0 && p->in_channels >= 1 && p->out_channels >= 1, "%s: %d tokens, %d -> %d channels", who, p->tokens, p->in_channels, p->out_channels);
    PB_REQUIRE(p->in_channels <= 131071, "%s: %d input channels could pass 32 bits (at most 131071)", who, p->in_channels);
    PB_REQUIRE(p->act >= 0 && p->act <= 2, "%s: activation %d (0 none, 1 relu, 2 relu6)", who, p->act);
    PB_REQUIRE(p->x_stride % 16 == 0 && p->w_stride % 16 == 0, "%s: rows of x and w start on 16 bytes (strides %lld, %lld)", who, (long long)p->x_stride, (long long)p->w_stride);
    PB_REQUIRE((p->x_stride >= p->in_channels || p->tokens <= 1) && (p->w_stride >= p->in_channels || p->out_channels == 1), "%s: rows overlap (strides %lld, %lld)", who, (long long)p->x_stride, (long long)p->w_stride);
    if (p->tokens > 0) {
        PB_REQUIRE(p->x && p->x_scale && p->w && p->w_scale && p->y, "%s: NULL buffer", who);
        PB_REQUIRE(aligned(p->x, 16) && aligned(p->w, 16), "%s: x and w must be 16-byte aligned", who);
        PB_REQUIRE(aligned(p->x_scale, 4) && aligned(p->w_scale, 4) && aligned(p->bias, 4) && aligned(p->y, dtype_bytes(p->y_dtype)), "%s: a buffer is not aligned to its elements", who);
    }
    return PB_OK;
}

}  // namespace
}  // namespace pb

using namespace pb;

extern "C" {

int pb_int8_quantize_info(const pb_int8_quantize_params* p, pb_launch_info* out) {
    const int rc = check_quantize(p);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_int8_quantize_info: NULL out");
    memset(out, 0, sizeof(*out));
    out->num_blocks = p->tokens > 0 ? (uint32_t)p->tokens : 1u;
    out->threads_per_block = 256;
    out->smem_per_block = 32;
    out->regs_per_thread = p->x_dtype == PB_F32 ? lm_regs(int8_quantize_kernel<float>) : p->x_dtype == PB_BF16 ? lm_regs(int8_quantize_kernel<__nv_bfloat16>) : lm_regs(int8_quantize_kernel<__half>);
    out->bytes = (uint64_t)p->tokens * ((dtype_bytes(p->x_dtype) + 1) * p->channels + 4);
    return PB_OK;
}

int pb_int8_quantize_launch(const pb_int8_quantize_params* p, void* stream, uint32_t job_id, void* notifier) {
    const int rc = check_quantize(p);
    if (rc != PB_OK) return rc;
    const dim3 grid(p->tokens > 0 ? (unsigned)p->tokens : 1u);
    FinishedBlockNotifier* nf = (FinishedBlockNotifier*)notifier;
    const char* who = "pb_int8_quantize";
#define PB_QUANTIZE(T) lm_launch(who, int8_quantize_kernel<T>, grid, dim3(256), 0, (cudaStream_t)stream, 1, (const T*)p->x, p->x_stride, p->q, p->q_stride, p->scale, p->tokens, p->channels, job_id, nf)
    if (p->x_dtype == PB_F32) return PB_QUANTIZE(float);
    if (p->x_dtype == PB_BF16) return PB_QUANTIZE(__nv_bfloat16);
    return PB_QUANTIZE(__half);
#undef PB_QUANTIZE
}

int pb_int8_dense_info(const pb_int8_dense_params* p, pb_launch_info* out) {
    const int rc = check_dense(p);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_int8_dense_info: NULL out");
    memset(out, 0, sizeof(*out));
    const uint64_t t = (uint64_t)p->tokens, k = (uint64_t)p->in_channels, n = (uint64_t)p->out_channels;
    const uint64_t blocks = ceil_div<uint64_t>(t, 64) * ceil_div<uint64_t>(n, 64);
    PB_REQUIRE(blocks <= 0x7fffffff, "pb_int8_dense: too many results for one launch");
    out->num_blocks = blocks > 0 ? (uint32_t)blocks : 1u;
    out->threads_per_block = 256;
    out->smem_per_block = 2 * 16 * 65 * 4;
    out->regs_per_thread = p->y_dtype == PB_F32 ? lm_regs(int8_dense_kernel<float>) : p->y_dtype == PB_BF16 ? lm_regs(int8_dense_kernel<__nv_bfloat16>) : lm_regs(int8_dense_kernel<__half>);
    out->flops = 2 * t * k * n;
    out->bytes = t * k + n * k + 4 * t + (p->bias ? 8 : 4) * n + t * n * dtype_bytes(p->y_dtype);
    return PB_OK;
}

int pb_int8_dense_launch(const pb_int8_dense_params* p, void* stream, uint32_t job_id, void* notifier) {
    pb_launch_info li;
    const int rc = pb_int8_dense_info(p, &li);
    if (rc != PB_OK) return rc;
    const DenseArgs a = {p->x, p->w, p->x_scale, p->w_scale, p->bias, p->y, p->x_stride, p->w_stride, p->y_stride, p->tokens, p->in_channels, p->out_channels, p->act};
    FinishedBlockNotifier* nf = (FinishedBlockNotifier*)notifier;
    const char* who = "pb_int8_dense";
    const dim3 grid(li.num_blocks);
    if (p->y_dtype == PB_F32) return lm_launch(who, int8_dense_kernel<float>, grid, dim3(256), 0, (cudaStream_t)stream, 1, a, job_id, nf);
    if (p->y_dtype == PB_BF16) return lm_launch(who, int8_dense_kernel<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, 1, a, job_id, nf);
    return lm_launch(who, int8_dense_kernel<__half>, grid, dim3(256), 0, (cudaStream_t)stream, 1, a, job_id, nf);
}

}  // extern "C"
