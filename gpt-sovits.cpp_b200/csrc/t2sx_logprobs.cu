// Log probabilities of given tokens, with the rows' entropy, the tokens' ranks and the best tokens.
//
//   m = max x,  s = sum e^(x - m),  w = sum e^(x - m) (x - m)     (over x > -inf)
//   logprob = x_t - m - log s,   entropy = log s - w / s
//   rank = #{x > x_t} + #{j < t: x_j = x_t}
#include "../../include/t2sx.h"
#include "t2sx_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>

using namespace t2sx;

int t2sx_set_error(int code, const char* msg);

namespace {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

constexpr int kThreads = 256;

// Value and id of a candidate as one key: greater keys come first (values descending, ids
// ascending).  -inf and NaN have no place in a list.
__device__ __forceinline__ unsigned long long order_key(float x, unsigned id) {
    unsigned b = __float_as_uint(x + 0.0f);   // one zero
    b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (unsigned long long)b << 32 | (0xFFFFFFFFu - id);
}

__device__ __forceinline__ float block_sum(float v, float* sh) {
    for (int x = 16; x; x >>= 1) v += __shfl_xor_sync(~0u, v, x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int i = 0; i < kThreads / 32; ++i) v += sh[i];
    return v;
}

// One CTA per row, the row read once for each statistic and each place of the list.
template <typename T>
__global__ void __launch_bounds__(kThreads)
k_logprobs(const T* __restrict__ logits, long long stride, int vocab, const int32_t* __restrict__ tokens, int top_k,
           float* __restrict__ logprob, float* __restrict__ entropy, int32_t* __restrict__ rank, int32_t* __restrict__ top_ids,
           float* __restrict__ top_logprobs) {
    __shared__ float sh[kThreads / 32];
    __shared__ unsigned long long shk[kThreads / 32];
    const long long row = blockIdx.x;
    const T* x = logits + row * stride;
    const int tid = threadIdx.x, t = tokens[row];
    const bool given = t >= 0 && t < vocab;
    const float xt = given ? to_f32(x[t]) : 0.0f;
    float m = -INFINITY, bad = 0.0f;
    for (int j = tid; j < vocab; j += kThreads) {
        const float v = to_f32(x[j]);
        if (!(v < INFINITY)) bad = 1.0f;
        m = fmaxf(m, v);
    }
    for (int y = 16; y; y >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, y));
    if ((tid & 31) == 0) sh[tid >> 5] = m;
    __syncthreads();
    for (int i = 0; i < kThreads / 32; ++i) m = fmaxf(m, sh[i]);
    bad = block_sum(bad, sh);
    float s = 0.0f, w = 0.0f, before = 0.0f;
    for (int j = tid; j < vocab; j += kThreads) {
        const float v = to_f32(x[j]);
        if (v > xt || (v == xt && j < t)) before += 1.0f;
        if (v == -INFINITY) continue;
        const float d = v - m, e = expf(d);
        s += e;
        w = fmaf(e, d, w);
    }
    s = block_sum(s, sh);
    w = block_sum(w, sh);
    before = block_sum(before, sh);
    const float log_s = s > 0.0f ? logf(s) : 0.0f;
    if (tid == 0) {
        logprob[row] = t == -1 ? 0.0f : !given || bad > 0.0f ? NAN : s > 0.0f ? xt - m - log_s : -INFINITY;
        if (entropy) entropy[row] = bad > 0.0f ? NAN : s > 0.0f ? log_s - w / s : 0.0f;
        if (rank) rank[row] = given ? (int)before : -1;
    }
    unsigned long long last = ~0ull;
    for (int i = 0; i < top_k; ++i) {
        unsigned long long best = 0;
        for (int j = tid; j < vocab; j += kThreads) {
            const float v = to_f32(x[j]);
            if (!(v > -INFINITY)) continue;
            const unsigned long long key = order_key(v, j);
            if (key < last && key > best) best = key;
        }
        for (int y = 16; y; y >>= 1) {
            const unsigned long long o = __shfl_xor_sync(~0u, best, y);
            best = o > best ? o : best;
        }
        __syncthreads();
        if ((tid & 31) == 0) shk[tid >> 5] = best;
        __syncthreads();
        for (int k = 0; k < kThreads / 32; ++k) best = shk[k] > best ? shk[k] : best;
        last = best;
        if (tid == 0) {
            const unsigned id = 0xFFFFFFFFu - (unsigned)best;
            top_ids[row * top_k + i] = best ? (int)id : -1;
            top_logprobs[row * top_k + i] = bad > 0.0f ? NAN : best ? to_f32(x[id]) - m - log_s : -INFINITY;
        }
    }
}

int bad(const char* m) { return t2sx_set_error(T2SX_ERR_INVALID, m); }

}  // namespace

extern "C" int t2sx_token_logprobs(int32_t device, int32_t type, int64_t rows, int64_t vocab, const void* logits_dev,
                                   int64_t stride, const int32_t* tokens_dev, int32_t top_k, float* logprob_dev,
                                   float* entropy_dev, int32_t* rank_dev, int32_t* top_ids_dev, float* top_logprobs_dev,
                                   void* stream) {
    if (type != T2SX_TYPE_F32 && type != T2SX_TYPE_F16 && type != T2SX_TYPE_BF16)
        return bad("t2sx_token_logprobs: the type must be f32, f16 or bf16");
    if (rows < 0 || rows > INT32_MAX || vocab <= 0 || vocab > (1 << 30) || stride < vocab || stride > (int64_t)1 << 40)
        return bad("t2sx_token_logprobs: rows, vocab or stride out of range");
    if (top_k < 0 || top_k > 32) return bad("t2sx_token_logprobs: top_k must be 0 to 32");
    if (rows == 0) return T2SX_OK;
    if (!logits_dev || !tokens_dev || !logprob_dev || (top_k > 0 && (!top_ids_dev || !top_logprobs_dev)))
        return bad("t2sx_token_logprobs: null logits, tokens or output");
    if (((uintptr_t)logits_dev % (type == T2SX_TYPE_F32 ? 4 : 2)) ||
        (((uintptr_t)tokens_dev | (uintptr_t)logprob_dev | (uintptr_t)entropy_dev | (uintptr_t)rank_dev | (uintptr_t)top_ids_dev |
          (uintptr_t)top_logprobs_dev) & 3))
        return bad("t2sx_token_logprobs: misaligned pointer");
    DeviceGuard dg;
    cudaError_t e = dg.set(device);
    if (e != cudaSuccess) return t2sx_set_error(T2SX_ERR_CUDA, cudaGetErrorString(e));
    cudaStream_t st = (cudaStream_t)stream;
    auto go = [&](auto kernel, auto* x) {
        kernel<<<(unsigned)rows, kThreads, 0, st>>>(x, (long long)stride, (int)vocab, tokens_dev, top_k, logprob_dev, entropy_dev,
                                                   rank_dev, top_ids_dev, top_logprobs_dev);
    };
    if (type == T2SX_TYPE_F32) go(k_logprobs<float>, (const float*)logits_dev);
    else if (type == T2SX_TYPE_F16) go(k_logprobs<__half>, (const __half*)logits_dev);
    else go(k_logprobs<__nv_bfloat16>, (const __nv_bfloat16*)logits_dev);
    e = cudaGetLastError();
    if (e != cudaSuccess) return t2sx_set_error(T2SX_ERR_CUDA, cudaGetErrorString(e));
    return T2SX_OK;
}
