// Logits of a decoding step before a token is chosen: penalties for tokens
// that the row's history holds, biases, and the mask of allowed tokens.
//
// Per logit v of token i, with c = how often i stands in the used history:
//     c > 0:  v = v > 0 ? v / r : v r,  then  v = v - c f - p
//     v = v + bias[i];   v = -inf where the mask's bit i is 0.
// A CTA owns kLogitsChunk consecutive tokens of one row.  It counts the
// history's ids that fall into them in shared memory (integer atomics: the
// counts do not depend on their order) and streams the chunk once.
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.hpp"
#include "pdl.cuh"

namespace emel {

namespace {

constexpr int kLogitsThreads = 256;
constexpr int kLogitsChunk = 8192;

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) logits_adjust_kernel(LogitsPlan p) {
    __shared__ uint32_t counts[kLogitsChunk];
    pdl_enter();
    const uint32_t chunks = (uint32_t)((p.vocab + kLogitsChunk - 1) / kLogitsChunk);
    const uint64_t row = blockIdx.x / chunks, base = (uint64_t)(blockIdx.x % chunks) * kLogitsChunk;
    const uint32_t here = (uint32_t)(p.vocab - base < kLogitsChunk ? p.vocab - base : kLogitsChunk);
    float r = 1.0f, f = 0.0f, pr = 0.0f;
    int64_t used = 0;
    if (p.history) {
        used = p.lengths[(int64_t)row * p.len_st];
        if (used < 0) used = 0;
        if ((uint64_t)used > p.history_len) used = (int64_t)p.history_len;
        const float* q = p.penalties + (p.penalty_rows ? (int64_t)row * p.pen_st[1] : 0);
        r = q[0];
        f = q[p.pen_st[0]];
        pr = q[2 * p.pen_st[0]];
    }
    if (used > 0) {
        for (uint32_t i = threadIdx.x; i < here; i += blockDim.x) counts[i] = 0;
        __syncthreads();
        const int32_t* ids = p.history + (int64_t)row * p.hist_st[1];
        for (int64_t i = threadIdx.x; i < used; i += blockDim.x) {
            const int64_t at = (int64_t)ids[i * p.hist_st[0]] - (int64_t)base;
            if (at >= 0 && at < (int64_t)here) atomicAdd(&counts[at], 1u);
        }
        __syncthreads();
    }
    const T* src = reinterpret_cast<const T*>(p.src + row * p.src_st) + base;
    T* dst = reinterpret_cast<T*>(p.dst + row * p.dst_st) + base;
    const float* bias = p.bias ? p.bias + (p.bias_rows ? (int64_t)row * p.bias_st : 0) + base : nullptr;
    const uint32_t* allowed = p.allowed ? p.allowed + (p.allowed_rows ? (int64_t)row * p.allowed_st : 0) + base / 32 : nullptr;
    for (uint32_t i = threadIdx.x; i < here; i += blockDim.x) {
        float v = (float)src[i];
        if (used > 0) {
            const uint32_t c = counts[i];
            if (c) {
                v = v > 0.0f ? v / r : v * r;
                v = v - (float)c * f;
                v = v - pr;
            }
        }
        if (bias) v = v + bias[i];
        if (allowed && !((allowed[i >> 5] >> (i & 31u)) & 1u)) v = -INFINITY;
        dst[i] = (T)v;
    }
}

template <typename T>
cudaError_t run_logits(const LaunchEnv& env, const LogitsPlan& p) {
    const uint64_t chunks = (p.vocab + kLogitsChunk - 1) / kLogitsChunk;
    const cudaError_t err = launch_dependent(logits_adjust_kernel<T>, dim3((unsigned)(chunks * p.rows)),
                                             dim3(kLogitsThreads), 0, env.stream, p);
    if (err == cudaSuccess) ++*env.launches;
    return err;
}

}  // namespace

uint64_t logits_blocks(uint64_t vocab, uint64_t rows) {
    const unsigned __int128 n = (unsigned __int128)((vocab + kLogitsChunk - 1) / kLogitsChunk) * rows;
    return n > UINT64_MAX ? UINT64_MAX : (uint64_t)n;
}

cudaError_t launch_logits_adjust(const LaunchEnv& env, const LogitsPlan& p) {
    return p.f16 ? run_logits<__half>(env, p) : run_logits<float>(env, p);
}

}  // namespace emel
