// Paged key/value cache: the append of new keys and values, and the attention
// of one new token of every sequence over its pages.
//
// A cache is [d, kv_heads, page_size, pages] in any order of strides; row b of
// the block table names the pages of sequence b in order.  Page numbers and
// positions live in device memory, so their guards run in the kernels: a page
// number or a position outside the cache is never used as an address, and the
// context's rejected word (reported by emel_cuda_stream_synchronize) is set.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.hpp"
#include "pdl.cuh"

namespace emel {

namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
    else return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

constexpr int kAppendThreads = 256;

// ---- append ------------------------------------------------------------------
template <typename S, typename C>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(PagedAppendPlan p) {
    pdl_enter();
    const uint64_t per = p.d * p.kv_heads;
    const uint64_t total = p.count * per;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t n = i / per, h = i % per / p.d, c = i % p.d;
        const int64_t pos = p.positions[(int64_t)n * p.pos_st];
        if (pos < 0) continue;
        const int64_t seq = p.sequences ? p.sequences[(int64_t)n * p.seq_st] : (int64_t)n;
        const uint64_t page_at = (uint64_t)pos / p.page_size, off = (uint64_t)pos % p.page_size;
        int64_t page = -1;
        if (seq >= 0 && (uint64_t)seq < p.sequences_count && page_at < p.table_pages)
            page = p.table[(int64_t)page_at * p.table_st[0] + seq * p.table_st[1]];
        if (page < 0 || (uint64_t)page >= p.pages) {
            atomicExch(p.reject, p.reject_code);
            continue;
        }
        const char* ks = p.key + c * sizeof(S) + h * p.key_st[1] + n * p.key_st[2];
        const char* vs = p.value + c * sizeof(S) + h * p.value_st[1] + n * p.value_st[2];
        char* kd = p.k_cache + c * 2 + h * p.k_st[1] + off * p.k_st[2] + page * p.k_st[3];
        char* vd = p.v_cache + c * 2 + h * p.v_st[1] + off * p.v_st[2] + page * p.v_st[3];
        if constexpr (std::is_same_v<S, C>) {
            *reinterpret_cast<C*>(kd) = *reinterpret_cast<const S*>(ks);
            *reinterpret_cast<C*>(vd) = *reinterpret_cast<const S*>(vs);
        } else {
            *reinterpret_cast<C*>(kd) = from_f32<C>(to_f32(*reinterpret_cast<const S*>(ks)));
            *reinterpret_cast<C*>(vd) = from_f32<C>(to_f32(*reinterpret_cast<const S*>(vs)));
        }
    }
}

// ---- attention ---------------------------------------------------------------
//
// One CTA per (query head, sequence): warp w takes tokens w, w + 4, ..., a
// lane d / 32 columns, with the running maximum and sum of a softmax:
//     M = max(m, s), l = l e^(m - M) + e^(s - M), o = o e^(m - M) + e^(s - M) v.
// The four warps' (m, l, o) join in shared memory.
constexpr int kAttnWarps = 4;
constexpr int kAttnCols = kPagedMaxD / 32;

template <typename Q, typename C>
__global__ void __launch_bounds__(kAttnWarps * 32) paged_attn_kernel(PagedAttnPlan p) {
    __shared__ float part_o[kAttnWarps][kPagedMaxD];
    __shared__ float part_m[kAttnWarps], part_l[kAttnWarps];
    pdl_enter();
    const uint64_t h = blockIdx.x % p.heads, b = blockIdx.x / p.heads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t kvh = h / p.rep;
    const char* qrow = p.q + h * p.q_st[1] + b * p.q_st[2];
    int64_t len = p.lengths[(int64_t)b * p.len_st];
    const int64_t cap = (int64_t)(p.table_pages * p.page_size);
    if (len < 0 || len > cap) {
        if (threadIdx.x == 0) atomicExch(p.reject, p.reject_code);
        len = len < 0 ? 0 : cap;
    }
    const int64_t first = p.window && (uint64_t)len > p.window ? len - (int64_t)p.window : 0;
    float q[kAttnCols], o[kAttnCols];
#pragma unroll
    for (int i = 0; i < kAttnCols; ++i) {
        const uint64_t c = lane + 32 * i;
        q[i] = c < p.d ? to_f32(reinterpret_cast<const Q*>(qrow)[c]) * p.scale : 0.0f;
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int64_t t = first + warp; t < len; t += kAttnWarps) {
        const int64_t page = p.table[(int64_t)((uint64_t)t / p.page_size) * p.table_st[0] + (int64_t)b * p.table_st[1]];
        if (page < 0 || (uint64_t)page >= p.pages) {
            if (lane == 0) atomicExch(p.reject, p.reject_code);
            continue;
        }
        const uint64_t off = (uint64_t)t % p.page_size;
        const C* k = reinterpret_cast<const C*>(p.k + kvh * p.k_st[1] + off * p.k_st[2] + page * p.k_st[3]);
        const C* v = reinterpret_cast<const C*>(p.v + kvh * p.v_st[1] + off * p.v_st[2] + page * p.v_st[3]);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kAttnCols; ++i) {
            const uint64_t c = lane + 32 * i;
            if (c < p.d) s = __fmaf_rn(q[i], to_f32(k[c]), s);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float top = fmaxf(m, s);
        const float ref = top == -INFINITY ? 0.0f : top;  // only -inf so far: every weight is 0
        const float keep = expf(m - ref), w = expf(s - ref);
        l = __fmaf_rn(l, keep, w);
#pragma unroll
        for (int i = 0; i < kAttnCols; ++i) {
            const uint64_t c = lane + 32 * i;
            if (c < p.d) o[i] = __fmaf_rn(w, to_f32(v[c]), o[i] * keep);
        }
        m = top;
    }
    if (lane == 0) {
        part_m[warp] = m;
        part_l[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < kAttnCols; ++i) part_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    char* drow = p.dst + h * p.dst_st[1] + b * p.dst_st[2];
    float top = -INFINITY, sum = 0.0f, w[kAttnWarps];
#pragma unroll
    for (int k = 0; k < kAttnWarps; ++k) top = fmaxf(top, part_m[k]);
#pragma unroll
    for (int k = 0; k < kAttnWarps; ++k) {
        w[k] = expf(part_m[k] - (top == -INFINITY ? 0.0f : top));
        sum = __fmaf_rn(w[k], part_l[k], sum);
    }
    for (uint64_t c = threadIdx.x; c < p.d; c += blockDim.x) {
        float x = 0.0f;
#pragma unroll
        for (int k = 0; k < kAttnWarps; ++k) x = __fmaf_rn(w[k], part_o[k][c], x);
        reinterpret_cast<Q*>(drow)[c] = from_f32<Q>(sum == 0.0f ? 0.0f : x / sum);
    }
}

template <typename S, typename C>
cudaError_t run_append(const LaunchEnv& env, const PagedAppendPlan& p) {
    const uint64_t total = p.count * p.d * p.kv_heads;
    const uint64_t want = (total + kAppendThreads - 1) / kAppendThreads;
    const uint64_t cap = (uint64_t)env.sm_count * 8;
    const cudaError_t err = launch_dependent(append_kernel<S, C>, dim3((unsigned)(want < cap ? want : cap)),
                                             dim3(kAppendThreads), 0, env.stream, p);
    if (err == cudaSuccess) ++*env.launches;
    return err;
}

template <typename Q, typename C>
cudaError_t run_attn(const LaunchEnv& env, const PagedAttnPlan& p) {
    const cudaError_t err = launch_dependent(paged_attn_kernel<Q, C>, dim3((unsigned)(p.heads * p.batch)),
                                             dim3(kAttnWarps * 32), 0, env.stream, p);
    if (err == cudaSuccess) ++*env.launches;
    return err;
}

}  // namespace

cudaError_t launch_paged_append(const LaunchEnv& env, const PagedAppendPlan& p) {
    if (p.cache_bf16) {
        return p.src_f32 ? run_append<float, __nv_bfloat16>(env, p) : run_append<__nv_bfloat16, __nv_bfloat16>(env, p);
    }
    return p.src_f32 ? run_append<float, __half>(env, p) : run_append<__half, __half>(env, p);
}

cudaError_t launch_paged_attn(const LaunchEnv& env, const PagedAttnPlan& p) {
    if (p.cache_bf16) {
        return p.q_f32 ? run_attn<float, __nv_bfloat16>(env, p) : run_attn<__nv_bfloat16, __nv_bfloat16>(env, p);
    }
    return p.q_f32 ? run_attn<float, __half>(env, p) : run_attn<__half, __half>(env, p);
}

}  // namespace emel
