// Logits of a decoding step before a token is chosen: penalties for tokens
// that the row's history holds, biases, and the mask of allowed tokens.
//
// Per logit v of token i, with c = how often i stands in the used history:
//     c > 0:  v = v > 0 ? v / r : v r,  then  v = v - c f - p
//     v = v + bias[i];   v = -inf where the mask's bit i is 0.
// Reading and writing every logit once is what bounds it.  A CTA owns
// kLogitsChunk consecutive tokens of one row, from a 16-byte boundary on.  It asks
// for its logits first, in 16-byte vectors that stay in registers; while they
// come it counts the history's ids that fall into its tokens in shared memory
// (integer atomics: the counts do not depend on their order).  A row is read
// once from HBM, its history once per chunk from L2.
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.hpp"
#include "pdl.cuh"

namespace emel {

namespace {

constexpr int kLogitsThreads = 256;
constexpr int kLogitsChunk = 8192;

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) logits_adjust_kernel(LogitsPlan p, uint32_t chunks) {
    constexpr int kVec = 16 / sizeof(T), kOwn = kLogitsChunk / kVec / kLogitsThreads;  // vectors of a thread
    __shared__ uint32_t counts[kLogitsChunk];
    pdl_enter();
    const uint64_t row = blockIdx.x / chunks;
    const T* src = reinterpret_cast<const T*>(p.src + row * p.src_st);
    T* dst = reinterpret_cast<T*>(p.dst + row * p.dst_st);
    // logits before the row's first 16-byte boundary in src belong to a vector that starts before the row
    const int64_t lead = (int64_t)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
    const int64_t base = (int64_t)(blockIdx.x % chunks) * kLogitsChunk - lead, vocab = (int64_t)p.vocab;
    if (base >= vocab) return;
    const bool alike = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & 15u) == 0;
    auto whole = [&](int64_t at) { return at >= 0 && at + kVec <= vocab; };
    uint4 raw[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int64_t at = base + (int64_t)(threadIdx.x + j * kLogitsThreads) * kVec;
        raw[j] = make_uint4(0, 0, 0, 0);
        if (whole(at)) raw[j] = __ldcs(reinterpret_cast<const uint4*>(src + at));
    }
    float r = 1.0f, f = 0.0f, pr = 0.0f;
    int64_t used = 0;
    if (p.history) {
        used = p.lengths[(int64_t)row * p.len_st];
        used = used < 0 ? 0 : (uint64_t)used > p.history_len ? (int64_t)p.history_len : used;
        const float* q = p.penalties + (p.penalty_rows ? (int64_t)row * p.pen_st[1] : 0);
        r = q[0];
        f = q[p.pen_st[0]];
        pr = q[2 * p.pen_st[0]];
    }
    if (used > 0) {
        uint4* clear = reinterpret_cast<uint4*>(counts);
#pragma unroll
        for (int i = 0; i < kLogitsChunk / 4 / kLogitsThreads; ++i) clear[threadIdx.x + i * kLogitsThreads] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int32_t* ids = p.history + (int64_t)row * p.hist_st[1];
        auto count = [&](int32_t id) {
            const int64_t at = (int64_t)id - base;
            if (at >= 0 && at < kLogitsChunk) atomicAdd(&counts[at], 1u);
        };
        constexpr int kIds = 8;  // in flight
        for (int64_t i = threadIdx.x; i < used; i += kIds * kLogitsThreads) {
            int32_t id[kIds];
#pragma unroll
            for (int u = 0; u < kIds; ++u) id[u] = i + u * kLogitsThreads < used ? ids[(i + u * kLogitsThreads) * p.hist_st[0]] : INT32_MIN;
#pragma unroll
            for (int u = 0; u < kIds; ++u) count(id[u]);
        }
        __syncthreads();
    }
    const float* bias = p.bias ? p.bias + (p.bias_rows ? (int64_t)row * p.bias_st : 0) : nullptr;
    const uint32_t* allowed = p.allowed ? p.allowed + (p.allowed_rows ? (int64_t)row * p.allowed_st : 0) : nullptr;
    auto adjusted = [&](float v, uint32_t c, float b, bool ok) {
        if (c) {
            v = v > 0.0f ? v / r : v * r;
            v = v - (float)c * f;
            v = v - pr;
        }
        if (bias) v = v + b;
        return ok ? v : -INFINITY;
    };
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const uint32_t in = (threadIdx.x + j * kLogitsThreads) * kVec;
        const int64_t at = base + in;
        if (!whole(at)) {
            for (int e = 0; e < kVec; ++e) {
                const int64_t i = at + e;
                if (i < 0 || i >= vocab) continue;
                const bool ok = !allowed || ((allowed[i >> 5] >> (i & 31)) & 1u);
                dst[i] = (T)adjusted((float)src[i], used > 0 ? counts[in + e] : 0u, bias ? bias[i] : 0.0f, ok);
            }
            continue;
        }
        float v[kVec];
        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            if constexpr (sizeof(T) == 4) v[e] = __uint_as_float(w[e]);
            else v[e] = __half2float(__ushort_as_half((uint16_t)(w[e >> 1] >> (16 * (e & 1)))));
        }
        float b[kVec] = {};
        if (bias) {
            const float* from = bias + at;
            if ((reinterpret_cast<uintptr_t>(from) & 15u) == 0) {
#pragma unroll
                for (int q = 0; q < kVec / 4; ++q) {
                    const float4 x = __ldg(reinterpret_cast<const float4*>(from) + q);
                    b[4 * q] = x.x, b[4 * q + 1] = x.y, b[4 * q + 2] = x.z, b[4 * q + 3] = x.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < kVec; ++e) b[e] = __ldg(from + e);
            }
        }
        uint32_t ok = 0xffffffffu;
        if (allowed) {  // the vector's bits, from one word or two
            const uint32_t lo = __ldg(allowed + (at >> 5)), hi = __ldg(allowed + ((at + kVec - 1) >> 5));
            ok = __funnelshift_r(lo, hi, (uint32_t)at & 31u);
        }
        uint32_t c[kVec] = {};
        if (used > 0) {
#pragma unroll
            for (int q = 0; q < kVec / 4; ++q) {
                const uint4 x = *reinterpret_cast<const uint4*>(counts + in + 4 * q);
                c[4 * q] = x.x, c[4 * q + 1] = x.y, c[4 * q + 2] = x.z, c[4 * q + 3] = x.w;
            }
        }
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[e] = adjusted(v[e], c[e], b[e], (ok >> e) & 1u);
        if (alike) {
            uint32_t o[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if constexpr (sizeof(T) == 4) o[q] = __float_as_uint(v[q]);
                else o[q] = __half_as_ushort(__float2half_rn(v[2 * q])) | (uint32_t)__half_as_ushort(__float2half_rn(v[2 * q + 1])) << 16;
            }
            __stcs(reinterpret_cast<uint4*>(dst + at), make_uint4(o[0], o[1], o[2], o[3]));
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) dst[at + e] = (T)v[e];
        }
    }
}

// Chunks of a row that starts anywhere between two 16-byte boundaries.
uint64_t logits_chunks(uint64_t vocab) { return vocab / kLogitsChunk + (vocab % kLogitsChunk + 7 + kLogitsChunk - 1) / kLogitsChunk; }

template <typename T>
cudaError_t run_logits(const LaunchEnv& env, const LogitsPlan& p) {
    const uint64_t chunks = logits_chunks(p.vocab);
    const cudaError_t err = launch_dependent(logits_adjust_kernel<T>, dim3((unsigned)(chunks * p.rows)),
                                             dim3(kLogitsThreads), 0, env.stream, p, (uint32_t)chunks);
    if (err == cudaSuccess) ++*env.launches;
    return err;
}

}  // namespace

uint64_t logits_blocks(uint64_t vocab, uint64_t rows) {
    const unsigned __int128 n = (unsigned __int128)logits_chunks(vocab) * rows;
    return n > UINT64_MAX ? UINT64_MAX : (uint64_t)n;
}

cudaError_t launch_logits_adjust(const LaunchEnv& env, const LogitsPlan& p) {
    return p.f16 ? run_logits<__half>(env, p) : run_logits<float>(env, p);
}

}  // namespace emel
