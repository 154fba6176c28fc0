// Logits of a decoding step before a token is chosen: penalties for tokens
// that the row's history holds, biases, and the mask of allowed tokens.
//
// Per logit v of token i, with c = how often i stands in the used history:
//     c > 0:  v = v > 0 ? v / r : v r,  then  v = v - c f - p
//     v = v + bias[i];   v = -inf where the mask's bit i is 0.
// Reading and writing every logit once is what bounds it.  A CTA owns
// kLogitsChunk consecutive tokens of one row, from a 16-byte boundary on, and asks
// for all that it needs before it waits for any of it: logits and biases in 16-byte
// vectors that stay in registers, mask words, the first ids of the history.  It
// counts the ids that fall into its tokens in shared memory (integer atomics: the
// counts do not depend on their order); a row is read once from HBM, its
// history once per chunk from L2.  64 rows of 151936 logits with biases and masks
// for each row: 18.9 us without a history (18.0 at the copy rate), 25.9 us with up to
// 4096 ids a row.  Chunks of 8192 took 33 us, chunks of 2048 42 us (more waves of
// history), and anything that spills registers a third more.
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.hpp"
#include "pdl.cuh"

namespace emel {

namespace {

constexpr int kLogitsThreads = 256;
constexpr int kLogitsChunk = 4096;
constexpr int kIds = 8;  // ids of a thread that are in flight from the start

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads, 4) logits_adjust_kernel(LogitsPlan p, uint32_t chunks) {
    constexpr int kVec = 16 / sizeof(T), kOwn = kLogitsChunk / kVec / kLogitsThreads;  // vectors of a thread
    __shared__ uint32_t counts[kLogitsChunk];
    pdl_enter();
    const uint32_t row = blockIdx.x / chunks;
    const T* src = reinterpret_cast<const T*>(p.src + row * p.src_st);
    T* dst = reinterpret_cast<T*>(p.dst + row * p.dst_st);
    // logits before the row's first 16-byte boundary in src belong to a vector that starts before the row
    const int32_t lead = (int32_t)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T)), vocab = (int32_t)p.vocab;
    const int32_t base = (int32_t)((blockIdx.x - row * chunks) * kLogitsChunk) - lead;
    if (base >= vocab) return;
    const int32_t own = base + (int32_t)threadIdx.x * kVec;  // and every kVec * kLogitsThreads logits on
    auto place = [&](int j) { return own + j * kVec * kLogitsThreads; };
    auto whole = [&](int32_t at) { return at >= 0 && at <= vocab - kVec; };
    // everything is asked for before anything is waited for: the history up to its
    // capacity, whatever part of it is in use
    const int32_t* ids = p.history ? p.history + (int64_t)row * p.hist_st[1] : nullptr;
    int32_t id[kIds];
#pragma unroll
    for (int u = 0; u < kIds; ++u) {
        const uint32_t i = threadIdx.x + u * kLogitsThreads;
        id[u] = ids && i < p.history_len ? ids[i * p.hist_st[0]] : INT32_MIN;
    }
    float r = 1.0f, f = 0.0f, pr = 0.0f;
    int32_t used = 0;
    if (p.history) {
        used = p.lengths[(int64_t)row * p.len_st];
        const float* q = p.penalties + (p.penalty_rows ? (int64_t)row * p.pen_st[1] : 0);
        r = q[0];
        f = q[p.pen_st[0]];
        pr = q[2 * p.pen_st[0]];
    }
    uint4 raw[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        raw[j] = make_uint4(0, 0, 0, 0);
        if (whole(place(j))) raw[j] = __ldcs(reinterpret_cast<const uint4*>(src + place(j)));
    }
    const float* bias = p.bias ? p.bias + (p.bias_rows ? (int64_t)row * p.bias_st : 0) : nullptr;
    const bool bias_vec = ((reinterpret_cast<uintptr_t>(bias) / 4 + (uint32_t)own) & 3u) == 0;
    float4 b[kOwn][kVec / 4];
    if (bias) {
#pragma unroll
        for (int j = 0; j < kOwn; ++j)
#pragma unroll
            for (int q = 0; q < kVec / 4; ++q) {
                const float* from = bias + place(j) + 4 * q;
                b[j][q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (!whole(place(j))) continue;
                if (bias_vec) b[j][q] = __ldg(reinterpret_cast<const float4*>(from));
                else b[j][q] = make_float4(__ldg(from), __ldg(from + 1), __ldg(from + 2), __ldg(from + 3));
            }
    }
    const uint32_t* allowed = p.allowed ? p.allowed + (p.allowed_rows ? (int64_t)row * p.allowed_st : 0) : nullptr;
    uint32_t lo[kOwn], hi[kOwn];  // the words of a vector's mask bits: one, or two where it crosses
    if (allowed) {
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
            lo[j] = hi[j] = 0;
            if (whole(place(j))) {
                lo[j] = __ldg(allowed + (place(j) >> 5));
                hi[j] = __ldg(allowed + ((place(j) + kVec - 1) >> 5));
            }
        }
    }
    used = used < 0 ? 0 : (uint64_t)used > p.history_len ? (int32_t)p.history_len : used;
    if (used > 0) {
        uint4* clear = reinterpret_cast<uint4*>(counts);
#pragma unroll
        for (int i = 0; i < kLogitsChunk / 4 / kLogitsThreads; ++i) clear[threadIdx.x + i * kLogitsThreads] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        auto count = [&](int32_t i, int32_t token) {
            // a chunk that starts before its row has no room for what lies there
            const uint32_t at = (uint32_t)token - (uint32_t)base;
            if (i < used && at < kLogitsChunk && token >= 0) atomicAdd(&counts[at], 1u);
        };
#pragma unroll
        for (int u = 0; u < kIds; ++u) count(threadIdx.x + u * kLogitsThreads, id[u]);
        for (int32_t i = threadIdx.x + kIds * kLogitsThreads; i < used; i += kLogitsThreads) count(i, ids[(int64_t)i * p.hist_st[0]]);
        __syncthreads();
    }
    auto penalized = [&](float v, uint32_t c) {
        if (c) {
            v = v > 0.0f ? v / r : v * r;
            v = v - (float)c * f;
            v = v - pr;
        }
        return v;
    };
    const bool alike = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & 15u) == 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int32_t at = place(j);
        const uint32_t* c = counts + (at - base);
        if (!whole(at)) {
            for (int e = 0; e < kVec; ++e) {
                const int32_t i = at + e;
                if (i < 0 || i >= vocab) continue;
                float v = (float)src[i];
                if (used > 0) v = penalized(v, c[e]);
                if (bias) v = v + bias[i];
                if (allowed && !((allowed[i >> 5] >> (i & 31)) & 1u)) v = -INFINITY;
                dst[i] = (T)v;
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
        if (used > 0) {
#pragma unroll
            for (int q = 0; q < kVec / 4; ++q) {
                const uint4 x = *reinterpret_cast<const uint4*>(c + 4 * q);
                if ((x.x | x.y | x.z | x.w) == 0) continue;  // nearly always
                v[4 * q] = penalized(v[4 * q], x.x);
                v[4 * q + 1] = penalized(v[4 * q + 1], x.y);
                v[4 * q + 2] = penalized(v[4 * q + 2], x.z);
                v[4 * q + 3] = penalized(v[4 * q + 3], x.w);
            }
        }
        if (bias) {
#pragma unroll
            for (int q = 0; q < kVec / 4; ++q) {
                v[4 * q] = v[4 * q] + b[j][q].x;
                v[4 * q + 1] = v[4 * q + 1] + b[j][q].y;
                v[4 * q + 2] = v[4 * q + 2] + b[j][q].z;
                v[4 * q + 3] = v[4 * q + 3] + b[j][q].w;
            }
        }
        if (allowed) {
            const uint32_t ok = __funnelshift_r(lo[j], hi[j], (uint32_t)at & 31u);
#pragma unroll
            for (int e = 0; e < kVec; ++e) v[e] = (ok >> e) & 1u ? v[e] : -INFINITY;
        }
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
