// Matrix-vector products with 4-bit weights and group scales (Q4_0, Q4_1,
// Q4_K rows), for one or a few activation rows.
//
// A group is 32 consecutive weights of a row; every format is
//     w = a (q - 8) + c,   q in 0..15,
// with a = d, c = 0 (Q4_0); a = d, c = m + 8 d (Q4_1); a = d s, c = 8 d s -
// e t with 6-bit s and t (Q4_K).  So
//     y = sum over groups of a * sum((q - 8) x) + c * sum(x),
// and the 4-bit integers meet the activations without a scale in between.
//
// Packed layout (emel_cuda_q4_pack): rows in tiles of 16, columns in blocks
// of 64.  Lane 4 g + t of a warp owns, of each 16 x 64 block, rows g and
// g + 8 and the columns 32 G + 8 t .. + 7 of both groups G: 32 quants, one
// 16-byte load.  Word j (columns 32 (j / 2) + 8 t + 4 (j % 2) + 0..3 =: k):
// nibble 2 s + (s's half) ... bits 4 r + 16 h hold, for r = 0..3 and h = 0, 1,
// row g + 8 (r & 1), column k + 2 (r >> 1) + h: what one m16n8k16 operand
// fragment holds in register r, half h.  The blocks of a tile are
// adjacent; the scales follow all quants, one record per tile and 256 columns:
//     Q4_0  lane: d of (row g, group 2t), (g, 2t+1), (g+8, 2t), (g+8, 2t+1)
//     Q4_1  lane: the same four as (d, m) pairs
//     Q4_K  lane: the same four as (s, t) byte pairs, then for each g the
//           (d, e) of rows g and g + 8
// Rows and columns beyond the matrix are quants of 8 under scales of 0.
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.hpp"
#include "pdl.cuh"

namespace emel {

namespace {

constexpr int kQ4Threads = 256;

__host__ __device__ constexpr uint64_t q4_scale_bytes(int code) {
    return code == kDtypeQ4_0 ? 256 : code == kDtypeQ4_1 ? 512 : 320;
}

// The quant of column k in a source row.
template <int CODE>
__device__ __forceinline__ uint32_t q4_quant(const uint8_t* row, uint64_t k) {
    const uint32_t i = (uint32_t)k & 31u;
    if constexpr (CODE == kDtypeQ4_K) {
        const uint32_t sub = ((uint32_t)k & 255u) >> 5;
        const uint8_t byte = row[(k >> 8) * 144 + 16 + 32 * (sub >> 1) + i];
        return (sub & 1u) ? byte >> 4 : byte & 15u;
    } else {
        constexpr int kBlock = CODE == kDtypeQ4_0 ? 18 : 20;
        const uint8_t byte = row[(k >> 5) * kBlock + (kBlock - 16) + (i & 15u)];
        return i < 16 ? byte & 15u : byte >> 4;
    }
}

__device__ __forceinline__ uint32_t load16(const uint8_t* p) { return (uint32_t)p[0] | ((uint32_t)p[1] << 8); }

// One thread per 16-byte piece of the quants, then one per lane of the scales.
template <int CODE>
__global__ void __launch_bounds__(kQ4Threads) q4_pack_kernel(Q4PackPlan p) {
    pdl_enter();
    const uint64_t tiles = (p.rows + 15) / 16, k64 = (p.k + 63) / 64, k256 = (p.k + 255) / 256;
    const uint64_t pieces = tiles * k64 * 32, records = tiles * k256 * 32;
    uint8_t* scales = p.dst + pieces * 16;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < pieces + records;
         i += (uint64_t)gridDim.x * blockDim.x) {
        const bool quants = i < pieces;
        const uint64_t at = quants ? i : i - pieces;
        const uint32_t lane = (uint32_t)at & 31u, g = lane >> 2, t = lane & 3u;
        const uint64_t block = at >> 5, per = quants ? k64 : k256, tile = block / per, kb = block % per;
        const uint64_t row[2] = {tile * 16 + g, tile * 16 + g + 8};
        if (quants) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint64_t k = kb * 64 + 32 * (j >> 1) + 8 * t + 4 * (j & 1);
                w[j] = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint64_t kk = k + 2 * (r >> 1) + h, rr = row[r & 1];
                        const uint32_t q = rr < p.rows && kk < p.k ? q4_quant<CODE>(p.src + rr * p.row_bytes, kk) : 8u;
                        w[j] |= q << (4 * r + 16 * h);
                    }
            }
            reinterpret_cast<uint4*>(p.dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
            continue;
        }
        uint8_t* rec = scales + block * q4_scale_bytes(CODE);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint64_t rr = row[s >> 1], group = kb * 8 + 2 * t + (s & 1);
            const bool in = rr < p.rows && group * 32 < p.k;
            const uint8_t* src = p.src + rr * p.row_bytes;
            if constexpr (CODE == kDtypeQ4_0) {
                reinterpret_cast<uint16_t*>(rec)[lane * 4 + s] = in ? (uint16_t)load16(src + group * 18) : 0;
            } else if constexpr (CODE == kDtypeQ4_1) {
                reinterpret_cast<uint16_t*>(rec)[lane * 8 + 2 * s] = in ? (uint16_t)load16(src + group * 20) : 0;
                reinterpret_cast<uint16_t*>(rec)[lane * 8 + 2 * s + 1] = in ? (uint16_t)load16(src + group * 20 + 2) : 0;
            } else {
                const uint8_t* c = src + kb * 144 + 4;  // 12 bytes of 6-bit scales and minimums
                const uint32_t j = 2 * t + (s & 1);
                uint32_t sc = 0, mn = 0;
                if (in) {
                    sc = j < 4 ? c[j] & 63u : (c[j + 4] & 15u) | ((uint32_t)(c[j - 4] >> 6) << 4);
                    mn = j < 4 ? c[j + 4] & 63u : (uint32_t)(c[j + 4] >> 4) | ((uint32_t)(c[j] >> 6) << 4);
                }
                rec[lane * 8 + 2 * s] = (uint8_t)sc;
                rec[lane * 8 + 2 * s + 1] = (uint8_t)mn;
                if (t == 0 && (s & 1) == 0) {
                    reinterpret_cast<uint16_t*>(rec + 256)[g * 4 + s] = in ? (uint16_t)load16(src + kb * 144) : 0;
                    reinterpret_cast<uint16_t*>(rec + 256)[g * 4 + s + 1] = in ? (uint16_t)load16(src + kb * 144 + 2) : 0;
                }
            }
        }
    }
}

// a and c of (scale slot s of lane `lane`) in one record.
template <int CODE>
__device__ __forceinline__ void q4_scale(const uint8_t* rec, uint32_t lane, uint32_t s, float& a, float& c) {
    if constexpr (CODE == kDtypeQ4_0) {
        a = __half2float(reinterpret_cast<const __half*>(rec)[lane * 4 + s]);
        c = 0.0f;
    } else if constexpr (CODE == kDtypeQ4_1) {
        a = __half2float(reinterpret_cast<const __half*>(rec)[lane * 8 + 2 * s]);
        c = __fmaf_rn(8.0f, a, __half2float(reinterpret_cast<const __half*>(rec)[lane * 8 + 2 * s + 1]));
    } else {
        const __half* de = reinterpret_cast<const __half*>(rec + 256) + (lane >> 2) * 4 + (s & 2u);
        a = __half2float(de[0]) * (float)rec[lane * 8 + 2 * s];
        c = __fmaf_rn(8.0f, a, -__half2float(de[1]) * (float)rec[lane * 8 + 2 * s + 1]);
    }
}

// One warp per output: lanes take blocks of 64 columns.
template <int CODE, typename X>
__global__ void __launch_bounds__(kQ4Threads) q4_matvec_kernel(Q4MatvecPlan p) {
    pdl_enter();
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t tiles = (p.rows + 15) / 16, k64 = (p.k + 63) / 64, k256 = (p.k + 255) / 256;
    const uint4* quants = reinterpret_cast<const uint4*>(p.weights);
    const uint8_t* scales = p.weights + tiles * k64 * 512;
    const uint64_t warps = (uint64_t)gridDim.x * (kQ4Threads / 32);
    for (uint64_t out = (uint64_t)blockIdx.x * (kQ4Threads / 32) + (threadIdx.x >> 5); out < p.rows * p.n; out += warps) {
        const uint64_t row = out % p.rows, n = out / p.rows;
        const uint64_t tile = row >> 4;
        const uint32_t g = (uint32_t)row & 7u, r = ((uint32_t)row >> 3) & 1u;
        const X* x = reinterpret_cast<const X*>(p.x + n * p.x_st);
        float sum = 0.0f;
        for (uint64_t kb = lane; kb < k64; kb += 32) {
            const uint8_t* rec = scales + (tile * k256 + (kb >> 2)) * q4_scale_bytes(CODE);
            for (uint32_t G = 0; G < 2; ++G) {
                float dot = 0.0f, total = 0.0f;
                for (uint32_t t = 0; t < 4; ++t) {
                    const uint4 q = quants[(tile * k64 + kb) * 32 + 4 * g + t];
                    for (uint32_t j = 0; j < 2; ++j) {
                        const uint32_t w = G ? (j ? q.w : q.z) : (j ? q.y : q.x);
                        for (uint32_t e = 0; e < 4; ++e) {
                            const uint64_t k = kb * 64 + 32 * G + 8 * t + 4 * j + e;
                            if (k >= p.k) continue;
                            const uint32_t nib = (w >> (4 * (r + 2 * (e >> 1)) + 16 * (e & 1))) & 15u;
                            const float xv = (float)x[k];
                            dot = __fmaf_rn((float)((int)nib - 8), xv, dot);
                            total += xv;
                        }
                    }
                }
                float a, c;
                q4_scale<CODE>(rec, 4 * g + ((uint32_t)kb & 3u), 2 * r + G, a, c);
                sum = __fmaf_rn(a, dot, sum);
                if constexpr (CODE != kDtypeQ4_0) sum = __fmaf_rn(c, total, sum);
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) {
            char* y = p.dst + n * p.dst_st;
            if (p.dst_f16) reinterpret_cast<__half*>(y)[row] = __float2half_rn(sum);
            else reinterpret_cast<float*>(y)[row] = sum;
        }
    }
}

template <int CODE>
cudaError_t run_q4_pack(const LaunchEnv& env, const Q4PackPlan& p) {
    const uint64_t tiles = (p.rows + 15) / 16;
    const uint64_t items = tiles * ((p.k + 63) / 64 + (p.k + 255) / 256) * 32;
    const uint64_t want = (items + kQ4Threads - 1) / kQ4Threads, cap = (uint64_t)env.sm_count * 8;
    const cudaError_t err = launch_dependent(q4_pack_kernel<CODE>, dim3((unsigned)(want < cap ? want : cap)),
                                             dim3(kQ4Threads), 0, env.stream, p);
    if (err == cudaSuccess) ++*env.launches;
    return err;
}

template <int CODE, typename X>
cudaError_t run_q4(const LaunchEnv& env, const Q4MatvecPlan& p) {
    const uint64_t want = (p.rows * p.n + kQ4Threads / 32 - 1) / (kQ4Threads / 32), cap = (uint64_t)env.sm_count * 8;
    const cudaError_t err = launch_dependent(q4_matvec_kernel<CODE, X>, dim3((unsigned)(want < cap ? want : cap)),
                                             dim3(kQ4Threads), 0, env.stream, p);
    if (err == cudaSuccess) ++*env.launches;
    return err;
}

template <int CODE>
cudaError_t run_q4_types(const LaunchEnv& env, const Q4MatvecPlan& p) {
    return p.x_f16 ? run_q4<CODE, __half>(env, p) : run_q4<CODE, float>(env, p);
}

}  // namespace

bool q4_packed_bytes(int code, uint64_t k, uint64_t rows, uint64_t* bytes) {
    const unsigned __int128 tiles = (rows >> 4) + ((rows & 15) != 0), k64 = (k >> 6) + ((k & 63) != 0),
                            k256 = (k >> 8) + ((k & 255) != 0);
    const unsigned __int128 total = tiles * (k64 * 512 + k256 * q4_scale_bytes(code));
    if (total > (unsigned __int128)INT64_MAX) return false;
    *bytes = (uint64_t)total;
    return true;
}

cudaError_t launch_q4_pack(const LaunchEnv& env, const Q4PackPlan& p) {
    if (p.code == kDtypeQ4_0) return run_q4_pack<kDtypeQ4_0>(env, p);
    if (p.code == kDtypeQ4_1) return run_q4_pack<kDtypeQ4_1>(env, p);
    return run_q4_pack<kDtypeQ4_K>(env, p);
}

cudaError_t launch_mul_mat_q4(const LaunchEnv& env, const Q4MatvecPlan& p) {
    if (p.code == kDtypeQ4_0) return run_q4_types<kDtypeQ4_0>(env, p);
    if (p.code == kDtypeQ4_1) return run_q4_types<kDtypeQ4_1>(env, p);
    return run_q4_types<kDtypeQ4_K>(env, p);
}

}  // namespace emel
