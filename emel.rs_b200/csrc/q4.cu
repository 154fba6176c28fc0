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
#include <cooperative_groups.h>
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

// ---- the product ---------------------------------------------------------------
//
// Reading the weights once is what bounds it (4.5 bits each); the work per
// weight has to stay under what an SM can issue while it waits for them: about
// three instructions a weight at full bandwidth.  So the quants become binary16
// integers q - 8 two at a time (a mask that leaves 1024 + q or 1024 + 16 q, one
// subtraction or multiply-add: exact), and m16n8k16 products multiply 16 rows
// with up to 8 columns of x at once, one instruction for 8 weights a lane.  The
// scales meet the products of a group, in binary32.
//
// Columns of x.  binary16: one for each token, as it is.  binary32: two for
// each token, x 2^e = hi + lo with both rounded to binary16 and e chosen per
// token (and CTA) so that the largest |x| lies in [2^14, 2^15): 22 bits and
// more, down to 2^-40 of the largest.  The tensor pipe is idle otherwise, so
// the second column costs no time.
//
// A persistent CTA of 16 warps keeps its columns of x in shared memory and
// walks tiles of 16 rows.  WK warps share a tile (each a part of its 256-column
// blocks), WR tiles are in work; a warp holds two blocks of weights in
// registers and asks for the next one piece by piece as it uses them up.  The
// warps' sums join in shared memory in a fixed order, one barrier a tile.  Where
// the columns of x do not fit in one SM, a cluster of 2, 4 or 8 CTAs
// splits k and joins through distributed shared memory.
constexpr int kQ4Warps = 16;
constexpr int kQ4MulThreads = kQ4Warps * 32;
constexpr int kQ4Tokens = 8;  // columns of one launch

struct Q4Shape {
    uint32_t wk, wr;       // warps of a tile, tiles in work: wk * wr = kQ4Warps
    uint32_t splits;       // CTAs of a cluster: parts of k
    uint32_t blocks;       // 256-column blocks of a CTA
    uint32_t rounds;       // tiles of a warp row
    uint32_t groups;       // clusters
    uint32_t x_row;        // bytes between columns of x in shared memory
    bool early, x_vec;
};

__device__ __forceinline__ uint4 ld_weights(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// (w & mask) | 0x64006400 in one instruction.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t biased(uint32_t w) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(MASK), "r"(0x64006400u));
    return r;
}

// The eight quants of a word as q - 8: operand registers 0..3.
__device__ __forceinline__ void quants(uint32_t w, uint32_t (&a)[4]) {
    const __half2 b1032 = __half2half2(__ushort_as_half(0x6408));  // 1024 + 8
    const __half2 b72 = __half2half2(__ushort_as_half(0xd480)), b16 = __half2half2(__ushort_as_half(0x2c00));  // -72, 1/16
    const uint32_t v = w >> 8;
    a[0] = h2_bits(__hsub2(bits_h2(biased<0x000f000fu>(w)), b1032));
    a[1] = h2_bits(__hfma2(bits_h2(biased<0x00f000f0u>(w)), b16, b72));
    a[2] = h2_bits(__hsub2(bits_h2(biased<0x000f000fu>(v)), b1032));
    a[3] = h2_bits(__hfma2(bits_h2(biased<0x00f000f0u>(v)), b16, b72));
}

// Scales of one 256-column block as a lane holds them: of its 64-column block
// t, slots (row g, group 0), (g, 1), (g + 8, 0), (g + 8, 1).
template <int CODE>
struct Q4Scales {
    uint32_t r[CODE == kDtypeQ4_0 ? 2 : 4];
    __device__ __forceinline__ void load(const uint8_t* rec, uint32_t lane) {
        if constexpr (CODE == kDtypeQ4_0) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(rec) + lane);
            r[0] = v.x;
            r[1] = v.y;
        } else if constexpr (CODE == kDtypeQ4_1) {
            const uint4 v = ld_weights(reinterpret_cast<const uint4*>(rec) + lane);
            r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
        } else {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(rec) + lane);
            const uint2 de = __ldg(reinterpret_cast<const uint2*>(rec + 256) + (lane >> 2));
            r[0] = v.x, r[1] = v.y, r[2] = de.x, r[3] = de.y;
        }
    }
    // a[row half][group], c likewise, of 64-column block j
    __device__ __forceinline__ void of(uint32_t lane, int j, float (&a)[2][2], float (&c)[2][2]) const {
        const uint32_t from = (lane & 28u) | (uint32_t)j;
        if constexpr (CODE == kDtypeQ4_0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2 f = __half22float2(bits_h2(__shfl_sync(0xffffffffu, r[h], from)));
                a[h][0] = f.x;
                a[h][1] = f.y;
            }
        } else if constexpr (CODE == kDtypeQ4_1) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float2 f = __half22float2(bits_h2(__shfl_sync(0xffffffffu, r[s], from)));
                a[s >> 1][s & 1] = f.x;
                c[s >> 1][s & 1] = __fmaf_rn(8.0f, f.x, f.y);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2 de = __half22float2(bits_h2(r[2 + h]));
                const uint32_t b = __shfl_sync(0xffffffffu, r[h], from);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    a[h][s] = de.x * (float)((b >> (16 * s)) & 255u);
                    c[h][s] = __fmaf_rn(8.0f, a[h][s], -de.y * (float)((b >> (16 * s + 8)) & 255u));
                }
            }
        }
    }
};

template <int CODE>
struct Q4Block {
    uint4 q[4];
    Q4Scales<CODE> s;
};

template <int CODE, int PARTS, int NT>
__global__ void __launch_bounds__(kQ4MulThreads, 1) q4_mul_kernel(const Q4MatvecPlan p, const Q4Shape shape) {
    constexpr int kCols = 8 * NT;
    constexpr bool kSums = CODE != kDtypeQ4_0;
    extern __shared__ __align__(16) unsigned char smem[];
    const uint32_t n = (uint32_t)p.n, cols = n * PARTS;
    float* red = reinterpret_cast<float*>(smem);                          // [2][warp][16][kCols]
    float* part = red + 2 * kQ4Warps * 16 * kCols;                        // [2][wr * 16 * n], splits > 1
    float* up = part + (shape.splits > 1 ? 2 * shape.wr * 16 * n : 0);    // [8]
    uint32_t* top = reinterpret_cast<uint32_t*>(up + kQ4Tokens);          // [8]
    float* xsum = reinterpret_cast<float*>(top + kQ4Tokens);              // [group][kCols]
    unsigned char* xs = reinterpret_cast<unsigned char*>(xsum + (kSums ? shape.blocks * 8 * kCols : 0));

    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3u;
    const uint32_t rank = shape.splits > 1 ? blockIdx.x % shape.splits : 0;
    const uint32_t group = shape.splits > 1 ? blockIdx.x / shape.splits : blockIdx.x;
    const uint64_t tiles = (p.rows + 15) / 16, k64 = (p.k + 63) / 64, k256 = (p.k + 255) / 256;
    const uint4* quads = reinterpret_cast<const uint4*>(p.weights);
    const uint8_t* scales = p.weights + tiles * k64 * 512;
    const uint32_t first = rank * shape.blocks;  // of this CTA's blocks
    const uint32_t here = first >= k256 ? 0u : (uint32_t)(k256 - first < shape.blocks ? k256 - first : shape.blocks);
    const uint32_t wk = warp % shape.wk, wr = warp / shape.wk;
    const uint32_t kb0 = wk * here / shape.wk, kb1 = (wk + 1) * here / shape.wk;

    // this warp's sequence of (tile, block): tiles group * wr + ..., blocks kb0 .. kb1
    struct At {
        uint64_t tile;
        uint32_t kb, round;
    };
    At ahead{(uint64_t)group * shape.wr + wr, kb0, 0};
    auto fetch_quads = [&](Q4Block<CODE>& b, const At& x, int j) {
        const uint64_t block = (uint64_t)(first + x.kb) * 4 + j;
        b.q[j] = x.round < shape.rounds && x.tile < tiles && block < k64 ? ld_weights(quads + (x.tile * k64 + block) * 32 + lane)
                                                                         : make_uint4(0, 0, 0, 0);
    };
    auto fetch_scales = [&](Q4Block<CODE>& b, const At& x) {
        if (x.round < shape.rounds && x.tile < tiles)
            b.s.load(scales + (x.tile * k256 + first + x.kb) * q4_scale_bytes(CODE), lane);
    };
    auto next = [&](At& x) {
        if (++x.kb == kb1) {
            x.kb = kb0;
            x.tile += (uint64_t)shape.groups * shape.wr;
            ++x.round;
        }
    };
    Q4Block<CODE> blk[2] = {};
    auto fill = [&]() {
        if (kb0 == kb1) return;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            fetch_scales(blk[s], ahead);
#pragma unroll
            for (int j = 0; j < 4; ++j) fetch_quads(blk[s], ahead, j);
            next(ahead);
        }
    };
    if (shape.early) fill();  // the previous kernel of the stream does not write the weights
    pdl_enter();
    if (!shape.early) fill();

    // ---- the columns of x
    const uint32_t pieces = here * 32;  // 8 values each; a multiple of 32: a warp stays in one token
    auto load8 = [&](uint32_t i, float (&v)[8]) {
        const uint32_t token = i / pieces;
        const uint64_t k = (uint64_t)first * 256 + (uint64_t)(i % pieces) * 8;
        const char* row = p.x + token * p.x_st;
        if constexpr (PARTS == 2) {
            const float* src = reinterpret_cast<const float*>(row) + k;
            if (shape.x_vec && k + 8 <= p.k) {
                const float4 lo = *reinterpret_cast<const float4*>(src), hi = *reinterpret_cast<const float4*>(src + 4);
                v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = k + e < p.k ? src[e] : 0.0f;
            }
        } else {
            const __half* src = reinterpret_cast<const __half*>(row) + k;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = k + e < p.k ? __half2float(src[e]) : 0.0f;
        }
    };
    if (here == 0 && threadIdx.x < kQ4Tokens) up[threadIdx.x] = 1.0f;  // a part of k beyond the matrix
    if constexpr (PARTS == 2) {
        if (threadIdx.x < kQ4Tokens) top[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n * pieces; i += kQ4MulThreads) {
            float v[8];
            load8(i, v);
            uint32_t big = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t b = fbits(v[e]) & 0x7fffffffu;
                big = b < 0x7f800000u && b > big ? b : big;
            }
            big = __reduce_max_sync(0xffffffffu, big);
            if (lane == 0) atomicMax(top + i / pieces, big);
        }
        __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < n * pieces; i += kQ4MulThreads) {
        const uint32_t token = i / pieces, at = i % pieces;
        float v[8];
        load8(i, v);
        float scale = 1.0f;
        if constexpr (PARTS == 2) {
            const int e = 127 + 14 + 127 - (int)(top[token] >> 23);  // exponent field of 2^14 / largest
            scale = top[token] == 0 ? 1.0f : bitsf((uint32_t)(e > 254 ? 254 : e) << 23);
            if (at == 0) up[token] = 1.0f / scale;
        } else if (at == 0) {
            up[token] = 1.0f;
        }
        float sum = 0.0f;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = v[2 * e] * scale, b = v[2 * e + 1] * scale;
            const __half2 h = __floats2half2_rn(a, b);
            hi[e] = h2_bits(h);
            if constexpr (PARTS == 2) {
                const float2 f = __half22float2(h);
                const float ra = a - f.x, rb = b - f.y;  // NaN for an infinity: the first part carries it alone
                lo[e] = h2_bits(__floats2half2_rn(fabsf(ra) < INFINITY ? ra : 0.0f, fabsf(rb) < INFINITY ? rb : 0.0f));
            }
            if constexpr (kSums) sum += a + b;
        }
        *reinterpret_cast<uint4*>(xs + token * shape.x_row + at * 16) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (PARTS == 2)
            *reinterpret_cast<uint4*>(xs + (n + token) * shape.x_row + at * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if constexpr (kSums) {  // of a group of 32: four lanes; it stands in the token's first column
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if ((at & 3u) == 0) {
                xsum[(at >> 2) * kCols + token] = sum;
                if constexpr (PARTS == 2) xsum[(at >> 2) * kCols + n + token] = 0.0f;
            }
        }
    }
    if constexpr (kSums) {
        const uint32_t rest = kCols - cols;  // columns that nobody reads: numbers, not what lay there
        for (uint32_t i = threadIdx.x; i < here * 8 * rest; i += kQ4MulThreads) xsum[i / rest * kCols + cols + i % rest] = 0.0f;
    }
    __syncthreads();

    // lanes of unused columns read the first one: their results are not used
    const unsigned char* x_at[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c) x_at[c] = xs + (8 * c + g < cols ? 8 * c + g : 0) * shape.x_row + t * 16;

    float total[NT][4];
    auto work = [&](Q4Block<CODE>& b, uint32_t kb) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a[2][2], c[2][2];
            b.s.of(lane, j, a, c);
            const uint32_t w[4] = {b.q[j].x, b.q[j].y, b.q[j].z, b.q[j].w};
            fetch_quads(b, ahead, j);
#pragma unroll
            for (int G = 0; G < 2; ++G) {
                const uint32_t at = (kb * 8 + j * 2 + G) * 64;
                float acc[NT][4] = {};
                uint32_t f[4], f2[4];
                quants(w[2 * G], f);
                quants(w[2 * G + 1], f2);
#pragma unroll
                for (int m = 0; m < NT; ++m) {
                    const uint4 x = *reinterpret_cast<const uint4*>(x_at[m] + at);
                    mma_f16(acc[m], f, x.x, x.y);
                    mma_f16(acc[m], f2, x.z, x.w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) total[m][e] = __fmaf_rn(a[e >> 1][G], acc[m][e], total[m][e]);
                    if constexpr (kSums) {
                        const float2 s = *reinterpret_cast<const float2*>(xsum + (kb * 8 + j * 2 + G) * kCols + 8 * m + 2 * t);
                        total[m][0] = __fmaf_rn(c[0][G], s.x, total[m][0]);
                        total[m][1] = __fmaf_rn(c[0][G], s.y, total[m][1]);
                        total[m][2] = __fmaf_rn(c[1][G], s.x, total[m][2]);
                        total[m][3] = __fmaf_rn(c[1][G], s.y, total[m][3]);
                    }
                }
            }
        }
        fetch_scales(b, ahead);
        next(ahead);
    };

    const uint32_t values = shape.wk * PARTS, outs = shape.wr * 16 * n;  // values of a sum: a power of two, at most 32
    auto store = [&](uint64_t tile0, uint32_t o, float y) {
        const uint32_t row = o & 15u, token = (o >> 4) % n;
        const uint64_t r = (tile0 + (o >> 4) / n) * 16 + row;
        if (r >= p.rows) return;
        char* at = p.dst + token * p.dst_st;
        if (p.dst_f16) reinterpret_cast<__half*>(at)[r] = __float2half_rn(y);
        else reinterpret_cast<float*>(at)[r] = y;
    };
    uint32_t odd = 0;  // which of the two blocks comes next
    for (uint32_t round = 0; round < shape.rounds; ++round) {
        const uint64_t tile0 = ((uint64_t)round * shape.groups + group) * shape.wr;
#pragma unroll
        for (int m = 0; m < NT; ++m) total[m][0] = total[m][1] = total[m][2] = total[m][3] = 0.0f;
        uint32_t kb = kb0;
        if (tile0 + wr < tiles) {
            if (odd && kb < kb1) {
                work(blk[1], kb++);
                odd = 0;
            }
            for (; kb + 2 <= kb1; kb += 2) {
                work(blk[0], kb);
                work(blk[1], kb + 1);
            }
            if (kb < kb1) {
                work(blk[0], kb);
                odd = 1;
            }
        }
        float* mine = red + ((round & 1u) * kQ4Warps + warp) * 16 * kCols;
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            *reinterpret_cast<float2*>(mine + g * kCols + 8 * m + 2 * t) = make_float2(total[m][0], total[m][1]);
            *reinterpret_cast<float2*>(mine + (g + 8) * kCols + 8 * m + 2 * t) = make_float2(total[m][2], total[m][3]);
        }
        __syncthreads();
        // output o = (tile, token, row): its values are summed by `values` adjacent lanes
        const uint32_t per = 32 / values, v = lane % values;
        for (uint32_t base = warp * per; base < outs; base += kQ4Warps * per) {
            const uint32_t o = base + lane / values;
            float y = 0.0f;
            if (o < outs) {
                const uint32_t token = (o >> 4) % n, w = (o >> 4) / n * shape.wk + v / PARTS;
                y = red[(((round & 1u) * kQ4Warps + w) * 16 + (o & 15u)) * kCols + (v % PARTS) * n + token];
            }
            for (uint32_t d = values >> 1; d > 0; d >>= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
            if (v == 0 && o < outs) {
                y *= up[(o >> 4) % n];
                if (shape.splits > 1) part[(round & 1u) * outs + o] = y;
                else store(tile0, o, y);
            }
        }
        if (shape.splits > 1) {
            cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
            cluster.sync();
            for (uint32_t o = threadIdx.x * shape.splits + rank; o < outs; o += kQ4MulThreads * shape.splits) {
                float y = 0.0f;
                for (uint32_t r = 0; r < shape.splits; ++r) y += cluster.map_shared_rank(part, r)[(round & 1u) * outs + o];
                store(tile0, o, y);
            }
        }
    }
    if (shape.splits > 1) cooperative_groups::this_cluster().sync();  // the others may still read this CTA's part
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

constexpr uint64_t kSharedMost = 227 * 1024;

uint64_t q4_shared_bytes(const Q4Shape& s, int code, int parts, int tiles8, uint64_t n) {
    const uint64_t cols = 8 * tiles8;
    return 2 * kQ4Warps * 16 * cols * 4 + (s.splits > 1 ? 2 * s.wr * 16 * n * 4 : 0) + kQ4Tokens * 8 +
           (code != kDtypeQ4_0 ? s.blocks * 8 * cols * 4 : 0) + n * parts * (uint64_t)s.x_row;
}

template <int CODE, int PARTS, int NT>
cudaError_t run_q4_at(const LaunchEnv& env, const Q4MatvecPlan& p, const Q4Shape& shape, uint64_t smem) {
    static DeviceFlags ready;
    if (!ready.done(env.device)) {
        const cudaError_t err = cudaFuncSetAttribute(q4_mul_kernel<CODE, PARTS, NT>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSharedMost);
        if (err != cudaSuccess) return err;
        ready.mark(env.device);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(shape.groups * shape.splits);
    cfg.blockDim = dim3(kQ4MulThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = env.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = shape.splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = shape.splits > 1 ? 2 : 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, q4_mul_kernel<CODE, PARTS, NT>, p, shape);
    if (err == cudaSuccess) ++*env.launches;
    return err;
}

// One launch: at most kQ4Tokens columns of x.
template <int CODE>
cudaError_t run_q4(const LaunchEnv& env, const Q4MatvecPlan& p, const Q4Shape& shape, uint64_t smem) {
    if (p.x_f16) return run_q4_at<CODE, 1, 1>(env, p, shape, smem);
    if (2 * p.n <= 8) return run_q4_at<CODE, 2, 1>(env, p, shape, smem);
    return run_q4_at<CODE, 2, 2>(env, p, shape, smem);
}

// How k and the rows are cut; false when the columns of x do not fit.
bool q4_shape(const LaunchEnv& env, const Q4MatvecPlan& p, Q4Shape* out, uint64_t* smem) {
    const int parts = p.x_f16 ? 1 : 2, tiles8 = (int)((p.n * parts + 7) / 8);
    const uint64_t tiles = (p.rows + 15) / 16, k256 = (p.k + 255) / 256;
    for (uint32_t splits = 1; splits <= 8; splits *= 2) {
        Q4Shape s{};
        s.splits = splits;
        s.blocks = (uint32_t)((k256 + splits - 1) / splits);
        s.x_row = s.blocks * 512 + 64;  // 64 mod 128: two columns' 16-byte pieces meet no bank twice
        const uint64_t groups = (uint64_t)env.sm_count / splits;
        // fewest blocks one after another in a warp; a round costs a barrier
        // and a join besides, about half a block's time
        uint64_t best = UINT64_MAX;
        for (uint32_t wk = 1; wk <= kQ4Warps; wk *= 2) {
            const uint32_t wr = kQ4Warps / wk;
            const uint64_t rounds = (tiles + groups * wr - 1) / (groups * wr), serial = (s.blocks + wk - 1) / wk;
            const uint64_t cost = rounds * (2 * serial + 1);
            if (cost >= best) continue;
            best = cost;
            s.wk = wk;
            s.wr = wr;
            s.rounds = (uint32_t)rounds;
            s.groups = (uint32_t)((tiles + rounds * wr - 1) / (rounds * wr));
        }
        *smem = q4_shared_bytes(s, p.code, parts, tiles8, p.n);
        *out = s;
        if (*smem <= kSharedMost) return true;
    }
    return false;
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

cudaError_t launch_mul_mat_q4(const LaunchEnv& env, const Q4MatvecPlan& plan) {
    uint64_t packed = 0;
    q4_packed_bytes(plan.code, plan.k, plan.rows, &packed);
    const bool early = reads_clear(env, plan.weights, packed);
    for (uint64_t at = 0; at < plan.n;) {
        Q4MatvecPlan p = plan;
        p.x = plan.x + at * plan.x_st;
        p.dst = plan.dst + at * plan.dst_st;
        p.n = plan.n - at < kQ4Tokens ? plan.n - at : kQ4Tokens;
        Q4Shape shape{};
        uint64_t smem = 0;
        while (!q4_shape(env, p, &shape, &smem)) {
            if (p.n == 1) return cudaErrorInvalidValue;
            p.n = (p.n + 1) / 2;
        }
        shape.early = at == 0 ? early : true;  // the product before it writes no weights
        shape.x_vec = !plan.x_f16 && ((reinterpret_cast<uintptr_t>(p.x) | (p.n > 1 ? p.x_st : 0)) & 15u) == 0;
        cudaError_t err = cudaSuccess;
        if (p.code == kDtypeQ4_0) err = run_q4<kDtypeQ4_0>(env, p, shape, smem);
        else if (p.code == kDtypeQ4_1) err = run_q4<kDtypeQ4_1>(env, p, shape, smem);
        else err = run_q4<kDtypeQ4_K>(env, p, shape, smem);
        if (err != cudaSuccess) return err;
        at += p.n;
    }
    stream_wrote(env.stream, plan.dst, (plan.n - 1) * plan.dst_st + plan.rows * (plan.dst_f16 ? 2 : 4));
    return cudaSuccess;
}

}  // namespace emel
