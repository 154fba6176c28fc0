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

// Quants k .. k + 3 of a source row (k a multiple of 4), one in the low half of
// each byte: adjacent columns stand in adjacent bytes, of one half or the other.
template <int CODE>
__device__ __forceinline__ uint32_t q4_quants(const uint8_t* row, uint64_t k, bool even) {
    const uint32_t i = (uint32_t)k & 31u;
    const uint8_t* from;
    bool high;
    if constexpr (CODE == kDtypeQ4_K) {
        const uint32_t sub = ((uint32_t)k & 255u) >> 5;
        from = row + (k >> 8) * 144 + 16 + 32 * (sub >> 1) + i;
        high = sub & 1u;
    } else {
        constexpr int kBlock = CODE == kDtypeQ4_0 ? 18 : 20;
        from = row + (k >> 5) * kBlock + (kBlock - 16) + (i & 15u);
        high = i >= 16;
    }
    uint32_t v;
    if (even) v = reinterpret_cast<const uint16_t*>(from)[0] | (uint32_t)reinterpret_cast<const uint16_t*>(from)[1] << 16;
    else v = from[0] | (uint32_t)from[1] << 8 | (uint32_t)from[2] << 16 | (uint32_t)from[3] << 24;
    return (high ? v >> 4 : v) & 0x0f0f0f0fu;
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
                for (int h = 0; h < 2; ++h) {  // rows g and g + 8: columns k, k + 2, k + 1, k + 3 in a word's bytes
                    const uint32_t q = row[h] < p.rows && k < p.k ? q4_quants<CODE>(p.src + row[h] * p.row_bytes, k, p.even) : 0x08080808u;
                    w[j] |= __byte_perm(q, 0, 0x3120) << (4 * h);
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
// three instructions a weight at full bandwidth, shared by all pipes.  So
// tensor products multiply 16 rows with 8 columns at once, and the quants reach
// them with as little work as the number of tokens allows.
//
// One or two tokens (q4_digits_kernel, m16n8k32 on 8-bit integers): a mask
// leaves four quants of a word, a shift and a mask the other four, three
// instructions for 8 weights.  A token is x 2^e rounded to an integer of 31
// bits (e per token and CTA: the largest finite |x| in [2^29, 2^30), subnormals below), and its four
// balanced digits to the base 256 are four columns.  A group's integer sum is exact; it
// comes out of the product on top of the bits of 1.5 2^23, so that one
// addition, of minus that and 8 times the digits' sum, makes sum((q - 8) digit) a
// binary32 number.
//
// More tokens (q4_halves_kernel, m16n8k16 on binary16): a mask leaves the bits
// of 1024 + q or, four bits higher up, of 1024 + 16 q, one subtraction or
// multiply-add makes q - 8 of them, exactly (the conversion by 1024's exponent as
// published for mixed-precision products: Kim, Henry, Fahim and Awadalla, "Who Says
// Elephants Can't Run", 2022); nine instructions for 8 weights.
// (The masked bits alone, as the subnormals q 2^-24, would take five, but
// their products came out with errors of 2^-17.)  A binary16
// token is one column as it is; a binary32 token is two, x 2^e = hi + lo, both
// rounded to binary16, the largest finite |x| in [2^14, 2^15): 22 bits and more, down to
// 2^-40 of the largest.
//
// The scales meet the products of a group, in binary32.
//
// A persistent CTA of 16 warps keeps its columns of x in shared memory and
// walks tiles of 16 rows.  WK warps share a tile (each a part of its 256-column
// blocks), WR tiles are in work; a warp holds two blocks of weights in
// registers and asks for the next one piece by piece as it uses them up.  The
// warps' sums join in shared memory in a fixed order, one barrier a tile.  Where
// the columns of x do not fit in one SM, a cluster of 2, 4 or 8 CTAs
// splits k and joins through distributed shared memory.
//
// One token, 4096 columns: 151936 rows of Q4_0, 350 MB, bound by HBM, 57 us in short
// runs, 6.1 TB/s, and 65 us where a long run meets the power limit; 14336 rows of
// Q4_K, 33 MB, 11.4 us, of which about 4 are start and preparation; whole rounds of
// tiles leave 112 of 148 SMs with work there.  Eight binary32 tokens,
// 11007 rows of Q4_1: 19.0 us, bound by instructions; binary16 tokens 13.0 us.
constexpr int kQ4Warps = 16;
constexpr int kQ4MulThreads = kQ4Warps * 32;
constexpr int kQ4Tokens = 8;  // columns of one launch
constexpr int kQ4DigitTokens = 2;

struct Q4Shape {
    uint32_t wk, wr;       // warps of a tile, tiles in work: wk * wr = kQ4Warps
    uint32_t splits;       // CTAs of a cluster: parts of k
    uint32_t blocks;       // 256-column blocks of a CTA
    uint32_t rounds;       // tiles of a warp row
    uint32_t groups;       // clusters
    uint32_t x_row;        // bytes between columns of x in shared memory
    bool early, x_vec;
};

// Loads into v where `in`; v keeps its value otherwise.
__device__ __forceinline__ void load_if(uint4& v, const uint4* p, bool in) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
        "@p ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}"
        : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
        : "l"(p), "r"((uint32_t)in));
}
__device__ __forceinline__ void load_if(uint2& v, const uint2* p, bool in) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\t"
        "@p ld.global.nc.v2.u32 {%0,%1}, [%2];\n\t}"
        : "+r"(v.x), "+r"(v.y)
        : "l"(p), "r"((uint32_t)in));
}

// d = a b + 0
__device__ __forceinline__ void mma_half(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// d += a b
__device__ __forceinline__ void mma_half_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a b + c in every element, integers
__device__ __forceinline__ void mma_digits(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                           uint32_t b0, uint32_t b1, uint32_t c) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c));
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// (w & MASK) | base in one instruction
template <uint32_t MASK>
__device__ __forceinline__ uint32_t mask_or(uint32_t w, uint32_t base) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(MASK), "r"(base));
    return r;
}

// The eight quants of a word as binary16 q - 8: operand registers 0..3.
__device__ __forceinline__ void half_quants(uint32_t w, uint32_t (&a)[4]) {
    const __half2 b1032 = __half2half2(__ushort_as_half(0x6408));  // 1024 + 8
    const __half2 b72 = __half2half2(__ushort_as_half(0xd480)), b16 = __half2half2(__ushort_as_half(0x2c00));  // -72, 1/16
    const uint32_t v = w >> 8, base = 0x64006400u;
    a[0] = h2_bits(__hsub2(bits_h2(mask_or<0x000f000fu>(w, base)), b1032));
    a[1] = h2_bits(__hfma2(bits_h2(mask_or<0x00f000f0u>(w, base)), b16, b72));
    a[2] = h2_bits(__hsub2(bits_h2(mask_or<0x000f000fu>(v, base)), b1032));
    a[3] = h2_bits(__hfma2(bits_h2(mask_or<0x00f000f0u>(v, base)), b16, b72));
}

// t += a (d + b) for the two columns of rows g (a0) and g + 8 (a1), on packed
// pairs of binary32: half the instructions (2 to 5 % of the time).
__device__ __forceinline__ void add_scaled(float (&t)[4], float a0, float a1, const uint32_t (&d)[4], float b0, float b1) {
    asm("{\n\t.reg .b64 x, y, b, p, q, t, u;\n\t"
        "mov.b64 x, {%4, %5};\n\tmov.b64 y, {%6, %7};\n\tmov.b64 b, {%8, %9};\n\t"
        "mov.b64 p, {%10, %10};\n\tmov.b64 q, {%11, %11};\n\tmov.b64 t, {%0, %1};\n\tmov.b64 u, {%2, %3};\n\t"
        "add.rn.f32x2 x, x, b;\n\tadd.rn.f32x2 y, y, b;\n\tfma.rn.f32x2 t, p, x, t;\n\tfma.rn.f32x2 u, q, y, u;\n\t"
        "mov.b64 {%0, %1}, t;\n\tmov.b64 {%2, %3}, u;\n\t}"
        : "+f"(t[0]), "+f"(t[1]), "+f"(t[2]), "+f"(t[3])
        : "r"(d[0]), "r"(d[1]), "r"(d[2]), "r"(d[3]), "f"(b0), "f"(b1), "f"(a0), "f"(a1));
}

// t += a x for the two columns of rows g (a0) and g + 8 (a1), likewise.
__device__ __forceinline__ void add_scaled(float (&t)[4], float a0, float a1, float x0, float x1, float x2, float x3) {
    asm("{\n\t.reg .b64 x, y, p, q, t, u;\n\t"
        "mov.b64 x, {%4, %5};\n\tmov.b64 y, {%6, %7};\n\tmov.b64 p, {%8, %8};\n\tmov.b64 q, {%9, %9};\n\t"
        "mov.b64 t, {%0, %1};\n\tmov.b64 u, {%2, %3};\n\tfma.rn.f32x2 t, p, x, t;\n\tfma.rn.f32x2 u, q, y, u;\n\t"
        "mov.b64 {%0, %1}, t;\n\tmov.b64 {%2, %3}, u;\n\t}"
        : "+f"(t[0]), "+f"(t[1]), "+f"(t[2]), "+f"(t[3])
        : "f"(x0), "f"(x1), "f"(x2), "f"(x3), "f"(a0), "f"(a1));
}

// Scales of one 256-column block as a lane holds them: of its 64-column block
// t, slots (row g, group 0), (g, 1), (g + 8, 0), (g + 8, 1).
template <int CODE>
struct Q4Scales {
    uint4 r;  // Q4_0: x, y; Q4_K: x, y and the (d, e) of its two rows
    __device__ __forceinline__ void load(const uint8_t* rec, uint32_t lane, bool in) {
        if constexpr (CODE == kDtypeQ4_1) {
            load_if(r, reinterpret_cast<const uint4*>(rec) + lane, in);
        } else {
            uint2 v = make_uint2(r.x, r.y);
            load_if(v, reinterpret_cast<const uint2*>(rec) + lane, in);
            r.x = v.x, r.y = v.y;
            if constexpr (CODE == kDtypeQ4_K) {
                uint2 de = make_uint2(r.z, r.w);
                load_if(de, reinterpret_cast<const uint2*>(rec + 256) + (lane >> 2), in);
                r.z = de.x, r.w = de.y;
            }
        }
    }
    // Q4_K: a and c of this lane's own slots, once a block (28 instructions; of
    // every 64-column block anew they took a quarter of all)
    __device__ __forceinline__ void own(float (&a)[4], float (&c)[4]) const {
        if constexpr (CODE == kDtypeQ4_K) {
            // a byte under the exponent of 2^23 is 2^23 + byte
            const auto value = [](uint32_t b, uint32_t at) { return bitsf(__byte_perm(b, 0x4b000000u, 0x7440u + at)) - 8388608.0f; };
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float2 de = __half22float2(bits_h2(s & 2 ? r.w : r.z));
                const uint32_t b = s & 2 ? r.y : r.x;
                a[s] = de.x * value(b, 2 * (s & 1));
                c[s] = __fmaf_rn(8.0f, a[s], -de.y * value(b, 2 * (s & 1) + 1));
            }
        }
    }
    // a[row half][group], c likewise (Q4_0: not used), of 64-column block j
    __device__ __forceinline__ void of(uint32_t lane, int j, const float (&own_a)[4], const float (&own_c)[4], float (&a)[2][2],
                                       float (&c)[2][2]) const {
        const uint32_t from = (lane & 28u) | (uint32_t)j;
        if constexpr (CODE == kDtypeQ4_0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2 f = __half22float2(bits_h2(__shfl_sync(0xffffffffu, h ? r.y : r.x, from)));
                a[h][0] = f.x;
                a[h][1] = f.y;
            }
        } else if constexpr (CODE == kDtypeQ4_1) {
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float2 f = __half22float2(bits_h2(__shfl_sync(0xffffffffu, w[s], from)));
                a[s >> 1][s & 1] = f.x;
                c[s >> 1][s & 1] = __fmaf_rn(8.0f, f.x, f.y);
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                a[s >> 1][s & 1] = __shfl_sync(0xffffffffu, own_a[s], from);
                c[s >> 1][s & 1] = __shfl_sync(0xffffffffu, own_c[s], from);
            }
        }
    }
};

template <int CODE>
struct Q4Block {
    uint4 q[4];
    Q4Scales<CODE> s;
};

// Where a CTA and a warp stand: their parts of k and of the tiles.
struct Q4Place {
    uint64_t tiles, k64, k256;
    uint32_t lane, warp, wk, wr, rank, group;
    uint32_t first, here;  // the CTA's 256-column blocks
    uint32_t kb0, kb1;     // the warp's, from `first` on
    __device__ __forceinline__ Q4Place(const Q4MatvecPlan& p, const Q4Shape& shape) {
        lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
        rank = shape.splits > 1 ? blockIdx.x % shape.splits : 0;
        group = shape.splits > 1 ? blockIdx.x / shape.splits : blockIdx.x;
        tiles = (p.rows + 15) / 16, k64 = (p.k + 63) / 64, k256 = (p.k + 255) / 256;
        first = rank * shape.blocks;
        here = first >= k256 ? 0u : (uint32_t)(k256 - first < shape.blocks ? k256 - first : shape.blocks);
        wk = warp % shape.wk, wr = warp / shape.wk;
        kb0 = wk * here / shape.wk, kb1 = (wk + 1) * here / shape.wk;
    }
};

// A warp's blocks in order: tiles group * wr + ..., of each kb0 .. kb1.  Quads
// that do not exist (the last block of a row may hold less than four) keep
// old bits: the columns of x under them are zeros, and so are their scales.
template <int CODE>
struct Q4Stream {
    const uint4* q;
    const uint8_t* s;
    uint64_t q_step, s_step;  // from the end of a tile's part to the next tile's
    uint32_t kb, kb0, kb1, left, lane, short_kb, short_n, quads;
    __device__ __forceinline__ Q4Stream(const Q4MatvecPlan& p, const Q4Shape& shape, const Q4Place& w) {
        const uint64_t tile = (uint64_t)w.group * shape.wr + w.wr, step = (uint64_t)shape.groups * shape.wr;
        lane = w.lane;
        kb = kb0 = w.kb0;
        kb1 = w.kb1;
        left = kb0 == kb1 || tile >= w.tiles ? 0u : (uint32_t)((w.tiles - 1 - tile) / step) + 1;
        q = reinterpret_cast<const uint4*>(p.weights) + (tile * w.k64 + (uint64_t)(w.first + kb0) * 4) * 32 + lane;
        s = p.weights + w.tiles * w.k64 * 512 + (tile * w.k256 + w.first + kb0) * q4_scale_bytes(CODE);
        q_step = (step * w.k64 - (uint64_t)(kb1 - kb0) * 4) * 32;
        s_step = (step * w.k256 - (kb1 - kb0)) * q4_scale_bytes(CODE);
        short_kb = w.first + w.here == w.k256 && (w.k64 & 3u) ? w.here - 1 : 0xffffffffu;
        short_n = (uint32_t)w.k64 & 3u;
        count();
    }
    __device__ __forceinline__ void count() { quads = left == 0 ? 0u : kb == short_kb ? short_n : 4u; }
    __device__ __forceinline__ void fetch_quads(Q4Block<CODE>& b, int j) { load_if(b.q[j], q + j * 32, (uint32_t)j < quads); }
    __device__ __forceinline__ void fetch_scales(Q4Block<CODE>& b) { b.s.load(s, lane, quads != 0); }
    __device__ __forceinline__ void next() {
        q += 128;
        s += q4_scale_bytes(CODE);
        if (++kb == kb1) {
            kb = kb0;
            q += q_step;
            s += s_step;
            left -= left != 0;
        }
        count();
    }
    __device__ __forceinline__ void fill(Q4Block<CODE> (&b)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fetch_scales(b[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) fetch_quads(b[i], j);
            next();
        }
    }
};

// Pieces of 8 values of x, shared out over the CTA; a warp stays in one token.
struct Q4Piece {
    uint32_t token, at;
    __device__ __forceinline__ void next(uint32_t pieces) {
        at += kQ4MulThreads;
        while (at >= pieces) {
            at -= pieces;
            ++token;
        }
    }
};

// The 8 values of a piece as they lie in memory: 16 bytes of binary16, or 32 of
// binary32; zeros beyond k (a multiple of 32: no piece is cut).
template <bool F32>
__device__ __forceinline__ void load_piece(const Q4MatvecPlan& p, bool vec, uint64_t k, uint32_t token, bool in, uint4 (&v)[F32 ? 2 : 1]) {
    const char* src = p.x + token * p.x_st + k * (F32 ? 4 : 2);
#pragma unroll
    for (int h = 0; h < (F32 ? 2 : 1); ++h) v[h] = make_uint4(0, 0, 0, 0);
    if (!in || k >= p.k) return;
    if (vec) {
#pragma unroll
        for (int h = 0; h < (F32 ? 2 : 1); ++h) v[h] = *reinterpret_cast<const uint4*>(src + 16 * h);
        return;
    }
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < (F32 ? 8 : 4); ++e) {
        if constexpr (F32) w[e] = reinterpret_cast<const uint32_t*>(src)[e];
        else w[e] = reinterpret_cast<const uint16_t*>(src)[2 * e] | (uint32_t)reinterpret_cast<const uint16_t*>(src)[2 * e + 1] << 16;
    }
    v[0] = make_uint4(w[0], w[1], w[2], w[3]);
    if constexpr (F32) v[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// The largest magnitude (bits) among eight binary32 values: above kInfinity if
// one is a NaN.
constexpr uint32_t kInfinity = 0x7f800000u;
__device__ __forceinline__ uint32_t largest_of(const uint32_t (&w)[8]) {
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) big = max(big, w[e] & 0x7fffffffu);
    return big;
}

// The exponent field (127 + e) of the power of two 2^e that brings `largest` (bits,
// finite) into [2^to, 2^(to + 1)), or below where it is subnormal; of 1 for 0.  Above
// 254 it is no number's: e is then 127 and a rest, two exact steps.
__device__ __forceinline__ uint32_t scale_to(uint32_t largest, int to) {
    return largest == 0 ? 127u : (uint32_t)(127 + to + 127 - (int)(largest >> 23));
}
__device__ __forceinline__ uint32_t first_step(uint32_t field) { return field > 254 ? 254u : field; }
__device__ __forceinline__ uint32_t rest_step(uint32_t field) { return 127 + field - first_step(field); }
__device__ __forceinline__ float power(uint32_t field) { return bitsf(field << 23); }
// 1 / power(field), a subnormal for the largest
__device__ __forceinline__ float inverse_power(uint32_t field) { return bitsf(field < 254 ? (254 - field) << 23 : 0x00400000u); }

// The sums of a round: every warp's [16 rows][COLS] lie in shared memory, 8
// floats apart beyond their size; the output (tile, row, token) is the sum over
// its WK warps and PARTS columns, part i weighted by `weight`^i.  Four lanes, 8
// apart, share an output: lane quarter s takes warps s, s + 4, ..., so the 32
// lanes read 32 banks.
constexpr uint32_t kQ4RedPad = 8;
template <int PARTS, int COLS>
__device__ __forceinline__ void q4_join(const Q4MatvecPlan& p, const Q4Shape& shape, const Q4Place& w, uint32_t round,
                                        const float* sums, float* part, const float* up, float weight) {
    constexpr uint32_t kWarp = 16 * COLS + kQ4RedPad;
    const uint32_t n = (uint32_t)p.n, outs = shape.wr * 16 * n, over_n = (65535 + n) / n;
    const uint64_t row0 = ((uint64_t)round * shape.groups + w.group) * shape.wr * 16;
    auto store = [&](uint32_t row, uint32_t token, float y) {
        const uint64_t r = row0 + row;
        if (r >= p.rows) return;
        char* at = p.dst + token * p.dst_st;
        if (p.dst_f16) reinterpret_cast<__half*>(at)[r] = __float2half_rn(y);
        else reinterpret_cast<float*>(at)[r] = y;
    };
    const uint32_t quarter = w.lane >> 3;
    for (uint32_t base = w.warp * 8; base < outs; base += kQ4Warps * 8) {
        const uint32_t o = base + (w.lane & 7u);  // outs is a multiple of 8
        const uint32_t row = (o * over_n) >> 16, token = o - row * n;  // o / n, exact for o <= 2048, n <= 8
        float y[PARTS] = {};
        const float* at = sums + ((row >> 4) * shape.wk + quarter) * kWarp + (row & 15u) * COLS + token;
#pragma unroll 4
        for (uint32_t v = quarter; v < shape.wk; v += 4, at += 4 * kWarp)
#pragma unroll
            for (int i = 0; i < PARTS; ++i) y[i] += at[i * n];
        float all = y[PARTS - 1];
#pragma unroll
        for (int i = PARTS - 2; i >= 0; --i) all = __fmaf_rn(all, weight, y[i]);
        all += __shfl_xor_sync(0xffffffffu, all, 8);
        all += __shfl_xor_sync(0xffffffffu, all, 16);
        if (quarter == 0) {
            if constexpr (PARTS == 4) all *= up[kQ4Tokens + token];  // digits: exact, the last rounding is the next one
            all *= up[token];
            if (shape.splits > 1) part[(round & 1u) * outs + o] = all;
            else store(row, token, all);
        }
    }
    if (shape.splits > 1) {
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster.sync();
        for (uint32_t o = threadIdx.x * shape.splits + w.rank; o < outs; o += kQ4MulThreads * shape.splits) {
            const uint32_t row = (o * over_n) >> 16, token = o - row * n;
            float y = 0.0f;
            for (uint32_t r = 0; r < shape.splits; ++r) y += cluster.map_shared_rank(part, r)[(round & 1u) * outs + o];
            store(row, token, y);
        }
    }
}

// Walks the rounds: `work(block, kb)` adds one block to the warp's `total`.
template <int CODE, int PARTS, int NT, typename Work>
__device__ __forceinline__ void q4_rounds(const Q4MatvecPlan& p, const Q4Shape& shape, const Q4Place& w, Q4Block<CODE> (&blk)[2],
                                          float (&total)[NT][4], float* red, float* part, const float* up, float weight,
                                          Work&& work) {
    constexpr int kCols = 8 * NT;
    const uint32_t g = w.lane >> 2, t = w.lane & 3u;
    uint32_t odd = 0;  // which of the two blocks comes next
    for (uint32_t round = 0; round < shape.rounds; ++round) {
#pragma unroll
        for (int m = 0; m < NT; ++m) total[m][0] = total[m][1] = total[m][2] = total[m][3] = 0.0f;
        uint32_t kb = w.kb0;
        if (((uint64_t)round * shape.groups + w.group) * shape.wr + w.wr < w.tiles) {
            if (odd && kb < w.kb1) {
                work(blk[1], kb++);
                odd = 0;
            }
            for (; kb + 2 <= w.kb1; kb += 2) {
                work(blk[0], kb);
                work(blk[1], kb + 1);
            }
            if (kb < w.kb1) {
                work(blk[0], kb);
                odd = 1;
            }
        }
        float* sums = red + (round & 1u) * kQ4Warps * (16 * kCols + kQ4RedPad);
        float* mine = sums + w.warp * (16 * kCols + kQ4RedPad);
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            *reinterpret_cast<float2*>(mine + g * kCols + 8 * m + 2 * t) = make_float2(total[m][0], total[m][1]);
            *reinterpret_cast<float2*>(mine + (g + 8) * kCols + 8 * m + 2 * t) = make_float2(total[m][2], total[m][3]);
        }
        __syncthreads();
        q4_join<PARTS, kCols>(p, shape, w, round, sums, part, up, weight);
    }
    if (shape.splits > 1) cooperative_groups::this_cluster().sync();  // the others may still read this CTA's part
}

// Shared memory of both kernels: the warps' sums, the cluster's, the tokens'
// scales, tables of the groups and the columns of x.
template <int NT>
struct Q4Shared {
    float* red;      // [2][warp][16][8 NT], padded
    float* part;     // [2][wr * 16 * n], splits > 1
    float* up;       // [2][kQ4Tokens]: 2^-e of the first step, of the rest
    uint32_t* top;   // [kQ4Tokens]: bits of the largest finite |x|
    float* table;    // per group
    unsigned char* xs;
    __device__ __forceinline__ Q4Shared(unsigned char* smem, const Q4Shape& shape, uint32_t n, uint32_t table_floats) {
        red = reinterpret_cast<float*>(smem);
        part = red + 2 * kQ4Warps * (16 * 8 * NT + kQ4RedPad);
        up = part + (shape.splits > 1 ? 2 * shape.wr * 16 * n : 0);
        top = reinterpret_cast<uint32_t*>(up + 2 * kQ4Tokens);
        table = reinterpret_cast<float*>(top + kQ4Tokens);
        xs = reinterpret_cast<unsigned char*>(table + shape.blocks * 8 * table_floats);
    }
};

constexpr int kQ4Batch = 4, kQ4DigitBatch = 2;  // pieces of x that a thread has in flight

// PARTS columns a token (1: binary16 x, 2: binary32 x), NT * 8 columns.
template <int CODE, int PARTS, int NT>
__global__ void __launch_bounds__(kQ4MulThreads, 1) q4_halves_kernel(const Q4MatvecPlan p, const Q4Shape shape) {
    constexpr int kCols = 8 * NT;
    constexpr bool kSums = CODE != kDtypeQ4_0;
    extern __shared__ __align__(16) unsigned char smem[];
    const uint32_t n = (uint32_t)p.n, cols = n * PARTS;
    const Q4Shared<NT> sh(smem, shape, n, kSums ? kCols : 0);
    const Q4Place w(p, shape);
    Q4Stream<CODE> ahead(p, shape, w);
    Q4Block<CODE> blk[2] = {};
    if (shape.early) ahead.fill(blk);  // the previous kernel of the stream does not write the weights
    pdl_enter();
    if (!shape.early) ahead.fill(blk);

    // ---- the columns of x
    const uint32_t pieces = w.here * 32, all = n * pieces;
    auto hi_slot = [&](const Q4Piece& x) { return reinterpret_cast<uint4*>(sh.xs + x.token * shape.x_row + x.at * 16); };
    auto lo_slot = [&](const Q4Piece& x) { return reinterpret_cast<uint4*>(sh.xs + (n + x.token) * shape.x_row + x.at * 16); };
    // sum of a piece's group of 32: four adjacent lanes; it stands in the token's first column
    auto group_sum = [&](const Q4Piece& x, float sum) {
        if constexpr (kSums) {
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if ((x.at & 3u) == 0) {
                sh.table[(x.at >> 2) * kCols + x.token] = sum;
                if constexpr (PARTS == 2) sh.table[(x.at >> 2) * kCols + n + x.token] = 0.0f;
            }
        }
    };
    if (threadIdx.x < kQ4Tokens) {
        sh.up[threadIdx.x] = sh.up[kQ4Tokens + threadIdx.x] = 1.0f;
        sh.top[threadIdx.x] = 0;
    }
    if constexpr (kSums) {  // columns that nobody reads
        for (uint32_t i = threadIdx.x; i < w.here * 8 * (kCols - cols); i += kQ4MulThreads)
            sh.table[i / (kCols - cols) * kCols + cols + i % (kCols - cols)] = 0.0f;
    }
    if (PARTS == 2) __syncthreads();
    if (threadIdx.x < all) {
        Q4Piece at{threadIdx.x / pieces, threadIdx.x % pieces};
        for (uint32_t i = threadIdx.x; i < all; i += kQ4Batch * kQ4MulThreads) {
            uint4 v[kQ4Batch][PARTS];
            Q4Piece x = at;
#pragma unroll
            for (int u = 0; u < kQ4Batch; ++u) {
                load_piece<PARTS == 2>(p, shape.x_vec, (uint64_t)w.first * 256 + (uint64_t)x.at * 8, x.token,
                                       i + u * kQ4MulThreads < all, v[u]);
                x.next(pieces);
            }
#pragma unroll
            for (int u = 0; u < kQ4Batch; ++u) {
                if (i + u * kQ4MulThreads < all) {
                    *hi_slot(at) = v[u][0];
                    if constexpr (PARTS == 2) {  // binary32 as it is, where its two parts will stand
                        *lo_slot(at) = v[u][1];
                        const uint32_t b[8] = {v[u][0].x, v[u][0].y, v[u][0].z, v[u][0].w,
                                               v[u][1].x, v[u][1].y, v[u][1].z, v[u][1].w};
                        const uint32_t big = __reduce_max_sync(0xffffffffu, largest_of(b));
                        if (w.lane == 0) atomicMax(sh.top + at.token, big);
                    } else {
                        const uint32_t b[4] = {v[u][0].x, v[u][0].y, v[u][0].z, v[u][0].w};
                        float sum = 0.0f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = __half22float2(bits_h2(b[e]));
                            sum += f.x + f.y;
                        }
                        group_sum(at, sum);
                    }
                }
                at.next(pieces);
            }
        }
    }
    __syncthreads();
    if (PARTS == 2) {
        uint32_t special = 0;  // tokens with an infinity or a NaN: their largest finite value is found anew
        for (uint32_t i = 0; i < n; ++i) special |= (uint32_t)(sh.top[i] >= kInfinity) << i;
        if (special) {
            __syncthreads();
            if (threadIdx.x < n && ((special >> threadIdx.x) & 1u)) sh.top[threadIdx.x] = 0;
            __syncthreads();
            if (threadIdx.x < all) {
                Q4Piece x{threadIdx.x / pieces, threadIdx.x % pieces};
                for (uint32_t i = threadIdx.x; i < all; i += kQ4MulThreads, x.next(pieces)) {
                    if (!((special >> x.token) & 1u)) continue;
                    const uint4 a = *hi_slot(x), b = *lo_slot(x);
                    const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                    for (int e = 0; e < 8; ++e)
                        if ((v[e] & 0x7fffffffu) < kInfinity) atomicMax(sh.top + x.token, v[e] & 0x7fffffffu);
                }
            }
            __syncthreads();
        }
        if (threadIdx.x < all) {
            Q4Piece x{threadIdx.x / pieces, threadIdx.x % pieces};
            for (uint32_t i = threadIdx.x; i < all; i += kQ4MulThreads) {
                const uint4 a = *hi_slot(x), b = *lo_slot(x);
                const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                // one step is enough: at 2^127 the parts' multiples of 2^-24 are finer than binary32's of 2^-149
                const uint32_t field = first_step(scale_to(sh.top[x.token], 14));
                const float scale = power(field);
                if (x.at == 0) sh.up[x.token] = inverse_power(field);
                float sum = 0.0f;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float y = bitsf(v[2 * q]) * scale, z = bitsf(v[2 * q + 1]) * scale;
                    const __half2 h = __floats2half2_rn(y, z);
                    const float2 f = __half22float2(h);
                    float ry = y - f.x, rz = z - f.y;
                    if (special) {  // NaN for an infinity: the first part carries it alone
                        ry = fabsf(ry) < INFINITY ? ry : 0.0f;
                        rz = fabsf(rz) < INFINITY ? rz : 0.0f;
                    }
                    hi[q] = h2_bits(h);
                    lo[q] = h2_bits(__floats2half2_rn(ry, rz));
                    sum += y + z;
                }
                *hi_slot(x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *lo_slot(x) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                group_sum(x, sum);
                x.next(pieces);
            }
        }
        __syncthreads();
    }

    // lanes of unused columns read the first one: their results are not used
    const uint32_t g = w.lane >> 2, t = w.lane & 3u;
    const unsigned char* x_at[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c) x_at[c] = sh.xs + (8 * c + g < cols ? 8 * c + g : 0) * shape.x_row + t * 16;
    float total[NT][4];
    auto work = [&](Q4Block<CODE>& b, uint32_t kb) {
        const float* sums = sh.table + kb * 8 * kCols + 2 * t;
        const uint32_t x_kb = kb * 512;
        float own_a[4], own_c[4];
        b.s.own(own_a, own_c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a[2][2], c[2][2];
            b.s.of(w.lane, j, own_a, own_c, a, c);
            const uint32_t q[4] = {b.q[j].x, b.q[j].y, b.q[j].z, b.q[j].w};
#pragma unroll
            for (int G = 0; G < 2; ++G) {
                uint32_t f[4], f2[4];
                half_quants(q[2 * G], f);
                half_quants(q[2 * G + 1], f2);
#pragma unroll
                for (int m = 0; m < NT; ++m) {
                    const uint4 x = *reinterpret_cast<const uint4*>(x_at[m] + x_kb + (j * 2 + G) * 64);
                    float acc[4];
                    mma_half(acc, f, x.x, x.y);
                    mma_half_add(acc, f2, x.z, x.w);
                    add_scaled(total[m], a[0][G], a[1][G], acc[0], acc[1], acc[2], acc[3]);
                    if constexpr (kSums) {
                        const float2 s = *reinterpret_cast<const float2*>(sums + (j * 2 + G) * kCols + 8 * m);
                        add_scaled(total[m], c[0][G], c[1][G], s.x, s.y, s.x, s.y);
                    }
                }
            }
            ahead.fetch_quads(b, j);
        }
        ahead.fetch_scales(b);
        ahead.next();
    };
    q4_rounds<CODE, PARTS, NT>(p, shape, w, blk, total, sh.red, sh.part, sh.up, 1.0f, work);
}

// One or two tokens of binary32 or binary16 as four digits each.
//
// Shared memory of a column: 16 bytes for each lane t of a 64-column block, of
// group 0 the digits of columns 8 t + (0, 2, 1, 3, 4, 6, 5, 7), then of group 1:
// the order in which the masks leave a word's quants.  The table holds for each
// 64-column block and t: of group 0 and 1, columns 2 t and 2 t + 1, what is added to
// the products; Q4_1 and Q4_K: then sum(x), in units of the
// highest digit, under the token's highest digit.
template <int CODE, bool F32>
__global__ void __launch_bounds__(kQ4MulThreads, 1) q4_digits_kernel(const Q4MatvecPlan p, const Q4Shape shape) {
    constexpr bool kSums = CODE != kDtypeQ4_0;
    constexpr uint32_t kTable = kSums ? 16 : 8;   // floats of a group
    constexpr float kBase = 12582912.0f;          // 1.5 2^23
    extern __shared__ __align__(16) unsigned char smem[];
    const uint32_t n = (uint32_t)p.n, cols = n * 4;
    const Q4Shared<1> sh(smem, shape, n, kTable);
    const Q4Place w(p, shape);
    Q4Stream<CODE> ahead(p, shape, w);
    Q4Block<CODE> blk[2] = {};
    if (shape.early) ahead.fill(blk);  // the previous kernel of the stream does not write the weights
    pdl_enter();
    if (!shape.early) ahead.fill(blk);

    // ---- the digits of x
    const uint32_t pieces = w.here * 32, all = n * pieces;
    // digit i of a piece; the columns stand digit by digit, as parts
    auto slot = [&](const Q4Piece& x, uint32_t i) {
        return reinterpret_cast<uint2*>(sh.xs + (i * n + x.token) * shape.x_row + (x.at >> 3) * 64 + (x.at & 3u) * 16 + ((x.at >> 2) & 1u) * 8);
    };
    // entry of (group, column) in the table
    auto entry = [&](uint32_t group, uint32_t col) -> float& {
        return sh.table[(group >> 1) * 2 * kTable + (col >> 1) * (kSums ? 8 : 4) + (group & 1u) * 2 + (col & 1u)];
    };
    if (threadIdx.x < kQ4Tokens) {
        sh.up[threadIdx.x] = sh.up[kQ4Tokens + threadIdx.x] = 1.0f;
        sh.top[threadIdx.x] = 0;
    }
    for (uint32_t i = threadIdx.x; i < w.here * 8 * (8 - cols); i += kQ4MulThreads) {  // columns that nobody reads
        float& e = entry(i / (8 - cols), cols + i % (8 - cols));
        e = -kBase;
        if constexpr (kSums) (&e)[4] = 0.0f;
    }
    __syncthreads();
    if (threadIdx.x < all) {
        Q4Piece at{threadIdx.x / pieces, threadIdx.x % pieces};
        for (uint32_t i = threadIdx.x; i < all; i += kQ4DigitBatch * kQ4MulThreads) {
            uint4 v[kQ4DigitBatch][F32 ? 2 : 1];
            Q4Piece x = at;
#pragma unroll
            for (int u = 0; u < kQ4DigitBatch; ++u) {
                load_piece<F32>(p, shape.x_vec, (uint64_t)w.first * 256 + (uint64_t)x.at * 8, x.token,
                                i + u * kQ4MulThreads < all, v[u]);
                x.next(pieces);
            }
#pragma unroll
            for (int u = 0; u < kQ4DigitBatch; ++u) {
                if (i + u * kQ4MulThreads < all) {
                    uint32_t b[8];
                    if constexpr (F32) {
                        b[0] = v[u][0].x, b[1] = v[u][0].y, b[2] = v[u][0].z, b[3] = v[u][0].w;
                        b[4] = v[u][F32].x, b[5] = v[u][F32].y, b[6] = v[u][F32].z, b[7] = v[u][F32].w;
                    } else {
                        const uint32_t h[4] = {v[u][0].x, v[u][0].y, v[u][0].z, v[u][0].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = __half22float2(bits_h2(h[e]));
                            b[2 * e] = fbits(f.x);
                            b[2 * e + 1] = fbits(f.y);
                        }
                    }
                    // binary32 as it is, where its digits will stand
#pragma unroll
                    for (int e = 0; e < 4; ++e) *slot(at, e) = make_uint2(b[2 * e], b[2 * e + 1]);
                    const uint32_t big = __reduce_max_sync(0xffffffffu, largest_of(b));
                    if (w.lane == 0) atomicMax(sh.top + at.token, big);
                }
                at.next(pieces);
            }
        }
    }
    __syncthreads();
    if (threadIdx.x < all) {
        Q4Piece x{threadIdx.x / pieces, threadIdx.x % pieces};
        for (uint32_t i = threadIdx.x; i < all; i += kQ4MulThreads) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint2 b = *slot(x, e);
                y[2 * e] = bitsf(b.x);
                y[2 * e + 1] = bitsf(b.y);
            }
            const uint32_t largest = sh.top[x.token], field = largest >= kInfinity ? 127u : scale_to(largest, 29);
            const float scale = power(first_step(field)), rest = power(rest_step(field));
            uint32_t d[8];
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float z = y[e] * scale;
                if constexpr (F32) z *= rest;  // binary16 columns never need it
                const int X = __float2int_rn(z);
                if constexpr (kSums) sum += (float)X;
                d[e] = ((uint32_t)X + 0x00808080u) ^ 0x00808080u;  // four balanced digits
            }
            // an infinity or NaN takes the whole column
            if (x.at == 0) {
                sh.up[x.token] = largest >= kInfinity ? bitsf(0x7fc00000u) : inverse_power(first_step(field));
                sh.up[kQ4Tokens + x.token] = inverse_power(rest_step(field));
            }
            // bytes i of the columns 0, 2, 1, 3 and 4, 6, 5, 7
            uint32_t digit[4][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t a = d[4 * h], b = d[4 * h + 2], c = d[4 * h + 1], e = d[4 * h + 3];
                const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab2 = __byte_perm(a, b, 0x7362);  // a0 b0 a1 b1, a2 b2 a3 b3
                const uint32_t ce0 = __byte_perm(c, e, 0x5140), ce2 = __byte_perm(c, e, 0x7362);
                digit[0][h] = __byte_perm(ab0, ce0, 0x5410);
                digit[1][h] = __byte_perm(ab0, ce0, 0x7632);
                digit[2][h] = __byte_perm(ab2, ce2, 0x5410);
                digit[3][h] = __byte_perm(ab2, ce2, 0x7632);
            }
            if constexpr (kSums) {
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                *slot(x, q) = make_uint2(digit[q][0], digit[q][1]);
                int s = __dp4a((int)digit[q][0], 0x01010101, __dp4a((int)digit[q][1], 0x01010101, 0));
                s += __shfl_xor_sync(0xffffffffu, s, 1);
                s += __shfl_xor_sync(0xffffffffu, s, 2);
                if ((x.at & 3u) == 0) {
                    float& e = entry(x.at >> 2, q * n + x.token);
                    e = -(kBase + (float)(8 * s));
                    if constexpr (kSums) (&e)[4] = q == 3 ? sum * (1.0f / 16777216.0f) : 0.0f;
                }
            }
            x.next(pieces);
        }
    }
    __syncthreads();

    const uint32_t g = w.lane >> 2, t = w.lane & 3u;
    // lanes of unused columns read the first one: their results are not used
    const unsigned char* x_at = sh.xs + (g < cols ? g : 0) * shape.x_row + t * 16;
    float total[1][4];
    auto work = [&](Q4Block<CODE>& b, uint32_t kb) {
        const float4* table = reinterpret_cast<const float4*>(sh.table + kb * 8 * kTable) + t * (kSums ? 2 : 1);
        const unsigned char* x_kb = x_at + kb * 256;
        float own_a[4], own_c[4];
        b.s.own(own_a, own_c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a[2][2], c[2][2];
            b.s.of(w.lane, j, own_a, own_c, a, c);
            const uint4 x = *reinterpret_cast<const uint4*>(x_kb + j * 64);
            const float4 base = table[j * (kSums ? 8 : 4)];
            const uint32_t q[4] = {b.q[j].x, b.q[j].y, b.q[j].z, b.q[j].w};
            constexpr uint32_t kMask = 0x0f0f0f0fu;
#pragma unroll
            for (int G = 0; G < 2; ++G) {
                uint32_t acc[4];
                mma_digits(acc, q[2 * G] & kMask, (q[2 * G] >> 4) & kMask, q[2 * G + 1] & kMask, (q[2 * G + 1] >> 4) & kMask,
                           G ? x.z : x.x, G ? x.w : x.y, 0x4b400000u);
                add_scaled(total[0], a[0][G], a[1][G], acc, G ? base.z : base.x, G ? base.w : base.y);
            }
            if constexpr (kSums) {
                const float4 s = table[j * 8 + 1];
                add_scaled(total[0], c[0][0], c[1][0], s.x, s.y, s.x, s.y);
                add_scaled(total[0], c[0][1], c[1][1], s.z, s.w, s.z, s.w);
            }
            ahead.fetch_quads(b, j);
        }
        ahead.fetch_scales(b);
        ahead.next();
    };
    q4_rounds<CODE, 4, 1>(p, shape, w, blk, total, sh.red, sh.part, sh.up, 256.0f, work);
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

bool q4_by_digits(const Q4MatvecPlan& p) { return p.n <= kQ4DigitTokens; }

uint64_t q4_shared_bytes(const Q4Shape& s, const Q4MatvecPlan& p) {
    const bool digits = q4_by_digits(p), sums = p.code != kDtypeQ4_0;
    const uint64_t parts = digits ? 4 : p.x_f16 ? 1 : 2, cols = (p.n * parts + 7) / 8 * 8;
    const uint64_t table = digits ? (sums ? 16 : 8) : sums ? cols : 0;
    return 2 * kQ4Warps * (16 * cols + kQ4RedPad) * 4 + (s.splits > 1 ? 2 * s.wr * 16 * p.n * 4 : 0) + kQ4Tokens * 12 +
           s.blocks * 8 * table * 4 + p.n * parts * s.x_row;
}

cudaError_t run_q4_kernel(void (*kernel)(Q4MatvecPlan, Q4Shape), DeviceFlags& ready, const LaunchEnv& env,
                          const Q4MatvecPlan& p, const Q4Shape& shape, uint64_t smem) {
    if (!ready.done(env.device)) {
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSharedMost);
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
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p, shape);
    if (err == cudaSuccess) ++*env.launches;
    return err;
}

// One launch: at most kQ4Tokens columns of x.
template <int CODE>
cudaError_t run_q4(const LaunchEnv& env, const Q4MatvecPlan& p, const Q4Shape& shape, uint64_t smem) {
    static DeviceFlags ready[5];
    if (q4_by_digits(p))
        return p.x_f16 ? run_q4_kernel(q4_digits_kernel<CODE, false>, ready[0], env, p, shape, smem)
                       : run_q4_kernel(q4_digits_kernel<CODE, true>, ready[1], env, p, shape, smem);
    if (p.x_f16) return run_q4_kernel(q4_halves_kernel<CODE, 1, 1>, ready[2], env, p, shape, smem);
    return 2 * p.n <= 8 ? run_q4_kernel(q4_halves_kernel<CODE, 2, 1>, ready[3], env, p, shape, smem)
                        : run_q4_kernel(q4_halves_kernel<CODE, 2, 2>, ready[4], env, p, shape, smem);
}

// How k and the rows are cut; false when the columns of x do not fit.
bool q4_shape(const LaunchEnv& env, const Q4MatvecPlan& p, Q4Shape* out, uint64_t* smem) {
    const uint64_t tiles = (p.rows + 15) / 16, k256 = (p.k + 255) / 256;
    for (uint32_t splits = 1; splits <= 8; splits *= 2) {
        Q4Shape s{};
        s.splits = splits;
        s.blocks = (uint32_t)((k256 + splits - 1) / splits);
        // 64 more than a multiple of 128: two columns' 16-byte pieces meet no bank twice
        s.x_row = s.blocks * (q4_by_digits(p) ? 256 : 512) + 64;
        const uint64_t groups = (uint64_t)env.sm_count / splits;
        // fewest blocks one after another in a warp; a round costs a barrier
        // and a join besides, about a quarter of a block's time
        uint64_t best = UINT64_MAX;
        for (uint32_t wk = 1; wk <= kQ4Warps; wk *= 2) {
            const uint32_t wr = kQ4Warps / wk;
            const uint64_t rounds = (tiles + groups * wr - 1) / (groups * wr), serial = (s.blocks + wk - 1) / wk;
            const uint64_t cost = rounds * (4 * serial + 1);
            if (cost >= best) continue;
            best = cost;
            s.wk = wk;
            s.wr = wr;
            s.rounds = (uint32_t)rounds;
            s.groups = (uint32_t)((tiles + rounds * wr - 1) / (rounds * wr));
        }
        *smem = q4_shared_bytes(s, p);
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
        shape.x_vec = ((reinterpret_cast<uintptr_t>(p.x) | (p.n > 1 ? p.x_st : 0)) & 15u) == 0;
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
