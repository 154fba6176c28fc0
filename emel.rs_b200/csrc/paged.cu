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
//     s_t = scale q . k_t,  m = max s,  out = sum e^(s - m) v / sum e^(s - m)
//
// Every key and value is read once from HBM, and that is what bounds the
// kernel: 4 flops a cached element and head are far under the tensor rate.
//
// Work.  A unit is one key/value head of one sequence with up to HPU of the
// query heads that share it; its tokens form tiles of 64.  All tiles of all
// units, in order, are cut into equal runs, one for each CTA, so a batch of
// any mixture of lengths loads every SM alike; a unit cut between CTAs leaves
// its pieces (m, l, o) in the workspace, and the CTA that finishes last (one
// ticket per cut unit) joins them in the order of the tiles, so the same
// inputs give the same bits.  The runs follow from the lengths on the device: no host
// knows them.
//
// Tile.  A warp takes 16 of a tile's tokens on its own: a ring of STAGES
// cp.async stages (16-byte chunks, rows padded by 16 bytes so that ldmatrix
// meets no bank twice) runs ahead across the ends of units, without a block
// barrier.  Rows outside [first, length) and the columns d .. DP are filled with zeros,
// so what lies there never meets an operand.
//
// Products on m16n8k16: S[head, token] = Q K^T, whose result fragments are
// the operand fragments of O[head, d] += P V.  Sixteen heads of a 16-bit
// query fill the 16 rows.  A binary32 query keeps its precision by parts
// instead: 8 heads, rows 0..7 the parts of highest weight, rows 8..15 the
// next ones -- binary16 caches: 2 parts of 11 bits, of the query divided by
// the power of two that brings its largest element into [1, 2), and of the
// weights; bfloat16 caches: 3 parts of 8 bits, the last one in a second
// operand.  The tensor pipe has room for that: the added products cost nothing
// in time.
constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kAttnSub = 16;                       // tokens of a warp's subtile
constexpr int kAttnTile = kAttnSub * kAttnWarps;   // tokens of a tile
constexpr float kLog2e = 1.4426950408889634f;
// Weights are held as 2^(s - m) with m 8 below the largest s (in units of
// log 2): binary16 keeps full precision down to 2^-22 of the largest weight
// instead of 2^-14.
constexpr float kWeightShift = 8.0f;

template <int DP>
struct AttnShape {
    static constexpr int kRow = DP * 2 + 16;                    // bytes of a staged row
    static constexpr int kStage = 2 * kAttnSub * kRow;          // K and V of a subtile
    // stages and CTAs per SM that fill shared memory: 2 CTAs up to 128
    // columns, one above
    static constexpr int kStages = DP == 64 ? 6 : DP == 96 ? 4 : DP == 128 ? 3 : DP == 192 ? 4 : 3;
    static constexpr int kCtas = DP <= 128 ? 2 : 1;
};

__device__ __forceinline__ uint32_t shared_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldsm2(uint32_t& r0, uint32_t& r1, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(at) : "memory");
}

template <typename C>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (std::is_same_v<C, __half>) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename C>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (std::is_same_v<C, __half>) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// What is left of x after its 16-bit rounding (0 for what is not finite: the
// first part carries it alone).
template <typename C>
__device__ __forceinline__ float rest_of(float x) {
    const float r = x - to_f32(from_f32<C>(x));
    return fabsf(r) < INFINITY ? r : 0.0f;
}

// A position in the order of all tiles.
struct TileAt {
    int64_t b;       // sequence
    uint32_t unit;   // key/value head and block of query heads
    int64_t tile;
    int64_t first, len, tiles;  // of sequence b
};

template <typename C, int PARTS, int DP>
__global__ void __launch_bounds__(kAttnThreads, AttnShape<DP>::kCtas) paged_attn_kernel(const PagedAttnPlan p) {
    using Shape = AttnShape<DP>;
    using Q = std::conditional_t<PARTS == 1, C, float>;
    constexpr int HPU = PARTS == 1 ? 16 : 8;
    constexpr int kRow = Shape::kRow, kStages = Shape::kStages;
    constexpr int kSlot = HPU * DP * 4 + HPU * 8;  // a warp's (o, m, l) in one of its own stages
    static_assert(kSlot <= Shape::kStage, "the pieces of a segment lie in one stage");
    extern __shared__ __align__(16) unsigned char smem[];
    unsigned char* q_tile = smem + kAttnWarps * kStages * Shape::kStage;
    constexpr int kQBytes = 16 * kRow * (PARTS == 3 ? 2 : 1);
    float* q_scale = reinterpret_cast<float*>(q_tile + kQBytes);           // [16]
    uint32_t* masks = reinterpret_cast<uint32_t*>(q_scale + 16);           // [warp][stage]
    int64_t* shared64 = reinterpret_cast<int64_t*>(masks + kAttnWarps * 8);  // [8]
    pdl_enter();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t g = lane >> 2, t4 = lane & 3;
    const uint32_t blocks = (uint32_t)((p.rep + HPU - 1) / HPU);
    const uint32_t units = (uint32_t)(p.heads / p.rep) * blocks;
    const int64_t cap = (int64_t)(p.table_pages * p.page_size);
    const int64_t batch = (int64_t)p.batch;

    auto span = [&](int64_t b, int64_t& first, int64_t& len) -> int64_t {  // tiles of sequence b
        len = p.lengths[b * p.len_st];
        len = len < 0 ? 0 : len > cap ? cap : len;
        first = p.window && len > (int64_t)p.window ? len - (int64_t)p.window : 0;
        return (len - first + kAttnTile - 1) / kAttnTile;
    };

    // ---- this CTA's run of tiles: the total first, then the place of its start
    int64_t mine = 0, first_tiles = 0;
    for (int64_t b = threadIdx.x; b < batch; b += kAttnThreads) {
        int64_t f, n;
        const int64_t tiles = span(b, f, n);
        if (b < kAttnThreads) first_tiles = tiles;
        mine += tiles;
        if (blockIdx.x == 0) {
            const int64_t raw = p.lengths[b * p.len_st];
            if (raw < 0 || raw > cap) atomicExch(p.reject, p.reject_code);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) shared64[warp] = mine;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) total += shared64[w];
    total *= units;
    int64_t run = (total + gridDim.x - 1) / gridDim.x;
    if (run < (int64_t)p.min_run) run = (int64_t)p.min_run;
    const int64_t start = run * blockIdx.x;
    const int64_t stop = start + run < total ? start + run : total;

    // sequences without tokens: zeros, spread over the CTAs
    for (int64_t b = blockIdx.x; b < batch; b += gridDim.x) {
        int64_t f, n;
        if (span(b, f, n) != 0) continue;
        for (uint64_t i = threadIdx.x; i < p.heads * p.d; i += kAttnThreads)
            reinterpret_cast<Q*>(p.dst + (i / p.d) * p.dst_st[1] + b * p.dst_st[2])[i % p.d] = from_f32<Q>(0.0f);
    }
    if (start >= stop) return;

    if (start == 0) {
        if (threadIdx.x == 0) {
            shared64[4] = 0;
            shared64[5] = 0;
        }
    } else {
        int64_t before = 0;
        __syncthreads();
        for (int64_t base = 0; base < batch; base += kAttnThreads) {
            const int64_t b = base + threadIdx.x;
            int64_t f, n;
            const int64_t tiles = b >= batch ? 0 : base == 0 ? first_tiles : span(b, f, n);
            int64_t sum = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            if (lane == 31) shared64[warp] = sum;
            __syncthreads();
            int64_t all = 0;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) {
                if (w < warp) sum += shared64[w];
                all += shared64[w];
            }
            const int64_t at = (before + sum - tiles) * units;  // first tile of sequence b
            if (tiles > 0 && at <= start && start < at + tiles * units) {
                shared64[4] = b;
                shared64[5] = start - at;
            }
            before += all;
            __syncthreads();
            if (start < before * units) break;
        }
    }
    __syncthreads();
    TileAt to;  // the next subtile to compute
    to.b = shared64[4];
    to.tiles = span(to.b, to.first, to.len);
    while (to.tiles == 0) to.tiles = span(++to.b, to.first, to.len);  // start == 0 only
    {
        const int64_t off = shared64[5];
        to.unit = (uint32_t)(off / to.tiles);
        to.tile = off % to.tiles;
    }
    auto advance = [&](TileAt& x) {
        if (++x.tile < x.tiles) return;
        x.tile = 0;
        if (++x.unit < units) return;
        x.unit = 0;
        do {
            if (++x.b >= batch) return;  // past the last tile: never used
            x.tiles = span(x.b, x.first, x.len);
        } while (x.tiles == 0);
    };

    // ---- the ring
    const uint32_t ring = shared_u32(smem) + warp * kStages * Shape::kStage;
    uint32_t* my_masks = masks + warp * 8;
    // the page of the token that this lane stands for (lanes 16.. repeat 0..15), -2: none
    auto page_of = [&](const TileAt& x) -> int32_t {
        const int64_t t = x.first + x.tile * kAttnTile + warp * kAttnSub + (lane & 15);
        if (t >= x.len) return -2;
        return p.table[(int64_t)((uint32_t)t / (uint32_t)p.page_size) * p.table_st[0] + x.b * p.table_st[1]];
    };
    auto issue = [&](const TileAt& x, int32_t page, int stage) {
        const int64_t t = x.first + x.tile * kAttnTile + warp * kAttnSub + (lane & 15);
        const bool in = page >= 0 && (uint64_t)page < p.pages;
        if (!in && page != -2) atomicExch(p.reject, p.reject_code);
        const uint32_t mask = __ballot_sync(0xffffffffu, in) & 0xffffu;
        if (lane == 0) my_masks[stage] = mask;
        const uint64_t off = in ? (uint32_t)t % (uint32_t)p.page_size : 0;
        const uint64_t pg = in ? (uint64_t)page : 0;
        const uint64_t h = x.unit / blocks;
        const uint64_t ko = pg * p.k_st[3] + off * p.k_st[2], vo = pg * p.v_st[3] + off * p.v_st[2];
        const char* kb = p.k + h * p.k_st[1];
        const char* vb = p.v + h * p.v_st[1];
        const uint32_t dst = ring + stage * Shape::kStage;
        if (p.vec) {
            constexpr int kChunks = DP / 8;
#pragma unroll
            for (int i = 0; i < kAttnSub * kChunks / 32; ++i) {
                const uint32_t c = lane + 32 * i, row = c / kChunks, col = c % kChunks;
                const uint64_t kr = __shfl_sync(0xffffffffu, ko, row), vr = __shfl_sync(0xffffffffu, vo, row);
                const bool use = ((mask >> row) & 1u) && col * 8 < p.d;
                cp16(dst + row * kRow + col * 16, use ? kb + kr + col * 16 : p.k, use);
                cp16(dst + kAttnSub * kRow + row * kRow + col * 16, use ? vb + vr + col * 16 : p.v, use);
            }
        } else {
            unsigned char* out = smem + (dst - shared_u32(smem));
            for (uint32_t row = 0; row < kAttnSub; ++row) {
                const uint64_t kr = __shfl_sync(0xffffffffu, ko, row), vr = __shfl_sync(0xffffffffu, vo, row);
                const bool use = (mask >> row) & 1u;
                for (uint32_t col = lane; col < DP; col += 32) {
                    uint16_t kx = 0, vx = 0;
                    if (use && col < p.d) {
                        kx = reinterpret_cast<const uint16_t*>(kb + kr)[col];
                        vx = reinterpret_cast<const uint16_t*>(vb + vr)[col];
                    }
                    *reinterpret_cast<uint16_t*>(out + row * kRow + col * 2) = kx;
                    *reinterpret_cast<uint16_t*>(out + (kAttnSub + row) * kRow + col * 2) = vx;
                }
            }
        }
    };

    const int64_t count = stop - start;
    TileAt ahead = to;
    int64_t left = count;  // subtiles not issued yet
    int into = 0;          // the stage that takes the next one
    int32_t page = page_of(ahead);
    auto issue_next = [&]() {
        if (left > 0) {
            issue(ahead, page, into);
            if (--left > 0) {
                advance(ahead);
                page = page_of(ahead);  // in flight until the next call
            }
        }
        into = into + 1 == kStages ? 0 : into + 1;
        cp_commit();
    };
#pragma unroll 1
    for (int s = 0; s < kStages - 1; ++s) issue_next();

    // ldmatrix addresses of this lane
    const uint32_t k_at = ((lane >> 4) * 8 + (lane & 7)) * kRow + ((lane >> 3) & 1) * 16;
    const uint32_t v_at = (((lane >> 3) & 1) * 8 + (lane & 7)) * kRow + (lane >> 4) * 16 + kAttnSub * kRow;
    const uint32_t q_at = shared_u32(q_tile) + (((lane >> 3) & 1) * 8 + (lane & 7)) * kRow + (lane >> 4) * 16;
    const uint32_t q2_at = shared_u32(q_tile) + 16 * kRow + (lane & 7) * kRow + ((lane >> 3) & 1) * 16;

    constexpr int kHeadsLane = PARTS == 1 ? 2 : 1;  // heads of a lane's result rows: g (and g + 8)
    float o[DP / 8][4];
    float m[kHeadsLane], l[kHeadsLane], sc[kHeadsLane];
    bool fresh = true;  // a new segment begins
    int stage = kStages - 1;
    int64_t seg_start = start;

#pragma unroll 1
    for (int64_t i = 0; i < count; ++i) {
        stage = stage + 1 == kStages ? 0 : stage + 1;
        if (fresh) {
            fresh = false;
            // the unit's query rows, in parts; every warp shares them
            const uint64_t h0 = (uint64_t)(to.unit / blocks) * p.rep + (uint64_t)(to.unit % blocks) * HPU;
            const uint32_t nh = (uint32_t)(p.rep - (to.unit % blocks) * HPU < HPU ? p.rep - (to.unit % blocks) * HPU : HPU);
            for (uint32_t r = warp; r < HPU; r += kAttnWarps) {
                const Q* row = reinterpret_cast<const Q*>(p.q + (h0 + r) * p.q_st[1] + to.b * p.q_st[2]);
                float x[DP / 32];
                float big = 0.0f;
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) {
                    const uint32_t col = lane + 32 * c;
                    x[c] = r < nh && col < p.d ? to_f32(row[col]) : 0.0f;
                    big = fmaxf(big, fabsf(x[c]));
                }
                float up = 1.0f, down = 1.0f;
                if constexpr (PARTS == 2) {
#pragma unroll
                    for (int s = 16; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
                    const int e = (int)((fbits(big) >> 23) & 255u) - 127;
                    if (big < INFINITY && e >= -126) {
                        down = bitsf((uint32_t)(e < 127 ? 127 - e : 1) << 23);
                        up = 1.0f / down;
                    }
                }
                if (lane == 0) q_scale[r] = p.scale * kLog2e * up;
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) {
                    const uint32_t col = lane + 32 * c;
                    const float y = x[c] * down;
                    *reinterpret_cast<C*>(q_tile + r * kRow + col * 2) = from_f32<C>(y);
                    if constexpr (PARTS >= 2) {
                        const float rest = rest_of<C>(y);
                        *reinterpret_cast<C*>(q_tile + (8 + r) * kRow + col * 2) = from_f32<C>(rest);
                        if constexpr (PARTS == 3)
                            *reinterpret_cast<C*>(q_tile + (16 + r) * kRow + col * 2) = from_f32<C>(rest_of<C>(rest));
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int h = 0; h < kHeadsLane; ++h) {
                m[h] = -INFINITY;
                l[h] = 0.0f;
                sc[h] = q_scale[g + 8 * h];
            }
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        }
        cp_wait<kStages - 2>();
        __syncwarp();
        const uint32_t mask = my_masks[stage];
        issue_next();  // into the stage that the previous iteration has read
        const uint32_t base = ring + stage * Shape::kStage;
        if (mask) {
            float s[2][4] = {}, s3[PARTS == 3 ? 2 : 1][4] = {};  // s3: the last parts, apart
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                uint32_t a[4], b[4];
                ldsm4(a, q_at + k * 32);
                ldsm4(b, base + k_at + k * 32);
                mma16816<C>(s[0], a[0], a[1], a[2], a[3], b[0], b[1]);
                mma16816<C>(s[1], a[0], a[1], a[2], a[3], b[2], b[3]);
                if constexpr (PARTS == 3) {
                    uint32_t a0, a2;
                    ldsm2(a0, a2, q2_at + k * 32);
                    mma16816<C>(s3[0], a0, 0u, a2, 0u, b[0], b[1]);
                    mma16816<C>(s3[PARTS == 3 ? 1 : 0], a0, 0u, a2, 0u, b[2], b[3]);
                }
            }
            // weights of this lane's tokens 2 t4, 2 t4 + 1 (n = 0) and 8 + those (n = 1)
            float w[kHeadsLane][4], keep[kHeadsLane];
            bool moved = false;
#pragma unroll
            for (int h = 0; h < kHeadsLane; ++h) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = s[n][2 * h + e];
                        if constexpr (PARTS >= 2) {
                            // an infinite key: the first part has its sign, a part of 0 would make it NaN
                            const float more = PARTS == 3 ? s[n][2 + e] + s3[PARTS == 3 ? n : 0][e] : s[n][2 + e];
                            x = fabsf(x) < INFINITY ? x + more : x;
                        }
                        w[h][2 * n + e] = (mask >> (8 * n + 2 * t4 + e)) & 1u ? x : -INFINITY;
                        top = fmaxf(top, w[h][2 * n + e]);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(m[h], __fmaf_rn(top, sc[h], -kWeightShift));
                const float ref = top == -INFINITY ? 0.0f : top;  // only -inf so far: every weight is 0
                keep[h] = m[h] == top ? 1.0f : ex2(m[h] - ref);
                moved = moved || keep[h] != 1.0f;
                m[h] = top;
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[h][e] = ex2(__fmaf_rn(w[h][e], sc[h], -ref));
                    sum += w[h][e];
                }
                l[h] = __fmaf_rn(l[h], keep[h], sum);
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) {
                    o[n][0] *= keep[0];
                    o[n][1] *= keep[0];
                    o[n][2] *= keep[kHeadsLane - 1];
                    o[n][3] *= keep[kHeadsLane - 1];
                }
            }
            uint32_t a0, a1, a2, a3, c0 = 0, c2 = 0;
            a0 = pack2<C>(w[0][0], w[0][1]);
            a2 = pack2<C>(w[0][2], w[0][3]);
            if constexpr (PARTS == 1) {
                a1 = pack2<C>(w[1][0], w[1][1]);
                a3 = pack2<C>(w[1][2], w[1][3]);
            } else {
                float r[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = rest_of<C>(w[0][e]);
                a1 = pack2<C>(r[0], r[1]);
                a3 = pack2<C>(r[2], r[3]);
                if constexpr (PARTS == 3) {
                    c0 = pack2<C>(rest_of<C>(r[0]), rest_of<C>(r[1]));
                    c2 = pack2<C>(rest_of<C>(r[2]), rest_of<C>(r[3]));
                }
            }
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                uint32_t b[4];
                ldsm4_t(b, base + v_at + n * 32);
                mma16816<C>(o[2 * n], a0, a1, a2, a3, b[0], b[1]);
                mma16816<C>(o[2 * n + 1], a0, a1, a2, a3, b[2], b[3]);
                if constexpr (PARTS == 3) {
                    mma16816<C>(o[2 * n], c0, 0u, c2, 0u, b[0], b[1]);
                    mma16816<C>(o[2 * n + 1], c0, 0u, c2, 0u, b[2], b[3]);
                }
            }
        }
        const bool unit_ends = to.tile + 1 == to.tiles;
        if (!unit_ends && i + 1 < count) {
            ++to.tile;
            continue;
        }

        // ---- the end of a segment: the warps' pieces join
        __syncwarp();
        float* piece = reinterpret_cast<float*>(smem + (warp * kStages + stage) * Shape::kStage);
#pragma unroll
        for (int h = 0; h < kHeadsLane; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if (t4 == 0) {
                piece[HPU * DP + g + 8 * h] = m[h];
                piece[HPU * DP + HPU + g + 8 * h] = l[h];
            }
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
            float* at = piece + g * DP + n * 8 + 2 * t4;
            if constexpr (PARTS == 1) {
                *reinterpret_cast<float2*>(at) = make_float2(o[n][0], o[n][1]);
                *reinterpret_cast<float2*>(at + 8 * DP) = make_float2(o[n][2], o[n][3]);
            } else {
                *reinterpret_cast<float2*>(at) = make_float2(o[n][0] + o[n][2], o[n][1] + o[n][3]);
            }
        }
        __syncthreads();
        const uint64_t h0 = (uint64_t)(to.unit / blocks) * p.rep + (uint64_t)(to.unit % blocks) * HPU;
        const uint32_t nh = (uint32_t)(p.rep - (to.unit % blocks) * HPU < HPU ? p.rep - (to.unit % blocks) * HPU : HPU);
        const int64_t unit_first = start + i - to.tile, unit_last = unit_first + to.tiles - 1;  // its tiles in the order
        const bool whole = seg_start == unit_first && unit_ends;
        const uint32_t d = (uint32_t)p.d;
        const uint64_t slot_floats = (uint64_t)HPU * (d + 2);
        float* slot = p.pieces + ((uint64_t)blockIdx.x * 2 + (seg_start == start ? 0 : 1)) * slot_floats;
        auto warp_piece = [&](int w) { return reinterpret_cast<const float*>(smem + (w * kStages + stage) * Shape::kStage); };
        for (uint32_t e = threadIdx.x; e < nh * d; e += kAttnThreads) {
            const uint32_t r = e / d, c = e % d;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, warp_piece(w)[HPU * DP + r]);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f, x = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) {
                const float f = ex2(warp_piece(w)[HPU * DP + r] - ref);
                sum = __fmaf_rn(f, warp_piece(w)[HPU * DP + HPU + r], sum);
                x = __fmaf_rn(f, warp_piece(w)[r * DP + c], x);
            }
            if (whole) {
                reinterpret_cast<Q*>(p.dst + (h0 + r) * p.dst_st[1] + to.b * p.dst_st[2])[c] =
                    from_f32<Q>(sum == 0.0f ? 0.0f : x / sum);
            } else {
                __stcg(slot + r * d + c, x);
                if (c == 0) {
                    __stcg(slot + HPU * d + r, top);
                    __stcg(slot + HPU * d + HPU + r, sum);
                }
            }
        }
        if (!whole) {
            const int64_t c0 = unit_first / run, c1 = unit_last / run;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                const unsigned before = atomicAdd(p.tickets + c0, 1u);
                shared64[6] = before == (unsigned)(c1 - c0);
            }
            __syncthreads();
            if (shared64[6]) {
                __threadfence();
                const int64_t n = c1 - c0 + 1;
                const float* first_slot = p.pieces + ((uint64_t)c0 * 2 + (c0 * run == unit_first ? 0 : 1)) * slot_floats;
                auto slot_of = [&](int64_t k) {
                    return k == 0 ? first_slot : p.pieces + (uint64_t)(c0 + k) * 2 * slot_floats;
                };
                for (uint32_t e = threadIdx.x; e < nh * d; e += kAttnThreads) {
                    const uint32_t r = e / d, c = e % d;
                    float top = -INFINITY;
#pragma unroll 4
                    for (int64_t k = 0; k < n; ++k) top = fmaxf(top, __ldcg(slot_of(k) + HPU * d + r));
                    const float ref = top == -INFINITY ? 0.0f : top;
                    float sum = 0.0f, x = 0.0f;
#pragma unroll 4
                    for (int64_t k = 0; k < n; ++k) {
                        const float* s = slot_of(k);
                        const float f = ex2(__ldcg(s + HPU * d + r) - ref);
                        sum = __fmaf_rn(f, __ldcg(s + HPU * d + HPU + r), sum);
                        x = __fmaf_rn(f, __ldcg(s + r * d + c), x);
                    }
                    reinterpret_cast<Q*>(p.dst + (h0 + r) * p.dst_st[1] + to.b * p.dst_st[2])[c] =
                        from_f32<Q>(sum == 0.0f ? 0.0f : x / sum);
                }
                if (threadIdx.x == 0) p.tickets[c0] = 0;
            }
        }
        __syncthreads();  // the pieces and the query rows may be overwritten
        if (i + 1 < count) advance(to);
        seg_start = start + i + 1;
        fresh = true;
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

template <typename C, int PARTS, int DP>
cudaError_t run_attn_at(const LaunchEnv& env, PagedAttnPlan p) {
    using Shape = AttnShape<DP>;
    constexpr int HPU = PARTS == 1 ? 16 : 8;
    constexpr int kSmem = kAttnWarps * Shape::kStages * Shape::kStage + 16 * Shape::kRow * (PARTS == 3 ? 2 : 1) + 64 +
                          kAttnWarps * 8 * 4 + 64;
    static DeviceFlags ready;
    if (!ready.done(env.device)) {
        const cudaError_t err = cudaFuncSetAttribute(paged_attn_kernel<C, PARTS, DP>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (err != cudaSuccess) return err;
        ready.mark(env.device);
    }
    // one wave, no more CTAs than there are tiles at most or slots for pieces
    const uint64_t slot = (uint64_t)HPU * (p.d + 2) * 4 * 2;
    uint64_t grid = (uint64_t)env.sm_count * Shape::kCtas;
    const uint64_t slots = paged_piece_bytes(env.sm_count) / slot, tickets = paged_tickets(env.sm_count);
    if (grid > slots) grid = slots;
    if (grid > tickets) grid = tickets;
    const unsigned __int128 most = (unsigned __int128)((p.table_pages * p.page_size + kAttnTile - 1) / kAttnTile) *
                                   p.batch * (p.heads / p.rep) * ((p.rep + HPU - 1) / HPU);
    if (most < grid) grid = (uint64_t)most;
    p.min_run = 1;
    const cudaError_t err = launch_dependent(paged_attn_kernel<C, PARTS, DP>, dim3((unsigned)grid), dim3(kAttnThreads),
                                             kSmem, env.stream, p);
    if (err == cudaSuccess) ++*env.launches;
    return err;
}

template <typename C, int PARTS>
cudaError_t run_attn(const LaunchEnv& env, const PagedAttnPlan& p) {
    if (p.d <= 64) return run_attn_at<C, PARTS, 64>(env, p);
    if (p.d <= 96) return run_attn_at<C, PARTS, 96>(env, p);
    if (p.d <= 128) return run_attn_at<C, PARTS, 128>(env, p);
    if (p.d <= 192) return run_attn_at<C, PARTS, 192>(env, p);
    return run_attn_at<C, PARTS, 256>(env, p);
}

}  // namespace

cudaError_t launch_paged_append(const LaunchEnv& env, const PagedAppendPlan& p) {
    if (p.cache_bf16) {
        return p.src_f32 ? run_append<float, __nv_bfloat16>(env, p) : run_append<__nv_bfloat16, __nv_bfloat16>(env, p);
    }
    return p.src_f32 ? run_append<float, __half>(env, p) : run_append<__half, __half>(env, p);
}

// Two pieces for each CTA of the widest shape (one CTA per SM, 16 heads of
// kPagedMaxD columns and their m and l), or for each of two CTAs per SM at
// half the columns.
uint64_t paged_piece_bytes(int sm_count) { return (uint64_t)sm_count * 2 * 16 * (kPagedMaxD + 4) * 4; }
uint64_t paged_tickets(int sm_count) { return (uint64_t)sm_count * 4; }

cudaError_t launch_paged_attn(const LaunchEnv& env, const PagedAttnPlan& p) {
    if (p.cache_bf16) return p.q_f32 ? run_attn<__nv_bfloat16, 3>(env, p) : run_attn<__nv_bfloat16, 1>(env, p);
    return p.q_f32 ? run_attn<__half, 2>(env, p) : run_attn<__half, 1>(env, p);
}

}  // namespace emel
