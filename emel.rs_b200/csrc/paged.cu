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
#include "tma.cuh"

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
//
// Bytes moved are all there is: every value is read and written once.

// The page of a position and the place in it; false: skipped or rejected.
__device__ __forceinline__ bool place_of(const PagedAppendPlan& p, int64_t pos, int64_t seq, uint64_t* page, uint64_t* off) {
    if (pos < 0) return false;
    const uint64_t at = (uint32_t)pos / (uint32_t)p.page_size;
    *off = (uint32_t)pos - (uint32_t)at * (uint32_t)p.page_size;
    int64_t pg = -1;
    if (seq >= 0 && (uint64_t)seq < p.sequences_count && at < p.table_pages)
        pg = p.table[(int64_t)at * p.table_st[0] + seq * p.table_st[1]];
    if (pg < 0 || (uint64_t)pg >= p.pages) {
        atomicExch(p.reject, p.reject_code);
        return false;
    }
    *page = (uint64_t)pg;
    return true;
}

template <typename S, typename C>
__device__ __forceinline__ C converted(S v) {
    if constexpr (std::is_same_v<S, C>) return v;  // bits unchanged
    else return from_f32<C>(to_f32(v));
}

// Eight values as one 16-byte store: from 16 bytes of the cache's type, or 32
// of binary32.
template <typename S, typename C>
struct AppendPiece {
    uint4 v[sizeof(S) == 4 ? 2 : 1];
    __device__ __forceinline__ void load(const char* p) {
#pragma unroll
        for (uint32_t i = 0; i < sizeof(v) / 16; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void store(char* p) const {
        if constexpr (std::is_same_v<S, C>) {
            *reinterpret_cast<uint4*>(p) = v[0];
        } else {
            const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const C lo = from_f32<C>(__uint_as_float(w[2 * i])), hi = from_f32<C>(__uint_as_float(w[2 * i + 1]));
                o[i] = *reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16;
            }
            *reinterpret_cast<uint4*>(p) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
};

// Rows of whole, aligned 16-byte pieces (p.vec).  A thread keeps its piece of a
// row and goes from row to row, kAppendRows of them in flight: two loads follow one
// another for each (position, page; the values come beside them).  8191 bfloat16 rows
// of 8 x 128 keys and values: 14.3 us, 4.7 TB/s (15.1 us with four rows in flight).
constexpr int kAppendRows = 2;
template <typename S, typename C>
__global__ void __launch_bounds__(kAppendThreads) append_rows_kernel(PagedAppendPlan p, uint32_t lanes) {
    pdl_enter();
    const uint32_t pieces = (uint32_t)p.d / 8, per = (uint32_t)p.kv_heads * pieces;
    const uint64_t step = (uint64_t)gridDim.x * (kAppendThreads / lanes);
    for (uint32_t x = threadIdx.x % lanes; x < per; x += lanes) {
        const uint32_t h = x / pieces, c = x - h * pieces;
        const char* ks = p.key + h * p.key_st[1] + c * 8 * sizeof(S);
        const char* vs = p.value + h * p.value_st[1] + c * 8 * sizeof(S);
        char* kd = p.k_cache + h * p.k_st[1] + c * 16;
        char* vd = p.v_cache + h * p.v_st[1] + c * 16;
        for (uint64_t n0 = (uint64_t)blockIdx.x * (kAppendThreads / lanes) + threadIdx.x / lanes; n0 < p.count; n0 += step * kAppendRows) {
            int32_t pos[kAppendRows], seq[kAppendRows];
            AppendPiece<S, C> k[kAppendRows], v[kAppendRows];
#pragma unroll
            for (int u = 0; u < kAppendRows; ++u) {
                const uint64_t n = n0 + u * step;
                if (n < p.count) {
                    pos[u] = p.positions[(int64_t)n * p.pos_st];
                    seq[u] = p.sequences ? p.sequences[(int64_t)n * p.seq_st] : (int32_t)n;
                    k[u].load(ks + n * p.key_st[2]);
                    v[u].load(vs + n * p.value_st[2]);
                }
            }
#pragma unroll
            for (int u = 0; u < kAppendRows; ++u) {
                const uint64_t n = n0 + u * step;
                uint64_t page, off;
                if (n < p.count && place_of(p, pos[u], seq[u], &page, &off)) {
                    k[u].store(kd + off * p.k_st[2] + page * p.k_st[3]);
                    v[u].store(vd + off * p.v_st[2] + page * p.v_st[3]);
                }
            }
        }
    }
}

// Anything else, value by value.
template <typename S, typename C>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(PagedAppendPlan p) {
    pdl_enter();
    const uint64_t per = p.d * p.kv_heads;
    const uint64_t total = p.count * per;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t n = i / per, h = i % per / p.d, c = i % p.d;
        uint64_t page, off;
        if (!place_of(p, p.positions[(int64_t)n * p.pos_st], p.sequences ? p.sequences[(int64_t)n * p.seq_st] : (int64_t)n, &page, &off))
            continue;
        const S* k = reinterpret_cast<const S*>(p.key + h * p.key_st[1] + n * p.key_st[2]);
        const S* v = reinterpret_cast<const S*>(p.value + h * p.value_st[1] + n * p.value_st[2]);
        reinterpret_cast<C*>(p.k_cache + h * p.k_st[1] + off * p.k_st[2] + page * p.k_st[3])[c] = converted<S, C>(k[c]);
        reinterpret_cast<C*>(p.v_cache + h * p.v_st[1] + off * p.v_st[2] + page * p.v_st[3])[c] = converted<S, C>(v[c]);
    }
}

// ---- attention ---------------------------------------------------------------
//
//     s_t = scale q . k_t,  m = max s,  out = sum e^(s - m) v / sum e^(s - m)
//
// Every key and value is read once from HBM for each unit, and that is what bounds
// the kernel: 4 flops a cached element and head are far under the tensor rate.
//
// Work.  A unit is one key/value head of one sequence with up to HPU (8 of binary32,
// 16 of 16 bits) of the query heads that share it; its tokens form tiles of 64.  More
// heads are more units, which read the same tiles again: 64 sequences of 8191 tokens
// over one head of 128, 269 MB, take 56 us with 8 binary32 query heads over binary16,
// 97 with 9, 180 with 32; in bfloat16 62 us with 16, 102 with 17.  All tiles of all
// units, in order, are cut into equal runs, one for each CTA, so a batch of
// any mixture of lengths loads every SM alike; a unit cut between CTAs leaves
// its pieces (m, l, o) in the workspace, and the CTA that finishes last (a
// ticket per cut unit) joins them in the order of the tiles, so the same
// inputs give the same bits.  Many pieces join in two steps of at most 8 and 37:
// one unit's 37 pieces by one CTA took 6 us of 37.  The runs follow from the lengths on the device: no host
// knows them.
//
// Bound by HBM once the lengths, the table and the rows have come one after another.
// 32 heads over 8 of 128: 64 sequences of up to 8191 tokens in bfloat16, 673 MB, 124 us,
// 5.4 TB/s; one of 32768 tokens, binary32 over binary16, 134 MB, 34.5 us, 3.9 TB/s
// (start and joins are latency).
//
// Tile.  Four warps take 16 of a tile's tokens each; two more find the rows
// and load them with cp.async (16-byte chunks, four or eight lanes a row), up to
// STAGES tiles ahead and across the ends of units; mbarriers say when a stage is
// there and when it is free, every wait is bounded.  With the computing warps finding
// their own rows that took 1 us a tile, more than the products; with one bulk copy for
// each row of 256 bytes the copy engine took 36 cycles a row, twice the time of all
// else.  Rows are padded by 16 bytes, so that ldmatrix meets no bank twice.  Tokens
// outside [first, length) or on rejected pages and the columns d .. DP are filled with
// zeros, so what lies there never meets an operand.  Rows that are not 16-byte
// aligned are loaded by the computing warps, element by element.
//
// Products on m16n8k16: S[head, token] = Q K^T, whose result fragments are
// the operand fragments of O[head, d] += P V.  Sixteen heads of a 16-bit
// query fill the 16 rows; their weights meet the values in two 16-bit parts (22 bits in
// binary16, 17 in bfloat16: the result is rounded to 11 or 8), one operand after the
// other.  A binary32 query keeps its precision by parts
// instead: 8 heads, rows 0..7 the parts of highest weight, rows 8..15 the
// next ones -- binary16 caches: 2 parts of 11 bits, of the query divided by
// the power of two that brings its largest finite element into [1, 2), and of the
// weights; bfloat16 caches: 3 parts of 8 bits, the last one in a second
// operand, of queries below 2^-40 brought up to that.  The tensor pipe has room for that: the added products cost nothing
// in time.
constexpr int kAttnWarps = 4;                      // that compute
constexpr int kAttnConsumers = kAttnWarps * 32;
constexpr int kAttnLoaders = 2;                    // that load: 32 rows of a tile each
constexpr int kAttnThreads = kAttnConsumers + 32 * kAttnLoaders;
constexpr int kAttnSub = 16;                       // tokens of a warp's subtile
constexpr int kAttnTile = kAttnSub * kAttnWarps;   // tokens of a tile
constexpr uint32_t kJoin = 16;                     // pieces whose loads are in flight together
constexpr uint32_t kJoinGroup = 8;
// What the end of a unit costs beside its tiles, in tiles: queries, joins and
// fences (about 2.5 us).  Runs are cut in these terms, or the CTAs with many short
// sequences would come last: a ragged batch of 24 sequences takes 24.5 us without
// it, 20.2, 19.6 and 20.4 with 1, 2 and 3; one of 64 sequences 127, 123, 122 and 121.
constexpr uint32_t kUnitCost = 2;
constexpr float kLog2e = 1.4426950408889634f;
// Weights are held as 2^(s - m) with m 8 below the largest s (in units of
// log 2): binary16 keeps full precision down to 2^-22 of the largest weight
// instead of 2^-14.
constexpr float kWeightShift = 8.0f;

template <int DP>
struct AttnShape {
    static constexpr int kRow = DP * 2 + 16;                    // bytes of a staged row
    static constexpr int kStage = 2 * kAttnTile * kRow;         // K and V of a tile
    // stages and CTAs per SM that fill shared memory: 2 CTAs up to 128
    // columns, one above
    static constexpr int kStages = DP == 64 ? 5 : DP == 96 ? 4 : DP == 128 ? 3 : DP == 192 ? 4 : 3;
    static constexpr int kCtas = DP <= 128 ? 2 : 1;
};

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const char* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
// arrives at the barrier when this thread's copies so far have landed
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// a barrier of the computing warps alone
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kAttnConsumers) : "memory"); }

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

// The smallest 16-bit number, with x's sign.
template <typename C>
__device__ __forceinline__ C smallest(float x) {
    const uint16_t bits = (uint16_t)(fbits(x) >> 31 << 15 | 1u);
    return *reinterpret_cast<const C*>(&bits);
}

// What is left of x after its 16-bit rounding (0 for what is not finite: the
// first part carries it alone).
template <typename C>
__device__ __forceinline__ float rest_of(float x) {
    const float r = x - to_f32(from_f32<C>(x));
    return fabsf(r) < INFINITY ? r : 0.0f;
}

// A place in the order of all tiles: sequence, key/value head, block of query
// heads, tile.
struct TileAt {
    int32_t b;
    uint32_t kvh, block;
    uint32_t tile, tiles;
    int32_t first, len;  // of sequence b
    int64_t at;          // in the order of all tiles and of what a unit costs besides
};

// a / b of numbers that nearly always have 32 bits: a 64-bit division is a call.
__device__ __forceinline__ int64_t divided(int64_t a, int64_t b) {
    return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// A token's row: its page as the table has it, whatever that is, and place in it
// (kNoToken: there is no token; a page has less than 2^31 places).
constexpr uint32_t kNoToken = 0xffffffffu;
struct RowAt {
    int32_t page;
    uint32_t off;
};

template <typename C, int PARTS, int DP>
__global__ void __launch_bounds__(kAttnThreads, AttnShape<DP>::kCtas) paged_attn_kernel(const PagedAttnPlan p) {
    using Shape = AttnShape<DP>;
    using Q = std::conditional_t<PARTS == 1, C, float>;
    constexpr int HPU = PARTS == 1 ? 16 : 8;
    constexpr int kRow = Shape::kRow, kStages = Shape::kStages;
    constexpr int kHeadsWarp = HPU / kAttnWarps;   // query rows that a warp stages
    constexpr int kSlot = HPU * DP * 4 + HPU * 8;  // a warp's (o, m, l) at the end of a segment
    static_assert(kAttnWarps * kSlot <= Shape::kStage, "the pieces of a segment lie in one stage");
    extern __shared__ __align__(16) unsigned char smem[];
    unsigned char* q_tile = smem + kStages * Shape::kStage;
    constexpr int kQBytes = 16 * kRow * (PARTS == 3 ? 2 : 1);
    float* q_scale = reinterpret_cast<float*>(q_tile + kQBytes);           // [16]
    uint2* masks = reinterpret_cast<uint2*>(q_scale + 16);                 // [stage]: bit t = token t (32 + t) is there
    uint64_t* full = reinterpret_cast<uint64_t*>(masks + kStages);         // [stage] barriers
    uint64_t* free_ = full + kStages;
    longlong2* places = reinterpret_cast<longlong2*>(smem + kStages * Shape::kStage + kQBytes + 64 + (kStages * 24 + 15) / 16 * 16);  // [kAttnTile]
    uint32_t* joins = reinterpret_cast<uint32_t*>(places + kAttnTile);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full + s, kAttnLoaders * 33);  // every lane's copies, and the masks
            mbar_init(free_ + s, kAttnWarps);
        }
        mbar_init_fence();
    }
    __syncthreads();
    pdl_enter();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t g = lane >> 2, t4 = lane & 3;
    const uint32_t rep = (uint32_t)p.rep, d = (uint32_t)p.d, page_size = (uint32_t)p.page_size;
    const uint32_t blocks = (rep + HPU - 1) / HPU, kv_heads = (uint32_t)p.heads / rep, units = kv_heads * blocks;
    const int64_t cap64 = (int64_t)(p.table_pages * p.page_size);
    const int32_t cap = cap64 < INT32_MAX ? (int32_t)cap64 : INT32_MAX;
    const int32_t batch = (int32_t)p.batch;

    auto span = [&](int32_t b, int32_t& first, int32_t& len) -> uint32_t {  // tiles of sequence b
        len = p.lengths[b * p.len_st];
        len = len < 0 ? 0 : len > cap ? cap : len;
        first = p.window && (uint64_t)len > p.window ? len - (int32_t)p.window : 0;
        return ((uint32_t)(len - first) + kAttnTile - 1) / kAttnTile;
    };

    // ---- this CTA's run of tiles, found by every warp for itself
    uint32_t mine = 0;
    bool empty = false, bad = false;
#pragma unroll 4
    for (int32_t base = 0; base < batch; base += 32) {
        const int32_t b = base + lane;
        int32_t f, n;
        const uint32_t tiles = b < batch ? span(b, f, n) : 0;
        mine += tiles ? tiles + kUnitCost : 0;
        empty = empty || (b < batch && tiles == 0);
    }
    const int64_t total = (((int64_t)__reduce_add_sync(0xffffffffu, mine >> 16) << 16) +
                           __reduce_add_sync(0xffffffffu, mine & 0xffffu)) * units;
    const int64_t run = total == 0 ? 1 : divided(total + gridDim.x - 1, gridDim.x);
    const int64_t start = run * blockIdx.x;
    const int64_t stop = start + run < total ? start + run : total;

    if (__any_sync(0xffffffffu, empty)) {  // sequences without tokens: zeros, spread over the CTAs
        for (int32_t b = blockIdx.x; b < batch; b += gridDim.x) {
            int32_t f, n;
            if (span(b, f, n) != 0) continue;
            for (uint64_t i = threadIdx.x; i < p.heads * d; i += kAttnThreads)
                reinterpret_cast<Q*>(p.dst + (i / d) * p.dst_st[1] + b * p.dst_st[2])[i % d] = from_f32<Q>(0.0f);
        }
    }
    if (blockIdx.x == 0) {
        for (int32_t b = threadIdx.x; b < batch; b += kAttnThreads) {
            bad = bad || p.lengths[b * p.len_st] > cap;  // a negative length is an empty sequence
        }
        if (bad) atomicExch(p.reject, p.reject_code);
    }
    if (start >= stop) return;

    TileAt to;  // the next tile to load or to compute
    {
        int64_t before = 0;  // tiles of the sequences before `base`
        uint32_t found = 0;
        int32_t base = 0;
        int64_t off = 0;
        for (; base < batch; base += 32) {
            const int32_t b = base + lane;
            int32_t f, n;
            uint32_t cost = b < batch ? span(b, f, n) : 0;
            cost += cost ? kUnitCost : 0;
            uint32_t sum = cost;  // of 32 sequences: at most 2^31
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            off = start - (before + sum - cost) * units;  // from the start of sequence b on
            found = __ballot_sync(0xffffffffu, off >= 0 && off < (int64_t)cost * units);
            if (found) break;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        const int from = __ffs(found) - 1;
        to.b = base + from;
        off = __shfl_sync(0xffffffffu, off, from);
        to.tiles = span(to.b, to.first, to.len);
        const uint32_t unit = (uint32_t)divided(off, to.tiles + kUnitCost), in = (uint32_t)(off - (int64_t)unit * (to.tiles + kUnitCost));
        to.tile = in < kUnitCost ? 0 : in - kUnitCost;
        to.at = in < kUnitCost ? start + kUnitCost - in : start;
        to.kvh = unit / blocks;
        to.block = unit % blocks;
    }
    if (to.at >= stop) return;
    auto advance = [&](TileAt& x) {
        ++x.at;
        if (++x.tile < x.tiles) return;
        x.at += kUnitCost;
        x.tile = 0;
        if (++x.block < blocks) return;
        x.block = 0;
        if (++x.kvh < kv_heads) return;
        x.kvh = 0;
        do {
            if (++x.b >= batch) return;  // past the last tile: never used
            x.tiles = span(x.b, x.first, x.len);
        } while (x.tiles == 0);
    };

    auto row_of = [&](const TileAt& x, uint32_t token) -> RowAt {
        const uint32_t t = (uint32_t)x.first + x.tile * kAttnTile + token;  // at most 63 beyond a length
        if (t >= (uint32_t)x.len) return RowAt{-1, kNoToken};
        // t / page_size by the host's multiplier (t < 2^31)
        const uint32_t at = (uint32_t)(((uint64_t)t * p.page_mul) >> p.page_shift);
        return RowAt{p.table[(int64_t)at * p.table_st[0] + (int64_t)x.b * p.table_st[1]], t - at * page_size};
    };
    auto known = [&](const RowAt& r) {
        const bool in = (uint64_t)(int64_t)r.page < p.pages;  // a negative page is a huge number
        if (!in && r.off != kNoToken) atomicExch(p.reject, p.reject_code);
        return in;
    };
    auto key_row = [&](const TileAt& x, const RowAt& r) {
        return p.k + x.kvh * p.k_st[1] + (uint64_t)(uint32_t)r.page * p.k_st[3] + r.off * p.k_st[2];
    };
    auto value_row = [&](const TileAt& x, const RowAt& r) {
        return p.v + x.kvh * p.v_st[1] + (uint64_t)(uint32_t)r.page * p.v_st[3] + r.off * p.v_st[2];
    };

    // ---- the loading warps
    if (warp >= kAttnWarps) {
        if (!p.vec) return;
        constexpr int kLanes = DP % 64 == 0 ? 8 : 4;  // lanes that bring a row, 32 / kLanes rows at a time
        const uint32_t half = warp - kAttnWarps, token = half * 32 + lane;
        const uint32_t sub = lane % kLanes, of = lane / kLanes;
        longlong2* my_places = places + half * 32;
        RowAt next = row_of(to, token);
        int stage = 0;
        uint32_t turn = 0;  // how often the ring has been filled
        for (bool more = true; more;) {
            const RowAt now = next;
            const bool in = known(now);
            const uint32_t mask = __ballot_sync(0xffffffffu, in);
            // every row's addresses, for the lanes that bring it
            __syncwarp();
            my_places[lane] = make_longlong2(reinterpret_cast<int64_t>(in ? key_row(to, now) : p.k),
                                             reinterpret_cast<int64_t>(in ? value_row(to, now) : p.v));
            advance(to);
            more = to.at < stop;
            if (more) next = row_of(to, token);  // in flight during this tile
            const bool waited = turn == 0 || mbar_try(free_ + stage, (turn - 1) & 1u) || mbar_wait(free_ + stage, (turn - 1) & 1u);
            if (!__all_sync(0xffffffffu, waited)) {
                if (lane == 0) atomicExch(p.fault, 1u);
                break;
            }
            if (lane == 0) {
                (half ? masks[stage].y : masks[stage].x) = mask;
                mbar_arrive(full + stage);
            }
            __syncwarp();
            const uint32_t dst = smem_u32(smem) + stage * Shape::kStage + (half * 32 + of) * kRow + sub * 16;
#pragma unroll
            for (int r = 0; r < 32; r += 32 / kLanes) {
                const longlong2 place = my_places[r + of];
                const char* k = reinterpret_cast<const char*>(place.x) + sub * 16;
                const char* v = reinterpret_cast<const char*>(place.y) + sub * 16;
                const bool here = (mask >> (r + of)) & 1u;
#pragma unroll
                for (int j = 0; j < DP / 8 / kLanes; ++j) {
                    const bool use = here && (sub + j * kLanes) * 8 < d;
                    cp16(dst + r * kRow + j * kLanes * 16, k + j * kLanes * 16, use);
                    cp16(dst + (r + kAttnTile) * kRow + j * kLanes * 16, v + j * kLanes * 16, use);
                }
            }
            cp_arrive(full + stage);
            if (++stage == kStages) {
                stage = 0;
                ++turn;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        return;
    }

    // ---- query rows: warp w stages rows w * kHeadsWarp ...
    Q x[kHeadsWarp][DP / 32];
    auto load_query = [&](const TileAt& at) {
#pragma unroll
        for (int i = 0; i < kHeadsWarp; ++i) {
            // loads without a condition are in flight together; what has no place becomes 0 later
            const uint32_t h = at.block * HPU + warp * kHeadsWarp + i, hh = h < rep ? h : rep - 1;
            const Q* row = reinterpret_cast<const Q*>(p.q + ((uint64_t)at.kvh * rep + hh) * p.q_st[1] + at.b * p.q_st[2]);
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                const uint32_t col = lane + 32 * c;
                x[i][c] = row[col < d ? col : d - 1];
            }
        }
    };
    auto stage_query = [&](const TileAt& at) {
#pragma unroll
        for (int i = 0; i < kHeadsWarp; ++i) {
            const uint32_t r = warp * kHeadsWarp + i;
            const bool there = at.block * HPU + r < rep;
            float y[DP / 32];
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) y[c] = there && lane + 32 * c < d ? to_f32(x[i][c]) : 0.0f;
            float up = 1.0f, down = 1.0f;
            if constexpr (PARTS >= 2) {
                float big = 0.0f;  // the largest finite one; a subnormal counts as 2^-126
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) big = fmaxf(big, fabsf(y[c]) < INFINITY ? fabsf(y[c]) : 0.0f);
                const uint32_t field = __reduce_max_sync(0xffffffffu, fbits(big)) >> 23;
                const int e = field > 0 ? (int)field - 127 : -126;
                // bfloat16 parts lose bits below 2^-133 only, and round the largest binary32 numbers to infinity
                const int by = PARTS == 2 ? (e < 127 ? -e : -126) : e < -40 ? -40 - e : e == 127 ? -1 : 0;
                down = bitsf((uint32_t)(127 + by) << 23);
                up = bitsf((uint32_t)(127 - by) << 23);
            }
            if (lane == 0) q_scale[r] = p.scale * up * kLog2e;
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                const uint32_t col = lane + 32 * c;
                const float z = y[c] * down;
                C first = from_f32<C>(z);
                // what rounds to 0 keeps its sign for a key that is infinite (0 would make a NaN of it); the
                // next part takes the smallest number back
                if (PARTS >= 2 && y[c] != 0.0f && to_f32(first) == 0.0f) first = smallest<C>(y[c]);
                *reinterpret_cast<C*>(q_tile + r * kRow + col * 2) = first;
                if constexpr (PARTS >= 2) {
                    const float left = z - to_f32(first), rest = fabsf(left) < INFINITY ? left : 0.0f;
                    *reinterpret_cast<C*>(q_tile + (8 + r) * kRow + col * 2) = from_f32<C>(rest);
                    if constexpr (PARTS == 3)
                        *reinterpret_cast<C*>(q_tile + (16 + r) * kRow + col * 2) = from_f32<C>(rest_of<C>(rest));
                }
            }
        }
    };
    load_query(to);
    stage_query(to);
    consumers_sync();

    // ldmatrix addresses of this lane
    const uint32_t k_at = ((lane >> 4) * 8 + (lane & 7)) * kRow + ((lane >> 3) & 1) * 16;
    const uint32_t v_at = (((lane >> 3) & 1) * 8 + (lane & 7)) * kRow + (lane >> 4) * 16 + kAttnTile * kRow;
    const uint32_t q_at = smem_u32(q_tile) + (((lane >> 3) & 1) * 8 + (lane & 7)) * kRow + (lane >> 4) * 16;
    const uint32_t q2_at = smem_u32(q_tile) + 16 * kRow + (lane & 7) * kRow + ((lane >> 3) & 1) * 16;

    constexpr int kHeadsLane = PARTS == 1 ? 2 : 1;  // heads of a lane's result rows: g (and g + 8)
    float o[DP / 8][4];
    float m[kHeadsLane], l[kHeadsLane], sc[kHeadsLane];
    auto begin_segment = [&]() {
#pragma unroll
        for (int h = 0; h < kHeadsLane; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.0f;
            sc[h] = q_scale[g + 8 * h];
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    };
    begin_segment();
    int stage = 0;
    uint32_t turn = 0;
    bool late = false;  // a wait has expired: what follows is only the walk to the end
    bool first_segment = true;

#pragma unroll 1
    for (;;) {
        unsigned char* rows = smem + stage * Shape::kStage + warp * kAttnSub * kRow;  // this warp's keys; values kAttnTile rows on
        uint32_t mask;  // of this warp's tokens
        if (p.vec) {
            if (!late && !__all_sync(0xffffffffu, mbar_try(full + stage, turn & 1u) || mbar_wait(full + stage, turn & 1u))) {
                late = true;
                if (lane == 0) atomicExch(p.fault, 1u);
            }
            mask = late ? 0u : ((warp < 2 ? masks[stage].x : masks[stage].y) >> ((warp & 1) * kAttnSub)) & 0xffffu;
        } else {
            const RowAt r = row_of(to, warp * kAttnSub + (lane & 15));
            const bool in = known(r);
            mask = __ballot_sync(0xffffffffu, in) & 0xffffu;
            const uint64_t kr = in ? reinterpret_cast<uint64_t>(key_row(to, r)) : 0, vr = in ? reinterpret_cast<uint64_t>(value_row(to, r)) : 0;
            for (int row = 0; row < kAttnSub; ++row) {
                const uint16_t* ks = reinterpret_cast<const uint16_t*>(__shfl_sync(0xffffffffu, kr, row));
                const uint16_t* vs = reinterpret_cast<const uint16_t*>(__shfl_sync(0xffffffffu, vr, row));
                for (uint32_t col = lane; col < DP; col += 32) {
                    const bool use = ((mask >> row) & 1u) && col < d;
                    *reinterpret_cast<uint16_t*>(rows + row * kRow + col * 2) = use ? ks[col] : (uint16_t)0;
                    *reinterpret_cast<uint16_t*>(rows + (kAttnTile + row) * kRow + col * 2) = use ? vs[col] : (uint16_t)0;
                }
            }
            __syncwarp();
        }
        const uint32_t base = smem_u32(rows);
        if (mask != 0) {
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
            // scores of this lane's tokens 2 t4, 2 t4 + 1 (n = 0) and 8 + those (n = 1)
            float w[kHeadsLane][4], keep[kHeadsLane];
#pragma unroll
            for (int h = 0; h < kHeadsLane; ++h)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float y = s[n][2 * h + e];
                        if constexpr (PARTS >= 2) {
                            // an infinite key: the first part has its sign, a part of 0 would make it NaN
                            const float more = PARTS == 3 ? s[n][2 + e] + s3[PARTS == 3 ? n : 0][e] : s[n][2 + e];
                            y = fabsf(y) < INFINITY ? y + more : y;
                        }
                        w[h][2 * n + e] = y;
                    }
            if (mask != 0xffffu) {
#pragma unroll
                for (int h = 0; h < kHeadsLane; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((mask >> ((e & 2) * 4 + 2 * t4 + (e & 1))) & 1u)) w[h][e] = -INFINITY;
            }
            bool moved = false;
#pragma unroll
            for (int h = 0; h < kHeadsLane; ++h) {
                float top = fmaxf(fmaxf(w[h][0], w[h][1]), fmaxf(w[h][2], w[h][3]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(m[h], __fmaf_rn(top, sc[h], -kWeightShift));
                const float ref = top == -INFINITY ? 0.0f : top;  // only -inf so far: every weight is 0
                keep[h] = ex2(m[h] - ref);
                moved = moved || m[h] != top;
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
            uint32_t a0, a1, a2, a3, c0 = 0, c1 = 0, c2 = 0, c3 = 0;
            a0 = pack2<C>(w[0][0], w[0][1]);
            a2 = pack2<C>(w[0][2], w[0][3]);
            if constexpr (PARTS == 1) {
                a1 = pack2<C>(w[1][0], w[1][1]);
                a3 = pack2<C>(w[1][2], w[1][3]);
                c0 = pack2<C>(rest_of<C>(w[0][0]), rest_of<C>(w[0][1]));
                c2 = pack2<C>(rest_of<C>(w[0][2]), rest_of<C>(w[0][3]));
                c1 = pack2<C>(rest_of<C>(w[1][0]), rest_of<C>(w[1][1]));
                c3 = pack2<C>(rest_of<C>(w[1][2]), rest_of<C>(w[1][3]));
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
                if constexpr (PARTS != 2) {
                    mma16816<C>(o[2 * n], c0, c1, c2, c3, b[0], b[1]);
                    mma16816<C>(o[2 * n + 1], c0, c1, c2, c3, b[2], b[3]);
                }
            }
        }
        const bool unit_ends = to.tile + 1 == to.tiles;
        auto release = [&]() {  // the stage may be filled again
            __syncwarp();
            if (p.vec && lane == 0) mbar_arrive(free_ + stage);
            if (++stage == kStages) {
                stage = 0;
                ++turn;
            }
        };
        const bool more = to.at + 1 + (unit_ends ? kUnitCost : 0) < stop;
        if (!unit_ends && more) {
            ++to.tile;
            ++to.at;
            release();
            continue;
        }

        // ---- the end of a segment: the warps' pieces join, in this stage
        const TileAt at = to;
        consumers_sync();  // every warp has read its rows
        unsigned char* stage_at = smem + stage * Shape::kStage;
        float* piece = reinterpret_cast<float*>(stage_at + warp * kSlot);
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
            float* spot = piece + g * DP + n * 8 + 2 * t4;
            if constexpr (PARTS == 1) {
                *reinterpret_cast<float2*>(spot) = make_float2(o[n][0], o[n][1]);
                *reinterpret_cast<float2*>(spot + 8 * DP) = make_float2(o[n][2], o[n][3]);
            } else {
                *reinterpret_cast<float2*>(spot) = make_float2(o[n][0] + o[n][2], o[n][1] + o[n][3]);
            }
        }
        if (more) {
            advance(to);
            load_query(to);  // in flight while the pieces join
        }
        consumers_sync();
        const uint32_t h0 = at.block * HPU, nh = rep - h0 < HPU ? rep - h0 : HPU;
        const int64_t unit_first = at.at - at.tile, unit_last = unit_first + at.tiles - 1;  // its tiles in the order
        const bool whole = unit_first >= start && unit_ends;
        const uint32_t quads = (d + 3) / 4;  // four columns at a time; rows of a slot are padded to them
        const uint64_t slot_floats = (uint64_t)HPU * (quads * 4 + 4);  // o, (m, l), a group's (m, l)
        char* out = p.dst + ((uint64_t)at.kvh * rep + h0) * p.dst_st[1] + at.b * p.dst_st[2];
        auto write = [&](uint32_t r, uint32_t q4, const float4& v, float sum) {
            Q* row = reinterpret_cast<Q*>(out + r * p.dst_st[1]) + q4 * 4;
            const float y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (q4 * 4 + c < d) row[c] = from_f32<Q>(sum == 0.0f ? 0.0f : y[c] / sum);
        };
        float* slot = p.pieces + ((uint64_t)blockIdx.x * 2 + (first_segment ? 0 : 1)) * slot_floats;
        auto warp_piece = [&](int w) { return reinterpret_cast<const float*>(stage_at + w * kSlot); };
        for (uint32_t e = threadIdx.x; e < nh * quads; e += kAttnConsumers) {
            const uint32_t r = e / quads, q4 = e - r * quads;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, warp_piece(w)[HPU * DP + r]);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) {
                const float f = ex2(warp_piece(w)[HPU * DP + r] - ref);
                const float4 y = *reinterpret_cast<const float4*>(warp_piece(w) + r * DP + q4 * 4);
                sum = __fmaf_rn(f, warp_piece(w)[HPU * DP + HPU + r], sum);
                v.x = __fmaf_rn(f, y.x, v.x);
                v.y = __fmaf_rn(f, y.y, v.y);
                v.z = __fmaf_rn(f, y.z, v.z);
                v.w = __fmaf_rn(f, y.w, v.w);
            }
            if (whole) {
                write(r, q4, v, sum);
            } else {
                __stcg(reinterpret_cast<float4*>(slot + r * quads * 4) + q4, v);
                if (q4 == 0) __stcg(reinterpret_cast<float2*>(slot + HPU * quads * 4) + r, make_float2(top, sum));
            }
        }
        if (!whole) {
            const int64_t c0 = divided(unit_first, run);
            const uint32_t pieces = (uint32_t)(divided(unit_last, run) - c0) + 1, me = (uint32_t)(blockIdx.x - c0);
            // of the unit's first piece: a CTA's first segment or its last one
            const uint64_t slot0 = (uint64_t)c0 * 2 + (unit_first - kUnitCost <= c0 * run ? 0 : 1);
            // many pieces join in two steps, eight CTAs' first: each step waits for
            // its loads about once
            const bool groups = pieces > kJoin;
            const uint32_t group = groups ? me / kJoinGroup : 0;
            const uint32_t of_group = !groups ? pieces : pieces - group * kJoinGroup < kJoinGroup ? pieces - group * kJoinGroup : kJoinGroup;
            const uint64_t head = group == 0 ? slot0 : (uint64_t)(c0 + group * kJoinGroup) * 2;  // the group's first slot
            auto last_of = [&](uint32_t* ticket, uint32_t n) {  // of n CTAs, the last one to come here
                __threadfence();
                consumers_sync();
                if (threadIdx.x == 0) {
                    *joins = atomicAdd(ticket, 1u) == n - 1;
                    if (*joins) *ticket = 0;
                }
                consumers_sync();
                const bool last = *joins != 0;
                if (last) __threadfence();
                return last;
            };
            // n slots from `first` on, then every `step` slots from `base`: the (m, l) at ml
            auto join = [&](uint64_t first, uint64_t base, uint32_t step, uint32_t n, uint32_t ml_at, auto&& done) {
                const float* s0 = p.pieces + first * slot_floats;
                const float* s1 = p.pieces + base * slot_floats;
                for (uint32_t e = threadIdx.x; e < nh * quads; e += kAttnConsumers) {
                    const uint32_t r = e / quads, q4 = e - r * quads;
                    float top = -INFINITY, sum = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (uint32_t k0 = 0; k0 < n; k0 += kJoin) {
                        float2 ml[kJoin];
                        float4 y[kJoin];
#pragma unroll
                        for (uint32_t k = 0; k < kJoin; ++k) {
                            ml[k] = make_float2(-INFINITY, 0.0f);
                            y[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (k0 + k < n) {
                                const float* s = k0 + k == 0 ? s0 : s1 + (uint64_t)(k0 + k) * step * slot_floats;
                                ml[k] = __ldcg(reinterpret_cast<const float2*>(s + ml_at) + r);
                                y[k] = __ldcg(reinterpret_cast<const float4*>(s + r * quads * 4) + q4);
                            }
                        }
                        float now = top;
#pragma unroll
                        for (uint32_t k = 0; k < kJoin; ++k) now = fmaxf(now, ml[k].x);
                        const float ref = now == -INFINITY ? 0.0f : now, keep = ex2(top - ref);
                        top = now;
                        sum *= keep;
                        v.x *= keep, v.y *= keep, v.z *= keep, v.w *= keep;
#pragma unroll
                        for (uint32_t k = 0; k < kJoin; ++k) {
                            const float f = ex2(ml[k].x - ref);
                            sum = __fmaf_rn(f, ml[k].y, sum);
                            v.x = __fmaf_rn(f, y[k].x, v.x);
                            v.y = __fmaf_rn(f, y[k].y, v.y);
                            v.z = __fmaf_rn(f, y[k].z, v.z);
                            v.w = __fmaf_rn(f, y[k].w, v.w);
                        }
                    }
                    done(r, q4, v, top, sum);
                }
            };
            auto finish = [&](uint32_t r, uint32_t q4, const float4& v, float, float sum) { write(r, q4, v, sum); };
            const uint32_t ml0 = HPU * quads * 4, ml1 = ml0 + HPU * 2;  // a piece's (m, l), a group's
            if (last_of(p.tickets + head, of_group)) {
                if (!groups) {
                    join(head, c0 * 2, 2, pieces, ml0, finish);
                } else {
                    // into the group's first slot: a thread overwrites what it alone has read
                    join(head, (uint64_t)(c0 + group * kJoinGroup) * 2, 2, of_group, ml0,
                         [&](uint32_t r, uint32_t q4, const float4& v, float top, float sum) {
                             float* s = p.pieces + head * slot_floats;
                             __stcg(reinterpret_cast<float4*>(s + r * quads * 4) + q4, v);
                             if (q4 == 0) __stcg(reinterpret_cast<float2*>(s + ml1) + r, make_float2(top, sum));
                         });
                    const uint32_t all = (pieces + kJoinGroup - 1) / kJoinGroup;
                    if (last_of(p.tickets + p.slots + slot0, all)) join(slot0, c0 * 2, 2 * kJoinGroup, all, ml1, finish);
                }
            }
        }
        if (!more) break;
        stage_query(to);
        first_segment = false;
        consumers_sync();  // the pieces have been read, the query rows are there
        release();
        begin_segment();
    }
}

template <typename S, typename C>
cudaError_t run_append(const LaunchEnv& env, const PagedAppendPlan& p) {
    if (p.vec) {
        // lanes of a row: a power of two, so that a thread keeps its place in every row
        const uint64_t per = p.kv_heads * (p.d / 8);
        uint32_t lanes = 8;
        while (lanes < kAppendThreads && lanes < per) lanes *= 2;
        const uint64_t rows = kAppendThreads / lanes, want = (p.count + rows - 1) / rows, cap = (uint64_t)env.sm_count * 8;
        const cudaError_t err = launch_dependent(append_rows_kernel<S, C>, dim3((unsigned)(want < cap ? want : cap)),
                                                 dim3(kAppendThreads), 0, env.stream, p, lanes);
        if (err == cudaSuccess) ++*env.launches;
        return err;
    }
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
    constexpr int kSmem = Shape::kStages * Shape::kStage + 16 * Shape::kRow * (PARTS == 3 ? 2 : 1) + 64 +
                          (Shape::kStages * 24 + 15) / 16 * 16 + kAttnTile * 16 + 16;
    static DeviceFlags ready;
    if (!ready.done(env.device)) {
        const cudaError_t err = cudaFuncSetAttribute(paged_attn_kernel<C, PARTS, DP>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (err != cudaSuccess) return err;
        ready.mark(env.device);
    }
    // one wave, no more CTAs than there are tiles at most or slots for pieces
    const uint64_t slot = (uint64_t)HPU * ((p.d + 3) / 4 * 4 + 4) * 4;
    uint64_t grid = (uint64_t)env.sm_count * Shape::kCtas;
    if (grid > paged_piece_bytes(env.sm_count) / (2 * slot)) grid = paged_piece_bytes(env.sm_count) / (2 * slot);
    p.slots = 2 * grid;
    if (2 * p.slots > paged_tickets(env.sm_count)) return cudaErrorInvalidValue;
    const unsigned __int128 most = (unsigned __int128)((p.table_pages * p.page_size + kAttnTile - 1) / kAttnTile) *
                                   p.batch * (p.heads / p.rep) * ((p.rep + HPU - 1) / HPU);
    if (most < grid) grid = (uint64_t)most;
    // t / page_size = (t * page_mul) >> page_shift for t < 2^31: page_mul is
    // 2^page_shift / page_size rounded up, with 2^page_shift >= 2^31 page_size
    p.page_shift = 31;
    while ((1ull << (p.page_shift - 31)) < p.page_size) ++p.page_shift;
    p.page_mul = (uint64_t)((((unsigned __int128)1 << p.page_shift) + p.page_size - 1) / p.page_size);
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
uint64_t paged_piece_bytes(int sm_count) { return (uint64_t)sm_count * 2 * 16 * (kPagedMaxD + 8) * 4; }
// A ticket for each slot's group and one for each slot's unit, at two CTAs per SM.
uint64_t paged_tickets(int sm_count) { return (uint64_t)sm_count * 8; }

cudaError_t launch_paged_attn(const LaunchEnv& env, const PagedAttnPlan& p) {
    if (p.cache_bf16) return p.q_f32 ? run_attn<__nv_bfloat16, 3>(env, p) : run_attn<__nv_bfloat16, 1>(env, p);
    return p.q_f32 ? run_attn<__half, 2>(env, p) : run_attn<__half, 1>(env, p);
}

}  // namespace emel
