// kv8.cu - the KV cache in 8 bits: append (quantise) and paged GQA decode
// attention over it, for sm_100a.
//
// A (page, KV head, plane) tile of 16 tokens x 128 dimensions is stored as
// code bytes with one fp32 scale; a sequence's unfinished page stays in bf16
// ("tail").  Layout: kv_layout.h; contract: rlrt.h.
//
// Both move bytes: their floor is what they read and write once, at the rate of a
// copy (6,547 GB/s measured here).  Times are of calls in a graph, inputs changing
// from call to call, merge included.
//   append     256 sequences x 1 token, 8 KV heads       5.3 us  (launch and the
//                                       dependent loads before a row's)
//              64 prompts of 64..1,024 tokens, bf16       46 us  75% of copy
//              the same, fp32                             72 us  80%
//              4 prompts of 30,001..32,768 tokens        127 us  92%
//   attention  1 sequence of 17 tokens                   4.4 us  (latency)
//              64 of 128..4,096, 32 heads on 8            60 us  80%
//              256 of 512..768, 32 heads on 8             63 us  83%
//              1 of 131,071, 32 heads on 4                29 us  70%
#include <cuda_fp16.h>

#include <cmath>
#include <cstdint>

#include "kv_layout.h"
#include "rlrt.h"
#include "rt_common.cuh"

namespace {

enum : int32_t { kErrLen = 1, kErrPage = 2, kErrCu = 3, kErrTimeout = 4 };
constexpr uint32_t kPlane = RT_KV8_PLANE_BYTES;

__device__ __forceinline__ void flag_error(int32_t *err, int32_t code)
{
    if (err)
        atomicCAS(err, 0, code);
}

// ------------------------------------------------------------------ append
struct AppendArgs {
    const void *k, *v;
    const int32_t *cu, *lens, *page_table;
    uint8_t *pages;
    float *scales;
    __nv_bfloat16 *tail;
    int32_t *error;
    uint64_t k_stride, v_stride, arena_pages;
    uint32_t num_seqs, num_kv_heads, num_tokens, max_pages;
    uint64_t n_items;  // units x KV heads
};

constexpr int kAppendWarps = 8;

// Four consecutive elements of a token's row, as loaded and as two bf16 pairs.  The
// loads are volatile so that they stay where they are written, ahead of the search
// for the warp's next item.
template <bool F32>
struct Four;
template <>
struct Four<true> {
    float4 v;
    __device__ __forceinline__ void load(const void *base, uint64_t elem)
    {
        asm volatile("ld.global.cs.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                     : "l"(static_cast<const float *>(base) + elem));
    }
    __device__ __forceinline__ uint2 bf16() const
    {
        return make_uint2(rt::pack_bf16x2(v.x, v.y), rt::pack_bf16x2(v.z, v.w));
    }
};
template <>
struct Four<false> {
    uint2 v;
    __device__ __forceinline__ void load(const void *base, uint64_t elem)
    {
        asm volatile("ld.global.cs.v2.u32 {%0, %1}, [%2];"
                     : "=r"(v.x), "=r"(v.y)
                     : "l"(static_cast<const uint16_t *>(base) + elem));
    }
    __device__ __forceinline__ uint2 bf16() const { return v; }
};

__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

// Codes of two quotients, in the two low bytes; the others hold anything.
template <uint32_t FMT>
__device__ __forceinline__ uint32_t codes2(rt::f32x2 y)
{
    if constexpr (FMT == RT_KV8_E4M3) {
        const float2 v = rt::halves(y);
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v.y), "f"(v.x));
        return r;
    } else {
        // 1.5 x 2^23 + y rounds y to the nearest integer, ties to even, and holds it in
        // its low bits
        constexpr float kRound = 12582912.0f;
        const float2 v = rt::halves(rt::add2(y, rt::pair(kRound, kRound)));
        return __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x0040);
    }
}

// Codes of four elements.  The quotient has to be the correctly rounded one, since
// codes change at quotients of k + 1/2: with inv the correctly rounded reciprocal,
// q = x inv and one step q + (x - q scale) inv, in fused operations, give it
// (Markstein, IBM J. Res. Dev. 34, 1990), as long as nothing leaves the normal
// range; tiles of other scales divide.
template <uint32_t FMT>
__device__ __forceinline__ uint32_t quantise4(uint2 x, float scale, float inv, bool plain)
{
    const uint32_t w[2] = {x.x, x.y};
    uint32_t r[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float lo = bf16_lo(w[i]), hi = bf16_hi(w[i]);
        if (plain) {
            const rt::f32x2 f = rt::pair(lo, hi), inv2 = rt::pair(inv, inv);
            const rt::f32x2 q = rt::mul2(f, inv2);
            r[i] = codes2<FMT>(rt::fma2(rt::fma2(q, rt::pair(-scale, -scale), f), inv2, q));
        } else {
            const float most = FMT == RT_KV8_E4M3 ? 448.0f : 127.0f;
            r[i] = codes2<FMT>(rt::pair(fminf(fmaxf(__fdiv_rn(lo, scale), -most), most),
                                        fminf(fmaxf(__fdiv_rn(hi, scale), -most), most)));
        }
    }
    return __byte_perm(r[0], r[1], 0x5410);
}

// Word w of a tile in shared memory: 16-byte vectors are permuted among the 8 of a
// 128-byte row so that the scattered word stores below meet few bank conflicts (K
// two ways, V none) and the vectors are read back without any.
__device__ __forceinline__ uint32_t staged(uint32_t w)
{
    return w ^ (((w >> 7) << 1 | (w >> 6 & 1u)) << 2);
}

// Quantise one tile (lane: dimensions 4 lane .. 4 lane + 3 of the 16 tokens) and
// store it in page order.
template <uint32_t FMT>
__device__ __forceinline__ void store_tile(const uint2 (&x)[16], uint32_t plane, uint32_t *stage,
                                           uint8_t *page, float *scale_out)
{
    const uint32_t lane = threadIdx.x & 31;
    uint32_t top2 = 0;  // per 16-bit half: the largest magnitude's bits
#pragma unroll
    for (int t = 0; t < 16; t++)
        top2 = __vmaxu2(top2, __vmaxu2(x[t].x & 0x7FFF7FFFu, x[t].y & 0x7FFF7FFFu));
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, max(top2 & 0xFFFFu, top2 >> 16));
    // a NaN's or infinity's bits are above every number's
    const float scale = top >= 0x7F80u ? __int_as_float(0x7FC00000)
                                       : __fdiv_rn(__uint_as_float(top << 16),
                                                   FMT == RT_KV8_E4M3 ? 448.0f : 127.0f);
    const bool plain = scale > 0x1p-90f && scale < 0x1p90f;
    const float inv = plain ? __frcp_rn(scale) : 0.0f;
    uint32_t w[16];
    if (plain) {
#pragma unroll
        for (int t = 0; t < 16; t++)
            w[t] = quantise4<FMT>(x[t], scale, inv, true);
    } else {
#pragma unroll
        for (int t = 0; t < 16; t++)
            w[t] = scale > 0.0f ? quantise4<FMT>(x[t], scale, 0.0f, false) : 0u;
    }
    if (plane == 0) {
#pragma unroll
        for (int t = 0; t < 16; t++)
            stage[staged(rt_kv8_k_offset(t, 4 * lane) / 4)] = w[t];
    } else {
        // words of tokens {2c, 2c+1, 2c+8, 2c+9} x 4 dimensions -> 4 words of 4 tokens
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint32_t r0 = w[2 * c], r1 = w[2 * c + 1], r2 = w[2 * c + 8], r3 = w[2 * c + 9];
            const uint32_t p0 = __byte_perm(r0, r1, 0x5140), p1 = __byte_perm(r0, r1, 0x7362);
            const uint32_t q0 = __byte_perm(r2, r3, 0x5140), q1 = __byte_perm(r2, r3, 0x7362);
            const uint32_t o[4] = {__byte_perm(p0, q0, 0x5410), __byte_perm(p0, q0, 0x7632),
                                   __byte_perm(p1, q1, 0x5410), __byte_perm(p1, q1, 0x7632)};
#pragma unroll
            for (int e = 0; e < 4; e++)
                stage[staged(rt_kv8_v_offset(2 * c, 4 * lane + e) / 4)] = o[e];
        }
    }
    __syncwarp();
    uint4 *dst = reinterpret_cast<uint4 *>(page);
#pragma unroll
    for (int i = 0; i < 4; i++)
        dst[i * 32 + lane] = *reinterpret_cast<const uint4 *>(stage + staged((i * 32 + lane) * 4));
    if (lane == 0)
        *scale_out = scale;
    __syncwarp();  // the stage has been read
}

// One warp per (unit, KV head), K and V; a unit is one page of one sequence that
// the call completes, and the first of a sequence its tail.  Sequence b owns the
// units from cu[b] / 16 + b on: n new tokens behind a remainder of up to 15 complete
// at most n / 16 + 1 pages, so the ranges are disjoint and a unit finds its sequence
// by a search of cu, 32 ways at a time, without a scan over the batch.  Lane i holds dimensions 4 i .. 4 i + 3 of all 16
// tokens of both planes, so they are read once, in whole rows, with 8 KiB a warp
// under way, and the maximum, the codes and the 4 x 4 byte transposes of V stay in
// registers.  The sequence's first unit alone reads and writes its tail, each lane
// the dimensions that it owns: the old tokens are in registers before the new ones
// are stored.
//
// A warp takes items in turn and looks for its next one while the loads of the
// current one are under way.  All registers of the SM hold 16 warps with one item
// each, so nothing of the next one can be loaded while the codes are computed (issue
// slots 55% busy): its rows are brought to L2 then (64 prompts 45 us, without 47; 4
// long ones 128 us, without 133; as one bulk prefetch a row 51 and 147).
template <uint32_t FMT, bool F32>
__global__ void __launch_bounds__(kAppendWarps * 32, 2) kv8_append_kernel(const AppendArgs a)
{
    __shared__ __align__(16) uint32_t stage[kAppendWarps][kPlane / 4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t threads = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t i = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; i < a.num_seqs; i += threads)
        if (a.cu[i] < 0 || a.cu[i + 1] < a.cu[i] || (uint32_t)a.cu[i + 1] > a.num_tokens)
            flag_error(a.error, kErrCu);

    struct Item {
        uint32_t b, h;
        uint32_t row, L0, L1, first;  // row: of position L0; first: the page's first position
        int32_t id;                   // the page's, where it becomes full
        bool full, tail;              // to do: the page, the sequence's tail
    };
    auto find = [&](uint64_t item) {
        Item w;
        w.full = w.tail = false;
        if (item >= a.n_items)
            return w;
        w.h = (uint32_t)(item % a.num_kv_heads);
        const int64_t unit = (int64_t)(item / a.num_kv_heads);
        uint32_t b = 0, n = a.num_seqs;  // the last b with cu[b] / 16 + b <= unit, or 0
        while (n > 1) {
            const uint32_t step = (n + 31) / 32, at = b + step * (uint32_t)lane;
            const bool before =
                step * (uint32_t)lane < n && (int64_t)(a.cu[at] >> 4) + (int64_t)at <= unit;
            // cu may decrease in a bad call: then any b will do
            const int last = 31 - __clz(__ballot_sync(0xFFFFFFFFu, before) | 1u);
            n = min(step, n - step * (uint32_t)last);
            b += step * (uint32_t)last;
        }
        const int64_t c0 = a.cu[b], c1 = a.cu[b + 1], L0 = a.lens[b], L1 = L0 + (c1 - c0);
        const int64_t j = unit - ((c0 >> 4) + (int64_t)b);
        if (j < 0 || c0 < 0 || c1 <= c0 || c1 > (int64_t)a.num_tokens)
            return w;
        if (L0 < 0 || (L1 >> 4) > (int64_t)a.max_pages) {
            if (lane == 0)
                flag_error(a.error, kErrLen);
            return w;
        }
        w.b = b;
        // L0 + the tokens of one call stay below 2^32
        w.row = (uint32_t)c0;
        w.L0 = (uint32_t)L0;
        w.L1 = (uint32_t)L1;
        const int64_t page = (L0 >> 4) + j;
        w.first = (uint32_t)page << 4;
        w.full = (page + 1) << 4 <= L1;
        w.tail = j == 0;
        w.id = -1;
        if (w.full) {
            w.id = a.page_table[(uint64_t)b * a.max_pages + (uint64_t)page];
            if (w.id < 0 || (uint64_t)w.id >= a.arena_pages) {
                if (lane == 0)
                    flag_error(a.error, kErrPage);
                w.full = false;
            }
        }
        return w;
    };

    // The next item's rows on their way to L2 while this one's codes are computed: lane l
    // asks for row l & 15 of K or V, in lines of 128 bytes.
    constexpr uint32_t kRowBytes = F32 ? 512u : 256u;
    auto ahead = [&](const Item &n) {
        if (n.full && n.first >= n.L0) {
            const uint64_t row = n.row + (n.first - n.L0) + (lane & 15);
            const uint8_t *p = lane < 16 ? (const uint8_t *)a.k + row * a.k_stride * (kRowBytes / 128u)
                                         : (const uint8_t *)a.v + row * a.v_stride * (kRowBytes / 128u);
            p += n.h * kRowBytes;
#pragma unroll
            for (uint32_t i = 0; i < kRowBytes; i += 128u)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(p + i));
        }
    };
    uint64_t item = (blockIdx.x * (uint64_t)blockDim.x + threadIdx.x) >> 5;
    const uint64_t warps = threads >> 5;
    Item w = find(item);
    for (; item < a.n_items; item += warps) {
        const uint64_t col = (uint64_t)w.h * 128u + 4u * lane;
        __nv_bfloat16 *tail = a.tail + rt_page_elem_offset(w.b, w.h, 0, 0, a.num_kv_heads) + 4 * lane;
        Item next;
        if (w.full && w.first >= w.L0) {  // a page of new tokens alone
            Four<F32> x[2][16];
            const uint64_t row = w.row + (w.first - w.L0);
            uint64_t at_k = row * a.k_stride + col, at_v = row * a.v_stride + col;
#pragma unroll
            for (int t = 0; t < 16; t++) {
                x[0][t].load(a.k, at_k);
                at_k += a.k_stride;
            }
            if constexpr (!F32) {
#pragma unroll
                for (int t = 0; t < 16; t++) {
                    x[1][t].load(a.v, at_v);
                    at_v += a.v_stride;
                }
            }
            next = find(item + warps);
            ahead(next);
            const uint64_t tile = ((uint64_t)w.id * a.num_kv_heads + w.h) * 2u;
            uint2 y[16];
#pragma unroll
            for (int t = 0; t < 16; t++)
                y[t] = x[0][t].bf16();
            store_tile<FMT>(y, 0, stage[warp], a.pages + tile * kPlane, a.scales + tile);
            if constexpr (F32) {  // twice the registers
#pragma unroll
                for (int t = 0; t < 16; t++) {
                    x[1][t].load(a.v, at_v);
                    at_v += a.v_stride;
                }
            }
#pragma unroll
            for (int t = 0; t < 16; t++)
                y[t] = x[1][t].bf16();
            store_tile<FMT>(y, 1, stage[warp], a.pages + (tile + 1) * kPlane, a.scales + tile + 1);
        } else {
            if (w.full) {  // old tokens from the tail, then new ones
                const uint64_t tile = ((uint64_t)w.id * a.num_kv_heads + w.h) * 2u;
                uint2 y[2][16];
#pragma unroll
                for (int t = 0; t < 16; t++) {
                    const uint32_t pos = w.first + t;
                    if (pos < w.L0) {
                        y[0][t] = *reinterpret_cast<const uint2 *>(tail + t * 128);
                        y[1][t] = *reinterpret_cast<const uint2 *>(tail + 2048 + t * 128);
                    } else {
                        const uint64_t row = w.row + (pos - w.L0);
                        Four<F32> k, v;
                        k.load(a.k, row * a.k_stride + col);
                        v.load(a.v, row * a.v_stride + col);
                        y[0][t] = k.bf16();
                        y[1][t] = v.bf16();
                    }
                }
                store_tile<FMT>(y[0], 0, stage[warp], a.pages + tile * kPlane, a.scales + tile);
                store_tile<FMT>(y[1], 1, stage[warp], a.pages + (tile + 1) * kPlane, a.scales + tile + 1);
            }
            next = find(item + warps);
        }
        if (w.tail) {
            const uint32_t base = w.L1 & ~15u, from = max(base, w.L0);
            const int n = (int)(w.L1 - from);
            // up to 15, of which 5 of K and of V are under way at once
            const uint64_t row = w.row + (from - w.L0);
            uint64_t at_k = row * a.k_stride + col, at_v = row * a.v_stride + col;
            __nv_bfloat16 *to = tail + (from - base) * 128;
#pragma unroll 1
            for (int t0 = 0; t0 < n; t0 += 5) {
                Four<F32> k[5], v[5];
#pragma unroll
                for (int t = 0; t < 5; t++) {
                    if (t0 + t < n) {
                        k[t].load(a.k, at_k);
                        v[t].load(a.v, at_v);
                    }
                    at_k += a.k_stride;
                    at_v += a.v_stride;
                }
#pragma unroll
                for (int t = 0; t < 5; t++) {
                    if (t0 + t < n) {
                        *reinterpret_cast<uint2 *>(to + (t0 + t) * 128) = k[t].bf16();
                        *reinterpret_cast<uint2 *>(to + 2048 + (t0 + t) * 128) = v[t].bf16();
                    }
                }
            }
        }
        w = next;
    }
}

// --------------------------------------------------------------- attention
constexpr int kWarps = 4;
constexpr int kStages = 2;
constexpr int kCtasPerSm = 3;
constexpr uint32_t kBlockBytes = 2 * kPlane;       // one (page, head): K plane, V plane
constexpr uint32_t kEntryBytes = 2 * kBlockBytes;  // two pages, or a tail's K and V rows
constexpr uint32_t kHeadPitch = 132;               // floats per column of the warps' merge
constexpr int kSmemBytes = kWarps * kStages * kEntryBytes;
constexpr uint32_t kMaxChunkPages = 32 * kWarps;   // a page to a lane
constexpr int kMergeWarps = 16;
constexpr uint64_t kWaitLimitNs = 2000000000ull;
static_assert(kWarps * 8 * kHeadPitch * 4 <= kSmemBytes, "the merge reuses the ring");

struct AttnArgs {
    const __nv_bfloat16 *q;
    const uint8_t *pages;
    const float *scales;
    const __nv_bfloat16 *tail;
    const int32_t *page_table, *lens;
    float *out;
    float *part_o;    // [num_seqs][num_kv_heads][max_chunks][G][128], each chunk's own mean
    float2 *part_ml;  // [num_seqs][num_kv_heads][max_chunks][G] (maximum, sum), base 2
    int32_t *error;
    uint64_t q_stride, arena_pages;
    uint32_t num_seqs, num_kv_heads, G, max_pages, max_seq_len, chunk_pages, max_chunks;
    float scale_log2;
};

__device__ __forceinline__ bool len_ok(const AttnArgs &a, int32_t L)
{
    return L >= 0 && (uint32_t)L <= a.max_seq_len && ((uint32_t)L >> 4) <= a.max_pages;
}
__device__ __forceinline__ uint32_t chunks_of(const AttnArgs &a, int32_t L)
{
    const uint32_t n = (((uint32_t)L >> 4) + a.chunk_pages - 1) / a.chunk_pages;
    return n ? n : 1u;
}

// D += A(16x16, row) * B(16x8, col), fp16 inputs, fp32 accumulate.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same for 32 codes a row: the cache's own format against the query's digits.
template <uint32_t FMT>
__device__ __forceinline__ void mma_codes_16832(uint32_t (&d)[4], const uint4 &a, uint32_t b0,
                                                uint32_t b1)
{
    if constexpr (FMT == RT_KV8_E4M3)
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 "
            "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 "
            "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
template <uint32_t FMT>
__device__ __forceinline__ float sum_of(uint32_t d)
{
    return FMT == RT_KV8_E4M3 ? __uint_as_float(d) : (float)(int32_t)d;
}

// Four codes as two fp16 pairs, exactly.  s8: with its sign bit flipped a
// code c is the byte c + 128, and 0x6400 | byte is the fp16 1024 + byte.
template <uint32_t FMT>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t &lo, uint32_t &hi)
{
    if constexpr (FMT == RT_KV8_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\t"
            "mov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        const uint32_t u = w ^ 0x80808080u;
        const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
        uint32_t x = __byte_perm(u, 0x64646464u, 0x4140);
        uint32_t y = __byte_perm(u, 0x64646464u, 0x4342);
        __half2 a = __hsub2(*reinterpret_cast<__half2 *>(&x), bias);
        __half2 b = __hsub2(*reinterpret_cast<__half2 *>(&y), bias);
        lo = *reinterpret_cast<uint32_t *>(&a);
        hi = *reinterpret_cast<uint32_t *>(&b);
    }
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi)
{
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&v);
}
__device__ __forceinline__ float2 unpack_f16x2(uint32_t v)
{
    return __half22float2(*reinterpret_cast<__half2 *>(&v));
}

// State of one warp's online softmax over its tokens, base 2: lane (g, c) =
// (lane / 4, lane % 4) has the columns 2c and 2c + 1, and of O^T the dimensions
// 16 i + g (o[i][0], o[i][1]) and 16 i + 8 + g (o[i][2], o[i][3]).
struct Softmax {
    float m0, m1, l0, l1;
    float o[8][4];
    int v;  // O's unit is 2^(v - 14), the same in all lanes
};

__device__ __forceinline__ float exp2i(int e) { return __int_as_float((127 + e) << 23); }

// V scales within 2^kFar of the largest leave P 2^-(38 - kFar) of 1 in two fp16 terms.
constexpr int kFar = 8;

// Bring O to a unit of 2^(v - 14) where it is below.
__device__ __forceinline__ void raise_unit(Softmax &st, int v)
{
    if (v > st.v) {
        // from -110 the step can be 237: in two factors
        const float f = exp2i(max(st.v - v, -126)), f2 = exp2i(min(0, st.v - v + 126));
        st.v = v;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int u = 0; u < 4; u++)
                st.o[i][u] = st.o[i][u] * f * f2;
    }
}
// The exponent above a V scale (bits of a float, no sign).
__device__ __forceinline__ int unit_of(uint32_t scale) { return min((int)(scale >> 23) - 126, 127); }

// New maxima for the scores of NP times 16 tokens (rows g and g + 8); s becomes
// exp2(s - m), and what was summed before is brought to the new maxima.  A warp
// in which no maximum has moved leaves O alone (the factor is exactly 1).
template <int NP>
__device__ __forceinline__ void softmax_step(Softmax &st, float (&s)[NP][4])
{
    float x0 = fmaxf(s[0][0], s[0][2]), x1 = fmaxf(s[0][1], s[0][3]);
#pragma unroll
    for (int p = 1; p < NP; p++) {
        x0 = fmaxf(x0, fmaxf(s[p][0], s[p][2]));
        x1 = fmaxf(x1, fmaxf(s[p][1], s[p][3]));
    }
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xFFFFFFFFu, x0, off));
        x1 = fmaxf(x1, __shfl_xor_sync(0xFFFFFFFFu, x1, off));
    }
    x0 = fmaxf(x0, st.m0);
    x1 = fmaxf(x1, st.m1);
    if (__any_sync(0xFFFFFFFFu, x0 != st.m0 || x1 != st.m1)) {
        const float f0 = rt::fast_exp2(st.m0 - x0), f1 = rt::fast_exp2(st.m1 - x1);
        st.m0 = x0;
        st.m1 = x1;
        st.l0 *= f0;
        st.l1 *= f1;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            st.o[i][0] *= f0;
            st.o[i][1] *= f1;
            st.o[i][2] *= f0;
            st.o[i][3] *= f1;
        }
    }
#pragma unroll
    for (int p = 0; p < NP; p++) {
        s[p][0] = rt::fast_exp2(s[p][0] - x0);
        s[p][2] = rt::fast_exp2(s[p][2] - x0);
        s[p][1] = rt::fast_exp2(s[p][1] - x1);
        s[p][3] = rt::fast_exp2(s[p][3] - x1);
        st.l0 += s[p][0] + s[p][2];
        st.l1 += s[p][1] + s[p][3];
    }
}

// The query in the codes' own format.  With an element q scaled by a power of
// two, s8 writes it as an integer in digits of base 256, each in [-128, 127]; e4m3
// as a sum of terms t_i 2^-4i, each the nearest to 16 times what the ones before have
// left.  Products with codes are exact and their sums kept in fp32 or integers, so K
// needs no conversion: a word of it is an operand as it lies.
//
// Up to 4 heads to a KV head (DUP): 4 digits, the 8 columns of one product taking
// two of them (columns 0..3 the one, 4..7 the other) and a second product the
// other two.  More heads: a product to a digit, 4 of s8 and 3 of e4m3.  The digits
// hold bf16's 8 bits down to elements 2^-22 (s8), 2^-21 (e4m3, 4 terms) or 2^-17 (3)
// of the row's largest.  What the last product adds is 0 unless an element is below
// 2^-14 (s8, more heads) or 2^-13 (e4m3), so most rows skip it (`deep` is false).  Rows
// with elements that the digits do not hold take wide_step (`left`): K may be
// 0 where they are large, and then their score is what the small elements say.
template <uint32_t FMT, bool DUP>
struct Query {
    static constexpr int kDigits = DUP || FMT == RT_KV8_S8 ? 4 : 3, kProducts = DUP ? 2 : kDigits;
    static constexpr bool kSkips = FMT == RT_KV8_E4M3 || !DUP;  // the last product is `deep`'s
    // The row's largest element is brought to [2^kTop, 2^(kTop + 1)): a first digit of up
    // to 63 (s8, with room for the carry) or 256 (e4m3).
    static constexpr int kTop = FMT == RT_KV8_E4M3 ? 7 : 29;
    static constexpr int kFirstUnit = FMT == RT_KV8_E4M3 ? 0 : 24;  // of the first digit: a score's
    uint32_t f[kProducts][4][2];
    float k0, k1;  // factors of the scores of the lane's columns 2c and 2c + 1
    bool deep;     // the same in all lanes
    bool left;     // the digits do not hold the lane's elements

    // Row g's elements of the lane, and the bits of the row's largest.
    static __device__ __forceinline__ uint32_t fetch(const __nv_bfloat16 *row, bool has, uint2 (&qv)[8])
    {
        const int c = threadIdx.x & 3;
#pragma unroll
        for (int s = 0; s < 8; s++)
            qv[s] = has ? *reinterpret_cast<const uint2 *>(row + 16 * s + 4 * c) : make_uint2(0u, 0u);
        uint32_t top2 = 0;
#pragma unroll
        for (int s = 0; s < 8; s++)
            top2 = __vmaxu2(top2, __vmaxu2(qv[s].x & 0x7FFF7FFFu, qv[s].y & 0x7FFF7FFFu));
        uint32_t top = max(top2 & 0xFFFFu, top2 >> 16);
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        return max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    }
    static __device__ __forceinline__ int exponent(uint32_t top)
    {
        return min(max((int)(top >> 7) - 127, kTop - 126), 127);
    }

    // Lane (g, c) holds, of column g, dimensions 16 s + 4 c .. + 3 for s = 0..7, as
    // K's words hold them.
    __device__ __forceinline__ void load(const __nv_bfloat16 *row, bool has, float scale_log2)
    {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        uint2 qv[8];
        const uint32_t top = fetch(row, has, qv);
        const int e = exponent(top);
        const float up = exp2i(kTop - e);
        // a row with a NaN or an infinity has no digits: its scores become NaN
        const float down = top >= 0x7F80u ? __int_as_float(0x7FC00000) : exp2i(e - kTop + kFirstUnit);
        auto element = [&](int s, int u) {
            const uint32_t w = u & 2 ? qv[s].y : qv[s].x;
            return __uint_as_float(u & 1 ? w & 0xFFFF0000u : w << 16) * up;
        };
        left = false;
        if constexpr (FMT == RT_KV8_E4M3) {
            // the first term cut off after 4 bits, the second has the other 4
            bool small = false;
#pragma unroll
            for (int s = 0; s < 8; s++) {
                uint32_t t0 = 0, t1 = 0;
#pragma unroll
                for (int u = 0; u < 4; u += 2) {
                    const float x = element(s, u), y = element(s, u + 1);
                    const float xh = __uint_as_float(__float_as_uint(x) & 0xFFF00000u);
                    const float yh = __uint_as_float(__float_as_uint(y) & 0xFFF00000u);
                    // below 2^-6 a term is not exact
                    small |= (fabsf(x) < 0.015625f && x != 0.0f) || (fabsf(y) < 0.015625f && y != 0.0f);
                    t0 |= term(xh, yh) << (8 * u);
                    t1 |= term((x - xh) * 16.0f, (y - yh) * 16.0f) << (8 * u);
                }
                if constexpr (DUP) {
                    f[0][s >> 1][s & 1] = g < 4 ? t0 : t1;
                    f[1][s >> 1][s & 1] = 0u;
                } else {
                    f[0][s >> 1][s & 1] = t0;
                    f[1][s >> 1][s & 1] = t1;
                    f[2][s >> 1][s & 1] = 0u;
                }
            }
            deep = __any_sync(0xFFFFFFFFu, small);
            if (deep) {
#pragma unroll 1
                for (int half = 0; half < 2; half++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint32_t d[kDigits];
#pragma unroll
                        for (int i = 0; i < kDigits; i++)
                            d[i] = 0;
#pragma unroll
                        for (int u = 0; u < 4; u += 2) {
                            float x = half ? element(2 * j + 1, u) : element(2 * j, u);
                            float y = half ? element(2 * j + 1, u + 1) : element(2 * j, u + 1);
#pragma unroll
                            for (int i = 0; i < kDigits; i++) {
                                const uint32_t t = term(x, y);
                                uint32_t back;
                                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"((uint16_t)t));
                                const float2 v = unpack_f16x2(back);
                                x = (x - v.x) * 16.0f;
                                y = (y - v.y) * 16.0f;
                                d[i] |= t << (8 * u);
                            }
                            left |= x != 0.0f || y != 0.0f;
                        }
#pragma unroll
                        for (int i = 0; i < kProducts; i++) {
                            const uint32_t w = DUP ? (g < 4 ? d[2 * i] : d[(2 * i + 1) % kDigits]) : d[i];
                            if (half)
                                f[i][j][1] = w;
                            else
                                f[i][j][0] = w;
                        }
                    }
                }
            }
        } else {
            // A byte plus 128, carried on, less 128 is a digit: all of them at once.
            constexpr uint32_t kBias = 0x00808080u;
            // bytes of the first and second product's digits, as selectors
            const uint32_t s0 = DUP && g >= 4 ? 0x62u : 0x73u;
            const uint32_t s1 = DUP ? (g < 4 ? 0x51u : 0x40u) : 0x62u;
            uint32_t low = 0;
#pragma unroll
            for (int s = 0; s < 8; s++) {
                uint32_t n[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const float x = element(s, u);
                    const int whole = __float2int_rn(x);
                    left |= (float)whole != x;
                    n[u] = ((uint32_t)whole + kBias) ^ kBias;
                }
                auto digit = [&](uint32_t sel) {
                    return __byte_perm(__byte_perm(n[0], n[1], sel), __byte_perm(n[2], n[3], sel), 0x5410);
                };
                f[0][s >> 1][s & 1] = digit(s0);
                f[1][s >> 1][s & 1] = digit(s1);
                if constexpr (!DUP) {
                    f[2][s >> 1][s & 1] = digit(0x51u);
                    f[3][s >> 1][s & 1] = digit(0x40u);
                    low |= f[3][s >> 1][s & 1];
                }
            }
            deep = !DUP && __any_sync(0xFFFFFFFFu, low != 0u);
        }
        k0 = scale_log2 * __shfl_sync(0xFFFFFFFFu, down, 8 * c);
        k1 = scale_log2 * __shfl_sync(0xFFFFFFFFu, down, 8 * c + 4);
    }

    static __device__ __forceinline__ uint32_t term(float x, float y)
    {
        uint16_t t;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(t) : "f"(y), "f"(x));
        return t;
    }

    // Scores of the 16 tokens of a K plane, but for K's scale: x[0], x[1] columns 2c,
    // 2c + 1 of token g, x[2], x[3] of token g + 8.
    __device__ __forceinline__ void scores(const uint4 *k, float (&x)[4]) const
    {
        uint32_t d[kProducts][4];
#pragma unroll
        for (int i = 0; i < kProducts; i++)
            d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0u;
        constexpr int kFirst = kSkips ? kProducts - 1 : kProducts;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint4 w = k[j * 32];
#pragma unroll
            for (int i = 0; i < kFirst; i++)
                mma_codes_16832<FMT>(d[i], w, f[i][j][0], f[i][j][1]);
        }
        if (kFirst < kProducts && deep) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                mma_codes_16832<FMT>(d[kProducts - 1], k[j * 32], f[kProducts - 1][j][0],
                                     f[kProducts - 1][j][1]);
        }
        // in units of the first digit, so that k0 and k1 stay in range with the query
        constexpr float kBase = FMT == RT_KV8_E4M3 ? 0x1p-4f : 0x1p-8f;
        if constexpr (DUP) {
            // digits 0 and 2 in columns 0..3, 1 and 3 in 4..7
            const float one = threadIdx.x & 2 ? kBase : 1.0f, two = one * (kBase * kBase);
#pragma unroll
            for (int u = 0; u < 4; u++) {
                x[u] = fmaf(sum_of<FMT>(d[0][u]), one, sum_of<FMT>(d[1][u]) * two);
                x[u] += __shfl_xor_sync(0xFFFFFFFFu, x[u], 2);
            }
        } else {
#pragma unroll
            for (int u = 0; u < 4; u++) {
                x[u] = sum_of<FMT>(d[kProducts - 1][u]);
#pragma unroll
                for (int i = kProducts - 2; i >= 0; i--)
                    x[u] = fmaf(x[u], kBase, sum_of<FMT>(d[i][u]));
            }
        }
    }
};

// NP pages of codes with the scales sk of K and sv of V: scores, softmax, and
// P.V added to O.
template <uint32_t FMT, bool DUP, int NP>
__device__ __forceinline__ void pages_step(Softmax &st, const uint4 *(&blk)[NP],
                                           const Query<FMT, DUP> &q, const float (&sk)[NP],
                                           const float (&sv)[NP])
{
    float x[NP][4];
#pragma unroll
    for (int p = 0; p < NP; p++) {
        q.scores(blk[p], x[p]);
        const float f0 = sk[p] * q.k0, f1 = sk[p] * q.k1;
        x[p][0] *= f0;
        x[p][1] *= f1;
        x[p][2] *= f0;
        x[p][3] *= f1;
    }
    softmax_step<NP>(st, x);
    const bool low_half = DUP && (threadIdx.x & 2) != 0;  // columns 4..7
#pragma unroll
    for (int p = 0; p < NP; p++) {
        const float vf = sv[p] * exp2i(14 - st.v);
#pragma unroll
        for (int u = 0; u < 4; u++)
            x[p][u] *= vf;
        // P as two fp16 terms, transposed into the second product's B operand
        const uint32_t h0 = pack_f16x2(x[p][0], x[p][1]), h1 = pack_f16x2(x[p][2], x[p][3]);
        const float2 r0 = unpack_f16x2(h0), r1 = unpack_f16x2(h1);
        const uint32_t l0 = pack_f16x2(x[p][0] - r0.x, x[p][1] - r0.y);
        const uint32_t l1 = pack_f16x2(x[p][2] - r1.x, x[p][3] - r1.y);
        const uint32_t p0 = rt::movmatrix_trans(low_half ? l0 : h0);
        const uint32_t p1 = rt::movmatrix_trans(low_half ? l1 : h1);
        uint32_t q0 = 0, q1 = 0;
        if constexpr (!DUP) {
            q0 = rt::movmatrix_trans(l0);
            q1 = rt::movmatrix_trans(l1);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint4 w = blk[p][128 + j * 32];
            uint32_t f[4];
            decode4<FMT>(w.x, f[0], f[2]);
            decode4<FMT>(w.y, f[1], f[3]);
            mma_f16_16816(st.o[2 * j], f, p0, p1);
            if constexpr (!DUP)
                mma_f16_16816(st.o[2 * j], f, q0, q1);
            decode4<FMT>(w.z, f[0], f[2]);
            decode4<FMT>(w.w, f[1], f[3]);
            mma_f16_16816(st.o[2 * j + 1], f, p0, p1);
            if constexpr (!DUP)
                mma_f16_16816(st.o[2 * j + 1], f, q0, q1);
        }
    }
}

// Four codes as two bf16 pairs, exactly.
template <uint32_t FMT>
__device__ __forceinline__ void decode4_bf16(uint32_t w, uint32_t &lo, uint32_t &hi)
{
    if constexpr (FMT == RT_KV8_E4M3) {
        decode4<FMT>(w, lo, hi);
        const float2 a = unpack_f16x2(lo), b = unpack_f16x2(hi);
        lo = rt::pack_bf16x2(a.x, a.y);
        hi = rt::pack_bf16x2(b.x, b.y);
    } else {
        lo = rt::pack_bf16x2((float)(int8_t)w, (float)(int8_t)(w >> 8));
        hi = rt::pack_bf16x2((float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24));
    }
}

// One page where pages_step's forms do not hold the values: all in bf16, which has the
// range.  The query as it is, times a power of two, against decoded codes; P in three
// terms.  With DUP the first four columns carry all of them.  Rare, so it is kept short.
template <uint32_t FMT, bool DUP>
__device__ __forceinline__ void wide_step(Softmax &st, const uint4 *blk, const Query<FMT, DUP> &q,
                                          const __nv_bfloat16 *q_row, bool has_q, float sk, float sv)
{
    uint2 qv[8];
    const int e = Query<FMT, DUP>::exponent(Query<FMT, DUP>::fetch(q_row, has_q, qv));
    const float up = exp2i(Query<FMT, DUP>::kTop - Query<FMT, DUP>::kFirstUnit - e);
    float x[1][4] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint4 w = blk[j * 32];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const uint2 y = qv[2 * j + s];
            uint32_t f[4];
            decode4_bf16<FMT>(s ? w.z : w.x, f[0], f[2]);
            decode4_bf16<FMT>(s ? w.w : w.y, f[1], f[3]);
            rt::mma_bf16_16816(x[0], f, rt::pack_bf16x2(bf16_lo(y.x) * up, bf16_hi(y.x) * up),
                               rt::pack_bf16x2(bf16_lo(y.y) * up, bf16_hi(y.y) * up));
        }
    }
    const float f0 = sk * q.k0, f1 = sk * q.k1;
    x[0][0] *= f0;
    x[0][1] *= f1;
    x[0][2] *= f0;
    x[0][3] *= f1;
    softmax_step<1>(st, x);
    const float vf = DUP && (threadIdx.x & 2) ? 0.0f : sv * exp2i(14 - st.v);
    uint32_t p[3][2];
#pragma unroll
    for (int u = 0; u < 4; u++)
        x[0][u] *= vf;
#pragma unroll
    for (int k = 0; k < 3; k++) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t w = rt::pack_bf16x2(x[0][2 * u], x[0][2 * u + 1]);
            x[0][2 * u] -= bf16_lo(w);
            x[0][2 * u + 1] -= bf16_hi(w);
            p[k][u] = rt::movmatrix_trans(w);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint4 w = blk[128 + (i >> 1) * 32];
        uint32_t f[4];
        decode4_bf16<FMT>(i & 1 ? w.z : w.x, f[0], f[2]);
        decode4_bf16<FMT>(i & 1 ? w.w : w.y, f[1], f[3]);
#pragma unroll
        for (int k = 0; k < 3; k++)
            rt::mma_bf16_16816(st.o[i], f, p[k][0], p[k][1]);
    }
}

// The bf16 tail, n_tail tokens of [16][128] K and V rows in shared memory: the
// same products on bf16 fragments, P in three bf16 terms (24 bits).  Rows past
// the tail's end hold anything: their scores are -inf and their V bits cleared.
// With DUP the first four columns carry all three terms.
//
// V has bf16's range: P is at most 2^-5, so that 16 products stay in fp32's, and they
// are summed apart, for O's unit may be so large that P in it would lose digits; with
// a unit of at least 2^6 O holds their sum.
template <bool DUP>
__device__ __forceinline__ void tail_step(Softmax &st, const uint8_t *tk, const uint8_t *tv,
                                          const __nv_bfloat16 *q_row, bool has_q, uint32_t n_tail,
                                          float scale_log2)
{
    const int g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
    float x[1][4] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int s = 0; s < 8; s++) {
        const uint2 qv = has_q ? *reinterpret_cast<const uint2 *>(q_row + 16 * s + 4 * c)
                               : make_uint2(0u, 0u);
        const uint2 a0 = *reinterpret_cast<const uint2 *>(tk + g * 256 + (16 * s + 4 * c) * 2);
        const uint2 a1 = *reinterpret_cast<const uint2 *>(tk + (g + 8) * 256 + (16 * s + 4 * c) * 2);
        const uint32_t f[4] = {a0.x, a1.x, a0.y, a1.y};
        rt::mma_bf16_16816(x[0], f, qv.x, qv.y);
    }
    const bool in0 = (uint32_t)g < n_tail, in1 = (uint32_t)g + 8u < n_tail;
    x[0][0] = in0 ? x[0][0] * scale_log2 : -INFINITY;
    x[0][1] = in0 ? x[0][1] * scale_log2 : -INFINITY;
    x[0][2] = in1 ? x[0][2] * scale_log2 : -INFINITY;
    x[0][3] = in1 ? x[0][3] * scale_log2 : -INFINITY;
    softmax_step<1>(st, x);
    uint32_t p[3][2];
    raise_unit(st, 20);
    const float unit = DUP && (threadIdx.x & 2) ? 0.0f : 0x1p-5f;
    const float back = exp2i(19 - st.v);
#pragma unroll
    for (int u = 0; u < 4; u++)
        x[0][u] *= unit;
#pragma unroll
    for (int k = 0; k < 3; k++) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t w = rt::pack_bf16x2(x[0][2 * u], x[0][2 * u + 1]);
            x[0][2 * u] -= __uint_as_float(w << 16);
            x[0][2 * u + 1] -= __uint_as_float(w & 0xFFFF0000u);
            p[k][u] = rt::movmatrix_trans(w);
        }
    }
    // lane c's tokens: 2c, 2c + 1 and 2c + 8, 2c + 9
    auto keep = [&](uint32_t t) {
        return (t < n_tail ? 0xFFFFu : 0u) | (t + 1u < n_tail ? 0xFFFF0000u : 0u);
    };
    const uint32_t keep0 = keep(2 * c), keep1 = keep(2 * c + 8);
    const uint16_t *v16 = reinterpret_cast<const uint16_t *>(tv);
    auto pair = [&](uint32_t t, uint32_t d) {
        return (uint32_t)v16[t * 128 + d] | (uint32_t)v16[(t + 1) * 128 + d] << 16;
    };
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t d0 = 16 * i + g;
        const uint32_t f[4] = {pair(2 * c, d0) & keep0, pair(2 * c, d0 + 8) & keep0,
                               pair(2 * c + 8, d0) & keep1, pair(2 * c + 8, d0 + 8) & keep1};
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 3; k++)
            rt::mma_bf16_16816(d, f, p[k][0], p[k][1]);
#pragma unroll
        for (int u = 0; u < 4; u++)
            st.o[i][u] = fmaf(d[u], back, st.o[i][u]);
    }
}

// One CTA per (sequence, KV head, chunk of pages), the pairs of pages dealt out to
// its warps.  Each warp has a ring of entries that bulk copies fill: the K and V
// codes of two pages for the KV head, or the tail's K and V rows.  The CTAs are
// handed out by the hardware, chunk by chunk of the whole batch: warps differ by
// 10% in the bandwidth they get, and equal shares dealt out beforehand end when
// the slowest does.
//
// Math, two pages at a time: S^T = K.Q^T with the codes as they are and the query
// in digits (Query), O^T += V^T.P^T on m16n8k16 with the codes in fp16, exactly;
// 16 tokens (or 16 dimensions) as rows, the KV group's heads as columns.  K's
// scale multiplies the scores in fp32.  V's multiplies P: with O's unit 2^(v -
// 14), v the exponent above the largest scale of the warp's pages, P times scale
// fills fp16's range from 2^14 down to 2^-24, and two fp16 terms of it are off by
// 2^-38 of the largest scale or 2^-22 of their own value.  With up to 4 heads (DUP) columns
// 4..7 repeat columns 0..3 and carry P's low terms, so one product covers both (64
// sequences of up to 4,096, 4 heads, e4m3: 59 us, without 64; s8: 59 and 60).
template <uint32_t FMT, bool DUP>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) kv8_decode_kernel(const AttnArgs a)
{
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kWarps][kStages];
    __shared__ float2 ml[kWarps][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    const uint32_t H = a.num_kv_heads, G = a.G;
    rt::grid_dep_launch();
    const uint32_t h = blockIdx.x % H, rest = blockIdx.x / H;
    const uint32_t b = rest % a.num_seqs, chunk = rest / a.num_seqs;
    const uint32_t p0 = chunk * a.chunk_pages;
    // Lane l has page l & 1 of the warp's pair l / 2: pair warp + kWarps (l / 2) of the
    // chunk.  Its id is read beside the length, which then says whether it counts.
    const uint32_t my_page = p0 + 2u * ((uint32_t)warp + kWarps * ((uint32_t)lane >> 1)) + (lane & 1);
    const bool in_table = my_page < a.max_pages && my_page < p0 + a.chunk_pages;
    const int32_t L = a.lens[b];
    const int32_t id = in_table ? a.page_table[(uint64_t)b * a.max_pages + my_page] : -1;
    const uint32_t head = DUP ? (uint32_t)g & 3u : (uint32_t)g;
    const bool has_q = head < G;
    const __nv_bfloat16 *q_row = a.q + (uint64_t)b * a.q_stride + ((uint64_t)h * G + head) * 128u;

    if (!len_ok(a, L)) {
        if (threadIdx.x == 0 && chunk == 0)
            flag_error(a.error, kErrLen);
        return;
    }
    const uint32_t n_chunks = chunks_of(a, L);
    if (chunk >= n_chunks)
        return;
    const uint32_t p1 = min((uint32_t)L >> 4, p0 + a.chunk_pages);
    const uint32_t pairs = (p1 - p0 + 1u) / 2u;
    const uint32_t n_pairs = (pairs + kWarps - 1u - (uint32_t)warp) / kWarps;
    // the tail goes to the first warp with the fewest pairs
    const uint32_t n_tail =
        chunk + 1 == n_chunks && (uint32_t)warp == pairs % kWarps ? (uint32_t)L & 15u : 0u;
    const uint32_t n_entries = n_pairs + (n_tail ? 1u : 0u);

    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < kStages; s++)
            rt::mbar_init(rt::smem_u32(&bars[warp][s]), 1);
        rt::mbar_fence_init();
    }
    __syncwarp();
    const bool mine = in_table && my_page < p1, ok = mine && id >= 0 && (uint64_t)id < a.arena_pages;
    if (mine && !ok)
        flag_error(a.error, kErrPage);
    const uint32_t have = __ballot_sync(0xFFFFFFFFu, ok);  // pages that are read
    const uint64_t block = ok ? (uint64_t)id * H + h : 0u;
    const uint32_t ring = rt::smem_u32(smem) + (uint32_t)warp * kStages * kEntryBytes;

    uint32_t issued = 0;
    auto issue = [&]() {
        const uint32_t s = issued % kStages;
        const uint32_t bar = rt::smem_u32(&bars[warp][s]), dst = ring + s * kEntryBytes;
        if (issued < n_pairs) {
            if ((uint32_t)lane >> 1 == issued) {
                const uint32_t both = have >> (2u * issued) & 3u, odd = lane & 1;
                if (!odd && both)
                    rt::mbar_arrive_expect_tx(bar, both == 3u ? 2u * kBlockBytes : kBlockBytes);
                if (ok)
                    rt::bulk_load(dst + odd * kBlockBytes, a.pages + block * kBlockBytes, kBlockBytes, bar);
            }
        } else if (lane == 0) {
            const __nv_bfloat16 *t = a.tail + rt_page_elem_offset(b, h, 0, 0, H);
            rt::mbar_arrive_expect_tx(bar, n_tail * 512u);
            rt::bulk_load(dst, t, n_tail * 256u, bar);
            rt::bulk_load(dst + kBlockBytes, t + 2048, n_tail * 256u, bar);
        }
        issued++;
    };
    while (issued < (uint32_t)kStages && issued < n_entries)
        issue();
    const float2 sc = ok ? *reinterpret_cast<const float2 *>(a.scales + block * 2u) : make_float2(0.f, 0.f);

    Query<FMT, DUP> q;
    q.load(q_row, has_q, a.scale_log2);
    Softmax st;
    st.m0 = st.m1 = -INFINITY;
    st.l0 = st.l1 = 0.0f;
    // O's unit holds the warp's largest V scale.  Where another is far below, P would lose
    // digits of what counts in dimensions that the large ones leave at 0: wide_step.
    const uint32_t sv_bits = __float_as_uint(sc.y) & 0x7FFFFFFFu;
    st.v = max(-110, unit_of(__reduce_max_sync(0xFFFFFFFFu, sv_bits)));
    const bool wide = __any_sync(0xFFFFFFFFu, q.left || (sv_bits != 0u && st.v - unit_of(sv_bits) > kFar));
#pragma unroll
    for (int i = 0; i < 8; i++)
        st.o[i][0] = st.o[i][1] = st.o[i][2] = st.o[i][3] = 0.0f;

    const uint8_t *slots = smem + (uint32_t)warp * kStages * kEntryBytes;
    uint32_t phases = 0, limit = n_entries;
    for (uint32_t i = 0; i < issued; i++) {
        const uint32_t s = i % kStages;
        const uint32_t both = i < n_pairs ? have >> (2u * i) & 3u : 4u;
        if (both) {
            // After an expired wait nothing is issued any more; what is in flight, this
            // entry included, is waited for, again with a limit.
            const uint32_t bar = rt::smem_u32(&bars[warp][s]), phase = (phases >> s) & 1u;
            if (!__all_sync(0xFFFFFFFFu, rt::mbar_wait_bounded(bar, phase, kWaitLimitNs))) {
                if (lane == 0)
                    flag_error(a.error, kErrTimeout);
                limit = 0;
                rt::mbar_wait_bounded(bar, phase, kWaitLimitNs);
            }
            phases ^= 1u << s;
            const uint8_t *base = slots + s * kEntryBytes;
            const uint4 *blk0 = reinterpret_cast<const uint4 *>(base) + lane;
            const uint4 *blk1 = blk0 + kBlockBytes / 16;
            if (both != 4u && wide) {
#pragma unroll 1
                for (int k = 2 * i; k < 2 * (int)i + 2; k++) {
                    const float sk = __shfl_sync(0xFFFFFFFFu, sc.x, k), sv = __shfl_sync(0xFFFFFFFFu, sc.y, k);
                    if (have >> k & 1u)
                        wide_step<FMT, DUP>(st, k & 1 ? blk1 : blk0, q, q_row, has_q, sk, sv);
                }
            } else if (both == 3u) {
                const uint4 *blk[2] = {blk0, blk1};
                const float sk[2] = {__shfl_sync(0xFFFFFFFFu, sc.x, 2 * i),
                                     __shfl_sync(0xFFFFFFFFu, sc.x, 2 * i + 1)};
                const float sv[2] = {__shfl_sync(0xFFFFFFFFu, sc.y, 2 * i),
                                     __shfl_sync(0xFFFFFFFFu, sc.y, 2 * i + 1)};
                pages_step<FMT, DUP, 2>(st, blk, q, sk, sv);
            } else if (both == 4u) {
                tail_step<DUP>(st, base, base + kBlockBytes, q_row, has_q, n_tail, a.scale_log2);
            } else {
                const uint4 *blk[1] = {both == 1u ? blk0 : blk1};
                const int k = 2 * i + (both == 1u ? 0 : 1);
                const float sk[1] = {__shfl_sync(0xFFFFFFFFu, sc.x, k)};
                const float sv[1] = {__shfl_sync(0xFFFFFFFFu, sc.y, k)};
                pages_step<FMT, DUP, 1>(st, blk, q, sk, sv);
            }
            __syncwarp();  // every lane has read the slot before it is filled again
        }
        if (issued < limit)
            issue();
    }

    // Merge the warps: sums over a column's lanes, then all states through shared memory.
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
        st.l0 += __shfl_xor_sync(0xFFFFFFFFu, st.l0, off);
        st.l1 += __shfl_xor_sync(0xFFFFFFFFu, st.l1, off);
    }
    if (g == 0) {
        ml[warp][2 * c] = make_float2(st.m0, st.l0);
        ml[warp][2 * c + 1] = make_float2(st.m1, st.l1);
    }
    __syncthreads();  // all slots have been read
    float *merge = reinterpret_cast<float *>(smem);
    // Divided by the sum here: a mean of V is in fp32's range where a sum may not be.
    const uint64_t row = (uint64_t)b * H + h, slot = row * a.max_chunks + chunk;
    {
        const float unit = exp2i(st.v - 14);
        // all maxima -infinity: no page was read, or all scores were NaN
        auto weight = [&](uint32_t col) {
            float M = -INFINITY, l = 0.0f, own = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++)
                M = fmaxf(M, ml[w][col].x);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float x = M == -INFINITY ? 1.0f : rt::fast_exp2(ml[w][col].x - M);
                l = fmaf(ml[w][col].y, x, l);
                own = w == warp ? x : own;
            }
            if (n_chunks > 1 && warp == 0 && g == 0 && col < G)
                a.part_ml[slot * G + col] = make_float2(M, l);
            return l == 0.0f ? 0.0f : __fdividef(own, l);
        };
        const float w0 = weight(2 * c), w1 = weight(2 * c + 1);
        float *to = merge + ((size_t)warp * 8 + 2 * c) * kHeadPitch + g;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            to[16 * i] = st.o[i][0] * w0 * unit;
            to[16 * i + kHeadPitch] = st.o[i][1] * w1 * unit;
            to[16 * i + 8] = st.o[i][2] * w0 * unit;
            to[16 * i + 8 + kHeadPitch] = st.o[i][3] * w1 * unit;
        }
    }
    __syncthreads();
    float *means = n_chunks == 1 ? a.out + row * G * 128u : a.part_o + slot * G * 128u;
    for (uint32_t r = warp; r < G; r += kWarps) {  // a warp to a head, four dimensions a lane
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
#pragma unroll
            for (uint32_t col = r; col < 8u; col += DUP ? 4u : 8u) {
                const float4 o = *reinterpret_cast<const float4 *>(merge + (w * 8 + col) * kHeadPitch + 4 * lane);
                acc.x += o.x;
                acc.y += o.y;
                acc.z += o.z;
                acc.w += o.w;
            }
        }
        reinterpret_cast<float4 *>(means + r * 128u)[lane] = acc;
    }
}

// Log-sum-exp merge of the chunks of sequences that have several.  It waits on
// memory alone, so each warp has U chunks' loads in flight, a lane four dimensions
// of each.
//
// WARPS = 1: one warp per (row, head), for batches of many rows and few chunks.  Else
// one CTA per (row, head), its warps taking the chunks in turn.
template <int WARPS, int U>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : WARPS * 32) kv8_merge_kernel(const AttnArgs a)
{
    __shared__ float2 warp_ml[WARPS];
    __shared__ float4 warp_o[WARPS][32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.G;
    const uint64_t item = WARPS == 1 ? blockIdx.x * 8ull + warp : blockIdx.x;
    const bool has_row = item < (uint64_t)a.num_seqs * a.num_kv_heads * G;
    const uint64_t row = item / G;
    const uint32_t sub = WARPS == 1 ? 0u : warp;
    const int32_t L = has_row ? a.lens[row / a.num_kv_heads] : 0;
    // Every CTA waits, also those without a part in it: this kernel's end stands for
    // both kernels' to what follows.
    rt::grid_dep_wait();
    if (!len_ok(a, L))
        return;
    const uint32_t n = chunks_of(a, L);
    if (n < 2)
        return;
    const uint64_t first = row * a.max_chunks * G + item % G;
    // all maxima -infinity: no page was read, or all scores were NaN
    auto weight = [](float x, float top) { return top == -INFINITY ? 1.0f : rt::fast_exp2(x - top); };
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t k0 = sub; k0 < n; k0 += WARPS * U) {
        float2 s[U];
        float4 o[U];
        float top = m;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t k = k0 + u * WARPS;
            s[u] = make_float2(-INFINITY, 0.0f);
            o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < n) {
                const uint64_t slot = first + (uint64_t)k * G;
                s[u] = a.part_ml[slot];
                o[u] = reinterpret_cast<const float4 *>(a.part_o + slot * 128u)[lane];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            top = fmaxf(top, s[u].x);
        // weights that sum to 1, so that acc stays a mean
        float w0 = l * weight(m, top), wt[U];
        l = w0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            wt[u] = s[u].y * weight(s[u].x, top);
            l += wt[u];
        }
        const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
        m = top;
        w0 *= inv;
        acc.x *= w0;
        acc.y *= w0;
        acc.z *= w0;
        acc.w *= w0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            wt[u] *= inv;
            acc.x += o[u].x * wt[u];
            acc.y += o[u].y * wt[u];
            acc.z += o[u].z * wt[u];
            acc.w += o[u].w * wt[u];
        }
    }
    if constexpr (WARPS == 1) {
        reinterpret_cast<float4 *>(a.out + item * 128u)[lane] = acc;
    } else {
        warp_o[warp][lane] = acc;
        if (lane == 0)
            warp_ml[warp] = make_float2(m, l);
        __syncthreads();
        if (threadIdx.x < 128) {
            float top = -INFINITY, sum = 0.0f, den = 0.0f, wt[WARPS];
#pragma unroll
            for (int w = 0; w < WARPS; w++)
                top = fmaxf(top, warp_ml[w].x);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                wt[w] = warp_ml[w].y * weight(warp_ml[w].x, top);
                den += wt[w];
            }
            const float inv = den == 0.0f ? 0.0f : __fdividef(1.0f, den);
#pragma unroll
            for (int w = 0; w < WARPS; w++)
                sum += reinterpret_cast<const float *>(warp_o[w])[threadIdx.x] * (wt[w] * inv);
            a.out[item * 128u + threadIdx.x] = sum;
        }
    }
}

// Pages per item.  Where all rows' pages make two items to an SM of up to 128 pages
// each, so many: fewer leave bandwidth idle, more are merged longer (1 x 131,071
// tokens, 4 KV heads: 29 us, with 48 pages an item 36, 32: 39).  Larger batches have
// more items than fit at once, and an item's start and end cost about as much as 14
// pages: 96 pages.  Of nine batches of 16 to 64 sequences of up to 4,096 or 8,192 tokens,
// 8 KV heads, in both formats, eight are in this class, and 96 is the best of 16, 32,
// 48, 64, 96 and 128 or within 3% of it (64 of 128..4,096: 59 us, 32 pages 66, 128 62;
// 16 of 128..8,192: 30, 32 pages 38, 128 32) but for one: 32 of 2,048..4,096, 1.4 turns
// of the GPU, take 44 and with 128 pages 40, which cost 64 such sequences 80 for 75.
// 16 of 2,048..4,096 have two items of 128 to an SM: 26 us in s8, 28 in e4m3, 25 and 27
// with 96.
struct AttnPlan {
    uint32_t chunk_pages, max_chunks;
    size_t part_o, part_ml;
};

AttnPlan plan_of(const rt_kv8_attn_params_t *p)
{
    AttnPlan r;
    const uint64_t rows = (uint64_t)p->num_seqs * p->num_kv_heads, pages = p->max_seq_len >> 4;
    uint64_t c = p->chunk_pages;
    if (!c) {
        const uint64_t per_row = rows ? 2ull * (uint64_t)rt::num_sms() / rows : 1u;
        c = per_row ? (pages + per_row - 1) / per_row : kMaxChunkPages + 1u;
        c = c > kMaxChunkPages ? 96u : c < 16u ? 16u : c;
    }
    r.chunk_pages = (uint32_t)((c + 1) / 2 * 2);  // whole pairs
    r.max_chunks = (uint32_t)((pages + r.chunk_pages - 1) / r.chunk_pages);
    r.max_chunks = r.max_chunks ? r.max_chunks : 1u;
    const size_t parts = r.max_chunks > 1u ? (size_t)p->num_seqs * p->num_q_heads * r.max_chunks : 0u;
    r.part_o = parts * 128u * sizeof(float);
    r.part_ml = parts * sizeof(float2);
    return r;
}

bool format_ok(uint32_t format) { return format == RT_KV8_E4M3 || format == RT_KV8_S8; }

int check_attn(const rt_kv8_attn_params_t *p)
{
    if (!p) {
        rt::set_error("kv8_decode_attention: null params");
        return RT_EINVAL;
    }
    if (!p->num_kv_heads || !p->num_q_heads || p->num_q_heads % p->num_kv_heads ||
        p->num_q_heads / p->num_kv_heads > 8u || !format_ok(p->format) ||
        p->chunk_pages > kMaxChunkPages || !(fabsf(p->scale) <= 2e38f) ||
        p->q_stride < (uint64_t)p->num_q_heads * 128u || p->q_stride % 8u ||
        p->max_seq_len > 0x7FFFFFFFu || (p->max_seq_len >> 4) > p->max_pages_per_seq) {
        rt::set_error("kv8_decode_attention: 1..8 query heads to a KV head (%u / %u), format e4m3 "
                      "or s8, q_stride >= num_q_heads * 128 and a multiple of 8, chunk_pages <= "
                      "%u, max_seq_len / 16 <= max_pages_per_seq",
                      p->num_q_heads, p->num_kv_heads, kMaxChunkPages);
        return RT_EINVAL;
    }
    if ((uint64_t)p->num_q_heads * p->num_seqs > 0x7FFFFFFFull ||
        (uint64_t)p->num_kv_heads * p->num_seqs * plan_of(p).max_chunks > 0x7FFFFFFFull) {
        rt::set_error("kv8_decode_attention: more than 2^31 - 1 work items");
        return RT_EINVAL;
    }
    return RT_OK;
}

}  // namespace

extern "C" int rt_kv8_append(const rt_kv8_append_params_t *p, const void *k, const void *v,
                             const int32_t *cu_tokens, const int32_t *seq_lens,
                             const int32_t *page_table, void *pages, float *scales, void *tail,
                             int32_t *error, void *stream)
{
    if (!p) {
        rt::set_error("kv8_append: null params");
        return RT_EINVAL;
    }
    if (p->num_seqs == 0 || p->num_tokens == 0)
        return RT_OK;
    const uint64_t row = (uint64_t)p->num_kv_heads * 128u;
    if (!p->num_kv_heads || !format_ok(p->format) || p->dtype > RT_DTYPE_BF16 ||
        p->k_stride < row || p->v_stride < row || p->k_stride % 8u || p->v_stride % 8u ||
        p->num_tokens > 0x7FFFFFFFu || p->num_seqs > 0x7FFFFFFFu) {
        rt::set_error("kv8_append: num_kv_heads > 0, format e4m3 or s8, dtype f32 or bf16, strides "
                      ">= num_kv_heads * 128 and multiples of 8");
        return RT_EINVAL;
    }
    // no page table or no arena: none of it is read
    if (!k || !v || !cu_tokens || !seq_lens || (!page_table && p->max_pages_per_seq) ||
        ((!pages || !scales) && p->arena_pages) || !tail) {
        rt::set_error("kv8_append: null argument");
        return RT_EINVAL;
    }
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)pages | (uintptr_t)tail) & 15u ||
        ((uintptr_t)cu_tokens | (uintptr_t)seq_lens | (uintptr_t)page_table | (uintptr_t)scales |
         (uintptr_t)error) & 3u) {
        rt::set_error("kv8_append: k, v, pages and tail must be 16-byte aligned, the rest 4-byte");
        return RT_EINVAL;
    }
    AppendArgs a;
    a.k = k;
    a.v = v;
    a.cu = cu_tokens;
    a.lens = seq_lens;
    a.page_table = page_table;
    a.pages = static_cast<uint8_t *>(pages);
    a.scales = scales;
    a.tail = static_cast<__nv_bfloat16 *>(tail);
    a.error = error;
    a.k_stride = p->k_stride;
    a.v_stride = p->v_stride;
    a.arena_pages = p->arena_pages;
    a.num_seqs = p->num_seqs;
    a.num_kv_heads = p->num_kv_heads;
    a.num_tokens = p->num_tokens;
    a.max_pages = p->max_pages_per_seq;
    const uint64_t units = (uint64_t)p->num_tokens / 16u + p->num_seqs;
    a.n_items = units * p->num_kv_heads;
    uint64_t blocks = (a.n_items + kAppendWarps - 1) / kAppendWarps;
    // Persistent warps hide the search behind the loads; a short call (many units with
    // a tail's few tokens alone) is over sooner with a warp to an item (512 sequences
    // of one token, 8 KV heads: 8.3 against 10.6 us).
    const uint64_t sms = (uint64_t)rt::num_sms();
    if (blocks > 6u * sms)
        blocks = 2u * sms;
    const dim3 grid((unsigned)blocks), block(kAppendWarps * 32);
    cudaStream_t s = (cudaStream_t)stream;
    const bool f32 = p->dtype == RT_DTYPE_F32;
    if (p->format == RT_KV8_E4M3) {
        if (f32)
            kv8_append_kernel<RT_KV8_E4M3, true><<<grid, block, 0, s>>>(a);
        else
            kv8_append_kernel<RT_KV8_E4M3, false><<<grid, block, 0, s>>>(a);
    } else {
        if (f32)
            kv8_append_kernel<RT_KV8_S8, true><<<grid, block, 0, s>>>(a);
        else
            kv8_append_kernel<RT_KV8_S8, false><<<grid, block, 0, s>>>(a);
    }
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? RT_OK : rt::cuda_fail(e, "kv8_append: launch");
}

extern "C" size_t rt_kv8_attn_workspace_bytes(const rt_kv8_attn_params_t *p)
{
    if (check_attn(p) != RT_OK)
        return 0;
    const AttnPlan r = plan_of(p);
    return r.part_o + r.part_ml;
}

extern "C" int rt_kv8_decode_attention(const rt_kv8_attn_params_t *p, const void *q,
                                       const void *pages, const float *scales, const void *tail,
                                       const int32_t *page_table, const int32_t *seq_lens,
                                       float *out, void *workspace, size_t workspace_bytes,
                                       int32_t *error, void *stream)
{
    const int rc = check_attn(p);
    if (rc != RT_OK)
        return rc;
    if (p->num_seqs == 0)
        return RT_OK;
    if (!q || ((!pages || !scales) && p->arena_pages) || !tail ||
        (!page_table && p->max_pages_per_seq) || !seq_lens || !out) {
        rt::set_error("kv8_decode_attention: null argument");
        return RT_EINVAL;
    }
    if (((uintptr_t)q | (uintptr_t)pages | (uintptr_t)tail | (uintptr_t)out | (uintptr_t)workspace) & 15u ||
        (uintptr_t)scales & 7u ||
        ((uintptr_t)page_table | (uintptr_t)seq_lens | (uintptr_t)error) & 3u) {
        rt::set_error("kv8_decode_attention: q, pages, tail, out and workspace must be 16-byte "
                      "aligned, scales 8-byte, the rest 4-byte");
        return RT_EINVAL;
    }
    const AttnPlan plan = plan_of(p);
    const size_t need = plan.part_o + plan.part_ml;
    if (need && (!workspace || workspace_bytes < need)) {
        rt::set_error("kv8_decode_attention: workspace of %zu bytes needed, %zu given", need,
                      workspace ? workspace_bytes : (size_t)0);
        return RT_ENOMEM;
    }
    AttnArgs a;
    a.q = static_cast<const __nv_bfloat16 *>(q);
    a.pages = static_cast<const uint8_t *>(pages);
    a.scales = scales;
    a.tail = static_cast<const __nv_bfloat16 *>(tail);
    a.page_table = page_table;
    a.lens = seq_lens;
    a.out = out;
    a.error = error;
    a.q_stride = p->q_stride;
    a.arena_pages = p->arena_pages;
    a.num_seqs = p->num_seqs;
    a.num_kv_heads = p->num_kv_heads;
    a.G = p->num_q_heads / p->num_kv_heads;
    a.max_pages = p->max_pages_per_seq;
    a.max_seq_len = p->max_seq_len;
    a.chunk_pages = plan.chunk_pages;
    a.max_chunks = plan.max_chunks;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    a.part_o = reinterpret_cast<float *>(ws);
    a.part_ml = reinterpret_cast<float2 *>(ws + plan.part_o);
    cudaStream_t s = (cudaStream_t)stream;
    void (*fn)(AttnArgs) = nullptr;
    if (p->format == RT_KV8_E4M3)
        fn = a.G <= 4 ? kv8_decode_kernel<RT_KV8_E4M3, true> : kv8_decode_kernel<RT_KV8_E4M3, false>;
    else
        fn = a.G <= 4 ? kv8_decode_kernel<RT_KV8_S8, true> : kv8_decode_kernel<RT_KV8_S8, false>;
    cudaError_t e = cudaFuncSetAttribute((const void *)fn,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess)
        return rt::cuda_fail(e, "kv8_decode_attention: shared memory");
    fn<<<p->num_kv_heads * p->num_seqs * plan.max_chunks, kWarps * 32, kSmemBytes, s>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess)
        return rt::cuda_fail(e, "kv8_decode_attention: launch");
    if (plan.max_chunks > 1u) {
        // a programmatic dependent: its CTAs are in place when the last items end
        const uint32_t items = p->num_seqs * p->num_q_heads;
        // A warp to a row once rows outweigh chunks: 24 sequences of 8,192 tokens (768 rows,
        // 6 chunks) 76 us, a CTA each 83; 4 of 32,768 (128 rows, 22 chunks) 58 against 52.
        const bool many = items >= 32u * plan.max_chunks;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(many ? (items + 7u) / 8u : items);
        cfg.blockDim = dim3((many ? 8 : kMergeWarps) * 32);
        cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = many ? cudaLaunchKernelEx(&cfg, kv8_merge_kernel<1, 4>, (const AttnArgs)a)
                 : cudaLaunchKernelEx(&cfg, kv8_merge_kernel<kMergeWarps, 14>, (const AttnArgs)a);
        if (e != cudaSuccess)
            return rt::cuda_fail(e, "kv8_decode_attention: merge launch");
    }
    return RT_OK;
}
