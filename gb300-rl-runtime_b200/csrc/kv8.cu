// kv8.cu - the KV cache in 8 bits: append (quantise) and paged GQA decode
// attention over it, for sm_100a.
//
// A (page, KV head, plane) tile of 16 tokens x 128 dimensions is stored as
// code bytes with one fp32 scale; a sequence's unfinished page stays in bf16
// ("tail").  Layout: kv_layout.h; contract: rlrt.h.
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
    uint64_t n_warps;  // units x heads x 2 planes
};

constexpr int kAppendWarps = 8;

// Four consecutive elements of a token's row, as two bf16 pairs.
template <bool F32>
__device__ __forceinline__ uint2 load4(const void *base, uint64_t elem)
{
    if constexpr (F32) {
        const float4 f = __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(base) + elem));
        return make_uint2(rt::pack_bf16x2(f.x, f.y), rt::pack_bf16x2(f.z, f.w));
    } else {
        return __ldcs(reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + elem));
    }
}

template <uint32_t FMT>
__device__ __forceinline__ uint32_t quantise4(uint2 x, float scale)
{
    const float f[4] = {__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xFFFF0000u),
                        __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xFFFF0000u)};
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        y[i] = __fdiv_rn(f[i], scale);
    if constexpr (FMT == RT_KV8_E4M3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y[1]), "f"(y[0]));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y[3]), "f"(y[2]));
        return (uint32_t)lo | (uint32_t)hi << 16;
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = __float2int_rn(fminf(fmaxf(y[i], -127.0f), 127.0f));
            w |= ((uint32_t)c & 0xFFu) << (8 * i);
        }
        return w;
    }
}

// One warp per (unit, KV head, plane); a unit is one page of one sequence that
// the call touches.  Sequence b owns the units from cu[b] / 16 + 2 b on: n new
// tokens behind any remainder touch at most n / 16 + 2 pages, so the ranges
// are disjoint and a unit finds its sequence by a binary search of cu, without
// a scan over the batch.  Lane i holds dimensions 4 i .. 4 i + 3 of all 16
// tokens, so a tile is read once, in whole rows, and the maximum, the codes
// and the 4 x 4 byte transposes of V stay in registers.  The sequence's first
// unit alone reads and writes its tail, each lane the dimensions that it owns:
// the old tokens are in registers before the new ones are stored.
template <uint32_t FMT, bool F32>
__global__ void __launch_bounds__(kAppendWarps * 32) kv8_append_kernel(const AppendArgs a)
{
    __shared__ __align__(16) uint32_t stage[kAppendWarps][kPlane / 4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t gid = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x;
    if (gid < a.num_seqs && (a.cu[gid] < 0 || a.cu[gid + 1] < a.cu[gid] ||
                             (uint32_t)a.cu[gid + 1] > a.num_tokens))
        flag_error(a.error, kErrCu);
    const uint64_t item = gid >> 5;
    if (item >= a.n_warps)
        return;
    const uint32_t plane = (uint32_t)(item & 1u);
    const uint32_t h = (uint32_t)((item >> 1) % a.num_kv_heads);
    const int64_t unit = (int64_t)((item >> 1) / a.num_kv_heads);

    uint32_t lo = 0, hi = a.num_seqs;  // the last b with cu[b] / 16 + 2 b <= unit
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) >> 1;
        if ((int64_t)(a.cu[mid] >> 4) + 2 * (int64_t)mid <= unit)
            lo = mid;
        else
            hi = mid;
    }
    const uint32_t b = lo;
    const int64_t c0 = a.cu[b], c1 = a.cu[b + 1], j = unit - ((c0 >> 4) + 2 * (int64_t)b);
    if (j < 0 || c0 < 0 || c1 <= c0 || c1 > (int64_t)a.num_tokens)
        return;
    const int64_t L0 = a.lens[b], L1 = L0 + (c1 - c0);
    if (L0 < 0 || (L1 >> 4) > (int64_t)a.max_pages) {
        if (lane == 0)
            flag_error(a.error, kErrLen);
        return;
    }
    const int64_t page = (L0 >> 4) + j, first = page << 4;
    const bool full = first + 16 <= L1;
    if (!full && j > 0)
        return;
    const void *src = plane ? a.v : a.k;
    const uint64_t stride = plane ? a.v_stride : a.k_stride;
    const uint64_t col = (uint64_t)h * 128u + 4u * lane;
    __nv_bfloat16 *tail = a.tail + rt_page_elem_offset(b, h, plane, 0, a.num_kv_heads) + 4 * lane;

    if (full) {
        uint2 x[16];
#pragma unroll
        for (int t = 0; t < 16; t++) {
            const int64_t pos = first + t;
            x[t] = pos < L0 ? *reinterpret_cast<const uint2 *>(tail + t * 128)
                            : load4<F32>(src, (uint64_t)(c0 + pos - L0) * stride + col);
        }
        uint32_t top2 = 0;  // per 16-bit half: the largest magnitude's bits
#pragma unroll
        for (int t = 0; t < 16; t++)
            top2 = __vmaxu2(top2, __vmaxu2(x[t].x & 0x7FFF7FFFu, x[t].y & 0x7FFF7FFFu));
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, max(top2 & 0xFFFFu, top2 >> 16));
        // a NaN's or infinity's bits are above every number's
        const float scale = top >= 0x7F80u ? __int_as_float(0x7FC00000)
                                           : __fdiv_rn(__uint_as_float(top << 16),
                                                       FMT == RT_KV8_E4M3 ? 448.0f : 127.0f);
        uint32_t w[16];
#pragma unroll
        for (int t = 0; t < 16; t++)
            w[t] = scale > 0.0f ? quantise4<FMT>(x[t], scale) : 0u;
        const int32_t id = a.page_table[(size_t)b * a.max_pages + page];
        if (id < 0 || (uint64_t)id >= a.arena_pages) {
            if (lane == 0)
                flag_error(a.error, kErrPage);
        } else {
            uint32_t *s = stage[warp];
            if (plane == 0) {
#pragma unroll
                for (int t = 0; t < 16; t++)
                    s[rt_kv8_k_offset(t, 4 * lane) / 4] = w[t];
            } else {
                // words of tokens {2c, 2c+1, 2c+8, 2c+9} x 4 dimensions -> 4 words of 4 tokens
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint32_t r0 = w[2 * c], r1 = w[2 * c + 1], r2 = w[2 * c + 8],
                                   r3 = w[2 * c + 9];
                    const uint32_t p0 = __byte_perm(r0, r1, 0x5140), p1 = __byte_perm(r0, r1, 0x7362);
                    const uint32_t q0 = __byte_perm(r2, r3, 0x5140), q1 = __byte_perm(r2, r3, 0x7362);
                    const uint32_t o[4] = {__byte_perm(p0, q0, 0x5410), __byte_perm(p0, q0, 0x7632),
                                           __byte_perm(p1, q1, 0x5410), __byte_perm(p1, q1, 0x7632)};
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        s[rt_kv8_v_offset(2 * c, 4 * lane + e) / 4] = o[e];
                }
            }
            __syncwarp();
            const uint64_t tile = ((uint64_t)id * a.num_kv_heads + h) * 2u + plane;
            uint4 *dst = reinterpret_cast<uint4 *>(a.pages + tile * kPlane);
#pragma unroll
            for (int i = 0; i < 4; i++)
                dst[i * 32 + lane] = reinterpret_cast<const uint4 *>(s)[i * 32 + lane];
            if (lane == 0)
                a.scales[tile] = scale;
        }
    }
    if (j == 0) {
        const int64_t base = (L1 >> 4) << 4;
        for (int64_t pos = base > L0 ? base : L0; pos < L1; pos++)
            *reinterpret_cast<uint2 *>(tail + (pos - base) * 128) =
                load4<F32>(src, (uint64_t)(c0 + pos - L0) * stride + col);
    }
}

// --------------------------------------------------------------- attention
constexpr int kWarps = 4;
constexpr int kStages = 4;
constexpr int kCtasPerSm = 3;
constexpr uint32_t kBlockBytes = 2 * kPlane;              // one (page, head): K plane, V plane
constexpr uint32_t kRingBytes = kWarps * kStages * kBlockBytes;
constexpr uint32_t kTailBytes = 2 * 16 * 256;             // bf16 K and V rows of the tail
constexpr uint32_t kHeadPitch = 132;                      // floats per head of the warps' merge
constexpr int kSmemBytes = kRingBytes + kTailBytes;
constexpr uint32_t kMaxChunkPages = 32 * kWarps;          // one page id per lane
constexpr uint64_t kWaitLimitNs = 2000000000ull;
static_assert(kWarps * 8 * kHeadPitch * 4 <= kRingBytes, "the merge reuses the ring");

struct AttnArgs {
    const __nv_bfloat16 *q;
    const uint8_t *pages;
    const float *scales;
    const __nv_bfloat16 *tail;
    const int32_t *page_table, *lens;
    float *out;
    float *part_o;    // [num_seqs][num_kv_heads][max_chunks][G][128], unnormalised
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

// Four codes as two fp16 pairs, exactly.  s8: with its sign bit flipped a
// code c is the byte c + 128, and 0x6400 | byte is the fp16 1024 + byte.
template <uint32_t FMT>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t &lo, uint32_t &hi)
{
    if constexpr (FMT == RT_KV8_E4M3) {
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)(w & 0xFFFFu)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
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
// (lane / 4, lane % 4) has the heads 2c and 2c + 1, and of O^T the dimensions
// 16 i + g (o[i][0], o[i][1]) and 16 i + 8 + g (o[i][2], o[i][3]).
struct Softmax {
    float m0, m1, l0, l1;
    float o[8][4];
};

// New maxima for scores of 16 tokens (rows g and g + 8); s becomes exp2(s - m).
// Returns the factors for what was summed before.
__device__ __forceinline__ float2 softmax_step(Softmax &st, float (&s)[4])
{
    float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xFFFFFFFFu, x0, off));
        x1 = fmaxf(x1, __shfl_xor_sync(0xFFFFFFFFu, x1, off));
    }
    x0 = fmaxf(x0, st.m0);
    x1 = fmaxf(x1, st.m1);
    const float2 f = make_float2(rt::fast_exp2(st.m0 - x0), rt::fast_exp2(st.m1 - x1));
    st.m0 = x0;
    st.m1 = x1;
    s[0] = rt::fast_exp2(s[0] - x0);
    s[2] = rt::fast_exp2(s[2] - x0);
    s[1] = rt::fast_exp2(s[1] - x1);
    s[3] = rt::fast_exp2(s[3] - x1);
    st.l0 = st.l0 * f.x + (s[0] + s[2]);
    st.l1 = st.l1 * f.y + (s[1] + s[3]);
    return f;
}

// One CTA per (sequence, KV head, chunk of pages), its warps taking the pages
// in turn.  A page's K and V codes are one 4 KiB bulk copy into the warp's
// ring.  Math per page: S^T = K.Q^T and O^T = V^T.P^T on m16n8k16 with the 16
// tokens (or 16 dimensions) as rows and the KV group's heads as columns.  Codes
// are exact in fp16; a query row is scaled by a power of two into fp16's range
// (exact for all that matters in fp32: see load_q) and the scales of K and V
// are applied in fp32, to the scores and to the page's part of O.  P is split
// into two fp16 terms, which keeps 22 bits of it.
template <uint32_t FMT>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) kv8_decode_kernel(const AttnArgs a)
{
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kWarps][kStages];
    __shared__ __align__(8) uint64_t tail_bar;
    __shared__ float2 ml[kWarps][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, c = lane & 3;
    const uint32_t h = blockIdx.x % a.num_kv_heads;
    const uint32_t rest = blockIdx.x / a.num_kv_heads;
    const uint32_t b = rest % a.num_seqs, chunk = rest / a.num_seqs;
    const int32_t L = a.lens[b];
    if (!len_ok(a, L)) {
        if (threadIdx.x == 0 && chunk == 0)
            flag_error(a.error, kErrLen);
        return;
    }
    const uint32_t n_chunks = chunks_of(a, L);
    if (chunk >= n_chunks)
        return;
    const uint32_t G = a.G;
    const uint32_t n_full = (uint32_t)L >> 4;
    const uint32_t p0 = chunk * a.chunk_pages;
    const uint32_t p1 = min(n_full, p0 + a.chunk_pages);
    const uint32_t n_tail = chunk + 1 == n_chunks ? (uint32_t)L & 15u : 0u;
    int n_mine = (int)((p1 - p0 + kWarps - 1 - warp) / kWarps);

    // barriers: each warp its own; warp 0 the tail's
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < kStages; s++)
            rt::mbar_init(rt::smem_u32(&bars[warp][s]), 1);
        if (warp == 0)
            rt::mbar_init(rt::smem_u32(&tail_bar), 1);
        rt::mbar_fence_init();
    }
    __syncwarp();

    // this warp's page ids and scales, one page per lane; -1: not read
    int32_t id = -1;
    float2 sc = make_float2(0.0f, 0.0f);
    if (lane < n_mine) {
        id = a.page_table[(size_t)b * a.max_pages + p0 + warp + lane * kWarps];
        if (id < 0 || (uint64_t)id >= a.arena_pages) {
            flag_error(a.error, kErrPage);
            id = -1;
        } else {
            sc = *reinterpret_cast<const float2 *>(a.scales +
                                                   ((uint64_t)id * a.num_kv_heads + h) * 2u);
        }
    }
    const uint32_t ring = rt::smem_u32(smem) + (uint32_t)warp * kStages * kBlockBytes;
    auto issue = [&](int i) {
        const int32_t pg = __shfl_sync(0xFFFFFFFFu, id, i);
        if (lane == 0 && pg >= 0) {
            const uint32_t s = (uint32_t)i % kStages;
            const uint32_t bar = rt::smem_u32(&bars[warp][s]);
            rt::mbar_arrive_expect_tx(bar, kBlockBytes);
            rt::bulk_load(ring + s * kBlockBytes,
                          a.pages + ((uint64_t)pg * a.num_kv_heads + h) * kBlockBytes, kBlockBytes,
                          bar);
        }
    };
    for (int i = 0; i < kStages && i < n_mine; i++)
        issue(i);
    const uint32_t tail_s = rt::smem_u32(smem) + kRingBytes;
    const int tail_warp = (int)((p1 - p0) % kWarps);  // the first one with fewer pages
    if (n_tail && warp == 0 && lane == 0) {
        const uint32_t bar = rt::smem_u32(&tail_bar), bytes = n_tail * 256u;
        const __nv_bfloat16 *src = a.tail + rt_page_elem_offset(b, h, 0, 0, a.num_kv_heads);
        rt::mbar_arrive_expect_tx(bar, 2 * bytes);
        rt::bulk_load(tail_s, src, bytes, bar);
        rt::bulk_load(tail_s + 4096u, src + 2048, bytes, bar);
    }

    // Query fragments: lane (g, c) holds, of head g, dimensions 16 s + 4 c .. + 3
    // for step s, as K's words hold them.  The row is multiplied by a power of
    // two so that its largest element lies in [2^14, 2^15): bf16 elements down to
    // 2^-31 of that are exact in fp16, and what the smaller ones lose is below
    // 2^-39 of the largest.
    const __nv_bfloat16 *q_row = a.q + (uint64_t)b * a.q_stride + ((uint64_t)h * G + g) * 128u;
    uint2 qv[8];
#pragma unroll
    for (int s = 0; s < 8; s++)
        qv[s] = (uint32_t)g < G ? *reinterpret_cast<const uint2 *>(q_row + 16 * s + 4 * c)
                                : make_uint2(0u, 0u);
    uint32_t top2 = 0;
#pragma unroll
    for (int s = 0; s < 8; s++)
        top2 = __vmaxu2(top2, __vmaxu2(qv[s].x & 0x7FFF7FFFu, qv[s].y & 0x7FFF7FFFu));
    uint32_t top = max(top2 & 0xFFFFu, top2 >> 16);
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    // 2^(14 - e) for a largest element of exponent e; within fp32's normal range
    const int e = min(max((int)(top >> 7) - 127, -112), 126);
    const float up = __int_as_float((127 + 14 - e) << 23), down = __int_as_float((127 - 14 + e) << 23);
    uint32_t qf[8][2];
#pragma unroll
    for (int s = 0; s < 8; s++) {
        qf[s][0] = pack_f16x2(__uint_as_float(qv[s].x << 16) * up,
                              __uint_as_float(qv[s].x & 0xFFFF0000u) * up);
        qf[s][1] = pack_f16x2(__uint_as_float(qv[s].y << 16) * up,
                              __uint_as_float(qv[s].y & 0xFFFF0000u) * up);
    }
    const float k0 = a.scale_log2 * __shfl_sync(0xFFFFFFFFu, down, 8 * c);       // head 2c
    const float k1 = a.scale_log2 * __shfl_sync(0xFFFFFFFFu, down, 8 * c + 4);   // head 2c + 1

    Softmax st;
    st.m0 = st.m1 = -INFINITY;
    st.l0 = st.l1 = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++)
        st.o[i][0] = st.o[i][1] = st.o[i][2] = st.o[i][3] = 0.0f;

    int n_issue = n_mine;
    uint32_t phases = 0;
    for (int i = 0; i < n_mine; i++) {
        const int32_t pg = __shfl_sync(0xFFFFFFFFu, id, i);
        const float sk = __shfl_sync(0xFFFFFFFFu, sc.x, i), sv = __shfl_sync(0xFFFFFFFFu, sc.y, i);
        const uint32_t s = (uint32_t)i % kStages;
        if (pg >= 0) {
            // after an expired wait no page is issued any more; those in flight are
            // waited for, each again with a limit
            if (!__all_sync(0xFFFFFFFFu,
                            rt::mbar_wait_bounded(rt::smem_u32(&bars[warp][s]), (phases >> s) & 1u,
                                                  kWaitLimitNs))) {
                if (lane == 0)
                    flag_error(a.error, kErrTimeout);
                n_issue = 0;
                n_mine = min(n_mine, i + kStages);
            }
            phases ^= 1u << s;
            const uint4 *blk = reinterpret_cast<const uint4 *>(smem + (ring - rt::smem_u32(smem)) +
                                                               s * kBlockBytes) + lane;
            float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint4 w = blk[j * 32];
                uint32_t f[4];
                decode4<FMT>(w.x, f[0], f[2]);
                decode4<FMT>(w.y, f[1], f[3]);
                mma_f16_16816(sa, f, qf[2 * j][0], qf[2 * j][1]);
                decode4<FMT>(w.z, f[0], f[2]);
                decode4<FMT>(w.w, f[1], f[3]);
                mma_f16_16816(sb, f, qf[2 * j + 1][0], qf[2 * j + 1][1]);
            }
            const float f0 = sk * k0, f1 = sk * k1;
            float x[4] = {(sa[0] + sb[0]) * f0, (sa[1] + sb[1]) * f1, (sa[2] + sb[2]) * f0,
                          (sa[3] + sb[3]) * f1};
            const float2 fac = softmax_step(st, x);
            // P as two fp16 terms, transposed into the second product's B operand
            const uint32_t h0 = pack_f16x2(x[0], x[1]), h1 = pack_f16x2(x[2], x[3]);
            const float2 r0 = unpack_f16x2(h0), r1 = unpack_f16x2(h1);
            const uint32_t l0 = pack_f16x2(x[0] - r0.x, x[1] - r0.y);
            const uint32_t l1 = pack_f16x2(x[2] - r1.x, x[3] - r1.y);
            const uint32_t ph0 = rt::movmatrix_trans(h0), ph1 = rt::movmatrix_trans(h1);
            const uint32_t pl0 = rt::movmatrix_trans(l0), pl1 = rt::movmatrix_trans(l1);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint4 w = blk[128 + j * 32];
                uint32_t f[4];
                float d[4] = {0.f, 0.f, 0.f, 0.f}, d2[4] = {0.f, 0.f, 0.f, 0.f};
                decode4<FMT>(w.x, f[0], f[2]);
                decode4<FMT>(w.y, f[1], f[3]);
                mma_f16_16816(d, f, ph0, ph1);
                mma_f16_16816(d, f, pl0, pl1);
                decode4<FMT>(w.z, f[0], f[2]);
                decode4<FMT>(w.w, f[1], f[3]);
                mma_f16_16816(d2, f, ph0, ph1);
                mma_f16_16816(d2, f, pl0, pl1);
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const float fu = u & 1 ? fac.y : fac.x;
                    st.o[2 * j][u] = fmaf(d[u], sv, st.o[2 * j][u] * fu);
                    st.o[2 * j + 1][u] = fmaf(d2[u], sv, st.o[2 * j + 1][u] * fu);
                }
            }
        }
        __syncwarp();  // every lane has read the slot before it is filled again
        if (i + kStages < n_issue)
            issue(i + kStages);
    }

    // The bf16 tail: the same products on bf16 fragments, P in three bf16 terms.
    // Rows past the tail's end hold anything: their scores are -inf and their V
    // bits are cleared.
    __syncthreads();  // tail_bar is initialised
    if (n_tail && warp == tail_warp) {
        if (!rt::mbar_wait_bounded(rt::smem_u32(&tail_bar), 0, kWaitLimitNs))
            flag_error(a.error, kErrTimeout);
        const uint8_t *tk = smem + kRingBytes, *tv = tk + 4096;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 8; s++) {
            const uint2 a0 = *reinterpret_cast<const uint2 *>(tk + g * 256 + (16 * s + 4 * c) * 2);
            const uint2 a1 = *reinterpret_cast<const uint2 *>(tk + (g + 8) * 256 + (16 * s + 4 * c) * 2);
            const uint32_t f[4] = {a0.x, a1.x, a0.y, a1.y};
            rt::mma_bf16_16816(x, f, qv[s].x, qv[s].y);
        }
        const bool in0 = (uint32_t)g < n_tail, in1 = (uint32_t)g + 8u < n_tail;
        x[0] = in0 ? x[0] * a.scale_log2 : -INFINITY;
        x[1] = in0 ? x[1] * a.scale_log2 : -INFINITY;
        x[2] = in1 ? x[2] * a.scale_log2 : -INFINITY;
        x[3] = in1 ? x[3] * a.scale_log2 : -INFINITY;
        const float2 fac = softmax_step(st, x);
        uint32_t p[3][2];
#pragma unroll
        for (int k = 0; k < 3; k++) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t w = rt::pack_bf16x2(x[2 * u], x[2 * u + 1]);
                x[2 * u] -= __uint_as_float(w << 16);
                x[2 * u + 1] -= __uint_as_float(w & 0xFFFF0000u);
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
#pragma unroll
            for (int u = 0; u < 4; u++)
                st.o[i][u] *= u & 1 ? fac.y : fac.x;
#pragma unroll
            for (int k = 0; k < 3; k++)
                rt::mma_bf16_16816(st.o[i], f, p[k][0], p[k][1]);
        }
    }

    // Merge the warps: sums over a head's lanes, then all states through shared memory.
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
        st.l0 += __shfl_xor_sync(0xFFFFFFFFu, st.l0, off);
        st.l1 += __shfl_xor_sync(0xFFFFFFFFu, st.l1, off);
    }
    __syncthreads();  // all slots have been read
    float *merge = reinterpret_cast<float *>(smem);
    {
        float *mine = merge + ((size_t)warp * 8 + 2 * c) * kHeadPitch + g;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            mine[16 * i] = st.o[i][0];
            mine[16 * i + kHeadPitch] = st.o[i][1];
            mine[16 * i + 8] = st.o[i][2];
            mine[16 * i + 8 + kHeadPitch] = st.o[i][3];
        }
        if (g == 0) {
            ml[warp][2 * c] = make_float2(st.m0, st.l0);
            ml[warp][2 * c + 1] = make_float2(st.m1, st.l1);
        }
    }
    __syncthreads();
    const uint32_t d = threadIdx.x;  // one dimension per thread
    const uint64_t bh = (uint64_t)b * a.num_kv_heads + h;
    for (uint32_t r = 0; r < G; r++) {
        float M = -INFINITY, l = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++)
            M = fmaxf(M, ml[w][r].x);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float wt = ml[w][r].x == -INFINITY ? 0.0f : rt::fast_exp2(ml[w][r].x - M);
            // a warp whose sum is NaN keeps it, whatever its maximum
            l += ml[w][r].y == 0.0f ? 0.0f : ml[w][r].y * (M == -INFINITY ? 1.0f : wt);
            acc += merge[(w * 8 + r) * kHeadPitch + d] * (M == -INFINITY ? 1.0f : wt);
        }
        if (n_chunks == 1) {
            a.out[(bh * G + r) * 128u + d] = l == 0.0f ? 0.0f : acc / l;
        } else {
            const uint64_t slot = (bh * a.max_chunks + chunk) * G + r;
            a.part_o[slot * 128u + d] = acc;
            if (d == 0)
                a.part_ml[slot] = make_float2(M, l);
        }
    }
}

// Log-sum-exp merge of the chunks of sequences that have several: one warp per
// (sequence, query head), each lane four dimensions.
__global__ void __launch_bounds__(128) kv8_merge_kernel(const AttnArgs a)
{
    const int lane = threadIdx.x & 31;
    const uint64_t row = blockIdx.x * 4ull + (threadIdx.x >> 5);
    const uint32_t Hq = a.num_kv_heads * a.G;
    if (row >= (uint64_t)a.num_seqs * Hq)
        return;
    const uint32_t b = (uint32_t)(row / Hq), hq = (uint32_t)(row % Hq);
    const int32_t L = a.lens[b];
    if (!len_ok(a, L))
        return;
    const uint32_t n = chunks_of(a, L);
    if (n == 1)
        return;
    const uint64_t first = (((uint64_t)b * a.num_kv_heads + hq / a.G) * a.max_chunks) * a.G + hq % a.G;
    float M = -INFINITY;
    for (uint32_t k = lane; k < n; k += 32)
        M = fmaxf(M, a.part_ml[first + (uint64_t)k * a.G].x);
#pragma unroll
    for (int off = 16; off; off >>= 1)
        M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, off));
    float l = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t k = 0; k < n; k++) {
        const uint64_t slot = first + (uint64_t)k * a.G;
        const float2 s = a.part_ml[slot];
        const float wt = M == -INFINITY ? 1.0f : s.x == -INFINITY ? 0.0f : rt::fast_exp2(s.x - M);
        const float4 o = reinterpret_cast<const float4 *>(a.part_o + slot * 128u)[lane];
        l += s.y == 0.0f ? 0.0f : s.y * wt;
        acc.x += o.x * wt;
        acc.y += o.y * wt;
        acc.z += o.z * wt;
        acc.w += o.w * wt;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    reinterpret_cast<float4 *>(a.out + row * 128u)[lane] =
        make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

// Pages per item: up to 64, fewer when the grid would not give every SM's slots
// two items.
uint32_t chunk_pages_of(const rt_kv8_attn_params_t *p)
{
    const uint64_t pages = p->max_seq_len >> 4;
    uint64_t c = p->chunk_pages;
    if (!c) {
        const uint64_t slots = 2ull * kCtasPerSm * (uint64_t)rt::num_sms();
        c = (pages * p->num_seqs * p->num_kv_heads + slots - 1) / slots;
        c = c < 8 ? 8 : c > 64 ? 64 : c;
    }
    return (uint32_t)c;
}
uint32_t max_chunks_of(const rt_kv8_attn_params_t *p, uint32_t chunk)
{
    const uint32_t n = ((p->max_seq_len >> 4) + chunk - 1) / chunk;
    return n ? n : 1u;
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
        p->chunk_pages > kMaxChunkPages || !(fabsf(p->scale) <= 3.4e38f) ||
        p->q_stride < (uint64_t)p->num_q_heads * 128u || p->q_stride % 8u ||
        p->max_seq_len > 0x7FFFFFFFu || (p->max_seq_len >> 4) > p->max_pages_per_seq) {
        rt::set_error("kv8_decode_attention: 1..8 query heads to a KV head (%u / %u), format e4m3 "
                      "or s8, q_stride >= num_q_heads * 128 and a multiple of 8, chunk_pages <= "
                      "%u, max_seq_len / 16 <= max_pages_per_seq",
                      p->num_q_heads, p->num_kv_heads, kMaxChunkPages);
        return RT_EINVAL;
    }
    const uint32_t chunk = chunk_pages_of(p);
    const uint64_t items = (uint64_t)p->num_kv_heads * p->num_seqs;
    if (items * max_chunks_of(p, chunk) > 0x7FFFFFFFull ||
        (uint64_t)p->num_q_heads * p->num_seqs > 0x7FFFFFFFull) {
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
    if (!k || !v || !cu_tokens || !seq_lens || !page_table || !pages || !scales || !tail) {
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
    const uint64_t units = (uint64_t)p->num_tokens / 16u + 2ull * p->num_seqs;
    a.n_warps = units * p->num_kv_heads * 2u;
    const uint64_t blocks = (a.n_warps + kAppendWarps - 1) / kAppendWarps;
    if (blocks > 0x7FFFFFFFull) {
        rt::set_error("kv8_append: more than 2^31 - 1 blocks of work; append in parts");
        return RT_EINVAL;
    }
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
    const uint32_t chunks = max_chunks_of(p, chunk_pages_of(p));
    return chunks > 1 ? (size_t)p->num_seqs * p->num_q_heads * chunks * (128u + 2u) * 4u : 0u;
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
    if (!q || !pages || !scales || !tail || !page_table || !seq_lens || !out) {
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
    const size_t need = rt_kv8_attn_workspace_bytes(p);
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
    a.chunk_pages = chunk_pages_of(p);
    a.max_chunks = max_chunks_of(p, a.chunk_pages);
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = need ? reinterpret_cast<float2 *>(a.part_o + (size_t)p->num_seqs * p->num_q_heads *
                                                                 a.max_chunks * 128u)
                     : nullptr;
    cudaStream_t s = (cudaStream_t)stream;
    const void *fn = p->format == RT_KV8_E4M3 ? (const void *)kv8_decode_kernel<RT_KV8_E4M3>
                                              : (const void *)kv8_decode_kernel<RT_KV8_S8>;
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess)
        return rt::cuda_fail(e, "kv8_decode_attention: shared memory");
    const dim3 grid(p->num_kv_heads * p->num_seqs * a.max_chunks);
    if (p->format == RT_KV8_E4M3)
        kv8_decode_kernel<RT_KV8_E4M3><<<grid, kWarps * 32, kSmemBytes, s>>>(a);
    else
        kv8_decode_kernel<RT_KV8_S8><<<grid, kWarps * 32, kSmemBytes, s>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess)
        return rt::cuda_fail(e, "kv8_decode_attention: launch");
    if (a.max_chunks > 1) {
        const uint64_t rows = (uint64_t)p->num_seqs * p->num_q_heads;
        kv8_merge_kernel<<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(a);
        e = cudaGetLastError();
        if (e != cudaSuccess)
            return rt::cuda_fail(e, "kv8_decode_attention: merge launch");
    }
    return RT_OK;
}
