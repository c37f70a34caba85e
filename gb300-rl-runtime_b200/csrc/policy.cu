// policy.cu - row operators of a policy-gradient update for sm_100a: the
// log-probability and entropy of one token per row of logits, their gradient,
// and the clipped policy loss with its gradient.  Contract: rlrt.h.
//
// A row is read from HBM once and its gradient written once.  A cluster of CTAs
// holds a row in shared memory, each of its warps a region that it alone loads
// (one bulk copy), reduces and turns into gradient, so regions need no barrier of
// their own; while a row is worked on the next one's copies are under way.  The
// warps send their statistics to every CTA of the cluster, whose mbarrier counts
// them; one warp of each CTA derives the row's coefficients from them, in the same
// order everywhere.
//
// Exponentials are taken in base 2: with c = log2(e) / T and an integer reference
// R, e = 2^z, z = l c - R in one fused multiply-add, whose one rounding is that of
// a small number where e is not small (c's own three roundings are a change of T by
// less than 2^-22 of itself, the same for all elements).  References differ between
// warps; sums move between them by exact powers of two.
//
// The floor is the logits read once and the gradient written once, at the rate of a
// copy (6,547 GB/s measured here).  fp32 is bound by that: 8,192 rows x 32,000 with
// gradient and entropy 343 us, 93% of copy.  bf16 has two exponentials for every 4
// bytes that move: 200 us, 80%, with the exponential unit 59% and the issue slots 60%
// busy (a quarter of the exponentials as polynomials on the multiply-add pipes: 220).
// Small calls are bound by latency: 256 rows x 32,000 fp32 without gradient 9.4 us
// (floor 5.0), 64 rows with gradient 8.7 us (floor 2.5).
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "rlrt.h"
#include "rt_common.cuh"

namespace {

enum : int32_t { kErrToken = 1, kErrSeq = 2, kErrTimeout = 4 };
constexpr int kCtasPerSm = 4;
constexpr int kRowWarps = 8;
constexpr int kThreads = kRowWarps * 32;
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kMaxRows = 32;  // of a group, one to a lane
constexpr uint32_t kMaxVocab = 262144;
constexpr uint64_t kWaitLimitNs = 2000000000ull;
constexpr uint32_t kMaxSmem = 224 * 1024;    // of a CTA, at most
constexpr uint32_t kSmemTarget = 72 * 1024;  // of a CTA: three to an SM

struct RowArgs {
    const void *logits;
    void *dlogits;
    const uint32_t *tokens;
    int32_t *error;
    uint64_t row_stride, grad_stride;
    uint32_t num_rows, vocab;
    uint32_t cluster, region, rows_each;  // region: elements of a warp, whole vectors
    float temperature;
    // log-probabilities
    const uint32_t *row_enable;
    float *logprobs, *entropy;
    const float *dlogprobs, *dentropy;
    // policy loss
    const float *weights, *advantages, *old_lp, *ref_lp;
    const uint32_t *row_seq;
    rt_policy_row_t *rows;
    uint32_t num_seqs;
    float clip_low, clip_high, kl_coef, entropy_coef;
};

enum Mode { kForward, kBackward, kPolicy };

// Statistics of a set of logits l: an integer reference R, s = sum of 2^z and u =
// sum of 2^z z, z = l c - R.
struct Stats {
    int R;
    float s, u;
};
constexpr int kNoRef = -4194304;  // -2^22: no logit that counts is below (see kMaxRef)
// The fused form holds while a row's reference is at most this in size, and then
// what lies below kNoRef is 0 beside it.  Rows beyond (logits of millions, or
// without a finite maximum) take differences to the maximum instead.
constexpr int kMaxRef = 2097152;

// Statistics for a reference that is higher by d.
__device__ __forceinline__ void raise(Stats &x, int R)
{
    const uint32_t d = (uint32_t)R - (uint32_t)x.R;
    const float w = __int_as_float((127 - (int)min(d, 127u)) << 23);  // 2^-d, 0 from 127 on
    x.u = w > 0.0f ? (x.u - x.s * (float)d) * w : 0.0f;
    x.s *= w;
    x.R = R;
}
// Of a warp's lanes, in all of them.
__device__ __forceinline__ void across_warp(Stats &x)
{
    raise(x, __reduce_max_sync(0xFFFFFFFFu, x.R));
#pragma unroll
    for (int off = 16; off; off >>= 1) {
        x.s += __shfl_xor_sync(0xFFFFFFFFu, x.s, off);
        x.u += __shfl_xor_sync(0xFFFFFFFFu, x.u, off);
    }
}

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Aligned: all lanes of a warp execute them together.
__device__ __forceinline__ void cluster_arrive()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait()
{
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Store to the shared memory of the cluster's CTA `rank`, at the addresses that
// `addr` and the mbarrier `bar` have here; counts 16 bytes on that mbarrier when it
// is there.  Unlike a cluster barrier it orders nothing else, so it does not wait
// for the gradient stores of the row before.
__device__ __forceinline__ void send_async(uint32_t addr, uint32_t bar, uint32_t rank, uint4 v)
{
    uint32_t to, to_bar;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(addr), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to_bar) : "r"(bar), "r"(rank));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                 ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"(to_bar)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ float to_float(T x)
{
    if constexpr (sizeof(T) == 2)
        return __bfloat162float(x);
    else
        return x;
}
template <typename T>
__device__ __forceinline__ T from_float(float x)
{
    if constexpr (sizeof(T) == 2)
        return __float2bfloat16_rn(x);
    else
        return x;
}

using rt::f32x2;
using rt::pair;
using rt::halves;
using rt::fma2;
using rt::add2;
using rt::mul2;
__device__ __forceinline__ f32x2 exp2_2(f32x2 z)
{
    const float2 v = halves(z);
    return pair(rt::fast_exp2(v.x), rt::fast_exp2(v.y));
}

// Eight logits of a lane: one 16-byte vector of bf16, or two of fp32 that lie 32
// vectors apart.  floor_of: a lower bound for them in the form that raise_to takes;
// it lets a NaN through.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
    static constexpr int kVectors = 2;
    typedef float Floor;
    float4 w[2];
    __device__ __forceinline__ void load(const uint8_t *p, bool second)
    {
        w[0] = *reinterpret_cast<const float4 *>(p);
        w[1] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (second)
            w[1] = *reinterpret_cast<const float4 *>(p + 512);
    }
    static __device__ __forceinline__ Floor floor_of(float x) { return x; }
    __device__ __forceinline__ void raise_to(Floor f)
    {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            w[i].x = rt::nan_max(w[i].x, f);
            w[i].y = rt::nan_max(w[i].y, f);
            w[i].z = rt::nan_max(w[i].z, f);
            w[i].w = rt::nan_max(w[i].w, f);
        }
    }
    __device__ __forceinline__ float top() const
    {
        return fmaxf(fmaxf(fmaxf(w[0].x, w[0].y), fmaxf(w[0].z, w[0].w)),
                     fmaxf(fmaxf(w[1].x, w[1].y), fmaxf(w[1].z, w[1].w)));
    }
    __device__ __forceinline__ f32x2 get(int i) const  // elements 2 i, 2 i + 1
    {
        return i & 1 ? pair(w[i >> 1].z, w[i >> 1].w) : pair(w[i >> 1].x, w[i >> 1].y);
    }
    __device__ __forceinline__ void set(int i, f32x2 v)
    {
        const float2 x = halves(v);
        if (i & 1) {
            w[i >> 1].z = x.x;
            w[i >> 1].w = x.y;
        } else {
            w[i >> 1].x = x.x;
            w[i >> 1].y = x.y;
        }
    }
    __device__ __forceinline__ void store(float *p, bool second) const
    {
        *reinterpret_cast<float4 *>(p) = w[0];
        if (second)
            *reinterpret_cast<float4 *>(p + 128) = w[1];
    }
};
template <>
struct Eight<__nv_bfloat16> {
    static constexpr int kVectors = 1;
    typedef uint32_t Floor;
    uint32_t w[4];
    __device__ __forceinline__ void load(const uint8_t *p, bool)
    {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
    }
    static __device__ __forceinline__ Floor floor_of(float x)
    {
        const __nv_bfloat162 f = __bfloat162bfloat162(__float2bfloat16_rd(x));
        return *reinterpret_cast<const uint32_t *>(&f);
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b)
    {
        const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162 *>(&a),
                                         *reinterpret_cast<const __nv_bfloat162 *>(&b));
        return *reinterpret_cast<const uint32_t *>(&m);
    }
    __device__ __forceinline__ void raise_to(Floor f)
    {
#pragma unroll
        for (int i = 0; i < 4; i++)
            asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(f));
    }
    __device__ __forceinline__ float top() const
    {
        const uint32_t m = larger(larger(w[0], w[1]), larger(w[2], w[3]));
        return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
    }
    __device__ __forceinline__ f32x2 get(int i) const
    {
        return pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    }
    __device__ __forceinline__ void set(int i, f32x2 v)
    {
        const float2 x = halves(v);
        w[i] = rt::pack_bf16x2(x.x, x.y);
    }
    __device__ __forceinline__ void store(__nv_bfloat16 *p, bool) const
    {
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// What the gradient of a row needs: dl[v] = [v = token] hit - 2^z (q0 + q1 z).
struct Gradient {
    float hit, q0, q1, R;
    float m;         // exact: z = (l - m) c
    uint32_t exact;
};
constexpr float kFloor = -200.0f;  // 2^z is 0 in fp32 from there on; keeps 0 times -infinity out
constexpr double kLn2 = 0.6931471805599453;

// ALONE: short rows, each a warp's own; no cluster, no barrier.
//
// 64 registers for four CTAs to an SM where shared memory allows (three of 64 KiB do
// for most vocabularies; a second buffer for a region, or regions in pieces, leave
// less in flight: 8,192 x 32,000 fp32 347..376 us against 343).
template <typename T, Mode MODE, bool ALONE>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) row_kernel(const RowArgs a)
{
    extern __shared__ __align__(128) uint8_t smem[];
    if (MODE == kPolicy)
        rt::grid_dep_launch();
    __shared__ __align__(8) uint64_t bars[kRowWarps];
    __shared__ __align__(8) uint64_t sent[2];
    // of every warp of the cluster: R, s, u, and the token's logit from its warp (else 0)
    __shared__ uint4 stats[2][kMaxCluster * kRowWarps];
    __shared__ Gradient grads;
    constexpr int N = 16 / sizeof(T), kStep = 32 * N * Eight<T>::kVectors;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = ALONE ? 0u : cluster_rank();
    const uint32_t group = ALONE ? blockIdx.x * kRowWarps + (uint32_t)warp : blockIdx.x / a.cluster;
    if (ALONE && (uint64_t)group * a.rows_each >= a.num_rows)
        return;
    const uint32_t row0 = group * a.rows_each;
    const uint32_t n_rows = min(a.rows_each, a.num_rows - row0);
    const uint32_t entry = ALONE ? 0u : rank * kRowWarps + (uint32_t)warp;
    const uint32_t n_entries = ALONE ? 1u : a.cluster * kRowWarps;
    const bool first = ALONE || (rank == 0 && warp == 0);  // of the row's warps

    // A row in vectors from the 16-byte boundary at or before its start: `skip`
    // elements of the first are not the row's, and the last one ends at or behind
    // `end`.  This warp's region is [lo, hi), of which [from, to) is the row's in
    // full vectors.
    struct Span {
        const T *base;
        uint32_t skip, end, lo, hi, from, to;
    };
    auto span = [&](const T *row) {
        Span r;
        r.skip = (uint32_t)((uintptr_t)row / sizeof(T)) % N;
        r.end = a.vocab + r.skip;
        r.base = row - r.skip;
        const uint32_t all = (r.end + N - 1) / N * N;
        r.lo = min(entry * a.region, all);
        r.hi = min(r.lo + a.region, all);
        r.from = r.lo == 0 && r.skip ? min((uint32_t)N, r.hi) : r.lo;
        r.to = max(r.from, min(r.hi, r.end / N * N));
        return r;
    };
    auto logits_of = [&](uint32_t i) {
        return static_cast<const T *>(a.logits) + (uint64_t)(row0 + i) * a.row_stride;
    };
    auto dlogits_of = [&](uint32_t i) {
        return static_cast<T *>(a.dlogits) + (uint64_t)(row0 + i) * a.grad_stride;
    };

    if (lane == 0) {
        rt::mbar_init(rt::smem_u32(&bars[warp]), 1);
        if (warp == 0) {
            rt::mbar_init(rt::smem_u32(&sent[0]), 1);
            rt::mbar_init(rt::smem_u32(&sent[1]), 1);
        }
        rt::mbar_fence_init();
    }
    __syncwarp();
    if (!ALONE)
        cluster_arrive();  // this CTA runs, its barriers are there: it may be sent to
    uint8_t *here = smem + (uint32_t)warp * a.region * (uint32_t)sizeof(T);
    T *slice = reinterpret_cast<T *>(here);
    auto copy = [&](const Span &r) {
        if (lane == 0 && r.from < r.to) {
            const uint32_t bar = rt::smem_u32(&bars[warp]), bytes = (r.to - r.from) * (uint32_t)sizeof(T);
            rt::fence_proxy_async_smem();  // a partial vector may have been stored there
            rt::mbar_arrive_expect_tx(bar, bytes);
            rt::bulk_load(rt::smem_u32(here) + (r.from - r.lo) * (uint32_t)sizeof(T), r.base + r.from, bytes, bar);
        }
    };
    uint32_t phase = 0;
    // After an expired wait the copy is waited for once more, again with a limit.
    auto arrived = [&](const Span &r) {
        if (r.from < r.to) {
            const uint32_t bar = rt::smem_u32(&bars[warp]);
            if (!rt::mbar_wait_bounded(bar, phase, kWaitLimitNs)) {
                if (a.error)
                    atomicCAS(a.error, 0, kErrTimeout);
                rt::mbar_wait_bounded(bar, phase, kWaitLimitNs);
            }
            phase ^= 1u;
        }
    };
    // What lies in a row's partial first and last vectors is loaded by lanes: 0 .. N -
    // 1 the first, N .. 2 N - 1 the last (a row inside one vector has it as the first).
    auto edge_at = [&](const Span &r, uint32_t &v) {
        v = lane < N ? (uint32_t)lane : r.end / N * N + (lane - N);
        const bool partial = lane < N ? r.skip != 0 : lane < 2 * N && r.end % N != 0 && !(r.skip != 0 && r.end < N);
        return partial && v >= r.lo && v < r.hi;
    };
    auto edge_of = [&](const Span &r) {
        uint32_t v;
        return edge_at(r, v) && v >= r.skip && v < r.end ? r.base[v] : from_float<T>(-INFINITY);
    };

    // Where rows are live whatever the arrays say, the first row's copy starts before
    // they are read; one that turns out to have a bad token is waited for and dropped.
    const bool early = MODE != kPolicy && !a.row_enable;
    Span r = span(logits_of(0));
    T edge = from_float<T>(0.0f);
    auto begin = [&]() {
        copy(r);
        edge = edge_of(r);
    };
    if (early)
        begin();
    // Lane i knows row i of the cluster.
    const uint32_t my_row = row0 + (uint32_t)lane;
    uint32_t token = 0;
    float weight = 0.0f, adv = 0.0f, old_lp = 0.0f, ref_lp = 0.0f, up_lp = 0.0f, up_h = 0.0f;
    bool live = false, bad = false;
    if ((uint32_t)lane < n_rows) {
        token = a.tokens[my_row];
        live = true;
        if constexpr (MODE == kPolicy) {
            weight = a.weights[my_row];
            live = weight != 0.0f;
            if (live) {
                const uint32_t seq = a.row_seq ? a.row_seq[my_row] : my_row;
                if (a.old_lp)
                    old_lp = a.old_lp[my_row];
                if (a.kl_coef != 0.0f)
                    ref_lp = a.ref_lp[my_row];
                bad = seq >= a.num_seqs;
                if (bad && first && a.error)
                    atomicCAS(a.error, 0, kErrSeq);
                adv = bad ? 0.0f : a.advantages[seq];
            }
        } else {
            live = !a.row_enable || a.row_enable[my_row] != 0u;
            if constexpr (MODE == kBackward) {
                up_lp = a.dlogprobs[my_row];
                up_h = a.dentropy ? a.dentropy[my_row] : 0.0f;
            }
        }
        if (live && !bad && token >= a.vocab) {
            bad = true;
            if (first && a.error)
                atomicCAS(a.error, 0, kErrToken);
        }
        if ((!live || bad) && first) {
            if constexpr (MODE == kPolicy) {
                float4 *r = reinterpret_cast<float4 *>(a.rows + my_row);
                r[0] = r[1] = make_float4(0.f, 0.f, 0.f, 0.f);
            } else if (MODE == kForward && bad) {
                a.logprobs[my_row] = 0.0f;
                if (a.entropy)
                    a.entropy[my_row] = 0.0f;
            }
        }
        live = live && !bad;
    }
    const uint32_t in_range = n_rows == 32u ? 0xFFFFFFFFu : (1u << n_rows) - 1u;
    uint32_t todo = __ballot_sync(0xFFFFFFFFu, live);  // the same in all warps of the cluster

    if (MODE != kForward && a.dlogits) {  // rows without a gradient
        for (uint32_t none = in_range & ~todo; none; none &= none - 1) {
            T *dst = dlogits_of(__ffs(none) - 1);
            const Span r = span(dst);
            T *out = dst - r.skip;
            for (uint32_t v = r.from + lane * N; v < r.to; v += 32 * N)
                *reinterpret_cast<uint4 *>(out + v) = make_uint4(0u, 0u, 0u, 0u);
            // a row may end inside its first vector
            for (uint32_t v = max(r.lo, r.skip) + lane; v < min(r.from, r.end); v += 32)
                out[v] = from_float<T>(0.0f);
            for (uint32_t v = r.to + lane; v < min(r.hi, r.end); v += 32)
                out[v] = from_float<T>(0.0f);
        }
    }
    uint32_t exchanges = 0;
    bool late = false;  // a statistics wait has expired (warp 0)
    if (early && !(todo & 1u))
        arrived(r);
    if (!ALONE)
        cluster_wait();
    if (!todo)
        return;

    const float inv_t = a.temperature > 0.0f ? 1.0f / a.temperature : 1.0f;
    const float c = inv_t * 1.4426950408889634f;
    const float inv_c = 1.0f / c;
    const f32x2 c2 = pair(c, c);
    if (!(early && (todo & 1u))) {
        r = span(logits_of(__ffs(todo) - 1));
        begin();
    }
    while (todo) {
        const uint32_t i = __ffs(todo) - 1;
        todo &= todo - 1;
        {
            uint32_t v;
            if (edge_at(r, v))
                slice[v - r.lo] = edge;
        }
        __syncwarp();
        // The region, when it is not needed any more, is filled from the next row.
        const Span next = todo ? span(logits_of(__ffs(todo) - 1)) : r;
        const T next_edge = todo ? edge_of(next) : edge;
        auto refill = [&]() {
            __syncwarp();
            if (todo)
                copy(next);
        };
        const uint32_t hit = __shfl_sync(0xFFFFFFFFu, token, i) + r.skip;
        float l_hit = 0.0f;  // the token's logit, in its warp

        // What lies more than 200 below the reference, in base 2, is 0 in fp32 and is
        // raised to there, which keeps 0 times -infinity out.
        Stats st{kNoRef, 0.0f, 0.0f};
        {
            arrived(r);
            const uint32_t bytes = (r.hi - r.lo) * (uint32_t)sizeof(T), mine = (uint32_t)lane * 16u;
            f32x2 s2, u2, minus_ref;
            auto add = [&](Eight<T> &x, typename Eight<T>::Floor floor) {
                x.raise_to(floor);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const f32x2 z = fma2(x.get(j), c2, minus_ref), e = exp2_2(z);
                    s2 = add2(s2, e);
                    u2 = fma2(e, z, u2);
                }
            };
            auto total = [&](f32x2 v) { return halves(v).x + halves(v).y; };
            // The warp's first vectors, and the token, which is often the row's peak, give its
            // reference.  It does not have to be the maximum: a logit so far above it that z and u lose digits (by more than 12 in
            // base 2) shows in the sums, and then the region's maximum is taken.
            Eight<T> head;
            float top = -INFINITY;
            if (mine < bytes) {
                head.load(here + mine, mine + 512u < bytes);
                top = head.top();
            }
            if (hit >= r.lo && hit < r.hi) {
                l_hit = to_float(slice[hit - r.lo]);
                top = fmaxf(top, l_hit);
            }
            // Statistics of the region for the lanes' largest `top`.
            auto sums = [&]() {
                st = Stats{max(__reduce_max_sync(0xFFFFFFFFu, __float2int_rn(top * c)), kNoRef), 0.0f, 0.0f};
                if (st.R > kMaxRef)
                    return;
                const typename Eight<T>::Floor floor = Eight<T>::floor_of(((float)st.R - 200.0f) * inv_c);
                minus_ref = pair(-(float)st.R, -(float)st.R);
                s2 = u2 = 0;
#pragma unroll 1
                for (uint32_t at = mine; at < bytes; at += kStep * (uint32_t)sizeof(T)) {
                    Eight<T> x;
                    x.load(here + at, at + 512u < bytes);
                    add(x, floor);
                }
                st.s = total(s2);
                st.u = total(u2);
            };
            sums();
            if (__builtin_expect(!__all_sync(0xFFFFFFFFu, st.s < 4096.0f), 0)) {
#pragma unroll 1
                for (uint32_t at = mine; at < bytes; at += kStep * (uint32_t)sizeof(T)) {
                    Eight<T> x;
                    x.load(here + at, at + 512u < bytes);
                    top = fmaxf(top, x.top());
                }
                sums();
            }
            if (MODE == kForward || !a.dlogits)
                refill();
        }
        float l_token = 0.0f;
        const bool leads = ALONE || warp == 0;
        // The row's statistics in warp 0 of every CTA, the same bits in each.  Entries
        // of one exchange land beside those of the one before; the CTA barrier behind
        // each exchange, and that no warp sends before it, keeps a third away.
        auto exchange = [&]() {
            across_warp(st);
            if constexpr (ALONE) {
                l_token = l_hit;
                return;
            }
            const uint32_t turn = exchanges & 1u, bar = rt::smem_u32(&sent[turn]);
            if (warp == 0 && lane == 0)
                rt::mbar_arrive_expect_tx(bar, n_entries * 16u);
            if ((uint32_t)lane < a.cluster)
                send_async(rt::smem_u32(&stats[turn][entry]), bar, lane,
                           make_uint4((uint32_t)st.R, __float_as_uint(st.s), __float_as_uint(st.u),
                                      __float_as_uint(l_hit)));
            if (warp == 0) {
                if (!rt::mbar_wait_bounded<true>(bar, exchanges >> 1 & 1u, kWaitLimitNs)) {
                    late = true;
                    if (a.error)
                        atomicCAS(a.error, 0, kErrTimeout);
                }
                st = Stats{INT32_MIN, 0.0f, 0.0f};
                l_token = 0.0f;
                for (uint32_t e = lane; e < n_entries; e += 32) {
                    const uint4 o = stats[turn][e];
                    Stats x{(int)o.x, __uint_as_float(o.y), __uint_as_float(o.z)};
                    const int top = max(st.R, x.R);
                    raise(st, top);
                    raise(x, top);
                    st.s += x.s;
                    st.u += x.u;
                    l_token += __uint_as_float(o.w);
                }
                across_warp(st);
#pragma unroll
                for (int off = 16; off; off >>= 1)
                    l_token += __shfl_xor_sync(0xFFFFFFFFu, l_token, off);
            }
            exchanges++;
        };
        Gradient gr = {};
        // Warp 0: the row's values and coefficients.
        auto finish = [&](bool exact, float m) {
            // the token's z, and log2 of the sum to 2^-24
            const double z_t = exact ? ((double)l_token - (double)m) * (double)c
                                     : (double)l_token * (double)c - (double)st.R;
            const uint32_t bits = __float_as_uint(st.s);
            const double log_s = st.s > 0.0f && st.s < INFINITY
                                     ? (double)((int)(bits >> 23) - 127) +
                                           (double)log2f(__uint_as_float((bits & 0x7FFFFFu) | 0x3F800000u))
                                     : (double)NAN;
            const double lp = kLn2 * (z_t - log_s);
            const float ent = (float)(kLn2 * (log_s - (double)(st.u / st.s)));
            float g_lp = 0.0f, g_h = 0.0f;
            const uint32_t row = row0 + i;
            if constexpr (MODE == kForward) {
                if (first && lane == 0) {
                    a.logprobs[row] = (float)lp;
                    if (a.entropy)
                        a.entropy[row] = ent;
                }
            } else if constexpr (MODE == kBackward) {
                g_lp = __shfl_sync(0xFFFFFFFFu, up_lp, i);
                g_h = __shfl_sync(0xFFFFFFFFu, up_h, i);
            } else {
                const float A = __shfl_sync(0xFFFFFFFFu, adv, i), w = __shfl_sync(0xFFFFFFFFu, weight, i);
                const float before = __shfl_sync(0xFFFFFFFFu, old_lp, i);
                const float ref = __shfl_sync(0xFFFFFFFFu, ref_lp, i);
                const float apart = a.old_lp ? (float)(lp - (double)before) : 0.0f;
                const float ratio = a.old_lp ? expf(apart) : 1.0f;
                const float held = fminf(fmaxf(ratio, 1.0f - a.clip_low), 1.0f + a.clip_high);
                // Where the ratio, or its product, leaves fp32, products of its root stay: an
                // advantage of 0 gives 0, and a weight may bring the slope back.
                float gain = ratio * A, pull = 0.0f;
                const bool large = !(fabsf(gain) < 0x1p100f) && apart == apart;
                if (large) {
                    const float half = expf(0.5f * apart), Aw = A * w;
                    gain = A == 0.0f ? 0.0f : half * (half * A);
                    pull = Aw == 0.0f ? 0.0f : half * (half * Aw);
                }
                const bool clipped = gain > held * A;
                const float policy = clipped ? -held * A : -gain;
                float kl = 0.0f, penalty = 0.0f, slope = clipped || large ? 0.0f : -gain;
                if (clipped)
                    pull = 0.0f;
                if (a.kl_coef != 0.0f) {
                    const float gap = (float)((double)ref - lp), x = expm1f(gap);
                    // e^g - 1 - g; by its series where the subtraction would lose digits
                    kl = x - gap;
                    if (fabsf(gap) < 0.5f)
                        kl = gap * gap *
                             (0.5f + gap * (1.f / 6 + gap * (1.f / 24 + gap * (1.f / 120 +
                              gap * (1.f / 720 + gap * (1.f / 5040 + gap * (1.f / 40320)))))));
                    penalty = a.kl_coef * kl;
                    if (gap > 80.0f) {  // as above
                        const float half = expf(0.5f * gap);
                        penalty = half * (half * a.kl_coef) - a.kl_coef * (gap + 1.0f);
                        pull += half * (half * (a.kl_coef * w));
                    } else {
                        slope -= a.kl_coef * x;
                    }
                }
                const float loss = policy + penalty - a.entropy_coef * ent;
                g_lp = slope * w - pull;
                g_h = -a.entropy_coef * w;
                if (first && lane == 0) {
                    float4 *to = reinterpret_cast<float4 *>(a.rows + row);
                    to[0] = make_float4((float)lp, ent, loss, policy);
                    to[1] = make_float4(kl, ratio, clipped ? 1.0f : 0.0f, w);
                }
            }
            // 2^z / s (g_lp + g_h (log p + H)) / T, log p = ln 2 (z - log2 s)
            const float scale = inv_t / st.s;
            gr.hit = g_lp * inv_t;
            gr.q0 = scale * (g_lp + g_h * (ent - (float)(kLn2 * log_s)));
            gr.q1 = scale * g_h * (float)kLn2;
            gr.R = (float)st.R;
            gr.m = m;
            gr.exact = exact ? 1u : 0u;
            if (!ALONE && lane == 0)
                grads = gr;
        };
        // What warp 0 has written to grads, in all warps.
        auto share = [&]() {
            if constexpr (!ALONE) {
                __syncthreads();
                gr = grads;
            }
        };
        exchange();
        if (leads) {
            if (st.R > kNoRef && st.R <= kMaxRef) {
                // bring a large sum to [1, 2): the gradient's factors are quotients by it
                raise(st, st.R + max((int)(__float_as_uint(st.s) >> 23 & 0xFFu) - 127, 0));
                finish(false, 0.0f);
            } else {
                gr.exact = 1u;
                if (!ALONE && lane == 0)
                    grads = gr;
            }
        }
        share();
        if (gr.exact) {  // once more, with differences to the maximum
            // from memory: the region may hold the next row already
            const uint32_t v0 = max(r.lo, r.skip) + lane, v1 = min(r.hi, r.end);
            float m = -INFINITY;
            for (uint32_t v = v0; v < v1; v += 32)
                m = fmaxf(m, to_float(r.base[v]));
            // bits whose order as integers is the floats'
            auto ordered = [](float x) {
                const int b = __float_as_int(x);
                return b ^ (b >> 31 & 0x7FFFFFFF);
            };
            st = Stats{__reduce_max_sync(0xFFFFFFFFu, ordered(m)), 0.0f, 0.0f};
            exchange();
            if (leads) {
                gr.m = __int_as_float(st.R ^ (st.R >> 31 & 0x7FFFFFFF));
                if (!ALONE && lane == 0)
                    grads = gr;
            }
            share();
            m = gr.m;
            st = Stats{0, 0.0f, 0.0f};
            f32x2 s2 = 0, u2 = 0;
            for (uint32_t v = v0; v < v1; v += 64) {
                const float y = v + 32 < v1 ? to_float(r.base[v + 32]) - m : -INFINITY;
                const f32x2 z = pair(rt::nan_max((to_float(r.base[v]) - m) * c, kFloor),
                                     rt::nan_max(y * c, kFloor));
                const f32x2 e = exp2_2(z);
                s2 = add2(s2, e);
                u2 = fma2(e, z, u2);
            }
            st.s = halves(s2).x + halves(s2).y;
            st.u = halves(u2).x + halves(u2).y;
            exchange();
            if (leads)
                finish(true, m);
            share();
        }

        if (MODE != kForward && a.dlogits) {
            auto slope = [&](uint32_t v) {
                const float l = to_float(slice[v - r.lo]);
                const float z = fmaxf(gr.exact ? (l - gr.m) * c : fmaf(l, c, -gr.R), kFloor);
                return from_float<T>((v == hit ? gr.hit : 0.0f) - rt::fast_exp2(z) * fmaf(gr.q1, z, gr.q0));
            };
            T *dst = dlogits_of(i), *out = dst - r.skip;
            if ((uint32_t)((uintptr_t)dst / sizeof(T)) % N == r.skip && !gr.exact) {
                const f32x2 minus_ref = pair(-gr.R, -gr.R);
                const f32x2 minus_q0 = pair(-gr.q0, -gr.q0), minus_q1 = pair(-gr.q1, -gr.q1);
                const typename Eight<T>::Floor floor = Eight<T>::floor_of((gr.R - 200.0f) * inv_c);
                {  // the partial vectors at the row's ends
                    uint32_t v;
                    if (edge_at(r, v) && v >= r.skip && v < r.end)
                        out[v] = slope(v);
                }
                const uint32_t start = (r.from - r.lo) * (uint32_t)sizeof(T) + (uint32_t)lane * 16u;
                const uint32_t stop = (r.to - r.lo) * (uint32_t)sizeof(T);
                T *to = out + r.from + lane * N;
                if (gr.q1 != 0.0f) {
#pragma unroll 1
                    for (uint32_t at = start; at < stop; at += kStep * (uint32_t)sizeof(T), to += kStep) {
                        Eight<T> x;
                        x.load(here + at, at + 512u < stop);
                        x.raise_to(floor);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const f32x2 z = fma2(x.get(j), c2, minus_ref);
                            x.set(j, mul2(exp2_2(z), fma2(minus_q1, z, minus_q0)));
                        }
                        x.store(to, at + 512u < stop);
                    }
                } else {  // no entropy term
#pragma unroll 1
                    for (uint32_t at = start; at < stop; at += kStep * (uint32_t)sizeof(T), to += kStep) {
                        Eight<T> x;
                        x.load(here + at, at + 512u < stop);
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            x.set(j, mul2(exp2_2(fma2(x.get(j), c2, minus_ref)), minus_q0));
                        x.store(to, at + 512u < stop);
                    }
                }
                // the token, by the lane that has stored its vector
                if (hit >= r.from && hit < r.to && (uint32_t)lane == (hit - r.from) / N % 32u)
                    out[hit] = slope(hit);
                refill();
            } else {
                for (uint32_t v = max(r.lo, r.skip) + lane; v < min(r.hi, r.end); v += 32)
                    out[v] = slope(v);
                refill();
            }
        }
        r = next;
        edge = next_edge;
    }
    // Statistics that have not come are still under way to this CTA's memory: it stays
    // until the cluster's other CTAs are through.
    if (!ALONE && __any_sync(0xFFFFFFFFu, late)) {
        cluster_arrive();
        cluster_wait();
    }
}

// Weighted sums over the rows' records, in fp64 and a fixed order: one cluster of
// CTAs, each an equal share of the rows, the shares' sums added by the first CTA.  As
// a programmatic dependent it is in place when the rows end; 32 bytes a row, from L2.
constexpr uint32_t kStatsCtas = 8;
__global__ void __launch_bounds__(512) policy_stats_kernel(const rt_policy_row_t *rows, uint32_t n,
                                                           float *stats)
{
    __shared__ double part[16][5];
    __shared__ double shares[kStatsCtas][5];
    const uint32_t rank = blockIdx.x;
    cluster_arrive();
    rt::grid_dep_wait();  // the rows' records are there
    double sum[5] = {0, 0, 0, 0, 0};
    for (uint64_t r = rank * 512u + threadIdx.x; r < n; r += kStatsCtas * 512u) {
        const float4 x = reinterpret_cast<const float4 *>(rows + r)[0];
        const float4 y = reinterpret_cast<const float4 *>(rows + r)[1];
        const double w = y.w;
        if (y.w != 0.0f) {
            sum[0] += w * (double)x.z;
            sum[1] += w * (double)x.w;
            sum[2] += w * (double)y.x;
            sum[3] += w * (double)x.y;
            sum[4] += w * (double)y.z;
        }
    }
#pragma unroll
    for (int i = 0; i < 5; i++) {
#pragma unroll
        for (int off = 16; off; off >>= 1)
            sum[i] += __shfl_xor_sync(0xFFFFFFFFu, sum[i], off);
        if ((threadIdx.x & 31) == 0)
            part[threadIdx.x >> 5][i] = sum[i];
    }
    cluster_wait();  // the first CTA runs
    __syncthreads();
    if (threadIdx.x < 5) {
        double s = 0.0;
        for (int w = 0; w < 16; w++)
            s += part[w][threadIdx.x];
        uint32_t to;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;"
                     : "=r"(to) : "r"(rt::smem_u32(&shares[rank][threadIdx.x])));
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(s) : "memory");
    }
    cluster_arrive();
    cluster_wait();
    if (rank == 0 && threadIdx.x < 5) {
        double s = 0.0;
        for (uint32_t k = 0; k < kStatsCtas; k++)
            s += shares[k][threadIdx.x];
        stats[threadIdx.x] = (float)s;
    }
}

// Short rows are a warp's own, those above 1,000 once there are more than CTAs for
// them at once (loss with gradient: 300 rows of 500 fp32 6.3 us, a CTA each 7.9; 8,192
// of 4,000 bf16 38 against 59; 592 of 4,000 fp32 10.3 against 9.3).
// Else CTAs to a row: as few as make a slice fit the target, then more while the
// rows would leave SMs idle and a slice keeps 8 KiB (16 rows of 32,000 bf16: 7.1 us,
// one CTA a row 10.0).  A group (a cluster or a warp)
// that takes several rows starts each row's copy as its warps end their parts of the
// row before.  Equal shares, all groups at once, where no group waits long for the
// last (4,096 rows of 8,000 fp32, 6.9 turns: 50 us, one row to a group 62); else one
// row to a group, balanced by the hardware (1,023 padded rows of 50,001 bf16, 3.5
// turns: 46 us, shares of 4 51); blocks of 8 where there are many (8,192 rows of
// 32,000 fp32: 343 us, one row to a group 380).
template <typename T, Mode MODE, bool ALONE>
int launch_rows(RowArgs &a, uint32_t k, cudaStream_t stream, const char *what)
{
    const uint32_t N = 16 / sizeof(T), esz = sizeof(T);
    const uint32_t warps = ALONE ? 1u : k * kRowWarps, groups = ALONE ? kRowWarps : 1u;
    a.cluster = k;
    a.region = ((a.vocab + N - 1 + N - 1) / N + warps - 1) / warps * N;
    const uint32_t one = a.region * kRowWarps * esz;
    const size_t bytes = (size_t)one;
    // the same value in every call: host threads may set it at once
    cudaError_t e = cudaFuncSetAttribute(row_kernel<T, MODE, ALONE>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(k);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = k;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int fit = 0;
    if (e == cudaSuccess)
        e = cudaOccupancyMaxActiveClusters(&fit, row_kernel<T, MODE, ALONE>, &cfg);
    if (e != cudaSuccess)
        return rt::cuda_fail(e, what);
    const uint64_t at_once = (uint64_t)(fit > 0 ? fit : 1) * groups;
    uint64_t each = ((uint64_t)a.num_rows + at_once - 1) / at_once;
    if (!ALONE && each > 24)
        each = 8;
    else if (!ALONE && each > 2 && a.num_rows * 100ull < each * at_once * 93u)
        each = 1;
    a.rows_each = (uint32_t)(each > kMaxRows ? kMaxRows : each);
    const uint64_t in_groups = ((uint64_t)a.num_rows + a.rows_each - 1) / a.rows_each;
    const uint64_t ctas = (in_groups + groups - 1) / groups * k;
    if (ctas > 0x7FFFFFFFull) {
        rt::set_error("%s: too many rows (%u)", what, a.num_rows);
        return RT_EINVAL;
    }
    cfg.gridDim = dim3((unsigned)ctas);
    e = cudaLaunchKernelEx(&cfg, row_kernel<T, MODE, ALONE>, (const RowArgs)a);
    return e == cudaSuccess ? RT_OK : rt::cuda_fail(e, what);
}

template <typename T, Mode MODE>
int launch_shape(RowArgs &a, cudaStream_t stream, const char *what)
{
    const uint64_t row = (uint64_t)a.vocab * sizeof(T) + 16u, sms = (uint64_t)rt::num_sms();
    if (a.vocab <= 1000u || (a.vocab <= 6000u && a.num_rows > kCtasPerSm * sms))
        return launch_rows<T, MODE, true>(a, 1u, stream, what);
    uint32_t k = 1;
    while (k < kMaxCluster && row > (uint64_t)k * kSmemTarget)
        k *= 2;
    while (k < kMaxCluster && a.num_rows * 2ull * k <= kCtasPerSm * sms && row / (2 * k) >= 8192)
        k *= 2;
    return launch_rows<T, MODE, false>(a, k, stream, what);
}

template <Mode MODE>
int launch_typed(RowArgs &a, uint32_t dtype, cudaStream_t stream, const char *what)
{
    return dtype == RT_DTYPE_BF16 ? launch_shape<__nv_bfloat16, MODE>(a, stream, what)
                                  : launch_shape<float, MODE>(a, stream, what);
}

// Arguments that all entry points share.
int check_rows(const char *what, uint32_t num_rows, uint32_t vocab, uint64_t row_stride,
               uint64_t grad_stride, uint32_t dtype, float temperature, const void *logits,
               const uint32_t *tokens, const void *dlogits, const int32_t *error)
{
    if (vocab == 0 || vocab > kMaxVocab || dtype > RT_DTYPE_BF16 || row_stride < vocab ||
        (dlogits && grad_stride < vocab) ||
        !(temperature == 0.0f || (temperature >= 1e-4f && temperature <= 1e4f))) {
        rt::set_error("%s: vocab 1..%u (%u), dtype f32 or bf16, strides >= vocab, temperature 0 "
                      "or 1e-4..1e4 (%g)", what, kMaxVocab, vocab, (double)temperature);
        return RT_EINVAL;
    }
    const uintptr_t esz = dtype == RT_DTYPE_BF16 ? 2 : 4;
    if (!logits || !tokens) {
        rt::set_error("%s: null argument", what);
        return RT_EINVAL;
    }
    if (((uintptr_t)logits | (uintptr_t)dlogits) % esz || ((uintptr_t)tokens | (uintptr_t)error) & 3u) {
        rt::set_error("%s: a pointer is not aligned to its element", what);
        return RT_EINVAL;
    }
    if (dlogits) {  // the same rows, or none in common
        const uintptr_t x = (uintptr_t)logits, y = (uintptr_t)dlogits;
        const uintptr_t nx = ((uintptr_t)(num_rows - 1) * row_stride + vocab) * esz;
        const uintptr_t ny = ((uintptr_t)(num_rows - 1) * grad_stride + vocab) * esz;
        if (!(x == y && row_stride == grad_stride) && x < y + ny && y < x + nx) {
            rt::set_error("%s: dlogits overlaps logits without being the same rows", what);
            return RT_EINVAL;
        }
    }
    return RT_OK;
}

bool misaligned(std::initializer_list<const void *> ptrs)
{
    uintptr_t bits = 0;
    for (const void *p : ptrs)
        bits |= (uintptr_t)p;
    return (bits & 3u) != 0;
}

int logprob_call(const char *what, const rt_logprob_params_t *p, const void *logits,
                 const uint32_t *tokens, const void *dlogits, int32_t *error, RowArgs &a)
{
    if (!p) {
        rt::set_error("%s: null params", what);
        return RT_EINVAL;
    }
    if (p->num_rows == 0)
        return RT_OK;
    const int rc = check_rows(what, p->num_rows, p->vocab, p->row_stride, p->grad_stride, p->dtype,
                              p->temperature, logits, tokens, dlogits, error);
    if (rc != RT_OK)
        return rc;
    a = RowArgs{};
    a.logits = logits;
    a.tokens = tokens;
    a.error = error;
    a.row_stride = p->row_stride;
    a.grad_stride = p->grad_stride;
    a.num_rows = p->num_rows;
    a.vocab = p->vocab;
    a.temperature = p->temperature;
    a.row_enable = p->row_enable;
    return RT_OK;
}

}  // namespace

extern "C" int rt_token_logprobs(const rt_logprob_params_t *p, const void *logits,
                                 const uint32_t *tokens, float *logprobs, float *entropy,
                                 int32_t *error, void *stream)
{
    RowArgs a;
    const int rc = logprob_call("token_logprobs", p, logits, tokens, nullptr, error, a);
    if (rc != RT_OK || p->num_rows == 0)
        return rc;
    if (!logprobs || misaligned({logprobs, entropy, p->row_enable})) {
        rt::set_error("token_logprobs: logprobs is null, or an output is not 4-byte aligned");
        return RT_EINVAL;
    }
    a.logprobs = logprobs;
    a.entropy = entropy;
    return launch_typed<kForward>(a, p->dtype, (cudaStream_t)stream, "token_logprobs: launch");
}

extern "C" int rt_token_logprobs_backward(const rt_logprob_params_t *p, const void *logits,
                                          const uint32_t *tokens, const float *dlogprobs,
                                          const float *dentropy, void *dlogits, int32_t *error,
                                          void *stream)
{
    RowArgs a;
    const int rc = logprob_call("token_logprobs_backward", p, logits, tokens, dlogits, error, a);
    if (rc != RT_OK || p->num_rows == 0)
        return rc;
    if (!dlogprobs || !dlogits || misaligned({dlogprobs, dentropy, p->row_enable})) {
        rt::set_error("token_logprobs_backward: dlogprobs or dlogits is null, or an input is not "
                      "4-byte aligned");
        return RT_EINVAL;
    }
    a.dlogits = dlogits;
    a.dlogprobs = dlogprobs;
    a.dentropy = dentropy;
    return launch_typed<kBackward>(a, p->dtype, (cudaStream_t)stream,
                                   "token_logprobs_backward: launch");
}

extern "C" int rt_policy_loss(const rt_policy_params_t *p, const void *logits,
                              const uint32_t *tokens, const float *weights,
                              const float *advantages, const uint32_t *row_seq,
                              const float *old_logprobs, const float *ref_logprobs,
                              rt_policy_row_t *rows, float *stats, void *dlogits, int32_t *error,
                              void *stream)
{
    if (!p || !stats || ((uintptr_t)stats & 3u)) {
        rt::set_error("policy_loss: params or stats is null, or stats not 4-byte aligned");
        return RT_EINVAL;
    }
    if (!(p->clip_low >= 0.0f && p->clip_low <= FLT_MAX) ||
        !(p->clip_high >= 0.0f && p->clip_high <= FLT_MAX) || !(fabsf(p->kl_coef) <= FLT_MAX) ||
        !(fabsf(p->entropy_coef) <= FLT_MAX)) {
        rt::set_error("policy_loss: clip_low, clip_high finite and >= 0, coefficients finite");
        return RT_EINVAL;
    }
    cudaStream_t s = (cudaStream_t)stream;
    if (p->num_rows) {
        const int rc = check_rows("policy_loss", p->num_rows, p->vocab, p->row_stride,
                                  p->grad_stride, p->dtype, p->temperature, logits, tokens,
                                  dlogits, error);
        if (rc != RT_OK)
            return rc;
        if (!weights || !advantages || !rows || (p->kl_coef != 0.0f && !ref_logprobs) ||
            (!row_seq && p->num_seqs < p->num_rows)) {
            rt::set_error("policy_loss: weights, advantages and rows are needed, ref_logprobs "
                          "when kl_coef != 0, num_seqs >= num_rows without row_seq");
            return RT_EINVAL;
        }
        if ((uintptr_t)rows & 15u ||
            misaligned({weights, advantages, row_seq, old_logprobs, ref_logprobs})) {
            rt::set_error("policy_loss: rows must be 16-byte aligned, the other arrays 4-byte");
            return RT_EINVAL;
        }
        RowArgs a = {};
        a.logits = logits;
        a.dlogits = dlogits;
        a.tokens = tokens;
        a.error = error;
        a.row_stride = p->row_stride;
        a.grad_stride = p->grad_stride;
        a.num_rows = p->num_rows;
        a.vocab = p->vocab;
        a.temperature = p->temperature;
        a.weights = weights;
        a.advantages = advantages;
        a.row_seq = row_seq;
        a.old_lp = old_logprobs;
        a.ref_lp = ref_logprobs;
        a.rows = rows;
        a.num_seqs = p->num_seqs;
        a.clip_low = p->clip_low;
        a.clip_high = p->clip_high;
        a.kl_coef = p->kl_coef;
        a.entropy_coef = p->entropy_coef;
        const int rc2 = launch_typed<kPolicy>(a, p->dtype, s, "policy_loss: launch");
        if (rc2 != RT_OK)
            return rc2;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kStatsCtas);
    cfg.blockDim = dim3(512);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kStatsCtas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    // in place when the last rows end
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, policy_stats_kernel, (const rt_policy_row_t *)rows,
                                             p->num_rows, stats);
    return e == cudaSuccess ? RT_OK : rt::cuda_fail(e, "policy_loss: stats launch");
}
