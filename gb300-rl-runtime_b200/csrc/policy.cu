// policy.cu - row operators of a policy-gradient update for sm_100a: the
// log-probability and entropy of one token per row of logits, their gradient,
// and the clipped policy loss with its gradient.  Contract: rlrt.h.
//
// A row is read from HBM once and its gradient written once.  A cluster of CTAs
// holds a row in shared memory: each CTA a slice, copied there by bulk copies
// whose pieces are reduced (running maximum, sum of exponentials, sum of
// e^z z for the entropy) while later pieces arrive.  The slices' statistics are
// exchanged through distributed shared memory, every CTA derives the row's
// coefficients from them in the same order, and the gradient is computed from
// the slice in shared memory.
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "rlrt.h"
#include "rt_common.cuh"

namespace {

enum : int32_t { kErrToken = 1, kErrSeq = 2, kErrTimeout = 4 };
constexpr int kThreads = 512;
constexpr int kPieces = 4;
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kMaxVocab = 262144;
constexpr uint64_t kWaitLimitNs = 2000000000ull;
// Three CTAs of this much on an SM: one loads while others reduce and store.
constexpr uint32_t kSliceTarget = 72 * 1024;

struct RowArgs {
    const void *logits;
    void *dlogits;
    const uint32_t *tokens;
    int32_t *error;
    uint64_t row_stride, grad_stride;
    uint32_t num_rows, vocab, cluster, slice;  // slice: elements per CTA, whole vectors
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

// Running statistics of a set of logits l: their maximum m, s = sum of
// e^((l - m) / T) and u = sum of e^((l - m) / T) (l - m).
struct Stats {
    float m, s, u;
};

// The sums of a set with maximum m, for a maximum shifted by d = m - m' <= 0;
// c = log2(e) / T.  A set without a logit above -infinity (m = -infinity, s = u =
// 0) shifts by 0.  Where the factor is 0 the set is gone, however far it was:
// its u is 0 and not 0 times an overflow; a NaN in s stays.
__device__ __forceinline__ void shift(float &s, float &u, float d, float c)
{
    const float w = rt::fast_exp2(d * c);
    u = w > 0.0f ? (u + s * d) * w : 0.0f;
    s *= w;
}
__device__ __forceinline__ Stats merge(Stats a, Stats b, float c)
{
    Stats r;
    r.m = fmaxf(a.m, b.m);
    shift(a.s, a.u, a.m == -INFINITY ? 0.0f : a.m - r.m, c);
    shift(b.s, b.u, b.m == -INFINITY ? 0.0f : b.m - r.m, c);
    r.s = a.s + b.s;
    r.u = a.u + b.u;
    return r;
}

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait()
{
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t rank, float v)
{
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
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

// One 16-byte vector of logits as floats, and back.
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    float f[N];
    __device__ __forceinline__ void load(const uint8_t *p)
    {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 2) {
                f[2 * i] = __uint_as_float(v[i] << 16);
                f[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
            } else {
                f[i] = __uint_as_float(v[i]);
            }
        }
    }
    __device__ __forceinline__ uint4 pack() const
    {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 2)
                v[i] = rt::pack_bf16x2(f[2 * i], f[2 * i + 1]);
            else
                v[i] = __float_as_uint(f[i]);
        }
        return make_uint4(v[0], v[1], v[2], v[3]);
    }
};

// What the gradient of a row needs: dl[v] = [v = token] hit - e^((l - m) / T)
// (q0 + q1 (l - m)).
struct Gradient {
    float hit, q0, q1;
};

template <typename T, Mode MODE>
__global__ void __launch_bounds__(kThreads) row_kernel(const RowArgs a)
{
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kPieces];
    __shared__ Stats warp_stats[kThreads / 32];
    __shared__ Stats slice_stats[kMaxCluster];
    __shared__ Gradient grad;
    constexpr int N = Vec<T>::N;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = cluster_rank();
    const uint32_t row = blockIdx.x / a.cluster;
    const T *src = static_cast<const T *>(a.logits) + (uint64_t)row * a.row_stride;
    T *dst = a.dlogits ? static_cast<T *>(a.dlogits) + (uint64_t)row * a.grad_stride : nullptr;

    // The row from the 16-byte boundary at or before its start: `skip` elements
    // of the first vector are not the row's.  This CTA has the vectors of
    // [lo, hi), of which [bulk_lo, bulk_hi) are the row's in full.
    const uint32_t skip = (uint32_t)((uintptr_t)src / sizeof(T)) % N;
    const uint32_t end = a.vocab + skip;
    const uint32_t lo = min(rank * a.slice, (end + N - 1) / N * N);
    const uint32_t hi = min(lo + a.slice, (end + N - 1) / N * N);
    const T *base = src - skip;

    const uint32_t token = a.tokens[row];
    float weight = 1.0f;
    uint32_t seq = row;
    bool live = true;
    if constexpr (MODE == kPolicy) {
        weight = a.weights[row];
        live = weight != 0.0f;
        if (live && a.row_seq) {
            seq = a.row_seq[row];
            if (seq >= a.num_seqs) {
                live = false;
                if (tid == 0 && rank == 0 && a.error)
                    atomicCAS(a.error, 0, kErrSeq);
            }
        }
    } else if (a.row_enable) {
        live = a.row_enable[row] != 0u;
    }
    bool bad = false;
    if (live && token >= a.vocab) {
        live = false;
        bad = true;
        if (tid == 0 && rank == 0 && a.error)
            atomicCAS(a.error, 0, kErrToken);
    }
    if (!live) {  // the same for all CTAs of the row
        if (dst) {
            const uint32_t from = lo > skip ? lo - skip : 0u, to = min(hi, end) - min(skip, hi);
            for (uint32_t v = from + tid; v < to; v += kThreads)
                dst[v] = from_float<T>(0.0f);
        }
        if (tid == 0 && rank == 0) {
            if constexpr (MODE == kPolicy) {
                float4 *r = reinterpret_cast<float4 *>(a.rows + row);
                r[0] = r[1] = make_float4(0.f, 0.f, 0.f, 0.f);
            } else if (MODE == kForward && bad) {
                a.logprobs[row] = 0.0f;
                if (a.entropy)
                    a.entropy[row] = 0.0f;
            }
        }
        return;
    }

    cluster_arrive();  // this CTA runs: its shared memory may be written from now on
    const uint32_t bulk_lo = lo == 0 && skip ? N : lo;
    const uint32_t bulk_hi = max(bulk_lo, min(hi, end / N * N));
    const uint32_t piece = ((bulk_hi - bulk_lo) / N + kPieces - 1) / kPieces * N;  // elements
    auto piece_lo = [&](int k) { return min(bulk_hi, bulk_lo + k * piece); };
    if (tid == 0) {
#pragma unroll
        for (int k = 0; k < kPieces; k++)
            rt::mbar_init(rt::smem_u32(&bars[k]), 1);
        rt::mbar_fence_init();
#pragma unroll
        for (int k = 0; k < kPieces; k++) {
            const uint32_t from = piece_lo(k), n = piece_lo(k + 1) - from;
            if (n) {
                const uint32_t bar = rt::smem_u32(&bars[k]);
                rt::mbar_arrive_expect_tx(bar, n * (uint32_t)sizeof(T));
                rt::bulk_load(rt::smem_u32(smem) + (from - lo) * (uint32_t)sizeof(T), base + from,
                              n * (uint32_t)sizeof(T), bar);
            }
        }
    }
    const float l_token = to_float(src[token]);
    // the row's partial first and last vectors, -infinity where they are not the row's
    T *slice = reinterpret_cast<T *>(smem);
    if (tid < 2 * N) {
        const uint32_t v = tid < N ? (uint32_t)tid : end / N * N + (tid - N);
        // a row inside one vector has its last vector filled as its first
        const bool partial = tid < N ? skip != 0 : end % N != 0 && !(skip != 0 && end < N);
        if (partial && v >= lo && v < hi)
            slice[v - lo] = v >= skip && v < end ? base[v] : from_float<T>(-INFINITY);
    }
    __syncthreads();

    const float inv_t = a.temperature > 0.0f ? 1.0f / a.temperature : 1.0f;
    const float c = inv_t * 1.4426950408889634f;
    Stats st{-INFINITY, 0.0f, 0.0f};
    auto take = [&](uint32_t v) {
        Vec<T> x;
        x.load(smem + (size_t)(v - lo) * sizeof(T));
        float top = x.f[0];
#pragma unroll
        for (int i = 1; i < N; i++)
            top = fmaxf(top, x.f[i]);
        if (top > st.m) {
            shift(st.s, st.u, st.m == -INFINITY ? 0.0f : st.m - top, c);
            st.m = top;
        }
        const float m = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float d = x.f[i] - m, e = rt::fast_exp2(d * c);
            st.s += e;
            st.u = fmaf(e, fmaxf(d, -FLT_MAX), st.u);
        }
    };
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
        const uint32_t from = piece_lo(k), to = piece_lo(k + 1);
        if (from < to && !rt::mbar_wait_bounded(rt::smem_u32(&bars[k]), 0, kWaitLimitNs) && a.error)
            atomicCAS(a.error, 0, kErrTimeout);
        for (uint32_t v = from + tid * N; v < to; v += kThreads * N)
            take(v);
    }
    if (tid == 0 && lo < bulk_lo && lo < hi)
        take(lo);
    if (tid == 32 && bulk_hi < hi)
        take(bulk_hi);

#pragma unroll
    for (int off = 16; off; off >>= 1) {
        Stats o;
        o.m = __shfl_xor_sync(0xFFFFFFFFu, st.m, off);
        o.s = __shfl_xor_sync(0xFFFFFFFFu, st.s, off);
        o.u = __shfl_xor_sync(0xFFFFFFFFu, st.u, off);
        st = merge(st, o, c);
    }
    if (lane == 0)
        warp_stats[warp] = st;
    cluster_wait();
    __syncthreads();
    if (warp == 0) {
        st = lane < kThreads / 32 ? warp_stats[lane] : Stats{-INFINITY, 0.0f, 0.0f};
#pragma unroll
        for (int off = 16; off; off >>= 1) {
            Stats o;
            o.m = __shfl_xor_sync(0xFFFFFFFFu, st.m, off);
            o.s = __shfl_xor_sync(0xFFFFFFFFu, st.s, off);
            o.u = __shfl_xor_sync(0xFFFFFFFFu, st.u, off);
            st = merge(st, o, c);
        }
        if ((uint32_t)lane < a.cluster) {
            const uint32_t at = rt::smem_u32(&slice_stats[rank]);
            store_cluster(at, lane, st.m);
            store_cluster(at + 4, lane, st.s);
            store_cluster(at + 8, lane, st.u);
        }
    }
    cluster_arrive();
    cluster_wait();

    if (tid == 0) {
        st = slice_stats[0];
        for (uint32_t k = 1; k < a.cluster; k++)
            st = merge(st, slice_stats[k], c);
        const double inv_td = a.temperature > 0.0f ? 1.0 / (double)a.temperature : 1.0;
        const double log_s = log((double)st.s);
        const double lp = ((double)l_token - (double)st.m) * inv_td - log_s;
        const double ent = log_s - (double)st.u / (double)st.s * inv_td;
        double g_lp = 0.0, g_h = 0.0;
        if constexpr (MODE == kForward) {
            if (rank == 0) {
                a.logprobs[row] = (float)lp;
                if (a.entropy)
                    a.entropy[row] = (float)ent;
            }
        } else if constexpr (MODE == kBackward) {
            g_lp = a.dlogprobs[row];
            g_h = a.dentropy ? a.dentropy[row] : 0.0f;
        } else {
            const double adv = a.advantages[seq];
            const double ratio = a.old_lp ? exp(lp - (double)a.old_lp[row]) : 1.0;
            const double held = fmin(fmax(ratio, 1.0 - (double)a.clip_low), 1.0 + (double)a.clip_high);
            const bool clipped = ratio * adv > held * adv;
            const double policy = clipped ? -held * adv : -ratio * adv;
            double kl = 0.0, slope = clipped ? 0.0 : -ratio * adv;
            if (a.kl_coef != 0.0f) {
                const double gap = (double)a.ref_lp[row] - lp, x = expm1(gap);
                kl = x - gap;
                slope -= (double)a.kl_coef * x;
            }
            const double loss = policy + (double)a.kl_coef * kl - (double)a.entropy_coef * ent;
            g_lp = slope * (double)weight;
            g_h = -(double)a.entropy_coef * (double)weight;
            if (rank == 0) {
                float4 *r = reinterpret_cast<float4 *>(a.rows + row);
                r[0] = make_float4((float)lp, (float)ent, (float)loss, (float)policy);
                r[1] = make_float4((float)kl, (float)ratio, clipped ? 1.0f : 0.0f, weight);
            }
        }
        // e / s (g_lp + g_h (log p + H)) / T, log p = (l - m) / T - log s
        const double scale = inv_td / (double)st.s;
        grad.hit = (float)(g_lp * inv_td);
        grad.q0 = (float)(scale * (g_lp + g_h * (ent - log_s)));
        grad.q1 = (float)(scale * g_h * inv_td);
        warp_stats[0].m = st.m;
    }
    if (MODE == kForward || !dst)
        return;
    __syncthreads();
    const Gradient gr = grad;
    const float m = warp_stats[0].m;
    const float floor_d = -200.0f / c;  // e^(d / T) is 0 in fp32 from there on
    auto slope = [&](float l) {
        const float d = fmaxf(l - m, floor_d);
        return -rt::fast_exp2(d * c) * fmaf(gr.q1, d, gr.q0);
    };
    const uint32_t hit = token + skip;
    const uint32_t dskip = (uint32_t)((uintptr_t)dst / sizeof(T)) % N;
    if (dskip == skip) {
        T *out = dst - skip;
        for (uint32_t v = bulk_lo + tid * N; v < bulk_hi; v += kThreads * N) {
            Vec<T> x;
            x.load(smem + (size_t)(v - lo) * sizeof(T));
#pragma unroll
            for (int i = 0; i < N; i++)
                x.f[i] = slope(x.f[i]);
            if (hit - v < (uint32_t)N) {
#pragma unroll
                for (int i = 0; i < N; i++)
                    x.f[i] += v + i == hit ? gr.hit : 0.0f;
            }
            *reinterpret_cast<uint4 *>(out + v) = x.pack();
        }
        // the partial vectors at the row's ends
        if (tid < 2 * N) {
            const uint32_t v = tid < N ? lo + tid : bulk_hi + (tid - N);
            const bool mine = tid < N ? v < bulk_lo : v >= bulk_lo;
            if (mine && v < hi && v >= skip && v < end)
                out[v] = from_float<T>(slope(to_float(slice[v - lo])) + (v == hit ? gr.hit : 0.0f));
        }
    } else {
        for (uint32_t v = max(lo, skip) + tid; v < min(hi, end); v += kThreads)
            dst[v - skip] = from_float<T>(slope(to_float(slice[v - lo])) + (v == hit ? gr.hit : 0.0f));
    }
}

// Weighted sums over the rows' records, in fp64 and a fixed order.
__global__ void __launch_bounds__(1024) policy_stats_kernel(const rt_policy_row_t *rows, uint32_t n,
                                                            float *stats)
{
    __shared__ double part[32][5];
    double sum[5] = {0, 0, 0, 0, 0};
    for (uint32_t r = threadIdx.x; r < n; r += 1024) {
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
    __syncthreads();
    if (threadIdx.x < 5) {
        double s = 0.0;
        for (int w = 0; w < 32; w++)
            s += part[w][threadIdx.x];
        stats[threadIdx.x] = (float)s;
    }
}

// CTAs to a row: as few as make a slice fit the target, then more while the
// rows would leave SMs idle and a slice keeps 8 KiB.
template <typename T, Mode MODE>
int launch_rows(RowArgs &a, cudaStream_t stream, const char *what)
{
    const uint32_t N = Vec<T>::N, esz = sizeof(T);
    auto slice_of = [&](uint32_t k) { return ((a.vocab + N - 1 + k - 1) / k + N - 1) / N * N; };
    uint32_t k = 1;
    while (k < kMaxCluster && (uint64_t)slice_of(k) * esz > kSliceTarget)
        k *= 2;
    const uint64_t slots = 2ull * (uint64_t)rt::num_sms();
    while (k < kMaxCluster && (uint64_t)a.num_rows * k * 2 <= slots && slice_of(2 * k) * esz >= 8192)
        k *= 2;
    a.cluster = k;
    a.slice = slice_of(k);
    if ((uint64_t)a.num_rows * k > 0x7FFFFFFFull) {
        rt::set_error("%s: too many rows (%u)", what, a.num_rows);
        return RT_EINVAL;
    }
    const size_t bytes = (size_t)a.slice * esz;
    cudaError_t e = cudaFuncSetAttribute(row_kernel<T, MODE>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess)
        return rt::cuda_fail(e, what);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.num_rows * k);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = k;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, row_kernel<T, MODE>, (const RowArgs)a);
    return e == cudaSuccess ? RT_OK : rt::cuda_fail(e, what);
}

template <Mode MODE>
int launch_typed(RowArgs &a, uint32_t dtype, cudaStream_t stream, const char *what)
{
    return dtype == RT_DTYPE_BF16 ? launch_rows<__nv_bfloat16, MODE>(a, stream, what)
                                  : launch_rows<float, MODE>(a, stream, what);
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
    policy_stats_kernel<<<1, 1024, 0, s>>>(rows, p->num_rows, stats);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? RT_OK : rt::cuda_fail(e, "policy_loss: stats launch");
}
