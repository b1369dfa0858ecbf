// answer.cu — from class sums to an answer: biases, allowed classes and
// penalties, the choice of a class and its log-probability, in one pass.
//
// z = allowed ? (pen(v) + b) / t : -inf, formed in 64 bits (divisions as products
// with reciprocals) and rounded once, so that equal and nearly equal class sums
// compare as the real numbers they stand for.  A thread forms E of a row's z at a time, finds their best, and
// sums exp(z' - z) over the others; two such triples (z, class, sum) merge into
// one.  The choice's log-probability is then -log1p(sum): without the
// cancellation of z - logsumexp(z) where the choice is nearly certain.
//
// Rows of up to 512 classes belong to 4 to 32 threads, whose next row is on its
// way while they work; longer ones to a block, or to a cluster of up to 16
// blocks where there are few rows, which merge through distributed shared
// memory.  How often a class stands in the row's history is counted in shared
// memory first, for the classes that the block holds.
//
// 65536 x 100 int32 takes 20 us on the GPU, 2.7 TB/s of its 54 MB, 22.5 a call: 52
// instructions a class, 9 us of issue, which the 16 warps of an SM, with 124
// registers a thread, fill to 53%: each round waits for 64-bit results, for the
// row's temperature and its reciprocal, and for the row's other threads.  Few long rows are bound by latency: one row
// of 131072 fp32 with a history of 2000 12 us, 64 x 32001 bf16 with a history of
// 700, masks and biases 16 us, both with the call's host time of 6 us.
#include <cooperative_groups.h>
#include <limits.h>
#include <math.h>

#include "common.cuh"
#include "elem.cuh"

namespace ytm {

namespace cg = cooperative_groups;

struct Best {
    float z;
    int k;  // INT_MAX: no allowed class seen
    float s;
};

// Order of numpy's argmax: NaN above all numbers, the lowest class of equals.
__device__ __forceinline__ bool above(float z, int k, float z2, int k2) {
    const bool n = z != z, n2 = z2 != z2, equal = n == n2 && (n || z == z2);
    return (z > z2) | (n & !n2) | (equal & (k < k2));
}

__device__ __forceinline__ float exp_of(float x) {  // within a few steps and x's rounding
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

__device__ __forceinline__ Best merge(const Best &a, const Best &b) {
    const bool ab = b.k == INT_MAX || (a.k != INT_MAX && above(a.z, a.k, b.z, b.k));
    const Best hi = ab ? a : b, lo = ab ? b : a;
    if (lo.k == INT_MAX) return hi;
    const float f = exp_of(lo.z - hi.z);
    // a term of -inf adds nothing, whatever its own sum came to
    return {hi.z, hi.k, f == 0.f ? hi.s : __fadd_rn(hi.s, __fmul_rn(f, 1.f + lo.s))};
}

__device__ __forceinline__ Best merge_lanes(Best b, int lanes) {
    for (int d = lanes / 2; d; d >>= 1)
        b = merge(b, {__shfl_xor_sync(0xFFFFFFFFu, b.z, d), __shfl_xor_sync(0xFFFFFFFFu, b.k, d),
                      __shfl_xor_sync(0xFFFFFFFFu, b.s, d)});
    return b;
}

struct AnswerRow {
    double rt, rr;  // 1 / temperature, 1 / repetition
    float r, f, p;
    int64_t len;    // of the history
};

__device__ __forceinline__ AnswerRow answer_row(const ytm_answer_args &a, int64_t n) {
    AnswerRow o;
    o.rt = 1.0 / (double)(a.temperature ? a.temperature[n] : a.temperature_all);
    o.len = 0;
    if (a.history) {
        o.r = a.repetition ? a.repetition[n] : a.repetition_all;
        o.rr = 1.0 / (double)o.r;
        o.f = a.frequency ? a.frequency[n] : a.frequency_all;
        o.p = a.presence ? a.presence[n] : a.presence_all;
        o.len = a.lengths ? max(0, min(a.history_len, a.lengths[n])) : a.history_len;
    }
    return o;
}

// Penalties for a class that stands `count` times in the history.
__device__ __forceinline__ double penalised(double v, uint32_t count, const AnswerRow &o) {
    return v * (v > 0.0 ? o.rr : (double)o.r) - (double)o.f * (double)count - (double)o.p;
}

// The best of E classes of a thread (z: -inf where closed) and the others' sum.
template <int E, typename K>
__device__ __forceinline__ Best best_of(const float (&z)[E], uint32_t open, K class_of) {
    float m = z[0];
#pragma unroll
    for (int e = 1; e < E; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(z[e]));
    int at = 0;
    float s = 0.f;
    if (m > -INFINITY) {  // a number, and no closed class has it
#pragma unroll
        for (int e = E - 1; e >= 0; --e) at = z[e] == m ? e : at;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float x = exp_of(z[e] - m);
            s += e == at ? 0.f : x;
        }
    } else {  // nothing open, -inf everywhere, or a NaN
        if (!open) return {-INFINITY, INT_MAX, 0.f};
        at = -1;
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
            if (((open >> e) & 1u) && (m == -INFINITY || z[e] != z[e])) at = e;
        if (m != m || __popc(open) > 1) s = NAN;
    }
    return {m, class_of(at), s};
}

__device__ __forceinline__ void write_answer(const ytm_answer_args &a, int64_t n, const Best &b) {
    const bool none = b.k == INT_MAX;
    if (a.choice) a.choice[n] = none ? -1 : b.k;
    if (a.logprob) a.logprob[n] = none ? -INFINITY : b.z != b.z ? b.z : -log1pf(b.s);
}

constexpr int AN_THREADS = 256;

// -------------------------------------------------- rows of few classes
// TPR threads hold a row, E classes each, neighbouring lanes neighbouring classes.

template <typename T, int TPR, int E, bool HIST>
__global__ void __launch_bounds__(AN_THREADS, E == 16 ? 2 : E == 8 ? 3 : 4) k_answer_small(const ytm_answer_args a) {
    constexpr int ROWS = AN_THREADS / TPR;
    extern __shared__ uint32_t counts[];  // [ROWS][TPR * E], with a history
    const int lane = threadIdx.x % TPR, team = threadIdx.x / TPR, K = a.k;
    uint32_t *const mine = counts + team * TPR * E;
    uint32_t shared_open = 0;
    float b[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int k = e * TPR + lane;
        b[e] = a.bias && k < K && !a.bias_stride ? a.bias[k] : 0.f;
        if (k < K && (a.allowed_stride || is_allowed(a.allowed, k))) shared_open |= 1u << e;
    }
    struct Row {
        T v[E];
        uint32_t open;
    };
    const auto clamped = [&](int64_t n) { return n < a.n ? n : a.n - 1; };
    const auto fetch = [&](int64_t n0) {
        Row r;
        const int64_t n = clamped(n0 + team);
        const T *cs = (const T *)a.cs + n * a.cs_stride + lane;
        r.open = shared_open;
#pragma unroll
        for (int e = 0; e < E; ++e) r.v[e] = e * TPR + lane < K ? cs[e * TPR] : T(0.f);
        if (a.allowed_stride) {
            const uint32_t *w = a.allowed + n * a.allowed_stride;
            uint32_t bits = 0;
            constexpr int STEP = TPR < 32 ? 32 / TPR : 1;  // classes of a thread in a word
#pragma unroll
            for (int e0 = 0; e0 < E; e0 += STEP) {
                const uint32_t word = e0 * TPR < K ? w[e0 * TPR / 32] >> lane : 0u;
#pragma unroll
                for (int e = e0; e < E && e < e0 + STEP; ++e) bits |= (word >> ((e - e0) * TPR) & 1u) << e;
            }
            r.open &= bits;
        }
        return r;
    };
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t n0 = (int64_t)blockIdx.x * ROWS;
    Row next = fetch(n0);
    for (; n0 < a.n; n0 += step) {
        const Row row = next;
        if (n0 + step < a.n) next = fetch(n0 + step);
        const bool live = n0 + team < a.n;
        const int64_t n = clamped(n0 + team);
        const AnswerRow o = answer_row(a, n);
        if (HIST) {
            __syncwarp();
#pragma unroll
            for (int e = 0; e < E; ++e) mine[e * TPR + lane] = 0;
            __syncwarp();
            for (int64_t i = lane; i < o.len; i += TPR) {
                const int64_t h = index_at(a.history, a.history_64, n * a.history_stride + i);
                if (h >= 0 && h < K) atomicAdd(&mine[h], 1u);
            }
            __syncwarp();
        }
        if (a.bias_stride) {
            const float *bias = a.bias + n * a.bias_stride + lane;
#pragma unroll
            for (int e = 0; e < E; ++e) b[e] = e * TPR + lane < K ? bias[e * TPR] : 0.f;
        }
        float z[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            double v = to_f64(row.v[e]);
            if (HIST) {
                const uint32_t c = mine[e * TPR + lane];
                if (c) v = penalised(v, c, o);
            }
            z[e] = row.open & (1u << e) ? (float)((v + (double)b[e]) * o.rt) : -INFINITY;
        }
        Best best = best_of(z, row.open, [&](int e) { return e * TPR + lane; });
        best = merge_lanes(best, TPR);
        if (!live) continue;
        if (a.adjusted) {
            float *const out = a.adjusted + n * (int64_t)K + lane;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e * TPR + lane < K) out[e * TPR] = z[e];
        }
        if (lane == 0) write_answer(a, n, best);
    }
}

// -------------------------------------------------- rows of many classes

// Classes whose counts a block holds at most; a multiple of every tile.
constexpr int AN_COUNTS = 16384;

template <typename T, int THREADS, int E, bool HIST>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 1 : 4) k_answer_big(const ytm_answer_args a, int cluster, int part, int hold) {
    __shared__ Best warp_best[32], block_best;
    extern __shared__ uint32_t counts[];  // [hold], with a history
    const int tid = threadIdx.x;
    const int64_t n = blockIdx.x / cluster;
    const int rank = (int)(blockIdx.x % cluster);
    const int from = (int)min((int64_t)a.k, (int64_t)rank * part), to = (int)min((int64_t)a.k, (int64_t)from + part);
    const T *cs = (const T *)a.cs + n * a.cs_stride;
    const float *bias = a.bias ? a.bias + n * a.bias_stride : nullptr;
    const uint32_t *allowed = a.allowed ? a.allowed + n * a.allowed_stride : nullptr;
    const AnswerRow o = answer_row(a, n);
    Best best = {-INFINITY, INT_MAX, 0.f};
    for (int64_t c = from; c < to; c += hold) {
        const int c0 = (int)c, c1 = (int)min((int64_t)to, c + hold);
        for (int k0 = c0 + tid; k0 - tid < c1; k0 += THREADS * E) {
            float z[E], b[E];
            uint32_t open = 0;
            T v[E];
            uint32_t word[E];
            const T *in = cs + k0;
            const float *bin = bias ? bias + k0 : nullptr;
            const uint32_t *win = allowed ? allowed + (k0 >> 5) : nullptr;
            // the tiles start at multiples of 32: a warp's bits are one word
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool there = k0 + e * THREADS < c1;
                v[e] = there ? in[e * THREADS] : T(0.f);
                b[e] = there && bin ? bin[e * THREADS] : 0.f;
                word[e] = !there ? 0u : win ? win[e * (THREADS / 32)] : ~0u;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) open |= (word[e] >> (k0 & 31) & 1u) << e;
            if (HIST && k0 == c0 + tid) {  // count, while the first tile is on its way
                __syncthreads();
                for (int i = tid; i < c1 - c0; i += THREADS) counts[i] = 0;
                __syncthreads();
                for (int64_t i = tid; i < o.len; i += THREADS) {
                    const int64_t h = index_at(a.history, a.history_64, n * a.history_stride + i) - c0;
                    if (h >= 0 && h < c1 - c0) atomicAdd(&counts[h], 1u);
                }
                __syncthreads();
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                double x = to_f64(v[e]);
                if (HIST) {
                    const uint32_t c = counts[k0 - c0 + e * THREADS];  // behind c1: not open
                    if (c) x = penalised(x, c, o);
                }
                z[e] = open & (1u << e) ? (float)((x + (double)b[e]) * o.rt) : -INFINITY;
            }
            if (a.adjusted) {
                float *const out = a.adjusted + n * a.k + k0;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (k0 + e * THREADS < c1) out[e * THREADS] = z[e];
            }
            best = merge(best, best_of(z, open, [&](int e) { return k0 + e * THREADS; }));
        }
    }
    best = merge_lanes(best, 32);
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid < 32) {
        best = merge_lanes(warp_best[tid % (THREADS / 32)], THREADS / 32);
        if (tid == 0) block_best = best;
    }
    if (cluster > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        if (rank == 0 && tid < 32) {
            best = {-INFINITY, INT_MAX, 0.f};
            if (tid < cluster) best = *cl.map_shared_rank(&block_best, tid);
            best = merge_lanes(best, 16);
        }
        cl.sync();  // nobody leaves while its best is read
    }
    if (rank == 0 && tid == 0) write_answer(a, n, best);
}

template <typename T, int TPR, int E>
static ytm_status launch_small(const ytm_answer_args &a, cudaStream_t st) {
    const int64_t rows = AN_THREADS / TPR;
    const unsigned grid = (unsigned)std::min<int64_t>(cdiv(a.n, rows), (int64_t)sm_count() * (E == 16 ? 2 : E == 8 ? 3 : 4));
    if (a.history) k_answer_small<T, TPR, E, true><<<grid, AN_THREADS, AN_THREADS * E * 4, st>>>(a);
    else k_answer_small<T, TPR, E, false><<<grid, AN_THREADS, 0, st>>>(a);
    return launch_check("answer");
}

template <typename T, int THREADS, int E>
static ytm_status launch_big(const ytm_answer_args &a, int cluster, cudaStream_t st) {
    if (a.n * cluster > INT_MAX) return fail(YTM_ERR_UNSUPPORTED, "answer: too many rows for one call");
    const int part = (int)(cdiv(cdiv(a.k, cluster), 32) * 32);
    // counts of whole tiles; narrow blocks hold fewer, so that four fit an SM
    const int tile = THREADS * E, most = THREADS == 1024 ? AN_COUNTS : AN_COUNTS / 2;
    const int64_t tiles = (int64_t)cdiv(part, tile) * tile;
    const int hold = (int)std::min<int64_t>(a.history ? most : tiles, tiles);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.n * cluster));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = a.history ? hold * 4 : 0;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    auto *f = a.history ? k_answer_big<T, THREADS, E, true> : k_answer_big<T, THREADS, E, false>;
    ytm_status rc;
    if (cluster > 8 && (rc = cuda_check(cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "answer cluster")))
        return rc;
    if (cfg.dynamicSmemBytes > 48 * 1024 &&
        (rc = cuda_check(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, AN_COUNTS * 4), "answer smem")))
        return rc;
    return cuda_check(cudaLaunchKernelEx(&cfg, f, a, cluster, part, hold), "answer");
}

template <typename T>
static ytm_status launch_answer(const ytm_answer_args &a, cudaStream_t st) {
    if (a.k <= 16) return launch_small<T, 4, 4>(a, st);
    if (a.k <= 64) return launch_small<T, 8, 8>(a, st);
    if (a.k <= 128) return launch_small<T, 8, 16>(a, st);
    if (a.k <= 256) return launch_small<T, 16, 16>(a, st);
    if (a.k <= 512) return launch_small<T, 32, 16>(a, st);
    if (a.k <= 1024) return launch_big<T, 256, 4>(a, 1, st);
    // few rows: wide blocks, and clusters of them while every block has an SM;
    // many (400 x 10000 fp32: 12.8 us in narrow blocks): four narrow blocks an SM
    if (a.k > 2048 && a.n <= sm_count()) {
        int cluster = 1;
        while (cluster < 16 && a.n * cluster * 2 <= sm_count() && a.k > cluster * 8192) cluster *= 2;
        return launch_big<T, 1024, 8>(a, cluster, st);
    }
    return launch_big<T, 256, 8>(a, 1, st);
}

}  // namespace ytm

using namespace ytm;

extern "C" {

ytm_status ytm_answer(const ytm_answer_args *args, void *stream) {
    if (!args) return fail(YTM_ERR_ARG, "args is NULL");
    ytm_answer_args a = *args;
    if (a.n < 0 || a.k <= 0) return fail(YTM_ERR_ARG, "answer: needs n >= 0 rows of k >= 1 classes");
    if (a.n > INT_MAX || a.k > (1 << 30)) return fail(YTM_ERR_UNSUPPORTED, "answer: more than 2^31 - 1 rows or 2^30 classes");
    if (!is_sum_type(a.cs_type)) return fail(YTM_ERR_ARG, "answer: class sums must be int32, fp32, fp16 or bf16");
    if (a.cs_stride < 0 || a.bias_stride < 0 || a.allowed_stride < 0 || a.history_stride < 0 || a.history_len < 0)
        return fail(YTM_ERR_ARG, "answer: negative stride or length");
    if (a.n == 0) return YTM_OK;
    if (!a.cs || (a.lengths && !a.history)) return fail(YTM_ERR_ARG, "null pointer");
    // the kernels take a stride to say that there is something to read row by row
    if (!a.bias) a.bias_stride = 0;
    if (!a.allowed) a.allowed_stride = 0;
    cudaStream_t st = as_stream(stream);
    switch (a.cs_type) {
        case YTM_I32: return launch_answer<int32_t>(a, st);
        case YTM_F32: return launch_answer<float>(a, st);
        case YTM_F16: return launch_answer<__half>(a, st);
        default: return launch_answer<__nv_bfloat16>(a, st);
    }
}

}  // extern "C"
