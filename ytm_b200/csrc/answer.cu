// answer.cu — from class sums to an answer: biases, allowed classes and
// penalties, the choice of a class and its log-probability.
#include <limits.h>
#include <math.h>

#include "common.cuh"
#include "elem.cuh"

namespace ytm {

// ------------------------------------------------------------ the choice
// z = allowed ? (pen(v) + b) / t : -inf, formed in 64 bits and rounded once, so
// that equal and nearly equal class sums compare as the real numbers they
// stand for.  One pass keeps, per thread, the best (z, class) and the sum s of
// exp(z' - z) over the other allowed classes; two such triples merge into
// one.  The choice's log-probability is then -log1p(s): without the
// cancellation of z - logsumexp(z) where the choice is nearly certain.

struct Best {
    float z;
    int k;  // INT_MAX: no allowed class seen
    float s;
};

// Order of numpy's argmax: NaN above all numbers, the lowest class of equals.
__device__ __forceinline__ bool above(float z, int k, float z2, int k2) {
    const bool n = z != z, n2 = z2 != z2;
    if (n || n2) return n && (!n2 || k < k2);
    return z > z2 || (z == z2 && k < k2);
}

__device__ __forceinline__ Best merge(const Best &a, const Best &b) {
    if (a.k == INT_MAX) return b;
    if (b.k == INT_MAX) return a;
    const bool ab = above(a.z, a.k, b.z, b.k);
    const Best hi = ab ? a : b, lo = ab ? b : a;
    const float f = expf(lo.z - hi.z);
    // a term of -inf adds nothing, whatever its own sum came to
    return {hi.z, hi.k, f == 0.f ? hi.s : hi.s + f * (1.f + lo.s)};
}

struct AnswerRow {
    double rt, r, f, p;
};

__device__ __forceinline__ AnswerRow answer_row(const ytm_answer_args &a, int64_t n) {
    AnswerRow o;
    o.rt = 1.0 / (double)(a.temperature ? a.temperature[n] : a.temperature_all);
    o.r = (double)(a.repetition ? a.repetition[n] : a.repetition_all);
    o.f = (double)(a.frequency ? a.frequency[n] : a.frequency_all);
    o.p = (double)(a.presence ? a.presence[n] : a.presence_all);
    return o;
}

__device__ __forceinline__ float adjust(double v, uint32_t count, double b, const AnswerRow &o) {
    if (count) v = (v > 0.0 ? v / o.r : v * o.r) - o.f * (double)count - o.p;
    return (float)((v + b) * o.rt);
}

constexpr int AN_THREADS = 256, AN_CHUNK = 8192;

template <typename T>
__global__ void __launch_bounds__(AN_THREADS) k_answer(const ytm_answer_args a) {
    __shared__ uint32_t cnt[AN_CHUNK];
    __shared__ Best part[AN_THREADS / 32];
    const int64_t n = blockIdx.x;
    const T *cs = (const T *)a.cs + n * a.cs_stride;
    const float *bias = a.bias ? a.bias + n * a.bias_stride : nullptr;
    const uint32_t *allowed = a.allowed ? a.allowed + n * a.allowed_stride : nullptr;
    const AnswerRow o = answer_row(a, n);
    const int64_t len = a.history ? (a.lengths ? max(0, min(a.history_len, a.lengths[n])) : a.history_len) : 0;
    Best best = {-INFINITY, INT_MAX, 0.f};
    for (int k0 = 0; k0 < a.k; k0 += AN_CHUNK) {
        const int kn = min(AN_CHUNK, a.k - k0);
        if (len) {
            for (int i = threadIdx.x; i < kn; i += AN_THREADS) cnt[i] = 0;
            __syncthreads();
            for (int64_t i = threadIdx.x; i < len; i += AN_THREADS) {
                const int64_t h = index_at(a.history, a.history_64, n * a.history_stride + i) - k0;
                if (h >= 0 && h < kn) atomicAdd(&cnt[h], 1u);
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < kn; i += AN_THREADS) {
            const int k = k0 + i;
            float z = -INFINITY;
            if (is_allowed(allowed, k)) {
                z = adjust(to_f64(cs[k]), len ? cnt[i] : 0u, bias ? (double)bias[k] : 0.0, o);
                best = merge(best, {z, k, 0.f});
            }
            if (a.adjusted) a.adjusted[n * a.k + k] = z;
        }
        if (len) __syncthreads();
    }
    for (int d = 16; d; d >>= 1) {
        const Best b = {__shfl_xor_sync(0xFFFFFFFFu, best.z, d), __shfl_xor_sync(0xFFFFFFFFu, best.k, d),
                        __shfl_xor_sync(0xFFFFFFFFu, best.s, d)};
        best = merge(best, b);
    }
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < AN_THREADS / 32; ++i) best = merge(best, part[i]);
        const bool none = best.k == INT_MAX;
        if (a.choice) a.choice[n] = none ? -1 : best.k;
        if (a.logprob) a.logprob[n] = none ? -INFINITY : best.z != best.z ? best.z : -log1pf(best.s);
    }
}

}  // namespace ytm

using namespace ytm;

extern "C" {

ytm_status ytm_answer(const ytm_answer_args *args, void *stream) {
    if (!args) return fail(YTM_ERR_ARG, "args is NULL");
    const ytm_answer_args &a = *args;
    if (a.n < 0 || a.k <= 0) return fail(YTM_ERR_ARG, "answer: needs n >= 0 rows of k >= 1 classes");
    if (a.n > INT_MAX) return fail(YTM_ERR_UNSUPPORTED, "answer: more than 2^31 - 1 rows");
    if (!is_sum_type(a.cs_type)) return fail(YTM_ERR_ARG, "answer: class sums must be int32, fp32, fp16 or bf16");
    if (a.cs_stride < 0 || a.bias_stride < 0 || a.allowed_stride < 0 || a.history_stride < 0 || a.history_len < 0)
        return fail(YTM_ERR_ARG, "answer: negative stride or length");
    if (a.n == 0) return YTM_OK;
    if (!a.cs || (a.lengths && !a.history)) return fail(YTM_ERR_ARG, "null pointer");
    cudaStream_t st = as_stream(stream);
    switch (a.cs_type) {
        case YTM_I32: k_answer<int32_t><<<(unsigned)a.n, AN_THREADS, 0, st>>>(a); break;
        case YTM_F32: k_answer<float><<<(unsigned)a.n, AN_THREADS, 0, st>>>(a); break;
        case YTM_F16: k_answer<__half><<<(unsigned)a.n, AN_THREADS, 0, st>>>(a); break;
        default: k_answer<__nv_bfloat16><<<(unsigned)a.n, AN_THREADS, 0, st>>>(a); break;
    }
    return launch_check("answer");
}

}  // extern "C"
