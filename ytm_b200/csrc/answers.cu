// answers.cu — from class sums to an answer: biases, allowed classes and
// penalties with the choice of a class, and the cross entropy of adjusted
// class sums with its gradients.
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

__device__ __forceinline__ int64_t index_at(const void *p, int is64, int64_t i) {
    return is64 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
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

// -------------------------------------------------------------- the loss
// z = allowed ? (v + b) / t : -inf, loss = w (log sum exp z - z_y),
// d = w (p - 1[y]), gradients d / t, sum_n d / t and -sum d z / t.

// One rounding for each operation: a product fused into z - m would leave the
// largest class's exponent off 0.
__device__ __forceinline__ float loss_z(float v, float b, float rt) { return __fmul_rn(__fadd_rn(v, b), rt); }

struct LossRow {
    float m, total;  // largest z and sum exp(z - m)
    float w;         // 0: the row counts for nothing
    int y;
};

template <typename T>
__global__ void __launch_bounds__(AN_THREADS) k_loss_rows(const ytm_loss_args a, LossRow *__restrict__ rows,
                                                          double *__restrict__ dts) {
    __shared__ float sm[AN_THREADS / 32], ss[AN_THREADS / 32];
    __shared__ double sd[AN_THREADS / 32];
    const int64_t n = blockIdx.x;
    const T *cs = (const T *)a.cs + n * a.cs_stride;
    const uint32_t *allowed = a.allowed ? a.allowed + n * a.allowed_stride : nullptr;
    const float rt = 1.f / (a.temperature ? *a.temperature : a.temperature_all);
    const int64_t y64 = index_at(a.target, a.target_64, n);
    const float w0 = a.weight ? a.weight[n] : 1.f;
    const bool use = y64 >= 0 && y64 < a.k && w0 != 0.f;
    const int y = use ? (int)y64 : -1;
    const bool open = use && is_allowed(allowed, y);
    T *dcs = a.dcs ? (T *)a.dcs + n * a.k : nullptr;
    if (!open) {  // no label, or one that the mask forbids: no gradient
        if (dcs)
            for (int k = threadIdx.x; k < a.k; k += AN_THREADS) dcs[k] = T(0.f);
        if (threadIdx.x == 0) {
            a.loss[n] = use ? w0 * INFINITY : 0.f;
            rows[n] = {0.f, 1.f, 0.f, -1};
            dts[n] = 0.0;
        }
        return;
    }
    float m = -INFINITY, s = 0.f;
    for (int k = threadIdx.x; k < a.k; k += AN_THREADS) {
        if (!is_allowed(allowed, k)) continue;
        const float z = loss_z(to_f32(cs[k]), a.bias ? a.bias[k] : 0.f, rt);
        if (z > m) { s = s * expf(m - z) + 1.f; m = z; }
        else if (z != -INFINITY) s += expf(z - m);  // NaN gets into the sum here
    }
    for (int d = 16; d; d >>= 1) {
        const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, d), s2 = __shfl_xor_sync(0xFFFFFFFFu, s, d);
        const float mm = fmaxf(m, m2);
        s = (m == mm ? s : s * expf(m - mm)) + (m2 == mm ? s2 : s2 * expf(m2 - mm));
        m = mm;
    }
    if ((threadIdx.x & 31) == 0) { sm[threadIdx.x >> 5] = m; ss[threadIdx.x >> 5] = s; }
    __syncthreads();
    m = sm[0];
    for (int i = 1; i < AN_THREADS / 32; ++i) m = fmaxf(m, sm[i]);
    s = 0.f;
    for (int i = 0; i < AN_THREADS / 32; ++i) s += sm[i] == m ? ss[i] : ss[i] * expf(sm[i] - m);
    const float zy = loss_z(to_f32(cs[y]), a.bias ? a.bias[y] : 0.f, rt);
    const float wt = w0 * rt;
    double dt = 0.0;
    for (int k = threadIdx.x; k < a.k; k += AN_THREADS) {
        float d = 0.f;
        if (is_allowed(allowed, k)) {
            const float z = loss_z(to_f32(cs[k]), a.bias ? a.bias[k] : 0.f, rt);
            const float p = expf(z - m) / s - (k == y ? 1.f : 0.f);
            if (p != 0.f) dt += (double)(p * (z - m));
            d = p * wt;
        }
        if (dcs) dcs[k] = from_f32<T>(d);
    }
    for (int d = 16; d; d >>= 1) dt += __shfl_xor_sync(0xFFFFFFFFu, dt, d);
    if ((threadIdx.x & 31) == 0) sd[threadIdx.x >> 5] = dt;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < AN_THREADS / 32; ++i) dt += sd[i];
        a.loss[n] = w0 * (logf(s) - (zy - m));
        rows[n] = {m, s, w0, y};
        dts[n] = -dt * (double)w0 * (double)rt;
    }
}

template <>
__device__ __forceinline__ int32_t from_f32<int32_t>(float v) { return (int32_t)v; }  // never stored

// Column sums of the gradients, and the temperature's (block 0 of the extra row).
template <typename T>
__global__ void __launch_bounds__(AN_THREADS) k_loss_cols(const ytm_loss_args a, const LossRow *__restrict__ rows,
                                                          const double *__restrict__ dts) {
    if (blockIdx.x == gridDim.x - 1) {
        __shared__ double sd[AN_THREADS];
        double s = 0.0;
        for (int64_t n = threadIdx.x; n < a.n; n += AN_THREADS) s += dts[n];
        sd[threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.x == 0 && a.dtemperature) {
            for (int i = 1; i < AN_THREADS; ++i) s += sd[i];
            *a.dtemperature = (float)s;
        }
        return;
    }
    const int k = blockIdx.x * AN_THREADS + threadIdx.x;
    if (k >= a.k || !a.dbias) return;
    const float rt = 1.f / (a.temperature ? *a.temperature : a.temperature_all);
    const float b = a.bias ? a.bias[k] : 0.f;
    double s = 0.0;
    for (int64_t n = 0; n < a.n; ++n) {
        const LossRow r = rows[n];
        if (r.y < 0 || !is_allowed(a.allowed ? a.allowed + n * a.allowed_stride : nullptr, k)) continue;
        const float z = loss_z(to_f32(((const T *)a.cs)[n * a.cs_stride + k]), b, rt);
        s += (double)((expf(z - r.m) / r.total - (k == r.y ? 1.f : 0.f)) * r.w);
    }
    a.dbias[k] = (float)(s * (double)rt);
}

static bool bad_type(int t) { return !is_float_type(t) && t != YTM_I32; }

}  // namespace ytm

using namespace ytm;

extern "C" {

ytm_status ytm_answer(const ytm_answer_args *args, void *stream) {
    if (!args) return fail(YTM_ERR_ARG, "args is NULL");
    const ytm_answer_args &a = *args;
    if (a.n < 0 || a.k <= 0) return fail(YTM_ERR_ARG, "answer: needs n >= 0 rows of k >= 1 classes");
    if (a.n > INT_MAX) return fail(YTM_ERR_UNSUPPORTED, "answer: more than 2^31 - 1 rows");
    if (bad_type(a.cs_type)) return fail(YTM_ERR_ARG, "answer: class sums must be int32, fp32, fp16 or bf16");
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

uint64_t ytm_class_loss_workspace_bytes(int64_t n, int32_t k) {
    (void)k;
    return n <= 0 ? 0 : (uint64_t)n * (sizeof(LossRow) + sizeof(double));
}

ytm_status ytm_class_loss(const ytm_loss_args *args, void *workspace, void *stream) {
    if (!args) return fail(YTM_ERR_ARG, "args is NULL");
    const ytm_loss_args &a = *args;
    if (a.n < 0 || a.k <= 0) return fail(YTM_ERR_ARG, "class loss: needs n >= 0 rows of k >= 1 classes");
    if (a.n > INT_MAX) return fail(YTM_ERR_UNSUPPORTED, "class loss: more than 2^31 - 1 rows");
    if (bad_type(a.cs_type)) return fail(YTM_ERR_ARG, "class loss: class sums must be int32, fp32, fp16 or bf16");
    if (a.cs_type == YTM_I32 && a.dcs) return fail(YTM_ERR_ARG, "class loss: int32 class sums have no gradient");
    if (a.cs_stride < 0 || a.allowed_stride < 0) return fail(YTM_ERR_ARG, "class loss: negative stride");
    cudaStream_t st = as_stream(stream);
    ytm_status rc;
    if (a.n == 0) {
        if (a.dbias && (rc = cuda_check(cudaMemsetAsync(a.dbias, 0, (size_t)a.k * 4, st), "memset"))) return rc;
        if (a.dtemperature && (rc = cuda_check(cudaMemsetAsync(a.dtemperature, 0, 4, st), "memset"))) return rc;
        return YTM_OK;
    }
    if (!a.cs || !a.target || !a.loss || !workspace) return fail(YTM_ERR_ARG, "null pointer");
    double *dts = (double *)workspace;
    LossRow *rows = (LossRow *)(dts + a.n);
    const unsigned cols = (unsigned)cdiv(a.k, AN_THREADS) + 1;
#define YTM_LOSS(T)                                                            \
    k_loss_rows<T><<<(unsigned)a.n, AN_THREADS, 0, st>>>(a, rows, dts);        \
    if ((rc = launch_check("class loss"))) return rc;                          \
    k_loss_cols<T><<<cols, AN_THREADS, 0, st>>>(a, rows, dts);
    switch (a.cs_type) {
        case YTM_I32: YTM_LOSS(int32_t) break;
        case YTM_F32: YTM_LOSS(float) break;
        case YTM_F16: YTM_LOSS(__half) break;
        default: YTM_LOSS(__nv_bfloat16) break;
    }
#undef YTM_LOSS
    return launch_check("class loss sums");
}

}  // extern "C"
