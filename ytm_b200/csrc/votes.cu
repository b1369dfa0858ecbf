// votes.cu — the vote of clause weights held in 4 bits with group scales.
#include "common.cuh"
#include "elem.cuh"

namespace ytm {

// Packed weights: row k holds the clauses of class k, two to a byte (clause c
// in the low half of byte c / 2 when c is even), offset by 8, row_bytes =
// 16 * ceil(C / 32).  One scale for `group` consecutive clauses of a class.

// Quantisation of weights [C][K] to [-7, 7]: with a = max |w| of the group,
// q = round-half-even(7 w / a) and scale = a / 7.  7 w and the quotient are
// formed in 64 bits, where a 24-bit w can meet a tie only exactly, so the
// rounding is that of the real quotient.  A thread per (class, group); lanes
// take consecutive classes, so every read of a weight row is coalesced.
template <typename T, typename S>
__global__ void k_q4_pack(const T *__restrict__ w, int64_t w_stride, int C, int K, int group, uint8_t *__restrict__ packed,
                          S *__restrict__ scales) {
    const int G = (int)((C + group - 1) / group);
    const int64_t row_bytes = q4_row_bytes(C);
    for (int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; u < (int64_t)K * G;
         u += (int64_t)gridDim.x * blockDim.x) {
        const int k = (int)(u % K), g = (int)(u / K);
        const int c0 = g * group, c1 = min(C, c0 + group);
        double a = 0.0;
        for (int c = c0; c < c1; ++c) a = fmax(a, fabs((double)to_f64(w[(int64_t)c * w_stride + k])));
        const S s = from_f32<S>((float)(a / 7.0));
        scales[(int64_t)k * G + g] = s;
        const int64_t end = min((int64_t)c0 + group, row_bytes * 2);
        for (int c = c0; c < end; c += 2) {
            uint32_t byte = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                double q = 0.0;
                if (c + h < c1 && a > 0.0) q = fmin(7.0, fmax(-7.0, rint(to_f64(w[(int64_t)(c + h) * w_stride + k]) * 7.0 / a)));
                byte |= (uint32_t)((int)q + 8) << (4 * h);
            }
            packed[(int64_t)k * row_bytes + c / 2] = (uint8_t)byte;
        }
    }
}

// y[n][k] = bias[k] + sum_g scale[k][g] * sum_{c in g} (q - 8) x[n][c].
// A block per (class, sample); a thread takes 32 clauses at a time, whose
// products it sums in fp32 before the scale.
template <int X, typename S, typename Y>
__global__ void __launch_bounds__(256) k_q4_votes(const void *__restrict__ x, int64_t x_stride, int C,
                                                  const uint8_t *__restrict__ packed, const S *__restrict__ scales,
                                                  int group, int K, const float *__restrict__ bias, Y *__restrict__ y) {
    const int64_t n = blockIdx.y;
    const int k = blockIdx.x, G = (C + group - 1) / group;
    const int units = (C + 31) / 32;
    const uint4 *row = reinterpret_cast<const uint4 *>(packed + (int64_t)k * q4_row_bytes(C));
    float acc = 0.f;
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
        const uint4 q = row[u];
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const int c = u * 32 + j;
            if (c < C) part += (float)((int)((w[j / 8] >> (4 * (j % 8))) & 15u) - 8) * load_x<X>(x, n * x_stride, c);
        }
        acc += part * to_f32(scales[(int64_t)k * G + u * 32 / group]);
    }
    __shared__ float s[8];
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xFFFFFFFFu, acc, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) acc += s[i];
        y[n * K + k] = from_f32<Y>(acc + (bias ? bias[k] : 0.f));
    }
}

template <int X, typename S>
static ytm_status launch_votes(const void *x, int64_t x_stride, int64_t N, int C, const uint8_t *packed, const S *scales,
                               int group, int K, const float *bias, void *y, int y_type, cudaStream_t st) {
    for (int64_t i = 0; i < N; i += 65535) {
        const int64_t m = N - i < 65535 ? N - i : 65535;
        const dim3 grid((unsigned)K, (unsigned)m);
        const char *xi = (const char *)x + i * x_stride * type_bytes(X);
        switch (y_type) {
            case YTM_F32: k_q4_votes<X, S, float><<<grid, 256, 0, st>>>(xi, x_stride, C, packed, scales, group, K, bias, (float *)y + i * K); break;
            case YTM_F16: k_q4_votes<X, S, __half><<<grid, 256, 0, st>>>(xi, x_stride, C, packed, scales, group, K, bias, (__half *)y + i * K); break;
            default: k_q4_votes<X, S, __nv_bfloat16><<<grid, 256, 0, st>>>(xi, x_stride, C, packed, scales, group, K, bias, (__nv_bfloat16 *)y + i * K); break;
        }
        ytm_status rc = launch_check("q4 votes");
        if (rc) return rc;
    }
    return YTM_OK;
}

template <int X>
static ytm_status launch_votes_x(const void *x, int64_t x_stride, int64_t N, int C, const uint8_t *packed,
                                 const void *scales, int scale_type, int group, int K, const float *bias, void *y,
                                 int y_type, cudaStream_t st) {
    switch (scale_type) {
        case YTM_F32: return launch_votes<X>(x, x_stride, N, C, packed, (const float *)scales, group, K, bias, y, y_type, st);
        case YTM_F16: return launch_votes<X>(x, x_stride, N, C, packed, (const __half *)scales, group, K, bias, y, y_type, st);
        default: return launch_votes<X>(x, x_stride, N, C, packed, (const __nv_bfloat16 *)scales, group, K, bias, y, y_type, st);
    }
}

static ytm_status check_q4(int32_t C, int32_t K, int32_t group, int32_t scale_type) {
    if (C <= 0 || K <= 0) return fail(YTM_ERR_ARG, "q4: clauses and classes must be positive");
    if (C > (1 << 30)) return fail(YTM_ERR_UNSUPPORTED, "q4: more than 2^30 clauses");
    if (group != 32 && group != 64 && group != 128) return fail(YTM_ERR_ARG, "q4: group must be 32, 64 or 128");
    if (!is_float_type(scale_type)) return fail(YTM_ERR_ARG, "q4: scales must be fp32, fp16 or bf16");
    return YTM_OK;
}

}  // namespace ytm

using namespace ytm;

extern "C" {

ytm_status ytm_q4_pack(const void *weights, int32_t w_type, int64_t w_stride, int32_t C, int32_t K, int32_t group,
                       uint8_t *packed, void *scales, int32_t scale_type, void *stream) {
    ytm_status rc = check_q4(C, K, group, scale_type);
    if (rc) return rc;
    if (w_type != YTM_I32 && w_type != YTM_F32) return fail(YTM_ERR_ARG, "q4: weights must be int32 or fp32");
    if (w_stride < K) return fail(YTM_ERR_ARG, "q4: weight row stride below the class count");
    if (!weights || !packed || !scales) return fail(YTM_ERR_ARG, "null pointer");
    cudaStream_t st = as_stream(stream);
    const uint64_t units = cdiv(C, group) * (uint64_t)K;
    const unsigned grid = (unsigned)std::min<uint64_t>(cdiv(units, 128), (uint64_t)sm_count() * 64);
    if (w_type == YTM_I32) {
        const int32_t *w = (const int32_t *)weights;
        if (scale_type == YTM_F32) k_q4_pack<<<grid, 128, 0, st>>>(w, w_stride, C, K, group, packed, (float *)scales);
        else if (scale_type == YTM_F16) k_q4_pack<<<grid, 128, 0, st>>>(w, w_stride, C, K, group, packed, (__half *)scales);
        else k_q4_pack<<<grid, 128, 0, st>>>(w, w_stride, C, K, group, packed, (__nv_bfloat16 *)scales);
    } else {
        const float *w = (const float *)weights;
        if (scale_type == YTM_F32) k_q4_pack<<<grid, 128, 0, st>>>(w, w_stride, C, K, group, packed, (float *)scales);
        else if (scale_type == YTM_F16) k_q4_pack<<<grid, 128, 0, st>>>(w, w_stride, C, K, group, packed, (__half *)scales);
        else k_q4_pack<<<grid, 128, 0, st>>>(w, w_stride, C, K, group, packed, (__nv_bfloat16 *)scales);
    }
    return launch_check("q4 pack");
}

ytm_status ytm_q4_votes(const void *x, int32_t x_type, int64_t x_stride, int64_t N, int32_t C, const uint8_t *packed,
                        const void *scales, int32_t scale_type, int32_t group, int32_t K, const float *bias, void *y,
                        int32_t y_type, void *stream) {
    ytm_status rc = check_q4(C, K, group, scale_type);
    if (rc) return rc;
    if (N < 0) return fail(YTM_ERR_ARG, "N < 0");
    if (!is_float_type(x_type) && x_type != YTM_BITS) return fail(YTM_ERR_ARG, "q4: x must be fp32, fp16, bf16 or packed bits");
    if (!is_float_type(y_type)) return fail(YTM_ERR_ARG, "q4: votes must be fp32, fp16 or bf16");
    if (x_stride < 0) return fail(YTM_ERR_ARG, "q4: negative row stride");
    if (N == 0) return YTM_OK;
    if (!x || !packed || !scales || !y) return fail(YTM_ERR_ARG, "null pointer");
    if ((uintptr_t)packed % 16) return fail(YTM_ERR_ARG, "q4: packed weights must start on a 16-byte boundary");
    cudaStream_t st = as_stream(stream);
    switch (x_type) {
        case YTM_F32: return launch_votes_x<YTM_F32>(x, x_stride, N, C, packed, scales, scale_type, group, K, bias, y, y_type, st);
        case YTM_F16: return launch_votes_x<YTM_F16>(x, x_stride, N, C, packed, scales, scale_type, group, K, bias, y, y_type, st);
        case YTM_BF16: return launch_votes_x<YTM_BF16>(x, x_stride, N, C, packed, scales, scale_type, group, K, bias, y, y_type, st);
        default: return launch_votes_x<YTM_BITS>(x, x_stride, N, C, packed, scales, scale_type, group, K, bias, y, y_type, st);
    }
}

}  // extern "C"
