// class_loss.cu — cross entropy of biased, masked, tempered class sums with
// its gradients.
//
// With u = v + b (allowed classes), m = max u and c = log2(e) / t,
//   x_k = (u_k - m) c, e_k = 2^x_k, s = sum e, h = sum e x
//   loss = w (ln s - (u_y - m) / t)
//   dcs_k = (w / t) (e_k / s - 1[k = y]),  dbias = sum_n dcs
//   dt = -(ln 2 / t) sum_n w (h / s - x_y)
// so that h gives the temperature's gradient without another look at u.  The
// factor comes after the difference: a row of the type's lowest value, whose
// product with c has left the type, keeps its u - m = 0.
//
// fp32 rounds whole numbers above 2^24.  Where a row's largest u reaches 2^23, they
// are taken less a whole number r near it, in 64 bits, so that their differences
// stay: that changes neither the loss nor a gradient.  r is 0 for other rows, whose
// rounded classes lie at least 2^23 below and so are off by 2^-23 of that at most.
//
// Rows of up to 512 classes stay in the registers of 4 to 32 threads between
// the sum and the gradient (k_loss_small).  Longer rows take two streams over
// the class sums, which need no barrier: k_loss_stat for (m, s, h), then
// k_loss_grad, whose threads keep their classes over a chunk of rows.  Both
// kernels sum dbias in registers and leave one part per team or chunk, which
// k_loss_join adds in a fixed order.
//
// Measured with a bias, calls back to back: 262144 x 100 int32 53 us (the first
// kernel 50, 2.1 TB/s: 37 instructions a class, 27 us of issue, which the 16 warps
// of an SM, with 122 registers a thread, fill to 57%: they wait for their loads and
// for the row's sums), fp32 62, bf16 56, bf16 with row masks 72; 2047 x 32001 bf16
// 119 us, with row masks 145 (393 MB in two streams, 3.3 and 2.7 TB/s; both issue
// 57% of the time, 60 and 64 registers: instructions, and loads waited for; the
// first reads the bias again for every row, 15 us of it).
// One pass with a cluster a row, the exponentials kept, took 583 us: labels and
// clusters waited for, with half of the clusters that would fill the SMs.
#include <float.h>
#include <limits.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "elem.cuh"

namespace ytm {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));  // within 2 steps, 2^0 = 1 exactly
    return y;
}

constexpr float WHOLE = 8388608.f;  // 2^23

// Whether whole numbers with the largest u of m are to be taken less an r.
__device__ __forceinline__ bool large_whole(float m) { return fabsf(m) >= WHOLE && m != -INFINITY; }

// A class sum less the row's r.
template <typename T>
__device__ __forceinline__ float class_sum(T v, int) { return to_f32(v); }
__device__ __forceinline__ float class_sum(int32_t v, int r) { return r ? (float)((int64_t)v - r) : (float)v; }

// u and x, the same operations for every use of a class's, so that the largest
// class's x is 0 exactly.
__device__ __forceinline__ float loss_u(float v, float b) { return __fadd_rn(v, b); }
__device__ __forceinline__ float loss_x(float u, float m, float c) { return __fmul_rn(__fsub_rn(u, m), c); }

// A row's label, weight and label's mask bit.  y < 0: the row counts for
// nothing; open: it has a gradient.
struct LossLabel {
    int y;
    float w;
    bool open;
};

__device__ __forceinline__ LossLabel loss_label(const ytm_loss_args &a, int64_t n) {
    LossLabel r;
    const int64_t y = index_at(a.target, a.target_64, n);
    r.w = a.weight ? a.weight[n] : 1.f;
    r.y = y >= 0 && y < a.k && r.w != 0.f ? (int)y : -1;
    r.open = r.y >= 0 && is_allowed(a.allowed ? a.allowed + n * a.allowed_stride : nullptr, r.y);
    return r;
}

__device__ __forceinline__ float loss_rt(const ytm_loss_args &a) {
    return 1.f / (a.temperature ? *a.temperature : a.temperature_all);
}
// Not 0, so that a masked class's -inf stays one under an infinite temperature.
__device__ __forceinline__ float loss_c(float rt) { return fmaxf(rt * LOG2E, FLT_MIN); }

// Partial sums of the teams or chunks: dbias [G][k], dt / (-ln 2 / t) [G].
struct LossPart {
    float *db;
    double *dt;
};

// -------------------------------------------------- rows of few classes
// TPR threads hold a row, E classes each (e TPR + lane), in pairs for the paired
// arithmetic.  The label's class is closed there and taken apart, by every thread
// of the row from the label's own load: its gradient is -(w / t) times the others'
// share, without the cancellation of p_y - 1.  The lane that holds the class adds
// that to its own sum in shared memory and stores the class's gradient once more.

constexpr int LS_THREADS = 256;

template <typename T, int TPR, int E>
__global__ void __launch_bounds__(LS_THREADS, E == 16 ? 2 : E == 8 ? 3 : 4) k_loss_small(const ytm_loss_args a, const LossPart part) {
    constexpr int ROWS = LS_THREADS / TPR, SLOTS = TPR * E;
    extern __shared__ float red[];  // [ROWS][SLOTS]: sums of the labels' gradients, at the end dbias of the teams
    __shared__ double red_dt[LS_THREADS / 32];
    const int lane = threadIdx.x % TPR, team = threadIdx.x / TPR, K = a.k;
    float *const mine = red + team * SLOTS + lane;
    const float rt = loss_rt(a), c = loss_c(rt);
    const F2 c2 = pair(c, c);
    F2 b[E / 2], acc[E / 2];
    uint32_t shared_open = 0;
    const uint32_t *const shared_mask = a.allowed_stride ? nullptr : a.allowed;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int k = e * TPR + lane;
        if (k < K && is_allowed(shared_mask, k)) shared_open |= 1u << e;
        mine[e * TPR] = 0.f;
    }
#pragma unroll
    for (int q = 0; q < E / 2; ++q) {
        const int k = 2 * q * TPR + lane;
        b[q] = pair(a.bias && k < K ? a.bias[k] : 0.f, a.bias && k + TPR < K ? a.bias[k + TPR] : 0.f);
        acc[q] = pair(0.f, 0.f);
    }
    // A row's loads are issued a round ahead, and its label's two rounds ahead,
    // so that the label's class sum, which waits for the label, comes in time.
    struct Row {
        T v[E];
        uint32_t open;
        T vy;
        float by;
        LossLabel label;
    };
    const auto clamped = [&](int64_t n) { return n < a.n ? n : a.n - 1; };
    const auto fetch = [&](int64_t n, const LossLabel &label) {
        Row r;
        const T *row = (const T *)a.cs + n * a.cs_stride, *cs = row + lane;
        r.open = shared_open;
        r.label = label;
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
        const int y = max(label.y, 0);
        r.vy = row[y];
        r.by = a.bias ? a.bias[y] : 0.f;
        return r;
    };
    double dt = 0.0;
    [[maybe_unused]] float top = 0.f;  // the largest |m|
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t n0 = (int64_t)blockIdx.x * ROWS;
    LossLabel label1 = loss_label(a, clamped(n0 + step + team));
    Row next = fetch(clamped(n0 + team), loss_label(a, clamped(n0 + team)));
    for (; n0 < a.n; n0 += step) {
        const Row row = next;
        if (n0 + step < a.n) {
            next = fetch(clamped(n0 + step + team), label1);
            label1 = loss_label(a, clamped(n0 + 2 * step + team));
        }
        const bool live = n0 + team < a.n;
        const int64_t n = clamped(n0 + team);
        // (of rows without a label, or with a closed one, nothing is used)
        const uint32_t y = (uint32_t)row.label.y;
        const bool own = y % TPR == lane;
        const uint32_t open = own ? row.open & ~(1u << (y / TPR % 32)) : row.open;  // without the label's class
        const float uy = loss_u(to_f32(row.vy), row.by);
        float z[E], m = uy;
#pragma unroll
        for (int q = 0; q < E / 2; ++q) {
            float x0, x1;
            split(add2(pair(to_f32(row.v[2 * q]), to_f32(row.v[2 * q + 1])), b[q]), x0, x1);
            z[2 * q] = open & (1u << (2 * q)) ? x0 : -INFINITY;
            z[2 * q + 1] = open & (2u << (2 * q)) ? x1 : -INFINITY;
            m = fmaxf(m, fmaxf(z[2 * q], z[2 * q + 1]));
        }
#pragma unroll
        for (int d = TPR / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
        F2 s2 = pair(0.f, 0.f), h2 = s2;
        const F2 m2 = pair(-m, -m);
#pragma unroll
        for (int q = 0; q < E / 2; ++q) {
            float x0, x1;
            split(mul2(add2(pair(z[2 * q], z[2 * q + 1]), m2), c2), x0, x1);
            z[2 * q] = ex2(x0);
            z[2 * q + 1] = ex2(x1);
            const F2 e2 = pair(z[2 * q], z[2 * q + 1]);
            s2 = add2(s2, e2);
            h2 = fma2(e2, pair(fmaxf(x0, -1024.f), fmaxf(x1, -1024.f)), h2);  // 0 * -inf counts for nothing
        }
        float s, h, t;
        split(s2, s, t);
        s += t;
        split(h2, h, t);
        h += t;
#pragma unroll
        for (int d = TPR / 2; d; d >>= 1) {
            s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
            h += __shfl_xor_sync(0xFFFFFFFFu, h, d);
        }
        const bool use = live && row.label.open;
        if constexpr (std::is_integral<T>::value) top = fmaxf(top, use ? fabsf(m) : 0.f);
        const float xy = loss_x(uy, m, c), ey = ex2(xy), others = s;
        s += ey;
        const float rs = 1.f / s, f = row.label.w * rt * rs;
        if (use) {
            const F2 f2 = pair(f, f);
#pragma unroll
            for (int q = 0; q < E / 2; ++q) {
                const F2 d2 = mul2(pair(z[2 * q], z[2 * q + 1]), f2);
                acc[q] = add2(acc[q], d2);
                split(d2, z[2 * q], z[2 * q + 1]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) z[e] = 0.f;
        }
        if constexpr (!std::is_integral<T>::value) {
            if (a.dcs && live) {
                T *const out = (T *)a.dcs + n * (int64_t)K + lane;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (e * TPR + lane < K) out[e * TPR] = from_f32<T>(z[e]);
            }
        }
        if (use && own) {
            const float dy = -others * f;
            mine[(int)y - lane] += dy;
            if constexpr (!std::is_integral<T>::value) {
                if (a.dcs) ((T *)a.dcs)[n * (int64_t)K + y] = from_f32<T>(dy);
            }
        }
        if (lane == 0 && live) {
            const float w = row.label.w, gap = uy - m;
            a.loss[n] = use ? w * (logf(s) - gap * rt) : row.label.y >= 0 ? w * INFINITY : 0.f;
            h = fmaf(ey, fmaxf(xy, -1024.f), h);
            if (use) dt += (double)w * ((double)(h * rs) - (double)gap * (double)c);
        }
    }
    if constexpr (std::is_integral<T>::value) {
        // Large whole numbers were among the block's rows: all of them once more, from
        // memory and class by class, as such rows are rare.
        if (__syncthreads_or(large_whole(top))) {
#pragma unroll
            for (int e = 0; e < E; ++e) mine[e * TPR] = 0.f;
#pragma unroll
            for (int q = 0; q < E / 2; ++q) acc[q] = pair(0.f, 0.f);
            dt = 0.0;
            for (n0 = (int64_t)blockIdx.x * ROWS; n0 < a.n; n0 += step) {
                const int64_t n = clamped(n0 + team);
                const LossLabel label = loss_label(a, n);
                const T *cs = (const T *)a.cs + n * a.cs_stride;
                const uint32_t *allowed = a.allowed ? a.allowed + n * a.allowed_stride : nullptr;
                const int y = label.y, last = n0 + team < a.n && label.open ? K : 0;  // 0: the row has its loss and no gradient
                const auto each = [&](auto f) {
                    for (int k = lane; k < last; k += TPR)
                        if (is_allowed(allowed, k)) f(k);
                };
                const auto over_team = [&](auto v, auto join) {
#pragma unroll
                    for (int d = TPR / 2; d; d >>= 1) v = join(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
                    return v;
                };
                const auto sum = [](float p, float q) { return p + q; };
                int r = INT_MIN;
                each([&](int k) { r = max(r, cs[k]); });
                r = over_team(r, [](int p, int q) { return max(p, q); });
                const auto u = [&](int k) { return loss_u(class_sum(cs[k], r), a.bias ? a.bias[k] : 0.f); };
                float m = -INFINITY, s = 0.f, h = 0.f;
                each([&](int k) { m = fmaxf(m, u(k)); });
                m = over_team(m, [](float p, float q) { return fmaxf(p, q); });
                each([&](int k) {
                    const float x = loss_x(u(k), m, c), e = ex2(x);
                    if (k != y) s += e, h = fmaf(e, fmaxf(x, -1024.f), h);
                });
                s = over_team(s, sum);
                h = over_team(h, sum);
                if (!last) continue;
                const float uy = u(y), xy = loss_x(uy, m, c), ey = ex2(xy), others = s;
                s += ey;
                h = fmaf(ey, fmaxf(xy, -1024.f), h);
                const float f = label.w * rt / s;
                each([&](int k) { mine[k - lane] += k == y ? -others * f : ex2(loss_x(u(k), m, c)) * f; });
                if (lane == 0) {
                    a.loss[n] = label.w * (logf(s) - (uy - m) * rt);
                    dt += (double)label.w * ((double)(h / s) - (double)(uy - m) * (double)c);
                }
            }
        }
    }
    // the block's sums, teams in order
#pragma unroll
    for (int q = 0; q < E / 2; ++q) {
        float x, y;
        split(acc[q], x, y);
        mine[2 * q * TPR] += x;
        mine[(2 * q + 1) * TPR] += y;
    }
    for (int d = 16; d; d >>= 1) dt += __shfl_xor_sync(0xFFFFFFFFu, dt, d);
    if ((threadIdx.x & 31) == 0) red_dt[threadIdx.x >> 5] = dt;
    __syncthreads();
    if (a.dbias)
        for (int k = threadIdx.x; k < K; k += LS_THREADS) {
            float t = 0.f;
            for (int i = 0; i < ROWS; ++i) t += red[i * SLOTS + k];
            if (gridDim.x == 1) a.dbias[k] = t;
            else part.db[(int64_t)blockIdx.x * K + k] = t;
        }
    if (threadIdx.x == 0) {
        for (int i = 1; i < LS_THREADS / 32; ++i) dt += red_dt[i];
        if (gridDim.x > 1) part.dt[blockIdx.x] = dt;
        else if (a.dtemperature) *a.dtemperature = (float)(-dt * (double)LN2 * (double)rt);
    }
}

// -------------------------------------------------- rows of many classes

// m: the largest u, less r.
struct LossStat {
    float m, s, h;
    int r;
};

// The largest u, less another r: exact where that is near.
__device__ __forceinline__ float largest_less(const LossStat &a, int r) {
    return (float)((double)a.m + (double)((int64_t)a.r - r));
}

// r next to the largest u (unless that is no number, or far from any class sum).
__device__ __forceinline__ void bring_near(LossStat &a) {
    if (!(fabsf(a.m) < 2.f * WHOLE)) return;
    const int64_t r = (int64_t)a.r + __float2int_rn(a.m);
    if (r != (int)r) return;
    a.m = largest_less(a, (int)r);
    a.r = (int)r;
}

__device__ __forceinline__ LossStat merge_alike(const LossStat &a, const LossStat &b, float c) {
    const float m = fmaxf(a.m, b.m);
    // a.m == m: the factor is 1 also where both are infinite
    const float da = a.m == m ? 0.f : loss_x(a.m, m, c), db = b.m == m ? 0.f : loss_x(b.m, m, c);
    const float fa = ex2(da), fb = ex2(db);
    // separate roundings: merge(a, b) == merge(b, a), so all lanes of an
    // exchange end with the same bits
    return {m, __fadd_rn(__fmul_rn(fa, a.s), __fmul_rn(fb, b.s)),
            __fadd_rn(__fmul_rn(fa, fmaf(a.s, fmaxf(da, -1024.f), a.h)),
                      __fmul_rn(fb, fmaf(b.s, fmaxf(db, -1024.f), b.h))), a.r};
}

// Of statistics less different r.  A call, as such rows are rare and this would be
// in the way of others.
__device__ __noinline__ LossStat merge_apart(LossStat a, LossStat b, float c) {
    if (a.m == -INFINITY) {
        a.r = b.r;
    } else if (b.m == -INFINITY) {
        b.r = a.r;
    } else {
        bring_near(a);
        bring_near(b);
        const int r = max(a.r, b.r);
        a.m = largest_less(a, r);
        b.m = largest_less(b, r);
        a.r = r;
    }
    return merge_alike(a, b, c);
}

template <typename T>
__device__ __forceinline__ LossStat merge(const LossStat &a, const LossStat &b, float c) {
    if (std::is_integral<T>::value && a.r != b.r) return merge_apart(a, b, c);
    return merge_alike(a, b, c);
}

// Over `lanes` neighbouring lanes of a whole warp.
template <typename T>
__device__ __forceinline__ LossStat merge_lanes(LossStat a, int lanes, float c) {
    if constexpr (std::is_integral<T>::value) {
        if (__any_sync(0xFFFFFFFFu, a.r != 0)) {
            for (int d = lanes / 2; d; d >>= 1)
                a = merge<T>(a, {__shfl_xor_sync(0xFFFFFFFFu, a.m, d), __shfl_xor_sync(0xFFFFFFFFu, a.s, d),
                                 __shfl_xor_sync(0xFFFFFFFFu, a.h, d), __shfl_xor_sync(0xFFFFFFFFu, a.r, d)}, c);
            return a;
        }
    }
#pragma unroll
    for (int d = lanes / 2; d; d >>= 1)
        a = merge_alike(a, {__shfl_xor_sync(0xFFFFFFFFu, a.m, d), __shfl_xor_sync(0xFFFFFFFFu, a.s, d),
                            __shfl_xor_sync(0xFFFFFFFFu, a.h, d), 0}, c);
    return a;
}

constexpr int LB_THREADS = 256;

// A row of class sums (or gradients) in 16-byte vectors from the 16-byte
// boundary at or below its start: class k is element off + k of them.
template <typename T>
struct RowVecs {
    static constexpr int V = 16 / (int)sizeof(T);
    const T *row;
    int off;

    __device__ __forceinline__ RowVecs(const void *base, int64_t row_index, int64_t stride)
        : row((const T *)base + row_index * stride), off((int)((uintptr_t)row % 16 / sizeof(T))) {}

    // Vectors first .. end - 1 lie inside the row; `slack` more classes must
    // follow them.  The classes before and behind are taken one by one.
    __device__ __forceinline__ int first() const { return off ? 1 : 0; }
    __device__ __forceinline__ int end(int K, int slack = 0) const { return max(first(), (int)(((int64_t)off + K - slack) / V)); }
    __device__ __forceinline__ const uint4 *at(int i) const { return (const uint4 *)(row - off + (int64_t)i * V); }
};

// Classes 2 q and 2 q + 1 of a vector.
template <typename T>
__device__ __forceinline__ F2 class_pair(const uint4 &raw, int q) {
    const T *v = (const T *)&raw;
    return pair(to_f32(v[2 * q]), to_f32(v[2 * q + 1]));
}

// Bits j: class k + j (of V, all of them in the row) is allowed.
template <int V>
__device__ __forceinline__ uint32_t open_classes(const uint32_t *allowed, int k) {
    if (!allowed) return ~0u;
    const uint32_t *w = allowed + (k >> 5);
    return __funnelshift_r(w[0], (k & 31) + V > 32 ? w[1] : 0u, k & 31);
}

// bias[k .. k + V), k = R below a multiple of four; reads up to R behind.
template <int V, int R>
__device__ __forceinline__ void load_bias(const float *bias, int k, F2 (&b)[V / 2]) {
    if (!bias) {
#pragma unroll
        for (int q = 0; q < V / 2; ++q) b[q] = pair(0.f, 0.f);
    } else if ((uintptr_t)bias % 16 == 0) {
        float f[V + 4];  // from the boundary at or below k
        const float *from = bias + (R ? k + R - 4 : k);
#pragma unroll
        for (int q = 0; q < (R ? V / 4 + 1 : V / 4); ++q) *(float4 *)&f[4 * q] = *(const float4 *)(from + 4 * q);
#pragma unroll
        for (int q = 0; q < V / 2; ++q) b[q] = pair(f[(R ? 4 - R : 0) + 2 * q], f[(R ? 4 - R : 0) + 2 * q + 1]);
    } else {
#pragma unroll
        for (int q = 0; q < V / 2; ++q) b[q] = pair(bias[k + 2 * q], bias[k + 2 * q + 1]);
    }
}

// A thread's round (vectors i0, i0 + LB_THREADS, ... below `to`) of large whole
// numbers, from memory and class by class, as such rows are rare.
template <int NV>
__device__ __noinline__ LossStat large_round(const int *row, int off, const uint32_t *allowed, const float *bias, int i0, int to,
                                             LossStat st, float c) {
    const auto each = [&](auto f) {
        for (int i = i0; i < to && i < i0 + NV * LB_THREADS; i += LB_THREADS)
            for (int k = i * 4 - off; k < i * 4 - off + 4; ++k)
                if (is_allowed(allowed, k)) f(k);
    };
    LossStat now = {-INFINITY, 0.f, 0.f, INT_MIN};
    each([&](int k) { now.r = max(now.r, row[k]); });
    const auto u = [&](int k) { return loss_u(class_sum(row[k], now.r), bias ? bias[k] : 0.f); };
    each([&](int k) { now.m = fmaxf(now.m, u(k)); });
    each([&](int k) {
        const float x = now.m == -INFINITY ? u(k) : loss_x(u(k), now.m, c), e = ex2(x);
        now.s += e;
        now.h = fmaf(e, fmaxf(x, -1024.f), now.h);
    });
    return merge<int>(st, now, c);
}

// (m, s, h) of `rounds` rounds of NV * LB_THREADS vectors of one row: block
// (part, row).
template <typename T, int NV>
__global__ void __launch_bounds__(LB_THREADS, 4) k_loss_stat(const ytm_loss_args a, LossStat *__restrict__ stats, int rounds) {
    constexpr int V = RowVecs<T>::V, STEP = NV * LB_THREADS;
    __shared__ LossStat warp_stat[LB_THREADS / 32];
    const int K = a.k;
    const int64_t n = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    if (n >= a.n) return;
    const float c = loss_c(loss_rt(a));
    const F2 c2 = pair(c, c);
    const RowVecs<T> row(a.cs, n, a.cs_stride);
    const uint32_t *allowed = a.allowed ? a.allowed + n * a.allowed_stride : nullptr;
    LossStat st = {-INFINITY, 0.f, 0.f, 0};
    const int first = row.first(), below = row.off & 3, end = row.end(K, below);  // the bias is read up to the next boundary
    const auto stream = [&](auto r) {
        constexpr int R = decltype(r)::value;
        const int64_t from = (int64_t)blockIdx.x * rounds * STEP;
        const int to = (int)min((int64_t)end, first + from + (int64_t)rounds * STEP);
        for (int i0 = (int)min((int64_t)end, first + from) + (int)threadIdx.x; i0 - (int)threadIdx.x < to; i0 += STEP) {
            uint4 raw[NV];
            uint32_t open[NV];
            F2 b[NV][V / 2];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = min(i0 + j * LB_THREADS, to - 1), k = i * V - row.off;
                raw[j] = *row.at(i);
                open[j] = open_classes<V>(allowed, k);
                load_bias<V, R>(a.bias, k, b[j]);
                if (i0 + j * LB_THREADS >= to) open[j] = 0;
            }
            float z[NV][V], m = st.m;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int q = 0; q < V / 2; ++q) {
                    float x, y;
                    split(add2(class_pair<T>(raw[j], q), b[j][q]), x, y);
                    z[j][2 * q] = open[j] & (1u << (2 * q)) ? x : -INFINITY;
                    z[j][2 * q + 1] = open[j] & (2u << (2 * q)) ? y : -INFINITY;
                    m = fmaxf(m, fmaxf(z[j][2 * q], z[j][2 * q + 1]));
                }
            [[maybe_unused]] const LossStat before = st;
            const float base = m == -INFINITY ? 0.f : -m;  // nothing yet: every e is 0
            const float d = st.m == m ? 0.f : loss_x(st.m, m, c), f = ex2(d);
            F2 s = pair(f * st.s, 0.f), h = pair(f * fmaf(st.s, fmaxf(d, -1024.f), st.h), 0.f);
            const F2 base2 = pair(base, base);
            st.m = m;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int q = 0; q < V / 2; ++q) {
                    float x, y;
                    split(mul2(add2(pair(z[j][2 * q], z[j][2 * q + 1]), base2), c2), x, y);
                    const F2 e = pair(ex2(x), ex2(y));
                    s = add2(s, e);
                    h = fma2(e, pair(fmaxf(x, -1024.f), fmaxf(y, -1024.f)), h);  // 0 * -inf counts for nothing
                }
            float x, y;
            split(s, x, y);
            st.s = x + y;
            split(h, x, y);
            st.h = x + y;
            if constexpr (std::is_integral<T>::value)
                if (large_whole(m) || before.r) st = large_round<NV>((const int *)row.row, row.off, allowed, a.bias, i0, to, before, c);
        }
    };
    switch (below) {  // where the bias lies against the vectors: the same for the block
        case 0: stream(std::integral_constant<int, 0>()); break;
        case 1: stream(std::integral_constant<int, 1>()); break;
        case 2: stream(std::integral_constant<int, 2>()); break;
        default: stream(std::integral_constant<int, 3>()); break;
    }
    if (blockIdx.x == 0) {  // the classes before the first and behind the last vector
        const int head = first * V - (first ? row.off : 0), tail = end * V - row.off;
        const int k = (int)threadIdx.x < head ? (int)threadIdx.x : tail + ((int)threadIdx.x - head);
        if (k < K && is_allowed(allowed, k)) {
            int r = 0;
            if constexpr (std::is_integral<T>::value) r = large_whole(to_f32(row.row[k])) ? (int)row.row[k] : 0;
            const float u = loss_u(class_sum(row.row[k], r), a.bias ? a.bias[k] : 0.f);
            // as in the streams: e of -inf is 0, and NaN that of NaN or +inf, which u - u is
            st = merge<T>(st, {u, u == -INFINITY ? 0.f : 1.f + (u - u), 0.f, r}, c);
        }
    }
    st = merge_lanes<T>(st, 32, c);
    if ((threadIdx.x & 31) == 0) warp_stat[threadIdx.x >> 5] = st;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    st = warp_stat[threadIdx.x % (LB_THREADS / 32)];
    st = merge_lanes<T>(st, LB_THREADS / 32, c);
    if (threadIdx.x == 0) stats[n * gridDim.x + blockIdx.x] = st;
}

// Gradients of a tile: block (tile, chunk of rows), a vector of memory a
// thread.  Where rows start off a 16-byte boundary, that vector holds other
// classes from row to row, with a period of 2, 4 or 8 rows: a chunk takes every
// `period`-th row only, so that its threads keep their classes, and loads,
// stores and sums of dbias need no shift.  Tile 0 writes the losses and the
// chunk's part of the temperature's gradient, and takes the classes outside
// the row's whole vectors; where the class sums' rows lie otherwise than the
// gradients', all classes are taken one by one.
constexpr int LB_ROWS = 128;  // rows of a chunk at most

struct GradRow {
    float m, f;  // the largest u less r, w / (t s)
    int r, y;    // y -1: no gradient
};

template <typename T>
__global__ void __launch_bounds__(LB_THREADS, 4) k_loss_grad(const ytm_loss_args a, const LossStat *__restrict__ stats,
                                                             int parts, int chunks, int chunk, int period, const LossPart part) {
    constexpr int V = RowVecs<T>::V, U = 4;
    __shared__ GradRow rows[LB_ROWS];
    __shared__ float wts[LB_ROWS];  // w / t
    __shared__ double red_dt[LB_THREADS / 32];
    cudaGridDependencySynchronize();
    const int K = a.k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the last rows first: the cache still holds their class sums
    const int id = chunks - 1 - (int)(blockIdx.y + blockIdx.z * gridDim.y);  // of the chunk
    if (id < 0) return;
    const int64_t n0 = id % period + (int64_t)(id / period) * chunk * period;  // the chunk's rows: n0 + i * period
    const int count = n0 < a.n ? (int)min((int64_t)chunk, (a.n - n0 + period - 1) / period) : 0;
    const float rt = loss_rt(a), c = loss_c(rt);
    double dt = 0.0;
    [[maybe_unused]] int large = 0;  // rows with an r
    for (int i = threadIdx.x; i < count; i += LB_THREADS) {
        const int64_t n = n0 + (int64_t)i * period;
        const LossLabel label = loss_label(a, n);
        GradRow r = {0.f, 0.f, 0, -1};
        float loss = label.y >= 0 ? label.w * INFINITY : 0.f;
        if (label.open) {
            LossStat st = stats[n * parts];
            for (int j0 = 1; j0 < parts; j0 += 4) {  // four loads at once
                LossStat next[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) next[j] = stats[n * parts + min(j0 + j, parts - 1)];
                if (std::is_integral<T>::value && (st.r | next[0].r | next[1].r | next[2].r | next[3].r)) {
                    for (int j = 0; j < 4 && j0 + j < parts; ++j) st = merge<T>(st, stats[n * parts + j0 + j], c);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (j0 + j < parts) st = merge_alike(st, next[j], c);
                }
            }
            r = {st.m, label.w * rt / st.s, st.r, label.y};
            wts[i] = label.w * rt;
            large |= st.r;
            if (blockIdx.x == 0) {
                const float gap = loss_u(class_sum(((const T *)a.cs)[n * a.cs_stride + label.y], st.r), a.bias ? a.bias[label.y] : 0.f) - st.m;
                loss = label.w * (logf(st.s) - gap * rt);
                dt += (double)label.w * ((double)(st.h / st.s) - (double)gap * (double)c);
            }
        }
        rows[i] = r;
        if (blockIdx.x == 0) a.loss[n] = loss;
    }
    if (blockIdx.x == 0) {
#pragma unroll
        for (int d = 16; d; d >>= 1) dt += __shfl_xor_sync(0xFFFFFFFFu, dt, d);
        if (lane == 0) red_dt[warp] = dt;
    }
    if constexpr (std::is_integral<T>::value) large = __syncthreads_or(large);
    else __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        for (int i = 1; i < LB_THREADS / 32; ++i) dt += red_dt[i];
        if (chunks > 1) part.dt[id] = dt;
        else if (a.dtemperature) *a.dtemperature = (float)(-dt * (double)LN2 * (double)rt);
    }
    if (!a.dcs && !a.dbias) return;
    float *const db = !a.dbias ? nullptr : chunks == 1 ? a.dbias : part.db + (int64_t)id * K;
    const int64_t row0 = min(n0, a.n - 1), in_step = (int64_t)period * a.cs_stride, out_step = (int64_t)period * K;
    const int64_t mask_step = (int64_t)period * a.allowed_stride;
    const uint32_t *const mask0 = a.allowed ? a.allowed + row0 * a.allowed_stride : nullptr;
    const RowVecs<T> in0(a.cs, row0, a.cs_stride), out0(a.dcs ? a.dcs : a.cs, row0, a.dcs ? K : a.cs_stride);
    // One class over the chunk's rows.
    const auto column = [&](int k) {
        const float b = a.bias ? a.bias[k] : 0.f;
        const T *in = in0.row + k;
        const uint32_t *mask = mask0 ? mask0 + (k >> 5) : nullptr;
        T *out = a.dcs ? (T *)a.dcs + row0 * (int64_t)K + k : nullptr;
        float sum = 0.f;
#pragma unroll 4
        for (int i = 0; i < count; ++i, in += in_step) {
            const GradRow r = rows[i];
            float d = 0.f;
            if (r.y >= 0) {
                if (!mask || (*mask >> (k & 31)) & 1u) d = ex2(loss_x(loss_u(class_sum(*in, r.r), b), r.m, c)) * r.f;
                if (r.y == k) d -= wts[i];
                sum += d;
            }
            if (mask) mask += mask_step;
            if constexpr (!std::is_integral<T>::value) {
                if (out) {
                    *out = from_f32<T>(d);
                    out += out_step;
                }
            }
        }
        if (db) db[k] = sum;
    };
    const int tile = blockIdx.x * LB_THREADS;
    if (in0.off != out0.off) {
        const int k1 = (int)min((int64_t)K, (int64_t)(tile + LB_THREADS) * V);
        for (int k = tile * V + (int)threadIdx.x; k < k1; k += LB_THREADS) column(k);
        return;
    }
    const int first = in0.first(), end = in0.end(K);
    if (blockIdx.x == 0) {
        const int head = first * V - (first ? in0.off : 0), tail = end * V - in0.off;
        const int k = (int)threadIdx.x < head ? (int)threadIdx.x : tail + ((int)threadIdx.x - head);
        if (threadIdx.x < 32 && k < K) column(k);
    }
    const int vec = first + tile + (int)threadIdx.x;
    if (vec >= end) return;
    const int k0 = vec * V - in0.off, warp_k = k0 - lane * V;
    const F2 c2 = pair(c, c);
    F2 b[V / 2], acc[V / 2];
#pragma unroll
    for (int q = 0; q < V / 2; ++q) {
        b[q] = a.bias ? pair(a.bias[k0 + 2 * q], a.bias[k0 + 2 * q + 1]) : pair(0.f, 0.f);
        acc[q] = pair(0.f, 0.f);
    }
    const uint32_t shared_open = open_classes<V>(a.allowed_stride ? nullptr : a.allowed, k0);
    const bool straddle = (k0 & 31) + V > 32, masked = a.allowed_stride != 0;
    const char *in = (const char *)in0.at(vec);
    char *out = (char *)out0.at(vec);
    const uint32_t *mask = mask0 + (k0 >> 5);
    const auto stream = [&](auto with_r) {
        for (int i0 = 0; i0 < count; i0 += U) {
            uint4 raw[U];
            uint32_t open[U], lo[U], hi[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {  // loads only: a use between them would wait for each in turn
                raw[u] = make_uint4(0, 0, 0, 0);
                lo[u] = hi[u] = 0u;
                if (i0 + u < count) {
                    raw[u] = *(const uint4 *)in;
                    if (masked) lo[u] = mask[0];
                    if (masked && straddle) hi[u] = mask[1];
                }
                in += in_step * (int64_t)sizeof(T);
                mask += mask_step;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) open[u] = masked ? __funnelshift_r(lo[u], hi[u], k0 & 31) : shared_open;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i0 + u >= count) break;
                const GradRow r = rows[i0 + u];
                float d[V];
                if (r.y >= 0) {
                    const F2 m2 = pair(-r.m, -r.m), f2 = pair(r.f, r.f);
#pragma unroll
                    for (int q = 0; q < V / 2; ++q) {
                        float x, y;
                        F2 v = class_pair<T>(raw[u], q);
                        if constexpr (decltype(with_r)::value)
                            v = pair(class_sum(((const T *)&raw[u])[2 * q], r.r), class_sum(((const T *)&raw[u])[2 * q + 1], r.r));
                        split(mul2(add2(add2(v, b[q]), m2), c2), x, y);
                        x = open[u] & (1u << (2 * q)) ? ex2(x) : 0.f;
                        y = open[u] & (2u << (2 * q)) ? ex2(y) : 0.f;
                        split(mul2(pair(x, y), f2), d[2 * q], d[2 * q + 1]);
                    }
                    if (r.y >= warp_k && r.y - warp_k < 32 * V) {  // the label's class is this warp's
#pragma unroll
                        for (int j = 0; j < V; ++j)
                            if (r.y - k0 == j) d[j] -= wts[i0 + u];
                    }
#pragma unroll
                    for (int q = 0; q < V / 2; ++q) acc[q] = add2(acc[q], pair(d[2 * q], d[2 * q + 1]));
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) d[j] = 0.f;
                }
                if constexpr (!std::is_integral<T>::value) {
                    if (a.dcs) {
                        alignas(16) T t[V];
#pragma unroll
                        for (int j = 0; j < V; ++j) t[j] = from_f32<T>(d[j]);
                        *(uint4 *)out = *(const uint4 *)t;
                        out += out_step * (int64_t)sizeof(T);
                    }
                }
            }
        }
    };
    if constexpr (std::is_integral<T>::value) {
        if (large) stream(std::true_type());
        else stream(std::false_type());
    } else {
        stream(std::false_type());
    }
    if (db) {
#pragma unroll
        for (int q = 0; q < V / 2; ++q) {
            float x, y;
            split(acc[q], x, y);
            db[k0 + 2 * q] = x;
            db[k0 + 2 * q + 1] = y;
        }
    }
}

// Sums of the teams' parts: 32 classes a block, 32 threads a class; the last
// block adds the temperature's.
__global__ void __launch_bounds__(1024) k_loss_join(const ytm_loss_args a, const LossPart part, int teams) {
    __shared__ double red[32][33];
    cudaGridDependencySynchronize();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const bool last = blockIdx.x == gridDim.x - 1;
    const int k = blockIdx.x * 32 + x;
    double t = 0.0;
    if (last)
        for (int i = threadIdx.x; i < teams; i += 1024) t += part.dt[i];
    else if (k < a.k)
        for (int i = y; i < teams; i += 32) t += (double)part.db[(int64_t)i * a.k + k];
    red[y][x] = t;
    __syncthreads();
    t = red[x][y];
#pragma unroll
    for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, d);
    if (!last) {
        if (x == 0 && blockIdx.x * 32 + y < a.k) a.dbias[blockIdx.x * 32 + y] = (float)t;
        return;
    }
    __syncthreads();
    if (x == 0) red[0][y] = t;
    __syncthreads();
    if (threadIdx.x < 32) {
        t = red[0][x];
#pragma unroll
        for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, d);
        if (x == 0 && a.dtemperature) *a.dtemperature = (float)(-t * (double)LN2 * (double)loss_rt(a));
    }
}

// ------------------------------------------------------------- launching

// How a call is cut: which kernels, and how many teams' parts there are to join.
struct LossPlan {
    bool big;
    int tpr, e;   // small: threads of a row, classes of a thread
    int nv;       // big: vectors of a thread in a round
    int parts, rounds, chunk, period;  // big: parts of a row, rounds of a part, rows of a chunk and their distance
    int64_t teams;             // blocks (small) or chunks (big)
};

constexpr int LOSS_CHAIN = 256;  // rows that one thread adds up in fp32 at most

static LossPlan loss_plan(int64_t n, int64_t k, int64_t elem, int64_t cs_stride) {
    LossPlan p = {};
    const int64_t sms = sm_count();
    if (k <= 512) {
        p.tpr = k <= 16 ? 4 : k <= 128 ? 8 : k <= 256 ? 16 : 32;
        p.e = k <= 32 ? 4 : k <= 64 ? 8 : 16;
        const int64_t rows = LS_THREADS / p.tpr;
        // up to four rounds of one block cost less than joining blocks
        p.teams = n <= 4 * rows ? 1 : std::min<int64_t>(cdiv(n, rows), sms * (p.e == 16 ? 2 : p.e == 8 ? 3 : 4));
        p.teams = std::max<int64_t>(p.teams, cdiv(n, rows * LOSS_CHAIN));
        return p;
    }
    p.big = true;
    // parts of a row until every SM has about eight blocks
    const int64_t vecs = cdiv(k * elem, 16);
    p.nv = vecs <= LB_THREADS ? 1 : (int)elem;    // 16 classes of a thread in a round
    const int64_t rounds = cdiv(vecs, (int64_t)LB_THREADS * p.nv);
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(32, cdiv(sms * 4, n)));
    p.rounds = (int)cdiv(rounds, std::min(want, rounds));
    p.parts = (int)cdiv(rounds, p.rounds);
    // the class sums' and the gradients' rows lie alike every `period` rows
    p.period = 1;
    while (k * elem * p.period % 16 || cs_stride * elem * p.period % 16) p.period *= 2;
    // chunks of rows until there are about eight blocks an SM
    p.chunk = (int)std::min<int64_t>(LB_ROWS, std::max<int64_t>(4, cdiv(n * cdiv(vecs, LB_THREADS), sms * 8)));
    p.teams = (int64_t)p.period * cdiv(cdiv(n, p.period), p.chunk);
    return p;
}

// A launch that may start while the kernel before it ends (it waits for that
// kernel's results itself).
template <typename... P, typename... A>
static ytm_status launch_after(void (*f)(P...), dim3 grid, unsigned block, cudaStream_t st, const char *what, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cuda_check(cudaLaunchKernelEx(&cfg, f, P(args)...), what);
}

// Workspace: dt parts, dbias parts, row statistics.
struct LossWs {
    uint64_t db, stats, total;
};

static LossWs loss_ws(const LossPlan &p, int64_t n, int64_t k) {
    LossWs w;
    const bool join = p.teams > 1;
    w.db = join ? align_up((uint64_t)p.teams * 8, 256) : 0;
    w.stats = w.db + (join ? align_up((uint64_t)p.teams * k * 4, 256) : 0);
    w.total = w.stats + (p.big ? (uint64_t)n * p.parts * sizeof(LossStat) : 0);
    return w;
}

template <typename T>
static ytm_status launch_big(const ytm_loss_args &a, const LossPlan &p, const LossPart &part, LossStat *stats, cudaStream_t st) {
    const unsigned gz = (unsigned)cdiv(a.n, 65535), gy = (unsigned)cdiv(a.n, gz);
    const dim3 grid(p.parts, gy, gz);
    if (p.nv == 1) k_loss_stat<T, 1><<<grid, LB_THREADS, 0, st>>>(a, stats, p.rounds);
    else k_loss_stat<T, (int)sizeof(T)><<<grid, LB_THREADS, 0, st>>>(a, stats, p.rounds);
    ytm_status rc = launch_check("class loss statistics");
    if (rc) return rc;
    const uint64_t vecs = cdiv((uint64_t)a.k * sizeof(T), 16);
    const unsigned tiles = a.dcs || a.dbias ? (unsigned)cdiv(vecs, LB_THREADS) : 1;
    const unsigned cz = (unsigned)cdiv(p.teams, 65535), cy = (unsigned)cdiv(p.teams, cz);
    return launch_after(k_loss_grad<T>, dim3(tiles, cy, cz), LB_THREADS, st, "class loss", a, stats, p.parts, (int)p.teams,
                        p.chunk, p.period, part);
}

template <typename T, int TPR, int E>
static ytm_status launch_small(const ytm_loss_args &a, const LossPlan &p, const LossPart &part, cudaStream_t st) {
    k_loss_small<T, TPR, E><<<(unsigned)p.teams, LS_THREADS, LS_THREADS * E * 4, st>>>(a, part);
    return launch_check("class loss");
}

template <typename T>
static ytm_status launch_loss(const ytm_loss_args &a, const LossPlan &p, const LossPart &part, LossStat *stats, cudaStream_t st) {
    if (p.big) return launch_big<T>(a, p, part, stats, st);
    if (p.tpr == 4) return launch_small<T, 4, 4>(a, p, part, st);
    if (p.tpr == 8 && p.e == 4) return launch_small<T, 8, 4>(a, p, part, st);
    if (p.tpr == 8 && p.e == 8) return launch_small<T, 8, 8>(a, p, part, st);
    if (p.tpr == 8) return launch_small<T, 8, 16>(a, p, part, st);
    if (p.tpr == 16) return launch_small<T, 16, 16>(a, p, part, st);
    return launch_small<T, 32, 16>(a, p, part, st);
}

}  // namespace ytm

using namespace ytm;

extern "C" {

uint64_t ytm_class_loss_workspace_bytes(int64_t n, int32_t k, int32_t cs_type, int64_t cs_stride) {
    if (n <= 0 || k <= 0 || !is_sum_type(cs_type) || cs_stride < 0) return 0;
    return loss_ws(loss_plan(n, k, type_bytes(cs_type), cs_stride), n, k).total;
}

ytm_status ytm_class_loss(const ytm_loss_args *args, void *workspace, void *stream) {
    if (!args) return fail(YTM_ERR_ARG, "args is NULL");
    ytm_loss_args a = *args;
    if (a.n < 0 || a.k <= 0) return fail(YTM_ERR_ARG, "class loss: needs n >= 0 rows of k >= 1 classes");
    if (a.n > INT_MAX || a.k > (1 << 30)) return fail(YTM_ERR_UNSUPPORTED, "class loss: more than 2^31 - 1 rows or 2^30 classes");
    if (!is_sum_type(a.cs_type)) return fail(YTM_ERR_ARG, "class loss: class sums must be int32, fp32, fp16 or bf16");
    if (a.cs_type == YTM_I32 && a.dcs) return fail(YTM_ERR_ARG, "class loss: int32 class sums have no gradient");
    if (a.cs_stride < 0 || a.allowed_stride < 0) return fail(YTM_ERR_ARG, "class loss: negative stride");
    if (!a.allowed) a.allowed_stride = 0;  // the kernels take a stride to say that there is something to read row by row
    cudaStream_t st = as_stream(stream);
    ytm_status rc;
    if (a.n == 0) {
        if (a.dbias && (rc = cuda_check(cudaMemsetAsync(a.dbias, 0, (size_t)a.k * 4, st), "memset"))) return rc;
        if (a.dtemperature && (rc = cuda_check(cudaMemsetAsync(a.dtemperature, 0, 4, st), "memset"))) return rc;
        return YTM_OK;
    }
    const LossPlan p = loss_plan(a.n, a.k, type_bytes(a.cs_type), a.cs_stride);
    const LossWs ws = loss_ws(p, a.n, a.k);
    if (!a.cs || !a.target || !a.loss || (ws.total && !workspace)) return fail(YTM_ERR_ARG, "null pointer");
    if ((uintptr_t)workspace % 16) return fail(YTM_ERR_ARG, "class loss: workspace must start on a 16-byte boundary");
    const LossPart part = {(float *)((char *)workspace + ws.db), (double *)workspace};
    LossStat *stats = (LossStat *)((char *)workspace + ws.stats);
    switch (a.cs_type) {
        case YTM_I32: rc = launch_loss<int32_t>(a, p, part, stats, st); break;
        case YTM_F32: rc = launch_loss<float>(a, p, part, stats, st); break;
        case YTM_F16: rc = launch_loss<__half>(a, p, part, stats, st); break;
        default: rc = launch_loss<__nv_bfloat16>(a, p, part, stats, st); break;
    }
    if (rc || p.teams == 1 || (!a.dbias && !a.dtemperature)) return rc;
    return launch_after(k_loss_join, dim3((unsigned)(a.dbias ? cdiv(a.k, 32) : 0) + 1), 1024, st, "class loss sums", a, part,
                        (int)p.teams);
}

}  // extern "C"
