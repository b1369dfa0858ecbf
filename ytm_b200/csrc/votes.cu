// votes.cu — the vote of clause weights held in 4 bits with group scales.
#include <cooperative_groups.h>

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
//
// The weights' bytes bound the call while there are few samples, so they are
// what streams: a block copies 16 KB of them a stage into shared memory with
// 16-byte asynchronous copies, four stages deep, and a warp multiplies 16
// classes by 256 clauses of a stage on the tensor cores (m16n8k16, fp32 sums).
// ldmatrix hands lane (g, t) word t of 32 clauses of classes g and g + 8, i.e.
// eight 4-bit weights, which the lane turns into bf16 or fp16 pairs (clauses i
// and i + 4) by or-ing them into the fraction of 128 (1024) and subtracting
// 136 (1032): exact.  The activations lie in shared memory in that order of
// clauses.  The sum of a group is exact up to the fp32 additions; its scale is
// applied in fp32.  Activations in fp32 take three columns, their leading,
// middle and last 8 bits, which are bf16 values exactly; clause bits are bf16
// zeros and ones.
//
// WM of a block's 8 warps lie along the classes, 8 / WM along the clauses, and
// up to 16 blocks of a cluster along the clauses, which add their sums through
// distributed shared memory in a fixed order.

namespace cg = cooperative_groups;

constexpr int Q4_THREADS = 256, Q4_WARPS = 8, Q4_STAGES = 4;
constexpr int Q4_SEG = 256;                                       // clauses of a warp in a stage
constexpr int Q4_WARP_BYTES = Q4_SEG / 32 * 17 * 16;              // 16 classes of a stage, rows of 17 x 16 bytes
constexpr int Q4_STAGE_BYTES = Q4_WARPS * Q4_WARP_BYTES;

struct Q4Args {
    const void *x;
    int64_t x_stride, n0, n;  // samples n0 .. n0 + n of this call
    const uint8_t *packed;
    const void *scales;
    const float *bias;
    void *y;
    int C, K, G, x_type, scale_type, y_type;
    int samples;              // of a block (grid z)
    int wm, log_wk, cluster;
    int xpitch;               // bytes between the activation columns in shared memory
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

__device__ __forceinline__ float load_scale(const void *p, int type, int64_t i) {
    if (type == YTM_F32) return ((const float *)p)[i];
    if (type == YTM_F16) return __half2float(((const __half *)p)[i]);
    return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
}

// Eight 4-bit weights -> four pairs (i, i + 4) of the value minus 8.
template <bool HALF>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // HALF: the odd nibbles stay 4 bits up, as 1024 + 16 q
        const uint32_t v = HALF ? (i < 2 ? w : w >> 8) : w >> (4 * i);
        const uint32_t mask = HALF && (i & 1) ? 0x00F000F0u : 0x000F000Fu;
        uint32_t b;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(b) : "r"(v), "r"(mask), "r"(HALF ? 0x64006400u : 0x43004300u));
        if (HALF) {
            const __half2 h = *(__half2 *)&b;
            const __half2 r = i & 1 ? __hfma2(h, __half2half2(__ushort_as_half(0x2C00)), __half2half2(__ushort_as_half(0xD480)))  // / 16 - 72
                                    : __hadd2(h, __half2half2(__ushort_as_half(0xE408)));                                          // - 1032
            p[i] = *(const uint32_t *)&r;
        } else {
            const __nv_bfloat162 r = __hadd2(*(__nv_bfloat162 *)&b, __bfloat162bfloat162(__ushort_as_bfloat16(0xC308)));  // - 136
            p[i] = *(const uint32_t *)&r;
        }
    }
}

template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (HALF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {  // of values that bf16 holds
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}

// Eight activations c .. c + 7 of a sample (0 behind the last clause).
struct Octet {
    uint32_t w[8];  // fp32: values; 16-bit: pairs in w[0..3]; bits: w[0]
};

__device__ __forceinline__ Octet load_octet(const Q4Args &a, int64_t row, int c) {
    Octet o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.w[i] = 0;
    if (c >= a.C) return o;
    if (a.x_type == YTM_BITS) {
        o.w[0] = ((const uint32_t *)a.x)[row + (c >> 5)] >> (c & 31) & 255u;
        if (c + 8 > a.C) o.w[0] &= (1u << (a.C - c)) - 1u;
        return o;
    }
    const bool all = c + 8 <= a.C;
    if (a.x_type == YTM_F32) {
        const float *p = (const float *)a.x + row + c;
        if (all && (uintptr_t)p % 16 == 0) {
            *(uint4 *)&o.w[0] = *(const uint4 *)p;
            *(uint4 *)&o.w[4] = *(const uint4 *)(p + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < a.C) o.w[i] = __float_as_uint(p[i]);
        }
        return o;
    }
    const uint16_t *p = (const uint16_t *)a.x + row + c;
    if (all && (uintptr_t)p % 16 == 0) {
        *(uint4 *)&o.w[0] = *(const uint4 *)p;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < a.C) o.w[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
    }
    return o;
}

// The octet in the order (0, 4, 1, 5, 2, 6, 3, 7), at byte `at` of its column
// (fp32: of its three columns).
__device__ __forceinline__ void store_octet(const Q4Args &a, char *at, const Octet &o) {
    if (a.x_type == YTM_BITS) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = ((o.w[0] >> i) & 1u) * 0x3F80u | ((o.w[0] >> (i + 4)) & 1u) * 0x3F800000u;
        *(uint4 *)at = make_uint4(v[0], v[1], v[2], v[3]);
    } else if (a.x_type == YTM_F32) {
        float rest[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] = __uint_as_float(o.w[i]);
#pragma unroll
        for (int part = 0; part < 3; ++part) {
            float top[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // the leading 8 bits; NaN stays NaN, infinity leaves nothing
                top[i] = __uint_as_float(__float_as_uint(rest[i]) & 0xFFFF0000u);
                if (part == 0 && rest[i] != rest[i]) top[i] = __uint_as_float(0x7FC00000u);
                rest[i] = part == 0 && !(fabsf(rest[i]) < INFINITY) ? 0.f : rest[i] - top[i];
            }
            *(uint4 *)(at + part * a.xpitch) = make_uint4(bf16_pair(top[0], top[4]), bf16_pair(top[1], top[5]),
                                                          bf16_pair(top[2], top[6]), bf16_pair(top[3], top[7]));
        }
    } else {
        *(uint4 *)at = make_uint4(__byte_perm(o.w[0], o.w[2], 0x5410), __byte_perm(o.w[0], o.w[2], 0x7632),
                                  __byte_perm(o.w[1], o.w[3], 0x5410), __byte_perm(o.w[1], o.w[3], 0x7632));
    }
}

template <bool HALF, int NT, int GROUP>
__global__ void __launch_bounds__(Q4_THREADS, NT <= 2 ? 2 : 1) k_q4_votes(const Q4Args a) {
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int WM = a.wm, WK = 1 << a.log_wk, wm = warp % WM, wk = warp / WM;
    const int rank = a.cluster > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int64_t row_bytes = q4_row_bytes(a.C);
    const int row0 = (int)(blockIdx.x / a.cluster) * 16 * WM;
    const int64_t sample0 = a.n0 + (int64_t)blockIdx.z * a.samples;
    const int samples = (int)min((int64_t)a.samples, a.n0 + a.n - sample0);
    const int parts = a.x_type == YTM_F32 ? 3 : 1, cols = samples * parts;
    // this block's stages of the C clauses: WK segments each
    const int stages_all = (a.C + Q4_SEG * WK - 1) / (Q4_SEG * WK);
    const int per = (stages_all + a.cluster - 1) / a.cluster;
    const int first = min(rank * per, stages_all), count = min(first + per, stages_all) - first;

    char *xs = smem + Q4_STAGES * Q4_STAGE_BYTES;
    const int xbuf = a.samples * parts * a.xpitch;
    const uint32_t smem_at = (uint32_t)__cvta_generic_to_shared(smem);

    // Weights of stage first + s: the thread's 16-byte unit of a row is the same
    // in its four rows.
    const int log_units = 3 + a.log_wk;  // 16-byte units of a row in a stage
    const int su = tid & ((1 << log_units) - 1), r0 = tid >> log_units, r_step = Q4_THREADS >> log_units;
    const uint8_t *src[4];
    uint32_t dst[4];
    bool row_there[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + i * r_step;
        row_there[i] = row0 + r < a.K;
        src[i] = a.packed + (row_there[i] ? (row0 + r) * row_bytes : 0) + (int64_t)first * (16 << log_units) + su * 16;
        dst[i] = smem_at + (((su >> 3) * WM + (r >> 4)) * 8 + (su & 7)) * 272 + (r & 15) * 16;
    }
    int64_t left = row_bytes - ((int64_t)first * (16 << log_units) + su * 16);  // bytes of the row from this stage's unit on
    int copied = 0;
    const auto copy_stage = [&]() {
        if (copied < count) {
            const uint32_t base = (copied % Q4_STAGES) * Q4_STAGE_BYTES;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool there = row_there[i] && left > 0;
                cp_async16(dst[i] + base, there ? src[i] : a.packed, there);
                src[i] += 16 << log_units;
            }
            left -= 16 << log_units;
        }
        ++copied;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const int log_octets = 5 + a.log_wk;  // of a sample in a stage
    const auto load_x = [&](int s, int u) {
        const int i = u >> log_octets;
        return load_octet(a, (sample0 + i) * a.x_stride, (first + s) * Q4_SEG * WK + (u - (i << log_octets)) * 8);
    };
    const auto store_x = [&](int s, int u, const Octet &o) {
        const int i = u >> log_octets;
        store_octet(a, xs + (s & 1) * xbuf + i * parts * a.xpitch + (u - (i << log_octets)) * 16, o);
    };
    const int x_units = samples << log_octets;

#pragma unroll
    for (int s = 0; s < Q4_STAGES - 1; ++s) copy_stage();
    if (count > 0)
        for (int u = tid; u < x_units; u += Q4_THREADS) store_x(0, u, load_x(0, u));

    // scales: lane t of a class holds groups t, t + 4, ... of a stage
    constexpr int GPS = Q4_SEG / GROUP, GPL = (GPS + 3) / 4;
    const int g = lane >> 2, t = lane & 3;
    const int class0 = row0 + wm * 16 + g, class1 = class0 + 8;
    const int64_t at0 = class0 < a.K ? (int64_t)class0 * a.G : 0, at1 = class1 < a.K ? (int64_t)class1 * a.G : 0;
    const auto load_scales = [&](int s, float (&sc)[GPL][2]) {
#pragma unroll
        for (int j = 0; j < GPL; ++j) {
            const int in_stage = j * 4 + t, grp = ((first + s) * WK + wk) * GPS + in_stage;
            const bool there = s < count && in_stage < GPS && grp < a.G;
            sc[j][0] = there ? load_scale(a.scales, a.scale_type, at0 + grp) : 0.f;
            sc[j][1] = there ? load_scale(a.scales, a.scale_type, at1 + grp) : 0.f;
        }
    };
    float next_sc[GPL][2];
    load_scales(0, next_sc);

    float tot[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) tot[n][i] = 0.f;
    int x_col[NT];  // columns behind the last are the last once more; nobody reads their sums
#pragma unroll
    for (int n = 0; n < NT; ++n) x_col[n] = min(n * 8 + g, cols - 1) * a.xpitch;
    const uint32_t mat = (warp * 8 + (lane >> 4)) * 272 + ((lane >> 3 & 1) * 8 + (lane & 7)) * 16;

    for (int s = 0; s < count; ++s) {
        asm volatile("cp.async.wait_group %0;" ::"n"(Q4_STAGES - 2) : "memory");
        __syncthreads();  // stage s and its activations are there; stage s - 1 is done with
        copy_stage();
        float sc[GPL][2];
#pragma unroll
        for (int j = 0; j < GPL; ++j) {
            sc[j][0] = next_sc[j][0];
            sc[j][1] = next_sc[j][1];
        }
        load_scales(s + 1, next_sc);
        Octet o;  // the next stage's first octet is on its way during the products
        const bool more = s + 1 < count;
        if (more && tid < x_units) o = load_x(s + 1, tid);

        const uint32_t w_at = smem_at + (s % Q4_STAGES) * Q4_STAGE_BYTES + mat;
        const char *x_at = xs + (s & 1) * xbuf + wk * Q4_SEG * 2 + t * 16;
        float acc[NT][4];
#pragma unroll
        for (int j2 = 0; j2 < Q4_SEG / 64; ++j2) {
            uint32_t q[4];
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]) : "r"(w_at + j2 * 2 * 272));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = j2 * 2 + h;  // 32 clauses
                if (j % (GROUP / 32) == 0) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
                }
                uint32_t lo[4], hi[4];
                unpack<HALF>(q[2 * h], lo);
                unpack<HALF>(q[2 * h + 1], hi);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 b = *(const uint4 *)(x_at + x_col[n] + j * 64);
                    mma<HALF>(acc[n], lo[0], hi[0], lo[1], hi[1], b.x, b.y);
                    mma<HALF>(acc[n], lo[2], hi[2], lo[3], hi[3], b.z, b.w);
                }
                if ((j + 1) % (GROUP / 32) == 0) {
                    const int grp = j / (GROUP / 32), from = (lane & ~3) | (grp & 3);
                    const float s0 = __shfl_sync(0xFFFFFFFFu, sc[grp / 4][0], from), s1 = __shfl_sync(0xFFFFFFFFu, sc[grp / 4][1], from);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        tot[n][0] = fmaf(s0, acc[n][0], tot[n][0]);
                        tot[n][1] = fmaf(s0, acc[n][1], tot[n][1]);
                        tot[n][2] = fmaf(s1, acc[n][2], tot[n][2]);
                        tot[n][3] = fmaf(s1, acc[n][3], tot[n][3]);
                    }
                }
            }
        }
        if (more) {
            if (tid < x_units) store_x(s + 1, tid, o);
            for (int u = tid + Q4_THREADS; u < x_units; u += Q4_THREADS) store_x(s + 1, u, load_x(s + 1, u));
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    // sums of the warps along the clauses and of the parts of an activation
    constexpr int COLS = NT * 8;
    float *red = (float *)smem;                      // [warp][16][COLS]
    float *mine = red + Q4_WARPS * 16 * COLS;        // [samples][16 * WM]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[(warp * 16 + g + (i >> 1) * 8) * COLS + n * 8 + t * 2 + (i & 1)] = tot[n][i];
    __syncthreads();
    const int rows = 16 * WM, outs = rows * samples;
    for (int u = tid; u < outs; u += Q4_THREADS) {
        const int i = u / rows, r = u - i * rows;
        float v = 0.f;
        for (int k = 0; k < WK; ++k)
            for (int p = 0; p < parts; ++p) v += red[((k * WM + r / 16) * 16 + r % 16) * COLS + i * parts + p];
        mine[u] = v;
    }
    __syncthreads();
    if (a.cluster > 1) cg::this_cluster().sync();
    for (int u = rank * Q4_THREADS + tid; u < outs; u += a.cluster * Q4_THREADS) {
        const int i = u / rows, r = u - i * rows;
        float v = 0.f;
        if (a.cluster > 1) {
            for (int k = 0; k < a.cluster; ++k) v += *cg::this_cluster().map_shared_rank(mine + u, k);
        } else {
            v = mine[u];
        }
        if (row0 + r >= a.K) continue;
        if (a.bias) v += a.bias[row0 + r];
        const int64_t at = (sample0 + i) * a.K + row0 + r;
        if (a.y_type == YTM_F32) ((float *)a.y)[at] = v;
        else if (a.y_type == YTM_F16) ((__half *)a.y)[at] = __float2half_rn(v);
        else ((__nv_bfloat16 *)a.y)[at] = __float2bfloat16_rn(v);
    }
    if (a.cluster > 1) cg::this_cluster().sync();  // nobody leaves while its sums are read
}

// How the warps lie (see above).  The cost of a cut, in stages of 16 KB: the
// blocks of the busiest SM times the stages of a block plus about three for its
// start and its end, half of which a second block on the SM hides.
struct Q4Plan {
    int wm, cluster, xpitch;
    size_t smem;
};

static Q4Plan q4_plan(int64_t C, int64_t K, int nt, int cols, int64_t z) {
    Q4Plan best = {};
    double least = 0;
    const int64_t sms = sm_count();
    for (int wm = 8; wm >= 1; wm /= 2) {
        const int wk = Q4_WARPS / wm, xpitch = Q4_SEG * 2 * wk + 64;
        const size_t red = (size_t)Q4_WARPS * 16 * nt * 8 * 4 + (size_t)cols * 16 * wm * 4;
        const size_t smem = std::max<size_t>((size_t)Q4_STAGES * Q4_STAGE_BYTES + 2 * (size_t)cols * xpitch, red);
        if (smem > 227 * 1024) continue;
        const int64_t tiles = cdiv(K, 16 * wm) * z, stages = cdiv(C, Q4_SEG * wk);
        const bool two = nt <= 2 && smem <= 113 * 1024;
        for (int cl = 1; cl <= 16; cl *= 2) {
            if (cl > 1 && cl > stages) break;
            // SMs that hold two blocks share their bandwidth between them
            const double cost = (double)cdiv(tiles * cl, sms) * ((double)cdiv(stages, cl) + (two ? 1.5 : 3));
            if (!best.wm || cost < least * 0.97) {
                best = {wm, cl, xpitch, smem};
                least = cost;
            }
        }
    }
    return best;
}

template <bool HALF, int NT, int GROUP>
static ytm_status launch_q4(const Q4Args &a, const Q4Plan &p, dim3 grid, cudaStream_t st) {
    auto *f = k_q4_votes<HALF, NT, GROUP>;
    ytm_status rc;
    if ((rc = cuda_check(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)p.smem), "q4 votes smem")))
        return rc;
    if (p.cluster > 8 && (rc = cuda_check(cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "q4 votes cluster")))
        return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(Q4_THREADS);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    return cuda_check(cudaLaunchKernelEx(&cfg, f, a), "q4 votes");
}

template <bool HALF, int NT>
static ytm_status launch_q4(const Q4Args &a, const Q4Plan &p, int group, dim3 grid, cudaStream_t st) {
    if (group == 32) return launch_q4<HALF, NT, 32>(a, p, grid, st);
    if (group == 64) return launch_q4<HALF, NT, 64>(a, p, grid, st);
    return launch_q4<HALF, NT, 128>(a, p, grid, st);
}

template <bool HALF>
static ytm_status launch_q4(const Q4Args &a, const Q4Plan &p, int nt, int group, dim3 grid, cudaStream_t st) {
    if (nt == 1) return launch_q4<HALF, 1>(a, p, group, grid, st);
    if (nt == 2) return launch_q4<HALF, 2>(a, p, group, grid, st);
    if (nt == 4) return launch_q4<HALF, 4>(a, p, group, grid, st);
    return launch_q4<HALF, 8>(a, p, group, grid, st);
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
    const int parts = x_type == YTM_F32 ? 3 : 1;
    const int64_t most = 64 / parts;  // samples of a block
    const int64_t z = std::min<int64_t>(cdiv(N, most), 65535);
    // samples evenly over the blocks, in tiles of 8 columns
    const int samples = (int)(N <= most ? N : most);
    const int cols = samples * parts, nt = cols <= 8 ? 1 : cols <= 16 ? 2 : cols <= 32 ? 4 : 8;
    const Q4Plan p = q4_plan(C, K, nt, cols, z);
    Q4Args a = {x, x_stride, 0, 0, packed, scales, bias, y, C, K, (int)cdiv(C, group), x_type, scale_type, y_type,
                samples, p.wm, p.wm == 8 ? 0 : p.wm == 4 ? 1 : p.wm == 2 ? 2 : 3, p.cluster, p.xpitch};
    for (int64_t i = 0; i < N; i += z * most) {
        a.n0 = i;
        a.n = std::min<int64_t>(N - i, z * most);
        const dim3 grid((unsigned)(cdiv(K, 16 * p.wm) * p.cluster), 1, (unsigned)cdiv(a.n, most));
        rc = x_type == YTM_F16 ? launch_q4<true>(a, p, nt, group, grid, as_stream(stream))
                               : launch_q4<false>(a, p, nt, group, grid, as_stream(stream));
        if (rc) return rc;
    }
    return YTM_OK;
}

}  // extern "C"
