// votes.cu — the vote of clause weights held in 4 bits with group scales.
#include <cooperative_groups.h>
#include <cuda.h>
#include <limits.h>
#include <string.h>

#include <atomic>
#include <type_traits>
#include <utility>

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
// take consecutive classes, so every read of a weight row is coalesced.  16384 x
// 4000 int32 327 us (0.9 TB/s): each weight is read twice and divided in 64 bits, and
// a warp's bytes are stored a packed row apart; done once for a model.
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
// what streams: one thread of a block copies 16 KB of them a stage into shared
// memory by TMA, four stages deep, and each of eight warps multiplies 16
// classes by 256 clauses of a stage on the tensor cores.  ldmatrix hands lane
// (g, t) word t of 32 clauses of classes g and g + 8, i.e. eight 4-bit weights.
// What is done with a word decides the speed, as it is done for every 4 bytes:
//
// - whole numbers (m16n8k32): two masks and a shift make the word's low and high
//   halves of the bytes two registers of unsigned bytes, an operand as they are.
//   Clause bits are the other operand; real activations become four signed
//   bytes, x = (d0 2^24 + d1 2^16 + d2 2^8 + d3) 2^e with e of the largest of 128
//   neighbours, i.e. x to 2^-30 of that one, in four columns.  The 8 that the
//   weights are offset by goes into the sums' start, -8 times the sum of a
//   group's digits.  Sums of a group are exact.
// - 16-bit products (m16n8k16): the word becomes four pairs (clauses i and i + 4)
//   by or-ing it into the fraction of 128 (fp16: 1024) and subtracting 136
//   (1032), exactly; four times the logic, but a column a sample.  Taken for 16-bit
//   activations from three samples on (16384 x 32768, bf16, groups of 128, on the
//   GPU: one sample 68 us against 50 in digits, three 68 against 61, five 69 against
//   73; 8192 x 8192: 13.8 against 12.3, 14.1 against 13.6, 14.5 against 15.3), and
//   where few classes leave the weights' stream short (65536 x 100: 7.7 against 9.1).
//   Many samples of many classes have a kernel of their own, k_q4_tiles.
//
// A group's sum is scaled in fp32.  k_q4_x lays the activations out before, in
// pieces of 256 clauses, so that a stage's are one piece of memory.
//
// WM of a block's 8 warps lie along the classes, 8 / WM along the clauses, and
// up to 16 blocks of a cluster along the clauses, which add their sums through
// distributed shared memory in a fixed order.

namespace cg = cooperative_groups;

enum Q4Mode { Q4_BITS, Q4_DIGITS, Q4_BF16, Q4_FP16 };

constexpr int Q4_WARPS = 8, Q4_THREADS = 32 * (Q4_WARPS + 1);  // the last warp copies
constexpr int Q4_STAGES = 4;
constexpr int Q4_SEG = 256;                        // clauses of a warp in a stage: 128 bytes of a class
constexpr int Q4_STAGE_BYTES = Q4_WARPS * 16 * 128;
constexpr int Q4_BARS = 128;                       // bytes of the barriers and the failure flag

// Bytes of 256 clauses of `cols` columns.  16-bit: [32 clauses][column][64].
// Whole numbers: digits [64 clauses][column][t][2 groups of 32][even 4, odd 4],
// the sums' starts i32 [group][column], and for real activations the factors
// f32 [128 clauses][column].
__host__ __device__ constexpr int q4_seg_bytes(Q4Mode mode, int cols, int group) {
    return mode >= Q4_BF16 ? cols * 512 : cols * (256 + Q4_SEG / group * 4 + (mode == Q4_DIGITS ? 8 : 0));
}

struct Q4Args {
    const char *xs;           // k_q4_x's activations: [block of samples][256 clauses][q4_seg_bytes]
    const void *scales;
    const float *bias;
    void *y;
    int64_t n0, n;            // samples n0 .. n0 + n of this launch
    int64_t xs_block;         // bytes of a block of samples in xs
    int K, G, stages, scale_type, y_type;
    int samples, parts;       // of a block (grid z); columns of a sample
    int log_wk, cluster, bars_at;
    uint32_t zero;            // 0, unknown to the compiler
};

// ---- activations

struct Q4XArgs {
    const void *x;
    int64_t x_stride, n0, n;
    char *xs;
    int64_t xs_block;
    int C, x_type, samples, parts, cols, segs, group;
    bool tiles;               // for k_q4_tiles
};

// Clauses c .. c + 7 of a row (0 behind the last clause) as fp32.
__device__ __forceinline__ void load_octet(const Q4XArgs &a, int64_t row, int c, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (a.x_type == YTM_F32) {
        const float *p = (const float *)a.x + row + c;
        if (c + 8 <= a.C && (uintptr_t)p % 16 == 0) {
            *(float4 *)&v[0] = *(const float4 *)p;
            *(float4 *)&v[4] = *(const float4 *)(p + 4);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < a.C) v[j] = p[j];
        }
    } else {
        const uint16_t *p = (const uint16_t *)a.x + row + c;
        uint32_t w[4] = {0, 0, 0, 0};
        if (c + 8 <= a.C && (uintptr_t)p % 16 == 0) {
            *(uint4 *)w = *(const uint4 *)p;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < a.C) w[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t h = w[j / 2] >> (16 * (j & 1)) & 0xFFFFu;
            v[j] = a.x_type == YTM_F16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16);
        }
    }
}

// A thread takes 8 clauses of a sample, 16 neighbours 128 clauses.
template <Q4Mode MODE>
__global__ void __launch_bounds__(256) k_q4_x(const Q4XArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int octets = a.segs * 32;
    const int64_t i = u / octets;  // sample of this launch: one for a warp
    if (i >= a.n) return;
    const int o = (int)(u - i * octets), c = o * 8, in_seg = o & 31;
    const int64_t row = (a.n0 + i) * a.x_stride;
    const int col = (int)(i % a.samples) * a.parts;
    char *const seg = a.xs + i / a.samples * a.xs_block + (int64_t)(o >> 5) * q4_seg_bytes(a.tiles ? Q4_FP16 : MODE, a.cols, a.group);
    // for tiles: rows of 64 clauses, their eight 16-byte pieces exchanged by the column's low bits
    const int tile_at = ((in_seg >> 3) * a.cols + col) * 128 + ((o & 7) ^ (col & 7)) * 16;
    if (MODE >= Q4_BF16) {
        // order (0, 4, 1, 5, 2, 6, 3, 7); the four 16-byte pieces of a (group,
        // column) are exchanged by the column's bits 1 and 2, so that the eight
        // lanes that read two columns together meet 32 different banks
        const uint16_t *p = (const uint16_t *)a.x + row + c;
        uint32_t w[4] = {0, 0, 0, 0};
        if (c + 8 <= a.C && (uintptr_t)p % 16 == 0) {
            *(uint4 *)w = *(const uint4 *)p;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < a.C) w[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
        }
        const int at = a.tiles ? tile_at : ((in_seg >> 2) * a.cols + col) * 64 + ((o & 3) ^ (col >> 1 & 3)) * 16;
        *(uint4 *)(seg + at) =
            make_uint4(__byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632), __byte_perm(w[1], w[3], 0x5410),
                       __byte_perm(w[1], w[3], 0x7632));
        return;
    }
    char *const digits = seg + ((in_seg >> 3) * a.cols + col) * 64 + (o & 3) * 16 + (in_seg >> 2 & 1) * 8;
    int *const starts = (int *)(seg + a.cols * 256) + in_seg * 8 / a.group * a.cols + col;
    const int lanes = a.group / 8;  // of a group
    const bool lead = (in_seg & (lanes - 1)) == 0;
    const auto start = [&](int part, int sum) {
        for (int d = lanes / 2; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        if (lead) starts[part] = -8 * sum;
    };
    if (MODE == Q4_BITS) {
        uint32_t w = c < a.C ? ((const uint32_t *)a.x)[row + (c >> 5)] >> (c & 31) & 255u : 0u;
        if (c < a.C && c + 8 > a.C) w &= (1u << (a.C - c)) - 1u;
        if (a.tiles) {  // fp16 ones, in the order above
            const auto ones = [&](int j) { return (w >> j & 1u) * 0x3C00u | (w >> (j + 4) & 1u) * 0x3C000000u; };
            *(uint4 *)(seg + tile_at) = make_uint4(ones(0), ones(1), ones(2), ones(3));
            return;
        }
        const auto spread = [](uint32_t v) { return (v & 1u) | (v & 4u) << 6 | (v & 16u) << 12 | (v & 64u) << 18; };
        *(uint2 *)digits = make_uint2(spread(w), spread(w >> 1));
        start(0, __popc(w));
        return;
    }
    float v[8], top = 0.f;
    load_octet(a, row, c, v);
    bool nan = false;
    int infs = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        nan |= v[j] != v[j];
        infs += fabsf(v[j]) == INFINITY;
        top = fmaxf(top, fabsf(v[j]));
    }
    for (int d = 8; d; d >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, d);
        infs += __shfl_xor_sync(0xFFFFFFFFu, infs, d);
    }
    // top < 2^(e + 1): |x| 2^(29 - e) < 2^30.  An infinity among the 128 becomes
    // the digit 1 of an infinite factor and the others 0; several of them, whose
    // signs would have to be told apart class by class, give NaN.
    const int e = (int)(__float_as_uint(top) >> 23) - 127;
    uint32_t even[4] = {0, 0, 0, 0}, odd[4] = {0, 0, 0, 0};
    int sums[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        int X = infs ? (fabsf(v[j]) == INFINITY ? (v[j] > 0.f ? 1 << 24 : -(1 << 24)) : 0) : __float2int_rn(scalbnf(v[j], 29 - e));
        if (nan) X = 0;
#pragma unroll
        for (int part = 3; part >= 0; --part) {
            const int d = part ? (int)(int8_t)(X & 255) : X;
            X = (X - d) >> 8;
            sums[part] += d;
            (j & 1 ? odd : even)[part] |= (uint32_t)(d & 255) << (8 * (j / 2));
        }
    }
    float *const factors = (float *)(seg + a.cols * (256 + Q4_SEG / a.group * 4)) + (in_seg >> 4) * a.cols + col;
#pragma unroll
    for (int part = 0; part < 4; ++part) {
        *(uint2 *)(digits + part * 64) = make_uint2(even[part], odd[part]);
        start(part, sums[part]);
        if ((in_seg & 15) == 0)
            factors[part] = nan || infs > 1 ? NAN : infs ? (part ? 0.f : INFINITY) : scalbnf(1.f, e - 5 - 8 * part);
    }
}

// ---- products

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{.reg .pred p;\n\tmbarrier.try_wait.parity.shared.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
__device__ __noinline__ bool bar_try_long(uint32_t bar, uint32_t parity) {
    uint64_t start, now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(start));
    for (int i = 0; i < (1 << 24); ++i) {
        if (bar_try(bar, parity)) return true;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
        if (now - start > 2000000000ull) break;
    }
    return false;
}
__device__ __noinline__ bool bar_wait_long(uint32_t bar, uint32_t parity, volatile int &failed) {
    if (failed) return false;
    if (bar_try_long(bar, parity)) return true;
    failed = 1;
    return false;
}
// Waits for the phase with this parity; false, and `failed` set, if it did not
// come within about two seconds, and at once after that.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int &failed) {
    return bar_try(bar, parity) || bar_wait_long(bar, parity, failed);
}

// Blocks whose votes are NaN because a wait gave up (ytm_q4_votes_gave_up).
__device__ unsigned long long g_gave_up;

__device__ __forceinline__ float scale_value(uint32_t raw, int type) {
    if (type == YTM_F32) return __uint_as_float(raw);
    if (type == YTM_F16) return __half2float(__ushort_as_half((unsigned short)raw));
    return __uint_as_float(raw << 16);
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

// Unsigned by signed bytes; `from`: the sums' start.
__device__ __forceinline__ void mma_int(int (&d)[4], const int (&from)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(from[0]), "r"(from[1]), "r"(from[2]), "r"(from[3]));
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

// Adds the cluster's sums `mine` [samples][2^log_rows classes from row0] in
// rank order, and the bias, and writes the votes.
__device__ __forceinline__ void q4_join(const Q4Args &a, float *mine, int rank, int row0, int log_rows, int64_t sample0, int samples) {
    const int outs = samples << log_rows;
    __syncthreads();
    if (a.cluster > 1) cg::this_cluster().sync();
    for (int u = rank * (int)blockDim.x + (int)threadIdx.x; u < outs; u += a.cluster * (int)blockDim.x) {
        const int i = u >> log_rows, r = u & ((1 << log_rows) - 1);
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

// COLS: the columns of a block, padded to a multiple of 8.
template <Q4Mode MODE, int COLS, int GROUP>
__global__ void __launch_bounds__(Q4_THREADS, COLS == 8 ? 3 : COLS <= 32 ? 2 : 1) k_q4_votes(const Q4Args a, const __grid_constant__ CUtensorMap weights) {
    constexpr int NT = COLS / 8, SEG_BYTES = q4_seg_bytes(MODE, COLS, GROUP);
    extern __shared__ __align__(1024) char smem[];  // weights, activations; barriers at the end
    uint64_t *const bars = (uint64_t *)(smem + a.bars_at);
    volatile int &failed = *(int *)(bars + 2 * Q4_STAGES), &copied = *((int *)(bars + 2 * Q4_STAGES) + 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int WK = 1 << a.log_wk, WM = Q4_WARPS >> a.log_wk;
    const int rank = a.cluster > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int row0 = (int)(blockIdx.x / a.cluster) * 16 * WM;
    // this block's stages of the clauses: WK segments each
    const int per = (a.stages + a.cluster - 1) / a.cluster;
    const int first = min(rank * per, a.stages), count = min(first + per, a.stages) - first;
    const int x_bytes = SEG_BYTES * WK;  // of a stage
    char *const xs = smem + Q4_STAGES * Q4_STAGE_BYTES;
    const uint32_t smem_at = (uint32_t)__cvta_generic_to_shared(smem);
    const uint32_t full = (uint32_t)__cvta_generic_to_shared(bars), empty = full + 8 * Q4_STAGES;
    if (tid == 0) {
        failed = 0;
        for (int s = 0; s < Q4_STAGES; ++s) {
            bar_init(full + 8 * s, 1);
            bar_init(empty + 8 * s, Q4_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    constexpr int GPS = Q4_SEG / GROUP, GPL = (GPS + 3) / 4;
    const int g = lane >> 2, t = lane & 3, wm = warp % WM, wk = warp / WM;
    float tot[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) tot[n][i] = 0.f;

    if (warp == Q4_WARPS) {
        if (lane == 0) {
            const char *const x0 = a.xs + blockIdx.z * a.xs_block + (int64_t)first * x_bytes;
            const auto copy_weights = [&](int s) {
                const uint32_t at = smem_at + (s % Q4_STAGES) * Q4_STAGE_BYTES, bar = full + 8 * (s % Q4_STAGES);
                bar_expect(bar, Q4_STAGE_BYTES + x_bytes);
                for (int k = 0; k < WK; ++k)
                    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                                 ::"r"(at + k * WM * 2048), "l"(&weights), "r"(((first + s) * WK + k) * 128), "r"(row0), "r"(bar)
                                 : "memory");
            };
            const auto copy_x = [&](int s) {
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"((uint32_t)__cvta_generic_to_shared(xs) + (s % Q4_STAGES) * x_bytes), "l"(x0 + (int64_t)s * x_bytes),
                               "r"(x_bytes), "r"(full + 8 * (s % Q4_STAGES)) : "memory");
            };
            // the weights do not wait for k_q4_x
            for (int s = 0; s < min(count, Q4_STAGES); ++s) copy_weights(s);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            int s = 0;
            for (; s < min(count, Q4_STAGES); ++s) copy_x(s);
            for (; s < count; ++s) {
                if (!bar_wait(empty + 8 * (s % Q4_STAGES), (s / Q4_STAGES - 1) & 1, failed)) break;
                copy_weights(s);
                copy_x(s);
            }
            copied = s;
        }
    } else {
        // scales: lane t of a class holds groups t, t + 4, ... of a stage; the
        // next stage's are on their way
        const int class0 = row0 + wm * 16 + g, class1 = class0 + 8;
        const bool wide = a.scale_type == YTM_F32;
        const int group0 = (first * WK + wk) * GPS + t, group_step = WK * GPS;
        const int bytes = wide ? 4 : 2;
        const char *sc0 = (const char *)a.scales + ((class0 < a.K ? (int64_t)class0 * a.G : 0) + group0) * bytes;
        const char *sc1 = (const char *)a.scales + ((class1 < a.K ? (int64_t)class1 * a.G : 0) + group0) * bytes;
        int last[GPL];  // stages that have this lane's group (group0 + 4 j + s group_step < G)
#pragma unroll
        for (int j = 0; j < GPL; ++j) last[j] = (a.G - group0 - 4 * j + group_step - 1) / group_step;
        uint32_t next_sc[2][GPL][2];
        const auto load_scales = [&](int s, uint32_t (&to)[GPL][2]) {
#pragma unroll
            for (int j = 0; j < GPL; ++j) {
                to[j][0] = to[j][1] = 0u;  // behind the last group: 0
                if (s < last[j]) {
                    if (wide) {
                        to[j][0] = *(const uint32_t *)(sc0 + 16 * j);
                        to[j][1] = *(const uint32_t *)(sc1 + 16 * j);
                    } else {
                        to[j][0] = *(const uint16_t *)(sc0 + 8 * j);
                        to[j][1] = *(const uint16_t *)(sc1 + 8 * j);
                    }
                }
            }
            sc0 += group_step * bytes;
            sc1 += group_step * bytes;
        };
        load_scales(0, next_sc[0]);
        load_scales(1, next_sc[1]);
        // rows of 128 bytes, their 16-byte pieces exchanged by the row's low bits (128-byte swizzle)
        const int mrow = (lane >> 3 & 1) * 8 + (lane & 7);
        const uint32_t mat = smem_at + (wk * WM + wm) * 2048 + mrow * 128;
        for (int s = 0; s < count; ++s) {
            float sc[GPL][2];
#pragma unroll
            for (int j = 0; j < GPL; ++j) {
                sc[j][0] = scale_value(next_sc[0][j][0], a.scale_type);
                sc[j][1] = scale_value(next_sc[0][j][1], a.scale_type);
                next_sc[0][j][0] = next_sc[1][j][0];
                next_sc[0][j][1] = next_sc[1][j][1];
            }
            load_scales(s + 2, next_sc[1]);
            bar_wait(full + 8 * (s % Q4_STAGES), (s / Q4_STAGES) & 1, failed);
            __syncwarp();
            const uint32_t w_at = mat + (s % Q4_STAGES) * Q4_STAGE_BYTES;
            const char *x_at = xs + (s % Q4_STAGES) * x_bytes + wk * SEG_BYTES;
            const auto words = [&](int j2, uint32_t (&q)[4]) {  // 64 clauses: classes g, g + 8 of the first 32, then of the others
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                             : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3])
                             : "r"(w_at + (((j2 * 2 + (lane >> 4)) ^ (lane & 7)) * 16)) : "memory");
            };
            const auto scales_of = [&](int grp, float &s0, float &s1) {
                const int from = (lane & ~3) | (grp & 3);
                s0 = __shfl_sync(0xFFFFFFFFu, sc[grp / 4][0], from);
                s1 = __shfl_sync(0xFFFFFFFFu, sc[grp / 4][1], from);
            };
            if constexpr (MODE <= Q4_DIGITS) {
                const int *starts = (const int *)(x_at + COLS * 256) + t * 2;
                const float *factors = (const float *)(x_at + COLS * (256 + GPS * 4)) + t * 2;
                constexpr bool SPLIT = MODE == Q4_DIGITS && GROUP < 128;  // several scales under one factor
                int acc[NT][4];
                float sum[SPLIT ? NT : 1][4];
#pragma unroll
                for (int j2 = 0; j2 < Q4_SEG / 64; ++j2) {
                    uint32_t q[4];
                    words(j2, q);
                    uint4 b[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) b[n] = *(const uint4 *)(x_at + (j2 * COLS + n * 8 + g) * 64 + t * 16);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int j = j2 * 2 + h, grp = j / (GROUP / 32);  // 32 clauses
                        const uint32_t a0 = q[2 * h] & 0x0F0F0F0Fu, a1 = q[2 * h + 1] & 0x0F0F0F0Fu;
                        const uint32_t a2 = q[2 * h] >> 4 & 0x0F0F0F0Fu, a3 = q[2 * h + 1] >> 4 & 0x0F0F0F0Fu;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint32_t b0 = h ? b[n].z : b[n].x, b1 = h ? b[n].w : b[n].y;
                            if (j % (GROUP / 32) == 0) {
                                const int2 c = *(const int2 *)(starts + grp * COLS + n * 8);
                                const int from[4] = {c.x, c.y, c.x, c.y};
                                mma_int(acc[n], from, a0, a1, a2, a3, b0, b1);
                            } else {
                                mma_int(acc[n], acc[n], a0, a1, a2, a3, b0, b1);
                            }
                        }
                        if ((j + 1) % (GROUP / 32)) continue;
                        float s0, s1;
                        scales_of(grp, s0, s1);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if constexpr (SPLIT) {
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    sum[n][i] = fmaf(i < 2 ? s0 : s1, (float)acc[n][i], j % 4 == GROUP / 32 - 1 ? 0.f : sum[n][i]);
                                if (j % 4 == 3) {
                                    const float2 f = *(const float2 *)(factors + j / 4 * COLS + n * 8);
#pragma unroll
                                    for (int i = 0; i < 4; ++i) tot[n][i] = fmaf(i & 1 ? f.y : f.x, sum[n][i], tot[n][i]);
                                }
                            } else if constexpr (MODE == Q4_DIGITS) {
                                const float2 f = *(const float2 *)(factors + j / 4 * COLS + n * 8);
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    tot[n][i] = fmaf((i & 1 ? f.y : f.x), (i < 2 ? s0 : s1) * (float)acc[n][i], tot[n][i]);
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; ++i) tot[n][i] = fmaf(i < 2 ? s0 : s1, (float)acc[n][i], tot[n][i]);
                            }
                        }
                    }
                }
            } else {
                constexpr bool HALF = MODE == Q4_FP16;
                const char *x_lane = x_at + g * 64 + (t ^ (g >> 1 & 3)) * 16;
                float acc[NT][4];
#pragma unroll
                for (int j2 = 0; j2 < Q4_SEG / 64; ++j2) {
                    uint32_t q[4];
                    words(j2, q);
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
                            const uint4 b = *(const uint4 *)(x_lane + (j * COLS + n * 8) * 64);
                            mma<HALF>(acc[n], lo[0], hi[0], lo[1], hi[1], b.x, b.y);
                            mma<HALF>(acc[n], lo[2], hi[2], lo[3], hi[3], b.z, b.w);
                        }
                        if ((j + 1) % (GROUP / 32)) continue;
                        float s0, s1;
                        scales_of(j / (GROUP / 32), s0, s1);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) tot[n][i] = fmaf(i < 2 ? s0 : s1, acc[n][i], tot[n][i]);
                    }
                }
            }
            // The stage is given back once its last words have come, not once their
            // loads are issued: the address waits for the sums that they went into
            // (`zero` is 0).  Without that, a warp's last 64 clauses of a stage were
            // now and then those of the stage copied over it.
            uint32_t come = 0;
#pragma unroll
            for (int n = 0; n < NT; ++n) come |= __float_as_uint(tot[n][0]);
            __syncwarp();
            if (lane == 0) bar_arrive(empty + 8 * (s % Q4_STAGES) + (come & a.zero));
        }
    }
    __syncthreads();  // all stages have been read
    if (failed) {  // copies may still be on their way: the memory is not used again, nor given back, before them
        if (tid < Q4_STAGES && tid < copied) {
            const int s = copied - 1 - tid;
            bar_try_long(full + 8 * (s % Q4_STAGES), (s / Q4_STAGES) & 1);
        }
        if (tid == 0) atomicAdd(&g_gave_up, 1ull);
        __syncthreads();
    }
    // sums of the warps along the clauses and of the parts of an activation
    float *red = (float *)smem;                      // [warp][16][COLS]
    float *mine = red + Q4_WARPS * 16 * COLS;        // [samples][16 * WM]
    if (warp < Q4_WARPS) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[(warp * 16 + g + (i >> 1) * 8) * COLS + n * 8 + t * 2 + (i & 1)] = tot[n][i];
    }
    __syncthreads();
    const int64_t sample0 = a.n0 + (int64_t)blockIdx.z * a.samples;
    const int samples = (int)min((int64_t)a.samples, a.n0 + a.n - sample0);
    const int rows = 16 * WM, log_rows = 7 - a.log_wk, outs = rows * samples;
    for (int u = tid; u < outs; u += Q4_THREADS) {
        const int i = u >> log_rows, r = u & (rows - 1);
        float v = failed ? NAN : 0.f;  // NaN: a copy did not come
        for (int k = 0; k < WK; ++k)
            for (int p = 0; p < a.parts; ++p) v += red[((k * WM + (r >> 4)) * 16 + (r & 15)) * COLS + i * a.parts + p];
        mine[u] = v;
    }
    q4_join(a, mine, rank, row0, log_rows, sample0, samples);
}

// ---- products of many samples on the tensor cores' own memory: 16-bit
// activations, and clause bits as fp16 ones (their group sums stay exact)
//
// A block takes 256 classes as two products of 128 by COLS.  Sixteen warps turn
// words into 16-bit pairs as above, a thread a class, and store them into the
// tensor memory as the products' first operand; the activations are the second,
// from shared memory.  A group's sums land in one of two accumulators a
// product, from which eight other warps add them, scaled, to theirs in
// registers.  Every step is handed on by a barrier in shared memory, so copies,
// conversion, products and scaling all run at once, and the hand-overs' latency
// bounds them: leaving out three products of four saves 5%, the conversion's
// arithmetic nothing.  That set the sizes: operands of 128 clauses (of 64: 15%
// slower), two halves of converting warps that take turns (one: 30% slower at 64
// samples), a warp for each product.  8192 x 16384, groups of 64, 64 samples:
// 38 us, 445 TFLOP/s (k_q4_votes 76); groups of 128 29 us.

constexpr int QT_TILES = 2;                           // products of a block
constexpr int QT_THREADS = 32 * 27;                   // 16 warps convert, 8 scale, one copies, one issues each product
constexpr int QT_SCALE = 16, QT_COPY = 24, QT_ISSUE = 25;  // their first
constexpr int QT_ROWS = 128 * QT_TILES, QT_W_BYTES = QT_ROWS * 128;
constexpr int QT_BARS = 384;

__host__ __device__ constexpr int qt_stages(int cols) { return cols == 64 ? 3 : 4; }  // what shared memory holds

struct QtBars {
    uint64_t full[4], empty[4], a_full[QT_TILES][4], a_empty[QT_TILES][4], d_full[QT_TILES][2], d_empty[QT_TILES][2], done[QT_TILES];
    uint32_t tmem;
    int failed, copied;
};
static_assert(sizeof(QtBars) <= QT_BARS, "barriers");

// bar_try_long and bar_wait without a call, which a kernel that deals out its
// registers cannot make; `stop`: ends the wait at once, or NULL.
__device__ __forceinline__ bool bar_poll(uint32_t bar, uint32_t parity, volatile int *stop) {
    if (bar_try(bar, parity)) return true;
    const long long start = clock64();
    do {
        if (bar_try(bar, parity)) return true;
        if (stop && *stop) return false;
    } while (clock64() - start < 4000000000ll);  // about two seconds
    return false;
}
__device__ __forceinline__ bool bar_wait_inline(uint32_t bar, uint32_t parity, volatile int &failed) {
    const bool ok = bar_poll(bar, parity, &failed);
    if (!ok) failed = 1;
    return ok;
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrives at the barrier when the products issued so far are done.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile("{.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;}"
                 ::"r"(d), "r"(a), "l"(b), "r"(shape), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void tc_store16(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                   "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tc_load16(uint32_t at, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at) : "memory");
}

// One lane of a whole warp, always the same.
__device__ __forceinline__ bool elected() {
    uint32_t is;
    asm volatile("{.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;}" : "=r"(is));
    return is;
}

// COLS: the samples of a block, padded to 32, 48 or 64.
template <bool HALF, int COLS, int GROUP>
__global__ void __launch_bounds__(QT_THREADS, 1) k_q4_tiles(const Q4Args a, const __grid_constant__ CUtensorMap weights) {
    constexpr int STAGES = qt_stages(COLS), X_BYTES = COLS * 512, STAGE = QT_W_BYTES + X_BYTES, GPS = Q4_SEG / GROUP;
    // columns of the tensor memory: accumulators [ND][tile][COLS], operands of 128
    // clauses [NA][tile][64]; a stage has a whole number of turns of both
    constexpr int ND = 2, NA = 2, KB = Q4_SEG / NA;
    constexpr uint32_t A_AT = ND * QT_TILES * COLS;
    static_assert(A_AT + NA * QT_TILES * KB / 2 <= 512 && GPS % ND == 0, "tensor memory");
    extern __shared__ __align__(1024) char smem[];
    QtBars &bars = *(QtBars *)(smem + a.bars_at);
    volatile int &failed = bars.failed, &copied = bars.copied;
    const auto bar = [](const uint64_t &b) { return (uint32_t)__cvta_generic_to_shared(&b); };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = a.cluster > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int row0 = (int)(blockIdx.x / a.cluster) * QT_ROWS;
    const int per = (a.stages + a.cluster - 1) / a.cluster;
    const int first = min(rank * per, a.stages), count = min(first + per, a.stages) - first;
    const uint32_t smem_at = (uint32_t)__cvta_generic_to_shared(smem);
    if (tid == 0) {
        failed = 0;
        copied = 0;
        for (int s = 0; s < STAGES; ++s) {
            bar_init(bar(bars.full[s]), 1);
            bar_init(bar(bars.empty[s]), 16 + QT_TILES);  // the converting warps and the products
        }
        for (int t = 0; t < QT_TILES; ++t) {
            for (int s = 0; s < NA; ++s) {
                bar_init(bar(bars.a_full[t][s]), 4);
                bar_init(bar(bars.a_empty[t][s]), 1);
            }
            for (int s = 0; s < ND; ++s) {
                bar_init(bar(bars.d_full[t][s]), 1);
                bar_init(bar(bars.d_empty[t][s]), 4);
            }
            bar_init(bar(bars.done[t]), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == QT_ISSUE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"((uint32_t)__cvta_generic_to_shared(&bars.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // all 512 columns are this block's, so they start at 0: the products' addresses are constants
    constexpr uint32_t tmem = 0;
    if (tid == 0 && *(volatile uint32_t *)&bars.tmem != tmem) failed = 1;
    const int part = warp >> 2 & 1;                       // product of a converting or scaling warp
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;    // its lanes of the tensor memory
    const int row = part * 128 + (warp & 3) * 32 + lane;  // and the thread's class

    const int64_t sample0 = a.n0 + (int64_t)blockIdx.z * a.samples;
    const int samples = (int)min((int64_t)a.samples, a.n0 + a.n - sample0);
    float *const mine = (float *)smem;  // [samples][QT_ROWS]

    if (warp == QT_COPY) {
        if (lane == 0) {
            const char *const x0 = a.xs + blockIdx.z * a.xs_block + (int64_t)first * X_BYTES;
            const auto copy_weights = [&](int s) {
                const uint32_t at = smem_at + s % STAGES * STAGE, b = bar(bars.full[s % STAGES]);
                bar_expect(b, STAGE);
                asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                             ::"r"(at), "l"(&weights), "r"((first + s) * 128), "r"(row0), "r"(b) : "memory");
            };
            const auto copy_x = [&](int s) {
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"(smem_at + s % STAGES * STAGE + QT_W_BYTES), "l"(x0 + (int64_t)s * X_BYTES), "r"(X_BYTES),
                               "r"(bar(bars.full[s % STAGES])) : "memory");
            };
            for (int s = 0; s < min(count, STAGES); ++s) copy_weights(s);  // they do not wait for k_q4_x
            asm volatile("griddepcontrol.wait;" ::: "memory");
            int s = 0;
            for (; s < min(count, STAGES); ++s) copy_x(s);
            for (; s < count; ++s) {
                if (!bar_wait_inline(bar(bars.empty[s % STAGES]), (s / STAGES - 1) & 1, failed)) break;
                copy_weights(s);
                copy_x(s);
            }
            copied = s;
        }
    } else if (warp >= QT_ISSUE) {
        // The whole warp goes along, so that addresses stay in uniform registers; one
        // lane issues (an `if (lane == 0)` around all of this took 100 cycles a product).
        // fp32 sums; operands fp16 or bf16, both with the clauses innermost; 128 by COLS
        constexpr uint32_t SHAPE = 1u << 4 | (HALF ? 0u : 1u << 7 | 1u << 10) | (uint32_t)(COLS / 8) << 17 | 8u << 24;
        // A stage's products; false if a wait gave up.  Its lanes may see that apart,
        // so all go on to the end of the stage (the waits end at once then, and what
        // the products find is this block's memory) and vote behind it.
        const auto issue = [&](auto product, int s) {
            constexpr int t = decltype(product)::value;
            bool ok = bar_wait_inline(bar(bars.full[s % STAGES]), (s / STAGES) & 1, failed);
            // rows of 128 bytes under the 128-byte swizzle, eight of them 1024 bytes from the next eight
            const uint64_t x = (uint64_t)((smem_at + s % STAGES * STAGE + QT_W_BYTES) >> 4) | 1ull << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61;
#pragma unroll
            for (int j = 0; j < NA; ++j) {
                ok &= bar_wait_inline(bar(bars.a_full[t][j]), s & 1, failed);
#pragma unroll
                for (int k0 = 0; k0 < KB; k0 += GROUP) {  // products into one accumulator
                    const int g = (j * KB + k0) / GROUP;  // of the stage
                    // the accumulator's last turn: in this stage or the one before
                    if (s > 0 || g >= ND) ok &= bar_wait_inline(bar(bars.d_empty[t][g % ND]), (s * (GPS / ND) + g / ND - 1) & 1, failed);
                    tc_fence_after();
                    if (elected()) {
#pragma unroll
                        for (int k = k0; k < k0 + GROUP; k += 16)
                            tc_mma((g % ND * QT_TILES + t) * COLS, A_AT + (j * QT_TILES + t) * (KB / 2) + k / 2,
                                   x + (uint64_t)((j * KB + k) / 64 * COLS * 8 + k % 64 / 8), SHAPE, k > k0);
                        tc_commit(bar(bars.d_full[t][g % ND]));
                        if (k0 + GROUP == KB) tc_commit(bar(bars.a_empty[t][j]));
                        if (k0 + GROUP == KB && j == NA - 1) tc_commit(bar(bars.empty[s % STAGES]));
                    }
                    __syncwarp();
                }
            }
            return ok;
        };
        const auto run = [&](auto product) {
            bool ok = true;
            for (int s = 0; s < count && ok; ++s) ok = __all_sync(0xFFFFFFFFu, issue(product, s));
            if (ok) {  // the last arrivals are still on their way to the barriers, whose memory goes with the block
                if (count) bar_wait_inline(bar(bars.empty[(count - 1) % STAGES]), ((count - 1) / STAGES) & 1, failed);
                return;
            }
            // the products on their way still read their operands
            if (elected()) tc_commit(bar(bars.done[decltype(product)::value]));
            bar_poll(bar(bars.done[decltype(product)::value]), 0, nullptr);
        };
        if (warp == QT_ISSUE) run(std::integral_constant<int, 0>());
        else run(std::integral_constant<int, 1>());
    } else if (warp < QT_SCALE) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        const char *const w_row = smem + row * 128;
        // a half of the warps has an operand each, so that one computes while the other waits
        const int j = warp >> 3;
        const uint32_t at = tmem + lanes + A_AT + (j * QT_TILES + part) * (KB / 2);
        for (int s = 0; s < count; ++s) {
            bar_wait_inline(bar(bars.full[s % STAGES]), (s / STAGES) & 1, failed);
            __syncwarp();
            const char *const w_at = w_row + s % STAGES * STAGE;
#pragma unroll
            for (int h = 0; h < KB / 32; ++h) {
                const uint4 q = *(const uint4 *)(w_at + ((j * (KB / 32) + h) ^ (row & 7)) * 16);
                uint32_t v[16], p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unpack<HALF>(i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w, p);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[i * 4 + e] = p[e];
                }
                if (h == 0) {
                    if (s > 0) bar_wait_inline(bar(bars.a_empty[part][j]), (s - 1) & 1, failed);
                    __syncwarp();
                    tc_fence_after();
                }
                tc_store16(at + h * 16, v);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                bar_arrive(bar(bars.a_full[part][j]));
                bar_arrive(bar(bars.empty[s % STAGES]));  // its words have come: their conversion is stored
            }
        }
    } else {
        // of the block's 864 * 72 registers: 512 * 48 for conversion, 256 * 120 here, 96 * 72
        asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
        F2 acc[COLS / 2];
#pragma unroll
        for (int i = 0; i < COLS / 2; ++i) acc[i] = pair(0.f, 0.f);
        // scales of a few groups; the next ones are on their way
        constexpr int CH = GPS < 4 || COLS == 64 ? 2 : 4, AT_ONCE = COLS == 64 ? 32 : COLS == 48 ? 16 : COLS;
        const int k = row0 + row, G = a.G;
        const int64_t of = k < a.K ? (int64_t)k * G : 0;
        const int chunks = count * (GPS / CH);
        uint32_t next[CH];
        const auto load_scales = [&](int c) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int g = first * GPS + c * CH + j;
                next[j] = 0u;  // behind the last group: 0
                if (g < G) next[j] = a.scale_type == YTM_F32 ? ((const uint32_t *)a.scales)[of + g] : ((const uint16_t *)a.scales)[of + g];
            }
        };
        load_scales(0);
        for (int c = 0, g = 0; c < chunks; ++c) {
            float sc[CH];
#pragma unroll
            for (int j = 0; j < CH; ++j) sc[j] = scale_value(next[j], a.scale_type);
            if (c + 1 < chunks) load_scales(c + 1);
#pragma unroll
            for (int j = 0; j < CH; ++j, ++g) {
                bar_wait_inline(bar(bars.d_full[part][g % ND]), (g / ND) & 1, failed);
                __syncwarp();
                tc_fence_after();
                const F2 s2 = pair(sc[j], sc[j]);
                const uint32_t at = tmem + lanes + (g % ND * QT_TILES + part) * COLS;
#pragma unroll
                for (int i0 = 0; i0 < COLS; i0 += AT_ONCE) {
                    uint32_t d[AT_ONCE / 16][16];
#pragma unroll
                    for (int i = 0; i < AT_ONCE / 16; ++i) tc_load16(at + i0 + i * 16, d[i]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (i0 + AT_ONCE == COLS) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(bar(bars.d_empty[part][g % ND]));
                    }
#pragma unroll
                    for (int i = 0; i < AT_ONCE / 2; ++i)
                        acc[i0 / 2 + i] = fma2(pair(__uint_as_float(d[i / 8][2 * i % 16]), __uint_as_float(d[i / 8][2 * i % 16 + 1])), s2, acc[i0 / 2 + i]);
                }
            }
        }
        // The sums go over the first stage, which the other product, up to two stages
        // behind, may still read: first the scaling warps wait for one another.
        asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
        for (int i = 0; i < COLS / 2; ++i) {
            float v, w;
            split(acc[i], v, w);
            if (2 * i < samples) mine[2 * i * QT_ROWS + row] = v;
            if (2 * i + 1 < samples) mine[(2 * i + 1) * QT_ROWS + row] = w;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == QT_ISSUE) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    if (failed) {  // copies may still be on their way; the sums are none
        if (tid < STAGES && tid < copied) {
            const int s = copied - 1 - tid;
            bar_poll(bar(bars.full[s % STAGES]), (s / STAGES) & 1, nullptr);
        }
        if (tid == 0) atomicAdd(&g_gave_up, 1ull);
        __syncthreads();
        for (int u = tid; u < samples * QT_ROWS; u += QT_THREADS) mine[u] = NAN;
    }
    q4_join(a, mine, rank, row0, 8, sample0, samples);
}

// How a call is cut.  The cost of a cut in microseconds, as measured: a stage of
// 16 KB takes 0.37 for each block that its SM holds (the SM's share of the
// memory's rate), or 0.15 to 0.3 for every 8 columns where the products bound
// it; every further round of blocks takes 3 to end and to start, and 6 if they
// are clusters (16384 x 32768, one sample: 256 blocks 49 us, 1024 in clusters of
// four 60 us; 65536 x 100: clusters of 16 6.8 us, 7 blocks 24 us).
struct Q4Plan {
    Q4Mode mode;
    int cols, samples, parts;  // of a block (columns padded); columns of a sample
    int wm, log_wk, cluster, stages;
    int64_t z, xs_block;       // blocks of samples of a launch, bytes of one's activations
    int64_t launches;
    size_t smem;
    bool tiles;                // k_q4_tiles
};

// Bytes of activations laid out at once (clause bits become 8 to 16 times as large): a
// call of more samples takes several launches (4096 bit samples of 65536 x 100 in two
// launches: 450 us against 435).
constexpr int64_t Q4_SCRATCH = 1 << 30;

// Launches of `blocks` blocks of samples, equal but for the last.
static void cut_launches(Q4Plan &p, int64_t blocks) {
    const int64_t most = std::min<int64_t>(65535, std::max<int64_t>(1, Q4_SCRATCH / p.xs_block));
    p.launches = cdiv(blocks, most);
    p.z = cdiv(blocks, p.launches);
}

// Blocks of k_q4_tiles, and the least cost: a stage takes 1.0 to 2.8 us by the
// number of its groups, a block 5 more to start and to end, 7 in a cluster.
static std::pair<Q4Plan, double> cut_tiles(Q4Plan p, int64_t N, int64_t C, int64_t K, int group) {
    p.tiles = true;
    p.samples = (int)cdiv(N, cdiv(N, (int64_t)64));
    p.cols = std::max(32, (p.samples + 15) / 16 * 16);
    p.wm = QT_ROWS / 16;
    p.stages = (int)cdiv(C, Q4_SEG);
    p.xs_block = (int64_t)p.cols * 512 * p.stages;
    cut_launches(p, cdiv(N, p.samples));
    p.smem = qt_stages(p.cols) * (QT_W_BYTES + (size_t)p.cols * 512) + QT_BARS;
    const double stage = (group == 32 ? 2.8 : group == 64 ? 1.7 : 1.15) * (p.cols == 32 ? 0.84 : 1.0);
    const int64_t sms = sm_count(), tiles = cdiv(K, QT_ROWS) * p.z;
    double least = 0;
    for (int cl = 1; cl <= 16 && (cl == 1 || cl <= p.stages); cl *= 2) {
        const int64_t place = cl == 16 ? sms * 3 / 4 : cl == 8 ? sms * 6 / 7 : sms;
        const double cost = p.launches * (double)cdiv(tiles * cl, place) * ((double)cdiv(p.stages, cl) * stage + (cl > 1 ? 7 : 5));
        if (!p.cluster || cost < least * 0.97) {
            p.cluster = cl;
            least = cost;
        }
    }
    return {p, least};
}

// Blocks of k_q4_votes of up to `most` samples, and the least cost.
static std::pair<Q4Plan, double> cut(Q4Plan p, int64_t N, int64_t C, int64_t K, int group, int64_t most) {
    p.samples = (int)cdiv(N, cdiv(N, most));
    const int used = p.samples * p.parts;
    p.cols = used <= 32 ? (used + 7) / 8 * 8 : used <= 48 ? 48 : 64;
    const int seg_bytes = q4_seg_bytes(p.mode, p.cols, group);
    const int64_t sms = sm_count();
    const int nt = p.cols / 8;
    double least = 0;
    for (int wm = 8, log_wk = 0; wm >= 1; wm /= 2, ++log_wk) {
        const int64_t wk = Q4_WARPS / wm;
        const size_t red = (size_t)Q4_WARPS * 16 * p.cols * 4 + (size_t)p.samples * 16 * wm * 4;
        const size_t smem = std::max<size_t>(Q4_STAGES * (Q4_STAGE_BYTES + (size_t)seg_bytes * wk), red) + Q4_BARS;
        if (smem > 227 * 1024) continue;
        const int64_t stages = cdiv(C, Q4_SEG * wk);
        Q4Plan q = p;
        q.xs_block = (int64_t)seg_bytes * wk * stages;
        cut_launches(q, cdiv(N, p.samples));
        const int64_t tiles = cdiv(K, 16 * wm) * q.z;
        const int64_t held = std::max<int64_t>(1, std::min<int64_t>(nt == 1 ? 3 : nt <= 4 ? 2 : 1, 227 * 1024 / (smem + 1024)));  // blocks of an SM
        for (int cl = 1; cl <= 16 && (cl == 1 || cl <= stages); cl *= 2) {
            const int64_t place = cl == 16 ? sms * 3 / 4 : cl == 8 ? sms * 6 / 7 : sms;  // SMs that such clusters reach
            const int64_t rounds = tiles * cl / (place * held), rest = tiles * cl % (place * held);
            const auto stage = [&](int64_t r) { return std::max(0.37 * r, nt > 4 ? 0.19 * nt * r : 0.15 * nt * (1 + r)); };
            const double per = (double)cdiv(stages, cl);
            const double cost = q.launches * (per * (rounds * stage(held) + (rest ? stage(cdiv(rest, place)) : 0)) +
                                              (rounds - (rest ? 0 : 1)) * (cl > 1 ? 6 : 3));
            if (!p.wm || cost < least * 0.97) {
                p.wm = wm;
                p.log_wk = log_wk;
                p.cluster = cl;
                p.stages = (int)stages;
                p.smem = smem;
                p.xs_block = q.xs_block;
                p.z = q.z;
                p.launches = q.launches;
                least = cost;
            }
        }
    }
    return {p, least};
}

static Q4Plan q4_plan_of(int64_t N, int64_t C, int64_t K, int x_type, int group) {
    Q4Plan p = {};
    p.mode = x_type == YTM_BITS ? Q4_BITS : x_type == YTM_F32 || (N <= 2 && K >= 1024) ? Q4_DIGITS : x_type == YTM_F16 ? Q4_FP16 : Q4_BF16;
    p.parts = p.mode == Q4_DIGITS ? 4 : 1;
    // digits: blocks of up to 8 samples, two an SM (21 samples of 8192 x 16384: 92 us
    // against 112 with 16)
    if (p.mode == Q4_DIGITS) return cut(p, N, C, K, group, 8).first;
    // else of up to 64 or 32, whichever costs less (bits, groups of 64: 64 samples of
    // 8192 x 16384 54 us against 58, 256 of 65536 x 100 48 against 37)
    const auto wide = cut(p, N, C, K, group, 64), narrow = cut(p, N, C, K, group, 32);
    const auto best = narrow.second < wide.second ? narrow : wide;
    // Tiles take as long for 3 samples as for 32 and suit many classes: 8192 x 16384,
    // groups of 64, fp16: 16 samples 25 us against 28 in k_q4_votes, 24 31 against 37,
    // 64 38 against 76; bits: 33 34 against 39, 64 38 against 54; groups of 32, fp16:
    // 17 44 against 39, 32 44 against 55.  16384 x 512, fp16: 17 13.0 against 11.9.
    if (K >= 512 && N > (p.mode == Q4_BITS ? group == 32 ? 48 : 32 : group == 32 ? 24 : 16)) {
        // cut's costs are those of bits under groups of 64, without the start
        const double more = (p.mode == Q4_BITS ? 1.0 : 1.35) * (group == 32 ? 1.27 : group == 64 ? 1.0 : 0.85);
        const auto tiles = cut_tiles(p, N, C, K, group);
        if (tiles.second < best.second * more + 7) return tiles.first;
    }
    return best.first;
}

// The thread's last plan again if the sizes are the same: the workspace's size
// and the call ask for it one after the other, and a server's calls are alike.
static const Q4Plan &q4_plan(int64_t N, int64_t C, int64_t K, int x_type, int group) {
    static thread_local int64_t of[6] = {-1, 0, 0, 0, 0, 0};
    static thread_local Q4Plan plan;
    const int64_t now[6] = {N, C, K, x_type, group, sm_count()};
    if (memcmp(of, now, sizeof now)) {
        plan = q4_plan_of(N, C, K, x_type, group);
        memcpy(of, now, sizeof now);
    }
    return plan;
}

// Lets kernel f have `smem` bytes and clusters of 16, once for a device.
template <typename F>
static ytm_status allow_smem(F *f, int smem, std::atomic<uint64_t> &done) {
    int dev = 0;
    ytm_status rc = cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
    if (rc || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return rc;
    if ((rc = cuda_check(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "q4 votes smem"))) return rc;
    if ((rc = cuda_check(cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "q4 votes cluster"))) return rc;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return YTM_OK;
}

// cuTensorMapEncodeTiled, which the driver hands out by name.
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static EncodeTiled f = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return f;
}

using Q4Kernel = void (*)(const Q4Args, const CUtensorMap);

static ytm_status launch_q4(Q4Kernel f, std::atomic<uint64_t> &done, unsigned threads, const Q4Args &a, const Q4Plan &p,
                            const CUtensorMap &map, dim3 grid, cudaStream_t st) {
    ytm_status rc = allow_smem(f, 227 * 1024, done);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)p.cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.cluster > 1 ? 2 : 1;
    return cuda_check(cudaLaunchKernelEx(&cfg, f, a, map), "q4 votes");
}

template <Q4Mode MODE, int COLS, int GROUP>
static ytm_status launch_q4(const Q4Args &a, const Q4Plan &p, const CUtensorMap &map, dim3 grid, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    return launch_q4(k_q4_votes<MODE, COLS, GROUP>, done, Q4_THREADS, a, p, map, grid, st);
}

template <bool HALF, int COLS, int GROUP>
static ytm_status launch_tiles(const Q4Args &a, const Q4Plan &p, const CUtensorMap &map, dim3 grid, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    return launch_q4(k_q4_tiles<HALF, COLS, GROUP>, done, QT_THREADS, a, p, map, grid, st);
}

template <bool HALF, int COLS>
static ytm_status launch_tiles(const Q4Args &a, const Q4Plan &p, const CUtensorMap &map, int group, dim3 grid, cudaStream_t st) {
    if (group == 32) return launch_tiles<HALF, COLS, 32>(a, p, map, grid, st);
    if (group == 64) return launch_tiles<HALF, COLS, 64>(a, p, map, grid, st);
    return launch_tiles<HALF, COLS, 128>(a, p, map, grid, st);
}

template <bool HALF>
static ytm_status launch_tiles(const Q4Args &a, const Q4Plan &p, const CUtensorMap &map, int group, dim3 grid, cudaStream_t st) {
    switch (p.cols) {
        case 32: return launch_tiles<HALF, 32>(a, p, map, group, grid, st);
        case 48: return launch_tiles<HALF, 48>(a, p, map, group, grid, st);
        default: return launch_tiles<HALF, 64>(a, p, map, group, grid, st);
    }
}

template <Q4Mode MODE, int COLS>
static ytm_status launch_q4(const Q4Args &a, const Q4Plan &p, const CUtensorMap &map, int group, dim3 grid, cudaStream_t st) {
    if (group == 32) return launch_q4<MODE, COLS, 32>(a, p, map, grid, st);
    if (group == 64) return launch_q4<MODE, COLS, 64>(a, p, map, grid, st);
    return launch_q4<MODE, COLS, 128>(a, p, map, grid, st);
}

template <Q4Mode MODE>
static ytm_status launch_q4(const Q4XArgs &xa, unsigned x_blocks, const Q4Args &a, const Q4Plan &p, const CUtensorMap &map, int group,
                            dim3 grid, cudaStream_t st) {
    k_q4_x<MODE><<<x_blocks, 256, 0, st>>>(xa);
    ytm_status rc = launch_check("q4 activations");
    if (rc) return rc;
    if constexpr (MODE != Q4_DIGITS)
        if (p.tiles) return launch_tiles<MODE != Q4_BF16>(a, p, map, group, grid, st);
    switch (p.cols) {
        case 8: return launch_q4<MODE, 8>(a, p, map, group, grid, st);
        case 16: return launch_q4<MODE, 16>(a, p, map, group, grid, st);
        case 24: return launch_q4<MODE, 24>(a, p, map, group, grid, st);
        case 32: return launch_q4<MODE, 32>(a, p, map, group, grid, st);
        default: break;
    }
    // digits have up to 8 samples, 32 columns, a block
    if constexpr (MODE != Q4_DIGITS) {
        if (p.cols == 48) return launch_q4<MODE, 48>(a, p, map, group, grid, st);
        if (p.cols == 64) return launch_q4<MODE, 64>(a, p, map, group, grid, st);
    }
    return fail(YTM_ERR_ARG, "q4 votes: no kernel of these columns");
}

static ytm_status check_q4(int32_t C, int32_t K, int32_t group, int32_t scale_type) {
    if (C <= 0 || K <= 0) return fail(YTM_ERR_ARG, "q4: clauses and classes must be positive");
    if (C > (1 << 30) || K > (1 << 30)) return fail(YTM_ERR_UNSUPPORTED, "q4: more than 2^30 clauses or classes");
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

ytm_status ytm_q4_votes_gave_up(uint64_t *out, void *stream) {
    if (!out) return fail(YTM_ERR_ARG, "null pointer");
    unsigned long long n = 0;
    cudaStream_t st = as_stream(stream);
    ytm_status rc = cuda_check(cudaMemcpyFromSymbolAsync(&n, g_gave_up, sizeof n, 0, cudaMemcpyDeviceToHost, st), "q4 votes given up");
    if (!rc) rc = cuda_check(cudaStreamSynchronize(st), "q4 votes given up");
    if (!rc) *out = n;
    return rc;
}

uint64_t ytm_q4_votes_workspace_bytes(int32_t x_type, int64_t N, int32_t C, int32_t K, int32_t group) {
    if (N <= 0 || check_q4(C, K, group, YTM_F32)) return 0;
    const Q4Plan &p = q4_plan(N, C, K, x_type, group);
    return (uint64_t)p.z * p.xs_block;
}

ytm_status ytm_q4_votes(const void *x, int32_t x_type, int64_t x_stride, int64_t N, int32_t C, const uint8_t *packed,
                        const void *scales, int32_t scale_type, int32_t group, int32_t K, const float *bias, void *y,
                        int32_t y_type, void *workspace, void *stream) {
    ytm_status rc = check_q4(C, K, group, scale_type);
    if (rc) return rc;
    if (N < 0) return fail(YTM_ERR_ARG, "N < 0");
    if (!is_float_type(x_type) && x_type != YTM_BITS) return fail(YTM_ERR_ARG, "q4: x must be fp32, fp16, bf16 or packed bits");
    if (!is_float_type(y_type)) return fail(YTM_ERR_ARG, "q4: votes must be fp32, fp16 or bf16");
    if (x_stride < 0) return fail(YTM_ERR_ARG, "q4: negative row stride");
    if (N == 0) return YTM_OK;
    if (!x || !packed || !scales || !y || !workspace) return fail(YTM_ERR_ARG, "null pointer");
    if ((uintptr_t)packed % 16 || (uintptr_t)workspace % 16)
        return fail(YTM_ERR_ARG, "q4: packed weights and workspace must start on a 16-byte boundary");
    cudaStream_t st = as_stream(stream);
    const Q4Plan p = q4_plan(N, C, K, x_type, group);
    // the weights as a matrix of bytes, tiles of 128 bytes by 16 WM classes; zeros outside
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)q4_row_bytes(C), (cuuint64_t)K}, strides[1] = {(cuuint64_t)q4_row_bytes(C)};
    const cuuint32_t box[2] = {128, (cuuint32_t)(16 * p.wm)}, step[2] = {1, 1};
    const EncodeTiled encode = encode_tiled();
    if (!encode) return fail(YTM_ERR_CUDA, "q4 votes: the driver has no cuTensorMapEncodeTiled");
    if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)packed, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return fail(YTM_ERR_CUDA, "q4 votes: cuTensorMapEncodeTiled refused the weights");
    const int64_t most = p.z * p.samples;  // samples of a launch
    const int segs = p.stages << p.log_wk;
    for (int64_t i = 0; i < N; i += most) {
        const int64_t n = std::min(N - i, most);
        const Q4XArgs xa = {x, x_stride, i, n, (char *)workspace, p.xs_block, C, x_type, p.samples, p.parts, p.cols, segs, group, p.tiles};
        const uint64_t blocks = cdiv((uint64_t)n * segs * 32, 256);
        if (blocks > INT_MAX) return fail(YTM_ERR_UNSUPPORTED, "q4 votes: too many activations for one call");
        const Q4Args a = {(const char *)workspace, scales, bias, y, i, n, p.xs_block, K, (int)cdiv(C, group), p.stages, scale_type,
                          y_type, p.samples, p.parts, p.log_wk, p.cluster, (int)p.smem - (p.tiles ? QT_BARS : Q4_BARS), 0u};
        const dim3 grid((unsigned)(cdiv(K, 16 * p.wm) * p.cluster), 1, (unsigned)cdiv(n, p.samples));
        switch (p.mode) {
            case Q4_BITS: rc = launch_q4<Q4_BITS>(xa, (unsigned)blocks, a, p, map, group, grid, st); break;
            case Q4_DIGITS: rc = launch_q4<Q4_DIGITS>(xa, (unsigned)blocks, a, p, map, group, grid, st); break;
            case Q4_BF16: rc = launch_q4<Q4_BF16>(xa, (unsigned)blocks, a, p, map, group, grid, st); break;
            default: rc = launch_q4<Q4_FP16>(xa, (unsigned)blocks, a, p, map, group, grid, st); break;
        }
        if (rc) return rc;
    }
    return YTM_OK;
}

}  // extern "C"
