// class_loss.cu — cross entropy of biased, masked, tempered class sums with
// its gradients, in one pass over the class sums.
//
// In units of log2 e: with c = log2(e) / t and z = (v + b) c (allowed classes),
//   e_k = 2^(z_k - m), s = sum e, h = sum e (z - m)         (m = max z)
//   loss = w (ln s - (z_y - m) ln 2)
//   dcs_k = (w / t) (e_k / s - 1[k = y]),  dbias = sum_n dcs
//   dt = -(ln 2 / t) sum_n w (h / s - (z_y - m))
// so the row's exponentials are kept in registers between the sum and the
// gradient, h needs no second look at z, and the class sums are read once.
// A thread keeps the same classes from row to row, so that dbias is summed in
// its registers; what the blocks have summed is added by a second small
// kernel in a fixed order.
#include <cooperative_groups.h>
#include <limits.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "elem.cuh"

namespace ytm {

namespace cg = cooperative_groups;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));  // within 2 steps, 2^0 = 1 exactly
    return y;
}

// One rounding for each operation: a product fused into z - m would leave the
// largest class's exponent off 0.
__device__ __forceinline__ float loss_z(float v, float b, float c) { return __fmul_rn(__fadd_rn(v, b), c); }

// What a row needs besides its class sums.
struct LossRow {
    float w, zy;
    int y;
    bool use, open;
};

template <typename T>
__device__ __forceinline__ LossRow loss_row(const ytm_loss_args &a, int64_t n, float c) {
    LossRow r;
    const int64_t y = index_at(a.target, a.target_64, n);
    r.w = a.weight ? a.weight[n] : 1.f;
    r.use = y >= 0 && y < a.k && r.w != 0.f;
    r.y = r.use ? (int)y : 0;
    r.open = r.use && is_allowed(a.allowed ? a.allowed + n * a.allowed_stride : nullptr, r.y);
    r.zy = loss_z(to_f32(((const T *)a.cs)[n * a.cs_stride + r.y]), a.bias ? a.bias[r.y] : 0.f, c);
    return r;
}

__device__ __forceinline__ float loss_rt(const ytm_loss_args &a) {
    return 1.f / (a.temperature ? *a.temperature : a.temperature_all);
}

// Partial sums of a block (or cluster): dbias [G][k], then dt / (-ln 2 / t) [G].
struct LossPart {
    float *db;
    double *dt;
};

// -------------------------------------------------- rows of few classes
// TPR threads hold a row, 4 * NV classes each: vectors of four where the rows
// are 16-byte (8-byte for 16-bit types) aligned, else neighbouring lanes take
// neighbouring classes.

constexpr int LS_THREADS = 256;

template <int TPR, int NV, bool VEC>
__device__ __forceinline__ int small_class(int lane, int j, int i) {
    return VEC ? (j * TPR + lane) * 4 + i : (j * 4 + i) * TPR + lane;
}

// Bits i = 0..3: class (j, i) is there and allowed.
template <int TPR, int NV, bool VEC>
__device__ __forceinline__ uint32_t small_open(const uint32_t *row, int lane, int j, int K) {
    uint32_t o = 0;
    if constexpr (VEC) {  // four neighbours: bits of one word
        const int k = small_class<TPR, NV, VEC>(lane, j, 0);
        if (k < K) o = (row ? row[k >> 5] >> (k & 31) : ~0u) & (k + 4 <= K ? 15u : (1u << (K - k)) - 1u);
    } else if constexpr (TPR <= 8) {  // the team's 4 * TPR classes: bits of one word
        const int k = small_class<TPR, NV, VEC>(0, j, 0);
        const uint32_t w = k < K ? (row ? row[k >> 5] >> (k & 31) : ~0u) : 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (small_class<TPR, NV, VEC>(lane, j, i) < K) o |= ((w >> (i * TPR + lane)) & 1u) << i;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = small_class<TPR, NV, VEC>(lane, j, i);
            if (k < K && is_allowed(row, k)) o |= 1u << i;
        }
    }
    return o;
}

template <typename T>
struct alignas(4 * sizeof(T)) Vec4 {
    T v[4];
};

template <typename T, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(LS_THREADS, NV >= 4 ? 2 : NV == 2 ? 3 : 4) k_loss_small(const ytm_loss_args a, const LossPart part) {
    constexpr int ROWS = LS_THREADS / TPR;
    extern __shared__ float red[];  // [ROWS][4 * NV * TPR]
    __shared__ double red_dt[LS_THREADS / 32];
    const int lane = threadIdx.x % TPR, team = threadIdx.x / TPR, K = a.k;
    const float rt = loss_rt(a), c = rt * LOG2E;
    // the bias stays in registers while there is room for it
    constexpr bool KEEP = NV < 8;
    const auto bias_of = [&](int j, int i) {
        const int k = small_class<TPR, NV, VEC>(lane, j, i);
        return a.bias && k < K ? a.bias[k] : 0.f;
    };
    float b[KEEP ? NV : 1][4], acc[NV][4];
    uint32_t shared_open = 0;  // bit 4 j + i
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        shared_open |= small_open<TPR, NV, VEC>(a.allowed_stride ? nullptr : a.allowed, lane, j, K) << (4 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (KEEP) b[KEEP ? j : 0][i] = bias_of(j, i);
            acc[j][i] = 0.f;
        }
    }
    double dt = 0.0;
    for (int64_t n0 = (int64_t)blockIdx.x * ROWS; n0 < a.n; n0 += (int64_t)gridDim.x * ROWS) {
        const bool live = n0 + team < a.n;
        const int64_t n = live ? n0 + team : a.n - 1;
        const T *cs = (const T *)a.cs + n * a.cs_stride;
        const LossRow row = loss_row<T>(a, n, c);
        float z[NV][4], m = -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            uint32_t open = shared_open >> (4 * j);
            if (a.allowed_stride) open &= small_open<TPR, NV, VEC>(a.allowed + n * a.allowed_stride, lane, j, K);
            Vec4<T> v;
            if (VEC) {
                const int k = small_class<TPR, NV, VEC>(lane, j, 0);
                if (k + 4 <= K) {
                    if constexpr (sizeof(T) == 4) *(uint4 *)&v = *(const uint4 *)(cs + k);
                    else *(uint2 *)&v = *(const uint2 *)(cs + k);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v.v[i] = cs[min(k + i, K - 1)];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v.v[i] = cs[min(small_class<TPR, NV, VEC>(lane, j, i), K - 1)];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                z[j][i] = (open >> i) & 1u ? loss_z(to_f32(v.v[i]), KEEP ? b[KEEP ? j : 0][i] : bias_of(j, i), c) : -INFINITY;
                m = fmaxf(m, z[j][i]);
            }
        }
#pragma unroll
        for (int d = TPR / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
        float s = 0.f, h = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = z[j][i] - m;
                z[j][i] = ex2(x);
                s += z[j][i];
                h = fmaf(z[j][i], fmaxf(x, -1024.f), h);  // 0 * -inf counts for nothing
            }
#pragma unroll
        for (int d = TPR / 2; d; d >>= 1) {
            s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
            h += __shfl_xor_sync(0xFFFFFFFFu, h, d);
        }
        const bool use = live && row.open;
        const float wt = row.w * rt, f = wt / s;
        T *dcs = (T *)a.dcs + n * (int64_t)K;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float d = z[j][i] * f;
                if (small_class<TPR, NV, VEC>(lane, j, i) == row.y) d -= wt;
                z[j][i] = use ? d : 0.f;
                acc[j][i] += z[j][i];
            }
            if constexpr (!std::is_integral<T>::value) {
                if (a.dcs && live) {
                    const int k = small_class<TPR, NV, VEC>(lane, j, 0);
                    Vec4<T> out;
#pragma unroll
                    for (int i = 0; i < 4; ++i) out.v[i] = from_f32<T>(z[j][i]);
                    if (VEC && k + 4 <= K) {
                        if constexpr (sizeof(T) == 4) *(uint4 *)(dcs + k) = *(uint4 *)&out;
                        else *(uint2 *)(dcs + k) = *(uint2 *)&out;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int ki = small_class<TPR, NV, VEC>(lane, j, i);
                            if (ki < K) dcs[ki] = out.v[i];
                        }
                    }
                }
            }
        }
        if (lane == 0 && live) {
            const float gap = row.zy - m;
            a.loss[n] = use ? row.w * (logf(s) - gap * LN2) : row.use ? row.w * INFINITY : 0.f;
            if (use) dt += (double)row.w * (double)(h / s - gap);
        }
    }
    // the block's sums, teams in order
    constexpr int SLOTS = 4 * NV * TPR;
    if (a.dbias) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[team * SLOTS + small_class<TPR, NV, VEC>(lane, j, i)] = acc[j][i];
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
// A block, or a cluster of up to 16 blocks, holds a row, E classes a thread:
// vectors of 16 bytes where the rows are 16-byte aligned, else neighbouring
// lanes take neighbouring classes.  Blocks of a cluster exchange (m, s, h) by
// writing into each other's shared memory.

struct LossStat {
    float m, s, h;
};

__device__ __forceinline__ LossStat merge(const LossStat &a, const LossStat &b) {
    const float m = fmaxf(a.m, b.m);
    // a.m == m: the factor is 1 also where both are infinite
    const float da = a.m == m ? 0.f : a.m - m, db = b.m == m ? 0.f : b.m - m;
    const float fa = ex2(da), fb = ex2(db);
    // separate roundings: merge(a, b) == merge(b, a), so all lanes of an
    // exchange end with the same bits
    return {m, __fadd_rn(__fmul_rn(fa, a.s), __fmul_rn(fb, b.s)),
            __fadd_rn(__fmul_rn(fa, fmaf(a.s, fmaxf(da, -1024.f), a.h)),
                      __fmul_rn(fb, fmaf(b.s, fmaxf(db, -1024.f), b.h)))};
}

// Blocks an SM holds: 128 registers a thread at 32 classes, 80 at 16, 64 at 8.
constexpr int big_blocks(int threads, int e) { return e == 32 ? 512 / threads : e == 16 ? 3 : 4; }

template <typename T, int THREADS, int E, bool VEC>
__global__ void __launch_bounds__(THREADS, big_blocks(THREADS, E)) k_loss_big(const ytm_loss_args a, const LossPart part, int cluster) {
    constexpr int V = VEC ? 16 / (int)sizeof(T) : 1, NV = E / V, WARPS = THREADS / 32;
    __shared__ LossStat warp_stat[2][WARPS], block_stat[2][16];
    const int tid = threadIdx.x, K = a.k;
    const int rank = cluster > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int team = blockIdx.x / cluster, teams = gridDim.x / cluster;
    const int k0 = rank * THREADS * E + tid * V;  // class (j, i): k0 + j * THREADS * V + i
    const float rt = loss_rt(a), c = rt * LOG2E;
    float b[E], acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int k = k0 + e / V * THREADS * V + e % V;
        b[e] = a.bias && k < K ? a.bias[k] : 0.f;
        acc[e] = 0.f;
    }
    double dt = 0.0;
    int turn = 0;  // changes with every row that is summed
    if (cluster > 1) cg::this_cluster().sync();  // all blocks are there to be written to
    for (int64_t n = team; n < a.n; n += teams) {
        const T *cs = (const T *)a.cs + n * a.cs_stride;
        T *dcs = (T *)a.dcs + n * (int64_t)K;
        const LossRow row = loss_row<T>(a, n, c);
        if (!row.open) {
            if (a.dcs) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int k = k0 + e / V * THREADS * V + e % V;
                    if (k < K) dcs[k] = T(0.f);
                }
            }
            if (tid == 0 && rank == 0) a.loss[n] = row.use ? row.w * INFINITY : 0.f;
            continue;  // the same for every block of the cluster
        }
        const uint32_t *allowed = a.allowed ? a.allowed + n * a.allowed_stride : nullptr;
        float z[E];
        LossStat st = {-INFINITY, 0.f, 0.f};
        uint32_t open = 0;  // bit e: class e of this thread is there and allowed
        if (VEC) {
            uint4 raw[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int k = k0 + j * THREADS * V;
                raw[j] = make_uint4(0, 0, 0, 0);
                if (k + V <= K) {
                    raw[j] = *(const uint4 *)(cs + k);
                    open |= ((1u << V) - 1u) << (j * V);
                } else if (k < K) {
                    for (int i = 0; i < K - k; ++i) ((T *)&raw[j])[i] = cs[k + i];
                    open |= ((1u << (K - k)) - 1u) << (j * V);
                }
            }
            if (allowed) {
                uint32_t bits = 0;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int k = k0 + j * THREADS * V;
                    if (k < K) bits |= (allowed[k >> 5] >> (k & 31) & ((1u << V) - 1u)) << (j * V);
                }
                open &= bits;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const T *v = (const T *)&raw[j];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int e = j * V + i;
                    z[e] = (open >> e) & 1u ? loss_z(to_f32(v[i]), b[e], c) : -INFINITY;
                    st.m = fmaxf(st.m, z[e]);
                }
            }
        } else {
            const T *c0 = cs + k0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool there = k0 + e * THREADS < K;
                z[e] = there ? to_f32(c0[e * THREADS]) : 0.f;
                if (there) open |= 1u << e;
            }
            if (allowed) {  // a warp's classes are the bits of one word
                const uint32_t *w0 = allowed + (k0 >> 5);
                uint32_t bits = 0;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (k0 + e * THREADS < K) bits |= (w0[e * (THREADS / 32)] >> (k0 & 31) & 1u) << e;
                open &= bits;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                z[e] = (open >> e) & 1u ? loss_z(z[e], b[e], c) : -INFINITY;
                st.m = fmaxf(st.m, z[e]);
            }
        }
        const float base = st.m == -INFINITY ? 0.f : st.m;  // nothing here: every e is 0
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float x = z[e] - base;
            z[e] = ex2(x);
            st.s += z[e];
            st.h = fmaf(z[e], fmaxf(x, -1024.f), st.h);
        }
        const float mine = st.m;
#pragma unroll
        for (int d = 16; d; d >>= 1)
            st = merge(st, {__shfl_xor_sync(0xFFFFFFFFu, st.m, d), __shfl_xor_sync(0xFFFFFFFFu, st.s, d),
                            __shfl_xor_sync(0xFFFFFFFFu, st.h, d)});
        if ((tid & 31) == 0) warp_stat[turn][tid >> 5] = st;
        __syncthreads();
        st = warp_stat[turn][tid & (WARPS - 1)];
#pragma unroll
        for (int d = WARPS / 2; d; d >>= 1)
            st = merge(st, {__shfl_xor_sync(0xFFFFFFFFu, st.m, d), __shfl_xor_sync(0xFFFFFFFFu, st.s, d),
                            __shfl_xor_sync(0xFFFFFFFFu, st.h, d)});
        if (cluster > 1) {
            // slots of the other turn may still be read by a slower block;
            // these were last read before the barrier of the turn between
            cg::cluster_group cl = cg::this_cluster();
            if (tid < cluster) *cl.map_shared_rank(&block_stat[turn][rank], tid) = st;
            cl.sync();
            st = block_stat[turn][0];
            for (int i = 1; i < cluster; ++i) st = merge(st, block_stat[turn][i]);
        }
        const float wt = row.w * rt;
        const float f = ex2(mine == st.m ? 0.f : mine - st.m) * (wt / st.s);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            z[e] *= f;
            acc[e] += z[e];
        }
        // the label's class: its owner takes w / t off
        const int o = row.y - k0, oj = o / (THREADS * V), oi = o - oj * THREADS * V;
        if (o >= 0 && oj < NV && oi < V) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e == oj * V + oi) {
                    z[e] -= wt;
                    acc[e] -= wt;
                }
        }
        if constexpr (!std::is_integral<T>::value) {
            if (a.dcs) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int k = k0 + j * THREADS * V;
                    T out[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) out[i] = from_f32<T>(z[j * V + i]);
                    if (VEC && k + V <= K) *(uint4 *)(dcs + k) = *(const uint4 *)out;
                    else
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            if (k + i < K) dcs[k + i] = out[i];
                }
            }
        }
        if (tid == 0 && rank == 0) {
            const float gap = row.zy - st.m;
            a.loss[n] = row.w * (logf(st.s) - gap * LN2);
            dt += (double)row.w * (double)(st.h / st.s - gap);
        }
        turn ^= 1;
    }
    float *db = teams == 1 ? a.dbias : part.db + (int64_t)team * K;
    if (a.dbias) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int k = k0 + e / V * THREADS * V + e % V;
            if (k < K) db[k] = acc[e];
        }
    }
    if (tid == 0 && rank == 0) {
        if (teams > 1) part.dt[team] = dt;
        else if (a.dtemperature) *a.dtemperature = (float)(-dt * (double)LN2 * (double)rt);
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

// How a call is cut: which kernel, how many teams of how many blocks.
struct LossPlan {
    bool big;
    int threads, e, cluster;  // big
    int tpr, nv;              // small
    int64_t teams;            // blocks (small) or clusters (big): parts to join
};

constexpr int LOSS_CHAIN = 256;  // rows that one team adds up in fp32 at most

static ytm_status loss_plan(int64_t n, int64_t k, LossPlan &p) {
    p = LossPlan{};
    const int sms = sm_count();
    if (k <= 1024) {
        p.tpr = k <= 16 ? 4 : k <= 128 ? 8 : k <= 256 ? 16 : 32;
        p.nv = k <= 32 ? 1 : k <= 64 ? 2 : k <= 512 ? 4 : 8;
        const int64_t rows = LS_THREADS / p.tpr;
        // up to four rounds of one block cost less than joining blocks
        p.teams = n <= 4 * rows ? 1 : std::min<int64_t>(cdiv(n, rows), (int64_t)sms * 4);
        p.teams = std::max<int64_t>(p.teams, cdiv(n, rows * LOSS_CHAIN));
        return YTM_OK;
    }
    p.big = true;
    p.threads = k <= 131072 ? 256 : 512;
    p.e = k <= 2048 ? 8 : k <= 4096 ? 16 : 32;
    p.cluster = 1;
    while ((int64_t)p.cluster * p.threads * p.e < k) p.cluster *= 2;
    if (p.cluster > 16) return fail(YTM_ERR_UNSUPPORTED, "class loss: more than 262,144 classes");
    p.teams = std::min<int64_t>(n, std::max<int64_t>(1, (int64_t)sms * big_blocks(p.threads, p.e) / p.cluster));
    p.teams = std::max<int64_t>(p.teams, cdiv(n, LOSS_CHAIN));
    return YTM_OK;
}

template <typename T, int THREADS, int E>
static ytm_status launch_big(const ytm_loss_args &a, const LossPlan &p, const LossPart &part, bool vec, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.teams * p.cluster));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    auto *f = vec ? k_loss_big<T, THREADS, E, true> : k_loss_big<T, THREADS, E, false>;
    ytm_status rc;
    if (p.cluster > 8 && (rc = cuda_check(cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                                          "class loss cluster")))
        return rc;
    return cuda_check(cudaLaunchKernelEx(&cfg, f, a, part, p.cluster), "class loss");
}

template <typename T, int TPR, int NV>
static ytm_status launch_small(const ytm_loss_args &a, const LossPlan &p, const LossPart &part, bool vec, cudaStream_t st) {
    const size_t smem = (size_t)LS_THREADS * NV * 16;
    if (vec) k_loss_small<T, TPR, NV, true><<<(unsigned)p.teams, LS_THREADS, smem, st>>>(a, part);
    else k_loss_small<T, TPR, NV, false><<<(unsigned)p.teams, LS_THREADS, smem, st>>>(a, part);
    return launch_check("class loss");
}

template <typename T>
static ytm_status launch_loss(const ytm_loss_args &a, const LossPlan &p, const LossPart &part, cudaStream_t st) {
    // vectors: 16 bytes in the big kernel, four classes in the small one
    const uint64_t step = p.big ? 16 : 4 * sizeof(T);
    const bool vec = (uintptr_t)a.cs % step == 0 && a.cs_stride * sizeof(T) % step == 0 &&
                     (!a.dcs || ((uintptr_t)a.dcs % step == 0 && (uint64_t)a.k * sizeof(T) % step == 0));
    if (p.big) {
        if (p.threads == 512) return launch_big<T, 512, 32>(a, p, part, vec, st);
        if (p.e == 8) return launch_big<T, 256, 8>(a, p, part, vec, st);
        if (p.e == 16) return launch_big<T, 256, 16>(a, p, part, vec, st);
        return launch_big<T, 256, 32>(a, p, part, vec, st);
    }
    if (p.tpr == 4) return launch_small<T, 4, 1>(a, p, part, vec, st);
    if (p.tpr == 8 && p.nv == 1) return launch_small<T, 8, 1>(a, p, part, vec, st);
    if (p.tpr == 8 && p.nv == 2) return launch_small<T, 8, 2>(a, p, part, vec, st);
    if (p.tpr == 8) return launch_small<T, 8, 4>(a, p, part, vec, st);
    if (p.tpr == 16) return launch_small<T, 16, 4>(a, p, part, vec, st);
    if (p.nv == 4) return launch_small<T, 32, 4>(a, p, part, vec, st);
    return launch_small<T, 32, 8>(a, p, part, vec, st);
}

}  // namespace ytm

using namespace ytm;

extern "C" {

uint64_t ytm_class_loss_workspace_bytes(int64_t n, int32_t k) {
    LossPlan p;
    if (n <= 0 || k <= 0 || loss_plan(n, k, p) || p.teams == 1) return 0;
    return align_up((uint64_t)p.teams * 8, 256) + (uint64_t)p.teams * k * 4;
}

ytm_status ytm_class_loss(const ytm_loss_args *args, void *workspace, void *stream) {
    if (!args) return fail(YTM_ERR_ARG, "args is NULL");
    const ytm_loss_args &a = *args;
    if (a.n < 0 || a.k <= 0) return fail(YTM_ERR_ARG, "class loss: needs n >= 0 rows of k >= 1 classes");
    if (a.n > INT_MAX) return fail(YTM_ERR_UNSUPPORTED, "class loss: more than 2^31 - 1 rows");
    if (!is_sum_type(a.cs_type)) return fail(YTM_ERR_ARG, "class loss: class sums must be int32, fp32, fp16 or bf16");
    if (a.cs_type == YTM_I32 && a.dcs) return fail(YTM_ERR_ARG, "class loss: int32 class sums have no gradient");
    if (a.cs_stride < 0 || a.allowed_stride < 0) return fail(YTM_ERR_ARG, "class loss: negative stride");
    cudaStream_t st = as_stream(stream);
    ytm_status rc;
    if (a.n == 0) {
        if (a.dbias && (rc = cuda_check(cudaMemsetAsync(a.dbias, 0, (size_t)a.k * 4, st), "memset"))) return rc;
        if (a.dtemperature && (rc = cuda_check(cudaMemsetAsync(a.dtemperature, 0, 4, st), "memset"))) return rc;
        return YTM_OK;
    }
    LossPlan p;
    if ((rc = loss_plan(a.n, a.k, p))) return rc;
    if (!a.cs || !a.target || !a.loss || (p.teams > 1 && !workspace)) return fail(YTM_ERR_ARG, "null pointer");
    LossPart part = {nullptr, nullptr};
    if (p.teams > 1) part = {(float *)((char *)workspace + align_up((uint64_t)p.teams * 8, 256)), (double *)workspace};
    switch (a.cs_type) {
        case YTM_I32: rc = launch_loss<int32_t>(a, p, part, st); break;
        case YTM_F32: rc = launch_loss<float>(a, p, part, st); break;
        case YTM_F16: rc = launch_loss<__half>(a, p, part, st); break;
        default: rc = launch_loss<__nv_bfloat16>(a, p, part, st); break;
    }
    if (rc || p.teams == 1 || (!a.dbias && !a.dtemperature)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.dbias ? cdiv(a.k, 32) : 0) + 1);
    cfg.blockDim = dim3(1024);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cuda_check(cudaLaunchKernelEx(&cfg, k_loss_join, a, part, (int)p.teams), "class loss sums");
}

}  // extern "C"
