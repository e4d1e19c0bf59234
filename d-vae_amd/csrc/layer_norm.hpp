// Layer norm over the last dimension, forward and backward.
//
//   forward   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), y = (x - mu) r gamma + beta
//   backward  xh = (x - mu) r, g = dy gamma, dx = r (g - mean(g) - xh mean(g xh)),
//             dgamma = sum over rows of dy xh, dbeta = sum over rows of dy
//
// Every statistic and sum is fp32 and taken from registers: the mean first, then the distances d from it.  sum(d) is what
// rounding left of the mean and corrects both it and sum(d^2), so that a row whose mean is large against its spread (a
// constant row at the extreme, where 1 / sqrt(eps) multiplies whatever is left) keeps its digits.  The backward pass starts from
// the mean as it was stored, in one fp32 number, and takes what that lost from the sum of its own distances: with h = (x - mean) r
// and c0 = mean(h), xh = h - c0 and mean(g xh) = mean(g h) - c0 mean(g), a third sum beside the two (at a mean of 1e6 spreads the
// stored number alone puts xh off by 0.03).  All orders are fixed: results are bitwise reproducible, and a row's y and dx do not
// depend on the other rows of the call.
//
// The bound is HBM: forward 2, backward 3 passes over the data.  A row lives in the registers of LPR lanes (a power of two,
// as few as cover it with 16-byte vectors, so that narrow rows leave no lane idle) or of a whole workgroup; dgamma / dbeta
// partials stay in registers over all rows a workgroup walks, and leave as one [2][C] slab per workgroup for a second
// launch to add up.  Rows may start at any element (vectors are loaded with element alignment, which costs nothing where
// the address is aligned).
#pragma once
#include "common.hpp"

namespace dvae {

template <typename T> struct LnVec;
template <> struct LnVec<float> {
    static constexpr int N = 4;
    using V = float __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct LnVec<bf16> {
    static constexpr int N = 8;
    using V = __bf16 __attribute__((ext_vector_type(8), aligned(2)));
};

// N values at p[0 .. N), of which `left` exist; what does not exist reads as zero and is not touched in memory.
template <typename T, bool TAIL>
__device__ inline typename LnVec<T>::V ln_load(const T* p, int left) {
    constexpr int N = LnVec<T>::N;
    if (left >= N) return *reinterpret_cast<const typename LnVec<T>::V*>(p);
    typename LnVec<T>::V r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (T)0.f;
    if (TAIL) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) r[i] = p[i];
    }
    return r;
}
template <typename T, bool TAIL>
__device__ inline void ln_store(T* p, int left, const float (&v)[LnVec<T>::N]) {
    constexpr int N = LnVec<T>::N;
    if (left >= N) {
        typename LnVec<T>::V r;
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = (T)v[i];
        *reinterpret_cast<typename LnVec<T>::V*>(p) = r;
    } else if (TAIL) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = (T)v[i];
    }
}
// A distance from the mean for element i of a vector of which `left` elements exist, 0 for the others.  Without a tail a
// vector exists whole or not at all, and a mean of 0 does it for all of an absent one.
template <bool TAIL, int N>
__device__ inline float ln_mean_of(float mean, int left) { return TAIL || left >= N ? mean : 0.f; }
template <bool TAIL>
__device__ inline float ln_only(float v, int i, int left) { return !TAIL || i < left ? v : 0.f; }
// gamma / beta (fp32), N of the columns from c on
template <int N>
__device__ inline void ln_param(const float* p, int c, int C, float missing, float (&v)[N]) {
    if (p && c + N <= C) {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const LnVec<float>::V r = *reinterpret_cast<const LnVec<float>::V*>(p + c + k);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[k + i] = r[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = p && c + i < C ? p[c + i] : missing;
    }
}

// Keeps the compiler from holding what it derived from a vector in registers instead of the vector itself (twice the size and more).
template <typename V>
__device__ inline void ln_forget(V& v) {
    u32x4 r = __builtin_bit_cast(u32x4, v);
    asm volatile("" : "+v"(r));
    v = __builtin_bit_cast(V, r);
}

// Sum over the LPR lanes of a row, in all of them: neighbours, pairs of pairs, halves of 8 and of 16 by data-parallel-primitive
// moves, then the rows of 16 by lane swaps.  Every step adds the same two numbers in either lane, so all lanes agree to the bit.
template <int CTRL>
__device__ inline float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int LPR>
__device__ inline float row_sum(float v) {
    if (LPR > 1) v = dpp_add<0xB1>(v);                   // quad_perm 1,0,3,2
    if (LPR > 2) v = dpp_add<0x4E>(v);                   // quad_perm 2,3,0,1
    if (LPR > 4) v = dpp_add<0x141>(v);                  // row_half_mirror
    if (LPR > 8) v = dpp_add<0x140>(v);                  // row_mirror
    if (LPR > 16) {
        const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false));
        v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    if (LPR > 32) {
        const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false));
        v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    return v;
}
// Sum over a workgroup of W waves; result in every thread.  `red` is W floats, free again after the second barrier.
template <int W>
__device__ inline float wg_sum(float v, float* red) {
    v = row_sum<64>(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += red[i];
    __syncthreads();
    return s;
}

// Several sums at once.
template <int W, int K>
__device__ inline void wg_sums(float (&v)[K], float (*red)[W]) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = row_sum<64>(v[k]);
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) red[k][threadIdx.x >> 6] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        v[k] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) v[k] += red[k][i];
    }
    __syncthreads();
}

// From the sums of d and d^2 over a row: the mean's correction and 1 / sqrt(v + eps).
struct LnStat {
    float off, inv;
};
__device__ inline LnStat ln_stat(float sum_d, float sum_d2, float inv_c, float eps) {
    LnStat t;
    t.off = sum_d * inv_c;
    const float v = sum_d2 * inv_c - t.off * t.off;
    t.inv = rsqrtf((v < 0.f ? 0.f : v) + eps);           // a NaN stays one
    return t;
}

// From the sums over a row of h, g and g h: the means the gradient takes away.
struct LnMeans {
    float c0, c1, c2;
};
__device__ inline LnMeans ln_means(float sum_h, float sum_g, float sum_gh, float inv_c) {
    LnMeans t;
    t.c0 = sum_h * inv_c;
    t.c1 = sum_g * inv_c;
    t.c2 = sum_gh * inv_c - t.c0 * t.c1;
    return t;
}

struct LnArgs {
    const void *x, *dy;
    void* y;                       // y, or dx
    const float *gamma, *beta;
    float *mean, *invstd;          // [rows]: written forward (or NULL), read backward
    float* partial;                // backward: [gridDim.x][2][C], or NULL when neither dgamma nor dbeta is wanted
    float* left;                   // backward, long rows: [rows], c0 for the columns' sums; or NULL
    long xs, ys, ds;               // row strides of x, y (dx), dy in elements
    long rows;
    int C;
    float eps;
};

// ---- rows in LPR lanes ------------------------------------------------------------------------------------------
// 256 threads hold 256 / LPR rows at a time, NV vectors a lane; a workgroup walks its rows U steps at a time with the
// loads of all steps issued together.
template <typename T, int LPR, int NV, int U, bool TAIL>
__global__ __launch_bounds__(256) void ln_fwd_rows_kernel(LnArgs a) {
    constexpr int N = LnVec<T>::N, RPB = 256 / LPR;
    const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const T* x = (const T*)a.x;
    T* y = (T*)a.y;
    float ga[NV][N], be[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + lane) * N;
        ln_param<N>(a.gamma, c, a.C, 1.f, ga[j]);
        ln_param<N>(a.beta, c, a.C, 0.f, be[j]);
    }
    const float inv_c = 1.f / (float)a.C;
    for (long r0 = (long)blockIdx.x * RPB * U; r0 < a.rows; r0 += (long)gridDim.x * RPB * U) {
        typename LnVec<T>::V v[U][NV];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long r = r0 + u * RPB + slot;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * LPR + lane) * N;
                v[u][j] = ln_load<T, TAIL>(x + r * a.xs + c, r < a.rows ? a.C - c : 0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long r = r0 + u * RPB + slot;
            float d[NV][N];
            float s = 0.f, q = 0.f, e = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < N; ++i) s += (float)v[u][j][i];
            const float mean = row_sum<LPR>(s) * inv_c;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int left = a.C - (j * LPR + lane) * N;
                const float m = ln_mean_of<TAIL, N>(mean, left);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    d[j][i] = ln_only<TAIL>((float)v[u][j][i] - m, i, left);
                    e += d[j][i];
                    q += d[j][i] * d[j][i];
                }
            }
            const LnStat t = ln_stat(row_sum<LPR>(e), row_sum<LPR>(q), inv_c, a.eps);
            if (r < a.rows) {
                if (lane == 0 && a.mean) { a.mean[r] = mean + t.off; a.invstd[r] = t.inv; }
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int c = (j * LPR + lane) * N;
#pragma unroll
                    for (int i = 0; i < N; ++i) d[j][i] = (d[j][i] - t.off) * t.inv * ga[j][i] + be[j][i];
                    ln_store<T, TAIL>(y + r * a.ys + c, a.C - c, d[j]);
                }
            }
        }
    }
}

// The next row's data is in flight, as it lies in memory, while a row is worked on.
template <typename T, int LPR, int NV, bool TAIL>
__global__ __launch_bounds__(256) void ln_bwd_rows_kernel(LnArgs a) {
    constexpr int N = LnVec<T>::N, RPB = 256 / LPR;
    __shared__ float red[4][LPR * NV * N];
    const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const T *x = (const T*)a.x, *dy = (const T*)a.dy;
    T* dx = (T*)a.y;
    float ga[NV][N], dg[NV][N], db[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        ln_param<N>(a.gamma, (j * LPR + lane) * N, a.C, 1.f, ga[j]);
#pragma unroll
        for (int i = 0; i < N; ++i) { dg[j][i] = 0.f; db[j][i] = 0.f; }
    }
    const float inv_c = 1.f / (float)a.C;
    const long step = (long)gridDim.x * RPB;
    typename LnVec<T>::V nx[NV], nd[NV];
    float nm, ni;
    auto fetch = [&](long r) {
        const bool in = r < a.rows;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + lane) * N;
            nx[j] = ln_load<T, TAIL>(x + r * a.xs + c, in ? a.C - c : 0);
            nd[j] = ln_load<T, TAIL>(dy + r * a.ds + c, in ? a.C - c : 0);
        }
        nm = in ? a.mean[r] : 0.f;
        ni = in ? a.invstd[r] : 0.f;
    };
    fetch((long)blockIdx.x * RPB + slot);
    for (long r0 = (long)blockIdx.x * RPB; r0 < a.rows; r0 += step) {
        const long r = r0 + slot;
        typename LnVec<T>::V vx[NV], vd[NV];
        const float mean = nm, inv = ni;
#pragma unroll
        for (int j = 0; j < NV; ++j) { vx[j] = nx[j]; vd[j] = nd[j]; }
        fetch(r + step);
        float s0 = 0.f, s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = a.C - (j * LPR + lane) * N;
            const float m = ln_mean_of<TAIL, N>(mean, left);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float h = ln_only<TAIL>(((float)vx[j][i] - m) * inv, i, left), g = (float)vd[j][i] * ga[j][i];
                s0 += h;
                s1 += g;
                s2 += g * h;
            }
        }
        const LnMeans t = ln_means(row_sum<LPR>(s0), row_sum<LPR>(s1), row_sum<LPR>(s2), inv_c);
        const bool put = r < a.rows && dx;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + lane) * N;
            float o[N];
            ln_forget(vx[j]);
            ln_forget(vd[j]);
#pragma unroll
            for (int i = 0; i < N; ++i) {                // of columns that do not exist dy is zero, and nothing is stored
                const float h = ((float)vx[j][i] - mean) * inv - t.c0, d = (float)vd[j][i];
                dg[j][i] += d * h;
                db[j][i] += d;
                o[i] = inv * (d * ga[j][i] - t.c1 - h * t.c2);
            }
            if (put) ln_store<T, TAIL>(dx + r * a.ys + c, a.C - c, o);
        }
    }
    if (!a.partial) return;
    // the row slots of a wave add up by shuffles, the waves through LDS; one slab leaves the workgroup
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float v = which ? db[j][i] : dg[j][i];
#pragma unroll
                for (int o = 32; o >= LPR; o >>= 1) v += __shfl_xor(v, o, 64);
                if ((threadIdx.x & 63) < LPR) red[wave][(j * LPR + lane) * N + i] = v;
            }
        __syncthreads();
        float* out = a.partial + ((long)blockIdx.x * 2 + which) * a.C;
        for (int c = threadIdx.x; c < a.C; c += 256) out[c] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
        __syncthreads();
    }
}

// ---- a row in a workgroup of W waves, the next row's data in flight ---------------------------------------------------
template <typename T, int W, int NV, bool TAIL>
__global__ __launch_bounds__(W * 64) void ln_fwd_wide_kernel(LnArgs a) {
    constexpr int N = LnVec<T>::N;
    __shared__ float red[W], red2[2][W];
    const T* x = (const T*)a.x;
    T* y = (T*)a.y;
    const float inv_c = 1.f / (float)a.C;
    float ga[NV][N], be[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * W * 64 + (int)threadIdx.x) * N;
        ln_param<N>(a.gamma, c, a.C, 1.f, ga[j]);
        ln_param<N>(a.beta, c, a.C, 0.f, be[j]);
    }
    typename LnVec<T>::V n[NV];
    auto fetch = [&](long r) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 64 + (int)threadIdx.x) * N;
            n[j] = ln_load<T, TAIL>(x + r * a.xs + c, r < a.rows ? a.C - c : 0);
        }
    };
    fetch(blockIdx.x);
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        float d[NV][N];
        float s = 0.f, eq[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                d[j][i] = (float)n[j][i];
                s += d[j][i];
            }
        fetch(r + gridDim.x);
        const float mean = wg_sum<W>(s, red) * inv_c;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = a.C - (j * W * 64 + (int)threadIdx.x) * N;
            const float m = ln_mean_of<TAIL, N>(mean, left);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                d[j][i] = ln_only<TAIL>(d[j][i] - m, i, left);
                eq[0] += d[j][i];
                eq[1] += d[j][i] * d[j][i];
            }
        }
        wg_sums<W>(eq, red2);
        const LnStat t = ln_stat(eq[0], eq[1], inv_c, a.eps);
        if (threadIdx.x == 0 && a.mean) { a.mean[r] = mean + t.off; a.invstd[r] = t.inv; }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 64 + (int)threadIdx.x) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) d[j][i] = (d[j][i] - t.off) * t.inv * ga[j][i] + be[j][i];
            ln_store<T, TAIL>(y + r * a.ys + c, a.C - c, d[j]);
        }
    }
}

template <typename T, int W, int NV, bool TAIL>
__global__ __launch_bounds__(W * 64) void ln_bwd_wide_kernel(LnArgs a) {
    constexpr int N = LnVec<T>::N;
    constexpr bool AHEAD = NV * N <= 8;                  // 16 columns a thread leave no registers for the next row
    __shared__ float red[3][W];
    const T *x = (const T*)a.x, *dy = (const T*)a.dy;
    T* dx = (T*)a.y;
    float dg[NV][N], db[NV][N], ga[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        ln_param<N>(a.gamma, (j * W * 64 + (int)threadIdx.x) * N, a.C, 1.f, ga[j]);
#pragma unroll
        for (int i = 0; i < N; ++i) { dg[j][i] = 0.f; db[j][i] = 0.f; }
    }
    const float inv_c = 1.f / (float)a.C;
    typename LnVec<T>::V nx[NV], nd[NV];
    auto fetch = [&](long r) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 64 + (int)threadIdx.x) * N;
            nx[j] = ln_load<T, TAIL>(x + r * a.xs + c, r < a.rows ? a.C - c : 0);
            nd[j] = ln_load<T, TAIL>(dy + r * a.ds + c, r < a.rows ? a.C - c : 0);
        }
    };
    if (AHEAD) fetch(blockIdx.x);
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        typename LnVec<T>::V vx[NV], vd[NV];
        if (!AHEAD) fetch(r);
        const float mean = a.mean[r], inv = a.invstd[r];
#pragma unroll
        for (int j = 0; j < NV; ++j) { vx[j] = nx[j]; vd[j] = nd[j]; }
        if (AHEAD) fetch(r + gridDim.x);
        float s[3] = {0.f, 0.f, 0.f};                    // of h, g and g h
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = a.C - (j * W * 64 + (int)threadIdx.x) * N;
            const float m = ln_mean_of<TAIL, N>(mean, left);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float h = ln_only<TAIL>(((float)vx[j][i] - m) * inv, i, left), g = (float)vd[j][i] * ga[j][i];
                s[0] += h;
                s[1] += g;
                s[2] += g * h;
            }
        }
        wg_sums<W>(s, red);
        const LnMeans t = ln_means(s[0], s[1], s[2], inv_c);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 64 + (int)threadIdx.x) * N;
            float o[N];
            ln_forget(vx[j]);
            ln_forget(vd[j]);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float h = ((float)vx[j][i] - mean) * inv - t.c0, d = (float)vd[j][i];
                dg[j][i] += d * h;
                db[j][i] += d;
                o[i] = inv * (d * ga[j][i] - t.c1 - h * t.c2);
            }
            if (dx) ln_store<T, TAIL>(dx + r * a.ys + c, a.C - c, o);
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (long)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (j * W * 64 + (int)threadIdx.x) * N + i;
            if (c < a.C) { out[c] = dg[j][i]; out[a.C + c] = db[j][i]; }
        }
}

// ---- rows of any length: read once per pass, the later passes out of the cache -------------------------------------
template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(LnArgs a) {
    __shared__ float red[16], red2[2][16];
    const float inv_c = 1.f / (float)a.C;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.xs;
        T* y = (T*)a.y + r * a.ys;
        float s = 0.f, eq[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < a.C; c += 1024) s += (float)x[c];
        const float mean = wg_sum<16>(s, red) * inv_c;
        for (int c = threadIdx.x; c < a.C; c += 1024) { const float d = (float)x[c] - mean; eq[0] += d; eq[1] += d * d; }
        wg_sums<16>(eq, red2);
        const LnStat t = ln_stat(eq[0], eq[1], inv_c, a.eps);
        if (threadIdx.x == 0 && a.mean) { a.mean[r] = mean + t.off; a.invstd[r] = t.inv; }
        for (int c = threadIdx.x; c < a.C; c += 1024)
            y[c] = (T)(((float)x[c] - mean - t.off) * t.inv * (a.gamma ? a.gamma[c] : 1.f) + (a.beta ? a.beta[c] : 0.f));
    }
}

// dx of long rows, and what the stored mean is off by, in spreads, for ln_cols_kernel, where the columns' sums come from
template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(LnArgs a) {
    __shared__ float red[3][16];
    const float inv_c = 1.f / (float)a.C;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = (const T*)a.x + r * a.xs, *dy = (const T*)a.dy + r * a.ds;
        T* dx = (T*)a.y + r * a.ys;
        const float mean = a.mean[r], inv = a.invstd[r];
        float s[3] = {0.f, 0.f, 0.f};
        for (int c = threadIdx.x; c < a.C; c += 1024) {
            const float g = (float)dy[c] * (a.gamma ? a.gamma[c] : 1.f), h = ((float)x[c] - mean) * inv;
            s[0] += h;
            s[1] += g;
            s[2] += g * h;
        }
        wg_sums<16>(s, red);
        const LnMeans t = ln_means(s[0], s[1], s[2], inv_c);
        if (threadIdx.x == 0 && a.left) a.left[r] = t.c0;
        if (!a.y) continue;
        for (int c = threadIdx.x; c < a.C; c += 1024) {
            const float g = (float)dy[c] * (a.gamma ? a.gamma[c] : 1.f);
            dx[c] = (T)(inv * (g - t.c1 - (((float)x[c] - mean) * inv - t.c0) * t.c2));
        }
    }
}

// dgamma / dbeta slabs of long rows: a thread per column, gridDim.y chunks of rows
template <typename T>
__global__ __launch_bounds__(256) void ln_cols_kernel(LnArgs a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.C) return;
    const T *x = (const T*)a.x, *dy = (const T*)a.dy;
    float dg = 0.f, db = 0.f;
    for (long r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float d = (float)dy[r * a.ds + c];
        dg += d * (((float)x[r * a.xs + c] - a.mean[r]) * a.invstd[r] - a.left[r]);
        db += d;
    }
    float* out = a.partial + (long)blockIdx.y * 2 * a.C;
    out[c] = dg;
    out[a.C + c] = db;
}

// slabs [G][2][C] -> dgamma, dbeta: 64 columns a workgroup at a time, its 16 waves take every 16th slab, eight loads in flight each
__global__ __launch_bounds__(1024) void ln_reduce_kernel(const float* partial, int G, int C, float* dgamma, float* dbeta) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long st = 2L * C;
    for (long e = (long)blockIdx.x * 64 + lane; e - lane < st; e += (long)gridDim.x * 64) {       // index into [2][C]
        float s = 0.f;
        if (e < st) {
            const float* p = partial + e;
            for (int g = wave; g < G; g += 128) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = g + 16 * i < G ? p[(g + 16 * i) * st] : 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += v[i];
            }
        }
        red[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && e < st) {
            s = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += red[i][lane];
            float* out = e < C ? dgamma : dbeta;
            if (out) out[e < C ? e : e - C] = s;
        }
        __syncthreads();
    }
}

}  // namespace dvae
