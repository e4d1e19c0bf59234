// Layer norm over the last dimension, forward and backward.
//
//   forward   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), y = (x - mu) r gamma + beta
//   backward  xh = (x - mu) r, g = dy gamma, dx = r (g - mean(g) - xh mean(g xh)),
//             dgamma = sum over rows of dy xh, dbeta = sum over rows of dy
//
// Every statistic and sum is fp32 and taken from registers: the mean first, then the distances d from it.  sum(d) is what
// rounding left of the mean and corrects both it and sum(d^2), so that a row whose mean is large against its spread (a
// constant row at the extreme, where 1 / sqrt(eps) multiplies whatever is left) keeps its digits.  All orders are fixed:
// results are bitwise reproducible, and a row's y and dx do not depend on the other rows of the call.
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
__device__ inline void ln_load(const T* p, int left, float (&v)[LnVec<T>::N]) {
    constexpr int N = LnVec<T>::N;
    if (left >= N) {
        const typename LnVec<T>::V r = *reinterpret_cast<const typename LnVec<T>::V*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)r[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.f;
        if (TAIL) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) v[i] = (float)p[i];
        }
    }
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
// gamma / beta (fp32), N of the columns from c on
template <int N>
__device__ inline void ln_param(const float* p, int c, int C, float missing, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = p && c + i < C ? p[c + i] : missing;
}

// Sum over the LPR lanes of a row; result in all of them.
template <int LPR>
__device__ inline float row_sum(float v) {
#pragma unroll
    for (int o = LPR >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
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

// Two sums at once.
template <int W>
__device__ inline void wg_sum2(float& a, float& b, float (*red)[W]) {
    a = row_sum<64>(a);
    b = row_sum<64>(b);
    if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = a; red[1][threadIdx.x >> 6] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) { a += red[0][i]; b += red[1][i]; }
    __syncthreads();
}

// From the sums of d and d^2 over a row: the mean's correction and 1 / sqrt(v + eps).
struct LnStat {
    float off, inv;
};
__device__ inline LnStat ln_stat(float sum_d, float sum_d2, float c, float eps) {
    LnStat t;
    t.off = sum_d / c;
    const float v = sum_d2 / c - t.off * t.off;
    t.inv = 1.f / sqrtf(fmaxf(v, 0.f) + eps);
    if (v != v) t.inv = v;                               // fmaxf would hide a NaN
    return t;
}

struct LnArgs {
    const void *x, *dy;
    void* y;                       // y, or dx
    const float *gamma, *beta;
    float *mean, *invstd;          // [rows]: written forward (or NULL), read backward
    float* partial;                // backward: [gridDim.x][2][C], or NULL when neither dgamma nor dbeta is wanted
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
    const float cf = (float)a.C;
    for (long r0 = (long)blockIdx.x * RPB * U; r0 < a.rows; r0 += (long)gridDim.x * RPB * U) {
        float v[U][NV][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long r = r0 + u * RPB + slot;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * LPR + lane) * N;
                ln_load<T, TAIL>(x + r * a.xs + c, r < a.rows ? a.C - c : 0, v[u][j]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long r = r0 + u * RPB + slot;
            float s = 0.f, q = 0.f, e = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < N; ++i) s += v[u][j][i];
            const float mean = row_sum<LPR>(s) / cf;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int left = a.C - (j * LPR + lane) * N;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float d = v[u][j][i] - mean;
                    v[u][j][i] = d;
                    e += i < left ? d : 0.f;
                    q += i < left ? d * d : 0.f;
                }
            }
            const LnStat t = ln_stat(row_sum<LPR>(e), row_sum<LPR>(q), cf, a.eps);
            if (r < a.rows) {
                if (lane == 0 && a.mean) { a.mean[r] = mean + t.off; a.invstd[r] = t.inv; }
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int c = (j * LPR + lane) * N;
#pragma unroll
                    for (int i = 0; i < N; ++i) v[u][j][i] = (v[u][j][i] - t.off) * t.inv * ga[j][i] + be[j][i];
                    ln_store<T, TAIL>(y + r * a.ys + c, a.C - c, v[u][j]);
                }
            }
        }
    }
}

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
    float nx[NV][N], nd[NV][N], nm, ni;                  // the next row's data, in flight while this row is worked on
    auto fetch = [&](long r) {
        const bool in = r < a.rows;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + lane) * N;
            ln_load<T, TAIL>(x + r * a.xs + c, in ? a.C - c : 0, nx[j]);
            ln_load<T, TAIL>(dy + r * a.ds + c, in ? a.C - c : 0, nd[j]);
        }
        nm = in ? a.mean[r] : 0.f;
        ni = in ? a.invstd[r] : 0.f;
    };
    fetch((long)blockIdx.x * RPB + slot);
    for (long r0 = (long)blockIdx.x * RPB; r0 < a.rows; r0 += step) {
        const long r = r0 + slot;
        float xh[NV][N], g[NV][N];
        const float mean = nm, inv = ni;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = a.C - (j * LPR + lane) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float h = (nx[j][i] - mean) * inv, d = nd[j][i];
                dg[j][i] += i < left ? d * h : 0.f;
                db[j][i] += d;
                const float gi = d * ga[j][i];
                xh[j][i] = h;
                g[j][i] = gi;
                s1 += gi;
                s2 += i < left ? gi * h : 0.f;
            }
        }
        fetch(r + step);
        const float c1 = row_sum<LPR>(s1) * inv_c, c2 = row_sum<LPR>(s2) * inv_c;
        if (r < a.rows && dx) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * LPR + lane) * N;
#pragma unroll
                for (int i = 0; i < N; ++i) g[j][i] = inv * (g[j][i] - c1 - xh[j][i] * c2);
                ln_store<T, TAIL>(dx + r * a.ys + c, a.C - c, g[j]);
            }
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

// ---- a row in a workgroup of W waves ------------------------------------------------------------------------------
template <typename T, int W, int NV>
__global__ __launch_bounds__(W * 64) void ln_fwd_wide_kernel(LnArgs a) {
    constexpr int N = LnVec<T>::N;
    __shared__ float red[W], red2[2][W];
    const T* x = (const T*)a.x;
    T* y = (T*)a.y;
    const float cf = (float)a.C;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        float v[NV][N];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 64 + (int)threadIdx.x) * N;
            ln_load<T, true>(x + r * a.xs + c, a.C - c, v[j]);
        }
        float s = 0.f, q = 0.f, e = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) s += v[j][i];
        const float mean = wg_sum<W>(s, red) / cf;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = a.C - (j * W * 64 + (int)threadIdx.x) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = v[j][i] - mean;
                v[j][i] = d;
                e += i < left ? d : 0.f;
                q += i < left ? d * d : 0.f;
            }
        }
        wg_sum2<W>(e, q, red2);
        const LnStat t = ln_stat(e, q, cf, a.eps);
        if (threadIdx.x == 0 && a.mean) { a.mean[r] = mean + t.off; a.invstd[r] = t.inv; }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 64 + (int)threadIdx.x) * N;
            float ga[N], be[N];
            ln_param<N>(a.gamma, c, a.C, 1.f, ga);
            ln_param<N>(a.beta, c, a.C, 0.f, be);
#pragma unroll
            for (int i = 0; i < N; ++i) v[j][i] = (v[j][i] - t.off) * t.inv * ga[i] + be[i];
            ln_store<T, true>(y + r * a.ys + c, a.C - c, v[j]);
        }
    }
}

template <typename T, int W, int NV>
__global__ __launch_bounds__(W * 64) void ln_bwd_wide_kernel(LnArgs a) {
    constexpr int N = LnVec<T>::N;
    __shared__ float red[2][W];
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
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        float xh[NV][N], g[NV][N];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 64 + (int)threadIdx.x) * N;
            ln_load<T, true>(x + r * a.xs + c, a.C - c, xh[j]);
            ln_load<T, true>(dy + r * a.ds + c, a.C - c, g[j]);
        }
        const float mean = a.mean[r], inv = a.invstd[r];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = a.C - (j * W * 64 + (int)threadIdx.x) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float h = (xh[j][i] - mean) * inv, d = g[j][i];
                dg[j][i] += i < left ? d * h : 0.f;
                db[j][i] += d;
                const float gi = d * ga[j][i];
                xh[j][i] = h;
                g[j][i] = gi;
                s1 += gi;
                s2 += i < left ? gi * h : 0.f;
            }
        }
        wg_sum2<W>(s1, s2, red);
        const float c1 = s1 * inv_c, c2 = s2 * inv_c;
        if (!dx) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * W * 64 + (int)threadIdx.x) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) g[j][i] = inv * (g[j][i] - c1 - xh[j][i] * c2);
            ln_store<T, true>(dx + r * a.ys + c, a.C - c, g[j]);
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
    const float cf = (float)a.C;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.xs;
        T* y = (T*)a.y + r * a.ys;
        float s = 0.f, q = 0.f, e = 0.f;
        for (int c = threadIdx.x; c < a.C; c += 1024) s += (float)x[c];
        const float mean = wg_sum<16>(s, red) / cf;
        for (int c = threadIdx.x; c < a.C; c += 1024) { const float d = (float)x[c] - mean; e += d; q += d * d; }
        wg_sum2<16>(e, q, red2);
        const LnStat t = ln_stat(e, q, cf, a.eps);
        if (threadIdx.x == 0 && a.mean) { a.mean[r] = mean + t.off; a.invstd[r] = t.inv; }
        for (int c = threadIdx.x; c < a.C; c += 1024)
            y[c] = (T)(((float)x[c] - mean - t.off) * t.inv * (a.gamma ? a.gamma[c] : 1.f) + (a.beta ? a.beta[c] : 0.f));
    }
}

// dx of long rows; the columns' sums come from ln_cols_kernel
template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(LnArgs a) {
    __shared__ float red[16];
    const float inv_c = 1.f / (float)a.C;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = (const T*)a.x + r * a.xs, *dy = (const T*)a.dy + r * a.ds;
        T* dx = (T*)a.y + r * a.ys;
        const float mean = a.mean[r], inv = a.invstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < a.C; c += 1024) {
            const float g = (float)dy[c] * (a.gamma ? a.gamma[c] : 1.f);
            s1 += g;
            s2 += g * (((float)x[c] - mean) * inv);
        }
        const float c1 = wg_sum<16>(s1, red) * inv_c, c2 = wg_sum<16>(s2, red) * inv_c;
        for (int c = threadIdx.x; c < a.C; c += 1024) {
            const float g = (float)dy[c] * (a.gamma ? a.gamma[c] : 1.f);
            dx[c] = (T)(inv * (g - c1 - ((float)x[c] - mean) * inv * c2));
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
        dg += d * (((float)x[r * a.xs + c] - a.mean[r]) * a.invstd[r]);
        db += d;
    }
    float* out = a.partial + (long)blockIdx.y * 2 * a.C;
    out[c] = dg;
    out[a.C + c] = db;
}

// slabs [G][2][C] -> dgamma, dbeta: 64 columns a workgroup, its four waves take every fourth slab
__global__ __launch_bounds__(256) void ln_reduce_kernel(const float* partial, int G, int C, float* dgamma, float* dbeta) {
    __shared__ float red[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int e = blockIdx.x * 64 + lane;                // index into [2][C]
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;        // four chains: their loads are in flight together
    if (e < 2 * C) {
        const float* p = partial + e;
        const long st = 2L * C;
        int g = wave;
        for (; g + 12 < G; g += 16) {
            s0 += p[g * st];
            s1 += p[(g + 4) * st];
            s2 += p[(g + 8) * st];
            s3 += p[(g + 12) * st];
        }
        for (; g < G; g += 4) s0 += p[g * st];
    }
    red[wave][lane] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    if (wave == 0 && e < 2 * C) {
        const float s = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
        float* out = e < C ? dgamma : dbeta;
        if (out) out[e < C ? e : e - C] = s;
    }
}

}  // namespace dvae
