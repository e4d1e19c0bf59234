// The whole iteration of a small matrix (p <= 64, q <= 768) in one workgroup and one launch: momentum, norm, every step, the
// result or the parameter's update.  What bounds such matrices is not work (64 x 576: 0.3 GFLOP of MFMAs) but the chain of
// dependent launches, four a step through the batched kernels, about 5 us each.  Measured: 64 x 576 48.5 us (7 a step), 64 x 27 21
// (3 a step); what a step waits for is the chain of latencies below, and, with several blocks a wave, their conversions.
//
// Eight waves; wave w owns the 32-column blocks w, w + 8, .. of X (NB at most) and keeps them in registers for good, as
// MFMA fragments: a product's accumulator X^T[q][p] has p across lanes and q down the registers, which is an operand of
// X X^T as it stands (contraction over q, in whatever order both operands share).  Per step:
//   Gram     every wave its blocks, 3 of the 4 subtiles of A (p x p), partial sums through LDS
//   square   A in LDS as plane pairs, B = a I + b A + c A^2, two of its sixteen subtiles a wave, back to LDS
//   apply    X^T <- X^T B, block by block: the one transposition (lanes to q) goes through a patch of LDS of the wave's own
// Three barriers a step.  Numbers are held as in the batched kernels: two fp16 pieces, three MFMAs, fp32 sums,
// those of hl and lh by themselves or first.
#pragma once
#include "newton_schulz.hpp"

namespace dvae {

using f16x4 = __attribute__((ext_vector_type(4))) _Float16;
using f32x2 = __attribute__((ext_vector_type(2))) float;

constexpr int NS_SMALL_P = 64, NS_SMALL_Q = 768, NS_SMALL_VEC = 1 << 15, NS_SMALL_JOBS = 32;
constexpr long NS_SMALL_SPAN = 1L << 28;                  // elements between a matrix's first and last: offsets of 32 bits

struct NsSmallArgs {
    NsJob jobs[NS_SMALL_JOBS];
    const NsJob* table;                                   // on the device, where there are more: then not NULL
    double eps;
    float a, b, c;
    float rate;                                           // see ns_shift
    float mu, nu, lr, decay;
    int nesterov, steps;
};
static_assert(sizeof(NsSmallArgs) <= 4096, "kernel arguments");

struct NsSmallLds {
    // A wave's partial Gram subtiles, two rows of a lane's column at a time: [3][8][lane][2].  Between two Grams the wave's
    // transposition patch lies in them: [32 q] rows of 64 (h, l) pairs of p, sixteen 16-byte chunks stored at chunk ^ turn(row)
    // (writes of 32 pairs in two rows 4 apart and reads of a chunk of sixteen rows meet all banks once), or, PITCH bytes apart, of
    // 64 floats while the matrix comes and goes.
    static constexpr int PITCH = 272;
    f32x2 sum[8][3 * 8 * 64];
    char a[64 * 256], b[64 * 256];                        // plane pairs, [line][row], chunks swizzled as in NsTile
    float diag[64];                                       // of A, see ns_polynomial
    double red[8];
};

// 16-byte chunk `chunk` of row `row` of line `line`
__device__ inline int ns_small_at(int line, int row, int chunk) { return (line * 64 + row) * 128 + ((chunk ^ (row >> 1 & 7)) << 4); }

// The lane, for a phase of a step.  Addresses are worked out anew in every one: the compiler would hold some hundred of them over
// the loop, in registers that the matrix needs.
__device__ inline int ns_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

struct NsBlock {
    f16x8 h[2][2], l[2][2];                               // [32 rows of p][half of the block's q]
};

template <typename T, bool MUON, int NB>
__global__ __launch_bounds__(512) void ns_small_kernel(NsSmallArgs g) {
    extern __shared__ __align__(16) char smem[];
    NsSmallLds& s = *reinterpret_cast<NsSmallLds*>(smem);
    const NsJob j = g.table ? g.table[blockIdx.x] : g.jobs[blockIdx.x];
    const int m = j.m, n = j.n;
    const cgbytes x = as_global<const char>(j.x);
    const gbytes out = as_global<char>(j.out), mom = as_global<char>(j.mom);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    if (MUON && j.vec) {
        const auto gr = as_global<const float>(j.x);
        const auto par = as_global<float>(j.out), mo = as_global<float>(j.mom);
        for (int e = threadIdx.x; e < m * n; e += 512) {
            const float mi = g.mu * mo[e] + g.nu * gr[e];
            mo[e] = mi;
            par[e] = par[e] * g.decay - g.lr * (g.nesterov ? g.nu * gr[e] + g.mu * mi : mi);
        }
        return;
    }
    const bool tall = m > n;
    const int p = tall ? n : m, q = tall ? m : n;
    constexpr int PITCH = NsSmallLds::PITCH / 4;
    float* patch = reinterpret_cast<float*>(s.sum[wave]);

    // A block's elements as the caller's memory has them along lanes: a tall matrix's rows hold p (one q at a time), another's
    // q (32 of two p's).  Of the sixteen of half t a lane has the first `count`, `leap` apart from `at` on (bytes; the host sees
    // to it that they fit 32 bits); those that do not exist read the first one of all and count as zero.
    struct Half {
        int count;
        unsigned at;
    };
    auto half_of = [&](int q0, int t, unsigned stride) {
        Half r;
        r.count = tall ? (lane < p ? q - q0 - t * 16 : 0) : (q0 + col < q ? (p - t * 32 - half + 1) >> 1 : 0);
        const unsigned at = (tall ? (q0 + t * 16) * stride + lane : (t * 32 + half) * stride + q0 + col) * (unsigned)sizeof(T);
        r.at = r.count > 0 ? at : 0u;
        return r;
    };
    // Stores of the elements that exist: of all sixteen in one run where a lane has them, else a branch each.
    auto put = [&](const Half& f, auto&& store) {
        if (f.count >= 16) {
#pragma unroll
            for (int i = 0; i < 16; ++i) store(i);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < f.count) store(i);
        }
    };
    const unsigned xleap = (unsigned)(tall ? j.xs : 2 * j.xs) * (unsigned)sizeof(T), oleap = (unsigned)(tall ? j.os : 2 * j.os) * (unsigned)sizeof(T);
    // where they lie in the patch, [q][p]
    const int patch_leap = tall ? PITCH : 2;
    auto patch_of = [&](int t) { return patch + (tall ? t * 16 * PITCH + lane : col * PITCH + t * 32 + half); };

    // ---- load, all of it in flight at once; then u and its norm, and through the patch to [q][p] ---------------------
    float raw[NB][2][16];
    double sq = 0.0;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        const int q0 = (wave + 8 * k) * 32;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const Half f = half_of(q0, t, (unsigned)j.xs);
#pragma unroll
            for (int i = 0; i < 16; ++i) raw[k][t][i] = (float)*(const DVAE_GLOBAL T*)(x + (f.at + (i < f.count ? i * xleap : 0u)));
        }
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        const int q0 = (wave + 8 * k) * 32;
        if (q0 < q) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const Half f = half_of(q0, t, (unsigned)j.xs);
                float* to = patch_of(t);
                float mv[16];
                if (MUON) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) mv[i] = *(const DVAE_GLOBAL float*)(mom + (f.at + (i < f.count ? i * xleap : 0u)));
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const bool in = i < f.count;
                    float v = in ? raw[k][t][i] : 0.f;
                    if (MUON) {
                        mv[i] = ns_rounded(in ? g.mu * mv[i] + g.nu * v : 0.f);
                        v = g.nesterov ? g.nu * v + g.mu * mv[i] : mv[i];
                    }
                    sq += (double)v * (double)v;
                    to[i * patch_leap] = v;
                }
                if (MUON) put(f, [&](int i) { *(DVAE_GLOBAL float*)(mom + (f.at + i * xleap)) = mv[i]; });
            }
            ns_wave_sync();
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = patch[(8 * (e >> 2) + 4 * half + (e & 3)) * PITCH + i * 32 + col];
                raw[k][i][e] = q0 < q ? v : 0.f;
            }
        ns_wave_sync();
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sq += __shfl_xor(sq, o, 64);
    if (lane == 0) s.red[wave] = sq;
    __syncthreads();
    sq = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sq += s.red[i];
    // times 2^(14 + shift) / (norm + eps), as a power of two and a factor near one: a float does not hold it for every norm
    int power;
    const float factor = (float)frexp(ns_inverse(sq, g.eps), &power);
    const int lead = ns_lead(sqrt(sq), g.eps);
    int shift = ns_shift(lead, g.rate, 0);
    power += shift;

    NsBlock blk[NB];
    // v times `by`, a power of two (so that the product is exact, see ns_rounded), in two pieces; element e of a subtile, e = 8 t + i, is element i of the fragment of half t
    auto hold = [&](NsBlock& b, int i, const float (&v)[16], float by) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const f16 h = (f16)(v[8 * t + e] * by);
                b.h[i][t][e] = h;
                b.l[i][t][e] = (f16)(__builtin_fmaf(v[8 * t + e], by, -(float)h) * NS_SL);
            }
    };
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = ns_rounded(ldexpf(raw[k][i][e], power) * factor);
            hold(blk[k], i, v, 1.f);
        }

    const int used = min(8, (q + 31) / 32);               // waves that own a block
    for (int step = 0; step < g.steps; ++step) {
        const int next = ns_shift(lead, g.rate, step + 1);
        const float gram = ldexpf(NS_SA / (NS_SX * NS_SX), -2 * shift), back = ldexpf(1.f / NS_SB, next - shift);
        // ---- Gram ----
        if (wave < used) {
            const int lane = ns_lane();
            f32x16 acc[3];
#pragma unroll
            for (int t = 0; t < 3; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][e] = 0.f;
            // subtiles (0,0), (1,0), (1,1); first hl and lh of all blocks, a block past q holding zeros, then hh on top
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                const NsBlock& b = blk[k];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.h[0][t], b.l[0][t], acc[0], 0, 0, 0);
                    acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.h[1][t], b.l[0][t], acc[1], 0, 0, 0);
                    acc[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.h[1][t], b.l[1][t], acc[2], 0, 0, 0);
                    acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.l[0][t], b.h[0][t], acc[0], 0, 0, 0);
                    acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.l[1][t], b.h[0][t], acc[1], 0, 0, 0);
                    acc[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.l[1][t], b.h[1][t], acc[2], 0, 0, 0);
                }
            }
#pragma unroll
            for (int t = 0; t < 3; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][e] *= 1.f / NS_SL;
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                const NsBlock& b = blk[k];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.h[0][t], b.h[0][t], acc[0], 0, 0, 0);
                    acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.h[1][t], b.h[0][t], acc[1], 0, 0, 0);
                    acc[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b.h[1][t], b.h[1][t], acc[2], 0, 0, 0);
                }
            }
#pragma unroll
            for (int t = 0; t < 3; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) s.sum[wave][(t * 8 + e) * 64 + lane] = f32x2{acc[t][2 * e], acc[t][2 * e + 1]};
        }
        __syncthreads();
        // ---- A: two rows of each subtile a lane ----
        {
            const int lane = ns_lane(), col = lane & 31, half = lane >> 5, part = wave & 1;
            f32x2 v[3];
            if (used == 8) {
#pragma unroll
                for (int t = 0; t < 3; ++t) {
                    f32x2 f[8];
#pragma unroll
                    for (int w = 0; w < 8; ++w) f[w] = s.sum[w][(t * 8 + wave) * 64 + lane];
                    v[t] = ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
                }
            } else {
#pragma unroll
                for (int t = 0; t < 3; ++t) v[t] = s.sum[0][(t * 8 + wave) * 64 + lane];
                for (int w = 1; w < used; ++w)
#pragma unroll
                    for (int t = 0; t < 3; ++t) v[t] += s.sum[w][(t * 8 + wave) * 64 + lane];
            }
#pragma unroll
            for (int t = 0; t < 3; ++t) {
                const int row = (t ? 32 : 0) + 8 * (wave >> 1) + 4 * half + 2 * part, c = (t == 2 ? 32 : 0) + col;
                f16x2 h, l;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float f = ns_rounded(v[t][i] * gram);
                    if (t != 1 && row + i == c) {
                        s.diag[c] = f;
                        f = 0.f;
                    }
                    h[i] = (f16)f;
                    l[i] = (f16)((f - (float)h[i]) * NS_SL);
                }
                // the lane's two rows of column c are two columns of row c; the subtile below the diagonal is stored as it is, too
                const int chunk = wave >> 1;
                *reinterpret_cast<f16x2*>(s.a + ns_small_at(row >> 5, c, chunk) + (row & 7) * 2) = h;
                *reinterpret_cast<f16x2*>(s.a + ns_small_at(row >> 5, c, 4 + chunk) + (row & 7) * 2) = l;
                if (t == 1) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        *reinterpret_cast<f16*>(s.a + ns_small_at(0, row + i, c >> 3) + (c & 7) * 2) = h[i];
                        *reinterpret_cast<f16*>(s.a + ns_small_at(0, row + i, 4 + (c >> 3)) + (c & 7) * 2) = l[i];
                    }
                }
            }
        }
        __syncthreads();
        // ---- square: two 16x16 subtiles a wave, their lines a 16x16x32 MFMA each ----
        {
            const int lane = ns_lane(), r16 = lane & 15, quarter = lane >> 4;
            const int ti = wave >> 1;
            f32x4 acc[2] = {}, low[2] = {};
#pragma unroll
            for (int line = 0; line < 2; ++line) {
                const f16x8 lh = *reinterpret_cast<const f16x8*>(s.a + ns_small_at(line, ti * 16 + r16, quarter));
                const f16x8 ll = *reinterpret_cast<const f16x8*>(s.a + ns_small_at(line, ti * 16 + r16, 4 + quarter));
                f16x8 rh[2], rl[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int row = ((wave & 1) * 2 + n) * 16 + r16;
                    rh[n] = *reinterpret_cast<const f16x8*>(s.a + ns_small_at(line, row, quarter));
                    rl[n] = *reinterpret_cast<const f16x8*>(s.a + ns_small_at(line, row, 4 + quarter));
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) low[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lh, rl[n], low[n], 0, 0, 0);
#pragma unroll
                for (int n = 0; n < 2; ++n) low[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ll, rh[n], low[n], 0, 0, 0);
#pragma unroll
                for (int n = 0; n < 2; ++n) acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lh, rh[n], acc[n], 0, 0, 0);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                // rows r0 .. r0 + 3 of column c, that is of row c, A being symmetric
                const int c = ((wave & 1) * 2 + n) * 16 + r16, r0 = ti * 16 + 4 * quarter;
                const int ah = ns_small_at(r0 >> 5, c, (r0 & 31) >> 3) + (r0 & 7) * 2, al = ns_small_at(r0 >> 5, c, 4 + ((r0 & 31) >> 3)) + (r0 & 7) * 2;
                const f16x4 vh = *reinterpret_cast<const f16x4*>(s.a + ah), vl = *reinterpret_cast<const f16x4*>(s.a + al);
                const float dc = s.diag[c];
                const f32x4 dr = *reinterpret_cast<const f32x4*>(s.diag + r0);
                f16x4 h, l;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float r = ns_rounded(ns_polynomial(g, acc[n][i] + low[n][i] * (1.f / NS_SL), __builtin_fmaf((float)vl[i], 1.f / NS_SL, (float)vh[i]),
                                                             dr[i], dc, r0 + i == c));
                    h[i] = (f16)r;
                    l[i] = (f16)((r - (float)h[i]) * NS_SL);
                }
                *reinterpret_cast<f16x4*>(s.b + ah) = h;
                *reinterpret_cast<f16x4*>(s.b + al) = l;
            }
        }
        __syncthreads();
        // ---- apply ----
        const int lane = ns_lane(), col = lane & 31, half = lane >> 5;
        char* xt = reinterpret_cast<char*>(s.sum[wave]);
        const int turn = (col & 3) | (col >> 3 & 1) << 2 | (col >> 2 & 1) << 3;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const int q0 = (wave + 8 * k) * 32;
            if (q0 < q) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {         // rows 8 (e / 4) + 4 half + e % 4 and 16 further down
                        char* at = xt + (8 * (e >> 2) + 4 * half + (e & 3)) * 256 + (((i * 8 + (col >> 2)) ^ (half << 3) ^ e) << 4) + (col & 3) * 4;
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            *reinterpret_cast<f16x2*>(at + t * 16 * 256) = f16x2{blk[k].h[i][t][e], blk[k].l[i][t][e]};
                    }
                ns_wave_sync();
                f32x16 acc[2], low[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][e] = low[i][e] = 0.f;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const int line = kk >> 1, t = kk & 1;
                    f16x8 lh, ll;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const f16x8 v = *reinterpret_cast<const f16x8*>(xt + col * 256 + (((kk * 4 + half * 2 + c) ^ turn) << 4));
#pragma unroll
                        for (int i = 0; i < 4; ++i) { lh[c * 4 + i] = v[2 * i]; ll[c * 4 + i] = v[2 * i + 1]; }
                    }
                    f16x8 rh[2], rl[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        rh[i] = *reinterpret_cast<const f16x8*>(s.b + ns_small_at(line, i * 32 + col, t * 2 + half));
                        rl[i] = *reinterpret_cast<const f16x8*>(s.b + ns_small_at(line, i * 32 + col, 4 + t * 2 + half));
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) low[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh, rl[i], low[i], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 2; ++i) low[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ll, rh[i], low[i], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 2; ++i) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh, rh[i], acc[i], 0, 0, 0);
                }
                ns_wave_sync();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float v[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] = ns_rounded(acc[i][e] + low[i][e] * (1.f / NS_SL));
                    hold(blk[k], i, v, back);
                }
            }
        }
        shift = next;
    }

    // ---- the result: back through the patch, so that lanes run along the caller's rows -------------------------------
    const float step_len = MUON ? g.lr * j.scale : 0.f, out_scale = ldexpf(1.f / NS_SX, -shift);
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        const int q0 = (wave + 8 * k) * 32;
        if (q0 < q) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    patch[(8 * (e >> 2) + 4 * half + (e & 3)) * PITCH + i * 32 + col] =
                        __builtin_fmaf((float)blk[k].l[i][e >> 3][e & 7], 1.f / NS_SL, (float)blk[k].h[i][e >> 3][e & 7]) * out_scale;
            ns_wave_sync();
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const Half f = half_of(q0, t, (unsigned)j.os);
                const float* from = patch_of(t);
                float old[16];
                if (MUON) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) old[i] = (float)*(const DVAE_GLOBAL T*)(out + (f.at + (i < f.count ? i * oleap : 0u)));
                }
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = from[i * patch_leap];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = ns_rounded(MUON ? old[i] * g.decay - step_len * v[i] : v[i]);
                put(f, [&](int i) { *(DVAE_GLOBAL T*)(out + (f.at + i * oleap)) = (T)v[i]; });
            }
            ns_wave_sync();
        }
    }
}

}  // namespace dvae
