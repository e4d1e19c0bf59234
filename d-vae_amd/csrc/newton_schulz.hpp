// Orthogonalising matrices by the quintic Newton-Schulz iteration, and the Muon update around it.
//
//   X_0 = X / (|X|_F + eps)     A = X X^T, B = a I + b A + c A^2, X <- B X      (`steps` times; p = min(m, n) rows)
//
// (a I folded into B saves the third product an operand.)  A matrix with more rows than columns is iterated as its
// transpose.  A list of matrices of any shapes runs as one batch: every phase is one launch over the tiles of all of them.
//
// Number format.  The iteration multiplies small singular values by up to a^steps (485 for the usual coefficients), so
// products of bf16 operands are off by 1 to 50 percent; fp32 operands would use the fp32 matrix rate, a sixteenth of
// the 16-bit one.  Here an operand is the sum of two fp16 pieces, x = h + l (22 bits), and a product is three MFMAs,
// hh + hl + lh, summed in fp32: the errors of an fp32 product at 3/16 of its time.  fp16's range is met by fixed scales: with
// the coefficients' bounds checked on the host, |X| <= 2, |A| <= 4 and |B| <= 7, held as 2^14 X, 2^13 A and 2^13 B.
//
// Layout.  A plane pair of an R x K operand is made of lines of 128 bytes: 32 h's of a row, then the 32 l's of the same
// columns.  The lines of the R rows follow each other, then those of the next 32 columns: what a tile reads or writes at a time
// is one run of memory.  R and K are padded to 64 with zeros, which the products keep zero.  X is kept with its transpose (two copies,
// taken in turn), so that every product reads both operands along its contraction and every store writes whole lines.
#pragma once
#include "common.hpp"

namespace dvae {

using f16 = _Float16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;

// Pointers that come out of the job table are told to be global memory: the compiler cannot know, and its flat accesses count
// as LDS traffic too, which makes every wait for a fragment one for the loads in flight as well.
#define DVAE_GLOBAL __attribute__((address_space(1)))
using gbytes = DVAE_GLOBAL char*;
using cgbytes = const DVAE_GLOBAL char*;
template <typename T>
__device__ inline DVAE_GLOBAL T* as_global(const void* p) { return (DVAE_GLOBAL T*)(uintptr_t)p; }

constexpr float NS_SX = 16384.f, NS_SA = 8192.f, NS_SB = 8192.f;

enum { NS_NORM, NS_SPLIT, NS_GRAM, NS_SYM, NS_APPLY, NS_PHASES };

struct NsJob {
    const void* x;            // source, or gradient
    void* out;                // result, or parameter
    float* mom;               // momentum (Muon)
    long xs, os;              // row strides in elements
    long off;                 // of X, XT (twice), A, B in the workspace, bytes
    int m, n;                 // as stored
    int vec;                  // Muon: no matrix, a plain momentum step
    int part;                 // first of its norm partials
    int nchunk;               // of its norm
    float scale;              // Muon: factor of the step
};

struct NsArgs {
    const int* first;         // [NS_PHASES][jp]: first workgroup of each job, INT_MAX beyond the last
    const NsJob* jobs;
    double* norm;             // partial sums of squares
    float* part;              // partial products of the Gram phase
    char* ws;
    int njobs, jp;
    int total;                // workgroups of this launch
    int turn;                 // which transposed copy is read
    int kc;                   // Gram: lines of 32 columns a workgroup sums
    float a, b, c;
    double eps;
    float mu, nu, lr, decay;  // momentum, 1 - momentum, step, 1 - step * weight decay: each rounded once from 64 bits
    int nesterov;
};

__host__ __device__ inline int ns_pad(int v) { return (v + 63) & ~63; }
__host__ __device__ inline long ns_job_bytes(int m, int n) {
    const long p = ns_pad(m < n ? m : n), q = ns_pad(m < n ? n : m);
    return 4 * (3 * p * q + 2 * p * p);
}

// ---- the table of jobs -----------------------------------------------------------------------------------------------
// It travels in kernel arguments: nothing on the host has to outlive the call, and a captured launch keeps its own copy.
struct NsBlob {
    static constexpr int WORDS = 896;
    unsigned w[WORDS];
};
__global__ __launch_bounds__(256) void ns_table_kernel(NsBlob blob, unsigned* dst, int words) {
    for (int i = threadIdx.x; i < words; i += 256) dst[i] = blob.w[i];
}

// The job of a workgroup, found by a wave at once: how many firsts are not beyond it.
__device__ inline int ns_find(const NsArgs& g, int phase, int wg, int& local) {
    const int* first = g.first + phase * g.jp;
    const int lane = threadIdx.x & 63;
    int job = -1, start = 0;
    for (int base = 0; base < g.jp; base += 64) {
        const int v = first[base + lane];
        const unsigned long long mask = __ballot(v <= wg);
        const int c = __popcll(mask);
        if (c) {
            job += c;
            start = __shfl(v, c - 1, 64);
        }
        if (c < 64) break;
    }
    local = wg - __builtin_amdgcn_readfirstlane(start);
    return __builtin_amdgcn_readfirstlane(job);
}

// Consecutive workgroups run on different XCDs; neighbouring tiles share operands and go to the same one's L2.
__device__ inline int ns_swizzle(int id, int total) {
    const int per = total >> 3, whole = per << 3;
    return id < whole ? (id & 7) * per + (id >> 3) : id;
}

struct NsPlanes {
    int P, Q;
    gbytes x, xt0, xt1, a, b;
    __device__ NsPlanes(const NsArgs& g, const NsJob& j) {
        P = ns_pad(min(j.m, j.n));
        Q = ns_pad(max(j.m, j.n));
        const long pq = 4L * P * Q;
        x = as_global<char>(g.ws) + j.off;
        xt0 = x + pq;
        xt1 = x + 2 * pq;
        a = x + 3 * pq;
        b = a + 4L * P * P;
    }
    __device__ gbytes xt(int which) const { return which ? xt1 : xt0; }
};

// A value that is about to be split is rounded to fp32 for good.  Left to itself the compiler converts a product to fp16 now
// from its rounded value and now, fused, from its exact one; at a tie the h that is stored and the h that l is the rest of are
// then two neighbours, and the pair is off by 2^-11.
__device__ inline float ns_rounded(float v) {
    asm("" : "+v"(v));
    return v;
}
__device__ inline unsigned ns_split(float v) {           // low half: h, high half: l
    v = ns_rounded(v);
    const f16 h = (f16)v;
    const f16 l = (f16)(v - (float)h);
    const f16x2 r = {h, l};
    return __builtin_bit_cast(unsigned, r);
}

// ---- momentum and norm ---------------------------------------------------------------------------------------------
__device__ inline float ns_momentum(const NsArgs& a, float g, float m) { return a.mu * m + a.nu * g; }
__device__ inline float ns_update(const NsArgs& a, float g, float m) { return a.nesterov ? a.nu * g + a.mu * m : m; }

constexpr int NS_CHUNK = 4096;                           // elements of a norm workgroup's trip

// Sums of squares in 64 bits: no matrix of finite fp32 values overflows them, and long sums keep their digits.
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs g) {
    __shared__ double red[4];
    int chunk;
    const NsJob j = g.jobs[ns_find(g, NS_NORM, blockIdx.x, chunk)];
    const long n = (long)j.m * j.n;
    const auto x = as_global<const T>(j.x);
    const auto mom = as_global<float>(j.mom), par = as_global<float>(j.out);
    double s = 0.0;
    for (long base = (long)chunk * NS_CHUNK; base < n; base += (long)j.nchunk * NS_CHUNK) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const long e = base + i * 256 + threadIdx.x;
            long at = e;
            if (!MUON && j.xs != j.n) at = (unsigned)e / (unsigned)j.n * j.xs + (unsigned)e % (unsigned)j.n;
            v[i] = e < n ? (float)x[at] : 0.f;
        }
        if (MUON) {
            float m[16], p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const long e = base + i * 256 + threadIdx.x;
                m[i] = e < n ? mom[e] : 0.f;
                p[i] = e < n && j.vec ? par[e] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const long e = base + i * 256 + threadIdx.x;
                const float mi = ns_momentum(g, v[i], m[i]);
                if (e < n) mom[e] = mi;
                v[i] = ns_update(g, v[i], mi);
                if (e < n && j.vec) par[e] = p[i] * g.decay - g.lr * v[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s += (double)v[i] * (double)v[i];
    }
    if (j.vec) return;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) g.norm[j.part + chunk] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- X_0 as plane pairs, in both orientations ------------------------------------------------------------------------
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ns_split_kernel(NsArgs g) {
    __shared__ unsigned tile[64][65];
    __shared__ double red[4];
    int t;
    const NsJob j = g.jobs[ns_find(g, NS_SPLIT, blockIdx.x, t)];
    double s = 0.0;
    for (int i = threadIdx.x; i < j.nchunk; i += 256) s += g.norm[j.part + i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    const double inv = (double)NS_SX / (sqrt((red[0] + red[1]) + (red[2] + red[3])) + g.eps);
    const NsPlanes w(g, j);
    const bool tall = j.m > j.n;
    const int ncol = ns_pad(j.n) >> 6;
    const int r0 = t / ncol * 64, c0 = t % ncol * 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = r0 + i * 4 + wave, c = c0 + lane;
        float v = 0.f;
        if (r < j.m && c < j.n) {
            const long e = (long)r * j.xs + c;
            v = (float)as_global<const T>(j.x)[e];
            if (MUON) v = ns_update(g, v, as_global<float>(j.mom)[e]);
            v = (float)((double)v * inv);
        }
        tile[i * 4 + wave][lane] = ns_split(v);
    }
    __syncthreads();
    // a thread writes 16 columns of a row: first in the source's orientation, then in the other
#pragma unroll
    for (int flip = 0; flip < 2; ++flip) {
        gbytes dst = flip ? (tall ? w.x : w.xt0) : (tall ? w.xt0 : w.x);
        const long rows = ns_pad(flip ? j.n : j.m);
        const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
        unsigned h[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned u0 = flip ? tile[c + 2 * i][r] : tile[r][c + 2 * i];
            const unsigned u1 = flip ? tile[c + 2 * i + 1][r] : tile[r][c + 2 * i + 1];
            h[i] = (u0 & 0xffffu) | (u1 << 16);
            l[i] = (u0 >> 16) | (u1 & 0xffff0000u);
        }
        const int row = (flip ? c0 : r0) + r, col = (flip ? r0 : c0) + c;
        gbytes p = dst + ((col >> 5) * rows + row) * 128 + (col & 31) * 2;
        *(DVAE_GLOBAL u32x4*)(p) = u32x4{h[0], h[1], h[2], h[3]};
        *(DVAE_GLOBAL u32x4*)(p + 16) = u32x4{h[4], h[5], h[6], h[7]};
        *(DVAE_GLOBAL u32x4*)(p + 64) = u32x4{l[0], l[1], l[2], l[3]};
        *(DVAE_GLOBAL u32x4*)(p + 80) = u32x4{l[4], l[5], l[6], l[7]};
    }
}

// ---- the products ----------------------------------------------------------------------------------------------------
// C[i][k] = sum over c of L[i][c] R[k][c] for a TS x TS tile: four waves, a quarter tile each, 32x32x16 MFMAs.  Two LDS
// stages of one line (32 columns) per row, one barrier a line: while one half of a line is multiplied, the fragments of the
// other half are on their way from LDS, and the lines after next are on their way from memory in two sets of registers.
// A line's eight 16-byte chunks are stored at chunk ^ (row / 2 & 7): of a fragment's rows any sixteen that are read at a time
// meet the 64 banks once each.
template <int TS>
struct NsTile {
    static constexpr int S = TS / 64;                    // subtiles of a wave each way
    static constexpr int PASS = TS / 32;                 // passes of 256 threads over a stage of one operand
    static constexpr int BYTES = 2 * 2 * TS * 128;
    f32x16 acc[S][S];

    struct Lines { u32x4 l[PASS], r[PASS]; };
    struct Frags { f16x8 lh[S], ll[S], rh[S], rl[S]; };

    __device__ inline void zero() {
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int k = 0; k < S; ++k)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][k][e] = 0.f;
    }

    // MFMAs FROM to TO of the 3 S^2 of half a line
    template <int FROM, int TO>
    __device__ inline void multiply(const Frags& f) {
#pragma unroll
        for (int m = FROM; m < TO; ++m) {
            const int w = m / (S * S), i = m / S % S, n = m % S;
            acc[i][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w == 1 ? f.ll[i] : f.lh[i], w == 0 ? f.rl[n] : f.rh[n], acc[i][n], 0, 0, 0);
        }
    }
    // `lines` is even; rows past lrows / rrows re-read the last one: their results are not stored
    __device__ inline void run(cgbytes L, int lrows, int l0, cgbytes R, int rrows, int r0, int line0, int lines, char* smem) {
        const int tid = threadIdx.x, row = tid >> 3, chunk = tid & 7;
        const int lane = tid & 63, wave = tid >> 6;
        cgbytes lp[PASS], rp[PASS];
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            lp[i] = L + ((long)line0 * lrows + min(l0 + i * 32 + row, lrows - 1)) * 128 + chunk * 16;
            rp[i] = R + ((long)line0 * rrows + min(r0 + i * 32 + row, rrows - 1)) * 128 + chunk * 16;
        }
        Lines set[2];
        int ahead = lines;
        auto fetch = [&](Lines& s) {                      // the next line; past the last one, that one again
#pragma unroll
            for (int i = 0; i < PASS; ++i) {
                s.l[i] = *(const DVAE_GLOBAL u32x4*)lp[i];
                s.r[i] = *(const DVAE_GLOBAL u32x4*)rp[i];
            }
            const bool more = --ahead > 0;
#pragma unroll
            for (int i = 0; i < PASS; ++i) {
                lp[i] += more ? lrows * 128L : 0L;
                rp[i] += more ? rrows * 128L : 0L;
            }
        };
        const int put = row * 128 + ((chunk ^ (row >> 1 & 7)) << 4);
        auto stage = [&](int at, const Lines& l) {
            char* s = smem + at * (2 * TS * 128) + put;
#pragma unroll
            for (int i = 0; i < PASS; ++i) {
                *reinterpret_cast<u32x4*>(s + i * 32 * 128) = l.l[i];
                *reinterpret_cast<u32x4*>(s + TS * 128 + i * 32 * 128) = l.r[i];
            }
        };
        const int half = lane >> 5, sw = lane >> 1 & 7;
        const char* sL = smem + ((wave >> 1) * (TS / 2) + (lane & 31)) * 128;
        const char* sR = smem + TS * 128 + ((wave & 1) * (TS / 2) + (lane & 31)) * 128;
        auto read = [&](Frags& f, int at, int k) {
            const int ch = at * (2 * TS * 128) + (((k * 2 + half) ^ sw) << 4), cl = at * (2 * TS * 128) + (((4 + k * 2 + half) ^ sw) << 4);
#pragma unroll
            for (int i = 0; i < S; ++i) {
                f.lh[i] = *reinterpret_cast<const f16x8*>(sL + i * 32 * 128 + ch);
                f.rl[i] = *reinterpret_cast<const f16x8*>(sR + i * 32 * 128 + cl);
            }
#pragma unroll
            for (int i = 0; i < S; ++i) {
                f.ll[i] = *reinterpret_cast<const f16x8*>(sL + i * 32 * 128 + cl);
                f.rh[i] = *reinterpret_cast<const f16x8*>(sR + i * 32 * 128 + ch);
            }
        };
        Frags f0, f1;
        fetch(set[0]);
        fetch(set[1]);
        stage(0, set[0]);
        fetch(set[0]);
        __syncthreads();
        read(f0, 0, 0);
        for (int k = 0; k < lines; k += 2) {
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                read(f1, d, 1);
                multiply<0, S * S>(f0);
                stage(d ^ 1, set[d ^ 1]);
                multiply<S * S, 3 * S * S>(f0);
                fetch(set[d ^ 1]);
                multiply<0, S * S>(f1);
                __syncthreads();                          // this line's fragments are out, the next line is in
                read(f0, d ^ 1, 0);
                multiply<S * S, 3 * S * S>(f1);
            }
        }
    }

    // of element e of subtile (i, k): row and column inside the tile
    __device__ static inline int row_of(int i, int e) {
        return (threadIdx.x >> 7) * (TS / 2) + i * 32 + 8 * (e >> 2) + 4 * ((threadIdx.x >> 5) & 1) + (e & 3);
    }
    __device__ static inline int col_of(int k) { return ((threadIdx.x >> 6) & 1) * (TS / 2) + k * 32 + (threadIdx.x & 31); }
};

// the line of a row that holds column `col`, a multiple of 32
__device__ inline gbytes ns_line(gbytes base, int rows, int row, int col) { return base + ((long)(col >> 5) * rows + row) * 128; }

// A 32x32 subtile (already scaled) to plane pairs: along its rows at `dst` (through a per-wave LDS patch) and, transposed,
// at `dst_t` straight from the registers, where a lane holds four consecutive rows of one column.  Either may be NULL.
__device__ inline void ns_store(const f32x16& v, unsigned* patch, gbytes dst, gbytes dst_t) {
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    unsigned u[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) u[e] = ns_split(v[e]);
    if (dst_t) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            gbytes p = dst_t + col * 128 + (8 * q + 4 * half) * 2;
            const unsigned* w = u + 4 * q;
            *(DVAE_GLOBAL u32x2*)(p) = u32x2{(w[0] & 0xffffu) | (w[1] << 16), (w[2] & 0xffffu) | (w[3] << 16)};
            *(DVAE_GLOBAL u32x2*)(p + 64) = u32x2{(w[0] >> 16) | (w[1] & 0xffff0000u), (w[2] >> 16) | (w[3] & 0xffff0000u)};
        }
    }
    if (dst) {
        constexpr int ST = 36;
#pragma unroll
        for (int e = 0; e < 16; ++e) patch[(8 * (e >> 2) + 4 * half + (e & 3)) * ST + col] = u[e];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int r = (lane >> 2) + 16 * k, c = (lane & 3) * 8;
            const u32x4 a = *reinterpret_cast<const u32x4*>(patch + r * ST + c), b = *reinterpret_cast<const u32x4*>(patch + r * ST + c + 4);
            gbytes p = dst + r * 128 + c * 2;
            *(DVAE_GLOBAL u32x4*)(p) = u32x4{(a[0] & 0xffffu) | (a[1] << 16), (a[2] & 0xffffu) | (a[3] << 16),
                                                 (b[0] & 0xffffu) | (b[1] << 16), (b[2] & 0xffffu) | (b[3] << 16)};
            *(DVAE_GLOBAL u32x4*)(p + 64) = u32x4{(a[0] >> 16) | (a[1] & 0xffff0000u), (a[2] >> 16) | (a[3] & 0xffff0000u),
                                                      (b[0] >> 16) | (b[1] & 0xffff0000u), (b[2] >> 16) | (b[3] & 0xffff0000u)};
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// tile t of a lower triangle, row by row
__device__ inline void ns_triangle(int t, int& i, int& k) {
    i = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    k = t - i * (i + 1) / 2;
}

// The symmetric products store the tiles at and below the diagonal and their mirror images.  Tiles on the diagonal are
// stored once: their two halves agree to rounding only, and two writers of one place would leave either's.
template <int TS>
__device__ inline void ns_store_symmetric(NsTile<TS>& c, char* smem, gbytes dst, int P, int ti, int tk) {
    constexpr int S = NsTile<TS>::S;
    const int wave = threadIdx.x >> 6, wr = (wave >> 1) * (TS / 2), wc = (wave & 1) * (TS / 2);
    unsigned* patch = reinterpret_cast<unsigned*>(smem) + wave * (32 * 36);
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int row = ti * TS + wr + i * 32, col = tk * TS + wc + k * 32;
            if (row >= P || col >= P) continue;
            ns_store(c.acc[i][k], patch, ns_line(dst, P, row, col), ti != tk ? ns_line(dst, P, col, row) : gbytes(nullptr));
        }
}

// A = X X^T, whole or, where the tiles alone would leave most of the chip idle, in `kc`-line pieces of the contraction that
// leave fp32 partial tiles for ns_gram_sum_kernel.
template <int TS, bool PIECES>
__global__ __launch_bounds__(256, 2) void ns_gram_kernel(NsArgs g) {
    __shared__ __align__(16) char smem[NsTile<TS>::BYTES];
    constexpr int S = NsTile<TS>::S;
    int t;
    const int wg = ns_swizzle(blockIdx.x, g.total);
    const NsJob j = g.jobs[ns_find(g, NS_GRAM, wg, t)];
    const NsPlanes w(g, j);
    const int lines = w.Q / 32, pieces = PIECES ? (lines + g.kc - 1) / g.kc : 1;
    int ti, tk;
    ns_triangle(t / pieces, ti, tk);
    const int line0 = PIECES ? t % pieces * g.kc : 0;
    NsTile<TS> c;
    c.zero();
    c.run(w.x, w.P, ti * TS, w.x, w.P, tk * TS, line0, PIECES ? min(g.kc, lines - line0) : lines, smem);
    if (PIECES) {
        float* out = g.part + (long)wg * (TS * TS) + threadIdx.x;
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int k = 0; k < S; ++k)
#pragma unroll
                for (int e = 0; e < 16; ++e) out[((i * S + k) * 16 + e) * 256] = c.acc[i][k][e];
        return;
    }
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) c.acc[i][k][e] *= NS_SA / (NS_SX * NS_SX);
    ns_store_symmetric<TS>(c, smem, w.a, w.P, ti, tk);
}

template <int TS>
__global__ __launch_bounds__(256) void ns_gram_sum_kernel(NsArgs g) {
    __shared__ __align__(16) char smem[4 * 32 * 36 * 4];
    constexpr int S = NsTile<TS>::S;
    int t;
    const int jn = ns_find(g, NS_SYM, blockIdx.x, t);
    const NsJob j = g.jobs[jn];
    const NsPlanes w(g, j);
    const int pieces = (w.Q / 32 + g.kc - 1) / g.kc;
    const float* in = g.part + ((long)g.first[NS_GRAM * g.jp + jn] + (long)t * pieces) * (TS * TS) + threadIdx.x;
    NsTile<TS> c;
    c.zero();
    static_assert(S == 1, "pieces are cut for tiles of 64");
    for (int s = 0; s < pieces; s += 4, in += 4 * TS * TS) {          // four pieces' loads in flight
        float v[4][16];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) v[u][e] = s + u < pieces ? in[u * TS * TS + e * 256] : 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) c.acc[0][0][e] += v[u][e];
    }
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) c.acc[i][k][e] *= NS_SA / (NS_SX * NS_SX);
    int ti, tk;
    ns_triangle(t, ti, tk);
    ns_store_symmetric<TS>(c, smem, w.a, w.P, ti, tk);
}

// B = a I + b A + c A^2
template <int TS>
__global__ __launch_bounds__(256, 2) void ns_square_kernel(NsArgs g) {
    __shared__ __align__(16) char smem[NsTile<TS>::BYTES];
    constexpr int S = NsTile<TS>::S;
    int t, ti, tk;
    const NsJob j = g.jobs[ns_find(g, NS_SYM, ns_swizzle(blockIdx.x, g.total), t)];
    const NsPlanes w(g, j);
    ns_triangle(t, ti, tk);
    NsTile<TS> c;
    c.zero();
    c.run(w.a, w.P, ti * TS, w.a, w.P, tk * TS, 0, w.P / 32, smem);
    const float s2 = g.c * (NS_SB / (NS_SA * NS_SA)), s1 = g.b * (NS_SB / NS_SA), s0 = g.a * NS_SB;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int col = tk * TS + NsTile<TS>::col_of(k), row = ti * TS + NsTile<TS>::row_of(i, 0);
            if (col >= w.P || row >= w.P) continue;
            // a lane's elements of A lie along a column: read as a row, A being symmetric
            cgbytes p = ns_line(w.a, w.P, col, row & ~31) + (row & 31) * 2;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const u32x2 h = *(const DVAE_GLOBAL u32x2*)(p + 16 * q), l = *(const DVAE_GLOBAL u32x2*)(p + 16 * q + 64);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f16x2 hv = __builtin_bit_cast(f16x2, (unsigned)h[e >> 1]), lv = __builtin_bit_cast(f16x2, (unsigned)l[e >> 1]);
                    const float av = (float)hv[e & 1] + (float)lv[e & 1];
                    float r = s2 * c.acc[i][k][4 * q + e] + s1 * av;
                    if (row + 8 * q + e == col) r += s0;
                    c.acc[i][k][4 * q + e] = r;
                }
            }
        }
    ns_store_symmetric<TS>(c, smem, w.b, w.P, ti, tk);
}

// X <- B X, left in both orientations
template <int TS>
__global__ __launch_bounds__(256, 2) void ns_apply_kernel(NsArgs g) {
    __shared__ __align__(16) char smem[NsTile<TS>::BYTES];
    constexpr int S = NsTile<TS>::S;
    int t;
    const NsJob j = g.jobs[ns_find(g, NS_APPLY, ns_swizzle(blockIdx.x, g.total), t)];
    const NsPlanes w(g, j);
    const int ni = (w.P + TS - 1) / TS, ti = t % ni, tk = t / ni;
    NsTile<TS> c;
    c.zero();
    c.run(w.b, w.P, ti * TS, w.xt(g.turn), w.Q, tk * TS, 0, w.P / 32, smem);
    const int wave = threadIdx.x >> 6, wr = (wave >> 1) * (TS / 2), wc = (wave & 1) * (TS / 2);
    unsigned* patch = reinterpret_cast<unsigned*>(smem) + wave * (32 * 36);
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int row = ti * TS + wr + i * 32, col = tk * TS + wc + k * 32;
            if (row >= w.P || col >= w.Q) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) c.acc[i][k][e] *= 1.f / NS_SB;
            ns_store(c.acc[i][k], patch, ns_line(w.x, w.P, row, col), ns_line(w.xt(g.turn ^ 1), w.Q, col, row));
        }
}

// The last product: its tile goes to the caller's matrix, or steps the parameter.  A tall matrix's tile is computed
// transposed (the operands trade places), so that lanes run along the caller's rows either way.
template <int TS, typename T, bool MUON>
__global__ __launch_bounds__(256, 2) void ns_last_kernel(NsArgs g) {
    __shared__ __align__(16) char smem[NsTile<TS>::BYTES];
    constexpr int S = NsTile<TS>::S;
    int t;
    const NsJob j = g.jobs[ns_find(g, NS_APPLY, ns_swizzle(blockIdx.x, g.total), t)];
    const NsPlanes w(g, j);
    const bool tall = j.m > j.n;
    const int ni = (w.P + TS - 1) / TS, tp = t % ni, tq = t / ni;
    NsTile<TS> c;
    c.zero();
    const cgbytes L = tall ? w.xt(g.turn) : w.b, R = tall ? w.b : w.xt(g.turn);
    const int lrows = tall ? w.Q : w.P, rrows = tall ? w.P : w.Q, ti = tall ? tq : tp, tk = tall ? tp : tq;
    c.run(L, lrows, ti * TS, R, rrows, tk * TS, 0, w.P / 32, smem);
    const auto out = as_global<T>(j.out);
    const float step = MUON ? g.lr * j.scale : 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int col = tk * TS + NsTile<TS>::col_of(k);
            if (col >= j.n) continue;
            float p[16];
            if (MUON) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int row = ti * TS + NsTile<TS>::row_of(i, e);
                    p[e] = row < j.m ? (float)out[row * j.os + col] : 0.f;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = ti * TS + NsTile<TS>::row_of(i, e);
                const float v = c.acc[i][k][e] * (1.f / (NS_SB * NS_SX));
                if (row < j.m) out[row * j.os + col] = (T)(MUON ? p[e] * g.decay - step * v : v);
            }
        }
}

}  // namespace dvae
