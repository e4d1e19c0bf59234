// Orthogonalising matrices by the quintic Newton-Schulz iteration, and the Muon update around it.
//
//   X_0 = X / (|X|_F + eps)     A = X X^T, B = a I + b A + c A^2, X <- B X      (`steps` times; p = min(m, n) rows)
//
// (K. Jordan and others, "Muon: an optimizer for hidden layers in neural networks", 2024, where the usual coefficients are from.)
// (a I folded into B saves the third product an operand.)  A matrix with more rows than columns is iterated as its
// transpose.  A list of matrices of any shapes runs as one batch: every phase is one launch over the tiles of all of them.
//
// Number format.  The iteration multiplies small singular values by up to a^steps (485 for the usual coefficients), so
// products of bf16 operands are off by 1 to 50 percent; fp32 operands would use the fp32 matrix rate, a sixteenth of
// the 16-bit one.  Here an operand is the sum of two fp16 pieces, x = h + l / 2^11 (22 bits), and a product is three MFMAs,
// hh + (hl + lh) / 2^11, summed in fp32: the errors of an fp32 product at 3/16 of its time.  fp16's range is met by scales: with
// the coefficients' bounds checked on the host, |X| <= 2, |A| <= 4 and |B| <= 7, held as 2^14 X, 2^13 A and 2^13 B.  l's own
// factor keeps it as far from fp16's lower end as h: without it elements below 6e-5 of the largest possible one would lose
// digits (rows of 1e-6 of the others' size were off by 1.5e-4).  What is left is an absolute error of 2^-50 an element, against
// matrices of norm up to 2: rows and columns of 1e-8 of the others' size are off by 1e-5, of 1e-10 by 1e-3.  A matrix that is small as
// a whole, its norm far below eps, has a larger power of two than 2^14, see ns_shift.
//
// Layout.  An R x K operand is made of lines of 32 columns: a row's 32 h's, then its 32 l's, 128 bytes in eight chunks of 16.  Equal
// chunks of the R rows follow each other, then the next chunk, then the next line: whatever a wave loads or stores, staged
// tiles, fragments or either orientation of a result, is runs of 16 rows and more.  R and K are padded to 64 with zeros, which
// the products keep zero.  X is kept with its transpose (two copies, taken in turn), so that every product reads both operands
// along its contraction.
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

constexpr float NS_SX = 16384.f, NS_SA = 8192.f, NS_SB = 8192.f, NS_SL = 2048.f;

// X_k is held as 2^(14 + shift) X_k: |X_0| is below 2^lead, lead the exponent of |X| / (|X| + eps), and a step multiplies every
// singular value by at most 2^rate, rate >= 0 by the host's bound on |a + b s^2 + c s^4|.  Past 96 nothing of fp32's range is left
// to be gained.
__device__ inline int ns_shift(int lead, float rate, int step) {
    const int v = -(lead + (int)ceilf(rate * (float)step));
    return v < 0 ? 0 : v > 96 ? 96 : v;
}
__device__ inline int ns_lead(double norm, double eps) {
    const double part = norm / (norm + eps);             // of a zero matrix without an eps, and of infinite ones, no number
    int e = 0;
    if (part > 0.0) (void)frexp(part, &e);
    return e;
}
// 2^14 / (|X| + eps) from |X|^2; a zero matrix stays one, whatever eps is
__device__ inline double ns_inverse(double square, double eps) { return square == 0.0 ? 0.0 : (double)NS_SX / (sqrt(square) + eps); }

enum { NS_NORM, NS_SPLIT, NS_GRAM, NS_GRAM_TILES, NS_SQUARE, NS_APPLY, NS_PHASES };

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
    int kc;                   // lines of 32 columns a workgroup of the Gram phase sums
    float scale;              // Muon: factor of the step
};

struct NsArgs {
    const int* first;         // [NS_PHASES][jp]: first workgroup of each job, INT_MAX beyond the last
    const NsJob* jobs;
    double* norm;             // partial sums of squares
    float* part;              // partial tiles of the symmetric products
    char* ws;
    int njobs, jp;
    int total;                // workgroups of this launch
    int turn;                 // which transposed copy is read
    int step;
    float rate;               // see ns_shift
    float a, b, c;
    double eps;
    NsJob one;                // the job, where there is only one: no table then
    float mu, nu, lr, decay;  // momentum, 1 - momentum, step, 1 - step * weight decay: each rounded once from 64 bits
    int nesterov;
};

__host__ __device__ inline int ns_pad(int v) { return (v + 63) & ~63; }
__host__ __device__ inline long ns_job_bytes(int m, int n) {
    const long p = ns_pad(m < n ? m : n), q = ns_pad(m < n ? n : m);
    return 4 * (3 * p * q + 2 * p * p + p + 64);         // A's diagonal and the matrix's lead last: p is a multiple of 64
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
    if (g.njobs == 1) {
        local = wg;
        return 0;
    }
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

__device__ inline NsJob ns_job_of(const NsArgs& g, int job) { return g.njobs == 1 ? g.one : g.jobs[job]; }

// Consecutive workgroups run on different XCDs; neighbouring tiles share operands and go to the same one's L2.
__device__ inline int ns_swizzle(int id, int total) {
    const int per = total >> 3, whole = per << 3;
    return id < whole ? (id & 7) * per + (id >> 3) : id;
}

// A row's part of the line that holds column `col`: its first chunk.  Chunks lie 16 * rows bytes apart, h's in 0..3, l's in 4..7.
__device__ inline gbytes ns_line(gbytes base, long rows, int row, int col) { return base + ((col >> 5) * rows * 8 + row) * 16; }

struct NsPlanes {
    int P, Q;
    gbytes x, xt0, xt1, a, b;
    DVAE_GLOBAL float* diag;
    DVAE_GLOBAL int* lead;
    __device__ NsPlanes(const NsArgs& g, const NsJob& j) {
        P = ns_pad(min(j.m, j.n));
        Q = ns_pad(max(j.m, j.n));
        const long pq = 4L * P * Q;
        x = as_global<char>(g.ws) + j.off;
        xt0 = x + pq;
        xt1 = x + 2 * pq;
        a = x + 3 * pq;
        b = a + 4L * P * P;
        diag = (DVAE_GLOBAL float*)(b + 4L * P * P);
        lead = (DVAE_GLOBAL int*)(diag + P);
    }
    __device__ int shift(const NsArgs& g, int step) const { return ns_shift(*lead, g.rate, step); }
    __device__ gbytes xt(int which) const { return which ? xt1 : xt0; }
};

// A value that is about to be split is rounded to fp32 for good.  Left to itself the compiler converts a product to fp16 now
// from its rounded value and now, fused, from its exact one; at a tie the h that is stored and the h that l is the rest of are
// then two neighbours, and the pair is off by 2^-11.  (What l is made from is exact: h's remainder times a power of two.)
__device__ inline float ns_rounded(float v) {
    asm("" : "+v"(v));
    return v;
}
__device__ inline unsigned ns_split(float v) {           // low half: h, high half: l
    v = ns_rounded(v);
    const f16 h = (f16)v;
    const f16 l = (f16)((v - (float)h) * NS_SL);
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
    const NsJob j = ns_job_of(g, ns_find(g, NS_NORM, blockIdx.x, chunk));
    const long n = (long)j.m * j.n;
    const auto x = as_global<const T>(j.x);
    const auto mom = as_global<float>(j.mom), par = as_global<float>(j.out);
    double s = 0.0;
    for (long base = (long)chunk * NS_CHUNK; base < n; base += (long)j.nchunk * NS_CHUNK) {
        // Loads are of elements that exist, whatever becomes of their values, and whole trips store without a condition: a condition
        // is a branch, and sixteen branches are sixteen latencies.
        const bool whole = base + NS_CHUNK <= n;
        float v[16], m[16], p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const long e = base + i * 256 + threadIdx.x, to = e < n ? e : 0;
            long at = to;
            if (!MUON && j.xs != j.n) at = (unsigned)to / (unsigned)j.n * j.xs + (unsigned)to % (unsigned)j.n;
            v[i] = (float)x[at];
            if (MUON) m[i] = mom[to];
            if (MUON && j.vec) p[i] = par[to];
        }
        if (MUON) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                m[i] = ns_rounded(ns_momentum(g, v[i], m[i]));
                v[i] = ns_update(g, v[i], m[i]);
                if (j.vec) p[i] = ns_rounded(p[i] * g.decay - g.lr * v[i]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const long e = base + i * 256 + threadIdx.x;
                if (whole || e < n) {
                    mom[e] = m[i];
                    if (j.vec) par[e] = p[i];
                }
            }
        }
        if (!whole)
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = base + i * 256 + threadIdx.x < n ? v[i] : 0.f;
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
    const NsJob j = ns_job_of(g, ns_find(g, NS_SPLIT, blockIdx.x, t));
    double s = 0.0;
    for (int i = threadIdx.x; i < j.nchunk; i += 256) s += g.norm[j.part + i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = (red[0] + red[1]) + (red[2] + red[3]);
    const NsPlanes w(g, j);
    const int lead = ns_lead(sqrt(s), g.eps);
    const double inv = ldexp(ns_inverse(s, g.eps), ns_shift(lead, g.rate, 0));
    if (t == 0 && threadIdx.x == 0) *w.lead = lead;
    const bool tall = j.m > j.n;
    const int ncol = ns_pad(j.n) >> 6;
    const int r0 = t / ncol * 64, c0 = t % ncol * 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = c0 + lane;
    float v[16], mom[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {                        // past the edges the last elements, which count as zero
        const long e = (long)min(r0 + i * 4 + wave, j.m - 1) * j.xs + min(c, j.n - 1);
        v[i] = (float)as_global<const T>(j.x)[e];
        if (MUON) mom[i] = as_global<float>(j.mom)[e];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (MUON) v[i] = ns_update(g, v[i], mom[i]);
        v[i] = (float)((double)v[i] * inv);
        tile[i * 4 + wave][lane] = ns_split(r0 + i * 4 + wave < j.m && c < j.n ? v[i] : 0.f);
    }
    __syncthreads();
    // a wave writes 16 columns of 64 rows: first in the source's orientation, then in the other
#pragma unroll
    for (int flip = 0; flip < 2; ++flip) {
        gbytes dst = flip ? (tall ? w.x : w.xt0) : (tall ? w.xt0 : w.x);
        const long rows = ns_pad(flip ? j.n : j.m);
        const int r = lane, c = wave * 16;
        unsigned h[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned u0 = flip ? tile[c + 2 * i][r] : tile[r][c + 2 * i];
            const unsigned u1 = flip ? tile[c + 2 * i + 1][r] : tile[r][c + 2 * i + 1];
            h[i] = (u0 & 0xffffu) | (u1 << 16);
            l[i] = (u0 >> 16) | (u1 & 0xffff0000u);
        }
        const int row = (flip ? c0 : r0) + r, col = (flip ? r0 : c0) + c;
        const gbytes p = ns_line(dst, rows, row, col) + (col & 31) / 8 * rows * 16;
        *(DVAE_GLOBAL u32x4*)p = u32x4{h[0], h[1], h[2], h[3]};
        *(DVAE_GLOBAL u32x4*)(p + rows * 16) = u32x4{h[4], h[5], h[6], h[7]};
        *(DVAE_GLOBAL u32x4*)(p + rows * 64) = u32x4{l[0], l[1], l[2], l[3]};
        *(DVAE_GLOBAL u32x4*)(p + rows * 80) = u32x4{l[4], l[5], l[6], l[7]};
    }
}

// what lanes of a wave wrote to LDS is there for its other lanes
__device__ inline void ns_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- the products ----------------------------------------------------------------------------------------------------
// C[i][k] = sum over c of L[i][c] R[k][c] for a TS x TS tile: four waves, a quarter tile each, 32x32x16 MFMAs; hl + lh has sums of
// its own.  Two LDS stages of one line (32 columns) per row, one barrier a line: while one half of a line is multiplied, the
// fragments of the other half are on their way from LDS, and the next lines are on their way from memory, two in two sets of
// registers, in tiles of 128, whose registers the sums take, one.
// A line's eight 16-byte chunks are stored at chunk ^ (row / 2 & 7): of a fragment's rows any sixteen that are read at a time
// meet the 64 banks once each.
//
// Two groups (G) of four waves share the contraction of one tile, each with stages of its own, and add up at the end (join): with
// no more tiles than CUs a CU has two waves a SIMD to cover each other's waits all the same.
template <int TS, int G = 1>
struct NsTile {
    static_assert(G <= 2, "one group or two");
    static constexpr int S = TS / 64;                    // subtiles of a wave each way
    static constexpr int PASS = TS / 32;                 // passes of 256 threads over a stage of one operand
    static constexpr int STAGES = 2 * 2 * TS * 128;      // bytes of a group
    static constexpr int BYTES = G * STAGES;
    static constexpr int SETS = S == 1 ? 2 : 1;          // lines on their way
    f32x16 acc[S][S], low[S][S];
    int from = 0, to = S;                                // rows of subtiles that are this group's after join

    struct Lines { u32x4 l[PASS], r[PASS]; };
    struct Frags { f16x8 lh[S], ll[S], rh[S], rl[S]; };

    __device__ inline void zero() {
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int k = 0; k < S; ++k)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][k][e] = low[i][k][e] = 0.f;
    }

    // MFMAs FROM to TO of the 3 S^2 of half a line
    template <int FROM, int TO>
    __device__ inline void multiply(const Frags& f) {
#pragma unroll
        for (int m = FROM; m < TO; ++m) {
            const int w = m / (S * S), i = m / S % S, n = m % S;
            f32x16& c = w == 2 ? acc[i][n] : low[i][n];
            c = __builtin_amdgcn_mfma_f32_32x32x16_f16(w == 1 ? f.ll[i] : f.lh[i], w == 0 ? f.rl[n] : f.rh[n], c, 0, 0, 0);
        }
    }
    // `lines` is even.  Operands have multiples of 64 rows: where a tile of 128 has only 64, it reads those twice, and what comes of the
    // second half is not stored.
    // SAME: both operands are the same rows, staged once.
    template <bool SAME = false>
    __device__ inline void run(cgbytes L, int lrows, int l0, cgbytes R, int rrows, int r0, int line0, int lines, char* smem) {
        const int tid = threadIdx.x & 255, row = tid & 31, chunk = tid >> 5, group = threadIdx.x >> 8;
        const int lane = tid & 63, wave = tid >> 6;
        int idle = 0;                                     // lines that the other group has more
        if (G > 1) {
            const int most = (lines / 2 + 1) & ~1;        // an even number for each
            if (group) {
                line0 += most;
                lines -= most;
                idle = most - lines;
                smem += STAGES;
            } else {
                lines = most;
            }
            if (lines == 0) {
                for (int k = 0; k <= idle; ++k) __syncthreads();
                return;
            }
        }
        cgbytes lp = L + (((long)line0 * 8 + chunk) * lrows + l0 + row) * 16, rp = R + (((long)line0 * 8 + chunk) * rrows + r0 + row) * 16;
        const int lup = l0 + TS <= lrows ? 64 * 16 : 0, rup = r0 + TS <= rrows ? 64 * 16 : 0;
        Lines set[SETS];
        int ahead = lines;
        auto fetch = [&](Lines& s) {                      // the next line; past the last one, that one again
#pragma unroll
            for (int i = 0; i < PASS; ++i) {
                s.l[i] = *(const DVAE_GLOBAL u32x4*)(lp + (i >> 1) * lup + (i & 1) * 32 * 16);
                if (!SAME) s.r[i] = *(const DVAE_GLOBAL u32x4*)(rp + (i >> 1) * rup + (i & 1) * 32 * 16);
            }
            const bool more = --ahead > 0;
            lp += more ? lrows * 128L : 0L;
            rp += more ? rrows * 128L : 0L;
        };
        const int put = row * 128 + ((chunk ^ (row >> 1 & 7)) << 4);
        auto stage = [&](int at, const Lines& l) {
            char* s = smem + at * (2 * TS * 128) + put;
#pragma unroll
            for (int i = 0; i < PASS; ++i) {
                *reinterpret_cast<u32x4*>(s + i * 32 * 128) = l.l[i];
                if (!SAME) *reinterpret_cast<u32x4*>(s + TS * 128 + i * 32 * 128) = l.r[i];
            }
        };
        const int half = lane >> 5, sw = lane >> 1 & 7;
        const char* sL = smem + ((wave >> 1) * (TS / 2) + (lane & 31)) * 128;
        const char* sR = smem + (SAME ? 0 : TS * 128) + ((wave & 1) * (TS / 2) + (lane & 31)) * 128;
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
        if (SETS == 2) fetch(set[SETS - 1]);
        stage(0, set[0]);
        fetch(set[0]);
        __syncthreads();
        read(f0, 0, 0);
        for (int k = 0; k < lines; k += 2) {
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                read(f1, d, 1);
                multiply<0, S * S>(f0);
                stage(d ^ 1, set[(d ^ 1) % SETS]);
                multiply<S * S, 3 * S * S>(f0);
                fetch(set[(d ^ 1) % SETS]);
                multiply<0, S * S>(f1);
                __syncthreads();                          // this line's fragments are out, the next line is in
                read(f0, d ^ 1, 0);
                multiply<S * S, 3 * S * S>(f1);
            }
        }
        for (int k = 0; k < idle; ++k) __syncthreads();
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int k = 0; k < S; ++k)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][k][e] += low[i][k][e] * (1.f / NS_SL);
    }

    // Adds the groups up: each keeps a row of subtiles.
    __device__ inline void join(char* smem) {
        static_assert(G == 1 || (G == 2 && S == 2), "two groups, two rows of subtiles");
        if (G == 1) return;
        const int tid = threadIdx.x & 255, group = threadIdx.x >> 8;
        __syncthreads();                                  // the stages are read
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if (i == group) continue;
#pragma unroll
            for (int k = 0; k < S; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f32x4*>(smem + group * STAGES + ((k * 4 + q) * 256 + tid) * 16) =
                        f32x4{acc[i][k][4 * q], acc[i][k][4 * q + 1], acc[i][k][4 * q + 2], acc[i][k][4 * q + 3]};
        }
        __syncthreads();
        from = group;
        to = group + 1;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if (i != group) continue;
#pragma unroll
            for (int k = 0; k < S; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 v = *reinterpret_cast<const f32x4*>(smem + (group ^ 1) * STAGES + ((k * 4 + q) * 256 + tid) * 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][k][4 * q + e] += v[e];
                }
        }
        __syncthreads();                                  // before the patches of the stores
    }

    // of element e of subtile (i, k): row and column inside the tile
    __device__ static inline int row_of(int i, int e) {
        return (threadIdx.x >> 7 & 1) * (TS / 2) + i * 32 + 8 * (e >> 2) + 4 * ((threadIdx.x >> 5) & 1) + (e & 3);
    }
    __device__ static inline int col_of(int k) { return ((threadIdx.x >> 6) & 1) * (TS / 2) + k * 32 + (threadIdx.x & 31); }
};

// A 32x32 subtile (already scaled) to plane pairs: along its rows at `dst`, of an operand of `rows` rows (through a per-wave LDS
// patch), and, transposed, at `dst_t` straight from the registers, where a lane holds four consecutive rows of one column,
// half a chunk.  Either may be NULL.
__device__ inline void ns_store(const f32x16& v, unsigned* patch, gbytes dst, long rows, gbytes dst_t, long rows_t) {
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    unsigned u[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) u[e] = ns_split(v[e]);
    if (dst_t) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const gbytes p = dst_t + (q * rows_t + col) * 16 + half * 8;
            const unsigned* w = u + 4 * q;
            *(DVAE_GLOBAL u32x2*)p = u32x2{(w[0] & 0xffffu) | (w[1] << 16), (w[2] & 0xffffu) | (w[3] << 16)};
            *(DVAE_GLOBAL u32x2*)(p + rows_t * 64) = u32x2{(w[0] >> 16) | (w[1] & 0xffff0000u), (w[2] >> 16) | (w[3] & 0xffff0000u)};
        }
    }
    if (dst) {
        constexpr int ST = 36;
#pragma unroll
        for (int e = 0; e < 16; ++e) patch[(8 * (e >> 2) + 4 * half + (e & 3)) * ST + col] = u[e];
        ns_wave_sync();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int r = (lane & 15) + 16 * k, c = lane >> 4;
            const u32x4 a = *reinterpret_cast<const u32x4*>(patch + r * ST + c * 8), b = *reinterpret_cast<const u32x4*>(patch + r * ST + c * 8 + 4);
            const gbytes p = dst + (c * rows + r) * 16;
            *(DVAE_GLOBAL u32x4*)p = u32x4{(a[0] & 0xffffu) | (a[1] << 16), (a[2] & 0xffffu) | (a[3] << 16),
                                           (b[0] & 0xffffu) | (b[1] << 16), (b[2] & 0xffffu) | (b[3] << 16)};
            *(DVAE_GLOBAL u32x4*)(p + rows * 64) = u32x4{(a[0] >> 16) | (a[1] & 0xffff0000u), (a[2] >> 16) | (a[3] & 0xffff0000u),
                                                         (b[0] >> 16) | (b[1] & 0xffff0000u), (b[2] >> 16) | (b[3] & 0xffff0000u)};
        }
        ns_wave_sync();
    }
}

// tile t of a lower triangle, row by row
__device__ inline void ns_triangle(int t, int& i, int& k) {
    i = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    k = t - i * (i + 1) / 2;
}

// tile t of `side` rows of tiles: those below the diagonal row by row, then the diagonal
__device__ inline void ns_diagonal_last(int t, int side, int& i, int& k) {
    const int below = side * (side - 1) / 2;
    if (t >= below) {
        i = k = t - below;
    } else {
        ns_triangle(t, i, k);
        ++i;
    }
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
            ns_store(c.acc[i][k], patch, ns_line(dst, P, row, col), P, ti != tk ? ns_line(dst, P, col, row) : gbytes(nullptr), P);
        }
}

// An element of B in row i, column k.  A is kept as its diagonal d, in fp32, and the rest R, in pieces: the matrix cores align the
// products of a group to the largest and cut off what lies below its last bit, so that in A^2 the squares beside a dominant one of
// the diagonal (X near orthogonal) lost some bits, always to one side.  In A^2 = R^2 + d_i R + R d_k + d^2 nothing is dominant:
// 64 x 576 came from 1.7e-6 to 6.1e-7 by it (fp32 products: 1.4e-6), for 0.5 to 4 % of the time.  `square` is R^2 (scaled), r the
// element of R.
template <typename Args>
__device__ inline float ns_polynomial(const Args& g, float square, float r, float di, float dk, bool diagonal) {
    const float t = diagonal ? dk : r, u = diagonal ? dk : di + dk;
    const float v = g.c * (NS_SB / (NS_SA * NS_SA)) * (square + u * t) + g.b * (NS_SB / NS_SA) * t;
    return diagonal ? v + g.a * NS_SB : v;
}
// element e of four pairs
__device__ inline float ns_whole(u32x2 h, u32x2 l, int e) {
    const f16x2 hv = __builtin_bit_cast(f16x2, (unsigned)h[e >> 1]), lv = __builtin_bit_cast(f16x2, (unsigned)l[e >> 1]);
    return __builtin_fmaf((float)lv[e & 1], 1.f / NS_SL, (float)hv[e & 1]);
}
// What turns sums of products of X as it is held into A as it is held; 0 for an X so small that A is nothing beside a I.
__device__ inline float ns_gram_scale(const NsArgs& g, const NsPlanes& w) { return ldexpf(NS_SA / (NS_SX * NS_SX), -2 * w.shift(g, g.step)); }
// An element of A: R's, or, on the diagonal, none there and d's.
__device__ inline float ns_off_diagonal(const NsPlanes& w, float v, int row, int col) {
    if (row != col) return v;
    w.diag[col] = v;
    return 0.f;
}

// What a symmetric product's subtile becomes: A = X X^T, or B = a I + b A + c A^2.  A lane's elements lie in column `col`, from
// `row` on; those of A that B needs are read along row `col`, A being symmetric.
template <bool SQUARE>
__device__ inline void ns_symmetric_value(const NsArgs& g, const NsPlanes& w, f32x16& v, int row, int col) {
    if (!SQUARE) {
        const float scale = ns_gram_scale(g, w);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= scale;
        if ((row ^ col) < 32) {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = ns_off_diagonal(w, v[e], row + 8 * (e >> 2) + (e & 3), col);
        }
        return;
    }
    const long rows = w.P;
    const cgbytes p = ns_line(w.a, rows, col, row & ~31) + (row & 4) * 2;
    const float dk = w.diag[col];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const u32x2 h = *(const DVAE_GLOBAL u32x2*)(p + q * rows * 16), l = *(const DVAE_GLOBAL u32x2*)(p + (4 + q) * rows * 16);
        const f32x4 di = *(const DVAE_GLOBAL f32x4*)(w.diag + row + 8 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = ns_polynomial(g, v[4 * q + e], ns_whole(h, l, e), di[e], dk, row + 8 * q + e == col);
    }
}

// One matrix in whole tiles: those on the diagonal, cheaper by half their loads, are spread over the XCDs by themselves and come last,
// so that they are what a CU with a tile more than the others has more (2048 x 2048, 528 tiles on 256 CUs: 775 -> 755 us; in line
// with the others, all on the last XCD, 780).
__device__ inline int ns_spread(const NsArgs& g, int ts, bool pieces) {
    return pieces || g.njobs != 1 ? g.total : g.total - (ns_pad(min(g.one.m, g.one.n)) + ts - 1) / ts;
}

// The symmetric products, tiles at and below the diagonal: whole or (Gram, where the tiles alone would leave much of the chip
// idle) in pieces of the contraction, a job's kc lines each, that leave fp32 partial tiles for ns_gram_sum_kernel.  Neighbouring
// workgroups take different tiles of the same lines: an XCD reads a part of X once.
template <int TS, bool SQUARE, bool PIECES>
__global__ __launch_bounds__(256, 2) void ns_symmetric_kernel(NsArgs g) {
    extern __shared__ __align__(16) char smem[];
    constexpr int S = NsTile<TS>::S;
    int t, ti, tk;
    const int spread = ns_spread(g, TS, PIECES), wg = (int)blockIdx.x < spread ? ns_swizzle(blockIdx.x, spread) : blockIdx.x;
    const NsJob j = ns_job_of(g, ns_find(g, SQUARE ? NS_SQUARE : NS_GRAM, wg, t));
    const NsPlanes w(g, j);
    const int side = (w.P + TS - 1) / TS, tiles = side * (side + 1) / 2;
    const int lines = (SQUARE ? w.P : w.Q) / 32, kc = j.kc, line0 = PIECES ? t / tiles * kc : 0;
    ns_diagonal_last(PIECES ? t % tiles : t, side, ti, tk);
    NsTile<TS> c;
    c.zero();
    const cgbytes m = SQUARE ? w.a : w.x;
    const int n = PIECES ? min(kc, lines - line0) : lines;
    if (ti == tk) c.template run<true>(m, w.P, ti * TS, m, w.P, tk * TS, line0, n, smem);
    else c.run(m, w.P, ti * TS, m, w.P, tk * TS, line0, n, smem);
    if (PIECES) {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const auto out = as_global<float>(g.part) + (long)wg * (TS * TS) + lane * 4;
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int k = 0; k < S; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    // subtile (row block, column block) of the tile, then its quarters, a lane's four values together
                    const int sub = ((wave >> 1) * S + i) * (2 * S) + (wave & 1) * S + k;
                    *(DVAE_GLOBAL f32x4*)(out + (sub * 4 + q) * 256) = f32x4{c.acc[i][k][4 * q], c.acc[i][k][4 * q + 1], c.acc[i][k][4 * q + 2], c.acc[i][k][4 * q + 3]};
                }
        return;
    }
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int row = ti * TS + NsTile<TS>::row_of(i, 0), col = tk * TS + NsTile<TS>::col_of(k);
            if (row < w.P && col < w.P) ns_symmetric_value<SQUARE>(g, w, c.acc[i][k], row, col);
        }
    ns_store_symmetric(c, smem, SQUARE ? w.b : w.a, w.P, ti, tk);
}

// Adds the pieces up, a workgroup for each 32x32 subtile: its waves take every fourth piece, four in flight, always in the same order.
template <int TS>
__global__ __launch_bounds__(256) void ns_gram_sum_kernel(NsArgs g) {
    constexpr int SUBS = (TS / 32) * (TS / 32);
    __shared__ f32x4 red[3][4][64];
    __shared__ unsigned patch[32 * 36];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sub = blockIdx.x % SUBS;
    int t, ti, tk;
    const int jn = ns_find(g, NS_GRAM_TILES, blockIdx.x / SUBS, t);
    const NsJob j = ns_job_of(g, jn);
    const NsPlanes w(g, j);
    const int side = (w.P + TS - 1) / TS, tiles = side * (side + 1) / 2;
    ns_diagonal_last(t, side, ti, tk);
    const int row = ti * TS + sub / (TS / 32) * 32, col = tk * TS + sub % (TS / 32) * 32;
    if (row >= w.P || col >= w.P) return;
    const int pieces = (w.Q / 32 + j.kc - 1) / j.kc;
    const auto in = as_global<const float>(g.part) + ((g.njobs == 1 ? 0L : (long)g.first[NS_GRAM * g.jp + jn]) + t) * (TS * TS) + sub * 1024 + lane * 4;
    f32x4 v[4] = {};
    for (int s = wave; s < pieces; s += 16) {
        f32x4 r[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int q = 0; q < 4; ++q) r[u][q] = *(const DVAE_GLOBAL f32x4*)(in + (long)min(s + 4 * u, pieces - 1) * tiles * (TS * TS) + q * 256);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (s + 4 * u < pieces) {
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] += r[u][q];
            }
    }
    if (wave) {
#pragma unroll
        for (int q = 0; q < 4; ++q) red[wave - 1][q][lane] = v[q];
    }
    __syncthreads();
    if (wave) return;
    f32x16 a;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const f32x4 f = (v[q] + red[0][q][lane]) + (red[1][q][lane] + red[2][q][lane]);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[4 * q + e] = f[e];
    }
    ns_symmetric_value<false>(g, w, a, row + 4 * (lane >> 5), col + (lane & 31));
    ns_store(a, patch, ns_line(w.a, w.P, row, col), w.P, ti != tk ? ns_line(w.a, w.P, col, row) : gbytes(nullptr), w.P);
}

// ---- symmetric products straight from memory -----------------------------------------------------------------------------
// Where the tiles of a symmetric product are few, tiles of 32, a workgroup of W waves each: many CUs fetch, the waves take every
// W-th line and feed their MFMAs from memory, four lines in flight (a tile's rows are read once a workgroup: LDS would only
// add its latency and a barrier a line), and add up through LDS at the end, a quarter of the tile for each of four waves.  What is
// left is a chain of latencies (arguments, loads, exchange, store) and, for long contractions, what the L2 gives a CU (35 B a
// clock).  The square: for p = 512, 36 staged tiles of 64 take 8.9 us, 136 of these 6.5 us; for p = 64 4.5 and 3.6.  X X^T: the
// D-VAE's matrices 7 + 5 us (with the sum of the longest one's pieces) against 8.5 + 7.5 us staged, 512 x 4608 20 against 17 us.

// A quarter of a 32x32 tile at (ti, tk) of a symmetric operand, four rows of a lane's column, to both of its places.
__device__ inline void ns_store_quarter(gbytes base, long rows, int ti, int tk, int quarter, const float (&v)[4]) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int row = ti * 32 + 8 * quarter + 4 * half, col = tk * 32 + (lane & 31);
    unsigned u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = ns_split(v[e]);
    const gbytes dst = ns_line(base, rows, col, ti * 32) + quarter * rows * 16 + half * 8;
    *(DVAE_GLOBAL u32x2*)dst = u32x2{(u[0] & 0xffffu) | (u[1] << 16), (u[2] & 0xffffu) | (u[3] << 16)};
    *(DVAE_GLOBAL u32x2*)(dst + rows * 64) = u32x2{(u[0] >> 16) | (u[1] & 0xffff0000u), (u[2] >> 16) | (u[3] & 0xffff0000u)};
    if (ti == tk) return;                                 // the tile holds both places' elements
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const gbytes p = ns_line(base, rows, row + e, tk * 32) + (lane >> 3 & 3) * rows * 16 + (lane & 7) * 2;
        *(DVAE_GLOBAL unsigned short*)p = (unsigned short)u[e];
        *(DVAE_GLOBAL unsigned short*)(p + rows * 64) = (unsigned short)(u[e] >> 16);
    }
}

// A = X X^T, in pieces of a job's kc lines (more than one leave fp32 partial tiles for ns_direct_sum_kernel), or
// B = a I + b A + c A^2.
template <bool SQUARE, int W>
__global__ __launch_bounds__(64 * W) void ns_direct_kernel(NsArgs g) {
    __shared__ f32x4 red[W][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    int t, ti, tk;
    const int wg = ns_swizzle(blockIdx.x, g.total);
    const NsJob j = ns_job_of(g, ns_find(g, SQUARE ? NS_SQUARE : NS_GRAM, wg, t));
    const NsPlanes w(g, j);
    const int all = (SQUARE ? w.P : w.Q) / 32, kc = SQUARE ? all : j.kc, tiles = (w.P / 32) * (w.P / 32 + 1) / 2;
    const int from = t / tiles * kc, to = min(from + kc, all);
    ns_triangle(t % tiles, ti, tk);
    const long rows = w.P;
    const gbytes m = SQUARE ? w.a : w.x;
    const cgbytes lp = ns_line(m, rows, ti * 32 + (lane & 31), 0) + half * rows * 16, rp = ns_line(m, rows, tk * 32 + (lane & 31), 0) + half * rows * 16;
    f32x16 acc[3];
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[k][e] = 0.f;
    for (int line = from + wave; line < to; line += 4 * W) {
        f16x8 l[4][4], r[4][4];                           // [line][two halves of h, then of l]; past the last line that one again, unused
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const long at = (min(line + W * u, to - 1) * 8 + c * 2) * rows * 16;
                l[u][c] = *(const DVAE_GLOBAL f16x8*)(lp + at);
                r[u][c] = *(const DVAE_GLOBAL f16x8*)(rp + at);
            }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (line + W * u >= to) break;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[u][k], r[u][2 + k], acc[0], 0, 0, 0);
                acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[u][2 + k], r[u][k], acc[1], 0, 0, 0);
                acc[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[u][k], r[u][k], acc[2], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[2][4 * q + e] + (acc[0][4 * q + e] + acc[1][4 * q + e]) * (1.f / NS_SL);
        red[wave][q][lane] = v;
    }
    __syncthreads();
    if (wave >= 4) return;
    f32x4 v = red[0][wave][lane];
#pragma unroll
    for (int o = 1; o < W; ++o) v += red[o][wave][lane];
    if (!SQUARE && kc < all) {
        as_global<f32x4>(g.part)[((long)wg * 4 + wave) * 64 + lane] = v;
        return;
    }
    float f[4];
    if (SQUARE) {
        // A's elements of this quarter: rows row .. row + 3 of column col, that is of row col, A being symmetric
        const int row = ti * 32 + 8 * wave + 4 * half, col = tk * 32 + (lane & 31);
        const cgbytes own = ns_line(w.a, rows, col, ti * 32) + wave * rows * 16 + half * 8;
        const u32x2 h = *(const DVAE_GLOBAL u32x2*)own, l = *(const DVAE_GLOBAL u32x2*)(own + rows * 64);
        const f32x4 di = *(const DVAE_GLOBAL f32x4*)(w.diag + row);
        const float dk = w.diag[col];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = ns_polynomial(g, v[e], ns_whole(h, l, e), di[e], dk, row + e == col);
    } else {
        const float scale = ns_gram_scale(g, w);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            f[e] = ns_off_diagonal(w, v[e] * scale, ti * 32 + 8 * wave + 4 * half + e, tk * 32 + (lane & 31));
    }
    ns_store_quarter(SQUARE ? w.b : w.a, rows, ti, tk, wave, f);
}

// Adds the pieces of the matrices that have several, a workgroup a tile, always in the same order.
__global__ __launch_bounds__(256) void ns_direct_sum_kernel(NsArgs g) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int t, ti, tk;
    const int jn = ns_find(g, NS_GRAM_TILES, blockIdx.x, t);
    const NsJob j = ns_job_of(g, jn);
    const NsPlanes w(g, j);
    const int all = w.Q / 32, tiles = (w.P / 32) * (w.P / 32 + 1) / 2, pieces = (all + j.kc - 1) / j.kc;
    if (pieces == 1) return;
    ns_triangle(t, ti, tk);
    const auto in = as_global<const f32x4>(g.part) + (((g.njobs == 1 ? 0L : (long)g.first[NS_GRAM * g.jp + jn]) + t) * 4 + wave) * 64 + lane;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < pieces; s += 8) {
        f32x4 r[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) r[u] = in[(long)min(s + u, pieces - 1) * tiles * 256];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (s + u < pieces) v += r[u];
    }
    float f[4];
    const float scale = ns_gram_scale(g, w);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        f[e] = ns_off_diagonal(w, v[e] * scale, ti * 32 + 8 * wave + 4 * (lane >> 5) + e, tk * 32 + (lane & 31));
    ns_store_quarter(w.a, w.P, ti, tk, wave, f);
}

// X <- B X, left in both orientations
template <int TS, int G>
__global__ __launch_bounds__(256 * G, G == 1 ? 2 : 1) void ns_apply_kernel(NsArgs g) {
    extern __shared__ __align__(16) char smem[];
    constexpr int S = NsTile<TS>::S;
    int t;
    const NsJob j = ns_job_of(g, ns_find(g, NS_APPLY, ns_swizzle(blockIdx.x, g.total), t));
    const NsPlanes w(g, j);
    const int ni = (w.P + TS - 1) / TS, ti = t % ni, tk = t / ni;
    const float scale = ldexpf(1.f / NS_SB, w.shift(g, g.step + 1) - w.shift(g, g.step));
    NsTile<TS, G> c;
    c.zero();
    c.run(w.b, w.P, ti * TS, w.xt(g.turn), w.Q, tk * TS, 0, w.P / 32, smem);
    c.join(smem);
    const int wave = threadIdx.x >> 6, wr = (wave >> 1 & 1) * (TS / 2), wc = (wave & 1) * (TS / 2);
    unsigned* patch = reinterpret_cast<unsigned*>(smem) + wave * (32 * 36);
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int row = ti * TS + wr + i * 32, col = tk * TS + wc + k * 32;
            if (row >= w.P || col >= w.Q || i < c.from || i >= c.to) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) c.acc[i][k][e] *= scale;
            ns_store(c.acc[i][k], patch, ns_line(w.x, w.P, row, col), w.P, ns_line(w.xt(g.turn ^ 1), w.Q, col, row), w.Q);
        }
}

// The last product: its tile goes to the caller's matrix, or steps the parameter.  A tall matrix's tile is computed
// transposed (the operands trade places), so that lanes run along the caller's rows either way.
template <int TS, typename T, bool MUON, int G>
__global__ __launch_bounds__(256 * G, G == 1 ? 2 : 1) void ns_last_kernel(NsArgs g) {
    extern __shared__ __align__(16) char smem[];
    constexpr int S = NsTile<TS>::S;
    int t;
    const NsJob j = ns_job_of(g, ns_find(g, NS_APPLY, ns_swizzle(blockIdx.x, g.total), t));
    const NsPlanes w(g, j);
    const bool tall = j.m > j.n;
    const float scale = ldexpf(1.f / (NS_SB * NS_SX), -w.shift(g, g.step));
    const int ni = (w.P + TS - 1) / TS, tp = t % ni, tq = t / ni;
    NsTile<TS, G> c;
    c.zero();
    const cgbytes L = tall ? w.xt(g.turn) : w.b, R = tall ? w.b : w.xt(g.turn);
    const int lrows = tall ? w.Q : w.P, rrows = tall ? w.P : w.Q, ti = tall ? tq : tp, tk = tall ? tp : tq;
    c.run(L, lrows, ti * TS, R, rrows, tk * TS, 0, w.P / 32, smem);
    c.join(smem);
    const auto out = as_global<T>(j.out);
    const float step = MUON ? g.lr * j.scale : 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int col = tk * TS + NsTile<TS>::col_of(k);
            if (col >= j.n || i < c.from || i >= c.to) continue;
            float p[16];
            if (MUON) {
#pragma unroll
                for (int e = 0; e < 16; ++e) p[e] = (float)out[min(ti * TS + NsTile<TS>::row_of(i, e), j.m - 1) * j.os + col];
            }
            const bool whole = ti * TS + NsTile<TS>::row_of(i, 15) < j.m;      // a lane's last row
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = c.acc[i][k][e] * scale;
                p[e] = ns_rounded(MUON ? p[e] * g.decay - step * v : v);
            }
            if (whole) {
#pragma unroll
                for (int e = 0; e < 16; ++e) out[(ti * TS + NsTile<TS>::row_of(i, e)) * j.os + col] = (T)p[e];
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int row = ti * TS + NsTile<TS>::row_of(i, e);
                    if (row < j.m) out[row * j.os + col] = (T)p[e];
                }
            }
        }
}

}  // namespace dvae
