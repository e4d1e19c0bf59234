// libdvae_hip.so: entry points of the learning operators that work on tensors of any shape -- layer norm, Newton-Schulz
// orthogonalisation, the Muon step.  A translation unit of its own: its kernels share nothing with the convolutions'.
// Host code here only validates, derives launch geometry and launches on the caller's stream.
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.hpp"
#include "layer_norm.hpp"
#include "newton_schulz.hpp"
#include "newton_schulz_small.hpp"

using namespace dvae;

namespace {

inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

// ---- layer norm -------------------------------------------------------------------------------------------------------
// How a row is held.  Up to 512 columns it lives in LPR lanes of at most 8 columns; up to 8192 in W waves, 8 columns a thread
// again (16 take twice the registers of the backward pass and half its occupancy: 3.0 instead of 4.4 TB/s at 4096 bf16
// columns); up to 16384 in 16 waves with 16; longer rows are read once per pass.
struct LnShape {
    int lpr, nv, waves;
    bool tail;
};
inline LnShape ln_shape(int C, int dtype) {
    const int N = dtype == DVAE_F32 ? 4 : 8;
    const int vecs = (C + N - 1) / N;
    LnShape s{0, 1, 0, C % N != 0};
    if (C <= 512) {
        s.lpr = 4;
        while (s.lpr < vecs && s.lpr < 64) s.lpr <<= 1;
        while (s.lpr * s.nv < vecs) s.nv <<= 1;
    } else if (C <= 16384) {
        s.waves = 2;
        while (s.waves < 16 && s.waves * 512 < C) s.waves <<= 1;
        s.nv = (C <= 8192 ? 8 : 16) / N;
    }
    return s;
}
// Workgroups of the backward pass, each of which leaves one slab of column sums: enough to fill the chip, but at least four
// trips each, so that the slabs stay a small part of the traffic.
inline int ln_bwd_groups(int64_t rows, int C, int dtype) {
    const LnShape s = ln_shape(C, dtype);
    const int64_t rpb = s.lpr ? 256 / s.lpr : 1;
    int64_t g = cdiv64(rows, rpb * 4);
    if (g > 256) g = cdiv64(rows, rpb * 8) > 256 ? cdiv64(rows, rpb * 8) : 256;      // eight trips once every CU has one
    const int64_t cap = s.lpr || s.waves <= 4 ? 1024 : s.waves ? 4096 / s.waves : 64;
    if (g > cap) g = cap;
    return (int)(g < 1 ? 1 : g);
}
// Workgroups of the slabs' sum, of 1024 threads: a launch holds fewer than 2^32 threads, rows may have 2^30 columns.
constexpr int64_t LN_REDUCE_GRID = 1 << 20;
// Forward: eight workgroups of four waves a CU, which then walk their rows with gamma / beta in registers.
constexpr int LN_GRID = 2048;

int ln_check(const char* what, int64_t rows, int C, int dtype) {
    if (dtype != DVAE_F32 && dtype != DVAE_BF16) DVAE_FAIL(DVAE_EDTYPE, "%s: unknown dtype %d", what, dtype);
    if (rows < 0 || C <= 0 || C >= (1 << 30)) DVAE_FAIL(DVAE_EINVAL, "%s: bad shape %lld x %d", what, (long long)rows, C);
    return DVAE_OK;
}
// an operand: present, element-aligned, rows that do not overlap where they are written
int ln_operand(const char* what, const char* name, const void* p, int64_t stride, int64_t rows, int C, int dtype, bool written) {
    const uintptr_t size = dtype == DVAE_F32 ? 4 : 2;
    if (!p) DVAE_FAIL(DVAE_EINVAL, "%s: %s is null", what, name);
    if ((uintptr_t)p % size) DVAE_FAIL(DVAE_EINVAL, "%s: %s is not aligned to its elements", what, name);
    if (stride < 0 || (written && rows > 1 && stride < C))
        DVAE_FAIL(DVAE_EINVAL, "%s: row stride %lld of %s (%d columns)", what, (long long)stride, name, C);
    return DVAE_OK;
}

template <typename T, int LPR, int NV>
void ln_launch_rows(const LnArgs& a, const LnShape& s, bool bwd, int groups, hipStream_t st) {
    constexpr int RPB = 256 / LPR, U = NV == 1 ? 4 : 2;
    if (bwd) {
        if (s.tail) hipLaunchKernelGGL((ln_bwd_rows_kernel<T, LPR, NV, true>), dim3(groups), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((ln_bwd_rows_kernel<T, LPR, NV, false>), dim3(groups), dim3(256), 0, st, a);
        return;
    }
    // several rows a lane only where that leaves the chip full: short calls want their rows spread out
    if (U > 1 && a.rows >= (int64_t)RPB * U * 512) {
        const int g = (int)(cdiv64(a.rows, RPB * U) < LN_GRID ? cdiv64(a.rows, RPB * U) : LN_GRID);
        if (s.tail) hipLaunchKernelGGL((ln_fwd_rows_kernel<T, LPR, NV, U, true>), dim3(g), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((ln_fwd_rows_kernel<T, LPR, NV, U, false>), dim3(g), dim3(256), 0, st, a);
    } else {
        const int g = (int)(cdiv64(a.rows, RPB) < LN_GRID ? cdiv64(a.rows, RPB) : LN_GRID);
        if (s.tail) hipLaunchKernelGGL((ln_fwd_rows_kernel<T, LPR, NV, 1, true>), dim3(g), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((ln_fwd_rows_kernel<T, LPR, NV, 1, false>), dim3(g), dim3(256), 0, st, a);
    }
}
template <typename T, int W, int NV>
void ln_launch_wide(const LnArgs& a, const LnShape& s, bool bwd, int groups, hipStream_t st) {
    if (bwd) {
        if (s.tail) hipLaunchKernelGGL((ln_bwd_wide_kernel<T, W, NV, true>), dim3(groups), dim3(W * 64), 0, st, a);
        else hipLaunchKernelGGL((ln_bwd_wide_kernel<T, W, NV, false>), dim3(groups), dim3(W * 64), 0, st, a);
        return;
    }
    const int g = (int)(a.rows < LN_GRID * 4 / W ? a.rows : LN_GRID * 4 / W);
    if (s.tail) hipLaunchKernelGGL((ln_fwd_wide_kernel<T, W, NV, true>), dim3(g), dim3(W * 64), 0, st, a);
    else hipLaunchKernelGGL((ln_fwd_wide_kernel<T, W, NV, false>), dim3(g), dim3(W * 64), 0, st, a);
}
template <typename T>
void ln_launch(const LnArgs& a, const LnShape& s, bool bwd, int groups, hipStream_t st) {
    constexpr int V = sizeof(T) == 4 ? 2 : 1;             // vectors of 8 columns
    if (s.lpr) {
        if (s.lpr == 4) ln_launch_rows<T, 4, 1>(a, s, bwd, groups, st);
        else if (s.lpr == 8) ln_launch_rows<T, 8, 1>(a, s, bwd, groups, st);
        else if (s.lpr == 16) ln_launch_rows<T, 16, 1>(a, s, bwd, groups, st);
        else if (s.lpr == 32) ln_launch_rows<T, 32, 1>(a, s, bwd, groups, st);
        else if (s.nv == 1) ln_launch_rows<T, 64, 1>(a, s, bwd, groups, st);
        else ln_launch_rows<T, 64, V>(a, s, bwd, groups, st);
    } else if (s.waves == 2) {
        ln_launch_wide<T, 2, V>(a, s, bwd, groups, st);
    } else if (s.waves == 4) {
        ln_launch_wide<T, 4, V>(a, s, bwd, groups, st);
    } else if (s.waves == 8) {
        ln_launch_wide<T, 8, V>(a, s, bwd, groups, st);
    } else if (s.waves == 16) {
        if (s.nv == V) ln_launch_wide<T, 16, V>(a, s, bwd, groups, st);
        else ln_launch_wide<T, 16, 2 * V>(a, s, bwd, groups, st);
    } else if (bwd) {
        hipLaunchKernelGGL((ln_bwd_long_kernel<T>), dim3((int)(a.rows < 2048 ? a.rows : 2048)), dim3(1024), 0, st, a);
        if (a.partial) hipLaunchKernelGGL((ln_cols_kernel<T>), dim3((a.C + 255) / 256, groups), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((ln_fwd_long_kernel<T>), dim3((int)(a.rows < 2048 ? a.rows : 2048)), dim3(1024), 0, st, a);
    }
}

// ---- Newton-Schulz ----------------------------------------------------------------------------------------------------
inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// Workgroups of a launch: 2^32 threads at 512 each.  Matrices that would need more do not fit the memory.
constexpr long NS_MOST = (1L << 23) - 1;

struct NsPlan {
    std::vector<unsigned> table;      // prefix arrays, then jobs, as they lie on the device
    int njobs = 0, jp = 0;
    long total[NS_PHASES] = {};
    int gram_ts = 64, square_ts = 64, apply_ts = 64;
    int apply_groups = 1;
    bool gram_pieces = false;
    size_t norm_off = 0, part_off = 0, bytes = 0;
    bool matrices = false;
};

// The largest singular value the iteration can reach from 1, and the largest |a + b s^2 + c s^4| it meets, by the polynomials'
// own extrema.  `rate`: the base-2 logarithm of the latter, rounded up and 0 at least.
bool ns_coefficients_fit(double a, double b, double c, int steps, float& rate) {
    double grows = 1.0;
    if (!isfinite(a) || !isfinite(b) || !isfinite(c)) return false;
    auto q = [&](double l) { return a + b * l + c * l * l; };
    double s = 1.0 + 1e-6;
    for (int k = 0; k < steps; ++k) {
        double l[4] = {0.0, s * s, 0.0, 0.0}, most_q = 0.0, most_x = 0.0;
        int n = 2;
        if (c != 0.0 && -b / (2 * c) > 0 && -b / (2 * c) < s * s) l[n++] = -b / (2 * c);
        for (int i = 0; i < n; ++i) most_q = fmax(most_q, fabs(q(l[i])));
        n = 2;                                            // x q(x^2): a + 3 b l + 5 c l^2 = 0
        if (c != 0.0) {
            const double d = 9 * b * b - 20 * a * c;
            if (d >= 0)
                for (int g = -1; g <= 1; g += 2) {
                    const double r = (-3 * b + g * sqrt(d)) / (10 * c);
                    if (r > 0 && r < s * s) l[n++] = r;
                }
        } else if (b != 0.0 && -a / (3 * b) > 0 && -a / (3 * b) < s * s) {
            l[n++] = -a / (3 * b);
        }
        for (int i = 0; i < n; ++i) most_x = fmax(most_x, sqrt(l[i]) * fabs(q(l[i])));
        if (!(most_q <= 7.001)) return false;                // a hair over, so that the bounds themselves pass
        grows = fmax(grows, most_q);
        rate = (float)(log2(grows) + 1e-6);
        s = most_x * (1.0 + 1e-4);
        if (!(s <= 2.001)) return false;
        if (s == 0.0) return true;
        if (s < 1e-30) s = 1e-30;
    }
    return true;
}

int ns_check(const char* what, const dvae_matrix* mats, int count, int dtype, bool muon) {
    if (count < 0 || (count > 0 && !mats)) DVAE_FAIL(DVAE_EINVAL, "%s: null list", what);
    if (count > 65536) DVAE_FAIL(DVAE_EINVAL, "%s: %d matrices (65536 at most)", what, count);
    if (dtype != DVAE_F32 && dtype != DVAE_BF16) DVAE_FAIL(DVAE_EDTYPE, "%s: unknown dtype %d", what, dtype);
    for (int i = 0; i < count; ++i) {
        const dvae_matrix& m = mats[i];
        const uintptr_t size = dtype == DVAE_F32 ? 4 : 2;
        if (m.rows <= 0 || m.cols <= 0 || m.rows > (1 << 30) || m.cols > (1 << 30) || m.rows * m.cols >= (1LL << 31))
            DVAE_FAIL(DVAE_EINVAL, "%s: matrix %d is %lld x %lld", what, i, (long long)m.rows, (long long)m.cols);
        if (!m.x || !m.out || (muon && !m.momentum)) DVAE_FAIL(DVAE_EINVAL, "%s: matrix %d has a null pointer", what, i);
        if (((uintptr_t)m.x | (uintptr_t)m.out) % size || (muon && (uintptr_t)m.momentum % 4))
            DVAE_FAIL(DVAE_EINVAL, "%s: matrix %d is not aligned to its elements", what, i);
        if (muon ? m.x_stride != m.cols || m.out_stride != m.cols : m.x_stride < 0 || (m.rows > 1 && m.out_stride < m.cols))
            DVAE_FAIL(DVAE_EINVAL, "%s: matrix %d has row strides %lld, %lld", what, i, (long long)m.x_stride, (long long)m.out_stride);
    }
    return DVAE_OK;
}

inline long ns_triangles(int P, int ts) {
    const long t = (P + ts - 1) / ts;
    return t * (t + 1) / 2;
}

void ns_job(const dvae_matrix& m, int scale_rule, NsJob& j) {
    j = NsJob{};
    j.x = m.x; j.out = m.out; j.mom = m.momentum;
    j.xs = m.x_stride; j.os = m.out_stride;
    j.m = (int)m.rows; j.n = (int)m.cols;
    j.vec = m.vector ? 1 : 0;
    const double r = (double)j.m, c = (double)j.n;
    j.scale = (float)(scale_rule == DVAE_MUON_RMS ? 0.2 * sqrt(fmax(r, c)) : sqrt(fmax(1.0, r / c)));
}

// Whether every matrix of a call fits the one-launch kernel.  One that does not makes the whole call go through the batched
// phases, where small matrices ride along for next to nothing.
bool ns_all_small(const dvae_matrix* mats, int count) {
    for (int i = 0; i < count; ++i) {
        const int64_t p = mats[i].rows < mats[i].cols ? mats[i].rows : mats[i].cols, q = mats[i].rows < mats[i].cols ? mats[i].cols : mats[i].rows;
        if (mats[i].vector ? mats[i].rows * mats[i].cols > NS_SMALL_VEC : p > NS_SMALL_P || q > NS_SMALL_Q) return false;
        if (mats[i].x_stride > NS_SMALL_SPAN / mats[i].rows || mats[i].out_stride > NS_SMALL_SPAN / mats[i].rows) return false;
    }
    return true;
}

// words of host memory to the device, as many kernel arguments at a time as fit
int ns_upload(const char* what, const unsigned* words, size_t count, unsigned* dst, hipStream_t st) {
    NsBlob blob;
    for (size_t at = 0; at < count; at += NsBlob::WORDS) {
        const size_t n = count - at < (size_t)NsBlob::WORDS ? count - at : (size_t)NsBlob::WORDS;
        memcpy(blob.w, words + at, n * 4);
        hipLaunchKernelGGL(ns_table_kernel, dim3(1), dim3(256), 0, st, blob, dst + at, (int)n);
        DVAE_CHECK_LAUNCH(what);
    }
    return DVAE_OK;
}

size_t ns_small_bytes(int count) { return count <= NS_SMALL_JOBS ? 256 : align256(count * sizeof(NsJob)); }

// A workgroup for each matrix: up to 32 in the kernel's arguments, more in a table.
template <typename T, bool MUON>
int ns_run_small(const char* what, const dvae_matrix* mats, int count, int scale_rule, const NsArgs& g, int steps, hipStream_t st) {
    static LdsOptIn opt[3];
    NsSmallArgs a{};
    a.eps = g.eps; a.a = g.a; a.b = g.b; a.c = g.c; a.mu = g.mu; a.nu = g.nu; a.lr = g.lr; a.decay = g.decay;
    a.nesterov = g.nesterov; a.steps = steps; a.rate = g.rate;
    std::vector<NsJob> many((size_t)(count > NS_SMALL_JOBS ? count : 0));
    NsJob* jobs = many.empty() ? a.jobs : many.data();
    int q = 1;
    for (int k = 0; k < count; ++k) {
        ns_job(mats[k], scale_rule, jobs[k]);
        if (!jobs[k].vec) q = std::max(q, std::max(jobs[k].m, jobs[k].n));
    }
    if (!many.empty()) {
        static_assert(sizeof(NsJob) % 4 == 0, "whole words");
        const int rc = ns_upload(what, (const unsigned*)many.data(), many.size() * sizeof(NsJob) / 4, (unsigned*)g.ws, st);
        if (rc) return rc;
        a.table = (const NsJob*)g.ws;
    }
    const int lds = (int)sizeof(NsSmallLds);
#define NS_SMALL_LAUNCH(NB)                                                                                          \
    do {                                                                                                             \
        opt[NB - 1].ensure((const void*)ns_small_kernel<T, MUON, NB>, lds);                                          \
        hipLaunchKernelGGL((ns_small_kernel<T, MUON, NB>), dim3(count), dim3(512), lds, st, a);                      \
    } while (0)
    if (q <= 256) NS_SMALL_LAUNCH(1);
    else if (q <= 512) NS_SMALL_LAUNCH(2);
    else NS_SMALL_LAUNCH(3);
#undef NS_SMALL_LAUNCH
    DVAE_CHECK_LAUNCH(what);
    return DVAE_OK;
}

int ns_plan(const char* what, const dvae_matrix* mats, int count, int scale_rule, NsPlan& p) {
    p.njobs = count;
    p.jp = (count + 1 + 63) / 64 * 64;
    std::vector<NsJob> jobs((size_t)count);
    std::vector<int> first((size_t)NS_PHASES * p.jp, INT_MAX);
    // Tile sizes by the work they make, in us of a CU: a line of a 128-tile costs it 0.78, of a 64-tile 0.28 (measured with the chip
    // full; a 128-tile is four of those), and a tile's start and end about 3 and 1.2.  Padding decides: 64-row matrices want 64.
    double cost[3][2] = {};                               // Gram, square, apply; tiles of 64, of 128
    long longest[2] = {1, 1}, lines[2] = {}, tiles[3][2] = {}, tiles32 = 0, lines32 = 0;
    for (int i = 0; i < count; ++i) {
        const dvae_matrix& m = mats[i];
        if (m.vector) continue;
        const int P = ns_pad((int)(m.rows < m.cols ? m.rows : m.cols)), Q = ns_pad((int)(m.rows < m.cols ? m.cols : m.rows));
        for (int big = 0; big < 2; ++big) {
            const int ts = big ? 128 : 64;
            const double line = big ? 0.78 : 0.28, ends = big ? 3.0 : 1.2;
            const long tri = ns_triangles(P, ts);
            cost[0][big] += tri * (Q / 32 * line + ends);
            cost[1][big] += tri * (P / 32 * line + ends);
            cost[2][big] += (double)((P + ts - 1) / ts) * ((Q + ts - 1) / ts) * (P / 32 * line + ends);
            lines[big] += tri * (Q / 32);
            tiles[0][big] += tri;
            tiles[1][big] += tri;
            tiles[2][big] += (long)((P + ts - 1) / ts) * ((Q + ts - 1) / ts);
        }
        tiles32 += ns_triangles(P, 32);
        lines32 += ns_triangles(P, 32) * (Q / 32);
        longest[0] = longest[0] > Q / 32 ? longest[0] : Q / 32;
        longest[1] = longest[1] > P / 32 ? longest[1] : P / 32;
        p.matrices = true;
    }
    // The Gram product is cut into pieces anyhow: 128 once that leaves each of 512 workgroups eight lines (below, their starts and
    // partial tiles cost more: 512 x 4608 210 us against 231, ResNet-18's matrices 575 against 560).
    p.gram_ts = cost[0][1] < cost[0][0] && lines[1] >= 4096 ? 128 : 64;
    // a product of one tile a workgroup: 128 only where that still gives every CU one
    p.apply_ts = cost[2][1] < cost[2][0] && cost[2][1] / 256 >= 0.9 * (longest[1] * 0.78 + 3.0) ? 128 : 64;
    // The Gram product in pieces: about 512 workgroups, two a CU, of at least 4 lines; none where tiles of 64 alone are as many
    // (2048 x 2048: 53 us whole in tiles of 64, 45 + 12 us in pieces of tiles of 128).
    const bool cut_gram = tiles[0][0] < 512;
    if (!cut_gram && tiles[0][1] < 512) p.gram_ts = 64;
    // Straight from memory in tiles of 32 where that is sooner done.  Times in us, measured: the pieces and their sum have 13 beside
    // their work (512 x 4608: 17 us in all, the D-VAE's matrices 16); a workgroup of the other 0.12 a line and 3, another 5 where it
    // leaves pieces (144 lines: 20 us; the D-VAE's: 12 us).
    const long direct_kc = lines32 / 256 > 32 ? lines32 / 256 : 32;
    auto direct_piece = [&](long all) {                   // lines of a workgroup: a CU's share of all, in equal pieces
        const long n = all / direct_kc > 1 ? all / direct_kc : 1;
        return (int)((all + n - 1) / n);
    };
    if (cut_gram) {
        int longest_piece = 0;
        bool several = false;
        for (int i = 0; i < count; ++i) {
            if (mats[i].vector) continue;
            const int all = ns_pad((int)(mats[i].rows < mats[i].cols ? mats[i].cols : mats[i].rows)) / 32, piece = direct_piece(all);
            longest_piece = std::max(longest_piece, piece);
            several = several || piece < all;
        }
        const double direct = fmax(longest_piece * 0.12, lines32 * 0.1 / 256) + (several ? 8.0 : 3.0);
        if (direct < cost[0][p.gram_ts == 128] / 256 + 13.0) p.gram_ts = 32;
    }
    const int gb = p.gram_ts == 128;
    const int gram_kc = (int)((lines[gb] + 511) / 512);
    // The square has p / 32 lines and few tiles: straight from memory in tiles of 32 up to about two workgroups of those a SIMD
    // (beyond, they read more than the L2 gives), whole in tiles of 64 until those of 128 fill the chip.
    p.square_ts = tiles32 <= 1280 ? 32 : tiles[1][1] >= 512 ? 128 : 64;
    // Two groups, see NsTile, where tiles of 128 are no more than the CUs.  Whole calls with one group and with two: 2048 x 2048 783
    // and 770 us, 1984 x 2048 772 and 760, 1856 x 2048 648 and 636, 1000 x 4000 385 and 380, 832 x 4608 and 700 x 5000 the same.
    p.apply_groups = p.apply_ts == 128 && tiles[2][1] <= 256 ? 2 : 1;
    auto piece = [](bool cut, int kc, int all) {          // at most 64 of a tile; even
        if (!cut) return all;
        if (kc < 4) kc = 4;
        if (kc < (all + 63) / 64) kc = (all + 63) / 64;
        return (kc + 1) & ~1;
    };
    long off = 0, part = 0;
    // The matrices with the longest contractions go first, so that no long tile starts when the short ones are done.
    std::vector<int> order((size_t)count);
    for (int i = 0; i < count; ++i) order[i] = i;
    auto side = [&](int i) { return mats[i].vector ? 0 : mats[i].rows < mats[i].cols ? mats[i].rows : mats[i].cols; };
    std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return side(a) > side(b); });
    for (int i = 0; i < count; ++i) {
        const dvae_matrix& m = mats[order[i]];
        NsJob& j = jobs[i];
        ns_job(m, scale_rule, j);
        const long chunks = ((long)j.m * j.n + NS_CHUNK - 1) / NS_CHUNK;
        j.nchunk = (int)(chunks < 1024 ? chunks : 1024);
        j.part = (int)part;
        for (int f = 0; f < NS_PHASES; ++f) {
            if (p.total[f] > NS_MOST) DVAE_FAIL(DVAE_EINVAL, "%s: too much work for one call", what);
            first[(size_t)f * p.jp + i] = (int)p.total[f];
        }
        p.total[NS_NORM] += j.nchunk;
        j.off = off;
        if (j.vec) continue;
        part += j.nchunk;
        const int P = ns_pad(j.m < j.n ? j.m : j.n), Q = ns_pad(j.m < j.n ? j.n : j.m);
        off += ns_job_bytes(j.m, j.n);
        p.total[NS_SPLIT] += (long)(P / 64) * (Q / 64);
        j.kc = p.gram_ts == 32 ? direct_piece(Q / 32) : piece(cut_gram, gram_kc, Q / 32);
        const long gp = (Q / 32 + j.kc - 1) / j.kc;
        if (gp > 1) p.gram_pieces = true;
        p.total[NS_GRAM] += ns_triangles(P, p.gram_ts) * gp;
        p.total[NS_GRAM_TILES] += ns_triangles(P, p.gram_ts);
        p.total[NS_SQUARE] += ns_triangles(P, p.square_ts);
        p.total[NS_APPLY] += (long)((P + p.apply_ts - 1) / p.apply_ts) * ((Q + p.apply_ts - 1) / p.apply_ts);
    }
    for (int f = 0; f < NS_PHASES; ++f)
        if (p.total[f] > NS_MOST) DVAE_FAIL(DVAE_EINVAL, "%s: too much work for one call", what);
    // jobs without tiles in a phase share their first with the next one that has some; those after the last such are beyond it
    const size_t words = first.size() + jobs.size() * sizeof(NsJob) / 4;
    p.table.resize(words);
    memcpy(p.table.data(), first.data(), first.size() * 4);
    if (count) memcpy(p.table.data() + first.size(), jobs.data(), jobs.size() * sizeof(NsJob));
    p.norm_off = align256(words * 4);
    p.part_off = p.norm_off + align256((size_t)part * sizeof(double));
    size_t parts = 0;
    if (p.gram_pieces) parts = (size_t)p.total[NS_GRAM] * p.gram_ts * p.gram_ts;
    const size_t planes = p.part_off + align256(parts * 4);
    NsJob* t = reinterpret_cast<NsJob*>(p.table.data() + first.size());
    for (int i = 0; i < count; ++i) t[i].off += (long)planes;
    p.bytes = planes + (size_t)off;
    return DVAE_OK;
}

template <typename T, bool MUON>
int ns_run(const char* what, const NsPlan& p, NsArgs g, int steps, hipStream_t st) {
    if (p.njobs == 1) {
        memcpy(&g.one, p.table.data() + (size_t)NS_PHASES * p.jp, sizeof(NsJob));
    } else {
        const int rc = ns_upload(what, p.table.data(), p.table.size(), (unsigned*)g.ws, st);
        if (rc) return rc;
    }
    g.first = (const int*)g.ws;
    g.jobs = (const NsJob*)(g.ws + (size_t)NS_PHASES * p.jp * 4);
    g.norm = (double*)(g.ws + p.norm_off);
    g.part = (float*)(g.ws + p.part_off);
    g.njobs = p.njobs;
    g.jp = p.jp;
    g.turn = 0;
// n workgroups of 256 * groups threads with tiles of ts in LDS (0: none); kernels that want over 64 KB of it say so once
#define NS_LAUNCH_N(n, groups, lds, ...)                                                             \
    do {                                                                                             \
        static LdsOptIn opt;                                                                         \
        if ((lds) > 65536) opt.ensure((const void*)(__VA_ARGS__), lds);                              \
        g.total = (int)(n);                                                                          \
        hipLaunchKernelGGL((__VA_ARGS__), dim3((unsigned)(n)), dim3(256 * (groups)), lds, st, g);    \
        DVAE_CHECK_LAUNCH(what);                                                                     \
    } while (0)
#define NS_LAUNCH(phase, ...) NS_LAUNCH_N(p.total[phase], 1, 0, __VA_ARGS__)
#define NS_LAUNCH_TILES(phase, ts, groups, ...) NS_LAUNCH_N(p.total[phase], groups, (NsTile<ts, groups>::BYTES), __VA_ARGS__)
    NS_LAUNCH(NS_NORM, ns_norm_kernel<T, MUON>);
    if (!p.matrices) return DVAE_OK;
    NS_LAUNCH(NS_SPLIT, ns_split_kernel<T, MUON>);
    for (int k = 0; k < steps; ++k) {
        g.step = k;
        if (p.gram_ts == 32) {
            NS_LAUNCH_N(p.total[NS_GRAM], 2, 0, ns_direct_kernel<false, 8>);
            if (p.gram_pieces) NS_LAUNCH(NS_GRAM_TILES, ns_direct_sum_kernel);
        } else if (p.gram_ts == 64) {
            if (!p.gram_pieces) NS_LAUNCH_TILES(NS_GRAM, 64, 1, ns_symmetric_kernel<64, false, false>);
            else {
                NS_LAUNCH_TILES(NS_GRAM, 64, 1, ns_symmetric_kernel<64, false, true>);
                NS_LAUNCH_N(p.total[NS_GRAM_TILES] * 4, 1, 0, ns_gram_sum_kernel<64>);
            }
        } else if (!p.gram_pieces) {
            NS_LAUNCH_TILES(NS_GRAM, 128, 1, ns_symmetric_kernel<128, false, false>);
        } else {
            NS_LAUNCH_TILES(NS_GRAM, 128, 1, ns_symmetric_kernel<128, false, true>);
            NS_LAUNCH_N(p.total[NS_GRAM_TILES] * 16, 1, 0, ns_gram_sum_kernel<128>);
        }
        if (p.square_ts == 32) NS_LAUNCH(NS_SQUARE, ns_direct_kernel<true, 4>);
        else if (p.square_ts == 64) NS_LAUNCH_TILES(NS_SQUARE, 64, 1, ns_symmetric_kernel<64, true, false>);
        else NS_LAUNCH_TILES(NS_SQUARE, 128, 1, ns_symmetric_kernel<128, true, false>);
        const bool last = k + 1 == steps;
        if (p.apply_ts == 128 && p.apply_groups == 1) {
            if (last) NS_LAUNCH_TILES(NS_APPLY, 128, 1, ns_last_kernel<128, T, MUON, 1>);
            else NS_LAUNCH_TILES(NS_APPLY, 128, 1, ns_apply_kernel<128, 1>);
        } else if (p.apply_ts == 128) {
            if (last) NS_LAUNCH_TILES(NS_APPLY, 128, 2, ns_last_kernel<128, T, MUON, 2>);
            else NS_LAUNCH_TILES(NS_APPLY, 128, 2, ns_apply_kernel<128, 2>);
        } else {
            if (last) NS_LAUNCH_TILES(NS_APPLY, 64, 1, ns_last_kernel<64, T, MUON, 1>);
            else NS_LAUNCH_TILES(NS_APPLY, 64, 1, ns_apply_kernel<64, 1>);
        }
        g.turn ^= 1;
    }
#undef NS_LAUNCH_TILES
#undef NS_LAUNCH
#undef NS_LAUNCH_N
    return DVAE_OK;
}

int ns_iteration_check(const char* what, const double* coefficients, int steps, double eps, float& rate) {
    if (!coefficients) DVAE_FAIL(DVAE_EINVAL, "%s: null coefficients", what);
    if (steps < 1 || steps > 100) DVAE_FAIL(DVAE_EINVAL, "%s: %d steps (1 to 100)", what, steps);
    if (!(eps >= 0.0) || !isfinite(eps)) DVAE_FAIL(DVAE_EINVAL, "%s: eps %g", what, eps);
    if (!ns_coefficients_fit(coefficients[0], coefficients[1], coefficients[2], steps, rate))
        DVAE_FAIL(DVAE_EINVAL, "%s: coefficients (%g, %g, %g) leave the range this iteration is computed in: from singular "
                  "values up to 1 every step has to stay at 2 or below, with |a + b s^2 + c s^4| at 7 or below", what,
                  coefficients[0], coefficients[1], coefficients[2]);
    return DVAE_OK;
}
int ns_workspace_check(const char* what, const void* ws, size_t have, size_t need) {
    if (!ws || (uintptr_t)ws & 255) DVAE_FAIL(DVAE_EINVAL, "%s: the workspace must be 256-byte aligned", what);
    if (have < need) DVAE_FAIL(DVAE_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, have, need);
    return DVAE_OK;
}

}  // namespace

extern "C" {

size_t dvae_layer_norm_workspace_bytes(int64_t rows, int C, int dtype) {
    if (rows < 0 || C <= 0 || C >= (1 << 30) || (dtype != DVAE_F32 && dtype != DVAE_BF16)) return 0;
    const LnShape s = ln_shape(C, dtype);
    return ((size_t)ln_bwd_groups(rows, C, dtype) * 2 * C + (s.lpr || s.waves ? 0 : (size_t)rows)) * sizeof(float);
}

int dvae_layer_norm_fwd(const void* x, int64_t x_stride, const float* gamma, const float* beta, void* y, int64_t y_stride,
                        float* save_mean, float* save_invstd, int64_t rows, int C, float eps, int dtype, void* st) {
    int rc = ln_check("layer_norm_fwd", rows, C, dtype);
    if (rc || rows == 0) return rc;
    if ((rc = ln_operand("layer_norm_fwd", "x", x, x_stride, rows, C, dtype, false))) return rc;
    if ((rc = ln_operand("layer_norm_fwd", "y", y, y_stride, rows, C, dtype, true))) return rc;
    if (!save_mean != !save_invstd) DVAE_FAIL(DVAE_EINVAL, "layer_norm_fwd: save_mean and save_invstd go together");
    if (!(eps >= 0.f)) DVAE_FAIL(DVAE_EINVAL, "layer_norm_fwd: eps %g", eps);
    LnArgs a{};
    a.x = x; a.xs = x_stride; a.y = y; a.ys = y_stride; a.gamma = gamma; a.beta = beta; a.mean = save_mean; a.invstd = save_invstd;
    a.rows = rows; a.C = C; a.eps = eps;
    const LnShape s = ln_shape(C, dtype);
    if (dtype == DVAE_F32) ln_launch<float>(a, s, false, 0, S(st));
    else ln_launch<bf16>(a, s, false, 0, S(st));
    DVAE_CHECK_LAUNCH("layer_norm_fwd");
    return DVAE_OK;
}

int dvae_layer_norm_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* gamma,
                        const float* save_mean, const float* save_invstd, void* dx, int64_t dx_stride, float* dgamma,
                        float* dbeta, void* workspace, size_t workspace_bytes, int64_t rows, int C, int dtype, void* st) {
    int rc = ln_check("layer_norm_bwd", rows, C, dtype);
    if (rc) return rc;
    const bool sums = dgamma || dbeta;
    if (!dx && !sums) return DVAE_OK;
    const int groups = ln_bwd_groups(rows, C, dtype);
    if (sums && rows) {
        if (!workspace || (uintptr_t)workspace & 15) DVAE_FAIL(DVAE_EINVAL, "layer_norm_bwd: the workspace must be 16-byte aligned");
        if (workspace_bytes < dvae_layer_norm_workspace_bytes(rows, C, dtype))
            DVAE_FAIL(DVAE_EWORKSPACE, "layer_norm_bwd: workspace of %zu bytes, %zu needed", workspace_bytes,
                      dvae_layer_norm_workspace_bytes(rows, C, dtype));
    }
    if (rows) {
        if ((rc = ln_operand("layer_norm_bwd", "dy", dy, dy_stride, rows, C, dtype, false))) return rc;
        if ((rc = ln_operand("layer_norm_bwd", "x", x, x_stride, rows, C, dtype, false))) return rc;
        if (dx && (rc = ln_operand("layer_norm_bwd", "dx", dx, dx_stride, rows, C, dtype, true))) return rc;
        if (!save_mean || !save_invstd) DVAE_FAIL(DVAE_EINVAL, "layer_norm_bwd: the forward pass's statistics are missing");
        LnArgs a{};
        a.x = x; a.xs = x_stride; a.dy = dy; a.ds = dy_stride; a.y = dx; a.ys = dx_stride; a.gamma = gamma;
        a.mean = const_cast<float*>(save_mean); a.invstd = const_cast<float*>(save_invstd);
        a.partial = sums ? (float*)workspace : nullptr;
        a.left = sums ? a.partial + (size_t)groups * 2 * C : nullptr;        // behind the slabs; long rows only
        a.rows = rows; a.C = C;
        const LnShape s = ln_shape(C, dtype);
        if (dtype == DVAE_F32) ln_launch<float>(a, s, true, groups, S(st));
        else ln_launch<bf16>(a, s, true, groups, S(st));
        DVAE_CHECK_LAUNCH("layer_norm_bwd");
    }
    if (sums) {
        const int64_t g = std::min(cdiv64(2LL * C, 64), LN_REDUCE_GRID);
        hipLaunchKernelGGL(ln_reduce_kernel, dim3((unsigned)g), dim3(1024), 0, S(st), (const float*)workspace,
                           rows ? groups : 0, C, dgamma, dbeta);
        DVAE_CHECK_LAUNCH("layer_norm_bwd");
    }
    return DVAE_OK;
}

size_t dvae_newton_schulz_workspace_bytes(const dvae_matrix* mats, int count) {
    try {
        if (count < 0 || (count > 0 && !mats) || count > 65536) return 0;
        for (int i = 0; i < count; ++i)
            if (mats[i].rows <= 0 || mats[i].cols <= 0 || mats[i].rows > (1 << 30) || mats[i].cols > (1 << 30) ||
                mats[i].rows * mats[i].cols >= (1LL << 31)) return 0;
        if (ns_all_small(mats, count)) return ns_small_bytes(count);
        NsPlan p;
        return ns_plan("newton_schulz", mats, count, DVAE_MUON_SPECTRAL, p) ? 0 : p.bytes;
    } catch (...) {
        return 0;
    }
}

int dvae_newton_schulz(const dvae_matrix* mats, int count, const double* coefficients, int steps, double eps, void* workspace,
                       size_t workspace_bytes, int dtype, void* st) {
    try {
        int rc = ns_check("newton_schulz", mats, count, dtype, false);
        if (rc) return rc;
        NsArgs g{};
        if ((rc = ns_iteration_check("newton_schulz", coefficients, steps, eps, g.rate))) return rc;
        for (int i = 0; i < count; ++i)
            if (mats[i].vector) DVAE_FAIL(DVAE_EINVAL, "newton_schulz: matrix %d is marked as a vector", i);
        if (count == 0) return DVAE_OK;
        g.ws = (char*)workspace;
        g.a = (float)coefficients[0]; g.b = (float)coefficients[1]; g.c = (float)coefficients[2];
        g.eps = eps;
        const bool small = ns_all_small(mats, count);
        if (small && (rc = ns_workspace_check("newton_schulz", workspace, workspace_bytes, ns_small_bytes(count)))) return rc;
        if (small)
            return dtype == DVAE_F32 ? ns_run_small<float, false>("newton_schulz", mats, count, DVAE_MUON_SPECTRAL, g, steps, S(st))
                                     : ns_run_small<bf16, false>("newton_schulz", mats, count, DVAE_MUON_SPECTRAL, g, steps, S(st));
        NsPlan p;
        if ((rc = ns_plan("newton_schulz", mats, count, DVAE_MUON_SPECTRAL, p))) return rc;
        if ((rc = ns_workspace_check("newton_schulz", workspace, workspace_bytes, p.bytes))) return rc;
        return dtype == DVAE_F32 ? ns_run<float, false>("newton_schulz", p, g, steps, S(st))
                                 : ns_run<bf16, false>("newton_schulz", p, g, steps, S(st));
    } catch (...) {
        DVAE_FAIL(DVAE_EINVAL, "newton_schulz: out of host memory");
    }
}

int dvae_muon_step(const dvae_matrix* mats, int count, double lr, double momentum, int nesterov, double weight_decay, int scale_rule,
                   const double* coefficients, int steps, double eps, void* workspace, size_t workspace_bytes, void* st) {
    try {
        int rc = ns_check("muon_step", mats, count, DVAE_F32, true);
        if (rc) return rc;
        NsArgs g{};
        if ((rc = ns_iteration_check("muon_step", coefficients, steps, eps, g.rate))) return rc;
        if (scale_rule != DVAE_MUON_SPECTRAL && scale_rule != DVAE_MUON_RMS) DVAE_FAIL(DVAE_EINVAL, "muon_step: scale rule %d", scale_rule);
        if (!(momentum >= 0.0 && momentum < 1.0) || !(lr >= 0.0) || !(weight_decay >= 0.0) || !isfinite(lr * weight_decay))
            DVAE_FAIL(DVAE_EINVAL, "muon_step: lr %g, momentum %g, weight decay %g", lr, momentum, weight_decay);
        if (count == 0) return DVAE_OK;
        g.ws = (char*)workspace;
        g.a = (float)coefficients[0]; g.b = (float)coefficients[1]; g.c = (float)coefficients[2];
        g.eps = eps;
        g.mu = (float)momentum; g.nu = (float)(1.0 - momentum); g.nesterov = nesterov; g.lr = (float)lr;
        g.decay = (float)(1.0 - lr * weight_decay);
        if (ns_all_small(mats, count)) {
            if ((rc = ns_workspace_check("muon_step", workspace, workspace_bytes, ns_small_bytes(count)))) return rc;
            return ns_run_small<float, true>("muon_step", mats, count, scale_rule, g, steps, S(st));
        }
        NsPlan p;
        if ((rc = ns_plan("muon_step", mats, count, scale_rule, p))) return rc;
        if ((rc = ns_workspace_check("muon_step", workspace, workspace_bytes, p.bytes))) return rc;
        return ns_run<float, true>("muon_step", p, g, steps, S(st));
    } catch (...) {
        DVAE_FAIL(DVAE_EINVAL, "muon_step: out of host memory");
    }
}

}  // extern "C"
