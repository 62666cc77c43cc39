// Which kernel and tile of fc_q4.cu a 4-bit layer of M x K x N takes: host
// arithmetic only (tests/q4_plan_check.cpp lists what the tests' sizes take).
#pragma once
#include <cstdint>

namespace ddg {

constexpr int Q4_MAX_K = 8 * 32768;     // a cluster of eight CTAs along K
constexpr int QT_MAX_K = Q4_MAX_K / 8;  // k per CTA: a column's sum, 2 * 255^2 * K, stays below 2^32

// ------------------------------------------------------------------ CUDA cores

constexpr int Q4_THREADS = 256, GV_WARPS = Q4_THREADS / 32;
constexpr int gv_outputs(int elem) { return elem == 4 ? 4 : 2; }  // per lane group and pass (registers: P limb sums each)
constexpr uint64_t GV_SMEM_MAX = 96 * 1024;

// units of 32 k; a group of L lanes takes one unit each, KS warps of the CTA split the units
struct GvGeom {
    int U, L, nseg, KS, slots, blocks;
};

inline GvGeom gv_geom(int K, int N, int R)
{
    GvGeom g;
    g.U = (K + 31) / 32;
    g.L = 1;
    while (g.L < 32 && g.L < g.U) g.L *= 2;
    g.nseg = (g.U + g.L - 1) / g.L;
    auto slots = [&](int ks) { return GV_WARPS / ks * (32 / g.L); };
    auto blocks = [&](int ks) { return int((int64_t(N) + slots(ks) * R - 1) / (slots(ks) * R)); };
    g.KS = 1;  // as many as leave one round of two CTAs an SM
    while (2 * g.KS <= GV_WARPS && g.KS < g.nseg && blocks(2 * g.KS) <= 2 * 148) g.KS *= 2;
    g.slots = slots(g.KS), g.blocks = blocks(g.KS);
    return g;
}

inline uint64_t gv_smem(const GvGeom &g, int rows, int elem)
{
    return uint64_t(rows) * g.U * (32 * elem + elem) + uint64_t(GV_WARPS) * 32 * gv_outputs(elem) * rows * elem;
}

// ------------------------------------------------------------------ tensor cores

// CTAs of a cluster that K is split over: while that leaves every CTA resident
// at once and two stages each, and for as long as a CTA's sums need it.
// Clusters of four: of eight, only 15 fit the device at a time (256 CTAs of a
// 4 x 4096 x 4096 product took three rounds).
inline int qt_split(int kc, int na, int K, int64_t ctas)
{
    int split = 1;
    while (na == 1 && split < 4 && ctas * split * 2 <= 148 && K >= 4 * kc * split) split *= 2;
    while (na == 1 && split < 8 && int64_t(K) > int64_t(QT_MAX_K) * split) split *= 2;
    return split;
}

// rows over Z_2^32 (half as many over Z_2^64), 128-output weight tiles, k per stage, us per 64 k
struct Q4Tile {
    int rows, na, kc;
    double us;
};
constexpr int Q4_TILES = 6;
constexpr Q4Tile Q4_TILE[Q4_TILES] = {{4, 1, 128, 0.22},  {8, 1, 128, 0.24}, {16, 1, 128, 0.28},
                                      {32, 1, 128, 0.42}, {64, 1, 64, 0.70}, {64, 2, 64, 0.90}};

// kernel: the index of a tile, or
constexpr int Q4_NONE = -1, Q4_GEMV = -2, Q4_EMPTY = -3;
struct Q4Plan {
    int kernel, split;  // split: CTAs along K
};

// elem: bytes of a ring element
inline Q4Plan q4_plan(int elem, int M, int K, int N)
{
    if (K == 0) return {Q4_EMPTY, 1};
    // The CUDA cores for one row over Z_2^32, for one over Z_2^64 (twice the limb products) up to 4096 x 4096, for two
    // of half that.  In us with the weights in L2 (from memory), CUDA cores against tensor cores: over Z_2^32
    // 1 x 1024 x 1024 4.1 (4.3) against 5.4 (5.4), 1 x 8192 x 8192 18.0 (21.6) against 22.2 (26.0), 2 x 2048 x 2048
    // 5.7 (7.1) against 6.8 (7.8), 2 x 4096 x 4096 10.5 (12.3) against 9.2 (10.9); over Z_2^64 1 x 4096 x 4096 10.6
    // (12.7) against 10.7 (11.7), 1 x 4096 x 8192 16.7 (19.9) against 15.9 (17.0), 2 x 2048 x 2048 7.6 (8.6) against
    // 7.8 (8.7).  The work alone decides, so one row of a wide, short layer over Z_2^64 is on the slower side:
    // 1 x 1024 x 16384 11.2 (14.4) against 9.7 (10.9).
    const uint64_t macs = uint64_t(M) * uint64_t(K) * uint64_t(N);
    const uint64_t most = M == 2 ? 1u << 26 : elem == 8 ? 1u << 27 : ~0ull;
    if (M <= 2 && macs * unsigned(elem) <= most && gv_smem(gv_geom(K, N, gv_outputs(elem)), M, elem) <= GV_SMEM_MAX)
        return {Q4_GEMV, 1};
    // The tile of least estimated time.  Wide tiles expand the weights fewer times
    // and split x for more outputs, narrow ones spread a small product over more
    // SMs: 256 x 1024 x 512 takes 7.4 us in tiles of 32 rows and 9.6 in tiles of
    // 64; 256 x 4096 x 8192 takes 93 us in tiles of 64 rows by 128 outputs and 58
    // by 256.  Stage times (us per 64 k) are fits to such measurements, with rows of x
    // on 16-byte boundaries; off them the copies of x add to every stage (256 x
    // 1004 x 4096 takes 19.7 us and 256 x 1003 x 4096 26.9).
    Q4Plan best = {Q4_NONE, 1};
    double least = 0;
    for (int i = 0; i < Q4_TILES; i++) {
        const Q4Tile &t = Q4_TILE[i];
        const int mt = t.rows * 4 / elem;
        const int64_t down = (int64_t(M) + mt - 1) / mt;
        const int64_t ctas = (int64_t(N) + t.na * 128 - 1) / (t.na * 128) * down;
        const int split = qt_split(t.kc, t.na, K, ctas);
        const double rounds = double((ctas * split + 147) / 148);
        const double us = rounds * (2.0 + t.us * double((K + 63) / 64) / split);
        const bool fits = (int64_t(K) + split - 1) / split <= QT_MAX_K && down <= 65535;
        if (fits && (best.kernel == Q4_NONE || us < least)) best = {i, split}, least = us;
    }
    return best;
}

}  // namespace ddg
