// hx_f8_plan.hpp -- which kernel of hx_f8.hip takes a call of the 8-bit linear or its gated pair, its parts of K and its workspace.  Host code
// only, of plain C++.
#pragma once
#include <algorithm>
#include <cstddef>

namespace hx {

constexpr int F8_BLOCK = 128;
constexpr int F8_ROWS = 8, F8_ROWS_THREADS = 1024;  // most rows of f8_rows_kernel; its workgroup

// LDS of f8_rows_kernel where x stays in it: rows of codes, whole KB, then the scales of all rows, [block][8].
constexpr int f8_far_row(int K) { return (K + 1023) / 1024 * 1024; }
constexpr int f8_far_blocks(int kb) { return (kb + 31) / 32 * 32; }  // whole rounds of 16 spans: zeros behind K
inline size_t f8_far_bytes(int M, int K) { return (size_t)M * f8_far_row(K) + f8_far_blocks((K + F8_BLOCK - 1) / F8_BLOCK) * F8_ROWS * sizeof(float); }

// Which kernel takes a call, and the parts of K.
struct F8Plan {
    enum Kind { ROWS, TILE64x32, TILE64x64, TILE128x64, TILE128x128, TILE256x32, TILE256x64, TILE256x256, NONE } kind;
    int splits, steps;
    long tiles;
    size_t partial, products;  // bytes of workspace
};
enum F8Sums { F8_FAST, F8_EXACT, F8_GATED };  // fp16 outputs; fp32 outputs, few rows, and where asked for; gated pair (exact)
constexpr int F8_CUS = 256, F8_COUNTERS = 16 * 1024;  // arrivals, at the start of a workspace
constexpr size_t F8_MOST_PRODUCTS = 48u << 20;
constexpr size_t F8_FAR_BYTES = (160 - 20) * 1024;  // next to the rows kernel's sums
constexpr int F8_NEAR = 2 * F8_ROWS_THREADS / 64;  // blocks of K whose spans are one round of the rows kernel's waves
constexpr long F8_MOST_TILES = 1l << 22;  // of at most 512 threads

// A tile, how many of its workgroups a CU holds, and what it costs, in us: to begin and end; a step of a workgroup at least; a step of each
// workgroup on a CU; where K is split, for the join and for each part of it, beside .36 us for each MB of sums.  Fitted to some 400 calls of fp16
// outputs, 240 of fp32 outputs and 480 of the gated pair (12 to 1500 rows, K and N 2048 to 12288), the model is within 5 % rms there, and its
// choice takes 1 % longer than the best of the tiles and splits on average, 10 % at most.  Beyond, 45 to 8000 rows with N from 2048 to 24576: from K = 2048 on
// at most 3 % longer, also over several rounds of tiles; at K = 1024 1 % on average and 13 % at most, at 512 4 and 30 %, at 128 13 and 46 % (2000 rows of
// 128 -> 8192, gated: 256 x 64 44.7 us, 256 x 256 30.7).  There `start`, charged once, is most of a call, and where tiles go in several rounds the times
// themselves are too low (8000 rows of 4096 -> 4096: 106 us, 143 to 150 measured).  (45 rows of 8192 -> 4096: 64 x 64 in 4 parts 12.9 us, in 2 parts
// 18.2, 128 x 64 in 8 parts 14.7; 1000 rows of 4096 -> 4096: 128 x 128 25.7, 64 x 64 38.8, 256 x 256 55.7.)
struct F8Tile {
    int bn, bm, resident;
    float start, step, each, join, part;
};
constexpr F8Tile F8_TILES[3][8] = {
    {{}, {64, 32, 4, 2.2f, 0.38f, 0.26f, 1.8f, 0.31f}, {64, 64, 3, 2.7f, 0.413f, 0.29f, 0.95f, 0.445f}, {128, 64, 2, 3.4f, 0.52f, 0.435f, 0.65f, 0.66f},
     {128, 128, 1, 3.9f, 0.65f, 0.66f, 0.f, 0.61f}, {}, {}, {256, 256, 1, 10.9f, 1.49f, 1.49f, 0.f, 0.f}},
    // exact, 128 x 128 is at most 3 % before 128 x 64
    {{}, {64, 32, 4, 3.1f, 0.43f, 0.292f, 1.65f, 0.2f}, {64, 64, 3, 3.2f, 0.552f, 0.37f, 0.93f, 0.38f}, {128, 64, 2, 4.25f, 0.80f, 0.596f, 0.2f, 0.62f},
     {}, {}, {}, {256, 256, 1, 9.6f, 2.94f, 2.94f, 0.f, 0.f}},
    // with the scaling; tiles of whole blocks of outputs do without products in memory (20 rows of 4096 -> 12288: 256 x 32 24.3 us, 64 x 32 26.7; 45
    // rows: 256 x 64 28.8, 64 x 64 30.3)
    {{}, {64, 32, 4, 6.2f, 0.446f, 0.333f, 0.93f, 0.16f}, {64, 64, 3, 7.4f, 0.543f, 0.39f, 0.62f, 0.16f}, {128, 64, 2, 7.2f, 0.867f, 0.649f, 0.1f, 0.56f},
     {}, {256, 32, 1, 4.5f, 1.0f, 1.0f, 0.94f, 0.65f}, {256, 64, 1, 6.0f, 1.17f, 1.17f, 0.46f, 0.5f}, {256, 256, 1, 11.6f, 2.9f, 2.9f, 0.f, 0.f}}};

inline F8Plan f8_plan(int M, int N, int K, F8Sums sums, bool split)
{
    F8Plan p{};
    const bool pair = sums == F8_GATED;
    const long nb = ((long)N + F8_BLOCK - 1) / F8_BLOCK;
    const int kb = (K + F8_BLOCK - 1) / F8_BLOCK;
    const size_t few = (size_t)nb * F8_ROWS * F8_BLOCK * sizeof(float);
    p.splits = 1;
    p.steps = kb;
    const bool fits = !(pair && (nb > F8_COUNTERS || few > F8_MOST_PRODUCTS)) && (kb <= F8_NEAR || f8_far_bytes(M, K) <= F8_FAR_BYTES);
    if (M <= F8_ROWS && fits) {
        p.kind = F8Plan::ROWS;
        if (pair) p.products = few;
        return p;
    }
    float least = 0.0f;
    p.kind = F8Plan::NONE;
    for (int kind = F8Plan::TILE64x32; kind <= F8Plan::TILE256x256; ++kind) {
        const F8Tile& t = F8_TILES[sums][kind];
        if (!t.bn) continue;
        const long mt = ((long)M + t.bm - 1) / t.bm, tiles = mt * (((long)N * (pair ? 2 : 1) + t.bn - 1) / t.bn);
        if (tiles > F8_MOST_TILES) continue;
        const bool whole = !pair || t.bn == 2 * F8_BLOCK;  // no blocks of outputs in parts, to be scaled later
        const size_t products = whole ? 0 : (size_t)(mt * nb) * t.bm * F8_BLOCK * sizeof(float);
        if (!whole && (tiles + mt * nb > F8_COUNTERS || products > F8_MOST_PRODUCTS)) continue;
        for (int s = 1; s <= 8; s *= 2) {
            const int steps = (kb + s - 1) / s;
            if (s > 1 && (!split || t.part == 0.f || steps < 4 || tiles * s > (long)F8_CUS * t.resident)) break;  // all are at work at once
            const float each = (float)((tiles * s + F8_CUS - 1) / F8_CUS);
            const float sums_mb = (float)(tiles * s * t.bn * std::min(t.bm, (M + 15) / 16 * 16)) * 4e-6f;
            const float join = s > 1 ? t.join + t.part * s + 0.36f * sums_mb : 0.0f;
            const float us = t.start + steps * std::max(t.step, each * t.each) + join;
            if (p.kind != F8Plan::NONE && us >= least) continue;
            least = us;
            p.kind = (F8Plan::Kind)kind;
            p.tiles = tiles;
            p.steps = steps;
            p.splits = (kb + steps - 1) / steps;
            p.partial = p.splits > 1 ? (size_t)tiles * p.splits * t.bn * t.bm * sizeof(float) : 0;
            p.products = products;
        }
    }
    return p;
}

inline size_t f8_workspace(const F8Plan& p) { return p.partial || p.products ? F8_COUNTERS * sizeof(int) + p.partial + p.products : 0; }

// Rows of a launch, a multiple of 256: 2^22 tiles of 256 x 256.
inline int f8_most_rows(int N, bool pair)
{
    const long columns = ((long)N * (pair ? 2 : 1) + 255) / 256, rows = F8_MOST_TILES / columns;  // columns <= 2^21
    return 256 * (int)std::min(rows, 1l << 22);
}

// Of the launches that a call is made of.
inline size_t f8_call_workspace(int M, int N, int K, F8Sums sums)
{
    const int most = f8_most_rows(N, sums == F8_GATED);
    size_t need = f8_workspace(f8_plan(M < most ? M : most, N, K, sums, true));
    if (M > most && M % most) {
        const size_t last = f8_workspace(f8_plan(M % most, N, K, sums, true));
        if (last > need) need = last;
    }
    return need;
}

}  // namespace hx
