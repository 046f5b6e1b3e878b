// How the gradient of the gated norm cuts its rows, and the workspace that takes: host code of its own, so that it can be asked without a GPU.
#pragma once
#include "row_threads.hpp"

#include <cstddef>

namespace cf {

// Threads of a row at most: 512 of up to 256 registers, 768 of 168, 1024 of 128.  Up to H = 8192 a thread has one or two chunks.  WIDE, up to 12288: two, and the next row's operands on a
// bf16 stream without groups alone, elsewhere they spill (us without them and with: 9216, bf16 98 and 87, with groups 110 and 145; fp32 131 and 221; all of it with 1024 threads 110, 161
// and 192).  WIDEST: four, with groups two, which spill either way, if little (16384, without groups: four 98, two 113; with them 247 and 222).
enum Width { USUAL, WIDE, WIDEST };
template <bool GROUPS, Width WIDTH>
constexpr int kGradThreads = WIDTH == WIDE ? 768 : WIDTH == WIDEST && GROUPS ? 1024 : 512;

// Whether a worker takes whole groups of rows that share a gate, every workers-th one; otherwise an equal share of the rows without regard to the groups.
constexpr bool whole_groups(unsigned groups, unsigned workers) { return groups >= 8ull * workers; }

// rows of up to kTallH: one chunk a thread; up to kWideH, two; the widest as kGradThreads has it
constexpr int kTallH = 8 * kGradThreads<false, USUAL>, kUsualH = 2 * kTallH, kWideH = 16 * kGradThreads<false, WIDE>;
// Workgroups of the backward pass: eight wavefronts a CU, which all kernels have registers for (292 workgroups of seven ran in two rounds: 8192 x 7168 196 us, 134 with 256), and four
// rows each, or the shares cost more than the rows; but 256 where there are as many rows.  Many kernels have registers for twelve wavefronts, whose additional shares mostly cost
// more than they bring above H = 256.  8 and 12, us, 16.8 M elements, bf16 rows, dx as bf16:
//                          no gate         four gates                                no gate         four gates
//     H = 256            51.2   47.5      61.9   73.7            H = 1536          43.3   51.2      46.2   48.6
//     H = 512            43.4   45.1      53.1   57.7            H = 2048          43.5   46.9      50.9   49.3
//     H = 1024           44.3   46.7      53.1   56.3            H = 2048, f32     62.6   62.8      66.8   73.9
inline int gated_parts(int rows, int H) {
    const int waves = H <= kOneWaveH ? 4 : row_threads(H, H <= kTallH ? 1 : 2) / kRowWave;
    const int turns = H <= kOneWaveH ? (rows - 1) / 4 + 1 : rows;
    int parts = 256 * (waves < 8 ? 8 / waves : 1);
    parts = parts < turns / 4 ? parts : turns / 4;
    parts = parts > 256 ? parts : 256;
    return parts < turns ? parts : turns;
}
struct GradPlan {
    int parts, workers, groups;         // groups: 0 = no gate
    bool several, segments;             // several groups; some of them in several workers' rows
    unsigned share;                     // rows of a worker
    int shares;                         // threads for a column of the segments
    size_t far, bytes;
};
inline GradPlan grad_plan(int rows, int H, int gate_rows) {
    GradPlan g{};
    if (rows == 0 || H == 0) return g;
    g.parts = gated_parts(rows, H);
    g.groups = gate_rows > 0 ? (rows - 1) / gate_rows + 1 : 0;
    g.several = g.groups > 1;
    g.workers = H <= kOneWaveH ? (4 * g.parts < rows ? 4 * g.parts : rows) : g.parts;
    g.share = static_cast<unsigned>((rows - 1) / g.workers + 1);
    g.segments = g.several && !whole_groups(g.groups, g.workers);
    // a group has some workers / groups segments
    g.shares = g.workers >= 16ll * g.groups ? 32 : g.workers >= 4ll * g.groups ? 8 : 2;
    const size_t shares = 2 * static_cast<size_t>(g.parts) + (g.segments ? 2 * static_cast<size_t>(g.workers) : 0);
    const size_t threads = H > kWideH ? kGradThreads<true, WIDEST> : kGradThreads<true, WIDE>;
    g.far = g.several && H > kUsualH ? static_cast<size_t>(g.parts) * 2 * 8 * threads * sizeof(double) : 0;
    g.bytes = g.far + (shares * H + g.parts) * sizeof(float);
    return g;
}

}  // namespace cf
