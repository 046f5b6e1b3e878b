// Which kernel runs the experts' block-scaled product, and how: host code of its own, so that the choice can be asked without a GPU.
#pragma once

namespace cf {

constexpr int kPlanEdge = 256, kPlanK = 128;            // the large tiles' edge, a K-tile
constexpr int kSlimEdge = 128, kSlimStages = 4;         // the 128 x 128 tiles', and the K-tiles that their kernel needs
constexpr int kMostExperts = 2048;                      // that the tile kernels count in LDS

// shape: the tile edge, or the number of a small-tile kernel (0: 16 x 16, 1: 32 x 32, 3: 64 x 64, 7: 32 x 64).  beside: workgroups that share the 64-row passes of an
// entry of 256 rows.
struct GroupedBlockPlan { int shape, beside; };

inline GroupedBlockPlan grouped_block_plan(int total_rows, int num_experts, int N, int K, int cus) {
    const float rows = static_cast<float>(total_rows), experts = static_cast<float>(num_experts < total_rows ? num_experts : total_rows);
    const int ktiles = K / kPlanK, columns64 = (N + 63) / 64;
    // Microseconds for rows that lie evenly (the counts are on the device; uneven ones were not part of the fit): rounds of workgroups or tiles over the CUs.  An expert has half of a tile (0.6 of a small one) more than its rows
    // fill, and one at least.  Fitted to 5200 sizes, of which 10 % run over 1.1 times the best kernel, 3 % over 1.25; some of them, us:
    //     rows  experts N x K     32 x 64  64 x 64  128 x 128  256 x 256        rows  experts N x K     32 x 64  64 x 64  128 x 128  256 x 256
    //     96    64  1408 x 2048     28.5     45       38         52             1000  16  1536 x 4096     46.3     38.8     25.9       38.5
    //     1280  64  1408 x 2048     41.3     64.9     46.8       56.0           4000  16  2048 x 7168       .      241      134        114
    //     2560  64  1408 x 2048     62.5     71.0     48.2       59.0           500    8  1024 x 2048     16.5     12.7     14.8       22.9
    //     8000  64  1408 x 2048     146      148      68.1       71.6           2000   8  1024 x 2048       .      28.6     15.9       30.4
    //     98304 64  1408 x 2048       .     1170      465        340            32768  8  1024 x 2048       .      274      114        93.4
    const auto tiles = [&](float edge, float more) { return rows / edge + more * experts > experts ? rows / edge + more * experts : experts; };
    const auto rounds = [&](float n) { const float r = n / static_cast<float>(cus); return static_cast<float>(static_cast<int>(r) + 1); };
    int shape = 3, beside = 1;      // of the small-tile kernel, or the tile edge; workgroups for the 64-row passes of an entry of 256 rows
    // Up to 24 rows an expert most have one pass of 32 x 64: their weights are read once, which is all of the time (4.6 TB/s).  Where that leaves CUs without
    // one, fewer columns and up to 36 rows (8 experts of 1024 x 2048, 200 rows: 10.1 us and 11.9), and few rows besides (12 rows, 64 experts of
    // 256 x 6144: 16 x 16 12.9, 32 x 32 13, 32 x 64 16.3; 16 rows, 2 of 512 x 4096: 9.2, 10.7, 12).
    const bool fills = experts * static_cast<float>(columns64) >= static_cast<float>(cus);
    if (rows <= (fills ? 24.0f : 36.0f) * static_cast<float>(num_experts)) {
        shape = fills ? 7 : rows <= 10.0f * experts ? 0 : 1;
    } else if (ktiles >= 3) {
        float best = 1e30f;
        // the LDS of the small-tile kernel holds the scales of 64 rows up to K = 16000
        if (ktiles >= 4 && ktiles <= 120) {
            const float passes = tiles(64.0f, 0.6f) * static_cast<float>(columns64) / static_cast<float>(cus);
            best = (passes > 0.8f ? passes + 0.5f : 1.0f) * (9.0f + static_cast<float>(ktiles) * 0.32f);
            const long long each = (static_cast<long long>(total_rows) + 64LL * num_experts - 1) / (64LL * num_experts);
            beside = each < 3 ? static_cast<int>(each) + 1 : 4;
        }
        if (ktiles >= kSlimStages && num_experts <= kMostExperts) {
            const float r = rounds(tiles(kSlimEdge, 0.5f) * static_cast<float>((N + kSlimEdge - 1) / kSlimEdge));
            const float t = (r > 1.0f ? r : 1.25f) * (static_cast<float>(ktiles) * 0.50f + 6.0f);
            if (t < best) { best = t; shape = kSlimEdge; }
        }
        if (num_experts <= kMostExperts) {
            const float t = rounds(tiles(kPlanEdge, 0.5f) * static_cast<float>((N + kPlanEdge - 1) / kPlanEdge)) * (static_cast<float>(ktiles) * 1.1f + 11.7f);
            if (t < best) shape = kPlanEdge;
        }
        if (shape == 3 && ktiles > 120) shape = 7;          // more experts than the tile kernels' LDS counts, and a long K
    }
    return {shape, shape == 3 ? beside : 1};
}

}  // namespace cf
