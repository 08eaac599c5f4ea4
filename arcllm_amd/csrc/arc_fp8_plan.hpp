// arc_fp8_plan.hpp -- which kernel takes an 8-bit product, its tiles and their parts, and the workspace that this
// needs.  Host code without HIP.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>

namespace arc {

constexpr uint32_t kFpBlock = 128;  // columns, and rows of weights, to a scale

// Which kernel takes a product, its tiles, and into how many parts their blocks are cut: what is expected to be quickest.
// A block costs a workgroup `one` us where it has a compute unit to itself, `two` where two share one; the last round may be
// short; beginning and end of a tile cost about 4 blocks; k_fp8_join 3 us and the sums' way there and back at 6 TB/s.  The
// constants come from products of 28 and 148 blocks, 24 to 4096 rows.  Expected times are from a third below those measured with weights
// from memory (8 blocks; 45 rows of 3584 x 18944) to a sixth or, in fp32, a quarter above (4096 rows).  What the choice has
// to tell apart, so measured, bf16: 3584 x 18944, 2048 rows, tiles of 128 183 us, of 256 in two parts 165; 1024 rows,
// tiles of 128 in one and two parts 145 and 113, of 256 in four 101; 4608 x 3584, 4096 rows, tiles of 128 105, of 256 108; 2048
// rows 71 and 64.
enum class Fp8Form { few, own, rows32, rows64, rows128, deep128, deep256 };
struct Fp8Plan {
    Fp8Form form;
    uint32_t mtiles, ntiles, splits;
    size_t bytes;  // of workspace
};
struct Fp8Tiles {
    Fp8Form form;
    uint32_t bm, bn;
    float one, two;  // deep256: alone on its compute unit; of few workgroups, of a full card
};
inline Fp8Plan fp8_plan_of(uint32_t N, uint32_t K, uint32_t M, bool gated, bool fast)
{
    Fp8Plan best{Fp8Form::few, 0, 0, 1, 256};
    // few rows: from about 6 on k_fp8_own reads them more cheaply where its workgroups come in one turn, and where they come in
    // many does not.  6, 8 and 16 rows with weights from memory, k_fp8_own and k_fp8_few, us: 3584 x 18944 18.0 and 19.1, 18.1 and
    // 19.3, 18.7 and 20.5; 4608 x 3584 8.3 and 7.9, 8.5 and 8.3, 9.1 and 9.9; 152064 x 3584 135 and 108, 139 and 117, 152
    // and 142.  The border stands high: at 18944 outputs 20.1 and 17.0, 20.5 and 18.0, 22.1 and 21.7, at 32768 31.7 and
    // 26.6, 32.4 and 28.2, 35.2 and 34.1
    if (M <= 16) {
        if (M >= 6 && N <= 32768) best.form = Fp8Form::own;
        return best;
    }
    float least = INFINITY;
    auto tiles = [](uint32_t n, uint32_t each) { return (n + each - 1) / each; };
    const uint32_t blocks = tiles(K, kFpBlock);
    const Fp8Tiles rows32{Fp8Form::rows32, 32, 128, fast ? 0.60f : 0.80f, fast ? 0.90f : 1.10f};
    const Fp8Tiles rows64{Fp8Form::rows64, 64, 128, fast ? 0.63f : 0.92f, fast ? 0.97f : 1.25f};
    const Fp8Tiles rows128{Fp8Form::rows128, 128, 128, fast ? 1.0f : 1.25f, fast ? 1.6f : 2.1f};
    const Fp8Tiles deep128{Fp8Form::deep128, 128, 128, 0.75f, 1.25f}, deep256{Fp8Form::deep256, 256, 256, 1.45f, 1.95f};
    const bool deep = fast && K % kFpBlock == 0;
    if (M <= 64) {
        // k_fp8_own, one workgroup to a compute unit: 2.5 us to begin and end, between them its copies, 1 KB each, or the weights
        // that all of them read at 5.2 TB/s
        const uint32_t copies = 2 * tiles(M, 16) + (gated ? 4 : 2);
        const float each = (fast ? 0.0105f : 0.0125f) * (copies <= 8 ? 1.0f : 1.25f);
        least = tiles(tiles(N, 16), 256) * (2.5f + std::max(blocks * copies * each, float(K) * (gated ? 8192 : 4096) / 5.2e6f));
        best.form = Fp8Form::own;
    }
    const Fp8Tiles of[2] = {M <= 32 ? rows32 : M <= 64 ? rows64 : deep ? deep128 : rows128, deep256};
    for (const Fp8Tiles& s : of) {
        if (s.form == Fp8Form::deep256 && (!deep || M <= 64)) continue;
        const uint32_t mtiles = tiles(M, s.bm), ntiles = tiles(N, gated ? s.bn / 2 : s.bn);
        for (uint32_t splits = 1; splits <= 16 && (splits == 1 || blocks / splits >= 4); splits *= 2) {
            const double parts = double(mtiles) * ntiles * splits, share = s.form == Fp8Form::deep256 ? 256 : 512;
            const double full = std::floor(parts / share), rest = parts - full * share;
            const double last = rest == 0 ? 0 : share == 256 ? s.one + (s.two - s.one) * rest / 256 : rest <= 256 ? s.one : s.two;
            const size_t sums = splits > 1 ? size_t(parts) * s.bm * s.bn * sizeof(float) : 0;
            const float time = float((full * s.two + last) * (tiles(blocks, splits) + 4) + (splits > 1 ? 3 + sums / 3e6 : 0));
            if (time >= least) continue;
            least = time;
            best = Fp8Plan{s.form, mtiles, ntiles, splits, sums ? sums : 256};
        }
    }
    return best;
}

// The most workspace that products of up to M rows take.  Up to 64 rows a plan depends on the number of 16 rows, beyond on
// that of 128, so one of each is asked.  Of a product cut in parts the sums' way alone, bytes / 3e6 us, is less than what
// cutting can save, the tiles' last round: two * (blocks + 4) us at most (`two` <= 2.1; with some room 7e6 for
// 3e6 * 2.1).  The sums of two parts or more are 8 bytes an output, so beyond `end` rows nothing is cut.
inline size_t fp8_most_bytes(uint32_t N, uint32_t K, uint32_t M, bool gated, bool fast)
{
    const uint64_t sums = 7000000ull * ((K + kFpBlock - 1) / kFpBlock + 4);
    const uint32_t end = uint32_t(std::min<uint64_t>(M, sums / (8ull * N * (gated ? 2 : 1)) + 256));
    size_t most = fp8_plan_of(N, K, M, gated, fast).bytes;
    for (uint32_t m = 16; m < end; m += m < 64 ? 16 : m < 128 ? 64 : 128)
        most = std::max(most, fp8_plan_of(N, K, m, gated, fast).bytes);
    return most;
}

}  // namespace arc
