// Reads lines "rows outputs columns gated y16" and prints for each the kernel that takes such a product, its tiles in both
// directions, their parts, the workspace of this call and the most of up to so many rows.
#include "arc_fp8_plan.hpp"

#include <cstdio>

int main()
{
    const char* names[] = {"few", "own", "rows32", "rows64", "rows128", "deep128", "deep256"};
    unsigned m, n, k, gated, fast;
    while (std::scanf("%u %u %u %u %u", &m, &n, &k, &gated, &fast) == 5) {
        const arc::Fp8Plan p = arc::fp8_plan_of(n, k, m, gated != 0, fast != 0);
        std::printf("%s %u %u %u %zu %zu\n", names[static_cast<int>(p.form)], p.mtiles, p.ntiles, p.splits, p.bytes,
                    arc::fp8_most_bytes(n, k, m, gated != 0, fast != 0));
    }
}
