// Prints the plan of the product with 4-bit weights for each "rows cols n swiglu parts" line of the input, on 256 CUs.
#include <cstdio>

#include "w4.h"

int main() {
    unsigned rows, cols, n, swiglu, parts;
    while (std::scanf("%u %u %u %u %u", &rows, &cols, &n, &swiglu, &parts) == 5) {
        const W4Plan p = w4_plan(rows, cols, n, swiglu, 256, parts);
        std::printf("%u %u %u %d %u %u %u %u %u %u\n", p.xl, p.panels, p.waves, (int)p.even, p.units, p.rounds, p.groups, p.run, p.blocks,
                    w4_rows_at_once(cols));
    }
}
