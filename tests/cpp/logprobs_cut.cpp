// Prints how the rows of each "rows vocab top bf16" line of the input are cut.
#include <cstdio>

#include "logprobs.h"

int main() {
    unsigned rows, vocab, top, bf16;
    while (std::scanf("%u %u %u %u", &rows, &vocab, &top, &bf16) == 4) {
        const LogprobsCut c = logprobs_cut(rows, vocab, top, bf16);
        std::printf("%u %u %u %u %u %u %u %llu\n", c.threads, c.each, c.count, c.length, c.join, c.at_once, logprobs_in_groups(c.threads),
                    (unsigned long long)logprobs_most_slices(rows, vocab, top, bf16));
    }
}
