// The kernel and the split of K that 4-bit layers take: reads lines
// "<bytes of a ring element> <M> <K> <N>", writes "<kernel> <split>" for each.
#include <cstdio>

#include "q4_plan.cuh"

int main()
{
    int elem, M, K, N;
    while (std::scanf("%d %d %d %d", &elem, &M, &K, &N) == 4) {
        const ddg::Q4Plan p = ddg::q4_plan(elem, M, K, N);
        std::printf("%d %d\n", p.kernel, p.split);
    }
    return 0;
}
