// Two host threads (two parties of one process) make their first tensor map at
// the same time.  Built with -fsanitize=thread against stand-ins of the runtime's
// calls; no device is touched.  Exit status 0 and "ok" when every map was made
// and the sanitizer saw no race.
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <thread>

#include <cuda_runtime.h>

// named by device functions that nothing here calls
inline size_t __cvta_generic_to_shared(const void *) { return 0; }
inline unsigned __byte_perm(unsigned, unsigned, unsigned) { return 0; }

#include "tma.cuh"

static std::atomic<int> maps{0}, lookups{0};

static CUresult fake_encode(CUtensorMap *map, CUtensorMapDataType, cuuint32_t rank, void *, const cuuint64_t *dims,
                            const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                            CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill)
{
    map->opaque[0] = rank == 2 ? dims[0] : 0;
    maps++;
    return CUDA_SUCCESS;
}

extern "C" cudaError_t cudaGetDriverEntryPoint(const char *, void **fn, unsigned long long,
                                               cudaDriverEntryPointQueryResult *q)
{
    lookups++;
    *fn = reinterpret_cast<void *>(&fake_encode);
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
extern "C" const char *cudaGetErrorString(cudaError_t) { return ""; }

namespace ddg {
void set_last_error(const char *, ...) {}
}  // namespace ddg

int main()
{
    std::atomic<int> ready{0}, good{0};
    auto party = [&] {
        ready++;
        while (ready < 2) {}
        for (int i = 0; i < 100; i++) {
            CUtensorMap m = {};
            if (ddg::tma_map_2d(&m, nullptr, 4, 64, 8, 256, 32, 8) == DDG_OK && m.opaque[0] == 64) good++;
        }
    };
    std::thread a(party), b(party);
    a.join(), b.join();
    const bool ok = good == 200 && maps == 200 && lookups >= 1;
    std::puts(ok ? "ok" : "failed");
    return ok ? 0 : 1;
}
